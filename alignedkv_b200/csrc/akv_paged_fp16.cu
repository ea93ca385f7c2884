// Attention over pages of fp16.
#include "akv_paged_attention.cuh"

namespace akv {

int launch_attend_fp16(const AttendArgs& a, const Plan& p, int D, bool joined, cudaStream_t st) {
    return D == 128 ? launch_rows<AKV_PAGE_FP16, 128>(a, p, joined, st) : launch_rows<AKV_PAGE_FP16, 64>(a, p, joined, st);
}

}  // namespace akv
