// Attention over pages of e4m3.
#include "akv_paged_attention.cuh"

namespace akv {

int launch_attend_e4m3(const AttendArgs& a, const Plan& p, int D, bool joined, cudaStream_t st) {
    return D == 128 ? launch_rows<AKV_PAGE_E4M3, 128>(a, p, joined, st) : launch_rows<AKV_PAGE_E4M3, 64>(a, p, joined, st);
}

}  // namespace akv
