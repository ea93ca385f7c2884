// Attention over pages of e2m1.
#include "akv_paged_attention.cuh"

namespace akv {

int launch_attend_e2m1(const AttendArgs& a, const Plan& p, int D, bool joined, cudaStream_t st) {
    return D == 128 ? launch_rows<AKV_PAGE_E2M1, 128>(a, p, joined, st) : launch_rows<AKV_PAGE_E2M1, 64>(a, p, joined, st);
}

}  // namespace akv
