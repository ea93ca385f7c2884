// Arguments of the attention over pages, and its launchers by page format (each has a file of its own).
#pragma once
#include "akv_paged.cuh"

namespace akv {

constexpr int CHUNK = 64, TEAM_CHUNK = 32, MOST_WARPS = 16;       // (TEAM_CHUNK: where a cluster has a unit to itself; a step where that is more)

// Warps of a CTA for units of 8 nt rows.  As many as have room for their sums and queries: 12 at 168 registers each, 8 at 255.  (16 rows of 128 channels in
// 12 warps spill 64 to 296 bytes; 32 x 8 heads x up to 4096 tokens, 12 rows: fp16 68.6 us, in 8 warps 57.5, e4m3 56.2 and 41.5, e2m1 46.3 and 43.7.
// 24 rows of 64 channels do with them in 8 and 4 bits: 20 rows, e4m3 40.2 us in 8 warps, 39.2 in 12, e2m1 41.4 and 39.7.)  One tile of
// 4-bit rows of 128 channels is bound by the instructions that unpack them: 16 (8 heads x 131072 tokens 43.9 us, 12 warps 45.5).  Spilled for all that, as
// ptxas says: one tile of 128 channels up to 24 bytes, two and three of 64 up to 32, four of 128 28 to 208.
constexpr int warps_of(int format, int D, int nt) {
    if (format == AKV_PAGE_E2M1 && D == 128 && nt == 1) return 16;
    return nt == 1 || (D == 64 && (nt == 2 || (nt == 3 && format != AKV_PAGE_FP16))) ? 12 : 8;
}

struct AttendArgs {
    Pool pool;
    const __half* q;
    __half* out;
    float *lse, *part;              // part: two records of each CTA, one of each warp, a border of each CTA
    int B, T, G, groups, rows, ctas, record, team, over_g;    // record: floats of one; team: CTAs of a cluster that has a unit to itself, or 0; over_g: 2^16 / G, rounded up
    // groups: units per (sequence, KV head); rows: query rows of a unit
    float scale2;                   // scale * log2(e)
};

// Rows of a unit in groups of 8 (nt), CTAs, workspace.
struct Plan {
    int nt, groups, rows, ctas, team;
    long long bytes;
};

// joined: units may be shared by CTAs.
int launch_attend_fp16(const AttendArgs& a, const Plan& p, int D, bool joined, cudaStream_t st);
int launch_attend_e4m3(const AttendArgs& a, const Plan& p, int D, bool joined, cudaStream_t st);
int launch_attend_e2m1(const AttendArgs& a, const Plan& p, int D, bool joined, cudaStream_t st);

}  // namespace akv
