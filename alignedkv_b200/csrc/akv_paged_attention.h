// Arguments of the attention over pages, and its launchers by page format (each has a file of its own).
#pragma once
#include "akv_paged.cuh"

namespace akv {

constexpr int CHUNK = 64, TEAM_CHUNK = 32, MOST_WARPS = 16;       // (TEAM_CHUNK: where a cluster has a unit to itself; a step where that is more)

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
