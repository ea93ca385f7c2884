// Attention of the newest tokens of each sequence over its pages: arguments, plan, entries.
#include "akv_paged_attention.h"

namespace akv {
namespace {

constexpr float LOG2E = 1.4426950408889634f;

long long chunks_of_table(const akv_pool* pool, int width, int chunk) { return ((long long)width * pool->page_size + chunk - 1) / chunk; }

// CTAs of a cluster per unit, where that is better than equal runs over all SMs, or 0.  A cluster joins its records itself, without a second
// kernel and without adding up lengths; but its SMs are a power of two per unit, all of them wait for the longest sequence, and not all SMs can be in
// clusters of one size.  So: where units leave SMs idle, and the longest sequence that the table can hold gives a warp few chunks.  No more CTAs than
// leave half of the warps without a chunk.
int team_of(long long units, long long most_chunks, int sms, int warps) {
    int team = 8;
    while (team > 1 && (units * team > sms * 3 / 4 || (team / 2) * warps >= 2 * most_chunks)) team /= 2;
    return units * team > sms || most_chunks > 8ll * warps * team ? 0 : team;
}

// Rows of a unit: as many as it takes, so that codes are unpacked once for all of them; but 8 where that still leaves a warp two chunks or fewer, since the
// time is then one warp's over all its rows (20 sequences of 42 tokens, 32 rows: 6.2 us, in units of 32 11.5).
Plan plan_of(int rows, const akv_pool* pool, int bsz, int width) {
    Plan p;
    const int D = pool->head_dim, eights = (rows + 7) / 8;
    const long long heads = (long long)bsz * pool->n_kv_heads;
    p.ctas = sm_count();
    p.groups = heads * eights * chunks_of_table(pool, width, CHUNK) <= 2ll * p.ctas * MOST_WARPS ? eights : (rows + 31) / 32;
    p.rows = (rows + p.groups - 1) / p.groups;
    p.nt = (p.rows + 7) / 8;
    p.team = team_of(heads * p.groups, chunks_of_table(pool, width, TEAM_CHUNK), p.ctas,
                     warps_of(pool->format, D, p.nt));
    p.bytes = p.team ? 0 : (2ll + MOST_WARPS) * p.ctas * 8 * p.nt * (D + 4) * 4 + 8ll * p.ctas;
    return p;
}

}  // namespace
}  // namespace akv

using namespace akv;

extern "C" {

long long akv_paged_scratch_bytes(const akv_pool* pool, int bsz, int width, int group, int tokens) {
    if (!pool || bsz <= 0 || width <= 0 || group <= 0 || tokens <= 0 || group > 64 || tokens > 64 || group * tokens > 64 ||
        (pool->head_dim != 64 && pool->head_dim != 128))
        return -1;
    return plan_of(group * tokens, pool, bsz, width).bytes;
}

int akv_paged_attention(const akv_pool* pool, const void* q, const void* pages, const void* lens, void* out, void* lse, void* scratch,
                        long long scratch_bytes, int bsz, int width, int group, int tokens, float scale, void* stream) {
    set_error("");
    AttendArgs a = {};
    int rc = fill_pool("paged_attention", pool, pages, lens, bsz, width, &a.pool);
    if (rc != AKV_OK) return rc;
    AKV_REQUIRE(q && out, AKV_ERR_NULL, "paged_attention: null pointer");
    AKV_REQUIRE(group > 0 && tokens > 0 && group <= 64 && tokens <= 64 && group * tokens <= 64, AKV_ERR_SHAPE,
                "paged_attention: %d new tokens of %d query heads per KV head (at most 64 rows)", tokens, group);
    AKV_REQUIRE(aligned16(q) && aligned16(out) && aligned16(scratch) && (reinterpret_cast<uintptr_t>(lse) & 3u) == 0, AKV_ERR_ALIGN,
                "paged_attention: q, out and scratch must be 16-byte aligned, lse 4-byte");
    const int D = pool->head_dim;
    const Plan p = plan_of(group * tokens, pool, bsz, width);
    AKV_REQUIRE(scratch || p.bytes == 0, AKV_ERR_NULL, "paged_attention: null pointer");
    AKV_REQUIRE(scratch_bytes >= p.bytes, AKV_ERR_SHAPE, "paged_attention: scratch of %lld bytes is too small", scratch_bytes);
    AKV_REQUIRE((long long)pool->n_pages * pool->n_kv_heads * pool->page_size <= 1ll << 32 && (long long)bsz * width < INT_MAX, AKV_ERR_OVERFLOW,
                "paged_attention: a pool of more than 2^32 rows");
    AKV_REQUIRE((long long)bsz * tokens * pool->n_kv_heads * group < INT_MAX / 256, AKV_ERR_OVERFLOW, "paged_attention: too many query rows");
    const long long most = chunks_of_table(pool, width, CHUNK) * bsz * pool->n_kv_heads * p.groups;
    AKV_REQUIRE(most < INT_MAX, AKV_ERR_OVERFLOW, "paged_attention: too many chunks of %d tokens", CHUNK);
    a.q = static_cast<const __half*>(q);
    a.out = static_cast<__half*>(out);
    a.lse = static_cast<float*>(lse);
    a.part = static_cast<float*>(scratch);
    a.B = bsz;
    a.T = tokens;
    a.G = group;
    a.over_g = (65536 + group - 1) / group;
    a.groups = p.groups;
    a.rows = p.rows;
    a.ctas = p.ctas;
    a.record = 8 * p.nt * (D + 4);
    a.scale2 = scale * LOG2E;
    a.team = p.team;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool joined = (long long)width * pool->page_size > CHUNK;      // (units of one chunk are nobody else's)
    if (pool->format == AKV_PAGE_FP16) return launch_attend_fp16(a, p, D, joined, st);
    if (pool->format == AKV_PAGE_E4M3) return launch_attend_e4m3(a, p, D, joined, st);
    return launch_attend_e2m1(a, p, D, joined, st);
}

}  // extern "C"
