// What enters and leaves the plane cache beside the decode step.
//   commit_kernel    the accepted path of a tree of drafted tokens: the state that one append after the other leaves
//   select_kernel    per (batch, KV head): the `keep` heaviest plane tokens, and with them who moves where
//   move_kernel      survivors behind `keep` into the places that became free in front of it
//   clear_kernel     K nibble planes, weights behind the survivors
#include <limits.h>

#include "akv_save.cuh"

namespace akv {
namespace {

constexpr int BLK = 64;

// ------------------------------------------------------------------ accepted path
// CTA = (batch, KV head) and one of K, V.  Rows in front of the accepted tokens: the residual buffer.  The two together are at most
// 127 rows: one block fills up at most, its rows go to the planes, and the rows behind it begin the next residual block.
__global__ void __launch_bounds__(256)
commit_kernel(uint8_t* __restrict__ f8, uint8_t* __restrict__ m4, uint8_t* __restrict__ l4, uint8_t* __restrict__ vf8,
              uint8_t* __restrict__ vm4, uint8_t* __restrict__ vl4, uint16_t* __restrict__ k_exp, uint16_t* __restrict__ v_exp,
              uint8_t* restk, uint8_t* restv, const uint8_t* __restrict__ kd, const uint8_t* __restrict__ vd,
              const int* __restrict__ path, int H, int D, int T, int n, int rest, int qn, int nmb, int L) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int node[BLK];
    pdl_enter();
    const int bh = blockIdx.x, b = bh / H, h = bh - b * H, tid = threadIdx.x;
    const bool value = blockIdx.y;
    uint8_t* buffer = value ? restv : restk;
    const uint8_t* drafted = value ? vd : kd;
    if (tid < n) node[tid] = min(max(path[(size_t)b * n + tid], 0), T - 1);
    __syncthreads();
    const size_t pitch = 2 * (size_t)D;
    auto slot = [&](int i) { return buffer + (((size_t)b * BLK + i) * H + h) * pitch; };
    auto fresh = [&](int i) { return drafted + (((size_t)b * T + node[i]) * H + h) * pitch; };
    // exponent maxima, two channels a word
    uint16_t* top = (value ? v_exp : k_exp) + (size_t)bh * (D >> 1);
    for (int c = tid; c < (D >> 1); c += blockDim.x) {
        uint32_t m = top[c];
        for (int i = 0; i < n; ++i) {
            const uint32_t w = reinterpret_cast<const uint32_t*>(fresh(i))[c];
            m = __vmaxu4(m, ((w >> 10) & 0x1Fu) | (((w >> 26) & 0x1Fu) << 8));
        }
        top[c] = (uint16_t)m;
    }
    int done = 0, at = rest;                           // accepted tokens that have gone, row of the next
    if (rest + n >= BLK) {
        auto row = [&](int i) { return i < rest ? static_cast<const uint8_t*>(slot(i)) : fresh(i - rest); };
        // (rows of the residual buffer are read and, further down, written: no read-only loads)
        const int vec = (int)(pitch >> 4);
        for (int i = tid; i < BLK * vec; i += blockDim.x) {
            const int r = i / vec, v = i - r * vec;
            reinterpret_cast<uint4*>(smem + r * pitch)[v] = reinterpret_cast<const uint4*>(row(r))[v];
        }
        __syncthreads();
        if (!value) {
            k_emit_block64<false, true>(smem, f8, m4, l4, (long long)bh * nmb + qn / BLK, D, nullptr);
        } else {
            const int per = D >> 5;
            for (int i = tid; i < BLK * per; i += blockDim.x) {
                const int r = i / per, c = i - r * per;
                const uint4* src = reinterpret_cast<const uint4*>(smem + r * pitch + c * 64);
                const size_t to = (size_t)bh * L + qn + r;
                v_write32(src[0], src[1], src[2], src[3], vf8 + to * D + c * 32, vm4 + to * (D >> 1) + c * 16,
                          vl4 + to * (D >> 1) + c * 16);
            }
        }
        done = BLK - rest;
        at = 0;
    }
    const int vec = (int)(pitch >> 4);
    for (int i = tid; i < (n - done) * vec; i += blockDim.x) {
        const int r = i / vec, v = i - r * vec;
        reinterpret_cast<uint4*>(slot(at + r))[v] = reinterpret_cast<const uint4*>(fresh(done + r))[v];
    }
}

// ------------------------------------------------------------------ eviction
// A weight as an unsigned key of the same order: NaN above infinity, -0 equal to +0; a protected token above all.
__device__ __forceinline__ uint32_t key_of(float w, bool safe) {
    if (safe) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(w + 0.f);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFEu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct EvictArgs {
    float* weights;
    int* positions;
    uint8_t *k8, *km, *kl, *v8, *vm, *vl;
    int *holes, *movers, *count;       // [rows][most], [rows][most], [rows]
    int D, L, nmb, n, rest, keep, recent, arranged, shift, most;
};

__device__ __forceinline__ int position_of(const EvictArgs& a, const int* pos, int i) { return i < a.arranged ? pos[i] : i + a.shift; }

// One CTA per row.  The keep-th largest key by four counts of eight bits; then one pass in order that numbers the free places and the
// survivors behind.
constexpr int SEL_NT = 1024;
__global__ void __launch_bounds__(SEL_NT) select_kernel(const EvictArgs a) {
    __shared__ int hist[256], warp_sum[3][SEL_NT / 32], total[3];
    __shared__ uint32_t found[2];
    pdl_enter();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const size_t row = blockIdx.x;
    const float* w = a.weights + row * a.L;
    int* pos = a.positions + row * a.L;
    const int safe_from = a.n + a.shift - a.recent;
    uint32_t prefix = 0;
    int want = a.keep;                                 // how many of the keys that share the prefix stay
    for (int bit = 24; bit >= 0; bit -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < a.n; i += SEL_NT) {
            const uint32_t k = key_of(w[i], position_of(a, pos, i) >= safe_from);
            if (bit == 24 || (k >> (bit + 8)) == (prefix >> (bit + 8))) atomicAdd(&hist[(k >> bit) & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int d = 255, above = 0;
            while (d > 0 && above + hist[d] < want) above += hist[d--];
            found[0] = d;
            found[1] = above;
        }
        __syncthreads();
        prefix |= found[0] << bit;
        want -= (int)found[1];
        __syncthreads();
    }
    int ties = 0, holes = 0, movers = 0;               // so far
    for (int i0 = 0; i0 < a.n; i0 += SEL_NT) {
        const int i = i0 + tid;
        const uint32_t k = i < a.n ? key_of(w[i], position_of(a, pos, i) >= safe_from) : 0;
        const bool tie = i < a.n && k == prefix;
        const uint32_t below = (1u << lane) - 1;
        const uint32_t tb = __ballot_sync(0xFFFFFFFFu, tie);
        if (lane == 0) warp_sum[0][warp] = __popc(tb);
        __syncthreads();
        int before = ties;
        for (int j = 0; j < warp; ++j) before += warp_sum[0][j];
        const bool stays = i < a.n && (k > prefix || (tie && before + __popc(tb & below) < want));
        const bool hole = i < a.keep && !stays, mover = stays && i >= a.keep;
        const uint32_t hb = __ballot_sync(0xFFFFFFFFu, hole), mb = __ballot_sync(0xFFFFFFFFu, mover);
        if (lane == 0) {
            warp_sum[1][warp] = __popc(hb);
            warp_sum[2][warp] = __popc(mb);
        }
        __syncthreads();
        int h = holes, m = movers;
        for (int j = 0; j < warp; ++j) {
            h += warp_sum[1][j];
            m += warp_sum[2][j];
        }
        if (hole) a.holes[row * a.most + h + __popc(hb & below)] = i;
        if (mover) a.movers[row * a.most + m + __popc(mb & below)] = i;
        if (stays && i < a.keep && i >= a.arranged) pos[i] = i + a.shift;
        if (tid < 3) {
            int s = 0;
            for (int j = 0; j < SEL_NT / 32; ++j) s += warp_sum[tid][j];
            total[tid] = s;
        }
        __syncthreads();
        ties += total[0];
        holes += total[1];
        movers += total[2];
        __syncthreads();
    }
    if (tid == 0) a.count[row] = movers;
}

// Index of the first free place that is not below `slot`.
__device__ __forceinline__ int first_hole(const int* holes, int count, int slot) {
    int lo = 0, hi = count;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (holes[mid] < slot) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// CTA = one block of 64 places in front of `keep`: its free places take the survivors of the same numbers.  Survivors are read
// only behind `keep` and places are written only in front of it, each by its own CTA: no order among the CTAs.
__global__ void __launch_bounds__(256) move_kernel(const EvictArgs a) {
    extern __shared__ __align__(16) uint8_t tile[];     // K: [D][64] high bytes, [D][32] twice
    __shared__ int src[BLK], dst[BLK];
    pdl_enter();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = a.D;
    const size_t row = blockIdx.x;
    const int blk = blockIdx.y;
    const int count = a.count[row];
    const int *holes = a.holes + row * a.most, *movers = a.movers + row * a.most;
    const int i0 = first_hole(holes, count, blk * BLK), i1 = first_hole(holes, count, blk * BLK + BLK), m = i1 - i0;
    if (m == 0) return;
    if (tid < m) {
        const int d = holes[i0 + tid], s = movers[i0 + tid];
        dst[tid] = d - blk * BLK;
        src[tid] = s;
        a.weights[row * a.L + d] = a.weights[row * a.L + s];
        a.positions[row * a.L + d] = position_of(a, a.positions + row * a.L, s);
    }
    const size_t t0 = row * a.nmb * D;                  // rows of 64 (32) bytes: [block][channel]
    const uint4 *k8 = reinterpret_cast<const uint4*>(a.k8 + (t0 + (size_t)blk * D) * 64),
                *km = reinterpret_cast<const uint4*>(a.km + (t0 + (size_t)blk * D) * 32),
                *kl = reinterpret_cast<const uint4*>(a.kl + (t0 + (size_t)blk * D) * 32);
    uint4* t4 = reinterpret_cast<uint4*>(tile);
    for (int i = tid; i < D * 8; i += 256)
        t4[i] = i < D * 4 ? k8[i] : i < D * 6 ? km[i - D * 4] : kl[i - D * 6];
    __syncthreads();
    uint8_t *tm = tile + D * 64, *tl = tm + D * 32;
    // high bytes and nibbles of one channel: a lane per free place; two places may share a nibble byte, so each nibble is
    // cleared and set with an atomic on its word
    for (int c = warp; c < D; c += 8)
        for (int j = lane; j < m; j += 32) {
            const int s = src[j], d = dst[j];
            const size_t at = t0 + (size_t)(s >> 6) * D + c;
            tile[c * 64 + d] = a.k8[at * 64 + (s & 63)];
            const int from = 4 * (1 - (s & 1)), to = 8 * ((d >> 1) & 3) + 4 * (1 - (d & 1));
            const uint32_t x = (a.km[at * 32 + ((s & 63) >> 1)] >> from) & 15u, y = (a.kl[at * 32 + ((s & 63) >> 1)] >> from) & 15u;
            unsigned* wm = reinterpret_cast<unsigned*>(tm + c * 32) + (d >> 3);
            unsigned* wl = reinterpret_cast<unsigned*>(tl + c * 32) + (d >> 3);
            atomicAnd(wm, ~(15u << to));
            atomicOr(wm, x << to);
            atomicAnd(wl, ~(15u << to));
            atomicOr(wl, y << to);
        }
    // V rows: 16 lanes per token, 16 bytes each (D = 128: 8 of high bytes, 4 of either nibble plane)
    const int per = D >> 3;
    for (int i = tid; i < m * per; i += 256) {
        const int j = i / per, v = i - j * per;
        const size_t s = row * a.L + src[j], d = row * a.L + (size_t)blk * BLK + dst[j];
        if (v < D / 16)
            reinterpret_cast<uint4*>(a.v8 + d * D)[v] = reinterpret_cast<const uint4*>(a.v8 + s * D)[v];
        else if (v < D / 16 + D / 32)
            reinterpret_cast<uint4*>(a.vm + d * (D / 2))[v - D / 16] = reinterpret_cast<const uint4*>(a.vm + s * (D / 2))[v - D / 16];
        else
            reinterpret_cast<uint4*>(a.vl + d * (D / 2))[v - D / 16 - D / 32] =
                reinterpret_cast<const uint4*>(a.vl + s * (D / 2))[v - D / 16 - D / 32];
    }
    __syncthreads();
    uint4 *o8 = reinterpret_cast<uint4*>(a.k8 + (t0 + (size_t)blk * D) * 64), *om = reinterpret_cast<uint4*>(a.km + (t0 + (size_t)blk * D) * 32),
          *ol = reinterpret_cast<uint4*>(a.kl + (t0 + (size_t)blk * D) * 32);
    for (int i = tid; i < D * 8; i += 256) {
        if (i < D * 4) o8[i] = t4[i];
        else if (i < D * 6) om[i - D * 4] = t4[i];
        else ol[i - D * 6] = t4[i];
    }
}

// blockIdx.y == 0: the weights of the residual tokens follow the survivors, zeros behind them; else: K nibble planes of a freed
// block (the K writer adds nibbles, so a block is zero before it is written again).
__global__ void __launch_bounds__(256) clear_kernel(const EvictArgs a) {
    __shared__ float tail[BLK];
    pdl_enter();
    const size_t row = blockIdx.x;
    const int tid = threadIdx.x;
    if (blockIdx.y == 0) {
        float* w = a.weights + row * a.L;
        if (tid < a.rest) tail[tid] = w[a.n + tid];
        __syncthreads();
        for (int i = a.keep + tid; i < a.n + a.rest; i += 256) w[i] = i - a.keep < a.rest ? tail[i - a.keep] : 0.f;
        return;
    }
    const size_t at = (row * a.nmb + a.keep / BLK + blockIdx.y - 1) * (size_t)a.D * 2;
    for (int i = tid; i < a.D * 2; i += 256) {
        reinterpret_cast<uint4*>(a.km)[at + i] = make_uint4(0, 0, 0, 0);
        reinterpret_cast<uint4*>(a.kl)[at + i] = make_uint4(0, 0, 0, 0);
    }
}

int check_planes(const char* fn, const akv_layer* a) {
    AKV_REQUIRE(a && a->k_first_8 && a->k_mid_4 && a->k_last_4 && a->v_first_8 && a->v_mid_4 && a->v_last_4, AKV_ERR_NULL,
                "%s: null pointer", fn);
    AKV_REQUIRE(a->bsz > 0 && a->n_kv_heads > 0 && (a->head_dim == 64 || a->head_dim == 128) && a->max_seq_len > 0 &&
                a->max_seq_len <= INT_MAX - 128, AKV_ERR_SHAPE,
                "%s: unsupported extent (bsz %d, KV heads %d, head_dim %d [64 or 128], max_seq_len %d)", fn, a->bsz, a->n_kv_heads,
                a->head_dim, a->max_seq_len);
    AKV_REQUIRE((long long)a->bsz * a->n_kv_heads < (1ll << 30), AKV_ERR_OVERFLOW, "%s: too many rows", fn);
    AKV_REQUIRE(aligned16(a->k_first_8) && aligned16(a->k_mid_4) && aligned16(a->k_last_4) && aligned16(a->v_first_8) &&
                aligned16(a->v_mid_4) && aligned16(a->v_last_4), AKV_ERR_ALIGN, "%s: pointers must be 16-byte aligned", fn);
    return AKV_OK;
}

}  // namespace
}  // namespace akv

using namespace akv;

extern "C" {

int akv_tree_commit(const akv_layer* layer, const void* k_new, const void* v_new, const void* path, int drafted, int accepted,
                    int rest_len, int rest_start, void* stream) {
    set_error("");
    const int rc = check_planes("tree_commit", layer);
    if (rc != AKV_OK) return rc;
    const akv_layer& a = *layer;
    AKV_REQUIRE(k_new && v_new && path && a.k_exp_max && a.v_exp_max && a.restk && a.restv, AKV_ERR_NULL,
                "tree_commit: null pointer");
    AKV_REQUIRE(drafted >= 1 && drafted <= BLK && accepted >= 1 && accepted <= BLK && rest_len >= 0 && rest_len < BLK &&
                rest_start >= 0 && rest_start % BLK == 0 && (long long)rest_start + rest_len + accepted <= a.max_seq_len,
                AKV_ERR_SHAPE, "tree_commit: %d of %d drafted tokens [1..64] behind %d + %d tokens of %d", accepted, drafted,
                rest_start, rest_len, a.max_seq_len);
    AKV_REQUIRE(aligned16(k_new) && aligned16(v_new) && aligned16(a.restk) && aligned16(a.restv) && aligned16(a.k_exp_max) &&
                aligned16(a.v_exp_max) && (reinterpret_cast<uintptr_t>(path) & 3u) == 0, AKV_ERR_ALIGN,
                "tree_commit: pointers must be 16-byte aligned");
    const int D = a.head_dim;
    launch_chained(commit_kernel, dim3(a.bsz * a.n_kv_heads, 2), dim3(256), rest_len + accepted >= BLK ? (size_t)BLK * 2 * D : 0,
                   static_cast<cudaStream_t>(stream), static_cast<uint8_t*>(a.k_first_8), static_cast<uint8_t*>(a.k_mid_4),
                   static_cast<uint8_t*>(a.k_last_4), static_cast<uint8_t*>(a.v_first_8), static_cast<uint8_t*>(a.v_mid_4),
                   static_cast<uint8_t*>(a.v_last_4), static_cast<uint16_t*>(a.k_exp_max), static_cast<uint16_t*>(a.v_exp_max),
                   static_cast<uint8_t*>(a.restk), static_cast<uint8_t*>(a.restv), static_cast<const uint8_t*>(k_new),
                   static_cast<const uint8_t*>(v_new), static_cast<const int*>(path), a.n_kv_heads, D, drafted, accepted, rest_len,
                   rest_start, (a.max_seq_len + BLK - 1) / BLK, a.max_seq_len);
    return cuda_status(cudaGetLastError(), "tree_commit launch");
}

long long akv_evict_scratch_bytes(int bsz, int n_kv_heads, int n_tokens, int keep) {
    if (bsz <= 0 || n_kv_heads <= 0 || keep <= 0 || keep > n_tokens) return -1;
    const long long most = keep < n_tokens - keep ? keep : n_tokens - keep;
    return (long long)bsz * n_kv_heads * (2 * most + 1) * 4;
}

int akv_evict(const akv_layer* layer, void* weights, void* positions, int rest_len, int rest_start, int keep, int recent,
              int arranged, int shift, void* stream) {
    set_error("");
    int rc = check_planes("evict", layer);
    if (rc != AKV_OK) return rc;
    const akv_layer& l = *layer;
    AKV_REQUIRE(weights && positions && l.scratch, AKV_ERR_NULL, "evict: null pointer");
    AKV_REQUIRE(rest_len >= 0 && rest_len < BLK && rest_start > 0 && rest_start % BLK == 0 &&
                (long long)rest_start + rest_len <= l.max_seq_len && keep > 0 && keep % BLK == 0 && keep <= rest_start &&
                recent >= 0 && recent <= keep && arranged >= 0 && arranged <= rest_start && shift >= 0 &&
                shift <= INT_MAX - 64 - l.max_seq_len, AKV_ERR_SHAPE,
                "evict: keep %d [multiple of 64], recent %d of %d + %d tokens of %d, %d arranged, shift %d", keep, recent, rest_start,
                rest_len, l.max_seq_len, arranged, shift);
    AKV_REQUIRE(rest_start / BLK < 65535, AKV_ERR_OVERFLOW, "evict: more than 65534 blocks");
    AKV_REQUIRE((reinterpret_cast<uintptr_t>(weights) & 3u) == 0 && (reinterpret_cast<uintptr_t>(positions) & 3u) == 0 &&
                aligned16(l.scratch), AKV_ERR_ALIGN, "evict: weights and positions must be 4-byte, scratch 16-byte aligned");
    AKV_REQUIRE(l.scratch_bytes >= akv_evict_scratch_bytes(l.bsz, l.n_kv_heads, rest_start, keep), AKV_ERR_SHAPE,
                "evict: scratch of %lld bytes is too small", l.scratch_bytes);
    const int rows = l.bsz * l.n_kv_heads;
    EvictArgs a = {};
    a.weights = static_cast<float*>(weights);
    a.positions = static_cast<int*>(positions);
    a.k8 = static_cast<uint8_t*>(l.k_first_8);
    a.km = static_cast<uint8_t*>(l.k_mid_4);
    a.kl = static_cast<uint8_t*>(l.k_last_4);
    a.v8 = static_cast<uint8_t*>(l.v_first_8);
    a.vm = static_cast<uint8_t*>(l.v_mid_4);
    a.vl = static_cast<uint8_t*>(l.v_last_4);
    a.most = keep < rest_start - keep ? keep : rest_start - keep;
    a.count = static_cast<int*>(l.scratch);
    a.holes = a.count + rows;
    a.movers = a.holes + (size_t)rows * a.most;
    a.D = l.head_dim;
    a.L = l.max_seq_len;
    a.nmb = (l.max_seq_len + BLK - 1) / BLK;
    a.n = rest_start;
    a.rest = rest_len;
    a.keep = keep;
    a.recent = recent;
    a.arranged = arranged;
    a.shift = shift;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    launch_chained(select_kernel, dim3(rows), dim3(SEL_NT), 0, st, a);
    if ((rc = cuda_status(cudaGetLastError(), "evict select launch")) != AKV_OK || keep == rest_start) return rc;
    launch_chained(move_kernel, dim3(rows, keep / BLK), dim3(256), (size_t)l.head_dim * 128, st, a);
    if ((rc = cuda_status(cudaGetLastError(), "evict move launch")) != AKV_OK) return rc;
    launch_chained(clear_kernel, dim3(rows, 1 + (rest_start - keep) / BLK), dim3(256), 0, st, a);
    return cuda_status(cudaGetLastError(), "evict clear launch");
}

}  // extern "C"
