// Attention of a tree of drafted tokens over the plane cache, and the entries of it and of its queries' weights.
//   tree_kernel         per (batch, KV head): up to 16 query rows against the planes, the residual tokens and the drafted tokens that
//                       the tree lets them see; one pass with a running maximum and sum (more rows: akv_tree_wide.cu)
//   tree_merge_kernel   joins the partial results of units that several runs share
//
//   s_rj = scale q_r . k_j (+ mask_j), o_r = sum_j exp(s_rj - m_r) v_j / l_r, l_r = sum_j exp(s_rj - m_r).
//
// All planes are read: 2 bytes per cached element, once.  Bound by HBM.
// Work: a unit is 16 query rows of one (batch, KV head); its tiles are 128 tokens of the planes each, and one tail tile of the
// residual tokens with the drafted ones behind them (at most 127).  The tiles of all units in a row are dealt to the warps in equal
// contiguous runs, so that every SM gets the same whatever the number of units and their length.  A warp needs no other one: it
// turns plane bytes into operand fragments in registers (akv_planes.cuh), keeps the scores of its tile and the output of its unit
// there, and leaves a record (maximum, sums, output) where a run begins or ends inside a unit.
// 8 x 32 x 4096 tokens, 16 rows: 103 us with the merge, 5.2 TB/s of 6.5 (its own share 96 us).
#include <limits.h>

#include "akv_planes.cuh"
#include "akv_tree.cuh"

namespace akv {
namespace {

constexpr int ROWS = 16, WARPS = 8;

// Token of line i of V step st within a tile, for lane column t: the tokens whose probabilities this lane holds.
__device__ __forceinline__ int v_token(int st, int t, int i) { return 32 * t + 2 * st + (i & 1) + (i >> 1) * 16; }

// A warp's ring of 4 KB steps in shared memory, filled STEPS - 1 steps ahead by its own asynchronous copies.
//   K step    16 channels of the tile's 128 tokens: high bytes [block][channel][64], nibbles [block][channel][32] twice
//   V step    32 (D = 128: 16) tokens: for each 16 of them high bytes [4t + i][D], nibbles [..][D / 2] twice
//   tail      16 tokens of the tail as fp16 rows [token][D]: a K step, then their V step
// The 16-byte pieces of a 128-byte line are swapped by XOR so that a quarter (half) warp's 16-byte (8-byte) loads of a line's
// pieces by lane (g, t) fall into different banks.
// Steps: four for eight warps with many tiles each (8 x 32 x 4096 tokens: 104 us, with three 107, with five 104).  A team (see
// Shape) has few warps with a tile or two each, which wait for the first bytes, not for the bandwidth: eight (1 x 32 x 1500 tokens:
// 12.9 us, with four 14.8).
constexpr int STEP_BYTES = 4096;
template <bool TEAM> constexpr int steps_of = TEAM ? 8 : 4;
template <bool TEAM> constexpr int warp_bytes = steps_of<TEAM> * STEP_BYTES + 8192;            // the ring, query fragments, probabilities
constexpr int TEAM_WARPS = 5;

template <int D, int STEPS>
struct Ring {
    static constexpr int KSTEPS = D / 16, VSTEPS = D / 16, SUB = 128 / D;     // SUB: products of 16 tokens per V step
    uint32_t base;                 // of the warp's ring
    int lane, put, get;            // steps: slots filled next, read next
    // what is copied next: step of a tile of (batch, KV head) bh; left = tiles from this one on
    int bh, left, step, tile, unit, plane_tiles;
    unsigned long long gone;       // a bit per tile from this one on: its mask leaves nothing

    // Tiles first .. last - 1 of units of p.tiles tiles, without those of `masked`.
    __device__ __forceinline__ void start(const TreeArgs& p, uint32_t at, int of_lane, int first, int last, unsigned long long masked) {
        base = at;
        lane = of_lane;
        put = get = step = 0;
        plane_tiles = (p.nb + 1) >> 1;
        unit = (unsigned)first / (unsigned)p.tiles;
        tile = first - unit * p.tiles;
        left = last - first;
        bh = unit;
        gone = masked;
        skip(p);
#pragma unroll 1
        for (int i = 0; i < STEPS - 1; ++i) fill(p);
    }
    __device__ __forceinline__ void next(const TreeArgs& p) {
        --left;
        gone >>= 1;
        if (++tile == p.tiles) {
            tile = 0;
            bh = ++unit;
        }
    }
    __device__ __forceinline__ void skip(const TreeArgs& p) {
        while (gone & 1) next(p);
    }
    __device__ __forceinline__ uint32_t slot(int i) const { return base + (uint32_t)i * STEP_BYTES; }

    __device__ __forceinline__ void copy_k(const TreeArgs& p, uint32_t to) const {
        const bool two = 2 * tile + 1 < p.nb;
        const long long row = ((long long)bh * p.nmb + 2 * tile) * D + 16 * step;
        const uint8_t *h = p.k8 + row * BLK + lane * 16, *m = p.km + row * (BLK / 2) + lane * 16, *l = p.kl + row * (BLK / 2) + lane * 16;
        // (lane: channel lane / 4 of 8, piece lane % 4; of nibbles channel lane / 2 of 16, piece lane % 2)
        const uint32_t at = (lane >> 3) * 128 + ((((lane >> 2) & 1) * 4 + (lane & 3)) ^ (2 * (lane >> 4))) * 16;
        const uint32_t nib = (lane >> 3) * 128 + ((((lane >> 1) & 3) * 2 + (lane & 1)) ^ (2 * (lane >> 3))) * 16;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const bool there = b == 0 || two;
            const long long o = there ? (long long)b * D : 0;
            copy16(to + b * 1024 + at, h + o * BLK, there);
            copy16(to + b * 1024 + 512 + (at ^ 64), h + o * BLK + 512, there);
            copy16(to + STEP_BYTES / 2 + b * 512 + nib, m + o * (BLK / 2), there);
            copy16(to + STEP_BYTES / 4 * 3 + b * 512 + nib, l + o * (BLK / 2), there);
        }
    }
    __device__ __forceinline__ void copy_v(const TreeArgs& p, uint32_t to, int vs) const {
        const bool two = 2 * tile + 1 < p.nb;
        const long long row = (long long)bh * p.L + tile * TILE;
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            const int st = vs * SUB + u;
            const uint32_t d = to + u * (STEP_BYTES / SUB);
            // rows of 128, 64 or 32 bytes: PIECES of 16 each
            auto rows = [&](const uint8_t* src, uint32_t dst, auto pieces) {
                constexpr int PIECES = decltype(pieces)::value;
#pragma unroll
                for (int j = 0; j < PIECES / 2; ++j) {
                    const int id = j * 32 + lane, r = id / PIECES, q = id % PIECES, t = r >> 2, i = r & 3;
                    const bool there = t < 2 || two;
                    const uint8_t* from = src + (row + (there ? v_token(st, t, i) : 0)) * (PIECES * 16) + q * 16;
                    copy16(dst + place<PIECES>(t, i, q), from, there);
                }
            };
            rows(p.v8, d, Int<D / 16>{});
            rows(p.vm, d + D * 16, Int<D / 32>{});
            rows(p.vl, d + D * 24, Int<D / 32>{});
        }
    }
    template <int X> struct Int { static constexpr int value = X; };
    // Where piece q of V row (t, i) lies, rows of PIECES pieces.
    template <int PIECES>
    static __device__ __forceinline__ uint32_t place(int t, int i, int q) {
        if constexpr (PIECES == 8) return (4 * t + i) * 128 + ((q ^ (2 * t)) << 4);
        else if constexpr (PIECES == 4) return (2 * i + (t >> 1)) * 128 + ((((t & 1) * 4 + q) ^ (2 * (t >> 1))) << 4);
        else return i * 128 + ((2 * t + q) << 4);
    }

    // Rows 16 c .. of the tail: the residual tokens, the drafted ones behind them; zeros behind those.
    __device__ __forceinline__ void copy_tail(const TreeArgs& p, uint32_t to, int c, bool value) const {
        const __half *rest = value ? p.restv : p.restk, *drafted = value ? p.vd : p.kd;
        const int b = (unsigned)bh / (unsigned)p.H, h = bh - b * p.H;
        constexpr int PIECES = D / 8;
#pragma unroll
        for (int j = 0; j < PIECES / 2; ++j) {
            const int id = j * 32 + lane, r = id / PIECES, q = id % PIECES, i = 16 * c + r, d = i - p.rest;
            const bool there = i < p.tail;
            const __half* row = d < 0 ? rest + ((long long)(b * BLK + i) * p.H + h) * D
                                      : drafted + ((long long)(b * p.T + (there ? d : 0)) * p.H + h) * D;
            copy16(to + tail_place(r, q, value), reinterpret_cast<const uint8_t*>(there ? row : p.q) + (there ? q * 16 : 0), there);
        }
    }
    // Where piece q of tail row r lies.  K is read by lane (g, t) = (row, 8 bytes of piece 2 kk + t / 2), V by (pieces of channels
    // N g .., rows 2t, 2t + 1, 2t + 8, 2t + 9).
    static __device__ __forceinline__ uint32_t tail_place(int r, int q, bool value) {
        const int t = (r >> 1) & 3;
        const int x = !value ? 2 * (r & 3) : D == 128 ? (t & 1) + 4 * (t >> 1) : 2 * t;
        return r * (2 * D) + ((q ^ x) << 4);
    }

    // One step further, if there is one; always a group, so that the groups count the steps.
    __device__ __forceinline__ void fill(const TreeArgs& p) {
        if (left > 0) {
            const uint32_t to = slot(put);
            int steps = KSTEPS + VSTEPS;
            if (tile == plane_tiles) {
                steps = ((p.tail + 15) >> 4) * 2;
                copy_tail(p, to, step >> 1, step & 1);
            } else if (step < KSTEPS) {
                copy_k(p, to);
            } else {
                copy_v(p, to, step - KSTEPS);
            }
            if (++step == steps) {
                step = 0;
                next(p);
                skip(p);
            }
        }
        cp_async_commit();
        put = put + 1 == STEPS ? 0 : put + 1;
    }
    // Waits for the step that is read next, requests the one whose slot the last read has left.
    __device__ __forceinline__ uint32_t take(const TreeArgs& p) {
        cp_async_wait<STEPS - 2>();
        __syncwarp();
        fill(p);
        const uint32_t at = slot(get);
        get = get + 1 == STEPS ? 0 : get + 1;
        return at;
    }

    __device__ __forceinline__ void lines_k(Line<16> (&x)[4], uint32_t at) const {
        const int g = lane >> 2, t = lane & 3;
        const uint32_t h = at + (g >> 2) * 1024 + 2 * t * 128 + (((g & 3) ^ (2 * t)) << 4);
        const uint32_t m = at + 2048 + (g >> 2) * 512 + t * 128 + (g & 1) * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t n = m + (((2 * i + ((g & 3) >> 1)) ^ (2 * t)) << 4);
            x[i].load((h ^ ((i & 1) * 64)) + (i >> 1) * 128, n, n + 1024);
        }
    }
    __device__ __forceinline__ void lines_v(Line<D / 8> (&x)[4], uint32_t at) const {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // the lane's D / 8 high bytes and D / 16 bytes of nibbles lie within one piece
            constexpr int HP = D / 16, NP = D / 32;
            const uint32_t h = at + place<HP>(t, i, D == 128 ? g : g >> 1) + (D == 128 ? 0 : (g & 1) * 8);
            const uint32_t n = at + D * 16 + place<NP>(t, i, D == 128 ? g >> 1 : g >> 2) + (D == 128 ? (g & 1) * 8 : (g & 3) * 4);
            x[i].load(h, n, n + D * 8);
        }
    }
};

// Of a run's first 64 tiles those whose mask takes every token away (left padding): neither copied nor looked at.  (A run is longer
// than that from 9.7 million cached (token, KV head) rows on; its tiles behind are masked score by score.)
__device__ __forceinline__ unsigned long long masked_tiles(const TreeArgs& p, int first, int last, int lane) {
    unsigned long long gone = 0;
    if (!p.mask) return gone;
#pragma unroll 4
    for (int i = 0; i < min(last - first, 64); ++i) {
        const int unit = (unsigned)(first + i) / (unsigned)p.tiles, tile = first + i - unit * p.tiles, count = p.nb * BLK - tile * TILE;
        const uint16_t* mask = reinterpret_cast<const uint16_t*>(p.mask) + (unsigned)unit / (unsigned)p.H * p.mask_stride + tile * TILE;
        bool none = tile < p.tiles - 1;
#pragma unroll
        for (int e = 0; e < TILE; e += 32)
            if (tile < p.tiles - 1 && lane + e < count) none = none && mask[lane + e] == 0xFC00u;
        gone |= (unsigned long long)__all_sync(0xFFFFFFFFu, none) << i;
    }
    return gone;
}

// Scores of a plane tile: s[j][c] = row g (c < 2) or g + 8, token 16 (2t + (c & 1)) + j.
template <int D, int STEPS>
__device__ __forceinline__ void plane_scores(float (&s)[16][4], const uint4* qf, const TreeArgs& p, Ring<D, STEPS>& ring) {
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll 1
    for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t at = ring.take(p);
        Line<16> x[4];
        ring.lines_k(x, at);
        mma_lines<16>(s, qf[kk * 32 + ring.lane], x);
    }
}

// Scores of 16 tail tokens: s[j][c] = row g (c < 2) or g + 8, token 8 j + 2t + (c & 1) of them.
template <int D>
__device__ __forceinline__ void tail_scores(float (&s)[2][4], const uint4* qf, uint32_t at, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int j = 0; j < 2; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint2 w = lds64(at + Ring<D, 4>::tail_place(g + 8 * j, 2 * kk + (t >> 1), false) + (t & 1) * 8);
            mma_f16(s[j], qf[kk * 32 + lane], w.x, w.y);
        }
}

// The unit's query rows as fragments in shared memory (every lane stores and reads its own).
template <int D>
__device__ __forceinline__ void load_q(uint4* qf, const TreeArgs& p, int b, int h, int lane) {
    const int g = lane >> 2, t = lane & 3, R = p.T * p.G;
    const __half* src[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = g + 8 * i;
        src[i] = r < R ? p.q + (long long)row_of(p, b, h, r) * D : nullptr;
    }
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
        uint2 w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = src[i] ? __ldg(reinterpret_cast<const uint2*>(src[i] + 16 * kk + 4 * t)) : make_uint2(0, 0);
        qf[kk * 32 + lane] = make_uint4(w[0].x, w[1].x, w[0].y, w[1].y);
    }
}

// Running maximum m, sums l and lr (of this lane's tokens) and output o of rows g and g + 8, taken on by scores s to base 2 of NJ n-tiles;
// s becomes the probabilities, relative to the maximum and times 2^LIFT.  (lr is taken on by `packed`.)
template <int NJ, int N>
__device__ __forceinline__ void soften(float (&s)[NJ][4], float (&m)[2], float (&l)[2], float (&lr)[2], float (&o)[N][4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float top = m[i];
#pragma unroll
        for (int j = 0; j < NJ; ++j) top = fmaxf(top, fmaxf(s[j][2 * i], s[j][2 * i + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        const float base = (top == -INFINITY ? 0.f : top) - LIFT;
        const float keep = ex2((m[i] - LIFT) - base);          // (nothing yet: 0)
        m[i] = top;
        l[i] *= keep;
        lr[i] *= keep;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            o[j][2 * i] *= keep;
            o[j][2 * i + 1] *= keep;
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                s[j][2 * i + c] = ex2(s[j][2 * i + c] - base);
                l[i] += s[j][2 * i + c];
            }
    }
}

// Two probabilities as they enter their product, added to lr.
__device__ __forceinline__ uint32_t packed(float x, float y, float& lr) {
    const uint32_t w = pack_half2(x, y);
    lr = plus_high(plus_low(lr, w), w);
    return w;
}

// One warp per query row: n records of its tokens, in their order, eight under way at a time; record i lies at at(i).
template <int D, class At>
__device__ __forceinline__ void join(const TreeArgs& p, At at, int n, long long to, int lane) {
    constexpr int C = D / 32, STEP = 8;                 // channels of a lane
    float acc[C], l = 0.f, lr = 0.f, top = -INFINITY;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = 0.f;
#pragma unroll 1
    for (int w = 0; w < n; w += STEP) {
        float4 ml[STEP];
        float o[STEP][C];
#pragma unroll
        for (int k = 0; k < STEP; ++k) {
            ml[k] = make_float4(-INFINITY, 0.f, 0.f, 0.f);
#pragma unroll
            for (int c = 0; c < C; ++c) o[k][c] = 0.f;
            if (w + k >= n) continue;
            const float* x = at(w + k);
            ml[k] = *reinterpret_cast<const float4*>(x);
            if constexpr (C == 4) {
                const float4 y = *reinterpret_cast<const float4*>(x + 4 + 4 * lane);
                o[k][0] = y.x; o[k][1] = y.y; o[k][2] = y.z; o[k][3] = y.w;
            } else {
                const float2 y = *reinterpret_cast<const float2*>(x + 4 + 2 * lane);
                o[k][0] = y.x; o[k][1] = y.y;
            }
        }
        float t = top;
#pragma unroll
        for (int k = 0; k < STEP; ++k) t = fmaxf(t, ml[k].x);
        const float base = t == -INFINITY ? 0.f : t, keep = ex2(top - base);
        top = t;
        l *= keep;
        lr *= keep;
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] *= keep;
#pragma unroll
        for (int k = 0; k < STEP; ++k) {
            const float f = ex2(ml[k].x - base);
            l = fmaf(f, ml[k].y, l);
            lr = fmaf(f, ml[k].z, lr);
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c] = fmaf(f, o[k][c], acc[c]);
        }
    }
    const float inv = lr == 0.f ? 0.f : 1.f / lr;
#pragma unroll
    for (int c = 0; c < C; c += 2)
        *reinterpret_cast<uint32_t*>(p.out + to * D + C * lane + c) = pack_half2(acc[c] * inv, acc[c + 1] * inv);
    if (p.lse && lane == 0) p.lse[to] = l == 0.f ? -INFINITY : ((top == -INFINITY ? 0.f : top) - LIFT + log2f(l)) * LN2;
}

// TEAM: the warps of a cluster have one unit between them and join their records themselves, in shared memory.
template <int D, bool TEAM>
__global__ void __launch_bounds__(32 * WARPS, 1) tree_kernel(const __grid_constant__ TreeArgs p) {
    constexpr int N = D / 8, WARP_BYTES = warp_bytes<TEAM>;
    using Ring = Ring<D, steps_of<TEAM>>;
    extern __shared__ __align__(128) uint8_t smem[];
    pdl_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int R = p.T * p.G;
    const int w = TEAM ? ((blockIdx.x % p.team) * blockDim.x >> 5) + warp : warp * gridDim.x + blockIdx.x;
    if (!TEAM && w >= p.nw) return;
    int first, last;
    if (TEAM) {                                        // p.nw runs of a unit, the first of them one tile longer, the last none
        const int each = p.tiles / p.nw, more = p.tiles - each * p.nw;
        first = blockIdx.x / (unsigned)p.team * p.tiles + w * each + min(w, more);
        last = first + each + (w < more);
    } else {
        first = run_start(p, w), last = run_start(p, w + 1);
    }
    const int unit0 = (unsigned)first / (unsigned)p.tiles;
    uint4* qf = reinterpret_cast<uint4*>(smem + (size_t)warp * WARP_BYTES + steps_of<TEAM> * STEP_BYTES);
    uint4* pf = qf + 256;
    Ring ring;
    unsigned long long gone = masked_tiles(p, first, last, lane);
    ring.start(p, smem_u32(smem) + warp * WARP_BYTES, lane, first, last, gone);
    // records: of a run's first unit in slot 0, of its last in slot 1 (those between are whole); a team's in place of the rings
    auto record = [&](int unit, int r) {
        return TEAM ? reinterpret_cast<float*>(smem + (size_t)warp * WARP_BYTES) + r * (D + 4)
                    : p.part + (size_t)((2 * w + (unit != unit0)) * ROWS + r) * (D + 4);
    };
    for (int at = first; at < last;) {
        // (one unit per KV head: more rows than 16 are the other kernel's)
        const int unit = (unsigned)at / (unsigned)p.tiles, b = (unsigned)unit / (unsigned)p.H, h = unit - b * p.H;
        const int t0 = at - unit * p.tiles, t1 = min(p.tiles, last - unit * p.tiles);
        const __half* mask = p.mask ? p.mask + b * p.mask_stride : nullptr;
        load_q<D>(qf, p, b, h, lane);
        float o[N][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, lr[2] = {0.f, 0.f};
        bool odd = false;                               // whether the tail has values that are not finite
#pragma unroll
        for (int j = 0; j < N; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
#pragma unroll 1
        for (int tile = t0; tile < min(t1, p.tiles - 1); ++tile) {
            const bool none = gone & 1;
            gone >>= 1;
            if (none) continue;
            {
                float s[16][4];
                plane_scores(s, qf, p, ring);
                const int count = p.nb * BLK - tile * TILE;
                if (mask || count < TILE) {             // tokens that do not exist or are masked away: -inf
#pragma unroll
                    for (int j = 0; j < 16; ++j)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int tok = 16 * (2 * t + c) + j;
                            const float add = mask && tok < count ? __half2float(mask[tile * TILE + tok]) : 0.f;
                            const bool gone = tok >= count || add == -INFINITY;
                            s[j][c] = gone ? -INFINITY : fmaf(s[j][c], p.scale2, add * LOG2E);
                            s[j][c + 2] = gone ? -INFINITY : fmaf(s[j][c + 2], p.scale2, add * LOG2E);
                        }
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
#pragma unroll
                        for (int c = 0; c < 4; ++c) s[j][c] *= p.scale2;
                }
                soften(s, m, l, lr, o);
                // (through shared memory, every lane its own: the loop over the V steps stays a loop - unrolled eight times, with
                // the copies in each, the kernel was bound by the fetch of its instructions, 195 us against 113 then at 8 x 32 x 4096 tokens)
#pragma unroll
                for (int st = 0; st < 8; ++st)
                    pf[st * 32 + lane] = make_uint4(packed(s[2 * st][0], s[2 * st + 1][0], lr[0]), packed(s[2 * st][2], s[2 * st + 1][2], lr[1]),
                                                    packed(s[2 * st][1], s[2 * st + 1][1], lr[0]), packed(s[2 * st][3], s[2 * st + 1][3], lr[1]));
            }
#pragma unroll 1
            for (int vs = 0; vs < Ring::VSTEPS; ++vs) {
                const uint32_t from = ring.take(p);
#pragma unroll
                for (int u = 0; u < Ring::SUB; ++u) {
                    const int st = vs * Ring::SUB + u;
                    Line<N> x[4];
                    ring.lines_v(x, from + u * (STEP_BYTES / Ring::SUB));
                    if (mask) {      // a token that is masked away counts as zero, whatever its values are: 0 * NaN would be NaN
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int tok = tile * TILE + v_token(st, t, i);
                            if (tok < p.nb * BLK && __half_as_ushort(mask[tok]) == 0xFC00u) x[i].clear();
                        }
                    }
                    mma_lines<N>(o, pf[st * 32 + lane], x);
                }
            }
        }
        if (t1 == p.tiles) {
            gone >>= 1;
            // The tail, 16 tokens at a time: rows of fp16 values.
            const uint8_t* seen = p.tree + b * p.tree_stride;
            const uint8_t* mine[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) mine[i] = seen + (unsigned)min(g + 8 * i, R - 1) / (unsigned)p.G * p.T;
#pragma unroll 1
            for (int c0 = 0; c0 < p.tail; c0 += 16) {
                float s[2][4];
                tail_scores<D>(s, qf, ring.take(p), lane);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int tok = c0 + 8 * j + 2 * t + c, d = tok - p.rest;
                        const float add = mask && d < 0 ? __half2float(mask[p.nb * BLK + tok]) : 0.f;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const bool here = d < 0 ? add != -INFINITY : d < p.T && mine[i][d];
                            s[j][2 * i + c] = here ? fmaf(s[j][2 * i + c], p.scale2, add * LOG2E) : -INFINITY;
                        }
                    }
                soften(s, m, l, lr, o);
                const uint4 a = make_uint4(packed(s[0][0], s[0][1], lr[0]), packed(s[0][2], s[0][3], lr[1]), packed(s[1][0], s[1][1], lr[0]),
                                           packed(s[1][2], s[1][3], lr[1]));
                const uint32_t from = ring.take(p);
                uint32_t x[4][N / 2];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 2 * t + (i & 1) + 8 * (i >> 1);
#pragma unroll
                    for (int v = 0; v < N / 8; ++v) {
                        const uint4 y = lds128(from + Ring::tail_place(r, N / 8 * g + v, true));
                        x[i][4 * v] = y.x; x[i][4 * v + 1] = y.y; x[i][4 * v + 2] = y.z; x[i][4 * v + 3] = y.w;
                    }
#pragma unroll
                    for (int v = 0; v < N / 2; ++v) x[i][v] = finite_halves(x[i][v], odd);
                }
#pragma unroll
                for (int v = 0; v < N / 2; ++v) {
                    mma_f16(o[2 * v], a, __byte_perm(x[0][v], x[1][v], 0x5410), __byte_perm(x[2][v], x[3][v], 0x5410));
                    mma_f16(o[2 * v + 1], a, __byte_perm(x[0][v], x[1][v], 0x7632), __byte_perm(x[2][v], x[3][v], 0x7632));
                }
            }
            odd = __any_sync(0xFFFFFFFFu, odd);
        }
        if (TEAM) __syncwarp();                        // (the ring has been read)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 1);
            l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 2);
            lr[i] += __shfl_xor_sync(0xFFFFFFFFu, lr[i], 1);
            lr[i] += __shfl_xor_sync(0xFFFFFFFFu, lr[i], 2);
            const int r = g + 8 * i;
            if (r >= R) continue;
            if (t0 == 0 && t1 == p.tiles) {
                const long long row = row_of(p, b, h, r);
                const float inv = lr[i] == 0.f ? 0.f : 1.f / lr[i];
                uint4* dst = reinterpret_cast<uint4*>(p.out + row * D + 2 * N * t);
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int v = 0; v < N / 8; ++v) {
                        uint32_t x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            x[e] = pack_half2(o[8 * v + 2 * e][2 * i + c] * inv, o[8 * v + 2 * e + 1][2 * i + c] * inv);
                        dst[c * (N / 8) + v] = make_uint4(x[0], x[1], x[2], x[3]);
                    }
                if (p.lse && t == 0) p.lse[row] = l[i] == 0.f ? -INFINITY : (m[i] - LIFT + log2f(l[i])) * LN2;
            } else {
                float* rec = record(unit, r);
                if (t == 0) *reinterpret_cast<float4*>(rec) = make_float4(m[i], l[i], lr[i], 0.f);
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int v = 0; v < N / 4; ++v)
                        reinterpret_cast<float4*>(rec + 4 + N * (2 * t + c))[v] =
                            make_float4(o[4 * v][2 * i + c], o[4 * v + 1][2 * i + c], o[4 * v + 2][2 * i + c],
                                        o[4 * v + 3][2 * i + c]);
            }
        }
        __syncwarp();
        if (odd && t == 0) {
#pragma unroll 1
            for (int i = 0; i < 2; ++i) {
                const int r = g + 8 * i;
                if (r >= R) continue;
                const float top = i ? m[1] : m[0], sum = i ? lr[1] : lr[0], base = (top == -INFINITY ? 0.f : top) - LIFT;
                if (t0 == 0 && t1 == p.tiles)
                    add_odd(p, b, h, r, D, base, sum == 0.f ? 0.f : 1.f / sum, p.out + (long long)row_of(p, b, h, r) * D);
                else
                    add_odd(p, b, h, r, D, base, 1.f, record(unit, r) + 4);
            }
        }
        at = unit * p.tiles + t1;
    }
    if constexpr (TEAM) {
        const int wpc = blockDim.x >> 5, unit = blockIdx.x / (unsigned)p.team, b = (unsigned)unit / (unsigned)p.H, h = unit - b * p.H;
        cluster_sync();
        for (int r = w; r < R; r += p.nw) {
            auto at = [&](int i) {
                const float* x = reinterpret_cast<const float*>(smem + (size_t)(i % wpc) * WARP_BYTES) + r * (D + 4);
                uint64_t y;
                asm("mapa.u64 %0, %1, %2;\n" : "=l"(y) : "l"(x), "r"(i / wpc));
                return reinterpret_cast<const float*>(y);
            };
            join<D>(p, at, min(p.nw, p.tiles), row_of(p, b, h, r), lane);
        }
        cluster_sync();                                // (no CTA leaves while another reads its records)
    }
}

// One warp per query row: the records of the runs that share its unit.  Bound by latency: where the row lies is worked out before the
// kernel in front has ended.
template <int D>
__global__ void __launch_bounds__(128) tree_merge_kernel(const __grid_constant__ TreeArgs p) {
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), unit = row / ROWS, r = row % ROWS;
    const int b = (unsigned)unit / (unsigned)p.H, h = unit - b * p.H;
    const int w0 = run_with(p, unit * p.tiles), w1 = run_with(p, unit * p.tiles + p.tiles - 1);
    const long long to = row_of(p, b, h, r);
    // a run's record of its first unit is in slot 0, of its last in slot 1: only the first of this unit's may have begun before it
    const float* rec = p.part + (size_t)(2 * w0 * ROWS + r) * (D + 4);
    constexpr size_t pitch = (size_t)2 * ROWS * (D + 4);
    const float* rec0 = run_start(p, w0) < unit * p.tiles ? rec + pitch / 2 : rec;
    pdl_wait();
    // (a whole unit has been written by its run)
    if ((unsigned)unit >= (unsigned)p.total / (unsigned)p.tiles || r >= p.T * p.G || w0 == w1) return;
    join<D>(p, [&](int i) { return i == 0 ? rec0 : rec + i * pitch; }, w1 - w0 + 1, to, lane);
}

// Warps for `total` tiles: one an SM while there are that few, then up to eight.
struct Deal {
    int grid, wpc, runs;
};
Deal deal(long long total, int most = WARPS) {
    const int sms = sm_count();
    Deal d;
    d.grid = (int)(total < sms ? total : sms);
    const long long per = (total + d.grid - 1) / d.grid;
    d.wpc = (int)(per < most ? per : most);
    d.runs = total < (long long)d.grid * d.wpc ? (int)total : d.grid * d.wpc;
    return d;
}

// How the attention of T drafted tokens behind rest_start tokens is cut up.
struct Shape {
    bool wide;
    int team, team_runs;       // CTAs of a cluster that has a unit to itself and its warps, or 0: runs of equal length
    int groups, rowsg, rowsu, rt, tiles;
    long long units, total;
    Deal d;
};
Shape shape_of(int bsz, int H, int G, int T, int rest_start) {
    Shape s;
    const int R = T * G;
    // More rows than a warp's product has: the tensor cores' kernel reads the planes once for up to 256 rows, this one would once
    // for 16 (20 rows, 8 x 131072 tokens: 125 us there, 187 here; 48 rows, 16 x 8 x 8190: 128 and 288).  Up to 16 rows it is
    // bound by HBM and has no chain through three roles of warps to wait for (8 x 32 x 4096, 16 rows: 103 us here, 130 there).
    s.wide = R > ROWS;
    s.groups = R > 128 ? 2 : 1;
    s.rt = s.wide ? (R + 128 * s.groups - 1) / (128 * s.groups) : 1;
    s.rowsu = s.wide ? (R + s.rt - 1) / s.rt : ROWS;
    s.rowsg = (s.rowsu + s.groups - 1) / s.groups;
    s.tiles = (rest_start / BLK + 1) / 2 + 1;
    s.units = (long long)bsz * H * s.rt;
    s.total = s.units * s.tiles;
    s.d = deal(s.total, s.wide ? 1 : WARPS);
    s.team = 0;
    // Short caches: a cluster per unit, one launch and no records in memory, wherever no warp gets more tiles by it (clusters of one
    // size leave some SMs without any: an eighth of them is not counted on).  On the device 12.3 us against 14.4 with equal runs and a
    // merge at 1 x 32 x 777 tokens, 15.7 against 18.0 at 1 x 8 x 4000, and a launch less for the host.
    int ctas = 8;
    while (ctas > 1 && s.units * ctas > sm_count() * 7 / 8) ctas /= 2;
    if (s.wide || s.tiles == 1 || s.units * ctas > sm_count()) return s;
    const int per = (s.tiles + ctas - 1) / ctas, wpc = per < TEAM_WARPS ? per : TEAM_WARPS, n = ctas * wpc;
    if ((s.tiles + n - 1) / n <= (s.total + s.d.runs - 1) / s.d.runs) {
        s.team = ctas;
        s.d.grid = (int)s.units * ctas;
        s.d.wpc = wpc;
        s.team_runs = n;
    }
    return s;
}

// (the limit is raised for what eight warps take, whatever this launch does: it is a property of the kernel, not of the call)
template <class Kernel>
int launch_warps(Kernel kernel, const Deal& d, cudaStream_t st, const TreeArgs& p) {
    const int bytes = p.team ? warp_bytes<true> : warp_bytes<false>;
    const int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (p.team ? TEAM_WARPS : WARPS) * bytes),
                               "tree kernel shared memory");
    if (rc != AKV_OK) return rc;
    const dim3 grid(d.grid), block(32 * d.wpc);
    if (p.team) launch_cluster(kernel, p.team, grid, block, (size_t)d.wpc * bytes, st, p);
    else launch_chained(kernel, grid, block, (size_t)d.wpc * bytes, st, p);
    return AKV_OK;
}

// Query rows per drafted token: so few that all indices of rows fit 32 bits.  (The first two factors alone fit 64 bits, not all three.)
bool few_rows(int bsz, int H, int G) {
    constexpr long long most = (1ll << 30) / BLK;
    return (long long)bsz * H < most && (long long)bsz * H * G < most;
}

int check_layer(const char* fn, const akv_layer* a, const void* q, int T, int rest_len, int rest_start, const void* mask,
                long long mask_stride) {
    AKV_REQUIRE(a && q && a->k_first_8 && a->k_mid_4 && a->k_last_4 && a->v_first_8 && a->v_mid_4 && a->v_last_4 && a->restk &&
                a->restv, AKV_ERR_NULL, "%s: null pointer", fn);
    AKV_REQUIRE(a->bsz > 0 && a->n_kv_heads > 0 && a->group > 0 && (a->head_dim == 64 || a->head_dim == 128) &&
                a->max_seq_len > 0 && a->max_seq_len <= INT_MAX - 128 && T >= 1 && T <= BLK, AKV_ERR_SHAPE,
                "%s: unsupported extent (bsz %d, KV heads %d, "
                "group %d, head_dim %d [64 or 128], max_seq_len %d, drafted tokens %d [1..64])", fn, a->bsz, a->n_kv_heads,
                a->group, a->head_dim, a->max_seq_len, T);
    AKV_REQUIRE(rest_len >= 0 && rest_len < BLK && rest_start >= 0 && rest_start % BLK == 0 &&
                (long long)rest_start + rest_len <= a->max_seq_len, AKV_ERR_SHAPE,
                "%s: rest_len %d [0..63] behind %d tokens [multiple of 64] of %d", fn, rest_len, rest_start, a->max_seq_len);
    AKV_REQUIRE(few_rows(a->bsz, a->n_kv_heads, a->group), AKV_ERR_OVERFLOW, "%s: too many rows", fn);
    AKV_REQUIRE(!mask || mask_stride >= 0, AKV_ERR_SHAPE, "%s: negative mask stride", fn);
    AKV_REQUIRE(aligned16(a->k_first_8) && aligned16(a->k_mid_4) && aligned16(a->k_last_4) && aligned16(a->v_first_8) &&
                aligned16(a->v_mid_4) && aligned16(a->v_last_4) && aligned16(a->restk) && aligned16(a->restv) && aligned16(q),
                AKV_ERR_ALIGN, "%s: pointers must be 16-byte aligned", fn);
    AKV_REQUIRE((reinterpret_cast<uintptr_t>(mask) & 1u) == 0, AKV_ERR_ALIGN, "%s: the mask must be 2-byte aligned", fn);
    return AKV_OK;
}

TreeArgs make_args(const akv_layer* a, const void* q, int T, int rest_len, int rest_start, const void* mask, long long mask_stride,
                   float scale) {
    TreeArgs p = {};
    p.k8 = static_cast<const uint8_t*>(a->k_first_8);
    p.km = static_cast<const uint8_t*>(a->k_mid_4);
    p.kl = static_cast<const uint8_t*>(a->k_last_4);
    p.v8 = static_cast<const uint8_t*>(a->v_first_8);
    p.vm = static_cast<const uint8_t*>(a->v_mid_4);
    p.vl = static_cast<const uint8_t*>(a->v_last_4);
    p.restk = static_cast<const __half*>(a->restk);
    p.restv = static_cast<const __half*>(a->restv);
    p.q = static_cast<const __half*>(q);
    p.mask = static_cast<const __half*>(mask);
    p.mask_stride = mask_stride;
    p.H = a->n_kv_heads;
    p.G = a->group;
    p.T = T;
    p.L = a->max_seq_len;
    p.nmb = (a->max_seq_len + BLK - 1) / BLK;
    p.nb = rest_start / BLK;
    p.rest = rest_len;
    p.scale = scale;
    p.scale2 = scale * LOG2E;
    return p;
}

}  // namespace
}  // namespace akv

using namespace akv;

extern "C" {

long long akv_tree_scratch_bytes(int bsz, int n_kv_heads, int group, int head_dim, int n_tokens, int drafted) {
    if (bsz <= 0 || n_kv_heads <= 0 || group <= 0 || (head_dim != 64 && head_dim != 128) || n_tokens < 0 || drafted < 1 ||
        drafted > BLK || !few_rows(bsz, n_kv_heads, group))
        return -1;
    const Shape s = shape_of(bsz, n_kv_heads, group, drafted, n_tokens);
    return 2ll * s.d.runs * s.rowsu * (head_dim + 4) * 4;
}

int akv_tree_attention(const akv_layer* layer, const void* q, const void* k_new, const void* v_new, const void* tree,
                       long long tree_stride, const void* mask, long long mask_stride, void* out, void* lse, int drafted,
                       int rest_len, int rest_start, float scale, void* stream) {
    set_error("");
    int rc = check_layer("tree_attention", layer, q, drafted, rest_len, rest_start, mask, mask_stride);
    if (rc != AKV_OK) return rc;
    AKV_REQUIRE(k_new && v_new && tree && out && layer->scratch, AKV_ERR_NULL, "tree_attention: null pointer");
    AKV_REQUIRE(tree_stride >= 0, AKV_ERR_SHAPE, "tree_attention: negative tree stride");
    AKV_REQUIRE(aligned16(k_new) && aligned16(v_new) && aligned16(out) && aligned16(layer->scratch), AKV_ERR_ALIGN,
                "tree_attention: pointers must be 16-byte aligned");
    AKV_REQUIRE((reinterpret_cast<uintptr_t>(lse) & 3u) == 0, AKV_ERR_ALIGN, "tree_attention: lse must be 4-byte aligned");
    const int D = layer->head_dim;
    AKV_REQUIRE(layer->scratch_bytes >= akv_tree_scratch_bytes(layer->bsz, layer->n_kv_heads, layer->group, D, rest_start, drafted),
                AKV_ERR_SHAPE, "tree_attention: scratch of %lld bytes is too small", layer->scratch_bytes);
    TreeArgs p = make_args(layer, q, drafted, rest_len, rest_start, mask, mask_stride, scale);
    p.kd = static_cast<const __half*>(k_new);
    p.vd = static_cast<const __half*>(v_new);
    p.tree = static_cast<const uint8_t*>(tree);
    p.tree_stride = tree_stride;
    p.out = static_cast<__half*>(out);
    p.lse = static_cast<float*>(lse);
    p.part = static_cast<float*>(layer->scratch);
    p.tail = rest_len + drafted;
    const Shape s = shape_of(layer->bsz, p.H, p.G, drafted, rest_start);
    p.groups = s.groups;
    p.rowsg = s.rowsg;
    p.rowsu = s.rowsu;
    p.rt = s.rt;
    p.tiles = s.tiles;
    AKV_REQUIRE(s.total < INT_MAX, AKV_ERR_OVERFLOW, "tree_attention: too many tiles of 128 tokens");
    p.total = (int)s.total;
    p.nw = s.team ? s.team_runs : s.d.runs;
    p.team = s.team;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (s.wide) return launch_tree_wide(p, D, s.d.grid, (int)s.units, st);
    rc = s.team ? launch_warps(D == 128 ? tree_kernel<128, true> : tree_kernel<64, true>, s.d, st, p)
                : launch_warps(D == 128 ? tree_kernel<128, false> : tree_kernel<64, false>, s.d, st, p);
    if (rc != AKV_OK) return rc;
    rc = cuda_status(cudaGetLastError(), "tree_attention launch");
    if (rc != AKV_OK || p.tiles == 1 || s.team) return rc;       // (units of one tile: none is shared)
    launch_chained(D == 128 ? tree_merge_kernel<128> : tree_merge_kernel<64>, dim3((unsigned)(s.units * (ROWS / 4))),
                   dim3(128), 0, st, p);
    return cuda_status(cudaGetLastError(), "tree_attention merge launch");
}

int akv_tree_weights(const akv_layer* layer, const void* q, const void* lse, const void* mask, long long mask_stride,
                     void* weights, int drafted, int rest_len, int rest_start, float scale, void* stream) {
    set_error("");
    int rc = check_layer("tree_weights", layer, q, drafted, rest_len, rest_start, mask, mask_stride);
    if (rc != AKV_OK) return rc;
    AKV_REQUIRE(lse && weights, AKV_ERR_NULL, "tree_weights: null pointer");
    AKV_REQUIRE(((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(weights)) & 3u) == 0, AKV_ERR_ALIGN,
                "tree_weights: lse and weights must be 4-byte aligned");
    TreeArgs p = make_args(layer, q, drafted, rest_len, rest_start, mask, mask_stride, scale);
    p.lse = static_cast<float*>(const_cast<void*>(lse));
    p.tiles = (p.nb + 1) / 2 + (rest_len > 0);
    p.tail = rest_len;
    const long long total = (long long)layer->bsz * p.H * p.tiles;
    AKV_REQUIRE(total < INT_MAX, AKV_ERR_OVERFLOW, "tree_weights: too many tiles of 128 tokens");
    p.total = (int)total;
    if (total == 0) return AKV_OK;
    const Deal d = deal(p.total, 1);
    p.nw = d.runs;
    p.rt = 1;
    return launch_weights_wide(p, layer->head_dim, d.grid, static_cast<float*>(weights), static_cast<cudaStream_t>(stream));
}

}  // extern "C"
