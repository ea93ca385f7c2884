// Attention of a tree of drafted tokens over the plane cache, and the attention weights of its queries.
//   tree_kernel      per (batch, KV head): the T * group query rows against the planes, the residual tokens and the drafted
//                    tokens that the tree lets them see; one pass with a running maximum and sum
//   tree_merge_kernel   joins the partial results of units that several warps share
//   weights_kernel   weights[t] += sum over the rows of exp(s_t - lse)
//
//   s_rj = scale q_r . k_j (+ mask_j), o_r = sum_j exp(s_rj - m_r) v_j / l_r, l_r = sum_j exp(s_rj - m_r).
//
// All planes are read: 2 bytes per cached element, once per 16 rows.  Bound by HBM while the rows of a KV head are few.
// Work: a unit is 16 query rows of one (batch, KV head); its tiles are 128 tokens of the planes each, and one tail tile of the
// residual (slots 0..63) and the drafted tokens (slots 64..127).  The tiles of all units in a row are dealt to the warps in equal
// contiguous runs, so that every SM gets the same whatever the number of units and their length.  A warp needs no other one: it
// turns plane bytes into operand fragments in registers (akv_planes.cuh), keeps the scores of its tile and the output of its unit
// there, and leaves a record (maximum, sum, output) where a run begins or ends inside a unit.
#include <limits.h>

#include "akv_planes.cuh"

namespace akv {
namespace {

constexpr int BLK = 64, TILE = 128, ROWS = 16, WARPS = 8;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// Probabilities enter their product as fp16, relative to the running maximum and times 2^15: at most 32768, and down to 2^-29 of the
// largest with all 11 bits (2^-14 without the factor).
constexpr float LIFT = 15.f;

struct TreeArgs {
    const uint8_t *k8, *km, *kl, *v8, *vm, *vl;
    const __half *restk, *restv, *q, *kd, *vd, *mask;
    const uint8_t* tree;
    long long tree_stride, mask_stride;
    __half* out;
    float *lse, *part;
    int H, G, T, nmb, L, nb, rest, rt, tiles;
    long long total, nw;       // tiles of all units, warps that they are dealt to (at most as many)
    float scale2;              // scale * log2(e)
};

__device__ __forceinline__ float ex2(float x) { return exp2f(x); }

// One K step: 16 channels of the tile's 128 tokens; lane (g, t): channels 16 kk + 4t .. + 3, tokens 16g .. 16g + 15.
template <int D>
__device__ __forceinline__ void load_k(Line<16> (&x)[4], const TreeArgs& p, long long bh, int tile, int kk, int g, int t) {
    const int blk = 2 * tile + (g >> 2);
    if (blk < p.nb) {
        const long long row = (bh * p.nmb + blk) * D + 16 * kk + 4 * t;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i].load(p.k8 + (row + i) * BLK + 16 * (g & 3), p.km + (row + i) * (BLK / 2) + 8 * (g & 3),
                      p.kl + (row + i) * (BLK / 2) + 8 * (g & 3));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i].clear();
    }
}

// Token of line i of V step st within a tile, for lane column t: the tokens whose probabilities this lane holds.
__device__ __forceinline__ int v_token(int st, int t, int i) { return 32 * t + 2 * st + (i & 1) + (i >> 1) * 16; }

template <int D>
__device__ __forceinline__ void load_v(Line<D / 8> (&x)[4], const TreeArgs& p, long long bh, int tile, int st, int g, int t,
                                       const __half* mask) {
    constexpr int N = D / 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int tok = tile * TILE + v_token(st, t, i);
        // (a token that the mask takes away counts as zero, whatever its values are: 0 * NaN would be NaN)
        if (tok < p.nb * BLK && !(mask && __ldg(reinterpret_cast<const uint16_t*>(mask) + tok) == 0xFC00u)) {
            const long long row = bh * p.L + tok;
            x[i].load(p.v8 + row * D + N * g, p.vm + row * (D / 2) + N / 2 * g, p.vl + row * (D / 2) + N / 2 * g);
        } else {
            x[i].clear();
        }
    }
}

// Scores of a plane tile: s[j][c] = row g (c < 2) or g + 8, token 16 (2t + (c & 1)) + j.
template <int D>
__device__ __forceinline__ void plane_scores(float (&s)[16][4], const uint4* qf, const TreeArgs& p, long long bh, int tile,
                                             int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll 1
    for (int kk = 0; kk < D / 16; ++kk) {
        Line<16> x[4];
        load_k<D>(x, p, bh, tile, kk, g, t);
        mma_lines<16>(s, qf[kk * 32 + lane], x);
    }
}

// Row of the tail tile's slot (0..63 residual, 64.. drafted) in an fp16 tensor pair; nullptr: there is none.
__device__ __forceinline__ const __half* tail_row(const __half* rest, const __half* drafted, const TreeArgs& p, int D, long long b,
                                                  int h, int slot) {
    if (slot < BLK) return slot < p.rest ? rest + ((b * BLK + slot) * p.H + h) * D : nullptr;
    return drafted && slot - BLK < p.T ? drafted + ((b * p.T + slot - BLK) * p.H + h) * D : nullptr;
}

template <int D>
__device__ __forceinline__ void tail_scores(float (&s)[16][4], const uint4* qf, const TreeArgs& p, long long b, int h, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const __half* row = tail_row(p.restk, p.kd, p, D, b, h, 16 * g + j);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            const uint2 w = row ? __ldg(reinterpret_cast<const uint2*>(row + 16 * kk + 4 * t)) : make_uint2(0, 0);
            mma_f16(s[j], qf[kk * 32 + lane], w.x, w.y);
        }
    }
}

// The unit's query rows as fragments in shared memory (every lane stores and reads its own).
template <int D>
__device__ __forceinline__ void load_q(uint4* qf, const TreeArgs& p, long long b, int h, int row0, int lane) {
    const int g = lane >> 2, t = lane & 3, R = p.T * p.G;
    const __half* src[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = row0 + g + 8 * i;
        src[i] = r < R ? p.q + ((b * p.T + r / p.G) * p.H * p.G + (long long)h * p.G + r % p.G) * D : nullptr;
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

// Scores to base 2 of a plane tile or of the tail's residual half; tokens that do not exist or are masked away: -inf.
__device__ __forceinline__ void scale_mask(float (&s)[16][4], const TreeArgs& p, const __half* mask, int first, int count, int t) {
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int tok = 16 * (2 * t + c) + j;
            float add = 0.f;
            if (mask && tok < count) add = __half2float(mask[first + tok]);
            const bool gone = tok >= count || add == -INFINITY;
            s[j][c] = gone ? -INFINITY : fmaf(s[j][c], p.scale2, add * LOG2E);
            s[j][c + 2] = gone ? -INFINITY : fmaf(s[j][c + 2], p.scale2, add * LOG2E);
        }
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <int D>
__global__ void __launch_bounds__(32 * WARPS, 1) tree_kernel(const TreeArgs p) {
    constexpr int N = D / 8;
    __shared__ __align__(16) uint4 frag[WARPS][256];
    pdl_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int R = p.T * p.G;
    const long long w = (long long)warp * gridDim.x + blockIdx.x;
    if (w >= p.nw) return;
    const long long first = w * p.total / p.nw, last = (w + 1) * p.total / p.nw;
    uint4* qf = frag[warp];
    for (long long at = first; at < last;) {
        const long long unit = at / p.tiles, bh = unit / p.rt, b = bh / p.H;
        const int h = (int)(bh - b * p.H), row0 = (int)(unit - bh * p.rt) * ROWS;
        const int t0 = (int)(at - unit * p.tiles), t1 = (int)min((long long)p.tiles, last - unit * p.tiles);
        const __half* mask = p.mask ? p.mask + b * p.mask_stride : nullptr;
        load_q<D>(qf, p, b, h, row0, lane);
        float o[N][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < N; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
#pragma unroll 1
        for (int tile = t0; tile < t1; ++tile) {
            const bool tail = tile == p.tiles - 1;
            float s[16][4];
            if (!tail) {
                plane_scores<D>(s, qf, p, bh, tile, lane);
                scale_mask(s, p, mask, tile * TILE, min(TILE, p.nb * BLK - tile * TILE), t);
            } else {
                tail_scores<D>(s, qf, p, b, h, lane);
                if (t < 2) {
                    scale_mask(s, p, mask, p.nb * BLK, p.rest, t);
                } else {
                    const uint8_t* seen = p.tree + b * p.tree_stride;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int r = row0 + g + 8 * i;
                        const uint8_t* mine = seen + (long long)(r / p.G) * p.T;
#pragma unroll
                        for (int j = 0; j < 16; ++j)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const int d = 16 * (2 * t + c) + j - BLK;
                                s[j][2 * i + c] = r < R && d < p.T && mine[d] ? s[j][2 * i + c] * p.scale2 : -INFINITY;
                            }
                    }
                }
            }
            uint32_t pf[16][2];      // probabilities of rows g and g + 8 as they enter the product: [j] = tokens 16 (2t) + j ...
            float base[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float top = m[i];
#pragma unroll
                for (int j = 0; j < 16; ++j) top = fmaxf(top, fmaxf(s[j][2 * i], s[j][2 * i + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                base[i] = (top == -INFINITY ? 0.f : top) - LIFT;
                const float keep = ex2((m[i] - LIFT) - base[i]);          // (nothing yet: 0)
                m[i] = top;
                l[i] *= keep;
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    o[j][2 * i] *= keep;
                    o[j][2 * i + 1] *= keep;
                }
#pragma unroll
                for (int j = 0; j < 16; ++j)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        s[j][2 * i + c] = ex2(s[j][2 * i + c] - base[i]);
                        l[i] += s[j][2 * i + c];
                    }
            }
#pragma unroll
            for (int st = 0; st < 8; ++st) {
                pf[2 * st][0] = pack_half2(s[2 * st][0], s[2 * st + 1][0]);
                pf[2 * st][1] = pack_half2(s[2 * st][2], s[2 * st + 1][2]);
                pf[2 * st + 1][0] = pack_half2(s[2 * st][1], s[2 * st + 1][1]);
                pf[2 * st + 1][1] = pack_half2(s[2 * st][3], s[2 * st + 1][3]);
            }
            if (!tail) {
#pragma unroll
                for (int st = 0; st < 8; ++st) {
                    Line<N> x[4];
                    load_v<D>(x, p, bh, tile, st, g, t, mask);
                    mma_lines<N>(o, make_uint4(pf[2 * st][0], pf[2 * st][1], pf[2 * st + 1][0], pf[2 * st + 1][1]), x);
                }
                continue;
            }
            // The tail: rows of fp16 values.  What one row of the tree sees is masked for another, and 0 * inf would be NaN:
            // drafted values that are not finite are left out of the product and added by the rows that see them.
            bool odd = false;
#pragma unroll
            for (int st = 0; st < 8; ++st) {
                uint32_t x[4][N / 2];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int slot = v_token(st, t, i);
                    const __half* row = tail_row(p.restv, p.vd, p, D, b, h, slot);
                    if (row && slot < BLK && mask && __half_as_ushort(mask[p.nb * BLK + slot]) == 0xFC00u) row = nullptr;
#pragma unroll
                    for (int v = 0; v < N / 8; ++v) {
                        const uint4 y = row ? __ldg(reinterpret_cast<const uint4*>(row + N * g) + v) : make_uint4(0, 0, 0, 0);
                        x[i][4 * v] = y.x; x[i][4 * v + 1] = y.y; x[i][4 * v + 2] = y.z; x[i][4 * v + 3] = y.w;
                    }
                    if (slot >= BLK) {
#pragma unroll
                        for (int v = 0; v < N / 2; ++v) {
                            if ((x[i][v] & 0x7C00u) == 0x7C00u) { x[i][v] &= 0xFFFF0000u; odd = true; }
                            if ((x[i][v] & 0x7C000000u) == 0x7C000000u) { x[i][v] &= 0xFFFFu; odd = true; }
                        }
                    }
                }
                const uint4 a = make_uint4(pf[2 * st][0], pf[2 * st][1], pf[2 * st + 1][0], pf[2 * st + 1][1]);
#pragma unroll
                for (int v = 0; v < N / 2; ++v) {
                    mma_f16(o[2 * v], a, __byte_perm(x[0][v], x[1][v], 0x5410), __byte_perm(x[2][v], x[3][v], 0x5410));
                    mma_f16(o[2 * v + 1], a, __byte_perm(x[0][v], x[1][v], 0x7632), __byte_perm(x[2][v], x[3][v], 0x7632));
                }
            }
            if (__any_sync(0xFFFFFFFFu, odd)) {
                float* pr = reinterpret_cast<float*>(qf);               // [16 rows][64 drafted tokens]; the unit's last use of qf
                __syncwarp();
                if (t >= 2) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
#pragma unroll
                        for (int c = 0; c < 4; ++c) pr[(g + 8 * (c >> 1)) * 64 + 16 * (2 * t + (c & 1)) + j - BLK] = s[j][c];
                }
                __syncwarp();
                const uint8_t* seen = p.tree + b * p.tree_stride;
                for (int d = 0; d < p.T; ++d) {
                    const uint16_t* v = reinterpret_cast<const uint16_t*>(p.vd) + ((b * p.T + d) * p.H + h) * D;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int r = row0 + g + 8 * i;
                        if (r >= R || !seen[(long long)(r / p.G) * p.T + d]) continue;
                        const float pd = pr[(g + 8 * i) * 64 + d];
#pragma unroll
                        for (int j = 0; j < N; ++j)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const uint16_t y = v[N * (2 * t + c) + j];
                                if ((y & 0x7C00u) == 0x7C00u) o[j][2 * i + c] += pd * __half2float(__ushort_as_half(y));
                            }
                    }
                }
                __syncwarp();
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 1);
            l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 2);
            const int r = row0 + g + 8 * i;
            if (r >= R) continue;
            if (t0 == 0 && t1 == p.tiles) {
                const long long row = (b * p.T + r / p.G) * p.H * p.G + (long long)h * p.G + r % p.G;
                const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
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
                // record of this warp: its first unit in slot 0, its last in slot 1 (those between are whole)
                const int slot = unit != first / p.tiles;
                float* rec = p.part + ((2 * w + slot) * ROWS + g + 8 * i) * (D + 4);
                if (t == 0) {
                    rec[0] = m[i];
                    rec[1] = l[i];
                }
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int v = 0; v < N / 4; ++v)
                        reinterpret_cast<float4*>(rec + 4 + N * (2 * t + c))[v] =
                            make_float4(o[4 * v][2 * i + c], o[4 * v + 1][2 * i + c], o[4 * v + 2][2 * i + c],
                                        o[4 * v + 3][2 * i + c]);
            }
        }
        at = unit * p.tiles + t1;
        __syncwarp();
    }
}

// Warp that holds tile i when `total` tiles are dealt to nw warps: the largest w with floor(w total / nw) <= i.
__device__ __forceinline__ long long warp_of(long long i, long long total, long long nw) { return ((i + 1) * nw - 1) / total; }

// One warp per query row: the records of the warps that share its unit, in the order of the tokens.
template <int D>
__global__ void __launch_bounds__(128) tree_merge_kernel(const TreeArgs p) {
    pdl_enter();
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);       // unit * 16 + row of the unit
    const long long unit = row / ROWS, bh = unit / p.rt, b = bh / p.H;
    if (unit * p.tiles >= p.total) return;
    const int h = (int)(bh - b * p.H), r = (int)(unit - bh * p.rt) * ROWS + (int)(row % ROWS);
    if (r >= p.T * p.G) return;
    const long long w0 = warp_of(unit * p.tiles, p.total, p.nw), w1 = warp_of(unit * p.tiles + p.tiles - 1, p.total, p.nw);
    if (w0 == w1) return;                                                       // a whole unit: written by its warp
    auto record = [&](long long w) {
        const int slot = unit != (w * p.total / p.nw) / p.tiles;
        return p.part + ((2 * w + slot) * ROWS + row % ROWS) * (D + 4);
    };
    float top = -INFINITY;
    for (long long w = w0 + lane; w <= w1; w += 32) top = fmaxf(top, record(w)[0]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    const float base = top == -INFINITY ? 0.f : top;
    constexpr int C = D / 32;
    float acc[C], l = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = 0.f;
#pragma unroll 4
    for (long long w = w0; w <= w1; ++w) {
        const float* rec = record(w);
        const float f = ex2(rec[0] - base);
        l = fmaf(f, rec[1], l);
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] = fmaf(f, rec[4 + C * lane + c], acc[c]);
    }
    const long long to = (b * p.T + r / p.G) * p.H * p.G + (long long)h * p.G + r % p.G;
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < C; c += 2)
        *reinterpret_cast<uint32_t*>(p.out + to * D + C * lane + c) = pack_half2(acc[c] * inv, acc[c + 1] * inv);
    if (p.lse && lane == 0) p.lse[to] = l == 0.f ? -INFINITY : (base - LIFT + log2f(l)) * LN2;
}

// A warp per 128 cached tokens of a (batch, KV head); all query rows of the head, 16 at a time, added in their order.
template <int D>
__global__ void __launch_bounds__(32 * WARPS, 1) weights_kernel(const TreeArgs p, float* __restrict__ weights) {
    __shared__ __align__(16) uint4 frag[WARPS][256];
    pdl_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int R = p.T * p.G, full = (p.nb + 1) >> 1;
    uint4* qf = frag[warp];
    for (long long at = (long long)warp * gridDim.x + blockIdx.x; at < p.total; at += p.nw) {
        const long long bh = at / p.tiles, b = bh / p.H;
        const int h = (int)(bh - b * p.H), tile = (int)(at - bh * p.tiles);
        const bool tail = tile == full;
        const int start = tail ? p.nb * BLK : tile * TILE, count = tail ? p.rest : min(TILE, p.nb * BLK - start);
        const __half* mask = p.mask ? p.mask + b * p.mask_stride : nullptr;
        float sum[16][2];
#pragma unroll
        for (int j = 0; j < 16; ++j) sum[j][0] = sum[j][1] = 0.f;
#pragma unroll 1
        for (int row0 = 0; row0 < R; row0 += ROWS) {
            load_q<D>(qf, p, b, h, row0, lane);
            float s[16][4], off[2];
            if (tail) tail_scores<D>(s, qf, p, b, h, lane);
            else plane_scores<D>(s, qf, p, bh, tile, lane);
            scale_mask(s, p, mask, start, count, t);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = row0 + g + 8 * i;
                off[i] = -INFINITY;
                if (r < R) off[i] = p.lse[(b * p.T + r / p.G) * p.H * p.G + (long long)h * p.G + r % p.G] * LOG2E;
#pragma unroll
                for (int j = 0; j < 16; ++j)
#pragma unroll
                    for (int c = 0; c < 2; ++c)        // (a row that sees nothing has lse = -inf)
                        if (off[i] != -INFINITY && s[j][2 * i + c] != -INFINITY) sum[j][c] += ex2(s[j][2 * i + c] - off[i]);
            }
        }
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) sum[j][c] += __shfl_xor_sync(0xFFFFFFFFu, sum[j][c], o);
                const int tok = 16 * (2 * t + c) + j;
                if (g == (j >> 1) && tok < count) weights[bh * p.L + start + tok] += sum[j][c];
            }
    }
}

// Warps for `total` tiles: one an SM while there are that few, then up to eight.
struct Deal {
    int grid, wpc;
    long long warps;
};
Deal deal(long long total) {
    const int sms = sm_count();
    Deal d;
    d.grid = (int)(total < sms ? total : sms);
    const long long per = (total + d.grid - 1) / d.grid;
    d.wpc = (int)(per < WARPS ? per : WARPS);
    d.warps = total < (long long)d.grid * d.wpc ? total : (long long)d.grid * d.wpc;
    return d;
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
    AKV_REQUIRE((long long)a->bsz * a->n_kv_heads * a->group < (1ll << 30) / BLK, AKV_ERR_OVERFLOW, "%s: too many rows", fn);
    AKV_REQUIRE(!mask || mask_stride >= 0, AKV_ERR_SHAPE, "%s: negative mask stride", fn);
    AKV_REQUIRE(aligned16(a->k_first_8) && aligned16(a->k_mid_4) && aligned16(a->k_last_4) && aligned16(a->v_first_8) &&
                aligned16(a->v_mid_4) && aligned16(a->v_last_4) && aligned16(a->restk) && aligned16(a->restv) && aligned16(q),
                AKV_ERR_ALIGN, "%s: pointers must be 16-byte aligned", fn);
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
    p.scale2 = scale * LOG2E;
    return p;
}

}  // namespace
}  // namespace akv

using namespace akv;

extern "C" {

long long akv_tree_scratch_bytes(int bsz, int n_kv_heads, int group, int head_dim, int n_tokens, int drafted) {
    if (bsz <= 0 || n_kv_heads <= 0 || group <= 0 || (head_dim != 64 && head_dim != 128) || n_tokens < 0 || drafted < 1 ||
        drafted > BLK)
        return -1;
    const long long units = (long long)bsz * n_kv_heads * (((long long)drafted * group + ROWS - 1) / ROWS);
    const Deal d = deal(units * ((n_tokens / BLK + 1) / 2 + 1));
    return 2 * d.warps * ROWS * (head_dim + 4) * 4;
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
    p.rt = (drafted * p.G + ROWS - 1) / ROWS;
    p.tiles = (p.nb + 1) / 2 + 1;
    const long long units = (long long)layer->bsz * p.H * p.rt;
    p.total = units * p.tiles;
    const Deal d = deal(p.total);
    p.nw = d.warps;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    launch_chained(D == 128 ? tree_kernel<128> : tree_kernel<64>, dim3(d.grid), dim3(32 * d.wpc), 0, st, p);
    rc = cuda_status(cudaGetLastError(), "tree_attention launch");
    if (rc != AKV_OK || p.tiles == 1) return rc;                 // (units of one tile: none is shared)
    launch_chained(D == 128 ? tree_merge_kernel<128> : tree_merge_kernel<64>, dim3((unsigned)(units * (ROWS / 4))), dim3(128), 0, st,
                   p);
    return cuda_status(cudaGetLastError(), "tree_attention merge launch");
}

int akv_tree_weights(const akv_layer* layer, const void* q, const void* lse, const void* mask, long long mask_stride,
                     void* weights, int drafted, int rest_len, int rest_start, float scale, void* stream) {
    set_error("");
    int rc = check_layer("tree_weights", layer, q, drafted, rest_len, rest_start, mask, mask_stride);
    if (rc != AKV_OK) return rc;
    AKV_REQUIRE(lse && weights, AKV_ERR_NULL, "tree_weights: null pointer");
    TreeArgs p = make_args(layer, q, drafted, rest_len, rest_start, mask, mask_stride, scale);
    p.lse = static_cast<float*>(const_cast<void*>(lse));
    p.tiles = (p.nb + 1) / 2 + (rest_len > 0);
    p.total = (long long)layer->bsz * p.H * p.tiles;
    if (p.total == 0) return AKV_OK;
    const Deal d = deal(p.total);
    p.nw = (long long)d.grid * d.wpc;
    launch_chained(layer->head_dim == 128 ? weights_kernel<128> : weights_kernel<64>, dim3(d.grid), dim3(32 * d.wpc), 0,
                   static_cast<cudaStream_t>(stream), p, static_cast<float*>(weights));
    return cuda_status(cudaGetLastError(), "tree_weights launch");
}

}  // extern "C"
