// What enters and leaves the plane cache beside the decode step.
//   commit_kernel    the accepted path of a tree of drafted tokens: the state that one append after the other leaves
//   select_kernel    per (batch, KV head): the `keep` heaviest plane tokens, and with them who moves where
//   move_kernel      survivors behind `keep` into the places that became free in front of it
//   clear_kernel     K nibble planes, weights behind the survivors
#include <limits.h>

#include "akv_planes.cuh"
#include "akv_save.cuh"

namespace akv {
namespace {

constexpr int BLK = 64;
constexpr int MOST_ROWS = 65535;                       // (batch, KV head) rows: along the grid's y

// ------------------------------------------------------------------ accepted path
// CTA = (batch, KV head) and one of K, V.  Rows in front of the accepted tokens: the residual buffer.  The two together are at most
// 127 rows: one block fills up at most, its rows go to the planes, and the rows behind it begin the next residual block.
// All rows that matter are requested at once and staged in shared memory; maxima, planes and residual rows are made from there.
// Bound by latency: one load, one barrier, one store.  (Maxima read row after row from global memory took 29 us at 512 heads and 48
// tokens.)
constexpr int COMMIT_NT = 256;
template <int D>
__global__ void __launch_bounds__(COMMIT_NT)
commit_kernel(uint8_t* __restrict__ f8, uint8_t* __restrict__ m4, uint8_t* __restrict__ l4, uint8_t* __restrict__ vf8,
              uint8_t* __restrict__ vm4, uint8_t* __restrict__ vl4, uint16_t* __restrict__ k_exp, uint16_t* __restrict__ v_exp,
              uint8_t* restk, uint8_t* restv, const uint8_t* __restrict__ kd, const uint8_t* __restrict__ vd,
              const int* __restrict__ path, int H, int T, int n, int rest, int qn, int nmb, int L) {
    constexpr int PITCH = 2 * D, VEC = D / 8, HD = D / 2;
    extern __shared__ __align__(16) uint8_t rows[];     // [row from `first` on][D] fp16
    __shared__ uint32_t part[COMMIT_NT];
    pdl_enter();
    const int bh = blockIdx.x, b = (unsigned)bh / (unsigned)H, h = bh - b * H, tid = threadIdx.x;
    const bool value = blockIdx.y, full = rest + n >= BLK;
    uint8_t* buffer = value ? restv : restk;
    const uint8_t* drafted = value ? vd : kd;
    const int first = full ? 0 : rest, count = rest + n - first;      // (without a full block the residual rows stay where they are)
    auto slot = [&](int i) { return buffer + ((size_t)(b * BLK + i) * H + h) * PITCH; };
#pragma unroll 4
    for (int i = tid; i < count * VEC; i += COMMIT_NT) {
        const int r = first + i / VEC, v = i % VEC;
        // (a node outside the tree is clamped into it; rows of the residual buffer are written further down: no read-only loads)
        const uint8_t* src = r < rest ? slot(r)
                                      : drafted + ((size_t)(b * T + min(max(path[b * n + r - rest], 0), T - 1)) * H + h) * PITCH;
        *reinterpret_cast<uint4*>(rows + i * 16) = *(reinterpret_cast<const uint4*>(src) + v);
    }
    __syncthreads();
    // exponent maxima, two channels a word, the tokens dealt to COMMIT_NT / HD shares
    uint32_t m = 0;
    for (int i = rest - first + tid / HD; i < count; i += COMMIT_NT / HD) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(rows + i * PITCH)[tid % HD];
        m = __vmaxu4(m, ((w >> 10) & 0x1Fu) | (((w >> 26) & 0x1Fu) << 8));
    }
    part[tid] = m;
    __syncthreads();
    if (tid < HD) {
        uint16_t* top = (value ? v_exp : k_exp) + (size_t)bh * HD + tid;
#pragma unroll
        for (int j = 1; j < COMMIT_NT / HD; ++j) m = __vmaxu4(m, part[j * HD + tid]);
        *top = (uint16_t)__vmaxu4(m, *top);
    }
    if (full) {
        const size_t block = (size_t)bh * nmb + qn / BLK;
        for (int i = tid; i < 2 * D; i += COMMIT_NT) {
            if (!value) {
                // 32 tokens of a channel
                const int c = i % D, t0 = i / D * 32;
                uint4 hi[2], mid, low;
                uint32_t *hw = reinterpret_cast<uint32_t*>(hi), *mw = reinterpret_cast<uint32_t*>(&mid), *lw = reinterpret_cast<uint32_t*>(&low);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint8_t* x = rows + (t0 + 8 * g + 2 * j) * PITCH + 2 * c;
                        w[j] = *reinterpret_cast<const uint16_t*>(x) | (uint32_t)*reinterpret_cast<const uint16_t*>(x + PITCH) << 16;
                    }
                    v_split4(w[0], w[1], w[2], w[3], hw[2 * g], hw[2 * g + 1], mw[g], lw[g]);
                }
                uint4* f = reinterpret_cast<uint4*>(f8 + (block * D + c) * BLK + t0);
                f[0] = hi[0];
                f[1] = hi[1];
                *reinterpret_cast<uint4*>(m4 + (block * D + c) * (BLK / 2) + t0 / 2) = mid;
                *reinterpret_cast<uint4*>(l4 + (block * D + c) * (BLK / 2) + t0 / 2) = low;
            } else {
                // 32 channels of a token
                const int r = i / (D / 32), c = i % (D / 32);
                const uint4* src = reinterpret_cast<const uint4*>(rows + r * PITCH + c * 64);
                const size_t to = (size_t)bh * L + qn + r;
                v_write32(src[0], src[1], src[2], src[3], vf8 + to * D + c * 32, vm4 + to * HD + c * 16, vl4 + to * HD + c * 16);
            }
        }
    }
    const int from = full ? BLK : rest - first;         // staged row that goes to residual row `at`
    const int at = full ? 0 : rest;
    for (int i = tid; i < (count - from) * VEC; i += COMMIT_NT)
        reinterpret_cast<uint4*>(slot(at + i / VEC))[i % VEC] = *reinterpret_cast<const uint4*>(rows + from * PITCH + i * 16);
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
    int *holes, *movers, *start;       // [rows][most] twice; [rows][keep / 64 + 1]: free places in front of each block's
    int D, L, nmb, n, rest, keep, recent, arranged, shift, most;
    int share;                         // places of a CTA of select_kernel's cluster, a multiple of its threads
    int held;                          // whether their keys are kept in shared memory
};

__device__ __forceinline__ int position_of(const EvictArgs& a, const int* pos, int i) { return i < a.arranged ? pos[i] : i + a.shift; }

// A word of another CTA's shared memory.
__device__ __forceinline__ uint32_t cluster_ld(const void* p, uint32_t cta) {
    uint32_t at, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(smem_u32(p)), "r"(cta));
    asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(at) : "memory");
    return v;
}

// A cluster per row; a CTA has `share` consecutive places and keeps their keys in shared memory: one read of the weights, whatever is
// counted.  The keep-th largest key by four counts of eight bits (in eight columns: few lanes of a warp meet, although weights crowd into
// few exponents), added up over the cluster through distributed shared memory; every CTA draws the same
// conclusion.  Then ties, free places and survivors behind are numbered in order: per warp, per CTA, per cluster.  Bound by latency: a
// load, four rounds of six barriers (one of them the cluster's), three numberings (256 rows of 4096: 18 us of 144; 8 rows of 131072: 32 of 137).
constexpr int SEL_MOST = 40960, SEL_CTAS = 8;      // keys a CTA can keep, CTAs of a row
template <int SEL_NT>
__global__ void __launch_bounds__(SEL_NT) select_kernel(const EvictArgs a) {
    constexpr int SEL_W = SEL_NT / 32;
    extern __shared__ __align__(16) uint32_t keys[];
    __shared__ int hist[8 * 257];                  // [column][digit], columns a bank apart
    __shared__ uint32_t sums[2][256];              // this CTA's counts: two buffers, so that one barrier a round is enough
    __shared__ uint32_t found[2], warp_sum[8], scan[3][SEL_W + 1], totals[2][2];
    pdl_enter();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t ctas, rank;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    auto sync_all = [&] {                              // (a cluster's barrier for one CTA costs 2 us of a call)
        if (ctas == 1) __syncthreads();
        else cluster_sync();
    };
    const size_t row = blockIdx.y;
    const float* w = a.weights + row * a.L;
    int* pos = a.positions + row * a.L;
    const int safe_from = a.n + a.shift - a.recent;
    const int first = min((int)rank * a.share, a.n), count = min(a.share, a.n - first);
    auto key = [&](int i) { return key_of(w[first + i], a.recent && position_of(a, pos, first + i) >= safe_from); };
    if (a.held) {
        // (eight at a time: all weights requested, then the positions that matter, then used)
#pragma unroll 1
        for (int i0 = tid; i0 < count; i0 += 8 * SEL_NT) {
            float x[8];
            int at[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = i0 + j * SEL_NT < count ? w[first + i0 + j * SEL_NT] : 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int i = first + i0 + j * SEL_NT;
                at[j] = i + a.shift;
                if (a.recent && i < a.arranged && i0 + j * SEL_NT < count) at[j] = pos[i];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i0 + j * SEL_NT < count) keys[i0 + j * SEL_NT] = key_of(x[j], a.recent && at[j] >= safe_from);
        }
    }
    auto at = [&](int i) { return a.held ? keys[i] : key(i); };
    uint32_t prefix = 0;
    uint32_t want = a.keep;                            // how many of the keys that share the prefix stay
    for (int round = 0; round < 4; ++round) {
        const int bit = 24 - 8 * round;
        for (int i = tid; i < 8 * 257; i += SEL_NT) hist[i] = 0;
        __syncthreads();
#pragma unroll 4
        for (int i = tid; i < count; i += SEL_NT) {
            const uint32_t k = at(i);
            if (round == 0 || (k >> (bit + 8)) == (prefix >> (bit + 8))) atomicAdd(&hist[(lane & 7) * 257 + ((k >> bit) & 255)], 1);
        }
        __syncthreads();
        if (tid < 256) {
            uint32_t c = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) c += hist[j * 257 + tid];
            sums[round & 1][tid] = c;
        }
        sync_all();
        // thread: digit 255 - tid; keys with a larger one, by the sums of the lanes and warps in front
        uint32_t c = 0, above = 0;
        if (tid < 256) {
            if (ctas == 1) c = sums[round & 1][255 - tid];
            else
                for (uint32_t r = 0; r < ctas; ++r) c += cluster_ld(&sums[round & 1][255 - tid], r);
            above = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, above, o);
                if (lane >= o) above += x;
            }
            if (lane == 31) warp_sum[warp] = above;
            above -= c;
        }
        __syncthreads();
        if (tid < 256) {
            for (int j = 0; j < warp; ++j) above += warp_sum[j];
            if (above < want && above + c >= want) {
                found[0] = 255 - tid;
                found[1] = above;
            }
        }
        __syncthreads();
        prefix |= found[0] << bit;
        want -= found[1];
        __syncthreads();
    }
    // A warp's places: share / 32 consecutive ones.  Numbers in front of it: `scan` of the CTA's warps, `base` of the CTAs before.
    const int part = a.share / SEL_W, i0 = warp * part, i1 = min(i0 + part, count);
    const uint32_t below = (1u << lane) - 1;
    auto number = [&](int s, uint32_t mine) {          // (lane 0: exclusive sums of the warps' counts)
        if (lane == 0) scan[s][warp] = mine;
        __syncthreads();
        if (warp == 0) {
            uint32_t x = lane < SEL_W ? scan[s][lane] : 0, y = x;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t z = __shfl_up_sync(0xFFFFFFFFu, y, o);
                if (lane >= o) y += z;
            }
            if (lane < SEL_W) scan[s][lane] = y - x;
            if (lane == 31) scan[s][SEL_W] = y;
        }
        __syncthreads();
    };
    uint32_t ties = 0;
    for (int i = i0; i < i1; i += 32) ties += __popc(__ballot_sync(0xFFFFFFFFu, i + lane < i1 && at(i + lane) == prefix));
    number(0, ties);
    if (tid == 0) totals[0][0] = scan[0][SEL_W];
    sync_all();
    uint32_t tie0 = scan[0][warp];
    for (uint32_t r = 0; r < rank; ++r) tie0 += cluster_ld(&totals[0][0], r);
    // (bits: the place's token stays; as many words as the warp has groups of 32, in the same order twice)
    uint32_t holes = 0, movers = 0, seen = tie0;
    auto stays = [&](int i, uint32_t& before) {
        const uint32_t k = i + lane < i1 ? at(i + lane) : 0;
        const bool tie = i + lane < i1 && k == prefix;
        const uint32_t tb = __ballot_sync(0xFFFFFFFFu, tie);
        const bool s = i + lane < i1 && (k > prefix || (tie && before + __popc(tb & below) < want));
        before += __popc(tb);
        return s;
    };
    for (int i = i0; i < i1; i += 32) {
        const bool s = stays(i, seen);
        const int place = first + i + lane;
        holes += __popc(__ballot_sync(0xFFFFFFFFu, i + lane < i1 && !s && place < a.keep));
        movers += __popc(__ballot_sync(0xFFFFFFFFu, s && place >= a.keep));
    }
    number(1, holes);
    number(2, movers);
    if (tid == 0) {
        totals[1][0] = scan[1][SEL_W];
        totals[1][1] = scan[2][SEL_W];
    }
    sync_all();
    uint32_t h = scan[1][warp], m = scan[2][warp];
    for (uint32_t r = 0; r < rank; ++r) {
        h += cluster_ld(&totals[1][0], r);
        m += cluster_ld(&totals[1][1], r);
    }
    int *hole_to = a.holes + row * a.most, *mover_to = a.movers + row * a.most, *start = a.start + row * (a.keep / BLK + 1);
    seen = tie0;
    for (int i = i0; i < i1; i += 32) {
        const bool s = stays(i, seen);
        const int place = first + i + lane;
        const bool hole = i + lane < i1 && !s && place < a.keep, mover = s && place >= a.keep;
        const uint32_t hb = __ballot_sync(0xFFFFFFFFu, hole), mb = __ballot_sync(0xFFFFFFFFu, mover);
        if (lane == 0 && place % BLK == 0 && place <= a.keep) start[place / BLK] = h;
        if (hole) hole_to[h + __popc(hb & below)] = place;
        if (mover) mover_to[m + __popc(mb & below)] = place;
        if (s && place < a.keep && place >= a.arranged) pos[place] = place + a.shift;
        h += __popc(hb);
        m += __popc(mb);
    }
    if (a.keep == a.n && rank == 0 && tid == 0) start[a.keep / BLK] = 0;      // (no place behind: nothing moves)
    sync_all();                                    // (no CTA leaves while another reads its counts)
}

// CTA = one block of 64 places in front of `keep`: its free places take the survivors of the same numbers.  Survivors are read
// only behind `keep` and places are written only in front of it, each by its own CTA: no order among the CTAs.
// K, token-minor: one survivor is a byte of each of D rows and half a byte of 2 D.  The block and the blocks that its survivors come
// from are put together to fp16 rows [channel][64 tokens] in shared memory, the latter one after the other; a warp takes a channel, a lane
// two neighbouring places, a survivor's value is one 2-byte load and store; at the end the block is split again.  (On the plane bytes
// themselves that were three loads and, with the neighbour's nibble in the same byte, more than one store per value: shared memory's
// pipe was 69% busy at 142 us for 8 x 32 x 4096 tokens to 2048.)  V: rows of 16-byte pieces through registers.
// Floor: the block twice, the blocks behind once, V's rows twice.
constexpr int MOVE_NT = 256, STAGED = 1;
template <int D>
__global__ void __launch_bounds__(MOVE_NT) move_kernel(const EvictArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];     // blocks of [D] rows of 128 bytes, 16-byte piece q of row c at q ^ (c & 1)
    __shared__ int from[BLK], to[BLK], src[BLK];
    constexpr int BYTES = D * 128, PIECES = D / 8, PER = BLK * PIECES / MOVE_NT, U = D * 4 / MOVE_NT;
    pdl_enter();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const size_t row = blockIdx.y;
    const int blk = blockIdx.x;
    const int* start = a.start + row * (a.keep / BLK + 1) + blk;
    const int i0 = start[0], m = start[1] - i0;
    if (m <= 0) return;
    // thread: 16 tokens of U channels of a block
    struct Bytes { uint4 h[U]; uint2 m[U], l[U]; };
    auto load = [&](Bytes& x, int b) {
        const size_t at = (row * a.nmb + b) * D;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t o = at * 4 + tid + u * MOVE_NT;
            x.h[u] = reinterpret_cast<const uint4*>(a.k8)[o];
            x.m[u] = reinterpret_cast<const uint2*>(a.km)[o];
            x.l[u] = reinterpret_cast<const uint2*>(a.kl)[o];
        }
    };
    auto place = [&](int u) {                           // of the first of the thread's two pieces
        const int i = tid + u * MOVE_NT, c = i >> 2;
        return c * 128 + (((2 * (i & 3)) ^ (c & 1)) << 4);
    };
    auto put = [&](const Bytes& x, int of) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int o = place(u);
            *reinterpret_cast<uint4*>(smem + of * BYTES + o) = halves8(x.h[u].x, x.h[u].y, x.m[u].x, x.l[u].x);
            *reinterpret_cast<uint4*>(smem + of * BYTES + (o ^ 16)) = halves8(x.h[u].z, x.h[u].w, x.m[u].y, x.l[u].y);
        }
    };
    Bytes mine, other[STAGED];
    load(mine, blk);
    if (tid < BLK) from[tid] = -1;
    __syncthreads();
    if (tid < m) {
        const int d = a.holes[row * a.most + i0 + tid], s = a.movers[row * a.most + i0 + tid];
        to[tid] = d;
        src[tid] = s;
        from[d - blk * BLK] = s;
        a.weights[row * a.L + d] = a.weights[row * a.L + s];
        a.positions[row * a.L + d] = position_of(a, a.positions + row * a.L, s);
    }
    __syncthreads();
    const int b0 = src[0] >> 6, b1 = src[m - 1] >> 6;   // (survivors ascend)
#pragma unroll
    for (int e = 0; e < STAGED; ++e)
        if (b0 + e <= b1) load(other[e], b0 + e);
    // V: thread = one 16-byte piece, of which plane is the same for all rows
    const int piece = tid % PIECES, j0 = tid / PIECES;
    const int pitch = piece < D / 16 ? D : D / 2;
    uint8_t* vp = (piece < D / 16 ? a.v8 + piece * 16 : piece < D * 3 / 32 ? a.vm + (piece - D / 16) * 16 : a.vl + (piece - D * 3 / 32) * 16) +
                  row * a.L * pitch;
    uint4 v[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int j = j0 + e * (MOVE_NT / PIECES);
        if (j < m) v[e] = *reinterpret_cast<const uint4*>(vp + (size_t)src[j] * pitch);
    }
    put(mine, 0);
    const int s0 = from[2 * lane], s1 = from[2 * lane + 1], swap = (warp & 1) << 4;      // (a warp's channels are all odd or all even)
    for (int b = b0; b <= b1; b += STAGED) {
#pragma unroll
        for (int e = 0; e < STAGED; ++e)
            if (b + e <= b1) put(other[e], 1 + e);
        __syncthreads();
#pragma unroll
        for (int e = 0; e < STAGED; ++e)
            if (b + STAGED + e <= b1) load(other[e], b + STAGED + e);
        const int r0 = s0 < 0 ? -1 : (s0 >> 6) - b, r1 = s1 < 0 ? -1 : (s1 >> 6) - b;
        const uint8_t *x0 = smem + (1 + r0) * BYTES + ((2 * (s0 & 63)) ^ swap), *x1 = smem + (1 + r1) * BYTES + ((2 * (s1 & 63)) ^ swap);
        uint8_t* y = smem + ((4 * lane) ^ swap);
        const bool t0 = r0 >= 0 && r0 < STAGED, t1 = r1 >= 0 && r1 < STAGED;
#pragma unroll 4
        for (int c = warp; c < D; c += MOVE_NT / 32) {
            if (t0) *reinterpret_cast<uint16_t*>(y + c * 128) = *reinterpret_cast<const uint16_t*>(x0 + c * 128);
            if (t1) *reinterpret_cast<uint16_t*>(y + c * 128 + 2) = *reinterpret_cast<const uint16_t*>(x1 + c * 128);
        }
        __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int j = j0 + e * (MOVE_NT / PIECES);
        if (j < m) *reinterpret_cast<uint4*>(vp + (size_t)to[j] * pitch) = v[e];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int o = place(u);
        const uint4 x = *reinterpret_cast<const uint4*>(smem + o), y = *reinterpret_cast<const uint4*>(smem + (o ^ 16));
        uint4 h;
        uint2 n, l;
        v_split4(x.x, x.y, x.z, x.w, h.x, h.y, n.x, l.x);
        v_split4(y.x, y.y, y.z, y.w, h.z, h.w, n.y, l.y);
        const size_t at = (row * a.nmb + blk) * D * 4 + tid + u * MOVE_NT;
        reinterpret_cast<uint4*>(a.k8)[at] = h;
        reinterpret_cast<uint2*>(a.km)[at] = n;
        reinterpret_cast<uint2*>(a.kl)[at] = l;
    }
}

// blockIdx.x == 0: the weights of the residual tokens follow the survivors, zeros behind them; else: K nibble planes of a freed
// block (the K writer adds nibbles, so a block is zero before it is written again).
__global__ void __launch_bounds__(256) clear_kernel(const EvictArgs a) {
    __shared__ float tail[BLK];
    pdl_enter();
    const size_t row = blockIdx.y;
    const int tid = threadIdx.x;
    if (blockIdx.x == 0) {
        float* w = a.weights + row * a.L;
        if (tid < a.rest) tail[tid] = w[a.n + tid];
        __syncthreads();
        for (int i = a.keep + tid; i < a.n + a.rest; i += 256) w[i] = i - a.keep < a.rest ? tail[i - a.keep] : 0.f;
        return;
    }
    const size_t at = (row * a.nmb + a.keep / BLK + blockIdx.x - 1) * (size_t)a.D * 2;
    for (int i = tid; i < a.D * 2; i += 256) {
        reinterpret_cast<uint4*>(a.km)[at + i] = make_uint4(0, 0, 0, 0);
        reinterpret_cast<uint4*>(a.kl)[at + i] = make_uint4(0, 0, 0, 0);
    }
}

// Threads: 512 where a CTA has few keys, so that two rows share an SM; 1024 for long ones.
int launch_select(const EvictArgs& a, int rows, int ctas, int threads, cudaStream_t st) {
    const size_t smem = a.held ? (size_t)a.share * 4 : 0;
    auto kernel = threads == 512 ? select_kernel<512> : select_kernel<1024>;
    int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SEL_MOST * 4),
                         "evict select shared memory");
    if (rc != AKV_OK) return rc;
    return cuda_status(launch_cluster(kernel, ctas, dim3(ctas, rows), dim3(threads), smem, st, a), "evict select launch");
}

int check_planes(const char* fn, const akv_layer* a) {
    AKV_REQUIRE(a && a->k_first_8 && a->k_mid_4 && a->k_last_4 && a->v_first_8 && a->v_mid_4 && a->v_last_4, AKV_ERR_NULL,
                "%s: null pointer", fn);
    AKV_REQUIRE(a->bsz > 0 && a->n_kv_heads > 0 && (a->head_dim == 64 || a->head_dim == 128) && a->max_seq_len > 0 &&
                a->max_seq_len <= INT_MAX - 128, AKV_ERR_SHAPE,
                "%s: unsupported extent (bsz %d, KV heads %d, head_dim %d [64 or 128], max_seq_len %d)", fn, a->bsz, a->n_kv_heads,
                a->head_dim, a->max_seq_len);
    AKV_REQUIRE((long long)a->bsz * a->n_kv_heads <= MOST_ROWS, AKV_ERR_OVERFLOW, "%s: more than %d (batch, KV head) rows", fn, MOST_ROWS);
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
    const int D = a.head_dim, staged = rest_len + accepted >= BLK ? rest_len + accepted : accepted;
    launch_chained(D == 128 ? commit_kernel<128> : commit_kernel<64>, dim3(a.bsz * a.n_kv_heads, 2), dim3(COMMIT_NT),
                   (size_t)staged * 2 * D, static_cast<cudaStream_t>(stream), static_cast<uint8_t*>(a.k_first_8),
                   static_cast<uint8_t*>(a.k_mid_4), static_cast<uint8_t*>(a.k_last_4), static_cast<uint8_t*>(a.v_first_8),
                   static_cast<uint8_t*>(a.v_mid_4), static_cast<uint8_t*>(a.v_last_4), static_cast<uint16_t*>(a.k_exp_max),
                   static_cast<uint16_t*>(a.v_exp_max), static_cast<uint8_t*>(a.restk), static_cast<uint8_t*>(a.restv),
                   static_cast<const uint8_t*>(k_new), static_cast<const uint8_t*>(v_new), static_cast<const int*>(path),
                   a.n_kv_heads, drafted, accepted, rest_len, rest_start, (a.max_seq_len + BLK - 1) / BLK, a.max_seq_len);
    return cuda_status(cudaGetLastError(), "tree_commit launch");
}

long long akv_evict_scratch_bytes(int bsz, int n_kv_heads, int n_tokens, int keep) {
    if (bsz <= 0 || n_kv_heads <= 0 || (long long)bsz * n_kv_heads > MOST_ROWS || keep <= 0 || keep > n_tokens) return -1;
    const long long most = keep < n_tokens - keep ? keep : n_tokens - keep;
    return (long long)bsz * n_kv_heads * (2 * most + keep / BLK + 1) * 4;
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
    a.holes = static_cast<int*>(l.scratch);
    a.movers = a.holes + (size_t)rows * a.most;
    a.start = a.movers + (size_t)rows * a.most;
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
    // CTAs of a row: twice as many, up to eight (what a cluster may have everywhere), while one has more places than it can keep the keys
    // of, or more than 2048 and some SMs have none
    int ctas = 1;
    while (ctas < SEL_CTAS && ((rest_start + ctas - 1) / ctas > SEL_MOST || (rows * ctas < sm_count() && rest_start / ctas > 2048))) ctas *= 2;
    const int threads = (rest_start + ctas - 1) / ctas > 8192 ? 1024 : 512;
    a.share = ((rest_start + ctas - 1) / ctas + threads - 1) / threads * threads;
    a.held = a.share <= SEL_MOST;
    if ((rc = launch_select(a, rows, ctas, threads, st)) != AKV_OK || keep == rest_start) return rc;
    const size_t smem = (size_t)(1 + STAGED) * l.head_dim * 128;
    auto move = l.head_dim == 128 ? move_kernel<128> : move_kernel<64>;
    rc = cuda_status(cudaFuncSetAttribute(move, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "evict shared memory");
    if (rc != AKV_OK) return rc;
    launch_chained(move, dim3(keep / BLK, rows), dim3(MOVE_NT), smem, st, a);
    if ((rc = cuda_status(cudaGetLastError(), "evict move launch")) != AKV_OK) return rc;
    launch_chained(clear_kernel, dim3(1 + (rest_start - keep) / BLK, rows), dim3(256), 0, st, a);
    return cuda_status(cudaGetLastError(), "evict clear launch");
}

}  // extern "C"
