// Which drafted tokens are accepted, and the token behind them, such that what comes out has the target's distribution.
//
// At an accepted node with target probabilities p and draft probabilities q its children, drawn from q, are asked in order: x is accepted
// with probability min(1, r(x) / (Z q(x))), r = max(p - c q, 0), c = 0 and Z = 1 at first.  A rejection leaves the residual max(r / Z - q, 0),
// normalised; times Z that is max(p - (c + Z) q, 0), since max(max(a, 0) - b, 0) = max(a - b, 0) for b >= 0.  So the residual after any number of
// rejections is one coefficient, and the tests are u Z q(x) < r(x) with Z = sum r.  Without q a child is a guess of probability one:
// accepted with probability p(x) / Z, and its p leaves the row when it is not.  Where no child is left, the smallest j with
// cumsum(r)[j] > u_0 sum(r) follows.  Products and sums in 64 bits: a difference p - c q is one fused operation, off by 2^-53 of itself, a sum of V by V 2^-53
// at most, so that a border moves across a random number only where that comes as near to it.
// A walk forms one sum over a vocabulary for each rejection that another child asks after, each behind the one before it, and one for the last token: of a
// chain that one alone.  A cluster of up to 8 CTAs has a sequence; of 64 chains of 8 nodes, 131072 words in fp32 (four CTAs each), 20.8 us.  Stamps in it: 1.5 us until the
// nodes' numbers are there, 1.0 of walk (3.3 the longest), 8.5 of pass over a row of p and one of q (66 MB in all, at the rate of a copy), 1.6 until the
// cluster has its sum, 1.6 for the token; the median CTA is done after 14.4, those of the longest walks, whose pass begins last, after 20.  (A CTA a sequence
// 526 us; a cluster whose CTAs take each step of the walk together 49; a warp that walks by itself 31; now loads in batches too.)  8 x 32 guesses of 32000 words: 9.6 us,
// one sequence of 5 nodes 6.0.
#include <cuda_bf16.h>

#include "akv_common.cuh"

namespace akv {
namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32, MOST = 64, MOST_CTAS = 8;

template <class P>
struct ChooseArgs {
    const P *target, *draft;
    long long target_batch, target_row, draft_batch, draft_row, parents_batch;
    const long long* ids;
    const float* coins;
    const int* parents;
    int *path, *count;
    long long* token;
    int T, V, ctas;            // ctas: of a sequence's cluster
};

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
// What is no probability counts as none: negative, infinite, NaN (as bits all are above the largest finite value).
__device__ __forceinline__ float chance(float x) { return __float_as_uint(x) < 0x7F800000u ? x : 0.f; }
__device__ __forceinline__ double left_of(double p, double c, double q) {
    const double r = fma(-c, q, p);
    return r > 0.0 ? r : 0.0;
}

// E = 16 bytes of probabilities from j on (zeros behind `end`).  VEC: rows begin on 16-byte boundaries.
template <class P, bool VEC>
__device__ __forceinline__ uint4 load(const P* row, int j, int end) {
    constexpr int E = 16 / sizeof(P);
    uint4 w = make_uint4(0, 0, 0, 0);
    if (VEC && j + E <= end) return __ldg(reinterpret_cast<const uint4*>(row + j));
    P* e = reinterpret_cast<P*>(&w);
#pragma unroll
    for (int i = 0; i < E; ++i)
        if (j + i < end) e[i] = row[j + i];
    return w;
}
template <class P>
__device__ __forceinline__ float element(const uint4& w, int i) {
    return chance(as_float(reinterpret_cast<const P*>(&w)[i]));
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
    return x;
}
// Address of a shared variable of this CTA in another CTA of the cluster.
__device__ __forceinline__ uint32_t there(const void* p, int cta) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(smem_u32(p)), "r"(cta));
    return a;
}

// Bound by HBM where the batch is large (a row of p, one of q, read once by the cluster of the sequence and once more, of one warp's part, from
// L2), by latency where it is small: the numbers of the nodes, the row, two barriers.  The vocabulary is cut into contiguous parts, a
// warp's each, so that the sums of the parts in front of one tell where the random number falls.
template <class P, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) choose_kernel(ChooseArgs<P> a) {
    constexpr int E = 16 / sizeof(P), STEP = 32 * E;
    __shared__ double s_sum[WARPS], s_step[WARPS], s_cta[2][MOST_CTAS];
    __shared__ int s_up[MOST], s_x[MOST], s_first, s_mine;     // (s_x: -1 outside the vocabulary)
    __shared__ float s_p[MOST], s_q[MOST], s_u[MOST];
    const int ctas = a.ctas, rank = blockIdx.x % ctas, b = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int T = a.T, V = a.V;
    cluster_arrive();
    pdl_turn();
    const P* target = a.target + b * a.target_batch;
    const P* draft = a.draft ? a.draft + b * a.draft_batch : nullptr;
    if (tid < T) {
        const int up = tid == 0 ? -1 : a.parents ? a.parents[b * a.parents_batch + tid] : tid - 1;
        const long long x = a.ids[(long long)b * T + tid];
        const bool word = x >= 0 && x < V, asked = up >= 0 && up < tid && word;
        s_up[tid] = up < tid ? up : -1;
        s_x[tid] = word ? (int)x : -1;
        s_u[tid] = a.coins[(long long)b * T + tid];
        s_p[tid] = asked ? chance(as_float(target[up * a.target_row + x])) : 0.f;
        s_q[tid] = asked && draft ? chance(as_float(draft[up * a.draft_row + x])) : 0.f;
    }
    if (tid == 0) s_first = s_mine = V;
    __syncthreads();
    if (!draft && tid < T) {                   // a guess that was made and rejected before has nothing left
        bool twice = false;
        for (int k = 1; k < tid; ++k) twice |= s_up[k] == s_up[tid] && s_x[k] == s_x[tid];
        if (twice) s_p[tid] = 0.f;
    }
    __syncthreads();
    cluster_wait();                            // (all CTAs of the cluster run: total() stores into their shared memory)
    // parts of whole steps; this warp's begins at `first`
    const int steps = (V + STEP - 1) / STEP, each = (steps + ctas * WARPS - 1) / (ctas * WARPS);
    const int first = min(V, (rank * WARPS + warp) * each * STEP), last = min(V, first + each * STEP);
    int now = 0, count = 1, turn = 0;
    unsigned long long gone = 0;               // bits: guesses that were rejected at this node
    double c = 0.0, left = 1.0;
    if (tid == 0 && rank == 0) a.path[(long long)b * T] = 0;
    // what is left of E probabilities from j on, in the step that begins with j0
    auto rest = [&](double (&r)[E], int j, int j0, int end) {
        const uint4 x = load<P, VEC>(target + now * a.target_row, j, end);
        if (c > 0.0) {
            const uint4 y = load<P, VEC>(draft + now * a.draft_row, j, end);
#pragma unroll
            for (int i = 0; i < E; ++i) r[i] = left_of(element<P>(x, i), c, element<P>(y, i));
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) r[i] = element<P>(x, i);
            for (unsigned long long g = gone; g; g &= g - 1) {
                const int k = s_x[__ffsll(g) - 1] - j0;
                if (k >= 0 && k < STEP)
#pragma unroll
                    for (int i = 0; i < E; ++i)
                        if (k == j - j0 + i) r[i] = 0.0;
            }
        }
    };
    auto total = [&]() -> double {
        constexpr int BATCH = 4;               // steps whose loads are on their way together
        double sum = 0.0;
        int j0 = first;
        if (VEC && c > 0.0) {
            const P *x = target + now * a.target_row + lane * E, *y = draft + now * a.draft_row + lane * E;
#pragma unroll 1
            for (; j0 + BATCH * STEP <= last; j0 += BATCH * STEP) {
                uint4 p[BATCH], q[BATCH];
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                    p[k] = __ldg(reinterpret_cast<const uint4*>(x + j0 + k * STEP));
                    q[k] = __ldg(reinterpret_cast<const uint4*>(y + j0 + k * STEP));
                }
#pragma unroll
                for (int k = 0; k < BATCH; ++k)
#pragma unroll
                    for (int i = 0; i < E; ++i) sum += left_of(element<P>(p[k], i), c, element<P>(q[k], i));
            }
        }
#pragma unroll 2
        for (; j0 < last; j0 += STEP) {
            double r[E];
            rest(r, j0 + lane * E, j0, last);
#pragma unroll
            for (int i = 0; i < E; ++i) sum += r[i];
        }
        sum = warp_sum(sum);
        __syncthreads();                       // (the last sums have been read)
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        turn ^= 1;
        if (warp == 0) {
            const double mine = warp_sum(lane < WARPS ? s_sum[lane] : 0.0);
            if (lane < ctas) asm volatile("st.shared::cluster.f64 [%0], %1;\n" ::"r"(there(&s_cta[turn][rank], lane)), "d"(mine) : "memory");
        }
        cluster_sync();
        sum = 0.0;
        for (int i = 0; i < ctas; ++i) sum += s_cta[turn][i];
        return sum;
    };
    // Every warp walks by itself, its lanes holding the nodes' parents.
    const int up0 = lane < T ? s_up[lane] : -1, up1 = lane + 32 < T ? s_up[lane + 32] : -1;
    for (bool on = true; on;) {
        on = false;
        unsigned long long children = __ballot_sync(0xFFFFFFFFu, up0 == now) | (unsigned long long)__ballot_sync(0xFFFFFFFFu, up1 == now) << 32;
        while (children) {
            const int i = __ffsll(children) - 1;
            children &= children - 1;
            const double u = s_u[i], p = s_p[i], q = s_q[i];
            if (draft) {
                on = u * left * q < left_of(p, c, q);
            } else {
                on = u * left < p;
                if (!on) {
                    left -= p;
                    gone |= 1ull << i;
                }
            }
            if (on) {
                now = i;
                c = 0.0;
                left = 1.0;
                gone = 0;
                if (tid == 0 && rank == 0) a.path[(long long)b * T + count] = i;
                ++count;
                break;
            }
            if (draft) {
                c += left;
                if (children) left = total();  // (the sum behind the last child is formed below)
            }
        }
    }
    double sum = total();
    if (!(sum > 0.0)) {                        // nothing is left of the row but rounding: the row itself
        c = 0.0;
        gone = 0;
        sum = total();
    }
    if (rank == 0) {
        if (tid == 0) a.count[b] = count;
        for (int i = count + tid; i < T; i += THREADS) a.path[(long long)b * T + i] = -1;
    }
    const double at = (double)fmaxf(s_u[0], 0.f) * sum;
    double before = 0.0;
    for (int i = 0; i < rank; ++i) before += s_cta[turn][i];
    // The warp's part in which `at` falls; the CTA looks through it together, a step per warp.
    int owner = -1;
    for (int w = 0; w < WARPS; ++w) {
        const double next = before + s_sum[w];
        if (before <= at && next > at) {
            owner = w;
            break;
        }
        before = next;
    }
    if (owner >= 0) {
        const int from = min(V, (rank * WARPS + owner) * each * STEP), to = min(V, from + each * STEP);
        for (int j1 = from; j1 < to; j1 += WARPS * STEP) {
            const int j0 = j1 + warp * STEP;
            double r[E], x = 0.0;
#pragma unroll
            for (int i = 0; i < E; ++i) r[i] = 0.0;
            if (j0 < to) rest(r, j0 + lane * E, j0, to);
#pragma unroll
            for (int i = 0; i < E; ++i) x += r[i];
            const double own = x;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xFFFFFFFFu, x, o);
                if (lane >= o) x += y;
            }
            if (lane == 31) s_step[warp] = x;
            __syncthreads();
            double z = before;
            for (int w = 0; w < WARPS; ++w) {
                if (w < warp) z += s_step[w];
                before += s_step[w];
            }
            z += x - own;
            int found = V;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                z += r[i];
                if (found == V && r[i] > 0.0 && z > at) found = j0 + lane * E + i;
            }
            found = __reduce_min_sync(0xFFFFFFFFu, found);
            if (lane == 0 && found < V) atomicMin(&s_mine, found);
            __syncthreads();
            if (s_mine < V) break;
        }
        if (tid == 0 && s_mine < V) asm volatile("red.shared::cluster.min.s32 [%0], %1;\n" ::"r"(there(&s_first, 0)), "r"(s_mine) : "memory");
    }
    // The first CTA waits for the others and has the rest to itself.
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    if (rank != 0) return;
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    if (s_first == V && sum > 0.0 && warp == 0) {
        // A random number of 1, or one between two parts whose sums were rounded: one warp adds up the row from its beginning, so that nothing lies
        // between; where that does not reach the number, the last entry.  Rare.
        before = 0.0;
        int low = V, high = -1;
        for (int j0 = 0; j0 < V && low == V; j0 += STEP) {
            double r[E], x = 0.0;
            rest(r, j0 + lane * E, j0, V);
#pragma unroll
            for (int i = 0; i < E; ++i) x += r[i];
            const double own = x;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xFFFFFFFFu, x, o);
                if (lane >= o) x += y;
            }
            double z = before + (x - own);
            int found = V, last_one = -1;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                z += r[i];
                if (r[i] > 0.0) {
                    last_one = j0 + lane * E + i;
                    if (found == V && z > at) found = last_one;
                }
            }
            low = __reduce_min_sync(0xFFFFFFFFu, found);
            high = max(high, __reduce_max_sync(0xFFFFFFFFu, last_one));
            before += __shfl_sync(0xFFFFFFFFu, x, 31);
        }
        if (lane == 0) s_first = low < V ? low : high;
    }
    if (tid == 0) a.token[b] = sum > 0.0 ? s_first : -1;
}

template <class P>
int launch_choose(ChooseArgs<P> a, const void* target, const void* draft, int bsz, cudaStream_t st) {
    a.target = static_cast<const P*>(target);
    a.draft = static_cast<const P*>(draft);
    constexpr int E = 16 / sizeof(P);
    const bool vec = aligned16(target) && aligned16(draft) && a.target_batch % E == 0 && a.target_row % E == 0 &&
                     (!draft || (a.draft_batch % E == 0 && a.draft_row % E == 0));
    // As many CTAs a sequence as keep a step or more for every warp, and all sequences' resident at once.
    a.ctas = MOST_CTAS;
    while (a.ctas > 1 && ((long long)a.ctas * WARPS * 32 * E > a.V || (long long)bsz * a.ctas > 2ll * sm_count())) a.ctas /= 2;
    launch_cluster(vec ? choose_kernel<P, true> : choose_kernel<P, false>, a.ctas, dim3((unsigned)bsz * a.ctas), dim3(THREADS), 0, st, a);
    return cuda_status(cudaGetLastError(), "accept_drafts launch");
}

}  // namespace
}  // namespace akv

using namespace akv;

extern "C" int akv_accept_drafts(const void* target, long long target_batch, long long target_row, const void* draft, long long draft_batch,
                                 long long draft_row, const void* ids, const void* coins, const void* parents, long long parents_batch,
                                 void* path, void* count, void* token, int bsz, int drafted, int vocab, int type, void* stream) {
    set_error("");
    AKV_REQUIRE(target && ids && coins && path && count && token, AKV_ERR_NULL, "accept_drafts: null pointer");
    AKV_REQUIRE(bsz > 0 && bsz <= 1 << 24 && drafted >= 1 && drafted <= MOST && vocab > 0, AKV_ERR_SHAPE,
                "accept_drafts: %d sequences, %d tokens each (1 to %d) of a vocabulary of %d", bsz, drafted, MOST, vocab);
    AKV_REQUIRE(vocab <= 1 << 24, AKV_ERR_OVERFLOW, "accept_drafts: a vocabulary of %d", vocab);
    AKV_REQUIRE(type == AKV_TYPE_FP32 || type == AKV_TYPE_FP16 || type == AKV_TYPE_BF16, AKV_ERR_SHAPE, "accept_drafts: type %d", type);
    AKV_REQUIRE(target_batch >= 0 && target_row >= 0 && draft_batch >= 0 && draft_row >= 0 && parents_batch >= 0, AKV_ERR_SHAPE,
                "accept_drafts: negative stride");
    const uintptr_t size = type == AKV_TYPE_FP32 ? 4 : 2;
    AKV_REQUIRE(((reinterpret_cast<uintptr_t>(target) | reinterpret_cast<uintptr_t>(draft)) & (size - 1)) == 0 &&
                    ((reinterpret_cast<uintptr_t>(ids) | reinterpret_cast<uintptr_t>(token)) & 7u) == 0 &&
                    ((reinterpret_cast<uintptr_t>(coins) | reinterpret_cast<uintptr_t>(parents) | reinterpret_cast<uintptr_t>(path) |
                      reinterpret_cast<uintptr_t>(count)) & 3u) == 0,
                AKV_ERR_ALIGN, "accept_drafts: pointers must be aligned to their types");
    auto run = [&](auto a) {
        a.target_batch = target_batch;
        a.target_row = target_row;
        a.draft_batch = draft_batch;
        a.draft_row = draft_row;
        a.parents_batch = parents_batch;
        a.ids = static_cast<const long long*>(ids);
        a.coins = static_cast<const float*>(coins);
        a.parents = static_cast<const int*>(parents);
        a.path = static_cast<int*>(path);
        a.count = static_cast<int*>(count);
        a.token = static_cast<long long*>(token);
        a.T = drafted;
        a.V = vocab;
        return launch_choose(a, target, draft, bsz, static_cast<cudaStream_t>(stream));
    };
    if (type == AKV_TYPE_FP32) return run(ChooseArgs<float>{});
    if (type == AKV_TYPE_FP16) return run(ChooseArgs<__half>{});
    return run(ChooseArgs<__nv_bfloat16>{});
}
