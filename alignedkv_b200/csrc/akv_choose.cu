// Which drafted tokens are accepted, and the token behind them, such that what comes out has the target's distribution.
//
// At an accepted node with target probabilities p and draft probabilities q its children, drawn from q, are asked in order: x is accepted
// with probability min(1, r(x) / (Z q(x))), r = max(p - c q, 0), c = 0 and Z = 1 at first.  A rejection leaves the residual max(r / Z - q, 0),
// normalised; times Z that is max(p - (c + Z) q, 0), since max(max(a, 0) - b, 0) = max(a - b, 0) for b >= 0.  So the residual after any number of
// rejections is one coefficient, and the tests are u Z q(x) < r(x) with Z = sum r.  Without q a child is a guess of probability one:
// accepted with probability p(x) / Z, and its p leaves the row when it is not.  Where no child is left, the smallest j with
// cumsum(r)[j] > u_0 sum(r) follows.  Products and sums in 64 bits: the differences of fp32 probabilities are exact there, and what the order
// of additions changes is too little to move a border across a random number.
#include <cuda_bf16.h>

#include "akv_common.cuh"

namespace akv {
namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32, MOST = 64;

template <class P>
struct ChooseArgs {
    const P *target, *draft;
    long long target_batch, target_row, draft_batch, draft_row, parents_batch;
    const long long* ids;
    const float* coins;
    const int* parents;
    int *path, *count;
    long long* token;
    int T, V;
};

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
// What is no probability counts as none.
template <class P>
__device__ __forceinline__ float chance(const P* at) {
    const float x = as_float(__ldg(at));
    return x > 0.f && x < INFINITY ? x : 0.f;
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
    return x;
}

template <class P>
__global__ void __launch_bounds__(THREADS) choose_kernel(ChooseArgs<P> a) {
    __shared__ double s_sum[WARPS];
    __shared__ int s_up[MOST], s_gone[MOST], s_found, s_last;
    __shared__ float s_p[MOST], s_q[MOST], s_u[MOST];
    __shared__ long long s_x[MOST];
    pdl_turn();
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int T = a.T, V = a.V;
    const P* target = a.target + b * a.target_batch;
    const P* draft = a.draft ? a.draft + b * a.draft_batch : nullptr;
    if (tid < T) {
        const int up = tid == 0 ? -1 : a.parents ? a.parents[b * a.parents_batch + tid] : tid - 1;
        const long long x = a.ids[(long long)b * T + tid];
        const bool asked = up >= 0 && up < tid && x >= 0 && x < V;
        s_up[tid] = up;
        s_x[tid] = x;
        s_u[tid] = a.coins[(long long)b * T + tid];
        s_p[tid] = asked ? chance(target + up * a.target_row + x) : 0.f;
        s_q[tid] = asked && draft ? chance(draft + up * a.draft_row + x) : 0.f;
    }
    __syncthreads();
    const int each = (V + WARPS - 1) / WARPS, first = min(V, warp * each), last = min(V, first + each);
    int now = 0, count = 1, gone = 0;
    double c = 0.0, left = 1.0;
    if (tid == 0) a.path[(long long)b * T] = 0;
    auto rest = [&](int j) -> double {
        double r = chance(target + now * a.target_row + j);
        if (draft) {
            if (c > 0.0) r = fmax(r - c * (double)chance(draft + now * a.draft_row + j), 0.0);
        } else {
            for (int g = 0; g < gone; ++g)
                if (s_gone[g] == j) r = 0.0;
        }
        return r;
    };
    auto total = [&]() -> double {
        double sum = 0.0;
        for (int j = first + lane; j < last; j += 32) sum += rest(j);
        sum = warp_sum(sum);
        __syncthreads();
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        sum = 0.0;
        for (int w = 0; w < WARPS; ++w) sum += s_sum[w];
        return sum;
    };
    for (int i = 1; i < T; ++i) {
        if (s_up[i] != now) continue;
        const double u = s_u[i], p = s_p[i], q = s_q[i];
        bool good;
        if (draft) {
            good = u * left * q < fmax(p - c * q, 0.0);
        } else {
            double r = p;
            for (int g = 0; g < gone; ++g)
                if (s_gone[g] == s_x[i]) r = 0.0;
            good = u * left < r;
            if (!good) {
                left -= r;
                __syncthreads();
                if (tid == 0) s_gone[gone] = s_x[i] >= 0 && s_x[i] < V ? (int)s_x[i] : -1;
                ++gone;
                __syncthreads();
            }
        }
        if (good) {
            now = i;
            c = 0.0;
            left = 1.0;
            gone = 0;
            if (tid == 0) a.path[(long long)b * T + count] = i;
            ++count;
        } else if (draft) {
            c += left;
            left = total();
        }
    }
    double sum = total();
    if (!(sum > 0.0)) {                        // nothing is left of the row but rounding: the row itself
        c = 0.0;
        gone = 0;
        sum = total();
    }
    if (tid == 0) {
        a.count[b] = count;
        s_found = V;
        s_last = -1;
    }
    for (int i = count + tid; i < T; i += THREADS) a.path[(long long)b * T + i] = -1;
    __syncthreads();
    const double at = (double)fmaxf(s_u[0], 0.f) * sum;
    double before = 0.0;
    for (int w = 0; w < warp; ++w) before += s_sum[w];
    int found = V, end = -1;
    for (int j0 = first; j0 < last; j0 += 32) {
        const int j = j0 + lane;
        const double r = j < last ? rest(j) : 0.0;
        double x = r;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xFFFFFFFFu, x, o);
            if (lane >= o) x += y;
        }
        if (r > 0.0) end = j;
        if (found == V && before + x > at && j < last) found = j;
        before += __shfl_sync(0xFFFFFFFFu, x, 31);
    }
    atomicMin(&s_found, found);
    atomicMax(&s_last, end);
    __syncthreads();
    if (tid == 0) a.token[b] = sum > 0.0 ? (s_found < V ? s_found : s_last) : -1;
}

template <class P>
int launch_choose(ChooseArgs<P> a, const void* target, const void* draft, int bsz, cudaStream_t st) {
    a.target = static_cast<const P*>(target);
    a.draft = static_cast<const P*>(draft);
    launch_chained(choose_kernel<P>, dim3(bsz), dim3(THREADS), 0, st, a);
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
    AKV_REQUIRE(bsz > 0 && drafted >= 1 && drafted <= MOST && vocab > 0, AKV_ERR_SHAPE,
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
