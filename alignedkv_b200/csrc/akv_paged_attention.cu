// Attention of the newest tokens of each sequence over its pages.
//
//   out_r = sum_j p_rj v_j / sum_j p_rj, p_rj = exp(scale q_r . k_j - m_r) over the tokens j that row r sees; fp32 throughout.
#include "akv_paged.cuh"

namespace akv {
namespace {

struct AttendArgs {
    Pool pool;
    const __half* q;
    __half* out;
    float* lse;
    int B, T, G;
    float scale;
};

constexpr int WARPS = 4;

// Channels N lane .. N lane + N - 1 of a row, times 2^e.
template <int F, int D>
__device__ __forceinline__ void load_row(float (&x)[D / 32], const uint8_t* codes, const int8_t* exps, const uint8_t* scales, long long row,
                                         int lane) {
    constexpr int N = D / 32;
    float unit = 1.f;
    if constexpr (F != AKV_PAGE_FP16) unit = power2(exps[row]);
    if constexpr (F == AKV_PAGE_E2M1) unit *= e4m3_float(scales[row * (D / 16) + lane * N / 16]);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        uint32_t h;
        if constexpr (F == AKV_PAGE_FP16) h = *reinterpret_cast<const uint32_t*>(codes + row * (2 * D) + (lane * N + i) * 2);
        else if constexpr (F == AKV_PAGE_E4M3) h = e4m3_halves(*reinterpret_cast<const uint16_t*>(codes + row * D + lane * N + i));
        else h = e2m1_halves(codes[row * (D / 2) + (lane * N + i) / 2]);
        const float2 f = halves_floats(h);
        x[i] = f.x * unit;
        x[i + 1] = f.y * unit;
    }
}

template <int F, int D>
__global__ void __launch_bounds__(32 * WARPS) attend_kernel(AttendArgs a) {
    constexpr int N = D / 32;
    __shared__ float part[WARPS][D + 2];
    pdl_turn();
    const Pool& p = a.pool;
    const int hq = blockIdx.x, t = blockIdx.y, b = blockIdx.z, h = hq / a.G, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = length_of(p, b) - (a.T - 1) + t;
    const long long at = ((long long)b * a.T + t) * (p.H * a.G) + hq;
    float q[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        q[i] = __half2float(a.q[at * D + lane * N + i]) * a.scale;
        o[i] = 0.f;
    }
    for (int j = warp; j < n; j += WARPS) {
        const long long row = pool_row(p, b, h, j);
        if (row < 0) continue;
        float k[N], v[N], s = 0.f;
        load_row<F, D>(k, p.kc, p.ke, p.ks, row, lane);
        load_row<F, D>(v, p.vc, p.ve, p.vs, row, lane);
#pragma unroll
        for (int i = 0; i < N; ++i) s = fmaf(q[i], k[i], s);
#pragma unroll
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, x);
        const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top, was = expf(m - base), pr = expf(s - base);
        m = top;
        l = l * was + pr;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = o[i] * was + pr * v[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) part[warp][lane * N + i] = o[i];
    if (lane == 0) {
        part[warp][D] = m;
        part[warp][D + 1] = l;
    }
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, part[w][D]);
    for (int w = 0; w < WARPS; ++w) sum += part[w][D] == -INFINITY ? part[w][D + 1] : part[w][D + 1] * expf(part[w][D] - top);
    for (int c = threadIdx.x; c < D; c += 32 * WARPS) {
        float x = 0.f;
        for (int w = 0; w < WARPS; ++w) x += part[w][D] == -INFINITY ? part[w][c] : part[w][c] * expf(part[w][D] - top);
        a.out[at * D + c] = __float2half_rn(sum == 0.f ? 0.f : x / sum);
    }
    if (a.lse && threadIdx.x == 0) a.lse[at] = top + logf(sum);
}

template <int F>
void launch_attend(const AttendArgs& a, int D, cudaStream_t st) {
    const dim3 grid(a.pool.H * a.G, a.T, a.B);
    if (D == 128) launch_chained(attend_kernel<F, 128>, grid, dim3(32 * WARPS), 0, st, a);
    else launch_chained(attend_kernel<F, 64>, grid, dim3(32 * WARPS), 0, st, a);
}

}  // namespace
}  // namespace akv

using namespace akv;

extern "C" {

long long akv_paged_scratch_bytes(const akv_pool* pool, int bsz, int width, int group, int tokens) {
    if (!pool || bsz <= 0 || width <= 0 || group <= 0 || tokens <= 0) return -1;
    return 0;
}

int akv_paged_attention(const akv_pool* pool, const void* q, const void* pages, const void* lens, void* out, void* lse, void* scratch,
                        long long scratch_bytes, int bsz, int width, int group, int tokens, float scale, void* stream) {
    set_error("");
    AttendArgs a = {};
    const int rc = fill_pool("paged_attention", pool, pages, lens, bsz, width, &a.pool);
    if (rc != AKV_OK) return rc;
    AKV_REQUIRE(q && out, AKV_ERR_NULL, "paged_attention: null pointer");
    AKV_REQUIRE(group > 0 && tokens > 0 && group <= 64 && tokens <= 64 && group * tokens <= 64, AKV_ERR_SHAPE,
                "paged_attention: %d new tokens of %d query heads per KV head (at most 64 rows)", tokens, group);
    AKV_REQUIRE(aligned16(q) && aligned16(out) && (reinterpret_cast<uintptr_t>(lse) & 3u) == 0, AKV_ERR_ALIGN,
                "paged_attention: q and out must be 16-byte aligned, lse 4-byte");
    (void)scratch;
    (void)scratch_bytes;
    a.q = static_cast<const __half*>(q);
    a.out = static_cast<__half*>(out);
    a.lse = static_cast<float*>(lse);
    a.B = bsz;
    a.T = tokens;
    a.G = group;
    a.scale = scale;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int D = pool->head_dim;
    if (pool->format == AKV_PAGE_FP16) launch_attend<AKV_PAGE_FP16>(a, D, st);
    else if (pool->format == AKV_PAGE_E4M3) launch_attend<AKV_PAGE_E4M3>(a, D, st);
    else launch_attend<AKV_PAGE_E2M1>(a, D, st);
    return cuda_status(cudaGetLastError(), "paged_attention launch");
}

}  // extern "C"
