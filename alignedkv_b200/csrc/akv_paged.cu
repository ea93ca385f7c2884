// The cache in pages: tokens are quantised as they enter it, and read back as fp16.
#include "akv_paged.cuh"

namespace akv {
namespace {

constexpr int THREADS = 256;
constexpr int PIECES = 2, ROWS_EACH = 2;       // a lane's 16-byte pieces of fp16 of a row, its rows; all are on their way together
template <int D> constexpr int lanes_of = D / (8 * PIECES);    // lanes of a row: lane i has pieces i, i + lanes, ...

struct AppendArgs {
    Pool pool;
    const __half *k, *v;
    long long k_batch, k_token, k_head, v_batch, v_token, v_head;
    const int* counts;
    int T, blocks;                             // blocks of a sequence's tokens
};

// The least e with a <= top 2^add 2^e for the bits of a >= 0 (top's fraction as bits); a = 0 counts as fp16's smallest.
__device__ __forceinline__ int least_exponent(uint32_t bits, uint32_t top_fraction, int add) {
    if (bits == 0) return -24 - add;
    return (int)(bits >> 23) - 127 - add + ((bits & 0x7FFFFFu) > top_fraction);
}
// x / s in the nearest fp32, s > 0 with reciprocal r to a few steps: x r is off by steps, what it leaves out is exact in one fused operation,
// and adding that part puts the quotient within 2^-40 before its one rounding.  Codes change at middles m of few bits; fp16 x is never
// nearer to m s than 2^-12 of it unless equal, and then the quotient is m itself.
__device__ __forceinline__ float quotient(float x, float s, float r) {
    const float y = x * r;
    return fmaf(fmaf(-y, s, x), r, y);
}
__device__ __forceinline__ float reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t max_halves(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
__device__ __forceinline__ uint32_t max_of(uint32_t two) { return max(two & 0xFFFFu, two >> 16); }
// 2^e in both halves, e in -14..15.
__device__ __forceinline__ uint32_t power2_halves(int e) { return (uint32_t)(e + 15) * 0x04000400u; }
// Two e4m3 codes of two halves (x, y of a word each): nearest, ties to even.
__device__ __forceinline__ uint32_t to_e4m3(uint32_t x, uint32_t y) {
    uint32_t w;
    asm("{\n.reg .b16 l, u;\ncvt.rn.satfinite.e4m3x2.f16x2 l, %1;\ncvt.rn.satfinite.e4m3x2.f16x2 u, %2;\nmov.b32 %0, {l, u};\n}\n" : "=r"(w) : "r"(x), "r"(y));
    return w;
}

// Codes of a lane's pieces, by the lanes that have a row; row < 0: takes part in the exchange, stores nothing.
template <int F, int D>
__device__ __forceinline__ void store_row(uint8_t* codes, int8_t* exps, uint8_t* scales, long long row, int lane, const uint4 (&raw)[PIECES]) {
    constexpr int LANES = lanes_of<D>;
    if constexpr (F == AKV_PAGE_FP16) {
#pragma unroll
        for (int q = 0; q < PIECES; ++q)
            if (row >= 0) *reinterpret_cast<uint4*>(codes + row * (2 * D) + (lane + q * LANES) * 16) = raw[q];
    } else {
        // magnitudes as 16 bits: NaN is above infinity, infinity above the rest
        uint32_t pair[PIECES], top = 0;        // (pair: of 16 channels, two neighbouring lanes)
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
            constexpr uint32_t ABS = 0x7FFF7FFFu;
            pair[q] = max_halves(max_halves(raw[q].x & ABS, raw[q].y & ABS), max_halves(raw[q].z & ABS, raw[q].w & ABS));
            if constexpr (F == AKV_PAGE_E2M1) pair[q] = max_halves(pair[q], __shfl_xor_sync(0xFFFFFFFFu, pair[q], 1));
            top = max_halves(top, pair[q]);
        }
#pragma unroll
        for (int o = F == AKV_PAGE_E2M1 ? 2 : 1; o < LANES; o <<= 1) top = max_halves(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        const uint32_t most = max_of(top);
        const bool finite = most < 0x7C00u;
        const uint32_t bits = __float_as_uint(halves_floats(most).x);
        const int e = F == AKV_PAGE_E4M3 ? least_exponent(bits, 0x600000u, 8) : least_exponent(bits, 0x280000u, 11);
        if (row >= 0 && lane == 0) exps[row] = (int8_t)(finite ? e : EXP_NAN);
        if constexpr (F == AKV_PAGE_E4M3) {
#pragma unroll
            for (int q = 0; q < PIECES; ++q) {
                // Times 2^-e: exact in fp16 where that makes a value larger; where it makes it smaller what gets lost is far below half
                // the smallest code.  -e beyond fp16 (a row below 2^-5) takes two factors, of the smallest rows three.
                const uint32_t one = power2_halves(min(-e, 14)), two = power2_halves(min(max(-e - 14, 0), 14));
                uint32_t x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = hmul2_bits(hmul2_bits(u4w(raw[q], i), one), two);
                if (e < -28) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = hmul2_bits(x[i], power2_halves(-e - 28));
                }
                const uint2 w = make_uint2(to_e4m3(x[0], x[1]), to_e4m3(x[2], x[3]));
                if (row >= 0) *reinterpret_cast<uint2*>(codes + row * D + (lane + q * LANES) * 8) = finite ? w : make_uint2(0, 0);
            }
        } else {
            const float unit = finite ? power2(e) : 0.f, back = finite ? power2(-e) : 0.f;
#pragma unroll
            for (int q = 0; q < PIECES; ++q) {
                uint16_t sc;
                const float sixth = finite ? quotient(halves_floats(max_of(pair[q])).x * back, 6.f, 1.f / 6.f) : 0.f;      // (middles of e4m3 have 5 bits)
                asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(sc) : "f"(0.f), "f"(sixth));
                if (row >= 0 && (lane & 1) == 0) scales[row * (D / 16) + ((lane + q * LANES) >> 1)] = (uint8_t)sc;
                const float s = e4m3_float(sc & 0xFFu) * unit, r = s > 0.f ? reciprocal(s) : 0.f;
                uint32_t c[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = halves_floats(u4w(raw[q], i));
                    asm("{\n.reg .b8 b;\ncvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\ncvt.u32.u8 %0, b;\n}\n"
                        : "=r"(c[i]) : "f"(quotient(f.y, s, r)), "f"(quotient(f.x, s, r)));
                }
                const uint32_t w = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
                if (row >= 0) *reinterpret_cast<uint32_t*>(codes + row * (D / 2) + (lane + q * LANES) * 4) = finite ? w : 0u;
            }
        }
    }
}

// What a block has: K and V of all heads side by side, then the next tokens, then the next sequence; so that what is written at one time lies
// together (16 sequences of 1000 tokens, 32 heads: 119 us, one head after the other 140).
struct Place {
    int b, block, h;
    bool which;
    __device__ __forceinline__ Place(int H, int blocks) {
        const unsigned x = blockIdx.x / (2u * H), y = blockIdx.x - x * 2u * H;
        which = y >= (unsigned)H;
        h = which ? y - H : y;
        b = x / (unsigned)blocks;
        block = x - b * blocks;
    }
};

// Rows of one tensor by LANES threads each; a block has consecutive tokens of one KV head, whose rows lie side by side in a page.  Bound by HBM
// and, nearly as much, by the instructions of the maxima and conversions: up to 1000 tokens of 16 x 32 heads of 128 channels 36 us in e4m3 (5.6 TB/s, 83%
// of the issue slots), up to 8190 of 4 x 8 13 us in e2m1.  (One row a lane, four, 128 or 512 threads: slower or the same.)
template <int F, int D>
__global__ void __launch_bounds__(THREADS) append_kernel(AppendArgs a) {
    constexpr int LANES = lanes_of<D>, ROWS = THREADS / LANES;
    pdl_turn();
    const Pool& p = a.pool;
    const Place at0(p.H, a.blocks);
    const int b = at0.b, h = at0.h, lane = threadIdx.x % LANES, begin = at0.block * (ROWS_EACH * ROWS), i0 = begin + threadIdx.x / LANES;
    const bool which = at0.which;
    const int n = a.counts ? min(a.T, a.counts[b]) : a.T;
    if (begin >= n) return;
    const long long at = max(0, p.lens[b]), room = (long long)p.width << p.shift;
    const __half* x = (which ? a.v + b * a.v_batch + h * a.v_head : a.k + b * a.k_batch + h * a.k_head) + lane * 8;
    const long long step = which ? a.v_token : a.k_token;
    uint4 raw[ROWS_EACH][PIECES];
    long long row[ROWS_EACH];
#pragma unroll
    for (int m = 0; m < ROWS_EACH; ++m) {
        const int i = i0 + m * ROWS;
        const bool there = i < n && at + i < room;
#pragma unroll
        for (int q = 0; q < PIECES; ++q)
            raw[m][q] = there ? __ldg(reinterpret_cast<const uint4*>(x + i * step + q * LANES * 8)) : make_uint4(0, 0, 0, 0);
        row[m] = there ? pool_row(p, b, h, at + i) : -1;
    }
#pragma unroll
    for (int m = 0; m < ROWS_EACH; ++m)
        if (begin + m * ROWS < n)              // (the same for the block)
            store_row<F, D>(which ? p.vc : p.kc, which ? p.ve : p.ke, which ? p.vs : p.ks, row[m], lane, raw[m]);
}

// fp16 of a value beyond its range: the largest.  (A code may be above the value it stands for: 65504 is held as 65536.)
__device__ __forceinline__ float saturated(float x) { return fabsf(x) > 65504.f ? copysignf(65504.f, x) : x; }

struct ReadArgs {
    Pool pool;
    __half *k, *v;
    int most, blocks;
};

// The same places.  Bound by HBM's writes: what append left above takes 51 us from e4m3 (5.1 TB/s, three
// quarters of them written), 27 us from e2m1.
template <int F, int D>
__global__ void __launch_bounds__(THREADS) read_kernel(ReadArgs a) {
    constexpr int LANES = lanes_of<D>, ROWS = THREADS / LANES, PIECE = row_bytes<F>(D) / (LANES * PIECES);
    pdl_turn();
    const Pool& p = a.pool;
    const Place at0(p.H, a.blocks);
    const int b = at0.b, h = at0.h, lane = threadIdx.x % LANES, i0 = at0.block * (ROWS_EACH * ROWS) + threadIdx.x / LANES;
    const bool which = at0.which;
    const int n = length_of(p, b);
    const uint8_t *codes = (which ? p.vc : p.kc) + lane * PIECE, *scales = which ? p.vs : p.ks;
    const int8_t* exps = which ? p.ve : p.ke;
    __half* out = (which ? a.v : a.k) + lane * 8;
    uint4 w[ROWS_EACH][PIECES];
    int exponent[ROWS_EACH];
    uint32_t scale[ROWS_EACH][PIECES];
#pragma unroll
    for (int m = 0; m < ROWS_EACH; ++m) {
        const int i = i0 + m * ROWS;
        const long long row = i < n && i < a.most ? pool_row(p, b, h, i) : -1;
        exponent[m] = 0;
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
            w[m][q] = make_uint4(0, 0, 0, 0);
            scale[m][q] = 0;
            if (row >= 0) {
                const uint8_t* x = codes + row * row_bytes<F>(D) + q * LANES * PIECE;
                if constexpr (F == AKV_PAGE_FP16) {
                    w[m][q] = __ldg(reinterpret_cast<const uint4*>(x));
                } else if constexpr (F == AKV_PAGE_E4M3) {
                    const uint2 y = __ldg(reinterpret_cast<const uint2*>(x));
                    w[m][q].x = y.x;
                    w[m][q].y = y.y;
                } else {
                    w[m][q].x = __ldg(reinterpret_cast<const uint32_t*>(x));
                    scale[m][q] = __ldg(scales + row * (D / 16) + ((lane + q * LANES) >> 1));
                }
            }
        }
        if (F != AKV_PAGE_FP16 && row >= 0) exponent[m] = __ldg(exps + row);
    }
#pragma unroll
    for (int m = 0; m < ROWS_EACH; ++m) {
        const int i = i0 + m * ROWS;
        if (i >= a.most) continue;
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
            if constexpr (F != AKV_PAGE_FP16) {
                uint32_t x[4], s = 0;
                if constexpr (F == AKV_PAGE_E4M3) {
                    uint32_t y[2], z[2];
                    e4m3_word(y, w[m][q].x);
                    e4m3_word(z, w[m][q].y);
                    x[0] = y[0]; x[1] = y[1]; x[2] = z[0]; x[3] = z[1];
                } else {
                    s = e4m3_halves(scale[m][q] * 0x0101u);
                    e2m1_word(x, w[m][q].x);
                }
                // In fp16 where the factor and every product fit it (448 * 2^7, 6 * 448 * 2^4; down to 2^-14 all are exact), else in fp32.
                if (exponent[m] >= -14 && exponent[m] <= (F == AKV_PAGE_E4M3 ? 7 : 4)) {
                    const uint32_t unit = power2_halves(exponent[m]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[k] = hmul2_bits(F == AKV_PAGE_E2M1 ? hmul2_bits(x[k], s) : x[k], unit);
                } else {
                    const float unit = power2(exponent[m]), f = F == AKV_PAGE_E2M1 ? halves_floats(s).x : 1.f;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float2 y = halves_floats(x[k]);
                        const __half2 r = __floats2half2_rn(saturated(y.x * f * unit), saturated(y.y * f * unit));
                        x[k] = *reinterpret_cast<const uint32_t*>(&r);
                    }
                }
                w[m][q] = make_uint4(x[0], x[1], x[2], x[3]);
            }
            __stcs(reinterpret_cast<uint4*>(out + (((long long)b * a.most + i) * p.H + h) * D + q * LANES * 8), w[m][q]);
        }
    }
}

// Blocks of a sequence's `tokens`; blocks of all (b, head, tensor) may not fit a grid.
int blocks_of(int tokens, int D) {
    const int rows = ROWS_EACH * THREADS / (D / (8 * PIECES));
    return (tokens + rows - 1) / rows;
}
template <int F>
void launch_append(const AppendArgs& a, int D, unsigned grid, cudaStream_t st) {
    if (D == 128) launch_chained(append_kernel<F, 128>, dim3(grid), dim3(THREADS), 0, st, a);
    else launch_chained(append_kernel<F, 64>, dim3(grid), dim3(THREADS), 0, st, a);
}
template <int F>
void launch_read(const ReadArgs& a, int D, unsigned grid, cudaStream_t st) {
    if (D == 128) launch_chained(read_kernel<F, 128>, dim3(grid), dim3(THREADS), 0, st, a);
    else launch_chained(read_kernel<F, 64>, dim3(grid), dim3(THREADS), 0, st, a);
}

bool misaligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

}  // namespace

int fill_pool(const char* what, const akv_pool* pool, const void* pages, const void* lens, int bsz, int width, Pool* p) {
    AKV_REQUIRE(pool && pages && lens, AKV_ERR_NULL, "%s: null pointer", what);
    const int D = pool->head_dim, f = pool->format;
    AKV_REQUIRE(f == AKV_PAGE_FP16 || f == AKV_PAGE_E4M3 || f == AKV_PAGE_E2M1, AKV_ERR_SHAPE, "%s: page format %d", what, f);
    AKV_REQUIRE(D == 64 || D == 128, AKV_ERR_SHAPE, "%s: head size %d (64 and 128 are covered)", what, D);
    AKV_REQUIRE(pool->n_pages > 0 && pool->n_kv_heads > 0 && pool->n_kv_heads <= 4096 && bsz > 0 && bsz <= 4096 && width > 0, AKV_ERR_SHAPE,
                "%s: bad extent (%d sequences, %d pages each, %d KV heads, %d pages in all)", what, bsz, width, pool->n_kv_heads, pool->n_pages);
    const int P = pool->page_size;
    AKV_REQUIRE(P >= 16 && P <= 256 && (P & (P - 1)) == 0, AKV_ERR_SHAPE, "%s: page size %d (a power of two from 16 to 256)", what, P);
    AKV_REQUIRE((long long)width * P <= INT_MAX / 2, AKV_ERR_OVERFLOW, "%s: %d pages of %d tokens in a sequence", what, width, P);
    AKV_REQUIRE(pool->k_codes && pool->v_codes && (f == AKV_PAGE_FP16 || (pool->k_exps && pool->v_exps)) &&
                    (f != AKV_PAGE_E2M1 || (pool->k_scales && pool->v_scales)),
                AKV_ERR_NULL, "%s: null pointer in the pool", what);
    AKV_REQUIRE(aligned16(pool->k_codes) && aligned16(pool->v_codes) && aligned16(pool->k_exps) && aligned16(pool->v_exps) &&
                    aligned16(pool->k_scales) && aligned16(pool->v_scales),
                AKV_ERR_ALIGN, "%s: the pool's pointers must be 16-byte aligned", what);
    AKV_REQUIRE(!misaligned(pages, 4) && !misaligned(lens, 4), AKV_ERR_ALIGN, "%s: pages and lens must be 4-byte aligned", what);
    *p = Pool{static_cast<uint8_t*>(pool->k_codes), static_cast<uint8_t*>(pool->v_codes), static_cast<int8_t*>(pool->k_exps),
              static_cast<int8_t*>(pool->v_exps), static_cast<uint8_t*>(pool->k_scales), static_cast<uint8_t*>(pool->v_scales),
              pool->n_pages, 0, pool->n_kv_heads, static_cast<const int*>(pages), static_cast<const int*>(lens), width};
    while ((1 << p->shift) < P) ++p->shift;
    return AKV_OK;
}

}  // namespace akv

using namespace akv;

extern "C" {

int akv_paged_append(const akv_pool* pool, const void* k, const void* v, const long long* strides, const void* pages, const void* lens,
                     const void* counts, int bsz, int width, int tokens, void* stream) {
    set_error("");
    AppendArgs a = {};
    const int rc = fill_pool("paged_append", pool, pages, lens, bsz, width, &a.pool);
    if (rc != AKV_OK) return rc;
    AKV_REQUIRE(k && v && strides, AKV_ERR_NULL, "paged_append: null pointer");
    AKV_REQUIRE(tokens > 0 && tokens <= 1 << 30, AKV_ERR_SHAPE, "paged_append: %d tokens", tokens);
    bool straight = aligned16(k) && aligned16(v) && !misaligned(counts, 4);
    for (int i = 0; i < 6; ++i) straight = straight && strides[i] % 8 == 0;
    AKV_REQUIRE(straight, AKV_ERR_ALIGN, "paged_append: rows of k and v must lie on 16-byte boundaries, counts on 4-byte ones");
    const int D = pool->head_dim;
    a.blocks = blocks_of(tokens, D);
    const long long grid = 2ll * pool->n_kv_heads * bsz * a.blocks;
    AKV_REQUIRE(grid < INT_MAX, AKV_ERR_OVERFLOW, "paged_append: too many rows");
    a.k = static_cast<const __half*>(k);
    a.v = static_cast<const __half*>(v);
    a.k_batch = strides[0];
    a.k_token = strides[1];
    a.k_head = strides[2];
    a.v_batch = strides[3];
    a.v_token = strides[4];
    a.v_head = strides[5];
    a.counts = static_cast<const int*>(counts);
    a.T = tokens;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (pool->format == AKV_PAGE_FP16) launch_append<AKV_PAGE_FP16>(a, D, (unsigned)grid, st);
    else if (pool->format == AKV_PAGE_E4M3) launch_append<AKV_PAGE_E4M3>(a, D, (unsigned)grid, st);
    else launch_append<AKV_PAGE_E2M1>(a, D, (unsigned)grid, st);
    return cuda_status(cudaGetLastError(), "paged_append launch");
}

int akv_paged_read(const akv_pool* pool, const void* pages, const void* lens, void* k, void* v, int bsz, int width, int most, void* stream) {
    set_error("");
    ReadArgs a = {};
    const int rc = fill_pool("paged_read", pool, pages, lens, bsz, width, &a.pool);
    if (rc != AKV_OK) return rc;
    AKV_REQUIRE(k && v, AKV_ERR_NULL, "paged_read: null pointer");
    AKV_REQUIRE(most > 0 && most <= 1 << 30, AKV_ERR_SHAPE, "paged_read: %d tokens", most);
    AKV_REQUIRE(aligned16(k) && aligned16(v), AKV_ERR_ALIGN, "paged_read: k and v must be 16-byte aligned");
    const int D = pool->head_dim;
    a.blocks = blocks_of(most, D);
    const long long grid = 2ll * pool->n_kv_heads * bsz * a.blocks;
    AKV_REQUIRE(grid < INT_MAX, AKV_ERR_OVERFLOW, "paged_read: too many rows");
    a.k = static_cast<__half*>(k);
    a.v = static_cast<__half*>(v);
    a.most = most;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (pool->format == AKV_PAGE_FP16) launch_read<AKV_PAGE_FP16>(a, D, (unsigned)grid, st);
    else if (pool->format == AKV_PAGE_E4M3) launch_read<AKV_PAGE_E4M3>(a, D, (unsigned)grid, st);
    else launch_read<AKV_PAGE_E2M1>(a, D, (unsigned)grid, st);
    return cuda_status(cudaGetLastError(), "paged_read launch");
}

}  // extern "C"
