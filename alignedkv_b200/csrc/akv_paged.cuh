// The cache in pages: how a page holds tokens, shared by the kernels that write, read and attend to them.
#pragma once
#include <limits.h>

#include "akv_common.cuh"

namespace akv {

// A pool of pages [n_pages, H, page_size]: rows of D channels per token and KV head.
//   AKV_PAGE_FP16  2 D bytes
//   AKV_PAGE_E4M3  D bytes and an exponent e, x = code 2^e.  e is the least with max |x| <= 448 2^e: a power of two costs e4m3 nothing (its
//                  steps are relative), multiplies without rounding, and leaves every code's rounding to the value alone.
//   AKV_PAGE_E2M1  D / 2 bytes (the even channel in the lower bits), an e4m3 scale s per 16 channels and an exponent e, x = code s 2^e.  e is the
//                  least with max |x| <= 6 * 448 2^e, s the nearest to max |x| 2^-e / 6 of its 16 channels.
// Exponent -128: a row with a value that is not finite; it stands for NaN throughout, its codes are zero.
constexpr int EXP_NAN = -128;
template <int F> __host__ __device__ constexpr int row_bytes(int D) { return F == AKV_PAGE_FP16 ? 2 * D : F == AKV_PAGE_E4M3 ? D : D / 2; }

struct Pool {
    uint8_t *kc, *vc;          // codes
    int8_t *ke, *ve;           // exponents
    uint8_t *ks, *vs;          // scales (e4m3)
    int n_pages, shift, H;     // shift: log2 of the page size
    const int* table;          // [B, width]
    const int* lens;           // [B]
    int width;
};

// Tokens of sequence b that its pages can hold at most.
__device__ __forceinline__ int length_of(const Pool& p, int b) {
    const long long room = (long long)p.width << p.shift;
    const int n = p.lens[b];
    return n < 0 ? 0 : n > room ? (int)room : n;
}
// Row of the pool that has position `at` (below the table's end) of KV head h; -1 where the page was given up.
__device__ __forceinline__ long long pool_row(const Pool& p, int b, int h, long long at) {
    const int page = __ldg(p.table + (long long)b * p.width + (at >> p.shift));
    if ((unsigned)page >= (unsigned)p.n_pages) return -1;
    return (((long long)page * p.H + h) << p.shift) + (at & ((1 << p.shift) - 1));
}

// 2^e (e in -126..127), NaN for EXP_NAN.
__device__ __forceinline__ float power2(int e) { return e == EXP_NAN ? NAN : __int_as_float((e + 127) << 23); }

// Two codes as halves; exact.
__device__ __forceinline__ uint32_t e4m3_halves(uint32_t two) {
    uint32_t h;
    asm("{\n.reg .b16 b;\ncvt.u16.u32 b, %1;\ncvt.rn.f16x2.e4m3x2 %0, b;\n}\n" : "=r"(h) : "r"(two));
    return h;
}
__device__ __forceinline__ uint32_t e2m1_halves(uint32_t two) {
    uint32_t h;
    asm("{\n.reg .b8 b;\ncvt.u8.u32 b, %1;\ncvt.rn.f16x2.e2m1x2 %0, b;\n}\n" : "=r"(h) : "r"(two));
    return h;
}
// Four codes of a word, eight.
__device__ __forceinline__ void e4m3_word(uint32_t (&h)[2], uint32_t word) {
    asm("{\n.reg .b16 l, u;\nmov.b32 {l, u}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, u;\n}\n" : "=r"(h[0]), "=r"(h[1]) : "r"(word));
}
__device__ __forceinline__ void e2m1_word(uint32_t (&h)[4], uint32_t word) {
    asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %4;\ncvt.rn.f16x2.e2m1x2 %0, a;\ncvt.rn.f16x2.e2m1x2 %1, b;\n"
        "cvt.rn.f16x2.e2m1x2 %2, c;\ncvt.rn.f16x2.e2m1x2 %3, d;\n}\n"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(word));
}
__device__ __forceinline__ float2 halves_floats(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }
__device__ __forceinline__ float e4m3_float(uint32_t code) { return halves_floats(e4m3_halves(code)).x; }

// Host side (akv_paged.cu): checks a pool and its table and fills the kernel parameters.
int fill_pool(const char* what, const akv_pool* pool, const void* pages, const void* lens, int bsz, int width, Pool* p);

}  // namespace akv
