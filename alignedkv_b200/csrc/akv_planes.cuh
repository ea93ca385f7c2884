// fp16 fragments of mma.m16n8k16 straight from the byte planes, in registers.
//
// K tiles run along tokens, V rows along channels; the contraction runs across them (q.k over channels, P.V over tokens).  Both
// are the same picture: four LINES of memory (four channels of K, four tokens of V) with N neighbouring elements each, where a
// product wants words (line 0, line 1) and (line 2, line 3) of one element.  Which element is which column of the product, and
// which line is which index of the sum, is free as long as the other operand agrees: lane (g, t) = (lane / 4, lane % 4) takes
// the elements N g .. N g + N - 1 (N = 16 or 8: wide loads) of its own four lines, and column g of n-tile j is element N g + j.
#pragma once
#include "akv_common.cuh"

namespace akv {

// D = A B + D, A 16 x 16 fp16 (row major), B 16 x 8 fp16, D fp32.  Lane (g, t): a[0], a[2] = row g, a[1], a[3] = row g + 8, with
// indices (2t, 2t+1) and (2t+8, 2t+9) of the sum; b0, b1 = column g, the same indices; d[0], d[1] = row g, columns 2t, 2t + 1,
// d[2], d[3] = row g + 8.
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// Eight elements of one line: h = their high bytes, m and l their nibbles (the even element in the high nibble) ->
// w[0] = elements 0 and 2, w[1] = 4 and 6, w[2] = 1 and 3, w[3] = 5 and 7, as fp16.
__device__ __forceinline__ void line8(uint32_t (&w)[4], uint32_t h0, uint32_t h1, uint32_t m, uint32_t l) {
    const uint32_t even = (m & 0xF0F0F0F0u) | ((l >> 4) & 0x0F0F0F0Fu);      // low bytes of elements 0, 2, 4, 6
    const uint32_t odd = ((m << 4) & 0xF0F0F0F0u) | (l & 0x0F0F0F0Fu);       // ... 1, 3, 5, 7
    w[0] = __byte_perm(even, h0, 0x6140);
    w[1] = __byte_perm(even, h1, 0x6342);
    w[2] = __byte_perm(odd, h0, 0x7150);
    w[3] = __byte_perm(odd, h1, 0x7352);
}

// The same eight elements in order.
__device__ __forceinline__ uint4 halves8(uint32_t h0, uint32_t h1, uint32_t m, uint32_t l) {
    const uint32_t even = (m & 0xF0F0F0F0u) | ((l >> 4) & 0x0F0F0F0Fu), odd = ((m << 4) & 0xF0F0F0F0u) | (l & 0x0F0F0F0Fu);
    const uint32_t a = __byte_perm(even, odd, 0x5140), b = __byte_perm(even, odd, 0x7362);
    return make_uint4(__byte_perm(a, h0, 0x5140), __byte_perm(a, h0, 0x7362), __byte_perm(b, h1, 0x5140), __byte_perm(b, h1, 0x7362));
}

// What a lane holds of one line: N elements, N / 8 groups of eight.
template <int N>
struct Line {
    uint32_t h[N / 4], m[N / 8], l[N / 8];
    __device__ __forceinline__ void load(uint32_t f8, uint32_t m4, uint32_t l4) {      // shared memory
        if constexpr (N == 16) {
            const uint4 a = lds128(f8);
            const uint2 b = lds64(m4), c = lds64(l4);
            h[0] = a.x; h[1] = a.y; h[2] = a.z; h[3] = a.w;
            m[0] = b.x; m[1] = b.y;
            l[0] = c.x; l[1] = c.y;
        } else {
            const uint2 a = lds64(f8);
            h[0] = a.x; h[1] = a.y;
            m[0] = lds32(m4);
            l[0] = lds32(l4);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) h[i] = 0;
#pragma unroll
        for (int i = 0; i < N / 8; ++i) m[i] = l[i] = 0;
    }
};

// acc[j] += A (16 x 16) times column j of the four lines, for the lane's N elements.
template <int N>
__device__ __forceinline__ void mma_lines(float (*acc)[4], const uint4& a, const Line<N> (&x)[4]) {
#pragma unroll
    for (int e = 0; e < N / 8; ++e) {
        uint32_t w[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) line8(w[i], x[i].h[2 * e], x[i].h[2 * e + 1], x[i].m[e], x[i].l[e]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int j = 8 * e + (r & 1) * 4 + (r >> 1);          // elements j and j + 2
            mma_f16(acc[j], a, __byte_perm(w[0][r], w[1][r], 0x5410), __byte_perm(w[2][r], w[3][r], 0x5410));
            mma_f16(acc[j + 2], a, __byte_perm(w[0][r], w[1][r], 0x7632), __byte_perm(w[2][r], w[3][r], 0x7632));
        }
    }
}

}  // namespace akv
