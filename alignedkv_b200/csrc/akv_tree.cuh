// What the kernels of the attention over drafted tokens share.
#pragma once
#include "akv_common.cuh"

namespace akv {

constexpr int BLK = 64, TILE = 128;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// Probabilities enter their product as fp16, since the values are fp16 and both operands of the tensor cores have one type: a second
// product with what the rounding leaves (half a step, 2^-11 of each) would double the work on P V.  Relative to the running maximum and
// times 2^15 they are at most 32768, and down to 2^-29 of the largest with all 11 bits (2^-14 without the factor).  Outputs are divided by
// the fp32 sum of the ROUNDED probabilities, so that what all of a row's have in common cancels: an average of equal values is
// that value, and a single dominating token comes out as it is.  The logarithm of the sum takes the exact ones.
// (Divided by the sum of the exact ones, up to a tenth of the elements of such averages were a step off; against 64 bits 2.5e-4 instead of
// 2.3e-4 at 16 x 8 x 8190 tokens, 48 rows, where the output's own rounding is 2.1e-4.  For 0 to 2% of the time.)
constexpr float LIFT = 15.f;

struct TreeArgs {
    const uint8_t *k8, *km, *kl, *v8, *vm, *vl;
    const __half *restk, *restv, *q, *kd, *vd, *mask;
    const uint8_t* tree;
    long long tree_stride, mask_stride;
    __half* out;
    float *lse, *part;
    int H, G, T, nmb, L, nb, rest;
    int rowsu, rt;             // query rows of a unit, units of a (batch, KV head)
    int tiles, tail;           // tiles of a unit; tokens of its last, the tail tile
    int total, nw;             // tiles of all units, runs that they are dealt to (at most as many): warps, or CTAs
    int team;                  // (tree_kernel) CTAs of a cluster that has a unit to itself, or 0
    int groups, rowsg;         // (tree_wide_kernel) row groups of a unit, rows of a group
    float scale, scale2;       // scale2 = scale * log2(e)
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// 16 bytes global -> shared past L1; with `there` false zeros, and nothing is read.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// x + the lower, the upper of two halves.
__device__ __forceinline__ float plus_low(float x, uint32_t h) {
    asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\nadd.rn.f32.f16 %0, lo, %0;\n}\n" : "+f"(x) : "r"(h));
    return x;
}
__device__ __forceinline__ float plus_high(float x, uint32_t h) {
    asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\nadd.rn.f32.f16 %0, hi, %0;\n}\n" : "+f"(x) : "r"(h));
    return x;
}

// (Indices of tiles, units and rows fit 32 bits - the launchers see to it - and are divided as such: a 64-bit division is a hundred
// instructions, and the kernels are bound by the fetch of their instructions before anything else is used up.)
// Row of the tensors [B,T,Hq,...]: query row r of KV head h of sequence b.
__device__ __forceinline__ int row_of(const TreeArgs& p, int b, int h, int r) {
    const int t = (unsigned)r / (unsigned)p.G;
    return (b * p.T + t) * (p.H * p.G) + h * p.G + r - t * p.G;
}
// First tile of run w (of run w + 1: its end): the first total % nw runs have one more.
__device__ __forceinline__ int run_start(const TreeArgs& p, int w) {
    const unsigned each = (unsigned)p.total / (unsigned)p.nw;
    return w * each + min(w, (int)(p.total - each * p.nw));
}
// Run that has tile i.
__device__ __forceinline__ int run_with(const TreeArgs& p, int i) {
    const unsigned each = (unsigned)p.total / (unsigned)p.nw, more = p.total - each * p.nw, bound = more * (each + 1);
    return (unsigned)i < bound ? (unsigned)i / (each + 1) : more + ((unsigned)i - bound) / each;
}

// Tail values that are not finite.  What one row sees of the drafted tokens is masked for another, and 0 * inf would be NaN: such
// values enter the product as zeros, and a row that sees them adds p . v to what it has written (p relative to 2^base, times `inv`).
// The rare way: by itself, and out of line.
template <class To>
static __device__ __noinline__ void add_odd(const TreeArgs& p, int b, int h, int r, int D, float base, float inv, To to) {
    const __half* q = p.q + (long long)row_of(p, b, h, r) * D;
    const __half* mask = p.mask ? p.mask + b * p.mask_stride + p.nb * BLK : nullptr;
    const uint8_t* seen = p.tree + b * p.tree_stride + (unsigned)r / (unsigned)p.G * p.T;
#pragma unroll 1
    for (int i = 0; i < p.tail; ++i) {
        const int d = i - p.rest;
        const long long at = ((long long)(d < 0 ? b * BLK + i : b * p.T + d) * p.H + h) * D;
        const __half *k = (d < 0 ? p.restk : p.kd) + at, *v = (d < 0 ? p.restv : p.vd) + at;
        const float add = d < 0 && mask ? __half2float(mask[i]) : 0.f;
        if (d < 0 ? add == -INFINITY : !seen[d]) continue;
        float pr = -1.f;
#pragma unroll 1
        for (int c = 0; c < D; ++c) {
            const float x = __half2float(v[c]);
            if (isfinite(x)) continue;
            if (pr < 0.f) {
                float dot = 0.f;
#pragma unroll 1
                for (int j = 0; j < D; ++j) dot = fmaf(__half2float(q[j]), __half2float(k[j]), dot);
                pr = ex2(fmaf(dot, p.scale2, add * LOG2E) - base) * inv;
            }
            auto& y = to[c];
            y = (float)y + pr * x;
        }
    }
}
__device__ __forceinline__ uint32_t finite_halves(uint32_t w, bool& odd) {
    if ((w & 0x7C00u) == 0x7C00u) { w &= 0xFFFF0000u; odd = true; }
    if ((w & 0x7C000000u) == 0x7C000000u) { w &= 0xFFFFu; odd = true; }
    return w;
}

// Tensor-core form (akv_tree_wide.cu).
int launch_tree_wide(const TreeArgs& p, int D, int ctas, int units, cudaStream_t st);
int launch_weights_wide(const TreeArgs& p, int D, int ctas, float* weights, cudaStream_t st);

}  // namespace akv
