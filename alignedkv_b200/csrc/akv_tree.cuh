// What the kernels of the attention over drafted tokens share.
#pragma once
#include "akv_common.cuh"

namespace akv {

constexpr int BLK = 64, TILE = 128;
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
    int H, G, T, nmb, L, nb, rest;
    int rowsu, rt;             // query rows of a unit, units of a (batch, KV head)
    int tiles, tail;           // tiles of a unit; tokens of its last, the tail tile
    int total, nw;             // tiles of all units, runs that they are dealt to (at most as many): warps, or CTAs
    int groups, rowsg;         // (tree_wide_kernel) row groups of a unit, rows of a group
    float scale, scale2;       // scale2 = scale * log2(e)
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
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

// Tensor-core form (akv_tree_wide.cu).
int launch_tree_wide(const TreeArgs& p, int D, int ctas, cudaStream_t st);
int launch_weights_wide(const TreeArgs& p, int D, int ctas, float* weights, cudaStream_t st);

}  // namespace akv
