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
    long long total, nw;       // tiles of all units, runs that they are dealt to (at most as many): warps, or CTAs
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

// Element of a row's tensors [B,T,Hq,...]: query row r of KV head h of sequence b.
__device__ __forceinline__ long long row_of(const TreeArgs& p, long long b, int h, int r) {
    return (b * p.T + r / p.G) * p.H * p.G + (long long)h * p.G + r % p.G;
}

// Tensor-core form (akv_tree_wide.cu).
int launch_tree_wide(const TreeArgs& p, int D, int ctas, cudaStream_t st);
int launch_weights_wide(const TreeArgs& p, int D, int ctas, float* weights, cudaStream_t st);

}  // namespace akv
