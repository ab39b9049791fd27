// SiLU without the library's expf and division: what the 8-bit product's SwiGLU and
// the DeltaNet mixer over trees share.
#pragma once

#include "common.hpp"

// x / (1 + exp(-x)) in a third of the instructions of expf and a division: exp2 of
// the product with log2 e, whose rounding error is put back, and a reciprocal
// with one Newton step; off by 3 + 1 + 1 + 1 roundings at most (the exponential,
// the sum, the reciprocal, the product) from kDeepGate up, +inf included. Below
// kDeepGate, where the exponential stays at exp(80), callers put their own value.
// Every fused multiply-add is written out, so that every use gives the same bits.
constexpr float kDeepGate = -80.0f;
__device__ __forceinline__ float silu_fast(float x) {
#pragma clang fp contract(off)
    constexpr float kLog2e = 1.44269502e0f, kRest = 1.92596303e-8f, kLn2 = 0.693147182f;
    // (past 200 the exponential is 0; an infinite x has no rounding error)
    const float c = __builtin_amdgcn_fmed3f(x, kDeepGate, 200.0f);
    const float hi = c * -kLog2e;
    const float lo = fmaf(-c, kRest, fmaf(c, -kLog2e, -hi));
    float e = __builtin_amdgcn_exp2f(hi);
    e = fmaf(e * kLn2, lo, e);
    const float d = 1.0f + e;
    float r = __builtin_amdgcn_rcpf(d);
    r = fmaf(fmaf(-d, r, 1.0f), r, r);
    return x * r;
}
