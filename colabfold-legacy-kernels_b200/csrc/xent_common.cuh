// Row arithmetic of the linear softmax cross entropy, shared by its general path and its path for heads
// of few classes.
#pragma once

#include "sm100.cuh"

namespace cflk {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_huge_valf();

// the token's class, -1 where the label names none
template <typename L>
__device__ __forceinline__ int label_of(const L* labels, long long t, long long V) {
    const long long l = (long long)labels[t];
    return l >= 0 && l < V ? (int)l : -1;
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    }
    return x;
}

__device__ __forceinline__ int warp_sum(int x) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, d);
    }
    return x;
}

// The power of two that brings a positive finite m into [2^13, 2^14); 1 for 0
__device__ __forceinline__ float grad_scale(float m) {
    if (!(m > 0.f)) {
        return 1.f;
    }
    int e;
    frexpf(m, &e);  // m = f 2^e, f in [0.5, 1)
    return exp2f((float)min(14 - e, 126));
}

// 32 logits of a row, columns c0.. of V, into its log2-domain maximum m and sum s (relative to m);
// at_label takes the label's logit. Columns past V count as -inf; where nothing is left m stays -inf
// and s 0.
__device__ __forceinline__ void row_stats(float (&y)[32], int c0, int V, int label, float& m,
                                          float& s, float& at_label) {
    if (c0 + 32 > V) {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            y[j] = c0 + j < V ? y[j] : -kInf;
        }
    }
    const int at = label - c0;
    if (at >= 0 && at < 32) {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            at_label = j == at ? y[j] : at_label;
        }
    }
    float top = y[0];
#pragma unroll
    for (int j = 1; j + 1 < 32; j += 2) {
        top = max3(top, y[j], y[j + 1]);
    }
    top = fmaxf(top, y[31]);
    const float m1 = fmaxf(m, top * kLog2e);
    const float ref = m1 == -kInf ? 0.f : m1;
    float part0 = 0.f, part1 = 0.f;
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
        part0 += ex2(fmaf(y[j], kLog2e, -ref));
        part1 += ex2(fmaf(y[j + 1], kLog2e, -ref));
    }
    s = s * ex2(m - ref) + (part0 + part1);
    m = m1;
}

// 32 logits to g = dl (softmax - onehot) with the row's log2-domain lse; zeros past V and in a dead row
__device__ __forceinline__ void row_grad(float (&y)[32], int c0, int V, int label, float lse2,
                                         float dl, bool dead) {
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        y[j] = ex2(fmaf(y[j], kLog2e, -lse2));
    }
    const int at = label - c0;
    if (at >= 0 && at < 32) {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            y[j] -= j == at ? 1.f : 0.f;
        }
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        y[j] = dead || c0 + j >= V ? 0.f : y[j] * dl;
    }
}

}  // namespace cflk
