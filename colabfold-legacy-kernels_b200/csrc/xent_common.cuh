// Row arithmetic of the linear softmax cross entropy, shared by its general path and its path for heads
// of few classes.
#pragma once

#include <climits>

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

// What a row's exponentials are taken against in the log2 domain: its largest logit m times log2 e,
// as a rounded product (never one fused into what it is subtracted from, so that all of a row's sums
// mean the same value), 0 where that is -inf.
__device__ __forceinline__ float log2_of(float m) { return __fmul_rn(m, kLog2e); }
__device__ __forceinline__ float log2_ref(float m) {
    const float r = log2_of(m);
    return r == -kInf ? 0.f : r;
}

// (m, s) of a row takes another part of it in: sums s of 2^(l log2 e - log2_ref(m))
__device__ __forceinline__ void join_stats(float& m, float& s, float m2, float s2) {
    const float m1 = fmaxf(m, m2), ref = log2_ref(m1);
    s = s * ex2(log2_of(m) - ref) + s2 * ex2(log2_of(m2) - ref);
    m = m1;
}

// A row's lse (log2 domain) and loss, from its largest logit m, the sum of 2^(l log2 e - m log2 e -
// off) and its label's logit. The loss is their difference, which the logits' size leaves exact to a
// rounding, and the logarithm of the sum, which is at least 1: log s + m - at_label in this order, or
// rows that are sure of their label lose what is left of the loss to the roundings of m log2 e. No
// loss where the lse is -inf.
__device__ __forceinline__ void row_loss(float m, float s, float off, float at_label, float& loss,
                                         float& lse) {
    const bool none = log2_of(m) == -kInf && s == s;
    const float l2 = log2f(s) + off, rest = kLn2 * l2;
    lse = none ? -kInf : fmaf(m, kLog2e, l2);
    loss = none ? 0.f : (m - at_label) + (rest < 0.f ? 0.f : rest);
}
// ... and `off` of sums against log2_ref(m)
__device__ __forceinline__ float ref_off(float m) { return fmaf(-m, kLog2e, log2_ref(m)); }

// N accumulators of a row (columns c0.. of V; `bias`, or null, their biases in shared memory, 16-byte
// aligned) into its maximum m and sum s (relative to log2_ref(m)); at_label takes the label's
// logit. Columns past V count as -inf; where nothing is left m stays -inf and s 0.
template <int N>
__device__ __forceinline__ void row_stats(const uint32_t (&v)[N], int c0, int V, int label,
                                          const float* bias, float& m, float& s,
                                          float& at_label) {
    float y[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        y[j] = __uint_as_float(v[j]);
    }
    if (bias != nullptr) {
#pragma unroll
        for (int q = 0; q < N / 4; ++q) {
            const float4 b = reinterpret_cast<const float4*>(bias)[q];
            y[4 * q] += b.x;
            y[4 * q + 1] += b.y;
            y[4 * q + 2] += b.z;
            y[4 * q + 3] += b.w;
        }
    }
    if (c0 + N > V) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            y[j] = c0 + j < V ? y[j] : -kInf;
        }
    }
    const int at = label - c0;
    if (at >= 0 && at < N) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            at_label = j == at ? y[j] : at_label;
        }
    }
    float top = y[0];
#pragma unroll
    for (int j = 1; j + 1 < N; j += 2) {
        top = max3(top, y[j], y[j + 1]);
    }
    top = fmaxf(top, y[N - 1]);
    const float m1 = fmaxf(m, top), ref = log2_ref(m1);
    const uint64_t log2e = pk2(kLog2e, kLog2e), off = pk2(-ref, -ref);
    float part0 = 0.f, part1 = 0.f;
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        const float2 e = upk2(fma2(pk2(y[j], y[j + 1]), log2e, off));
        part0 += ex2(e.x);
        part1 += ex2(e.y);
    }
    s = s * ex2(log2_of(m) - ref) + (part0 + part1);
    m = m1;
}

// What a row needs to turn logits into g = dl (softmax - onehot): its log2-domain lse, dl and
// label (relative to the columns). A row without a token or with no class left is set so that its g
// comes out as zeros.
struct GradRow {
    float lse2, dl;
    int label;
    __device__ __forceinline__ void kill() {
        lse2 = kInf;
        dl = 0.f;
        label = INT_MIN / 2;
    }
};

// N accumulators of a row to g, as row_stats takes them. Columns past V give zeros. Pairs of
// columns share an instruction where they can.
template <int N>
__device__ __forceinline__ void row_grad(const uint32_t (&v)[N], float (&y)[N], int c0, int V,
                                         const GradRow& row, const float* bias) {
    const uint64_t log2e = pk2(kLog2e, kLog2e), ref = pk2(-row.lse2, -row.lse2);
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        uint64_t l0 = pk2(__uint_as_float(v[4 * q]), __uint_as_float(v[4 * q + 1]));
        uint64_t l1 = pk2(__uint_as_float(v[4 * q + 2]), __uint_as_float(v[4 * q + 3]));
        if (bias != nullptr) {
            const float4 b = reinterpret_cast<const float4*>(bias)[q];
            l0 = add2(l0, pk2(b.x, b.y));
            l1 = add2(l1, pk2(b.z, b.w));
        }
        const float2 e0 = upk2(fma2(l0, log2e, ref)), e1 = upk2(fma2(l1, log2e, ref));
        y[4 * q] = ex2(e0.x);
        y[4 * q + 1] = ex2(e0.y);
        y[4 * q + 2] = ex2(e1.x);
        y[4 * q + 3] = ex2(e1.y);
    }
    const int at = row.label - c0;
    if (at >= 0 && at < N) {
        const unsigned bit = 1u << at;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (bit & (1u << j)) {
                y[j] -= 1.f;
            }
        }
    }
    const uint64_t dl = pk2(row.dl, row.dl);
#pragma unroll
    for (int q = 0; q < N / 2; ++q) {
        const float2 g = upk2(mul2(pk2(y[2 * q], y[2 * q + 1]), dl));
        y[2 * q] = g.x;
        y[2 * q + 1] = g.y;
    }
    if (c0 + N > V) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            y[j] = c0 + j < V ? y[j] : 0.f;
        }
    }
}

}  // namespace cflk
