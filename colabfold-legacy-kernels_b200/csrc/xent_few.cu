// Linear softmax cross entropy of at most 64 tokens over many classes (scoring single tokens): the
// weights are read once, at HBM's rate, and nothing else matters.
//
//   * the product is taken the other way round, l^T = w x^T: 128 classes are the M rows (tensor-
//     memory lanes) of an MMA, the tokens its 16 to 64 columns, so the tensor cores do no padding
//     work and a thread holds one class;
//   * a CTA takes a range of classes (whole groups of 32, the TMA box, so that all SMs read the
//     same share) and streams it through eight 24 KB stages;
//   * a thread keeps a running (max, sum of exponentials against it) a token over all classes it
//     sees, one exponential a logit; lanes and warps are joined once, at the end, and the CTAs by a second
//     kernel in order. No token list: a row without a label is computed and dropped.
//
// 4 tokens, 32000 classes, 1024 channels (66 MB of weights): 17 us with the join, 27 us through the
// 256 x 256 tiles of the general path. What is left beside the stream (10 us at the copy rate) is
// the start of the CTAs and of the second kernel.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "capi_internal.h"
#include "cflk_b200.h"
#include "launch.cuh"
#include "sm100.cuh"
#include "tmap.h"
#include "vec_io.cuh"
#include "xent_common.cuh"

namespace cflk {
namespace {

__device__ unsigned g_status;

constexpr int kFew = 64;             // tokens
constexpr int kThreads = 384;        // TMA warp, MMA warp, two idle, two warpgroups of 32 tokens each
constexpr int kEpiWarp0 = 4;
constexpr int kGroup = 32;           // classes a TMA box
constexpr int kStages = 8;
// 64 channels of w and x (of up to kFew tokens)
constexpr int kW = 128 * 128, kX = kFew * 128, kStageBytes = kW + kX;
constexpr int kSmemBytes = kStages * kStageBytes + 1024;
constexpr int kSms = 148;
constexpr float kLowest = -3.402823466e38f;  // a maximum of nothing that subtracts without NaN
constexpr unsigned long long kDrainLimitNs = 200000000ull;

struct FewArgs {
    const void* bias;
    const void* labels;
    float2* part;       // [CTA][kFew]
    float* lab_logit;   // [kFew]
    int T, V, C;
    int per;            // classes a CTA
};

template <typename T, typename L>
__global__ void __launch_bounds__(kThreads, 1)
    few_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx,
               const FewArgs a) {
    begin_next();
    using E = Elem<T>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2], drain;
    __shared__ uint32_t tmem_sh;
    __shared__ int abort_flag;
    __shared__ float2 joined[8][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int v0 = blockIdx.x * a.per;
    const int v1 = a.V - v0 < a.per ? a.V : v0 + a.per;  // (v0 + per may pass 2^31)
    const int tiles = (v1 - v0 + 127) / 128, nk = (a.C + 63) / 64;
    const int cols = (a.T + 15) & ~15;

    if (warp == 1) {
        if (lane == 0) {
            for (int i = 0; i < kStages; ++i) {
                mbar_init(&full[i], 1);
                mbar_init(&empty[i], 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(&acc_full[i], 1);
                mbar_init(&acc_empty[i], 8);
            }
            mbar_init(&drain, 1);
            abort_flag = 0;
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(&tmem_sh, 128);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_sh;

    if (warp == 0 && lane == 0) {
        int g = 0;
        bool ok = true;
        for (int t = 0; ok && t < tiles; ++t) {
            const int c0 = v0 + 128 * t, groups = (min(128, v1 - c0) + kGroup - 1) / kGroup;
            for (int kb = 0; kb < nk; ++kb, ++g) {
                const int s = g % kStages;
                if (g >= kStages && !mbar_wait(&empty[s], ((g - kStages) / kStages) & 1, &g_status,
                                               kStatusMmaWait, &abort_flag)) {
                    ok = false;
                    break;
                }
                uint8_t* st = smem + s * kStageBytes;
                mbar_arrive_expect_tx(&full[s], groups * (kGroup * 128) + cols * 128);
                for (int i = 0; i < groups; ++i) {
                    tma_load_2d(st + i * kGroup * 128, &tw, &full[s], 64 * kb, c0 + kGroup * i);
                }
                tma_load_2d(st + kW, &tx, &full[s], 64 * kb, 0);
            }
        }
        for (int h = g > kStages ? g - kStages : 0; h < g; ++h) {
            mbar_wait(&full[h % kStages], (h / kStages) & 1, &g_status, kStatusTmaWait, nullptr,
                      kDrainLimitNs);
        }
    } else if (warp == 1 && lane == 0) {
        const uint32_t idesc = idesc_f16(E::kBf16, 128, cols, false, false);
        int g = 0;
        bool ok = true;
        for (int t = 0; ok && t < tiles; ++t) {
            if (t >= 2 && !mbar_wait(&acc_empty[t & 1], ((t >> 1) - 1) & 1, &g_status,
                                     kStatusSyncWait, &abort_flag)) {
                break;
            }
            tc_fence_after();
            for (int kb = 0; kb < nk; ++kb, ++g) {
                const int s = g % kStages;
                if (!mbar_wait(&full[s], (g / kStages) & 1, &g_status, kStatusTmaWait,
                               &abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t at = smem_u32(smem + s * kStageBytes);
                mma_ss_k4(tmem + 64 * (t & 1), desc_lo(at, 16), desc_lo(at + kW, 16), 2, 2, idesc,
                          kb);
                mma_commit(&empty[s]);
            }
            if (ok) {
                mma_commit(&acc_full[t & 1]);
            }
        }
        mma_commit(&drain);
        mbar_wait(&drain, 0, &g_status, kStatusMmaWait, nullptr, kDrainLimitNs);
    } else if (warp >= kEpiWarp0) {
        const int g = (warp - kEpiWarp0) >> 2, r = ((warp & 3) << 5) | lane;  // tokens 32 g ..
        const int tok0 = 32 * g;
        const bool some = tok0 < a.T;
        // this lane's token of the group, and its class
        const int my_tok = tok0 + lane;
        const int my_label = my_tok < a.T ? label_of(static_cast<const L*>(a.labels), my_tok, a.V) : -1;
        float m[32], s[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            m[j] = kLowest;
            s[j] = 0.f;
        }
        for (int t = 0; t < tiles; ++t) {
            const int c0 = v0 + 128 * t, cls = c0 + r;
            const float bias = a.bias != nullptr && cls < v1
                                   ? E::to_f(static_cast<const T*>(a.bias)[cls])
                                   : 0.f;
            mbar_wait(&acc_full[t & 1], (t >> 1) & 1, &g_status, kStatusMmaWait, &abort_flag);
            tc_fence_after();
            if (some) {
                uint32_t v[32];
                tmem_ld32(tmem + 64 * (t & 1) + tok0 + tmem_lane_base(warp), v);
                tmem_wait_ld();
                // tokens whose label is among this warp's 32 classes
                const int rel = my_label - (c0 + 32 * (warp & 3));
                unsigned hit = __ballot_sync(0xffffffffu, rel >= 0 && rel < 32);
                while (hit != 0) {
                    const int j = __ffs(hit) - 1;
                    hit &= hit - 1;
                    const int at = __shfl_sync(0xffffffffu, rel, j);
                    float z = 0.f;
#pragma unroll
                    for (int q = 0; q < 32; ++q) {
                        z = q == j ? __uint_as_float(v[q]) : z;
                    }
                    if (lane == at && cls < v1) {
                        a.lab_logit[tok0 + j] = z + bias;
                    }
                }
                if (cls < v1) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        if (j % 8 == 0 && tok0 + j >= a.T) {
                            break;  // eights of tokens
                        }
                        // one exponential: of the smaller of the two, relative to the larger
                        const float y = __uint_as_float(v[j]) + bias;
                        const float d = (y - m[j]) * kLog2e;
                        const float e = ex2(-fabsf(d));
                        s[j] = d > 0.f ? fmaf(s[j], e, 1.f) : s[j] + e;
                        m[j] = fmaxf(m[j], y);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&acc_empty[t & 1]);
            }
        }
        // lanes, then the warps of the group
        if (some) {
            float keep_m = kLowest, keep_s = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                if (j % 8 == 0 && tok0 + j >= a.T) {
                    break;
                }
                float top = m[j];
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) {
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                }
                float sum = s[j] * ex2((m[j] - top) * kLog2e);
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) {
                    sum += __shfl_xor_sync(0xffffffffu, sum, d);
                }
                keep_m = lane == j ? top : keep_m;
                keep_s = lane == j ? sum : keep_s;
            }
            joined[warp - kEpiWarp0][lane] = make_float2(keep_m, keep_s);
            named_sync(1 + g, 128);
            if ((warp & 3) == 0) {
                float2 p = joined[4 * g][lane];
#pragma unroll
                for (int w = 1; w < 4; ++w) {
                    const float2 q = joined[4 * g + w][lane];
                    const float top = fmaxf(p.x, q.x);
                    p.y = p.y * ex2((p.x - top) * kLog2e) + q.y * ex2((q.x - top) * kLog2e);
                    p.x = top;
                }
                // nothing left: as the other path's pieces say it
                a.part[blockIdx.x * kFew + my_tok] =
                    make_float2(p.x == kLowest && p.y == 0.f ? -kInf : p.x, p.y);
            }
        }
    }
    tc_fence_before();
    __syncwarp();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 128);
    }
}

// The CTAs' pieces of a token in order: a warp a token.
template <typename L>
__global__ void __launch_bounds__(256)
    few_join_kernel(const float2* part, const float* lab_logit,
                    const L* __restrict__ labels, int T, int V, int pieces,
                    float* loss, float* lse) {
    wait_before();
    const int t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (t >= T) {
        return;
    }
    float m = -kInf, s = 0.f;
    const auto join = [&](float x, float y) {
        const float m1 = fmaxf(m, x);
        const float ref = m1 == -kInf ? 0.f : m1;
        s = s * ex2((m - ref) * kLog2e) + y * ex2((x - ref) * kLog2e);
        m = m1;
    };
    float2 p[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {  // at most 8 * 32 CTAs
        const int q = lane + 32 * u;
        p[u] = q < pieces ? part[q * kFew + t] : make_float2(-kInf, 0.f);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        join(p[u].x, p[u].y);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const float x = __shfl_xor_sync(0xffffffffu, m, d), y = __shfl_xor_sync(0xffffffffu, s, d);
        join(x, y);
    }
    if (lane == 0) {
        if (label_of(labels, t, V) < 0) {
            loss[t] = 0.f;
            lse[t] = -kInf;
        } else {
            row_loss(m, s, 0.f, lab_logit[t], loss[t], lse[t]);
        }
    }
}

// classes a CTA: equal shares in whole boxes
int few_per(int64_t V) {
    const int64_t groups = (V + kGroup - 1) / kGroup;
    return (int)((groups + kSms - 1) / kSms * kGroup);
}

}  // namespace

bool xent_few_fits(int64_t T) {
    return T <= kFew;
}

size_t xent_few_workspace() {
    return (size_t)kSms * kFew * sizeof(float2) + kFew * sizeof(float);
}

cudaError_t xent_few(const HeadCall& c, bool& map_ok) {
    FewArgs a{};
    a.bias = c.bias;
    a.labels = c.labels;
    a.part = static_cast<float2*>(c.workspace);
    a.lab_logit = reinterpret_cast<float*>(a.part + kSms * kFew);
    a.T = (int)c.T;
    a.V = (int)c.V;
    a.C = (int)c.C;
    a.per = few_per(c.V);
    const int grid = (int)((c.V + a.per - 1) / a.per);
    const CUtensorMapDataType t =
        c.dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap tw, tx;
    const uint64_t dw[2] = {(uint64_t)c.C, (uint64_t)c.V}, dx[2] = {(uint64_t)c.C, (uint64_t)c.T};
    const uint64_t st[1] = {(uint64_t)c.C};
    const uint32_t bw[2] = {64, kGroup}, bx[2] = {64, (uint32_t)((c.T + 15) & ~15)};
    map_ok = encode_tiled(&tw, t, 2, 2, c.w, dw, st, bw, CU_TENSOR_MAP_SWIZZLE_128B) &&
             encode_tiled(&tx, t, 2, 2, c.x, dx, st, bx, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!map_ok) {
        return cudaSuccess;
    }
    const auto run = [&](auto tag, auto ltag) -> cudaError_t {
        using T = decltype(tag);
        using L = decltype(ltag);
        auto kern = few_kernel<T, L>;
        static bool done[kMaxDevices] = {};
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e == cudaSuccess && (dev >= kMaxDevices || !done[dev])) {
            e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
            if (e == cudaSuccess && dev < kMaxDevices) {
                done[dev] = true;
            }
        }
        if (e != cudaSuccess) {
            return e;
        }
        kern<<<grid, kThreads, kSmemBytes, c.stream>>>(tw, tx, a);
        launch_behind(few_join_kernel<L>, (a.T + 7) / 8, 256, 0, c.stream, a.part, a.lab_logit,
                      static_cast<const L*>(c.labels), a.T, a.V, grid, c.loss, c.lse);
        return cudaGetLastError();
    };
    if (c.labels_64) {
        return c.dtype == kBF16 ? run(__nv_bfloat16{}, (long long)0) : run(__half{}, (long long)0);
    }
    return c.dtype == kBF16 ? run(__nv_bfloat16{}, 0) : run(__half{}, 0);
}

unsigned read_and_clear_status_few() {
    unsigned v = 0, z = 0;
    cudaMemcpyFromSymbol(&v, g_status, sizeof(v));
    cudaMemcpyToSymbol(g_status, &z, sizeof(z));
    return v;
}

}  // namespace cflk
