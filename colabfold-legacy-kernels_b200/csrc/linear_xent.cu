// Softmax cross entropy of a linear layer's classes without keeping the logits, and its gradients.
//
//   l = x w^T + b (T tokens, V classes, C channels);  lse = log sum_v exp l;  loss = lse - l[label]
//   g = dloss (softmax(l) - onehot(label));  dx = g w;  dw = g^T x;  db = sum_t g
//
// A token whose label lies outside [0, V) has no loss and no gradient; its row of x is never used
// (it may hold anything). The labelled rows are gathered into consecutive rows first, so the
// products cost what the labelled tokens cost; their number stays on the device, where every
// kernel reads it.
//
//   * one persistent GEMM kernel serves the four products: a pair of CTAs (cta_group::2) computes
//     256 x 256 tiles, each CTA streaming its 128 rows of A and its 128 of B by TMA through a ring
//     of five 32 KB stages, the leader issuing the MMAs into one of two tensor-memory
//     accumulators, two warpgroups a CTA (four where g is made) draining the other;
//   * forward: the epilogue reduces each row's 128 columns to (max, sum of exponentials), a second
//     kernel joins a row's pieces in order;
//   * backward: the classes are taken in pieces; per piece the epilogue turns recomputed logits
//     into g, rounded to the 16-bit type into the workspace, and g is multiplied by w (adding to
//     float32 sums of dx) and, transposed, by x. The rounding of g (relative 2^-8 in bf16, 2^-11
//     in f16) is of the size of the outputs' own rounding and is what feeding the tensor cores
//     takes; dloss is first scaled by a power of two that brings its largest magnitude to 2^13,
//     so that f16 keeps g's small values, and the factor is taken out before the outputs round;
//   * sums, exponentials and row statistics are float32; products whose tiles are too few for the
//     machine are split along K into float32 slabs added in order. No atomics: the same bits
//     every run;
//   * heads of few classes (xent_head.cu) and the forward of few tokens (xent_few.cu), which HBM
//     bounds, have kernels of their own.
//
// Bound by the tensor cores: 2 T V C operations forward, 6 T V C backward, 2 of them the logits
// again, which not keeping them costs. T 4096, V 16384, C 1024, bf16, under a profiler: the logits'
// product 96 us (tensor pipe active 82 %), g 111 (69 %), dx 101 (88 %), dw 109 (77 %). T 8192,
// V 100003, C 2048: 13.4 TFLOP in 9.6 to 10.6 ms, 1.27 to 1.40 PFLOP/s where a library product of
// 8192^3 holds 1.41 for seconds; the GPU's power is the limit there.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <string>

#include "capi_internal.h"
#include "cflk_b200.h"
#include "launch.cuh"
#include "pair_mma.cuh"
#include "sm100.cuh"
#include "tmap.h"
#include "vec_io.cuh"
#include "xent_common.cuh"

namespace cflk {
namespace {

__device__ unsigned g_status;

// ------------------------------------------------------------------------------------------
// the labelled tokens
// ------------------------------------------------------------------------------------------
constexpr int kPrepThreads = 256, kPrepItems = 1024;  // tokens a block

// counts[b]: the block's labelled tokens; maxs[b]: the largest finite |dloss| among them (backward)
template <typename L>
__global__ void __launch_bounds__(kPrepThreads)
    xent_count_kernel(const L* __restrict__ labels, const float* __restrict__ dloss, int T,
                      long long V, int* __restrict__ counts, float* __restrict__ maxs) {
    begin_next();
    __shared__ int sc[8];
    __shared__ float sm[8];
    int n = 0;
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < kPrepItems / kPrepThreads; ++j) {
        const long long t = (long long)blockIdx.x * kPrepItems + j * kPrepThreads + threadIdx.x;
        if (t < T && label_of(labels, t, V) >= 0) {
            ++n;
            if (dloss != nullptr) {
                const float d = fabsf(dloss[t]);
                m = d < kInf ? fmaxf(m, d) : m;
            }
        }
    }
    n = warp_sum(n);
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) {
        sc[threadIdx.x >> 5] = n;
        sm[threadIdx.x >> 5] = m;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int s = 0;
        float mm = 0.f;
        for (int i = 0; i < 8; ++i) {
            s += sc[i];
            mm = fmaxf(mm, sm[i]);
        }
        counts[blockIdx.x] = s;
        maxs[blockIdx.x] = mm;
    }
}

struct PrepArgs {
    const float* dloss;  // backward, with lse
    const float* lse;
    float* loss;         // forward: rows without a label get 0 and lse -inf
    float* lse_out;
    const int* counts;
    const float* maxs;
    int T, nblocks;
    long long V;
    int* perm;           // [T]: the labelled tokens in order, the others from the end
    int* lab;            // labels of the labelled tokens
    float* lse_c;        // their lse and scaled dloss (backward)
    float* dl_c;
    int* count;          // labelled tokens
    float* inv;          // 1 / grad_scale
};

// Blocks put their tokens at their places: thread i holds 4 consecutive tokens.
template <typename L>
__global__ void __launch_bounds__(kPrepThreads)
    xent_compact_kernel(const L* __restrict__ labels, const PrepArgs a) {
    wait_before();
    begin_next();
    __shared__ int sc[8], so[8];
    __shared__ float sm[8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // labelled tokens before this block, and the largest |dloss| of all
    // (a single block needs no counts, and finds the largest |dloss| below)
    int before = 0;
    float m = 0.f;
    for (int i = tid; a.nblocks > 1 && i < a.nblocks; i += kPrepThreads) {
        before += i < (int)blockIdx.x ? a.counts[i] : 0;
        m = fmaxf(m, a.maxs[i]);
    }
    before = warp_sum(before);
    const long long t0 = (long long)blockIdx.x * kPrepItems + tid * 4;
    int lab[4], mine = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        lab[j] = t0 + j < a.T ? label_of(labels, t0 + j, a.V) : -1;
        mine += lab[j] >= 0;
        if (a.nblocks == 1 && a.dloss != nullptr && lab[j] >= 0) {
            const float d = fabsf(a.dloss[t0 + j]);
            m = d < kInf ? fmaxf(m, d) : m;
        }
    }
    m = warp_max(m);
    int x = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        x += lane >= d ? y : 0;
    }
    if (lane == 31) {
        so[warp] = x;
    }
    if (lane == 0) {
        sc[warp] = before;
        sm[warp] = m;
    }
    __syncthreads();
    before = 0;
    int at = x - mine, total = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        before += sc[w];
        m = fmaxf(m, sm[w]);
        at += w < warp ? so[w] : 0;
        total += so[w];
    }
    at += before;
    const float scale = grad_scale(m);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const long long t = t0 + j;
        if (t < a.T) {
            if (lab[j] >= 0) {
                a.perm[at] = (int)t;
                a.lab[at] = lab[j];
                if (a.dloss != nullptr) {
                    a.lse_c[at] = a.lse[t];
                    a.dl_c[at] = a.dloss[t] * scale;
                }
                ++at;
            } else {
                // t - at tokens without a label come before this one
                a.perm[a.T - 1 - (t - at)] = (int)t;
                if (a.loss != nullptr) {
                    a.loss[t] = 0.f;
                    a.lse_out[t] = -kInf;
                }
            }
        }
    }
    if (blockIdx.x == gridDim.x - 1 && tid == 0) {
        *a.count = before + total;
        *a.inv = 1.f / scale;
    }
}

// xc[i] = x[perm[i]] for the labelled tokens, zeros up to the next multiple of 64 (the K slices
// of dw read that far); a warp a row, 16 bytes a lane.
__global__ void __launch_bounds__(256)
    xent_gather_kernel(const uint4* __restrict__ x, const int* perm, const int* count, uint4* xc,
                       int cv) {
    wait_before();
    begin_next();
    const int n = *count, lane = threadIdx.x & 31;
    const int end = (n + 63) & ~63;
    for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < end;
         i += (long long)gridDim.x * 8) {
        const uint4* src = i < n ? x + (long long)perm[i] * cv : nullptr;
        uint4* dst = xc + i * cv;
        for (int c = lane; c < cv; c += 128) {
            uint4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                v[u] = src != nullptr && c + 32 * u < cv ? src[c + 32 * u] : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (c + 32 * u < cv) {
                    dst[c + 32 * u] = v[u];
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------
// the products
// ------------------------------------------------------------------------------------------
// kStats: rows of x w^T to (max, sum) pieces; kGrad: to g (16-bit); kDx: g w to float32 slabs;
// kDw: g^T x to the 16-bit output; kDwSlab: g^T x to float32 slabs.
enum Kind : int { kStats = 0, kGrad = 1, kDx = 2, kDw = 3, kDwSlab = 4 };

constexpr int PN = 256, PM = 256, PK = 64;  // a pair's tile, and the depth of a stage
// A TMA warp, an MMA warp, two idle, and the epilogue's warpgroups, each 256 / groups columns of
// the CTA's 128 rows. g's exponentials, roundings and stores take four, or at C = 512 the tensor
// cores wait for them (T 4095, V 32001, forward and backward: 457 us with two, 451 with four).
__host__ __device__ constexpr int epi_groups(int kind) { return kind == 1 ? 4 : 2; }
__host__ __device__ constexpr int gemm_threads(int kind) { return 128 + 128 * epi_groups(kind); }
constexpr int kEpiWarp0 = 4;
constexpr int kStages = 5;
constexpr int kHalfBytes = 128 * PK * 2;    // a CTA's rows of A, or of B, in a stage
constexpr int kStageBytes = 2 * kHalfBytes;
constexpr int kBoxBytes = 128 * 128;        // output staging: 128 rows of 128 bytes
constexpr int kSmemBytes = kStages * kStageBytes + 4 * kBoxBytes + 1024;
static_assert(kSmemBytes <= 227 * 1024, "shared memory");
constexpr unsigned long long kDrainLimitNs = 200000000ull;

struct GemmArgs {
    const int* count;     // labelled tokens
    int row0, rows;       // kStats: the rows of this launch
    int V, C;
    int v0, vp;           // the piece of the classes (vp a multiple of 256)
    int splits;           // along K (kDx, kDwSlab)
    int accumulate;       // kDx: add to the slab
    long long cap;        // rows of a statistics piece
    const int* lab;
    const void* bias;     // or null
    float2* part;         // kStats
    float* lab_logit;
    const float* lse_c;   // kGrad
    const float* dl_c;
    const float* inv;     // kDw
};

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::
                     "l"(map),
                 "r"(src), "r"(c0), "r"(c1)
                 : "memory");
}

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int c0, int c1,
                                             int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::
            "l"(map),
        "r"(src), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

__device__ __forceinline__ void tma_add_3d(const CUtensorMap* map, uint32_t src, int c0, int c1,
                                           int c2) {
    asm volatile(
        "cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], "
        "[%1];" ::"l"(map),
        "r"(src), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

__device__ __forceinline__ void bulk_commit() {
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void bulk_wait_all() {
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// The items of a pair of CTAs, one after the other: an output tile and a range of K each. The logits'
// products take rows fastest: the pairs at work share w's tiles in L2, where x stays. Those of g take
// columns fastest, so that g, the largest operand, is read from HBM once (dw at T 4096, V 16384,
// C 1024 read 471 MB with rows fastest, 3.5 times g). Positions advance by additions: the divisions
// of an item's number take the thread that issues the MMAs about as long as two of a tile's stages.
template <int KIND>
struct Walk {
    int n0, m0, kb0, kb1, split;
    long long left;

    __device__ __forceinline__ Walk(const GemmArgs& a, int n) {
        constexpr bool kDwLike = KIND == kDw || KIND == kDwSlab;
        const int rows = KIND == kStats ? max(0, min(a.rows, n - a.row0)) : n;
        const int classes = min(a.vp, a.V - a.v0);
        const int ntm = ((kDwLike ? classes : rows) + PM - 1) / PM;
        const int ntn = ((KIND == kStats || KIND == kGrad ? classes : a.C) + PN - 1) / PN;
        const int k = kDwLike ? n : KIND == kDx ? classes : a.C;
        const int nkb = (k + PK - 1) / PK;
        const int splits = KIND == kDx || KIND == kDwSlab ? a.splits : 1;
        base_ = nkb / splits;
        extra_ = nkb - base_ * splits;
        fast_n_ = KIND >= kDx ? ntn : ntm;
        slow_n_ = KIND >= kDx ? ntm : ntn;
        const int pairs = (int)(gridDim.x >> 1), first = (int)(blockIdx.x >> 1);
        left = (long long)ntm * ntn * splits - first;
        step_ = pairs;
        if (left <= 0) {
            return;  // also: no tile at all
        }
        fast_ = first % fast_n_;
        slow_ = first / fast_n_ % slow_n_;
        split = first / fast_n_ / slow_n_;
        d_fast_ = pairs % fast_n_;
        d_slow_ = pairs / fast_n_ % slow_n_;
        d_split_ = pairs / fast_n_ / slow_n_;
        place();
    }
    __device__ __forceinline__ bool more() const { return left > 0; }
    __device__ __forceinline__ void next() {
        left -= step_;
        fast_ += d_fast_;
        slow_ += d_slow_;
        split += d_split_;
        if (fast_ >= fast_n_) {
            fast_ -= fast_n_;
            ++slow_;
        }
        if (slow_ >= slow_n_) {
            slow_ -= slow_n_;
            ++split;
        }
        place();
    }

private:
    int base_, extra_, fast_n_, slow_n_, fast_, slow_, d_fast_, d_slow_, d_split_, step_;
    __device__ __forceinline__ void place() {
        m0 = (KIND >= kDx ? slow_ : fast_) * PM;
        n0 = (KIND >= kDx ? fast_ : slow_) * PN;
        kb0 = split * base_ + min(split, extra_);
        kb1 = kb0 + base_ + (split < extra_ ? 1 : 0);
    }
};

template <typename T, int KIND>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(gemm_threads(KIND), 1)
    xent_gemm_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                     const __grid_constant__ CUtensorMap to, const GemmArgs a) {
    wait_before();
    begin_next();
    using E = Elem<T>;
    constexpr bool A_MN = KIND == kDw || KIND == kDwSlab;
    constexpr bool B_MN = KIND >= kDx;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2], drain;
    __shared__ uint32_t tmem_sh;
    __shared__ int abort_flag;
    __shared__ __align__(16) float bias_sh[PN];  // of the tile's columns
    constexpr int kGroups = epi_groups(KIND), kCols = PN / kGroups, kSlots = 4 / kGroups;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int n = *a.count;

    if (warp == 1) {
        if (lane == 0) {
            for (int i = 0; i < kStages; ++i) {
                mbar_init(&full[i], 1);
                mbar_init(&empty[i], 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(&acc_full[i], 1);
                mbar_init(&acc_empty[i], 8 * kGroups);  // the epilogue warps of both CTAs
            }
            mbar_init(&drain, 1);
            abort_flag = 0;
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc_pair(&tmem_sh, 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = tmem_sh;

    if (warp == 0 && lane == 0) {
        // TMA: this CTA's halves of A and B; the leader's barrier counts both CTAs' bytes. A
        // stage is refilled once the MMAs that read it are done (in both CTAs).
        int g = 0, s = 0;  // stages filled; the next one
        uint32_t phase = 1;
        bool ok = true;
        for (Walk<KIND> it(a, n); ok && it.more(); it.next()) {
            for (int kb = it.kb0; kb < it.kb1; ++kb, ++g) {
                if (g >= kStages && !mbar_wait(&empty[s], phase, &g_status, kStatusMmaWait,
                                               &abort_flag)) {
                    ok = false;
                    break;
                }
                uint8_t* st = smem + s * kStageBytes;
                uint8_t* sb = st + kHalfBytes;
                const int k0 = kb * PK;
                if (rank == 0) {
                    mbar_arrive_expect_tx(&full[s], 2 * kStageBytes);
                }
                const uint32_t bar = map_rank(smem_u32(&full[s]), 0);
                const int m = it.m0 + 128 * (int)rank + (KIND == kStats ? a.row0 : 0);
                const int nn = it.n0 + 128 * (int)rank;
                if constexpr (A_MN) {
                    tma_load_2d_pair(st, &ta, bar, m, k0);
                    tma_load_2d_pair(st + kHalfBytes / 2, &ta, bar, m + 64, k0);
                } else {
                    tma_load_2d_pair(st, &ta, bar, k0, m);
                }
                if constexpr (B_MN) {
                    const int kr = KIND == kDx ? a.v0 + k0 : k0;
                    tma_load_2d_pair(sb, &tb, bar, nn, kr);
                    tma_load_2d_pair(sb + kHalfBytes / 2, &tb, bar, nn + 64, kr);
                } else {
                    tma_load_2d_pair(sb, &tb, bar, k0, a.v0 + nn);
                }
                if (++s == kStages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
        if (rank == 0) {
            // the last loads (one a stage at most) land before the pair can exit
            for (int h = g > kStages ? g - kStages : 0; h < g; ++h) {
                mbar_wait(&full[h % kStages], (h / kStages) & 1, &g_status, kStatusTmaWait,
                          nullptr, kDrainLimitNs);
            }
        }
    } else if (warp == 1 && lane == 0 && rank == 0) {
        const uint32_t idesc = idesc_f16(E::kBf16, PM, PN, A_MN, B_MN);
        // Descriptors of 128-byte-swizzled operands, 8-row groups 1 KB apart. K-major: a K step of 16
        // is 32 bytes along the row; MN-major: 64-wide atoms 8 KB apart, a K step is 16 rows of
        // 128 bytes. The low word holds the address and the atoms' distance in 16-byte units.
        constexpr uint32_t kAStep = A_MN ? 128 : 2, kBStep = B_MN ? 128 : 2;
        const uint32_t a0 = desc_lo(smem_u32(smem), A_MN ? 8192 : 16);
        const uint32_t b0 = desc_lo(smem_u32(smem) + kHalfBytes, B_MN ? 8192 : 16);
        int s = 0, lt = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (Walk<KIND> it(a, n); ok && it.more(); it.next()) {
            if (it.kb0 == it.kb1) {
                continue;
            }
            const int buf = lt & 1;
            if (lt >= 2 && !mbar_wait(&acc_empty[buf], ((lt - 2) >> 1) & 1, &g_status,
                                      kStatusSyncWait, &abort_flag)) {
                break;
            }
            tc_fence_after();
            const uint32_t acc = tmem + buf * PN;
            for (int kb = it.kb0; kb < it.kb1; ++kb) {
                if (!mbar_wait(&full[s], phase, &g_status, kStatusTmaWait, &abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t at = s * (kStageBytes >> 4);
                mma_pair_k4<kAStep, kBStep>(acc, a0 + at, b0 + at, idesc, kb > it.kb0);
                mma_commit_pair(&empty[s]);
                if (++s == kStages) {
                    s = 0;
                    phase ^= 1;
                }
            }
            if (ok) {
                mma_commit_pair(&acc_full[buf]);
            }
            ++lt;
        }
        // every MMA issued is complete before tensor memory is freed
        mma_commit_pair(&drain);
        mbar_wait(&drain, 0, &g_status, kStatusMmaWait, nullptr, kDrainLimitNs);
    } else if (warp >= kEpiWarp0) {
        // epilogue: warpgroup g takes columns [kCols g, kCols (g + 1)) of the CTA's 128 rows (thread
        // r = row = tensor-memory lane), with its own staging boxes, named barrier and leader
        const int g = (warp - kEpiWarp0) >> 2;
        const int r = ((warp & 3) << 5) | lane;
        const bool leader = lane == 0 && (warp & 3) == 0;
        const uint32_t lane_base = tmem_lane_base(warp);
        uint8_t* slots = smem + kStages * kStageBytes + g * kSlots * kBoxBytes;
        int lt = 0, box = 0;
        // a box of this warpgroup is free once the store of the box kSlots before it has read it
        const auto next_slot = [&]() -> uint8_t* {
            if (leader) {
                bulk_wait_read<kSlots - 1>();
            }
            named_sync(1 + g, 128);
            return slots + (box++ & (kSlots - 1)) * kBoxBytes;
        };
        [[maybe_unused]] float out_scale = 1.f;
        if constexpr (KIND == kDw) {
            out_scale = *a.inv;
        }
        for (Walk<KIND> it(a, n); it.more(); it.next()) {
            const bool none = it.kb0 == it.kb1;  // an empty K range: zeros
            const int buf = lt & 1;
            const int row = it.m0 + 128 * (int)rank + r;  // of the launch's rows
            const int col0 = it.n0 + kCols * g;
            [[maybe_unused]] int lab = INT_MIN / 2;  // no token
            [[maybe_unused]] GradRow grad;
            grad.kill();
            if constexpr (KIND == kStats || KIND == kGrad) {
                const int tok = row + (KIND == kStats ? a.row0 : 0);
                if (tok < n) {
                    lab = a.lab[tok] - a.v0;
                    // (a NaN lse is that of a row whose gradients are NaN in every class)
                    if (KIND == kGrad && !(a.lse_c[tok] == -kInf)) {
                        grad.lse2 = a.lse_c[tok];
                        grad.dl = a.dl_c[tok];
                        grad.label = lab;
                    }
                }
                if (a.bias != nullptr) {
                    named_sync(1 + g, 128);  // the previous tile's reads are done
                    if (r < kCols) {
                        const int c = a.v0 + col0 + r;
                        bias_sh[kCols * g + r] =
                            c < a.V ? E::to_f(static_cast<const T*>(a.bias)[c]) : 0.f;
                    }
                    named_sync(1 + g, 128);
                }
            }
            if (!none) {
                mbar_wait(&acc_full[buf], (lt >> 1) & 1, &g_status, kStatusMmaWait, &abort_flag);
                tc_fence_after();
                ++lt;
            }
            const uint32_t acc = tmem + buf * PN + kCols * g + lane_base;
            // the accumulator's 32 columns of chunk ch
            const auto load = [&](int ch, uint32_t (&v)[32]) {
                tmem_ld32(acc + 32 * ch, v);
                tmem_wait_ld();
            };
            if constexpr (KIND == kStats) {
                // maximum and sum of this row's columns; -inf where nothing is left
                float m = -kInf, s = 0.f, at_label = 0.f;
                const int limit = min(a.vp, a.V - a.v0);
                for (int ch = 0; ch < kCols / 32; ++ch) {
                    const int c0 = col0 + 32 * ch;
                    if (c0 >= limit) {
                        break;
                    }
                    uint32_t v[32];
                    load(ch, v);
                    row_stats<32>(v, c0, limit, lab,
                                  a.bias != nullptr ? &bias_sh[kCols * g + 32 * ch] : nullptr, m, s,
                                  at_label);
                }
                if (lab >= col0 && lab < min(col0 + 128, limit)) {
                    a.lab_logit[row + a.row0] = at_label;
                }
                const int piece = (it.n0 / PN) * 2 + g;
                a.part[piece * a.cap + row] = make_float2(m, s);
            } else if constexpr (KIND == kGrad) {
                const int limit = min(a.vp, a.V - a.v0);
                for (int j = 0; j < kCols / 64; ++j) {
                    const int b0 = col0 + 64 * j;
                    if (b0 >= limit) {
                        break;
                    }
                    uint8_t* dst = next_slot() + r * 128;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int c0 = b0 + 32 * h;
                        uint32_t v[32];
                        load(2 * j + h, v);
                        float y[32];
                        row_grad<32>(v, y, c0, limit, grad,
                                 a.bias != nullptr ? &bias_sh[kCols * g + 64 * j + 32 * h] : nullptr);
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            *reinterpret_cast<uint4*>(dst + (((4 * h + q) ^ (r & 7)) << 4)) =
                                make_uint4(E::pack(y[8 * q], y[8 * q + 1]),
                                           E::pack(y[8 * q + 2], y[8 * q + 3]),
                                           E::pack(y[8 * q + 4], y[8 * q + 5]),
                                           E::pack(y[8 * q + 6], y[8 * q + 7]));
                        }
                    }
                    fence_async_smem();
                    named_sync(1 + g, 128);
                    if (leader) {
                        tma_store_2d(&to, smem_u32(dst), b0, it.m0 + 128 * (int)rank);
                        bulk_commit();
                    }
                }
            } else if constexpr (KIND == kDw) {
                for (int j = 0; j < kCols / 64; ++j) {
                    const int b0 = col0 + 64 * j;
                    if (b0 >= a.C) {
                        break;
                    }
                    uint8_t* dst = next_slot() + r * 128;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t v[32];
                        if (!none) {
                            load(2 * j + h, v);
                        }
                        float y[32];
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            y[k] = none ? 0.f : __uint_as_float(v[k]) * out_scale;
                        }
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            *reinterpret_cast<uint4*>(dst + (((4 * h + q) ^ (r & 7)) << 4)) =
                                make_uint4(E::pack(y[8 * q], y[8 * q + 1]),
                                           E::pack(y[8 * q + 2], y[8 * q + 3]),
                                           E::pack(y[8 * q + 4], y[8 * q + 5]),
                                           E::pack(y[8 * q + 6], y[8 * q + 7]));
                        }
                    }
                    fence_async_smem();
                    named_sync(1 + g, 128);
                    if (leader) {
                        const int orow = a.v0 + it.m0 + 128 * (int)rank;
                        if (orow < a.V) {
                            tma_store_2d(&to, smem_u32(dst), b0, orow);
                        }
                        bulk_commit();
                    }
                }
            } else {
                for (int ch = 0; ch < kCols / 32; ++ch) {
                    const int c0 = col0 + 32 * ch;
                    if (c0 >= a.C) {
                        break;
                    }
                    uint32_t v[32];
                    if (!none) {
                        load(ch, v);
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            v[k] = 0;
                        }
                    }
                    uint8_t* dst = next_slot() + r * 128;
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        *reinterpret_cast<uint4*>(dst + ((q ^ (r & 7)) << 4)) =
                            make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                    }
                    fence_async_smem();
                    named_sync(1 + g, 128);
                    if (leader) {
                        const int orow = it.m0 + 128 * (int)rank;
                        if (KIND == kDx && a.accumulate) {
                            tma_add_3d(&to, smem_u32(dst), c0, orow, it.split);
                        } else {
                            tma_store_3d(&to, smem_u32(dst), c0, orow, it.split);
                        }
                        bulk_commit();
                    }
                }
            }
            if (!none) {
                // this warp's columns of the accumulator are read
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive_cluster(map_rank(smem_u32(&acc_empty[buf]), 0));
                }
            }
        }
        if (leader) {
            bulk_wait_all();
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (rank == 1 && warp == 1 && lane == 0) {
        // the leader commits `drain` after every other arrive on this CTA's barriers: once it has
        // come, none is under way to a CTA that exits
        mbar_wait(&drain, 0, &g_status, kStatusMmaWait, nullptr, 2 * kDrainLimitNs);
    }
    __syncwarp();
    cluster_sync_all();  // no CTA leaves while its pair may still signal or load into it
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

// ------------------------------------------------------------------------------------------
// joins
// ------------------------------------------------------------------------------------------
// Rows' pieces to lse and loss: 32 rows a block, eight threads a row over every eighth piece,
// joined in order. A row with no class left (every logit -inf) counts as without a label.
__global__ void __launch_bounds__(256)
    xent_join_kernel(const float2* part, const float* lab_logit, const int* perm, const int* count,
                     int row0, int rows, long long cap, int pieces, float* loss, float* lse) {
    wait_before();
    __shared__ float2 sh[8][32];
    const int n = *count;
    const int r = threadIdx.x & 31, seg = threadIdx.x >> 5;
    const int row = blockIdx.x * 32 + r;
    const bool live = row < rows && row0 + row < n;
    float m = -kInf, s = 0.f;
    const auto join = [&](float2 p) { join_stats(m, s, p.x, p.y); };
    if (live) {
        for (int p = seg; p < pieces; p += 32) {
            float2 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                v[u] = p + 8 * u < pieces ? part[(p + 8 * u) * cap + row] : make_float2(-kInf, 0.f);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                join(v[u]);
            }
        }
    }
    sh[seg][r] = make_float2(m, s);
    __syncthreads();
    if (seg == 0 && live) {
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            join(sh[i][r]);
        }
        const int t = perm[row0 + row];
        row_loss(m, s, ref_off(m), lab_logit[row0 + row], loss[t], lse[t]);
    }
}

// dx rows: the slabs of a labelled token's row added in order, scaled and rounded; zeros for the
// others. A warp a row, eight channels a lane.
template <typename T>
__global__ void __launch_bounds__(256)
    xent_dx_kernel(const float* acc, long long slab, int splits, const int* perm, const int* count,
                   const float* inv, T* dx, int rows, int C) {
    wait_before();
    const int n = *count, lane = threadIdx.x & 31;
    const float by = *inv;
    for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < rows;
         i += (long long)gridDim.x * 8) {
        T* dst = dx + (long long)perm[i] * C;
        for (int c = lane * 8; c < C; c += 256) {
            float s[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                s[k] = 0.f;
            }
            if (i < n) {
                load_vec<float, 8>(acc + i * C + c, s);
                for (int p = 1; p < splits; ++p) {
                    float v[8];
                    load_vec<float, 8>(acc + p * slab + i * C + c, v);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        s[k] += v[k];
                    }
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    s[k] *= by;
                }
            }
            store_vec<T, 8>(dst + c, s);
        }
    }
}

// dw of a piece from its slabs, eight channels a thread
template <typename T>
__global__ void __launch_bounds__(256)
    xent_dw_kernel(const float* acc, long long slab, int splits, const float* inv, T* dw,
                   long long total8) {
    wait_before();
    begin_next();
    const float by = *inv;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total8;
         i += (long long)gridDim.x * 256) {
        float s[8];
        load_vec<float, 8>(acc + i * 8, s);
        for (int p = 1; p < splits; ++p) {
            float v[8];
            load_vec<float, 8>(acc + p * slab + i * 8, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                s[k] += v[k];
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            s[k] *= by;
        }
        store_vec<T, 8>(dw + i * 8, s);
    }
}

constexpr int kBiasChunks = 256;  // at most

// column sums of a piece of g: a block 256 columns of one of gridDim.y row ranges
template <typename T>
__global__ void __launch_bounds__(256)
    xent_colsum_kernel(const T* g, const int* count, int vp, int limit, float* part) {
    wait_before();
    begin_next();
    __shared__ float sh[8][256];
    const int n = *count;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int col = blockIdx.x * 256 + lane * 8;
    const int r0 = (int)((long long)n * blockIdx.y / gridDim.y);
    const int r1 = (int)((long long)n * (blockIdx.y + 1) / gridDim.y);
    float s[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        s[k] = 0.f;
    }
    if (col < limit) {  // g holds whole 64-column boxes up to the limit
        for (int r = r0 + w; r < r1; r += 32) {
            float v[4][8];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (r + 8 * u < r1) {
                    load_vec<T, 8>(g + (long long)(r + 8 * u) * vp + col, v[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (r + 8 * u < r1) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        s[k] += v[u][k];
                    }
                }
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        sh[w][lane * 8 + k] = s[k];
    }
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        t += sh[i][threadIdx.x];
    }
    part[(long long)blockIdx.y * vp + blockIdx.x * 256 + threadIdx.x] = t;
}

// the ranges' sums in order: 32 columns a block, eight threads a column
template <typename T>
__global__ void __launch_bounds__(256)
    xent_dbias_kernel(const float* part, int chunks, int vp, int limit, const float* inv,
                      T* dbias) {
    wait_before();
    begin_next();
    __shared__ float sh[8][32];
    const int lane = threadIdx.x & 31, seg = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (c < limit) {
#pragma unroll 8
        for (int i = seg; i < chunks; i += 8) {
            s += part[(long long)i * vp + c];
        }
    }
    sh[seg][lane] = s;
    __syncthreads();
    if (seg == 0 && c < limit) {
#pragma unroll
        for (int k = 1; k < 8; ++k) {
            s += sh[k][lane];
        }
        dbias[c] = Elem<T>::from_f(s * *inv);
    }
}

// ------------------------------------------------------------------------------------------
// plans
// ------------------------------------------------------------------------------------------
size_t round256(size_t n) {
    return (n + 255) & ~size_t(255);
}

constexpr int64_t kMax = int64_t(1) << 31;
constexpr size_t kPartBytes = size_t(256) << 20;   // statistics pieces of one launch
// g of one piece of the classes. Pieces that stay in L2 do not pay for their launches and part-
// filled waves: T 8192, V 100003, C 2048 11.4 ms at 64 and 128 MB, 11.3 at 256, 11.1 at 512.
constexpr size_t kPieceBytes = size_t(512) << 20;
constexpr int kPairs = 74;

struct Plan {
    // few classes, or (forward) few tokens: xent_head.cu and xent_few.cu, whose workspace is all
    // they need
    bool head, few;
    int64_t tp;        // rows of the gathered tokens, whole tiles
    int64_t row_step;  // forward: rows a launch
    int64_t vp;        // classes a piece (backward), whole tiles
    int dx_splits, dw_splits;
    size_t counts, maxs, perm, lab, lse_c, dl_c, scalars, xc;
    size_t part, lab_logit;             // forward
    size_t g, dx_acc, dw_acc, db_part;  // backward
    size_t bytes;
};

// False where a size overflows what the kernels index.
bool make_plan(int64_t T, int64_t V, int64_t C, bool bwd, Plan& p) {
    if (T >= kMax - 1024 || V >= kMax - 1024 || C >= kMax - 1024) {
        return false;
    }
    int64_t mul = 0;
    if (__builtin_mul_overflow(T + 256, C * 64, &mul) || __builtin_mul_overflow(V, C * 64, &mul)) {
        return false;
    }
    // Both sides, in us (head kernels / the tiles below), forward and backward: T 589824, V 64,
    // C 128, nine tenths labelled 37 / 172 and 83 / 615; T 262144, V 23, C 256, 15 % labelled
    // 17 / 30 and 51 / 142, all 30 / 108 and 83 / 387; T 100000, V 128, C 128 16 / 46 and 37 / 151;
    // T 1000, V 64, C 128 8.1 / 12.7 and 14 / 38; T 50000, V 100, C 200 forward 14 / 32. Backward
    // that width (V above 64 with C above 128) does not fit the heads' shared memory and takes the
    // tiles: 95 to 110.
    p.head = xent_head_fits(V, C, bwd);
    if (p.head) {
        p.bytes = xent_head_workspace(T, V, C, bwd);
        return true;
    }
    // V 32000, C 1024, us (few / the tiles below): T 1 17 / 27, T 64 21 / 28; more tokens than one
    // MMA's columns would read the weights twice.
    p.few = !bwd && xent_few_fits(T);
    if (p.few) {
        p.bytes = xent_few_workspace();
        return true;
    }
    p.tp = (T + PM - 1) / PM * PM;
    const int64_t tiles_v = (V + PN - 1) / PN, tiles_c = (C + PN - 1) / PN, tiles_t = p.tp / PM;
    size_t at = 0;
    const auto take = [&](size_t n) {
        const size_t o = at;
        at += round256(n);
        return o;
    };
    const int64_t nb = (T + kPrepItems - 1) / kPrepItems;
    p.counts = take(nb * 4);
    p.maxs = take(nb * 4);
    p.perm = take(T * 4);
    p.lab = take(T * 4);
    p.scalars = take(256);
    p.xc = take((size_t)p.tp * C * 2);
    if (!bwd) {
        const int64_t row_bytes = tiles_v * 2 * 8;
        p.row_step = std::min<int64_t>(
            p.tp, std::max<int64_t>(PM, (int64_t)kPartBytes / row_bytes / PM * PM));
        p.part = take((size_t)p.row_step * row_bytes);
        p.lab_logit = take(p.tp * 4);
    } else {
        p.lse_c = take(T * 4);
        p.dl_c = take(T * 4);
        // pieces of equal size, whole tiles, each at most kPieceBytes of g
        const int64_t most = std::max<int64_t>(1, (int64_t)kPieceBytes / (p.tp * 2) / PN);
        const int64_t pieces = (tiles_v + most - 1) / most;
        p.vp = (tiles_v + pieces - 1) / pieces * PN;
        const int64_t tiles_p = p.vp / PN;
        // K in as many ranges as cost least: waves of tiles over the pairs, 0.4 us a 64-deep stage
        // (a 256 x 256 tile under load), against the float32 slabs, written and read once at
        // 6 TB/s; ranges of at least 8 stages. `direct`: one range needs no slab.
        const auto splits = [](int64_t tiles, int64_t k, double slab_bytes, bool direct) {
            const int64_t stages = (k + PK - 1) / PK;
            int best = 1;
            double least = 0;
            for (int s = 1; s <= 64 && (s == 1 || stages / s >= 8); ++s) {
                const double waves = (double)((tiles * s + kPairs - 1) / kPairs);
                const double cost = waves * (double)((stages + s - 1) / s) * 0.4 +
                                    (s == 1 && direct ? 0 : 2 * s * slab_bytes / 6e6);
                if (s == 1 || cost < 0.98 * least) {
                    best = s;
                    least = cost;
                }
            }
            return best;
        };
        p.dx_splits = splits(tiles_t * tiles_c, p.vp, 4.0 * p.tp * C, false);
        p.dw_splits = splits(tiles_p * tiles_c, T, 4.0 * p.vp * C, true);
        p.g = take((size_t)p.tp * p.vp * 2);
        p.dx_acc = take((size_t)p.dx_splits * p.tp * C * 4);
        p.dw_acc = p.dw_splits > 1 ? take((size_t)p.dw_splits * p.vp * C * 4) : 0;
        p.db_part = take((size_t)kBiasChunks * p.vp * 4);
    }
    p.bytes = at;
    return true;
}

template <typename T, int KIND>
cudaError_t launch_gemm(cudaStream_t s, const CUtensorMap& ta, const CUtensorMap& tb,
                        const CUtensorMap& to, const GemmArgs& a, int64_t items) {
    auto kern = xent_gemm_kernel<T, KIND>;
    // the pairs that fit the device at once, found once a device
    static int pairs[kMaxDevices] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) {
        return e;
    }
    if (dev >= kMaxDevices || pairs[dev] == 0) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
        if (e != cudaSuccess) {
            return e;
        }
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * kPairs);
        cfg.blockDim = dim3(gemm_threads(KIND));
        cfg.dynamicSmemBytes = kSmemBytes;
        int fit = 0;
        e = cudaOccupancyMaxActiveClusters(&fit, kern, &cfg);
        if (e != cudaSuccess) {
            return e;
        }
        fit = std::max(1, std::min(fit, kPairs));
        if (dev >= kMaxDevices) {
            return launch_behind(kern, 2 * (unsigned)std::min<int64_t>(items, fit),
                                 gemm_threads(KIND), kSmemBytes, s, ta, tb, to, a);
        }
        pairs[dev] = fit;
    }
    const unsigned grid = 2 * (unsigned)std::max<int64_t>(1, std::min<int64_t>(items, pairs[dev]));
    return launch_behind(kern, grid, gemm_threads(KIND), kSmemBytes, s, ta, tb, to, a);
}

// a row-major [rows][cols] matrix in boxes of box_cols x box_rows (128-byte rows)
bool map2(CUtensorMap* m, CUtensorMapDataType t, int es, const void* p, int64_t rows, int64_t cols,
          uint32_t box_rows) {
    const uint64_t d[2] = {(uint64_t)cols, (uint64_t)rows}, st[1] = {(uint64_t)cols};
    const uint32_t box[2] = {(uint32_t)(128 / es), box_rows};
    return encode_tiled(m, t, es, 2, p, d, st, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

bool map3(CUtensorMap* m, const void* p, int64_t slabs, int64_t rows, int64_t cols) {
    const uint64_t d[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)slabs};
    const uint64_t st[2] = {(uint64_t)cols, (uint64_t)(cols * rows)};
    const uint32_t box[3] = {32, 128, 1};
    return encode_tiled(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, 3, p, d, st, box,
                        CU_TENSOR_MAP_SWIZZLE_128B);
}

uint8_t* ws_of(const HeadCall& c) {
    return static_cast<uint8_t*>(c.workspace);
}

// label compaction and the gather of x
cudaError_t prepare(const HeadCall& c, const Plan& p) {
    const int64_t nb = (c.T + kPrepItems - 1) / kPrepItems;
    PrepArgs a{};
    a.dloss = c.dloss;
    a.lse = c.lse_in;
    a.loss = c.loss;
    a.lse_out = c.lse;
    a.counts = reinterpret_cast<int*>(ws_of(c) + p.counts);
    a.maxs = reinterpret_cast<float*>(ws_of(c) + p.maxs);
    a.T = (int)c.T;
    a.nblocks = (int)nb;
    a.V = c.V;
    a.perm = reinterpret_cast<int*>(ws_of(c) + p.perm);
    a.lab = reinterpret_cast<int*>(ws_of(c) + p.lab);
    a.lse_c = reinterpret_cast<float*>(ws_of(c) + p.lse_c);
    a.dl_c = reinterpret_cast<float*>(ws_of(c) + p.dl_c);
    a.count = reinterpret_cast<int*>(ws_of(c) + p.scalars);
    a.inv = reinterpret_cast<float*>(ws_of(c) + p.scalars + 4);
    int* counts = reinterpret_cast<int*>(ws_of(c) + p.counts);
    float* maxs = reinterpret_cast<float*>(ws_of(c) + p.maxs);
    const auto run = [&](auto tag) {
        using L = decltype(tag);
        const L* labels = static_cast<const L*>(c.labels);
        if (nb > 1) {
            xent_count_kernel<L><<<(unsigned)nb, kPrepThreads, 0, c.stream>>>(
                labels, c.dloss, (int)c.T, c.V, counts, maxs);
        }
        if (nb > 1) {
            launch_behind(xent_compact_kernel<L>, (unsigned)nb, kPrepThreads, 0, c.stream, labels,
                          a);
        } else {
            xent_compact_kernel<L><<<1, kPrepThreads, 0, c.stream>>>(labels, a);
        }
    };
    if (c.labels_64) {
        run((long long)0);
    } else {
        run(0);
    }
    const unsigned grid = (unsigned)std::min<int64_t>((c.T + 63 + 7) / 8, 148 * 8);
    launch_behind(xent_gather_kernel, grid, 256, 0, c.stream, static_cast<const uint4*>(c.x),
                  a.perm, a.count, reinterpret_cast<uint4*>(ws_of(c) + p.xc), (int)(c.C / 8));
    return cudaGetLastError();
}

template <typename T>
cudaError_t forward(const HeadCall& c, const Plan& p, bool& map_ok) {
    const CUtensorMapDataType t =
        c.dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap tx, tw;
    map_ok = map2(&tx, t, 2, ws_of(c) + p.xc, p.tp, c.C, 128) && map2(&tw, t, 2, c.w, c.V, c.C, 128);
    if (!map_ok) {
        return cudaSuccess;
    }
    cudaError_t e = prepare(c, p);
    GemmArgs a{};
    a.count = reinterpret_cast<int*>(ws_of(c) + p.scalars);
    a.V = (int)c.V;
    a.C = (int)c.C;
    a.vp = (int)((c.V + PN - 1) / PN * PN);
    a.splits = 1;
    a.cap = p.row_step;
    a.lab = reinterpret_cast<int*>(ws_of(c) + p.lab);
    a.bias = c.bias;
    a.part = reinterpret_cast<float2*>(ws_of(c) + p.part);
    a.lab_logit = reinterpret_cast<float*>(ws_of(c) + p.lab_logit);
    for (int64_t r0 = 0; e == cudaSuccess && r0 < c.T; r0 += p.row_step) {
        a.row0 = (int)r0;
        a.rows = (int)std::min(p.row_step, c.T - r0);
        const int64_t items = (int64_t)((a.rows + PM - 1) / PM) * (a.vp / PN);
        e = launch_gemm<T, kStats>(c.stream, tx, tw, tw, a, items);
        if (e == cudaSuccess) {
            launch_behind(xent_join_kernel, (a.rows + 31) / 32, 256, 0, c.stream, a.part,
                          a.lab_logit, reinterpret_cast<int*>(ws_of(c) + p.perm), a.count, a.row0,
                          a.rows, a.cap, 2 * (a.vp / PN), c.loss, c.lse);
            e = cudaGetLastError();
        }
    }
    return e;
}

template <typename T>
cudaError_t backward(const HeadCall& c, const Plan& p, bool& map_ok) {
    const CUtensorMapDataType t =
        c.dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    T* g = reinterpret_cast<T*>(ws_of(c) + p.g);
    float* dx_acc = reinterpret_cast<float*>(ws_of(c) + p.dx_acc);
    float* dw_acc = reinterpret_cast<float*>(ws_of(c) + p.dw_acc);
    float* db_part = reinterpret_cast<float*>(ws_of(c) + p.db_part);
    const float* inv = reinterpret_cast<float*>(ws_of(c) + p.scalars + 4);
    // K-major operands in boxes of 128 rows, MN-major ones in boxes of 64 K rows
    CUtensorMap x_k, w_k, g_k, x_n, w_n, g_m, g_out, dx_out, dw_out;
    map_ok = map2(&x_k, t, 2, ws_of(c) + p.xc, p.tp, c.C, 128) &&
             map2(&w_k, t, 2, c.w, c.V, c.C, 128) && map2(&g_k, t, 2, g, p.tp, p.vp, 128) &&
             map2(&x_n, t, 2, ws_of(c) + p.xc, p.tp, c.C, 64) && map2(&w_n, t, 2, c.w, c.V, c.C, 64) &&
             map2(&g_m, t, 2, g, p.tp, p.vp, 64) && map3(&dx_out, dx_acc, p.dx_splits, p.tp, c.C) &&
             (p.dw_splits > 1 ? map3(&dw_out, dw_acc, p.dw_splits, p.vp, c.C)
                              : map2(&dw_out, t, 2, c.dw, c.V, c.C, 128));
    if (!map_ok) {
        return cudaSuccess;
    }
    g_out = g_k;
    cudaError_t e = prepare(c, p);
    GemmArgs a{};
    a.count = reinterpret_cast<int*>(ws_of(c) + p.scalars);
    a.V = (int)c.V;
    a.C = (int)c.C;
    a.vp = (int)p.vp;
    a.lab = reinterpret_cast<int*>(ws_of(c) + p.lab);
    a.bias = c.bias;
    a.lse_c = reinterpret_cast<float*>(ws_of(c) + p.lse_c);
    a.dl_c = reinterpret_cast<float*>(ws_of(c) + p.dl_c);
    a.inv = inv;
    const int64_t tiles_t = p.tp / PM, tiles_c = (c.C + PN - 1) / PN;
    for (int64_t v0 = 0; e == cudaSuccess && v0 < c.V; v0 += p.vp) {
        a.v0 = (int)v0;
        const int64_t classes = std::min(p.vp, c.V - v0);
        const int64_t tiles_p = (classes + PN - 1) / PN;
        a.splits = 1;
        e = launch_gemm<T, kGrad>(c.stream, x_k, w_k, g_out, a, tiles_t * tiles_p);
        if (e == cudaSuccess && c.dbias != nullptr) {
            // eight blocks an SM, of at least 64 rows
            const int chunks = (int)std::max<int64_t>(
                1, std::min<int64_t>({kBiasChunks, 8 * 2 * kPairs / tiles_p, c.T / 64}));
            launch_behind(xent_colsum_kernel<T>, dim3((unsigned)tiles_p, chunks), 256, 0, c.stream,
                          g, a.count, a.vp, (int)classes, db_part);
            launch_behind(xent_dbias_kernel<T>, (unsigned)((classes + 31) / 32), 256, 0, c.stream,
                          db_part, chunks, a.vp, (int)classes, inv, static_cast<T*>(c.dbias) + v0);
            e = cudaGetLastError();
        }
        if (e == cudaSuccess) {
            a.splits = p.dx_splits;
            a.accumulate = v0 > 0;
            e = launch_gemm<T, kDx>(c.stream, g_k, w_n, dx_out, a, tiles_t * tiles_c * a.splits);
        }
        if (e == cudaSuccess) {
            a.splits = p.dw_splits;
            const int64_t items = tiles_p * tiles_c * a.splits;
            if (p.dw_splits == 1) {
                e = launch_gemm<T, kDw>(c.stream, g_m, x_n, dw_out, a, items);
            } else {
                e = launch_gemm<T, kDwSlab>(c.stream, g_m, x_n, dw_out, a, items);
                if (e == cudaSuccess) {
                    const int64_t total8 = classes * c.C / 8;
                    launch_behind(xent_dw_kernel<T>,
                                  (unsigned)std::min<int64_t>((total8 + 255) / 256, 148 * 8), 256,
                                  0, c.stream, dw_acc, p.vp * c.C, a.splits, inv,
                                  static_cast<T*>(c.dw) + v0 * c.C, total8);
                    e = cudaGetLastError();
                }
            }
        }
    }
    if (e == cudaSuccess) {
        launch_behind(xent_dx_kernel<T>, (unsigned)std::min<int64_t>((c.T + 7) / 8, 148 * 8), 256,
                      0, c.stream, dx_acc, p.tp * c.C, p.dx_splits,
                      reinterpret_cast<int*>(ws_of(c) + p.perm), a.count, inv,
                      static_cast<T*>(c.dx), (int)c.T, (int)c.C);
        e = cudaGetLastError();
    }
    return e;
}

int check(const char* who, int dtype, int labels_64, int64_t T, int64_t V, int64_t C) {
    const auto bad = [&](const char* what) {
        return fail(kInvalidArgument, std::string(who) + ": " + what);
    };
    if (dtype != kF16 && dtype != kBF16) {
        return bad("dtype must be f16 or bf16");
    }
    if (labels_64 != 0 && labels_64 != 1) {
        return bad("labels are int32 (labels_64 0) or int64 (1)");
    }
    if (T < 0 || V < 1 || C < 8 || C % 8 != 0) {
        return bad("T non-negative, V at least 1, C a positive multiple of 8");
    }
    return kOk;
}

int workspace_size(const char* who, int64_t T, int64_t V, int64_t C, bool bwd, size_t* bytes) {
    const int rc = check(who, kBF16, 0, T, V, C);
    if (rc != kOk) {
        return rc;
    }
    if (bytes == nullptr) {
        return fail(kInvalidArgument, std::string(who) + ": null size");
    }
    *bytes = 0;
    Plan p{};
    if (T > 0) {
        if (!make_plan(T, V, C, bwd, p)) {
            return fail(kInvalidArgument, std::string(who) + ": sizes must be below 2^31");
        }
        *bytes = p.bytes;
    }
    return kOk;
}

int finish(const char* who, bool map_ok, cudaError_t e) {
    if (!map_ok) {
        return fail(kInvalidArgument, std::string(who) + ": TMA descriptor rejected");
    }
    if (e != cudaSuccess) {
        return fail(kInternal, std::string(who) + " launch: " + cudaGetErrorString(e));
    }
    return kOk;
}

int check_workspace(const char* who, const void* ws, size_t have, size_t need) {
    if ((ws == nullptr && need > 0) || have < need || reinterpret_cast<uintptr_t>(ws) % 256 != 0) {
        return fail(kInvalidArgument,
                    std::string(who) + ": workspace below the size function's or not 256-byte "
                                       "aligned");
    }
    return kOk;
}

}  // namespace

unsigned read_and_clear_status_xent() {
    unsigned v = 0, z = 0;
    cudaMemcpyFromSymbol(&v, g_status, sizeof(v));
    cudaMemcpyToSymbol(g_status, &z, sizeof(z));
    return v;
}

}  // namespace cflk

using namespace cflk;

extern "C" int cflk_linear_xent_workspace_size(int64_t T, int64_t V, int64_t C, size_t* bytes) {
    clear_error();
    return workspace_size("linear_xent", T, V, C, false, bytes);
}

extern "C" int cflk_linear_xent(void* stream, int dtype, int labels_64, const void* x,
                                const void* w, const void* bias, const void* labels, float* loss,
                                float* lse, int64_t T, int64_t V, int64_t C, void* workspace,
                                size_t ws_bytes) {
    clear_error();
    const char* who = "linear_xent";
    int rc = check(who, dtype, labels_64, T, V, C);
    if (rc != kOk || T == 0) {
        return rc;
    }
    if (x == nullptr || w == nullptr || labels == nullptr || loss == nullptr || lse == nullptr) {
        return fail(kInvalidArgument, "linear_xent: null buffer");
    }
    if (!aligned16(x) || !aligned16(w)) {
        return fail(kInvalidArgument, "linear_xent: x and w must be 16-byte aligned");
    }
    Plan p{};
    if (!make_plan(T, V, C, false, p)) {
        return fail(kInvalidArgument, "linear_xent: sizes must be below 2^31");
    }
    rc = check_workspace(who, workspace, ws_bytes, p.bytes);
    if (rc != kOk) {
        return rc;
    }
    HeadCall c{};
    c.stream = static_cast<cudaStream_t>(stream);
    c.dtype = dtype;
    c.labels_64 = labels_64;
    c.x = x;
    c.w = w;
    c.bias = bias;
    c.labels = labels;
    c.loss = loss;
    c.lse = lse;
    c.T = T;
    c.V = V;
    c.C = C;
    c.workspace = workspace;
    bool map_ok = true;
    const cudaError_t e = p.head           ? xent_head(c, false, map_ok)
                          : p.few          ? xent_few(c, map_ok)
                          : dtype == kBF16 ? forward<__nv_bfloat16>(c, p, map_ok)
                                           : forward<__half>(c, p, map_ok);
    return finish(who, map_ok, e);
}

extern "C" int cflk_linear_xent_bwd_workspace_size(int64_t T, int64_t V, int64_t C,
                                                   size_t* bytes) {
    clear_error();
    return workspace_size("linear_xent_bwd", T, V, C, true, bytes);
}

extern "C" int cflk_linear_xent_bwd(void* stream, int dtype, int labels_64, const void* x,
                                    const void* w, const void* bias, const void* labels,
                                    const float* lse, const float* dloss, void* dx, void* dw,
                                    void* dbias, int64_t T, int64_t V, int64_t C, void* workspace,
                                    size_t ws_bytes) {
    clear_error();
    const char* who = "linear_xent_bwd";
    int rc = check(who, dtype, labels_64, T, V, C);
    if (rc != kOk) {
        return rc;
    }
    if (dw == nullptr || (bias == nullptr) != (dbias == nullptr)) {
        return fail(kInvalidArgument, "linear_xent_bwd: null buffer (dbias goes with bias)");
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (T == 0) {
        cudaError_t e = cudaMemsetAsync(dw, 0, (size_t)V * (size_t)C * 2, s);
        if (e == cudaSuccess && dbias != nullptr) {
            e = cudaMemsetAsync(dbias, 0, (size_t)V * 2, s);
        }
        return finish(who, true, e);
    }
    if (x == nullptr || w == nullptr || labels == nullptr || lse == nullptr || dloss == nullptr ||
        dx == nullptr) {
        return fail(kInvalidArgument, "linear_xent_bwd: null buffer");
    }
    if (!aligned16(x) || !aligned16(w) || !aligned16(dx) || !aligned16(dw)) {
        return fail(kInvalidArgument,
                    "linear_xent_bwd: x, w, dx and dw must be 16-byte aligned");
    }
    Plan p{};
    if (!make_plan(T, V, C, true, p)) {
        return fail(kInvalidArgument, "linear_xent_bwd: sizes must be below 2^31");
    }
    rc = check_workspace(who, workspace, ws_bytes, p.bytes);
    if (rc != kOk) {
        return rc;
    }
    HeadCall c{};
    c.stream = s;
    c.dtype = dtype;
    c.labels_64 = labels_64;
    c.x = x;
    c.w = w;
    c.bias = bias;
    c.labels = labels;
    c.lse_in = lse;
    c.dloss = dloss;
    c.dx = dx;
    c.dw = dw;
    c.dbias = dbias;
    c.T = T;
    c.V = V;
    c.C = C;
    c.workspace = workspace;
    bool map_ok = true;
    const cudaError_t e = p.head           ? xent_head(c, true, map_ok)
                          : dtype == kBF16 ? backward<__nv_bfloat16>(c, p, map_ok)
                                           : backward<__half>(c, p, map_ok);
    return finish(who, map_ok, e);
}
