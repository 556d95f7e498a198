// Linear softmax cross entropy and its gradients for heads of few classes over many positions (a
// masked-MSA head's 23, a distance head's 64), where HBM bounds the work: x is read once and dx
// written once, nothing else of that size moves.
//
//   forward, per 128 labelled tokens:  l = x w^T in tensor memory; a thread a row: lse, loss
//   backward:  l again, g = dloss (softmax - onehot) as 16-bit rows in shared memory; one
//     accumulator dx = g w, another, kept over all tiles of the CTA, dw += g^T x
//
//   * a persistent CTA an SM; it lists its labelled tokens in shared memory (blocks of 128 tokens
//     in turn over the CTAs) and works through them 128 at a time, so positions without a label
//     cost nothing but dx's zeros, which a warp sends as bulk copies;
//   * w stays in shared memory in one layout that serves as the K-major B of the logits and the
//     N-major B of dx; a tile of x, gathered row by row by four warps' asynchronous copies, is the K-major A of the logits, then the N-major B of dw, then the staging of dx, whose rows
//     leave in whole lines; g is the K-major A of dx and the M-major A of dw;
//   * two warpgroups take the tiles in turn, each with its own tensor-memory slot, so one's
//     exponentials overlap the other's products and stores; one warp issues all MMAs in a fixed
//     order;
//   * each CTA leaves a float32 dw (and dbias), a second kernel adds them in order: the same bits
//     every run.
//
// g is rounded to 16 bits as in the general path, and for the same reason; float16 scales dloss by a
// power of two first (by the CTA's largest, taken out of dx and dw in float32 before they round).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <string>
#include <type_traits>

#include "capi_internal.h"
#include "cflk_b200.h"
#include "sm100.cuh"
#include "tmap.h"
#include "vec_io.cuh"
#include "xent_common.cuh"

namespace cflk {
namespace {

__device__ unsigned g_status;

// two warpgroups of workers, then the zeroing, the MMA and four loading warps
constexpr int kThreads = 448;
constexpr int kZeroWarp = 8, kMmaWarp = 9, kLoad0 = 10, kLoaders = 4;
constexpr int kRoundBlocks = 32;      // blocks of 128 tokens a CTA lists at a time
constexpr int kRound = kRoundBlocks * 128;
constexpr int kAtom = 128 * 128;      // 128 rows of 64 16-bit columns, 128-byte swizzle
constexpr int kDynamicMax = 227 * 1024 - 2048;  // beside the static shared memory
constexpr int kSms = 148;
constexpr unsigned long long kDrainLimitNs = 200000000ull;

struct Layout {
    int vp;       // rows of w in shared memory: 64 or 128
    int atoms;    // 64-column atoms of a row of x
    int nx;       // x tiles in flight (even: a warpgroup keeps its tiles)
    int off_x, off_g, off_list, bytes;
};

// False where the tiles do not fit shared memory or dw does not fit tensor memory.
bool make_layout(int64_t V, int64_t C, bool bwd, Layout& l) {
    if (V > 128 || C > 256) {
        return false;
    }
    l.vp = V <= 64 ? 64 : 128;
    l.atoms = (int)((C + 63) / 64);
    const int w = l.atoms * l.vp * 128, x = l.atoms * kAtom;
    const int g = bwd ? 2 * (l.vp / 64) * kAtom : 0;
    const int rest = w + g + kRound * 4 + 1024;  // alignment
    for (l.nx = 4; l.nx >= 2; l.nx -= 2) {
        if (rest + l.nx * x <= kDynamicMax) {
            l.off_x = w;
            l.off_g = l.off_x + l.nx * x;
            l.off_list = l.off_g + g;
            l.bytes = l.off_list + kRound * 4 + 1024;
            return true;
        }
    }
    return false;
}

struct HeadArgs {
    const void* x;
    const void* labels;
    const void* bias;
    const float* dloss;  // backward, with lse_in
    const float* lse_in;
    float* loss;         // forward
    float* lse;
    void* dx;
    float* dw_part;      // [CTA][V][C]
    float* db_part;      // [CTA][V]
    int T, V, C;
    Layout l;
};

// 16 bytes from global to shared memory, zeros where `bytes` is 0
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void copy_wait_all() {
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// `bytes` (a multiple of 16) from shared to global memory, both 16-byte aligned
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst),
                 "r"(src), "r"(bytes)
                 : "memory");
}

// whether the phase with the given parity is complete
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

template <typename T, typename L, bool BWD>
__global__ void __launch_bounds__(kThreads, 1)
    head_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ HeadArgs a) {
    using E = Elem<T>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t w_full, x_full[4], x_free[4], l_full[2], g_full[2], d_full[2], d_free[2],
        drain;
    __shared__ uint32_t tmem_sh;
    __shared__ int abort_flag;
    __shared__ float bias_sh[128];
    __shared__ __align__(16) uint4 zero_sh[32];
    __shared__ int block_count[kRoundBlocks + 1];
    __shared__ float max_sh[kThreads / 32];

    const Layout& l = a.l;
    const L* labels = static_cast<const L*>(a.labels);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int xbytes = l.atoms * kAtom, gbytes = (l.vp / 64) * kAtom;
    uint8_t* xs = smem + l.off_x;
    uint8_t* gs = smem + l.off_g;
    int* list = reinterpret_cast<int*>(smem + l.off_list);
    const int vn = (a.V + 15) & ~15;   // logits columns, and K of dx
    const int cn = (a.C + 15) & ~15;   // dw columns
    const int nch = (a.C + 127) / 128; // dx goes through the slot 128 columns at a time
    const int blocks = (int)(((long long)a.T + 127) / 128);
    const int rounds = (blocks + kRoundBlocks * (int)gridDim.x - 1) / (kRoundBlocks * (int)gridDim.x);
    // token j of this CTA's block i of round rd
    const auto token = [&](int rd, int i, int j) -> long long {
        return (((long long)rd * kRoundBlocks + i) * gridDim.x + blockIdx.x) * 128 + j;
    };

    if (warp == kMmaWarp) {
        if (lane == 0) {
            mbar_init(&w_full, 1);
            for (int i = 0; i < 4; ++i) {
                mbar_init(&x_full[i], 32 * kLoaders / l.nx);  // the loading warps' lanes
                mbar_init(&x_free[i], BWD ? 128 : 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(&l_full[i], 1);
                mbar_init(&g_full[i], 128);
                mbar_init(&d_full[i], 1);
                mbar_init(&d_free[i], 128);
            }
            mbar_init(&drain, 1);
            abort_flag = 0;
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(&tmem_sh, 512);
        tmem_relinquish();
    }
    if (warp == kZeroWarp) {
        zero_sh[lane] = make_uint4(0, 0, 0, 0);
        fence_async_smem();
    }
    if (threadIdx.x < 128) {
        bias_sh[threadIdx.x] = a.bias != nullptr && (int)threadIdx.x < a.V
                                   ? E::to_f(static_cast<const T*>(a.bias)[threadIdx.x])
                                   : 0.f;
    }
    float scale = 1.f, inv = 1.f;
    if constexpr (BWD && std::is_same<T, __half>::value) {
        // the power of two for float16, over all of this CTA's labelled tokens
        float m = 0.f;
        for (int b = warp; b < rounds * kRoundBlocks; b += kThreads / 32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const long long t = token(0, b, 32 * j + lane);
                if (t < a.T && label_of(labels, t, a.V) >= 0) {
                    const float d = fabsf(a.dloss[t]);
                    m = d < kInf ? fmaxf(m, d) : m;
                }
            }
        }
        m = warp_max(m);
        if (lane == 0) {
            max_sh[warp] = m;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) {
            m = fmaxf(m, max_sh[w]);
        }
        scale = grad_scale(m);
        inv = 1.f / scale;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_sh;
    const uint32_t dw_col = tmem + 256;

    if (warp == kZeroWarp && lane == 0) {
        mbar_arrive_expect_tx(&w_full, l.atoms * l.vp * 128);
        for (int i = 0; i < l.atoms; ++i) {
            tma_load_2d(smem + i * l.vp * 128, &tw, &w_full, 64 * i, 0);
        }
    }

    int base = 0;             // tiles of earlier rounds
    int df = 0;               // workers: dx chunks seen
    int freed[2] = {0, 0};    // MMA: slots drained
    float db[4] = {0.f, 0.f, 0.f, 0.f};
    bool ok = true, w_ready = false;
    for (int rd = 0; rd < rounds; ++rd) {
        // list this round's tokens: the labelled ones in order from the front, the others from
        // the back
        constexpr int kMine = (kRoundBlocks * 32 + kThreads - 1) / kThreads;  // blocks a warp
        unsigned ballots[kMine][4];
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
            const int i = warp + k * (kThreads / 32);
            int n = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const long long t = i < kRoundBlocks ? token(rd, i, 32 * j + lane) : a.T;
                ballots[k][j] =
                    __ballot_sync(0xffffffffu, t < a.T && label_of(labels, t, a.V) >= 0);
                n += __popc(ballots[k][j]);
            }
            if (lane == 0 && i < kRoundBlocks) {
                block_count[i] = n;
            }
        }
        __syncthreads();
        if (warp == 0) {
            const int n = block_count[lane];
            int x = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, d);
                x += lane >= d ? y : 0;
            }
            __syncwarp();
            block_count[lane] = x - n;
            if (lane == 31) {
                block_count[32] = x;
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
            const int i = warp + k * (kThreads / 32);
            if (i >= kRoundBlocks) {
                break;
            }
            int at = block_count[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const long long t = token(rd, i, 32 * j + lane);
                const unsigned ballot = ballots[k][j];
                const int before = at + __popc(ballot & ((1u << lane) - 1));
                if ((ballot >> lane) & 1) {
                    list[before] = (int)t;
                } else {
                    // token 128 i + 32 j + lane of the round, `before` of them labelled
                    const bool in = t < a.T;
                    list[kRound - 1 - (128 * i + 32 * j + lane - before)] = in ? (int)t : -1;
                    if (!BWD && in) {
                        a.loss[t] = 0.f;
                        a.lse[t] = -kInf;
                    }
                }
                at += __popc(ballot);
            }
        }
        __syncthreads();
        const int count = block_count[kRoundBlocks];
        const int n = (count + 127) / 128;

        if (warp >= kLoad0) {
            // the labelled rows of x, 16 bytes a copy, 8, 16 or 32 lanes a row; the last tile's
            // missing rows repeat the last token (their g is zero). Each tile buffer has its
            // own one or two warps, so as many tiles are under way as there are buffers.
            const int wpt = kLoaders / l.nx, b = (warp - kLoad0) / wpt;  // warps a tile, buffer
            const int part = (warp - kLoad0) % wpt, rows = 128 / wpt;
            const int lpr = cn <= 64 ? 8 : cn <= 128 ? 16 : 32, rpw = 32 / lpr;
            const int piece = lane & (lpr - 1), sub = lane / lpr;
            const bool on = piece * 8 < cn;
            const uint32_t bytes = piece * 8 < a.C ? 16 : 0;  // zeros up to the K step
            const T* x = static_cast<const T*>(a.x) + (bytes ? piece * 8 : 0);
            const uint32_t dst = smem_u32(xs + b * xbytes) + (piece >> 3) * kAtom;
            // tiles g = base + c with g % nx == b
            for (int c = (b - base % l.nx + l.nx) % l.nx; c < n; c += l.nx) {
                const int g = base + c;
                if (lane == 0) {
                    ok = g < l.nx || mbar_wait(&x_free[b], (g / l.nx - 1) & 1, &g_status,
                                               kStatusSyncWait, &abort_flag);
                }
                ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
                if (!ok) {
                    break;
                }
                for (int i = part * rows + sub; i < (part + 1) * rows; i += 8 * rpw) {
                    int t[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        t[u] = list[min(c * 128 + i + u * rpw, count - 1)];
                    }
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const int row = i + u * rpw;
                        if (on) {
                            copy16(dst + row * 128 + (((piece & 7) ^ (row & 7)) << 4),
                                   x + (long long)t[u] * a.C, bytes);
                        }
                    }
                }
                copy_wait_all();
                fence_async_smem();
                mbar_arrive(&x_full[b]);
            }
        } else if (warp == kMmaWarp && lane == 0) {
            const uint32_t sw = smem_u32(smem);
            const uint32_t id_l = idesc_f16(E::kBf16, 128, vn, false, false);
            const auto k_major = [](uint32_t at) { return smem_desc(at, 16, 1024, kSwizzle128B); };
            const auto logits = [&](int c) {
                const int g = base + c, b = g % l.nx;
                if (!w_ready) {
                    ok = ok && mbar_wait(&w_full, 0, &g_status, kStatusTmaWait, &abort_flag);
                    w_ready = true;
                }
                ok = ok && mbar_wait(&x_full[b], (g / l.nx) & 1, &g_status, kStatusTmaWait,
                                     &abort_flag);
                if (!ok) {
                    return;
                }
                tc_fence_after();
                const uint32_t sx = smem_u32(xs + b * xbytes);
                for (int ks = 0; ks < cn / 16; ++ks) {
                    mma_ss(tmem + 128 * (g & 1), k_major(sx + (ks >> 2) * kAtom + 32 * (ks & 3)),
                           k_major(sw + (ks >> 2) * l.vp * 128 + 32 * (ks & 3)), id_l, ks > 0);
                }
                if constexpr (!BWD) {
                    mma_commit(&x_free[b]);
                }
                mma_commit(&l_full[g & 1]);
            };
            if constexpr (!BWD) {
                for (int c = 0; ok && c < n; ++c) {
                    const int g = base + c;
                    if (g >= 2) {
                        ok = mbar_wait(&d_free[g & 1], ((g >> 1) - 1) & 1, &g_status,
                                       kStatusSyncWait, &abort_flag);
                        tc_fence_after();
                    }
                    if (ok) {
                        logits(c);
                    }
                }
            } else {
                // dx's columns [128 ch, ...) of tile c into its slot
                const auto dx_chunk = [&](int c, int ch) {
                    const int g = base + c, cols = min(128, cn - 128 * ch);
                    const uint32_t id = idesc_f16(E::kBf16, 128, cols, false, true);
                    const uint32_t sg = smem_u32(gs + (g & 1) * gbytes);
                    for (int ks = 0; ks < vn / 16; ++ks) {
                        mma_ss(tmem + 128 * (g & 1),
                               k_major(sg + (ks >> 2) * kAtom + 32 * (ks & 3)),
                               smem_desc(sw + 2 * ch * l.vp * 128 + ks * 2048, l.vp * 128, 1024,
                                         kSwizzle128B),
                               id, ks > 0);
                    }
                };
                const uint32_t id_w = idesc_f16(E::kBf16, l.vp, cn, true, true);
                // Each warpgroup's tile goes through: logits (x has come) -> dx's first columns and
                // dw (g is written; tiles in order, so dw's sum is always the same one) -> dx's
                // other columns (the slot is drained) -> the tile after next. Whatever is ready
                // is issued.
                int tile[2] = {base & 1, 1 - (base & 1)}, stage[2] = {0, 0}, next_dw = 0;
                unsigned long long t0 = globaltimer();
                while (tile[0] < n || tile[1] < n) {
                    bool moved = false;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int c = tile[h], g = base + c;
                        if (c >= n) {
                            continue;
                        }
                        if (stage[h] == 0) {
                            if (mbar_test(&x_full[g % l.nx], (g / l.nx) & 1)) {
                                logits(c);
                                stage[h] = 1;
                                moved = true;
                            }
                        } else if (stage[h] == 1) {
                            if (next_dw == c && mbar_test(&g_full[h], (g >> 1) & 1)) {
                                tc_fence_after();
                                dx_chunk(c, 0);
                                const uint32_t sg = smem_u32(gs + h * gbytes);
                                const uint32_t sx = smem_u32(xs + (g % l.nx) * xbytes);
                                for (int ks = 0; ks < 8; ++ks) {
                                    mma_ss(dw_col,
                                           smem_desc(sg + ks * 2048, kAtom, 1024, kSwizzle128B),
                                           smem_desc(sx + ks * 2048, kAtom, 1024, kSwizzle128B),
                                           id_w, g > 0 || ks > 0);
                                }
                                mma_commit(&d_full[h]);  // also: x's and g's reads are done
                                ++next_dw;
                                stage[h] = 2;
                                moved = true;
                            }
                        } else if (mbar_test(&d_free[h], freed[h] & 1)) {
                            ++freed[h];
                            tc_fence_after();
                            const int ch = stage[h] - 1;
                            if (ch < nch) {
                                dx_chunk(c, ch);
                                mma_commit(&d_full[h]);
                                ++stage[h];
                            } else {
                                tile[h] += 2;
                                stage[h] = 0;
                            }
                            moved = true;
                        }
                    }
                    if (moved) {
                        t0 = globaltimer();
                    } else if (!ok || *(volatile int*)&abort_flag ||
                               globaltimer() - t0 > kWaitLimitNs) {
                        atomicOr(&g_status, kStatusSyncWait);
                        abort_flag = 1;
                        break;
                    }
                }
            }
        } else if (BWD && warp == kZeroWarp) {
            // zeros for the rows without a label: a bulk copy of a zeroed row each
            for (int i = lane; i < kRound - count; i += 32) {
                const int t = list[kRound - 1 - i];
                if (t >= 0) {
                    bulk_store(static_cast<T*>(a.dx) + (long long)t * a.C, smem_u32(zero_sh),
                               a.C * 2);
                }
            }
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        } else if (warp < kZeroWarp) {
            const int h = warp >> 2;                       // warpgroup
            const int r = ((warp & 3) << 5) | lane;        // row of the tile, tensor-memory lane
            const uint32_t slot = tmem + 128 * h + tmem_lane_base(warp);
            for (int c = (base + h) & 1; c < n; c += 2) {
                const int g = base + c, b = g % l.nx;
                const bool live = c * 128 + r < count;
                const int tok = list[min(c * 128 + r, count - 1)];
                const int lab = label_of(labels, tok, a.V);
                [[maybe_unused]] float lse2 = 0.f, dl = 0.f;
                if constexpr (BWD) {
                    lse2 = a.lse_in[tok];
                    dl = a.dloss[tok] * scale;
                }
                mbar_wait(&l_full[h], (g >> 1) & 1, &g_status, kStatusMmaWait, &abort_flag);
                tc_fence_after();
                if constexpr (!BWD) {
                    float m = -kInf, s = 0.f, at_label = 0.f;
                    for (int c0 = 0; c0 < a.V; c0 += 32) {
                        uint32_t v[32];
                        tmem_ld32(slot + c0, v);
                        tmem_wait_ld();
                        float y[32];
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            y[j] = __uint_as_float(v[j]) + bias_sh[c0 + j];
                        }
                        row_stats(y, c0, a.V, lab, m, s, at_label);
                    }
                    tc_fence_before();
                    mbar_arrive(&d_free[h]);
                    if (live) {
                        const bool none = m == -kInf && s == 0.f;
                        const float l2 = log2f(s);
                        a.lse[tok] = none ? -kInf : m + l2;
                        a.loss[tok] = none ? 0.f : kLn2 * (m + l2) - at_label;
                    }
                } else {
                    const bool dead = !live || lse2 == -kInf;
                    uint8_t* grow = gs + h * gbytes + r * 128;
                    for (int c0 = 0; c0 < vn; c0 += 32) {
                        uint32_t v[32];
                        tmem_ld32(slot + c0, v);
                        tmem_wait_ld();
                        float y[32];
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            y[j] = __uint_as_float(v[j]) + bias_sh[c0 + j];
                        }
                        row_grad(y, c0, a.V, lab, lse2, dl, dead);
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            *reinterpret_cast<uint4*>(
                                grow + (c0 >> 6) * kAtom +
                                (((((c0 >> 3) & 4) + q) ^ (r & 7)) << 4)) =
                                make_uint4(E::pack(y[8 * q], y[8 * q + 1]),
                                           E::pack(y[8 * q + 2], y[8 * q + 3]),
                                           E::pack(y[8 * q + 4], y[8 * q + 5]),
                                           E::pack(y[8 * q + 6], y[8 * q + 7]));
                        }
                    }
                    fence_async_smem();
                    tc_fence_before();
                    mbar_arrive(&g_full[h]);
                    if (a.bias != nullptr) {
                        // columns 2 lane, 2 lane + 1 of each atom over this warp's 32 rows
                        named_sync(1 + h, 128);
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            if (q * 64 >= vn) {
                                break;
                            }
                            const uint8_t* p = gs + h * gbytes + q * kAtom;
#pragma unroll 8
                            for (int i = 0; i < 32; ++i) {
                                const int row = 32 * (warp & 3) + i;
                                const float2 w = E::unpack(*reinterpret_cast<const uint32_t*>(
                                    p + row * 128 + (((lane >> 2) ^ (row & 7)) << 4) +
                                    (lane & 3) * 4));
                                db[2 * q] += w.x;
                                db[2 * q + 1] += w.y;
                            }
                        }
                    }
                    // dx into the tile of x, which its products no longer read
                    uint8_t* xrow = xs + b * xbytes + r * 128;
                    for (int ch = 0; ch < nch; ++ch) {
                        mbar_wait(&d_full[h], df & 1, &g_status, kStatusMmaWait, &abort_flag);
                        ++df;
                        tc_fence_after();
                        const int end = min(128, a.C - 128 * ch);
                        for (int c0 = 0; c0 < end; c0 += 32) {
                            uint32_t v[32];
                            tmem_ld32(slot + c0, v);
                            tmem_wait_ld();
                            const int col = 128 * ch + c0;
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                uint32_t o[4];
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    o[i] = E::pack(__uint_as_float(v[8 * q + 2 * i]) * inv,
                                                   __uint_as_float(v[8 * q + 2 * i + 1]) * inv);
                                }
                                *reinterpret_cast<uint4*>(
                                    xrow + (col >> 6) * kAtom +
                                    (((((col >> 3) & 4) + q) ^ (r & 7)) << 4)) =
                                    make_uint4(o[0], o[1], o[2], o[3]);
                            }
                        }
                        tc_fence_before();
                        mbar_arrive(&d_free[h]);
                    }
                    named_sync(1 + h, 128);
                    // whole rows out: 8, 16 or 32 lanes a row of up to 64, 128 or 256 columns
                    const int lpr = a.C <= 64 ? 8 : a.C <= 128 ? 16 : 32;
                    const int piece = lane & (lpr - 1), sub = lane / lpr, rpw = 32 / lpr;
                    for (int i = (warp & 3) * rpw + sub; i < 128; i += 4 * rpw) {
                        if (c * 128 + i < count && piece * 8 < a.C) {
                            const uint4 w = *reinterpret_cast<const uint4*>(
                                xs + b * xbytes + (piece >> 3) * kAtom + i * 128 +
                                (((piece & 7) ^ (i & 7)) << 4));
                            reinterpret_cast<uint4*>(static_cast<T*>(a.dx) +
                                                     (long long)list[c * 128 + i] * a.C)[piece] = w;
                        }
                    }
                    fence_async_smem();
                    mbar_arrive(&x_free[b]);
                }
            }
        }
        base += n;
        __syncwarp();
        __syncthreads();
    }
    // every copy has landed and every MMA is done before shared and tensor memory go
    if (warp == kZeroWarp && lane == 0) {
        mbar_wait(&w_full, 0, &g_status, kStatusTmaWait, nullptr, kDrainLimitNs);
    }
    if (BWD && warp == kZeroWarp) {
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    if (warp == kMmaWarp && lane == 0) {
        mma_commit(&drain);
        mbar_wait(&drain, 0, &g_status, kStatusMmaWait, nullptr, kDrainLimitNs);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if constexpr (BWD) {
        float* db_sh = reinterpret_cast<float*>(list);  // [warp of the workers][128]
        if (warp < kZeroWarp) {
            const int h = warp >> 2, w = warp & 3;
            // dw: lane = class; with 64 rows lanes 32 w + i (i < 16) hold class 16 w + i
            const int v = l.vp == 128 ? 32 * w + lane : 16 * w + lane;
            const bool mine = v < a.V && (l.vp == 128 || lane < 16);
            float* dst = a.dw_part + ((long long)blockIdx.x * a.V + v) * a.C;
            for (int c0 = 32 * h; c0 < a.C; c0 += 64) {
                uint32_t x[32];
                if (base > 0) {
                    tmem_ld32(dw_col + tmem_lane_base(warp) + c0, x);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        x[j] = 0;
                    }
                }
                if (mine) {
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        if (c0 + 4 * q < a.C) {
                            reinterpret_cast<float4*>(dst + c0)[q] = make_float4(
                                __uint_as_float(x[4 * q]) * inv, __uint_as_float(x[4 * q + 1]) * inv,
                                __uint_as_float(x[4 * q + 2]) * inv,
                                __uint_as_float(x[4 * q + 3]) * inv);
                        }
                    }
                }
            }
            if (a.bias != nullptr) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    db_sh[(4 * h + w) * 128 + 64 * (q >> 1) + 2 * lane + (q & 1)] = db[q];
                }
            }
        }
        __syncthreads();
        if (a.bias != nullptr && (int)threadIdx.x < a.V) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s += db_sh[i * 128 + threadIdx.x];
            }
            a.db_part[(long long)blockIdx.x * a.V + threadIdx.x] = s * inv;
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// The CTAs' dw and dbias added in order: four values a thread, eight threads over the CTAs.
template <typename T>
__global__ void __launch_bounds__(256)
    head_reduce_kernel(const float* __restrict__ dw_part, const float* __restrict__ db_part,
                       int ctas, int V, int C, T* __restrict__ dw, T* __restrict__ dbias) {
    __shared__ float4 sh[8][32];
    const int r = threadIdx.x & 31, seg = threadIdx.x >> 5;
    const int total = V * C / 4;
    const int i = blockIdx.x * 32 + r;
    const int wblocks = (total + 31) / 32;
    if ((int)blockIdx.x < wblocks) {
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < total) {
#pragma unroll 8
            for (int c = seg; c < ctas; c += 8) {
                const float4 v = reinterpret_cast<const float4*>(dw_part)[(long long)c * total + i];
                s.x += v.x;
                s.y += v.y;
                s.z += v.z;
                s.w += v.w;
            }
        }
        sh[seg][r] = s;
        __syncthreads();
        if (seg == 0 && i < total) {
#pragma unroll
            for (int k = 1; k < 8; ++k) {
                s.x += sh[k][r].x;
                s.y += sh[k][r].y;
                s.z += sh[k][r].z;
                s.w += sh[k][r].w;
            }
            const float o[4] = {s.x, s.y, s.z, s.w};
            store_vec<T, 4>(dw + 4ll * i, o);
        }
    } else {
        const int v = ((int)blockIdx.x - wblocks) * 32 + r;
        float s = 0.f;
        if (v < V) {
            for (int c = seg; c < ctas; c += 8) {
                s += db_part[(long long)c * V + v];
            }
        }
        sh[seg][r].x = s;
        __syncthreads();
        if (seg == 0 && v < V) {
#pragma unroll
            for (int k = 1; k < 8; ++k) {
                s += sh[k][r].x;
            }
            dbias[v] = Elem<T>::from_f(s);
        }
    }
}

int head_grid(int64_t T) {
    return (int)std::min<int64_t>(kSms, (T + 127) / 128);
}

template <typename T, typename L, bool BWD>
cudaError_t launch(const HeadCall& c, const CUtensorMap& tw, const HeadArgs& a) {
    auto kern = head_kernel<T, L, BWD>;
    static bool done[kMaxDevices] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) {
        return e;
    }
    if (dev >= kMaxDevices || !done[dev]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kDynamicMax);
        if (e != cudaSuccess) {
            return e;
        }
        if (dev < kMaxDevices) {
            done[dev] = true;
        }
    }
    kern<<<head_grid(c.T), kThreads, a.l.bytes, c.stream>>>(tw, a);
    return cudaGetLastError();
}

}  // namespace

bool xent_head_fits(int64_t V, int64_t C, bool bwd) {
    Layout l;
    return make_layout(V, C, bwd, l);
}

size_t xent_head_workspace(int64_t T, int64_t V, int64_t C, bool bwd) {
    return bwd ? (size_t)head_grid(T) * (size_t)(V * C + V) * sizeof(float) : 0;
}

cudaError_t xent_head(const HeadCall& c, bool bwd, bool& map_ok) {
    HeadArgs a{};
    make_layout(c.V, c.C, bwd, a.l);
    a.x = c.x;
    a.labels = c.labels;
    a.bias = c.bias;
    a.dloss = c.dloss;
    a.lse_in = c.lse_in;
    a.loss = c.loss;
    a.lse = c.lse;
    a.dx = c.dx;
    a.T = (int)c.T;
    a.V = (int)c.V;
    a.C = (int)c.C;
    const int grid = head_grid(c.T);
    a.dw_part = static_cast<float*>(c.workspace);
    a.db_part = a.dw_part + (size_t)grid * c.V * c.C;
    const CUtensorMapDataType t =
        c.dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap tw;
    const uint64_t dw[2] = {(uint64_t)c.C, (uint64_t)c.V}, st[1] = {(uint64_t)c.C};
    const uint32_t bw[2] = {64, (uint32_t)a.l.vp};
    map_ok = encode_tiled(&tw, t, 2, 2, c.w, dw, st, bw, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!map_ok) {
        return cudaSuccess;
    }
    const auto run = [&](auto tag) -> cudaError_t {
        using T = decltype(tag);
        if (!bwd) {
            return c.labels_64 ? launch<T, long long, false>(c, tw, a)
                               : launch<T, int, false>(c, tw, a);
        }
        cudaError_t e = c.labels_64 ? launch<T, long long, true>(c, tw, a)
                                    : launch<T, int, true>(c, tw, a);
        if (e == cudaSuccess) {
            const int blocks = (a.V * a.C / 4 + 31) / 32 + (c.bias != nullptr ? (a.V + 31) / 32 : 0);
            head_reduce_kernel<T><<<blocks, 256, 0, c.stream>>>(
                a.dw_part, a.db_part, grid, a.V, a.C, static_cast<T*>(c.dw),
                static_cast<T*>(c.dbias));
            e = cudaGetLastError();
        }
        return e;
    };
    return c.dtype == kBF16 ? run(__nv_bfloat16{}) : run(__half{});
}

unsigned read_and_clear_status_head() {
    unsigned v = 0, z = 0;
    cudaMemcpyFromSymbol(&v, g_status, sizeof(v));
    cudaMemcpyToSymbol(g_status, &z, sizeof(z));
    return v;
}

}  // namespace cflk
