// Linear softmax cross entropy and its gradients for heads of few classes over many positions (a
// masked-MSA head's 23, a distance head's 64), where HBM bounds the work: x is read once and dx
// written once, nothing else of that size moves. What fits shared memory: forward V <= 128 and
// C <= 256; backward C <= 256 for V <= 64 and C <= 128 for V <= 128. Others take the general path.
//
//   forward, per 128 labelled tokens:  l = x w^T in tensor memory; a thread a row: lse, loss
//   backward:  l again, g = dloss (softmax - onehot) as 16-bit rows in shared memory; one
//     accumulator dx = g w, another, kept over all tiles of the CTA, dw += g^T x
//
//   * a persistent CTA an SM; it lists its labelled tokens in shared memory (blocks of 128 tokens
//     in turn over the CTAs) and works through them 128 at a time, so positions without a label
//     cost nothing but dx's zeros, which two warps send as bulk copies. Where most tokens carry a
//     label it takes whole blocks as tiles instead, x and dx as TMA boxes;
//   * w stays in shared memory in one layout that serves as the K-major B of the logits and the
//     N-major B of dx; a tile of x, gathered row by row by four warps' asynchronous copies, is the
//     K-major A of the logits, then the N-major B of dw; g is the K-major A of dx and the M-major
//     A of dw;
//   * four warpgroups work on two tiles (forward: four), each tile with its own tensor-memory
//     slot, so one's exponentials overlap the other's products and stores; each has a warp that
//     issues its MMAs, and dw's are issued in the order of the tiles;
//   * each CTA leaves a float32 dw (and dbias), a second kernel adds them in order: the same bits
//     every run.
//
// g is rounded to 16 bits as in the general path, and for the same reason; float16 scales dloss by
// a power of two first (by the CTA's largest, taken out of dx and dw in float32 before they round).
//
// 768 x 768 tokens, 64 classes, 128 channels, nine tenths labelled, f16: forward 41 us (151 MB
// read, 3.8 TB/s), backward 86 us (151 MB read, 151 written, 3.5 TB/s) and 5 for the sums of dw.
// 512 x 512 tokens, 23 classes, 256 channels, 15 % labelled, bf16: 20, 41 (20 MB read, 134
// written) and 5 us. Issue slots are 46 % (forward) and 56 % (backward) busy, the tensor pipe 13
// and 23 %: what bounds them is the chain from a tile's load over its logits to its exponentials
// in each of the tiles at work beside one another: four at most, however small V is, forward, and
// two backward.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <string>
#include <type_traits>

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

// four warpgroups of workers; a warp for each tile at work: the column sums of g (dbias), the MMAs;
// and four loading warps
constexpr int kThreads = 768;
constexpr int kSumWarp = 16, kMmaWarp = 18, kLoad0 = 20, kLoaders = 4;
constexpr int kFwdSlots = 4;  // of logits in tensor memory
constexpr int kRoundBlocks = 32;      // blocks of 128 tokens a CTA lists at a time
constexpr int kRound = kRoundBlocks * 128;
constexpr int kZeroRows = 8;          // rows of zeros in shared memory
// The eighths of labelled tokens from which on whole blocks are taken. 300000 tokens, 40 classes,
// gathered / whole blocks, two GPUs each: C 128 (four tiles fit) half labelled forward 17.8 and 23.9 /
// 18.0 us, backward 41.9 and 53.9 / 48; three quarters 22.0 / 18.0 and 50.7 / 47; C 256 (two) half
// forward 27.2 and 39.3 / 33.5, backward 70.5 and 89.2 / 95; three quarters 86.9 and 114.5 / 95.
__device__ __forceinline__ int dense_eighths(bool bwd, int nx) {
    return bwd && nx == 2 ? 5 : 4;
}
constexpr int kAtom = 128 * 128;      // 128 rows of 64 16-bit columns, 128-byte swizzle
constexpr int kDynamicMax = 227 * 1024 - 3072;  // beside the static shared memory
constexpr int kSms = 148;
constexpr unsigned long long kDrainLimitNs = 200000000ull;

struct Layout {
    int vp;       // rows of w in shared memory: 64 or 128
    int atoms;    // 64-column atoms of a row of x
    int nx;       // x tiles in flight (even: a warpgroup keeps its tiles)
    int off_x, off_g, off_list, off_zero, bytes;
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
    const int zero = bwd ? kZeroRows * (int)C * 2 : 0;
    const int rest = w + g + kRound * 4 + zero + 1024;  // alignment
    for (l.nx = 4; l.nx >= 2; l.nx -= 2) {
        if (rest + l.nx * x <= kDynamicMax) {
            l.off_x = w;
            l.off_g = l.off_x + l.nx * x;
            l.off_list = l.off_g + g;
            l.off_zero = l.off_list + kRound * 4;
            l.bytes = l.off_zero + zero + 1024;
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
    bool wide;           // dx rows in 32-byte accesses
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

// 32 bytes to a 32-byte boundary in one access
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]),
                 "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::
                     "l"(map),
                 "r"(src), "r"(c0), "r"(c1)
                 : "memory");
}

// `bytes` (a multiple of 16) from shared to global memory, both 16-byte aligned
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst),
                 "r"(src), "r"(bytes)
                 : "memory");
}

template <typename T, typename L, bool BWD>
__global__ void __launch_bounds__(kThreads, 1)
    head_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw,
                const __grid_constant__ CUtensorMap tdx, const __grid_constant__ HeadArgs a) {
    if constexpr (BWD) {
        begin_next();
    }
    using E = Elem<T>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t w_full, x_full[4], x_free[4], dx_ready[4], l_full[kFwdSlots], d_free[kFwdSlots],
        g_full[2], g_free[2], d_full[2], dw_done[2], drain;
    __shared__ uint32_t tmem_sh;
    __shared__ int abort_flag;
    __shared__ __align__(16) float bias_sh[128];
    __shared__ int block_count[kRoundBlocks + 1], block_list[kRoundBlocks], dense_sh, blocks_sh;
    __shared__ unsigned labelled[4 * kRoundBlocks];  // a bit a token of the round
    __shared__ float max_sh[kThreads / 32], db_sh[2][128];

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
    const int nmask = l.nx - 1, nshift = l.nx == 4 ? 2 : 1;  // tile g: buffer g & nmask
    const int blocks = (int)(((long long)a.T + 127) / 128);
    const int rounds = (blocks + kRoundBlocks * (int)gridDim.x - 1) / (kRoundBlocks * (int)gridDim.x);
    // token j of this CTA's block i of round rd
    const auto token = [&](int rd, int i, int j) -> long long {
        return (((long long)rd * kRoundBlocks + i) * gridDim.x + blockIdx.x) * 128 + j;
    };

    // the first round's labels on their way while the CTA sets itself up
    for (int i = warp; i < kRoundBlocks; i += kThreads / 32) {
        const long long t = token(0, i, 4 * lane);
        if (t < a.T) {
            asm volatile("prefetch.global.L2 [%0];" ::"l"(labels + t));
        }
    }
    if (warp == kMmaWarp) {
        if (lane == 0) {
            mbar_init(&w_full, 1);
            for (int i = 0; i < 4; ++i) {
                mbar_init(&x_full[i], 32 * kLoaders / l.nx);  // the loading warps' lanes
                mbar_init(&x_free[i], 1);
                // a worker warp arrives once: eight a tile (backward) or four
                mbar_init(&dx_ready[i], 8);
            }
            for (int i = 0; i < kFwdSlots; ++i) {
                mbar_init(&l_full[i], 1);
                mbar_init(&d_free[i], BWD ? 8 : 4);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(&g_full[i], 8);
                mbar_init(&g_free[i], 1);
                mbar_init(&d_full[i], 1);
                mbar_init(&dw_done[i], 1);
            }
            mbar_init(&drain, 2);
            abort_flag = 0;
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(&tmem_sh, 512);
        tmem_relinquish();
    }
    if constexpr (BWD) {
        for (int i = threadIdx.x; i < kZeroRows * a.C / 8; i += kThreads) {
            reinterpret_cast<uint4*>(smem + l.off_zero)[i] = make_uint4(0, 0, 0, 0);
        }
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
    // Tensor memory: two slots of 128 columns for dx and 256 columns for dw; where dw takes at most
    // 128 and the logits at most 64, the logits have columns of their own and run a tile ahead,
    // else they share the slot with dx.
    const bool ahead = BWD && cn <= 128 && l.vp == 64;
    const uint32_t dw_col = tmem + (ahead ? 384 : 256);
    const auto logits_col = [&](int slot) {
        return tmem + (ahead ? 256 + 64 * slot : 128 * slot);
    };

    if (warp == kSumWarp && lane == 0) {
        mbar_arrive_expect_tx(&w_full, l.atoms * l.vp * 128);
        for (int i = 0; i < l.atoms; ++i) {
            tma_load_2d(smem + i * l.vp * 128, &tw, &w_full, 64 * i, 0);
        }
    }

    int base = 0;             // tiles of earlier rounds
    int df = 0;               // dx chunks seen (workers) or drained (MMA)
    int stored = 0;           // loading warps: tiles of dx stored
    float db[4] = {0.f, 0.f, 0.f, 0.f};
    bool ok = true, w_ready = false;
#pragma unroll 1
    for (int rd = 0; rd < rounds; ++rd) {
        // list this round's labelled tokens in order
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
                if (BWD && lane == 0 && i < kRoundBlocks) {
                    labelled[4 * i + j] = ballots[k][j];
                }
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
            // the blocks with a labelled token, and whether whole blocks are worth taking
            const unsigned some = __ballot_sync(0xffffffffu, n > 0);
            if (n > 0) {
                block_list[__popc(some & ((1u << lane) - 1))] = lane;
            }
            const long long left = a.T - token(rd, lane, 0);
            const int in = warp_sum((int)min(128ll, max(0ll, left)));
            if (lane == 31) {
                block_count[32] = x;
                blocks_sh = __popc(some);
                dense_sh = 8 * x >= dense_eighths(BWD, l.nx) * in;
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
                } else if (!BWD && t < a.T) {
                    a.loss[t] = 0.f;
                    a.lse[t] = -kInf;
                }
                at += __popc(ballot);
            }
        }
        __syncthreads();
        const int count = block_count[kRoundBlocks];
        // Dense rounds take whole blocks of tokens as tiles, x and dx as TMA boxes, and rows without a
        // label as rows without a gradient; the others gather the labelled rows
        const bool dense = dense_sh != 0;
        const int n = dense ? blocks_sh : (count + 127) / 128;

        const auto arrive_warp = [&](uint64_t* bar) {
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(bar);
            }
        };
        if (warp >= kLoad0) {
            // Each tile buffer has its own one or two warps, so as many tiles are under way as
            // there are buffers. Gathered rows: 16 bytes a copy, 8, 16 or 32 lanes a row; the last
            // tile's missing rows repeat the last token (their g is zero).
            const int wpt = kLoaders / l.nx, b = (warp - kLoad0) / wpt;  // warps a tile, buffer
            const int part = (warp - kLoad0) % wpt, rows = 128 / wpt;
            const int lpr = cn <= 64 ? 8 : cn <= 128 ? 16 : 32, rpw = 32 / lpr;
            const int piece = lane & (lpr - 1), sub = lane / lpr;
            const bool on = piece * 8 < cn;
            const uint32_t bytes = piece * 8 < a.C ? 16 : 0;  // zeros up to the K step
            const T* x = static_cast<const T*>(a.x) + (bytes ? piece * 8 : 0);
            const uint32_t dst = smem_u32(xs + b * xbytes) + (piece >> 3) * kAtom;
            int staged = -1;  // dense backward: the tile whose dx this buffer will hold
            const auto store_dx = [&] {
                ok = mbar_wait(&dx_ready[b], stored & 1, &g_status, kStatusSyncWait, &abort_flag);
                ++stored;
                const int t0 = (int)token(rd, block_list[staged], 0);
#pragma unroll 1
                for (int i = 0; i < l.atoms; ++i) {
                    tma_store_2d(&tdx, smem_u32(xs + b * xbytes + i * kAtom), 64 * i, t0);
                }
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            };
            // tiles g = base + c with g % nx == b
#pragma unroll 1
            for (int c = (b - base) & nmask; c < n; c += l.nx) {
                const int g = base + c;
                if (dense) {
                    if (lane == 0) {
                        if (staged >= 0) {
                            store_dx();
                        } else {
                            ok = g < l.nx || mbar_wait(&x_free[b], ((g >> nshift) - 1) & 1, &g_status,
                                                       kStatusSyncWait, &abort_flag);
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
                    if (!ok) {
                        break;
                    }
                    // (every lane arrives: the barrier counts those of the gathering form)
                    if (lane == 0 && part == 0) {
                        staged = BWD ? c : -1;
                        const int t0 = (int)token(rd, block_list[c], 0);
                        mbar_arrive_expect_tx(&x_full[b], xbytes);
#pragma unroll 1
                        for (int i = 0; i < l.atoms; ++i) {
                            tma_load_2d(xs + b * xbytes + i * kAtom, &tx, &x_full[b], 64 * i, t0);
                        }
                    } else {
                        mbar_arrive(&x_full[b]);
                    }
                    continue;
                }
                if (lane == 0) {
                    ok = g < l.nx || mbar_wait(&x_free[b], ((g >> nshift) - 1) & 1, &g_status,
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
            if (staged >= 0 && ok) {
                store_dx();
            }
            __syncwarp();
        } else if (warp >= kMmaWarp && lane == 0) {
            // Descriptors' low words, made once: a step along an operand is an addition in 16-byte
            // units. K-major: a K step of 16 columns is 32 bytes, 64 columns an atom; MN-major: a K
            // step of 16 rows is 2 KB.
            const uint32_t id_l = idesc_f16(E::kBf16, 128, vn, false, false);
            const uint32_t w_k = desc_lo(smem_u32(smem), 16);
            const uint32_t w_n = desc_lo(smem_u32(smem), l.vp * 128);
            const uint32_t x_k0 = desc_lo(smem_u32(xs), 16), g_k0 = desc_lo(smem_u32(gs), 16);
            [[maybe_unused]] const uint32_t x_n0 = desc_lo(smem_u32(xs), kAtom);
            [[maybe_unused]] const uint32_t g_m0 = desc_lo(smem_u32(gs), kAtom);
            const uint32_t w_atom = l.vp * 8, x_tile = xbytes >> 4, g_tile = gbytes >> 4;
            constexpr uint32_t kAtom16 = kAtom >> 4;
            // K-major A (atoms kAtom apart) times B, ksteps steps of K; b_step and b_atom: B's
            // advance a step, and four
            const auto product = [&](uint32_t d, uint32_t da, uint32_t dbp, uint32_t b_step,
                                     uint32_t b_atom, uint32_t id, int ksteps) {
                int k = 0;
#pragma unroll 1
                for (; k + 4 <= ksteps; k += 4) {
                    mma_ss_k4(d, da, dbp, 2, b_step, id, k);
                    da += kAtom16;
                    dbp += b_atom;
                }
#pragma unroll 1
                for (; k < ksteps; ++k) {
                    mma_ss_lo(d, da, dbp, id, k);
                    da += 2;
                    dbp += b_step;
                }
            };
            const auto logits = [&](int c, int slot) {
                const int g = base + c, b = g & nmask;
                if (!w_ready) {
                    ok = ok && mbar_wait(&w_full, 0, &g_status, kStatusTmaWait, &abort_flag);
                    w_ready = true;
                }
                ok = ok && mbar_wait(&x_full[b], (g >> nshift) & 1, &g_status, kStatusTmaWait,
                                     &abort_flag);
                if (!ok) {
                    return;
                }
                tc_fence_after();
                product(logits_col(slot), x_k0 + b * x_tile, w_k, 2, w_atom, id_l, cn >> 4);
                if constexpr (!BWD) {
                    mma_commit(&x_free[b]);
                }
                mma_commit(&l_full[slot]);
            };
            const auto wait = [&](uint64_t* bar, int parity) {
                ok = ok && mbar_wait(bar, parity & 1, &g_status, kStatusSyncWait, &abort_flag);
                tc_fence_after();
            };
            if constexpr (!BWD) {
                // the two warps take the tiles in turn: one issues an MMA of these sizes in about 100
                // cycles, 1650 a tile
#pragma unroll 1
                for (int c = (base + warp - kMmaWarp) & 1; ok && c < n; c += 2) {
                    const int g = base + c;
                    if (g >= kFwdSlots) {
                        wait(&d_free[g % kFwdSlots], g / kFwdSlots - 1);
                    }
                    logits(c, g % kFwdSlots);
                }
            } else {
                // This warp's tiles are those of worker group h: the logits, dx's first 128 columns
                // and dw once g is written, dx's other columns as the slot is drained. The two
                // warps add to dw in turn, so that its sum is always the same one.
                const int h = warp - kMmaWarp;
                const uint32_t id_w = idesc_f16(E::kBf16, l.vp, cn, true, true);
#pragma unroll 1
                for (int c = (base + h) & 1; ok && c < n; c += 2) {
                    const int g = base + c;
                    const auto dx_chunk = [&](int ch) {
                        product(tmem + 128 * h, g_k0 + h * g_tile, w_n + 2 * ch * w_atom, 128, 512,
                                idesc_f16(E::kBf16, 128, min(128, cn - 128 * ch), false, true),
                                vn >> 4);
                        mma_commit(&d_full[h]);
                    };
                    if (!ahead || c < 2) {
                        logits(c, h);
                    }
                    wait(&g_full[h], g >> 1);
                    if (ahead && c >= 2) {
                        wait(&d_free[h], df++);
                    }
                    if (!ok) {
                        break;
                    }
                    dx_chunk(0);
                    if (g > 0) {
                        wait(&dw_done[h ^ 1], (g - 1) >> 1);
                        if (!ok) {
                            break;
                        }
                    }
                    const uint32_t dg = g_m0 + h * g_tile, dx = x_n0 + (g & nmask) * x_tile;
                    mma_ss_k4(dw_col, dg, dx, 128, 128, id_w, g);
                    mma_ss_k4(dw_col, dg + 512, dx + 512, 128, 128, id_w, 1);
                    mma_commit(&x_free[g & nmask]);
                    mma_commit(&dw_done[h]);
                    if (ahead) {
                        if (c + 2 < n) {
                            logits(c + 2, h);
                        } else {
                            wait(&d_free[h], df++);
                        }
                        continue;
                    }
#pragma unroll 1
                    for (int ch = 1; ok && ch <= nch; ++ch) {
                        wait(&d_free[h], df++);
                        if (ok && ch < nch) {
                            dx_chunk(ch);
                        }
                    }
                }
            }
        } else if (BWD && (warp == kSumWarp || warp == kSumWarp + 1)) {
            // zeros for the rows without a label (dense: of the blocks without one): a lane 32 tokens,
            // each run of them as bulk copies of up to kZeroRows zeroed rows (a copy a row is what
            // the copy engine then waits for: 114 MB in 31 us)
            for (int w = threadIdx.x - 32 * kSumWarp; w < 4 * kRoundBlocks; w += 64) {
                const int blk = w >> 2;
                const long long t0 = token(rd, blk, 32 * (w & 3));
                const long long left = a.T - t0;
                unsigned todo = left <= 0 ? 0 : left >= 32 ? 0xffffffffu : (1u << left) - 1;
                todo &= ~labelled[w];
                if (dense && block_count[blk + 1] != block_count[blk]) {
                    todo = 0;
                }
                while (todo != 0) {
                    const int first = __ffs(todo) - 1;
                    const unsigned rest = ~(todo >> first);  // a zero ends the run
                    const int run = min(rest == 0 ? 32 : __ffs(rest) - 1, kZeroRows);
                    bulk_store(static_cast<T*>(a.dx) + (t0 + first) * a.C,
                               smem_u32(smem + l.off_zero), run * a.C * 2);
                    todo &= ~(((1u << run) - 1) << first);
                }
            }
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            const int h = warp - kSumWarp;
            for (int c = (base + h) & 1; a.bias != nullptr && c < n; c += 2) {
                const int g = base + c;
                mbar_wait(&g_full[h], (g >> 1) & 1, &g_status, kStatusSyncWait, &abort_flag);
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    if (q * 64 >= vn) {
                        break;
                    }
                    const uint8_t* p = gs + h * gbytes + q * kAtom + (lane & 3) * 4;
                    float s0[2] = {0.f, 0.f}, s1[2] = {0.f, 0.f};
#pragma unroll 8
                    for (int row = 0; row < 128; ++row) {
                        const float2 w = E::unpack(*reinterpret_cast<const uint32_t*>(
                            p + row * 128 + (((lane >> 2) ^ (row & 7)) << 4)));
                        s0[row & 1] += w.x;
                        s1[row & 1] += w.y;
                    }
                    db[2 * q] += s0[0] + s0[1];
                    db[2 * q + 1] += s1[0] + s1[1];
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&g_free[h]);
                }
            }
        } else if (warp < kSumWarp) {
            // forward: a warpgroup a tile; backward: two, half of the columns each
            const int h = BWD ? (warp >> 2) & 1 : warp >> 2;
            [[maybe_unused]] const int half = warp >> 3;
            const int r = ((warp & 3) << 5) | lane;        // row of the tile, tensor-memory lane
            // a tile's row: its token, and what is loaded for it a tile ahead (without a branch round
            // a load: the loads' latency is a quarter of a tile's time)
            struct Row {
                long long tok;
                int lab;
                bool in;
                float lse2, dl;
            };
            const auto fetch = [&](int c, Row& row) {
                const long long at = dense ? token(rd, block_list[c], r)
                                           : (long long)list[min(c * 128 + r, count - 1)];
                row.tok = min(at, (long long)a.T - 1);
                row.in = dense ? at < a.T : c * 128 + r < count;
                row.lab = label_of(labels, row.tok, a.V);
                if constexpr (BWD) {
                    row.lse2 = a.lse_in[row.tok];
                    row.dl = a.dloss[row.tok];
                }
            };
            constexpr int kStep = BWD ? 2 : 4;
            int c = BWD ? (base + h) & 1 : (h - base) & 3;
            Row next = {};
            if (c < n) {
                fetch(c, next);
            }
#pragma unroll 1
            for (; c < n; c += kStep) {
                const int g = base + c;
                const int sl = BWD ? h : g % kFwdSlots, turn = BWD ? g >> 1 : g / kFwdSlots;
                const uint32_t slot = logits_col(sl) + tmem_lane_base(warp);
                [[maybe_unused]] const uint32_t dx_slot = tmem + 128 * sl + tmem_lane_base(warp);
                const long long tok = next.tok;
                const int lab = next.lab;
                const bool live = next.in && lab >= 0;
                [[maybe_unused]] GradRow grad;
                if constexpr (BWD) {
                    grad.lse2 = next.lse2;
                    grad.dl = next.dl * scale;
                    grad.label = lab;
                    if (!live || grad.lse2 == -kInf) {
                        grad.kill();
                    }
                }
                if (!BWD && c + kStep < n) {
                    fetch(c + kStep, next);
                }
                if constexpr (BWD) {
                    if (a.bias != nullptr && g >= 2) {
                        // dbias has been summed from this warpgroup's last g
                        mbar_wait(&g_free[h], ((g >> 1) - 1) & 1, &g_status, kStatusSyncWait,
                                  &abort_flag);
                    }
                }
                mbar_wait(&l_full[sl], turn & 1, &g_status, kStatusMmaWait, &abort_flag);
                tc_fence_after();
                if constexpr (!BWD) {
                    float m = -kInf, s = 0.f, at_label = 0.f;
#pragma unroll 1
                    for (int c0 = 0; c0 < a.V; c0 += 16) {
                        uint32_t v[16];
                        tmem_ld16(slot + c0, v);
                        tmem_wait_ld();
                        row_stats<16>(v, c0, a.V, lab, a.bias != nullptr ? bias_sh + c0 : nullptr,
                                      m, s, at_label);
                    }
                    tc_fence_before();
                    arrive_warp(&d_free[sl]);
                    if (live) {
                        row_loss(m, s, ref_off(m), at_label, a.loss[tok], a.lse[tok]);
                    }
                } else {
                    uint8_t* grow = gs + h * gbytes + r * 128;
                    const int b = g & nmask;
                    uint8_t* xrow = xs + b * xbytes + r * 128;
#pragma unroll 1
                    for (int c0 = 16 * half; c0 < vn; c0 += 32) {
                        uint32_t v[16];
                        tmem_ld16(slot + c0, v);
                        tmem_wait_ld();
                        if (dense && !live && c0 == 0 && !isfinite(__uint_as_float(v[0]))) {
                            // a row without a label may hold anything, and dw multiplies it by
                            // its zeros of g: NaN and infinities (which every logit shows) are
                            // cleared
#pragma unroll 1
                            for (int p = 0; p < 8 * l.atoms; ++p) {
                                *reinterpret_cast<uint4*>(
                                    xrow + (p >> 3) * kAtom + (((p & 7) ^ (r & 7)) << 4)) =
                                    make_uint4(0, 0, 0, 0);
                            }
                        }
                        float y[16];
                        row_grad<16>(v, y, c0, a.V, grad,
                                     a.bias != nullptr ? bias_sh + c0 : nullptr);
                        if (!live) {  // zeros, whatever the logits were: a product with 0 keeps NaN
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                y[j] = 0.f;
                            }
                        }
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            *reinterpret_cast<uint4*>(
                                grow + (c0 >> 6) * kAtom +
                                (((((c0 >> 3) & 7) + q) ^ (r & 7)) << 4)) =
                                make_uint4(E::pack(y[8 * q], y[8 * q + 1]),
                                           E::pack(y[8 * q + 2], y[8 * q + 3]),
                                           E::pack(y[8 * q + 4], y[8 * q + 5]),
                                           E::pack(y[8 * q + 6], y[8 * q + 7]));
                        }
                    }
                    fence_async_smem();
                    tc_fence_before();
                    arrive_warp(&g_full[h]);
                    if (c + kStep < n) {
                        fetch(c + kStep, next);
                    }
                    // dx. Dense: into the tile of x, which its products no longer read, for the loading
                    // warp to store. Gathered: a thread stores its row, whole 32-byte sectors where
                    // the rows allow it
                    T* out = static_cast<T*>(a.dx) + (long long)tok * a.C;
#pragma unroll 1
                    for (int ch = 0; ch < nch; ++ch) {
                        mbar_wait(&d_full[h], df & 1, &g_status, kStatusMmaWait, &abort_flag);
                        ++df;
                        tc_fence_after();
                        const int end = min(128, a.C - 128 * ch);
                        if (ch == 0) {
                            // dw has read g and x
                            mbar_wait(&dw_done[h], (g >> 1) & 1, &g_status, kStatusMmaWait,
                                      &abort_flag);
                        }
#pragma unroll 1
                        for (int c0 = 32 * half; c0 < end; c0 += 64) {
                            uint32_t v[32], o[16];
                            tmem_ld32(dx_slot + c0, v);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                o[i] = E::pack(__uint_as_float(v[2 * i]) * inv,
                                               __uint_as_float(v[2 * i + 1]) * inv);
                            }
                            const int col = 128 * ch + c0;
                            if (dense) {
                                uint8_t* p = xrow + (col >> 6) * kAtom;
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    *reinterpret_cast<uint4*>(
                                        p + (((((col >> 3) & 4) + q) ^ (r & 7)) << 4)) =
                                        live ? make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2],
                                                          o[4 * q + 3])
                                             : make_uint4(0, 0, 0, 0);
                                }
                            } else if (live) {
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    if (c0 + 8 * q >= end) {
                                        break;
                                    }
                                    if (!a.wide) {
                                        *reinterpret_cast<uint4*>(out + col + 8 * q) = make_uint4(
                                            o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
                                    } else if (q % 2 == 0) {
                                        store32(out + col + 8 * q, &o[4 * q]);
                                    }
                                }
                            }
                        }
                        tc_fence_before();
                        arrive_warp(&d_free[h]);
                    }
                    if (dense) {
                        fence_async_smem();
                        arrive_warp(&dx_ready[b]);
                    }
                }
            }
        }
        base += n;
        __syncwarp();
        __syncthreads();
    }
    // every copy has landed and every MMA is done before shared and tensor memory go
    if (warp == kSumWarp && lane == 0) {
        mbar_wait(&w_full, 0, &g_status, kStatusTmaWait, nullptr, kDrainLimitNs);
    }
    if (BWD && warp >= kSumWarp) {
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    if ((warp == kMmaWarp || warp == kMmaWarp + 1) && lane == 0) {
        mma_commit(&drain);
        mbar_wait(&drain, 0, &g_status, kStatusMmaWait, nullptr, kDrainLimitNs);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if constexpr (BWD) {
        if (warp < 8) {
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
        } else if ((warp == kSumWarp || warp == kSumWarp + 1) && a.bias != nullptr) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                db_sh[warp - kSumWarp][64 * (q >> 1) + 2 * lane + (q & 1)] = db[q];
            }
        }
        __syncthreads();
        if (a.bias != nullptr && (int)threadIdx.x < a.V) {
            a.db_part[(long long)blockIdx.x * a.V + threadIdx.x] =
                (db_sh[0][threadIdx.x] + db_sh[1][threadIdx.x]) * inv;
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// The CTAs' dw and dbias added in order: four values a thread, kSegs threads over the CTAs.
constexpr int kSegs = 16;

template <typename T>
__global__ void __launch_bounds__(32 * kSegs)
    head_reduce_kernel(const float* dw_part, const float* db_part, int ctas, int V, int C, T* dw,
                       T* dbias) {
    wait_before();
    __shared__ float4 sh[kSegs][32];
    const int r = threadIdx.x & 31, seg = threadIdx.x >> 5;
    const int total = V * C / 4;
    const int i = blockIdx.x * 32 + r;
    const int wblocks = (total + 31) / 32;
    if ((int)blockIdx.x < wblocks) {
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < total) {
#pragma unroll 10
            for (int c = seg; c < ctas; c += kSegs) {
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
            for (int k = 1; k < kSegs; ++k) {
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
            for (int c = seg; c < ctas; c += kSegs) {
                s += db_part[(long long)c * V + v];
            }
        }
        sh[seg][r].x = s;
        __syncthreads();
        if (seg == 0 && v < V) {
#pragma unroll
            for (int k = 1; k < kSegs; ++k) {
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
cudaError_t launch(const HeadCall& c, const CUtensorMap& tx, const CUtensorMap& tw,
                   const CUtensorMap& tdx, const HeadArgs& a) {
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
    kern<<<head_grid(c.T), kThreads, a.l.bytes, c.stream>>>(tx, tw, tdx, a);
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
    a.wide = c.C % 16 == 0 && reinterpret_cast<uintptr_t>(c.dx) % 32 == 0;
    const int grid = head_grid(c.T);
    a.dw_part = static_cast<float*>(c.workspace);
    a.db_part = a.dw_part + (size_t)grid * c.V * c.C;
    const CUtensorMapDataType t =
        c.dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap tx, tw, tdx;
    const uint64_t dims[2] = {(uint64_t)c.C, (uint64_t)c.T}, dw[2] = {(uint64_t)c.C, (uint64_t)c.V};
    const uint64_t st[1] = {(uint64_t)c.C};
    const uint32_t box[2] = {64, 128}, bw[2] = {64, (uint32_t)a.l.vp};
    map_ok = encode_tiled(&tx, t, 2, 2, c.x, dims, st, box, CU_TENSOR_MAP_SWIZZLE_128B) &&
             encode_tiled(&tw, t, 2, 2, c.w, dw, st, bw, CU_TENSOR_MAP_SWIZZLE_128B);
    tdx = tx;
    if (map_ok && bwd) {
        map_ok = encode_tiled(&tdx, t, 2, 2, c.dx, dims, st, box, CU_TENSOR_MAP_SWIZZLE_128B);
    }
    if (!map_ok) {
        return cudaSuccess;
    }
    const auto run = [&](auto tag) -> cudaError_t {
        using T = decltype(tag);
        if (!bwd) {
            return c.labels_64 ? launch<T, long long, false>(c, tx, tw, tdx, a)
                               : launch<T, int, false>(c, tx, tw, tdx, a);
        }
        cudaError_t e = c.labels_64 ? launch<T, long long, true>(c, tx, tw, tdx, a)
                                    : launch<T, int, true>(c, tx, tw, tdx, a);
        if (e == cudaSuccess) {
            const int blocks = (a.V * a.C / 4 + 31) / 32 + (c.bias != nullptr ? (a.V + 31) / 32 : 0);
            launch_behind(head_reduce_kernel<T>, blocks, 32 * kSegs, 0, c.stream, a.dw_part,
                          a.db_part, grid, a.V, a.C, static_cast<T*>(c.dw),
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
