// Embedding lookup with scaling and its gradient by sorted tokens.
//
//   forward   out[t] = scale * table[ids[t]]        (a row of zeros for an id outside [0, V))
//   backward  dtable[v] = scale * sum over t with ids[t] = v of dout[t], float32
//
// Both are bound by HBM: the forward by the T output rows, the backward by the T rows of dout and
// the V float32 rows it writes. The backward sorts (id, token) pairs by id (a stable radix sort:
// the tokens of one id stay in order), cuts the sorted list into equal chunks so that an id with
// many tokens is spread over many warps, and adds the chunks' partial sums in the order of the
// list. Tables of few rows sort in shared memory instead, each CTA its own tokens. No float atomics,
// the same bits every run; sums are float32 and round nowhere else.
//
// Measured: 589824 tokens, 65 rows, 128 channels, bf16: lookup 34 us (151 MB written, 4.4 TB/s;
// a plain fill reaches 3.9, a copy 6.5), gradient 41 us (151 MB read, 3.7 TB/s). 16384 tokens,
// 50001 rows, 1024 channels, f16: gradient 66 us, of which 205 MB of zeros and sums are about 50
// at the fill's rate; four launches of the sort are too short to fill the machine and carry
// most of the zeros.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <type_traits>

#include "capi_internal.h"
#include "cflk_b200.h"
#include "launch.cuh"
#include "sm100.cuh"
#include "vec_io.cuh"

namespace cflk {
namespace {

constexpr int kSms = 148;

// ------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------
constexpr int kFwdThreads = 256, kFwdUnroll = 4;

// A thread takes kFwdUnroll vectors of VEC channels a step (their loads all in flight before the
// first store). Rows and columns of its vectors advance by the constant stride's quotient and
// remainder, so the loop divides nothing. (Unsigned: a position plus a step may pass 2^31.)
template <typename TI, typename TO, typename Id, int VEC>
__global__ void __launch_bounds__(kFwdThreads)
    embed_kernel(const Id* __restrict__ ids, const TI* __restrict__ table, TO* __restrict__ out,
                 long long T, long long V, unsigned cv, float scale) {
    const long long stride = (long long)gridDim.x * kFwdThreads;
    const long long first = (long long)blockIdx.x * kFwdThreads + threadIdx.x;
    const long long drow = stride / cv;
    const unsigned dcol = (unsigned)(stride - drow * cv);
    long long row = first / cv;
    unsigned col = (unsigned)(first - row * cv);
    while (row < T) {
        long long r[kFwdUnroll], id[kFwdUnroll];
        unsigned c[kFwdUnroll];
#pragma unroll
        for (int u = 0; u < kFwdUnroll; ++u) {
            r[u] = row;
            c[u] = col;
            id[u] = (long long)ids[min(row, T - 1)];
            row += drow;
            col += dcol;
            if (col >= cv) {
                col -= cv;
                ++row;
            }
        }
        // no branch round a load: an id outside the table reads its row 0 and drops it
        float v[kFwdUnroll][VEC];
#pragma unroll
        for (int u = 0; u < kFwdUnroll; ++u) {
            const bool ok = id[u] >= 0 && id[u] < V;
            load_vec<TI, VEC>(table + ((ok ? id[u] : 0) * cv + c[u]) * VEC, v[u]);
        }
#pragma unroll
        for (int u = 0; u < kFwdUnroll; ++u) {
            const bool ok = id[u] >= 0 && id[u] < V;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                v[u][i] = ok ? v[u][i] * scale : 0.f;
            }
        }
#pragma unroll
        for (int u = 0; u < kFwdUnroll; ++u) {
            if (r[u] < T) {
                store_vec<TO, VEC>(out + (r[u] * cv + c[u]) * VEC, v[u]);
            }
        }
    }
}

template <typename TI, typename TO, typename Id>
cudaError_t launch_embed(cudaStream_t s, const void* ids, const void* table, void* out, int64_t T,
                         int64_t V, int64_t C, float scale) {
    // 16-byte accesses of the narrower type when the rows allow them, else one channel a thread
    constexpr int VEC = sizeof(TO) == 2 || sizeof(TI) == 2 ? 8 : 4;
    const bool vec = C % VEC == 0 && aligned16(table) && aligned16(out);
    const int64_t cv = vec ? C / VEC : C;
    const int64_t need = (T * cv + kFwdThreads * kFwdUnroll - 1) / (kFwdThreads * kFwdUnroll);
    const unsigned grid = (unsigned)std::min<int64_t>(need, 8 * kSms);
    if (vec) {
        embed_kernel<TI, TO, Id, VEC><<<grid, kFwdThreads, 0, s>>>(
            static_cast<const Id*>(ids), static_cast<const TI*>(table), static_cast<TO*>(out), T,
            V, (unsigned)cv, scale);
    } else {
        embed_kernel<TI, TO, Id, 1><<<grid, kFwdThreads, 0, s>>>(
            static_cast<const Id*>(ids), static_cast<const TI*>(table), static_cast<TO*>(out), T,
            V, (unsigned)cv, scale);
    }
    return cudaGetLastError();
}

// ------------------------------------------------------------------------------------------
// backward: stable radix sort of (id, token)
// ------------------------------------------------------------------------------------------
constexpr int kSortThreads = 256, kSortWarps = kSortThreads / 32, kSortRounds = 4;
constexpr int kSortItems = kSortThreads * kSortRounds;  // a block's consecutive pairs
constexpr int kMaxDigit = 9;                            // bits of a pass
constexpr int kFewBlocks = 32;                          // no scan kernel up to these

// An id outside [0, V) sorts as V, behind every row.
template <typename Id>
__device__ __forceinline__ unsigned sort_key(const Id* ids, long long t, unsigned V) {
    const long long id = (long long)ids[t];
    return id >= 0 && id < (long long)V ? (unsigned)id : V;
}

// Rows without a token get zeros. The first kernel of the sort marks the rows that have one; the
// kernels after it, whose own blocks leave most SMs idle, each carry blocks that write a share of
// the others.
struct ZeroShare {
    const uint8_t* present;   // a byte a row
    float* dtable;
    int row0, row1;           // rows of this launch, multiples of 32 (or V)
    int C, blocks;            // channels; blocks at the end of the grid
    int vec;
};

// `block` of s.blocks, `warps` warps a block: 32 rows a block a step, its warps in turn
__device__ __forceinline__ void zero_rows(const ZeroShare& s, int block, int warps) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // (a step past the last row may pass 2^31)
    for (long long r0 = (long long)s.row0 + block * 32; r0 < s.row1; r0 += s.blocks * 32) {
        for (int r = warp; r < min(32ll, s.row1 - r0); r += warps) {
            if (s.present[r0 + r] != 0) {
                continue;
            }
            float* dst = s.dtable + (r0 + r) * s.C;
            if (s.vec) {
                for (unsigned c = lane * 4; c < (unsigned)s.C; c += 128) {
                    *reinterpret_cast<float4*>(dst + c) = make_float4(0.f, 0.f, 0.f, 0.f);
                }
            } else {
                for (unsigned c = lane; c < (unsigned)s.C; c += 32) {
                    dst[c] = 0.f;
                }
            }
        }
    }
}

// Whether this is the block's first look at `key` (a hash table of twice the block's tokens, so a
// free place is always found): a frequent row is marked once a block, by a plain store of a byte
// (600000 tokens of 2000 rows: 150 us with an atomic a token on a bitmap, 61 us so).
constexpr int kSeen = 2 * kSortItems;
constexpr unsigned kUnseen = 0xffffffffu;
__device__ __forceinline__ bool first_of_block(unsigned* seen, unsigned key) {
    unsigned h = (key * 2654435761u) >> 16;
    while (true) {
        h &= kSeen - 1;
        const unsigned old = atomicCAS(&seen[h], kUnseen, key);
        if (old == kUnseen || old == key) {
            return old == kUnseen;
        }
        ++h;
    }
}

// counts[digit][block]
template <typename Key>
__global__ void __launch_bounds__(kSortThreads)
    sort_count_kernel(const Key* keys, int T, unsigned V, int shift, int bits, int* counts,
                      int nblocks, uint8_t* mark, const ZeroShare zero) {
    wait_before();
    begin_next();
    if ((int)blockIdx.x >= nblocks) {
        zero_rows(zero, blockIdx.x - nblocks, kSortWarps);
        return;
    }
    __shared__ int hist[1 << kMaxDigit];
    __shared__ unsigned seen[kSeen];
    const int bins = 1 << bits;
    for (int i = threadIdx.x; mark != nullptr && i < kSeen; i += kSortThreads) {
        seen[i] = kUnseen;
    }
    for (int i = threadIdx.x; i < bins; i += kSortThreads) {
        hist[i] = 0;
    }
    __syncthreads();
    unsigned key[kSortRounds];
#pragma unroll
    for (int j = 0; j < kSortRounds; ++j) {
        const long long t = (long long)blockIdx.x * kSortItems + j * kSortThreads + threadIdx.x;
        key[j] = sort_key(keys, min(t, (long long)T - 1), V);
    }
#pragma unroll
    for (int j = 0; j < kSortRounds; ++j) {
        const long long t = (long long)blockIdx.x * kSortItems + j * kSortThreads + threadIdx.x;
        if (t < T) {
            atomicAdd(&hist[(key[j] >> shift) & (bins - 1)], 1);
            if (mark != nullptr && key[j] < V && first_of_block(seen, key[j])) {
                mark[key[j]] = 1;
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += kSortThreads) {
        counts[(long long)i * nblocks + blockIdx.x] = hist[i];
    }
}

// A warp a digit: counts[digit][*] becomes its exclusive prefix over the blocks, totals[digit]
// the sum.
__global__ void __launch_bounds__(kSortThreads)
    sort_scan_kernel(int* counts, int* totals, int bins, int nblocks) {
    wait_before();
    begin_next();
    const int digit = blockIdx.x * kSortWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (digit >= bins) {
        return;
    }
    int* row = counts + (long long)digit * nblocks;
    int base = 0;
    for (int b0 = 0; b0 < nblocks; b0 += 32) {
        const int b = b0 + lane;
        const int n = b < nblocks ? row[b] : 0;
        int x = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, d);
            x += lane >= d ? y : 0;
        }
        if (b < nblocks) {
            row[b] = base + x - n;
        }
        base += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) {
        totals[digit] = base;
    }
}

// Each block puts its pairs at their places. Where the blocks are few (scanned 0) it adds the
// counts of a digit itself, else it takes their prefix from sort_scan_kernel. Warp w owns the
// block's pairs [w 32 kSortRounds, (w + 1) 32 kSortRounds) in rounds of 32: a pair's rank among the
// warp's of its digit is the digit's running count plus the lower lanes of the round with the same
// digit, so equal digits keep their order. FIRST: the pairs are (ids[t], t).
template <typename Key, bool FIRST>
__global__ void __launch_bounds__(kSortThreads)
    sort_scatter_kernel(const Key* keys, const int* toks, int T, unsigned V, int shift, int bits,
                        const int* counts, const int* totals, int nblocks, int scanned,
                        unsigned* okeys, int* otoks, const ZeroShare zero) {
    wait_before();
    begin_next();
    if ((int)blockIdx.x >= nblocks) {
        zero_rows(zero, blockIdx.x - nblocks, kSortWarps);
        return;
    }
    __shared__ int run[kSortWarps][1 << kMaxDigit];
    __shared__ int base[1 << kMaxDigit];
    __shared__ int warp_sum[kSortWarps];
    const int bins = 1 << bits, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    for (int i = tid; i < bins; i += kSortThreads) {
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            run[w][i] = 0;
        }
    }
    // exclusive prefix of the totals: two digits a thread, a scan over the warps
    const int d0 = 2 * tid;
    int t[2] = {0, 0}, lower[2] = {0, 0};  // a digit's pairs in all blocks, and in those before
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (d0 + k >= bins) {
            continue;
        }
        const int* row = counts + (long long)(d0 + k) * nblocks;
        if (scanned) {
            t[k] = totals[d0 + k];
            lower[k] = row[blockIdx.x];
        } else {
#pragma unroll 8
            for (int b = 0; b < nblocks; ++b) {
                const int n = row[b];
                t[k] += n;
                lower[k] += b < (int)blockIdx.x ? n : 0;
            }
        }
    }
    const int t0 = t[0], t1 = t[1];
    int x = t0 + t1;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        x += lane >= d ? y : 0;
    }
    if (lane == 31) {
        warp_sum[warp] = x;
    }
    __syncthreads();
    int before = x - t0 - t1;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
        before += w < warp ? warp_sum[w] : 0;
    }
    if (d0 < bins) {
        base[d0] = before + lower[0];
    }
    if (d0 + 1 < bins) {
        base[d0 + 1] = before + t0 + lower[1];
    }
    const long long at = (long long)blockIdx.x * kSortItems + warp * 32 * kSortRounds + lane;
    unsigned key[kSortRounds];
    int tok[kSortRounds], rank[kSortRounds];
#pragma unroll
    for (int j = 0; j < kSortRounds; ++j) {
        const long long t = at + 32 * j;
        key[j] = 0;
        tok[j] = 0;
        rank[j] = 0;
        if (t < T) {
            key[j] = sort_key(keys, t, V);
            tok[j] = FIRST ? (int)t : toks[t];
        }
    }
#pragma unroll
    for (int j = 0; j < kSortRounds; ++j) {
        const bool live = at + 32 * j < T;
        // lanes past the end match nothing that counts: a digit of their own
        const unsigned digit = live ? (key[j] >> shift) & (bins - 1) : 0xffffffffu;
        const unsigned same = __match_any_sync(0xffffffffu, digit);
        if (live) {
            rank[j] = run[warp][digit] + __popc(same & ((1u << lane) - 1));
        }
        __syncwarp();
        if (live && lane == 31 - __clz(same)) {
            run[warp][digit] += __popc(same);
        }
        __syncwarp();
    }
    __syncthreads();
    // each warp's first place a digit
    for (int i = tid; i < bins; i += kSortThreads) {
        int sum = base[i];
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            const int n = run[w][i];
            run[w][i] = sum;
            sum += n;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortRounds; ++j) {
        if (at + 32 * j < T) {
            const int place = run[warp][(key[j] >> shift) & (bins - 1)] + rank[j];
            okeys[place] = key[j];
            otoks[place] = tok[j];
        }
    }
}

// ------------------------------------------------------------------------------------------
// backward: sums over the sorted list
// ------------------------------------------------------------------------------------------
constexpr int kSumThreads = 256, kSumWarps = kSumThreads / 32;

// A warp sums chunk `c` of the sorted list (len pairs) over one slab of 32 VEC channels. Rows
// whose pairs all lie in the chunk are written; the sum of a row that began before the chunk goes
// to partial[c][0], that of a row that began in it and goes on after it to partial[c][1]. The
// blocks past the first sum_blocks write their share of the rows without a token.
template <typename T, int VEC>
__global__ void __launch_bounds__(kSumThreads)
    embed_sum_kernel(const unsigned* keys, const int* toks, const T* __restrict__ dout,
                     float* dtable, float* partial, int n, unsigned V, int C, int slabs, int chunks,
                     int len, int sum_blocks, float scale, const ZeroShare zero) {
    wait_before();
    if (chunks > 1) {
        begin_next();
    }
    constexpr int kUnroll = 8;
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * kSumWarps + (threadIdx.x >> 5);
    if ((int)blockIdx.x >= sum_blocks) {
        zero_rows(zero, blockIdx.x - sum_blocks, kSumWarps);
        return;
    }
    if (item >= (long long)chunks * slabs) {
        return;
    }
    const int c = (int)(item / slabs), slab = (int)(item - (long long)c * slabs);
    const unsigned col = ((unsigned)slab * 32 + lane) * VEC;  // (past 2^31 in the last slab)
    const bool on = col < (unsigned)C;
    const int p0 = c * len, p1 = n - p0 < len ? n : p0 + len;  // (p0 + len may pass 2^31)
    const unsigned prev = p0 > 0 ? keys[p0 - 1] : 0xffffffffu;
    const unsigned next = p1 < n ? keys[p1] : 0xffffffffu;
    const T* src = dout + (on ? col : 0);
    float acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        acc[i] = 0.f;
    }
    unsigned cur = keys[p0];
    bool first = true;  // the chunk's first row
    const auto flush = [&](bool last) {
        if (cur < V && on) {
            const bool before = first && cur == prev, after = last && cur == next;
            float* dst = before ? partial + (long long)c * 2 * C + col
                         : after ? partial + ((long long)c * 2 + 1) * C + col
                                 : dtable + (long long)cur * C + col;
            const float by = before || after ? 1.f : scale;
            float o[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                o[i] = acc[i] * by;
            }
            store_vec<float, VEC>(dst, o);
        }
    };
    for (int p = p0; p < p1; p += kUnroll) {
        unsigned k[kUnroll];
        int t[kUnroll];
        float v[kUnroll][VEC];
        // (no branch round a load: what is past the chunk or outside the table is dropped below)
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            k[u] = keys[min(p + u, p1 - 1)];
            t[u] = toks[min(p + u, p1 - 1)];
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            load_vec<T, VEC>(src + (long long)t[u] * C, v[u]);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (p + u < p1) {
                if (k[u] != cur) {
                    flush(false);
                    first = false;
                    cur = k[u];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        acc[i] = 0.f;
                    }
                }
                if (k[u] < V && on) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        acc[i] += v[u][i];
                    }
                }
            }
        }
    }
    flush(true);
}

// Rows that cross a chunk's end, by the chunk they begin in: its part and the following chunks' in
// order. A warp an item (chunk, slab); rows of more than kLong parts by the block's warps together,
// each a contiguous share of the parts.
constexpr int kLong = 9;

template <int VEC>
__device__ __forceinline__ void add_parts(const float* partial, int q0, int q1, int C, unsigned col,
                                          float (&acc)[VEC]) {
    for (int q = q0; q < q1; q += 8) {
        float v[8][VEC];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            load_vec<float, VEC>(partial + (long long)min(q + u, q1 - 1) * 2 * C + col, v[u]);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (q + u < q1) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    acc[i] += v[u][i];
                }
            }
        }
    }
}

template <int VEC>
__global__ void __launch_bounds__(kSumThreads)
    embed_join_kernel(const unsigned* keys, float* dtable, const float* partial, int n, unsigned V,
                      int C, int slabs, int chunks, int len, float scale) {
    wait_before();
    __shared__ int long_last[kSumWarps];  // the last chunk of a warp's long row, or -1
    __shared__ __align__(32) float part_sum[kSumWarps][32 * VEC];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long item0 = (long long)blockIdx.x * kSumWarps;
    // (chunks fastest: the slabs of a long row fall to different blocks)
    const auto column = [&](long long item) {
        return ((unsigned)(item / chunks) * 32 + lane) * VEC;
    };
    const long long item = item0 + warp;
    int last = -1;
    if (item < (long long)chunks * slabs) {
        const int c = (int)(item % chunks);
        const long long end = (long long)(c + 1) * len;
        // a row that begins in chunk c and goes on: its following chunks, 32 looks at a time
        if (end < n) {
            const unsigned row = keys[end - 1];
            const unsigned before = c > 0 ? keys[(long long)c * len - 1] : 0xffffffffu;
            if (row < V && before != row && keys[end] == row) {
                last = c;
                for (int q = c + 1; q < chunks; q += 32) {
                    const long long at = (long long)(q + lane) * len;
                    const unsigned same =
                        __ballot_sync(0xffffffffu, q + lane < chunks && keys[min(at, n - 1ll)] == row);
                    const int run = same == 0xffffffffu ? 32 : __ffs(~same) - 1;
                    last += run;
                    if (run < 32) {
                        break;
                    }
                }
                const unsigned col = column(item);
                if (last - c < kLong && col < (unsigned)C) {
                    float acc[VEC];
                    load_vec<float, VEC>(partial + ((long long)c * 2 + 1) * C + col, acc);
                    add_parts<VEC>(partial, c + 1, last + 1, C, col, acc);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        acc[i] *= scale;
                    }
                    store_vec<float, VEC>(dtable + (long long)row * C + col, acc);
                }
                last = last - c < kLong ? -1 : last;
            }
        }
    }
    if (lane == 0) {
        long_last[warp] = last;
    }
    __syncthreads();
    for (int w = 0; w < kSumWarps; ++w) {
        if (long_last[w] < 0) {
            continue;
        }
        const int c = (int)((item0 + w) % chunks), parts = long_last[w] - c;
        const unsigned col = column(item0 + w);
        const bool on = col < (unsigned)C;
        float acc[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            acc[i] = 0.f;
        }
        if (on) {
            if (warp == 0) {
                load_vec<float, VEC>(partial + ((long long)c * 2 + 1) * C + col, acc);
            }
            add_parts<VEC>(partial, c + 1 + parts * warp / kSumWarps,
                           c + 1 + parts * (warp + 1) / kSumWarps, C, col, acc);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            part_sum[warp][lane * VEC + i] = acc[i];
        }
        __syncthreads();
        if (warp == 0 && on) {
            for (int k = 1; k < kSumWarps; ++k) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    acc[i] += part_sum[k][lane * VEC + i];
                }
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                acc[i] *= scale;
            }
            store_vec<float, VEC>(dtable + (long long)keys[(long long)(c + 1) * len] * C + col, acc);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------
// backward of a small table: sorted CTA by CTA
// ------------------------------------------------------------------------------------------
// Where the table's slab of 4 GL channels fits shared memory, a CTA sorts its own tokens there, up to
// kLocalTokens at a time: a counting sort by row whose ranks keep the tokens' order. Groups of GL
// lanes then take equal ranges of the sorted list, each row's sum in registers, so the only
// traffic is dout's; rows that end inside a range go to the table, those at its ends to a list
// whose runs of one row are added in order. The CTAs' tables are added in order by
// embed_local_reduce_kernel.
constexpr int kLocalThreads = 1024, kLocalWarps = kLocalThreads / 32;
constexpr int kLocalTokens = 4096, kLocalRounds = kLocalTokens / kLocalThreads;
constexpr int kLocalSmem = 200 * 1024;

struct LocalSmem {
    int table, ends, end_row, base, count, key, tok, bytes;
};
__host__ __device__ inline LocalSmem local_smem(int V, int lanes) {
    LocalSmem m;
    int at = 0;
    const auto take = [&](int n) {
        const int o = at;
        at += (n + 15) / 16 * 16;
        return o;
    };
    m.table = take(V * lanes * 16);
    m.ends = take(kLocalThreads * 2 * 16);
    m.end_row = take(kLocalThreads / lanes * 2 * 4);
    m.base = take((V + 1) * 4);
    m.count = take(kLocalWarps * V * 2);
    m.key = take(kLocalTokens * 2);
    m.tok = take(kLocalTokens * 2);
    m.bytes = at;
    return m;
}

template <typename T, typename Id, int GL>
__global__ void __launch_bounds__(kLocalThreads, 1)
    embed_local_kernel(const Id* __restrict__ ids, const T* __restrict__ dout,
                       float* __restrict__ partial, long long n, int V, int C, long long per) {
    begin_next();
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int kGroups = kLocalThreads / GL, kUnroll = 8;
    const LocalSmem m = local_smem(V, GL);
    float4* table = reinterpret_cast<float4*>(smem + m.table);
    float4* ends = reinterpret_cast<float4*>(smem + m.ends);
    int* end_row = reinterpret_cast<int*>(smem + m.end_row);
    int* base = reinterpret_cast<int*>(smem + m.base);
    uint16_t* count = reinterpret_cast<uint16_t*>(smem + m.count);
    uint16_t* skey = reinterpret_cast<uint16_t*>(smem + m.key);
    uint16_t* stok = reinterpret_cast<uint16_t*>(smem + m.tok);
    __shared__ int warp_total[kLocalWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = tid / GL, gl = tid % GL;
    const int col = (blockIdx.y * GL + gl) * 4;
    const bool on = col < C;
    for (int i = tid; i < V * GL; i += kLocalThreads) {
        table[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const long long t_end = min(n, (blockIdx.x + 1) * per);
    for (long long t0 = blockIdx.x * per; t0 < t_end; t0 += kLocalTokens) {
        // ranks among the warp's tokens of the same row
        for (int i = tid; i < kLocalWarps * V; i += kLocalThreads) {
            count[i] = 0;
        }
        int key[kLocalRounds], rank[kLocalRounds];
#pragma unroll
        for (int r = 0; r < kLocalRounds; ++r) {
            const long long t = t0 + warp * (32 * kLocalRounds) + 32 * r + lane;
            const long long id = t < t_end ? (long long)ids[t] : -1;
            key[r] = id >= 0 && id < V ? (int)id : -1;
        }
        __syncthreads();
        uint16_t* mine = count + warp * V;
#pragma unroll
        for (int r = 0; r < kLocalRounds; ++r) {
            const unsigned same = __match_any_sync(0xffffffffu, key[r]);
            const int before = __popc(same & ((1u << lane) - 1));
            rank[r] = key[r] >= 0 ? mine[key[r]] + before : 0;
            __syncwarp();
            if (key[r] >= 0 && lane == 31 - __clz(same)) {
                mine[key[r]] = (uint16_t)(rank[r] + 1);
            }
            __syncwarp();
        }
        __syncthreads();
        // a thread a row: the warps' first places; then the rows' (V at most kLocalThreads)
        int total = 0;
        if (tid < V) {
#pragma unroll 8
            for (int w = 0; w < kLocalWarps; ++w) {
                const int c = count[w * V + tid];
                count[w * V + tid] = (uint16_t)total;
                total += c;
            }
        }
        int x = total;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, d);
            x += lane >= d ? y : 0;
        }
        if (lane == 31) {
            warp_total[warp] = x;
        }
        __syncthreads();
        int lower = x - total, listed = 0;
#pragma unroll
        for (int w = 0; w < kLocalWarps; ++w) {
            lower += w < warp ? warp_total[w] : 0;
            listed += warp_total[w];
        }
        if (tid < V) {
            base[tid] = lower;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kLocalRounds; ++r) {
            if (key[r] >= 0) {
                const int at = base[key[r]] + mine[key[r]] + rank[r];
                skey[at] = (uint16_t)key[r];
                stok[at] = (uint16_t)(warp * (32 * kLocalRounds) + 32 * r + lane);
            }
        }
        __syncthreads();
        // sums of this group's range
        const int len = (listed + kGroups - 1) / kGroups;
        const int p0 = group * len, p1 = min(listed, p0 + len);
        if (gl == 0) {
            end_row[2 * group] = -1;
            end_row[2 * group + 1] = -1;
        }
        if (p0 < p1) {
            const T* src = dout + t0 * C + (on ? col : 0);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            int cur = skey[p0];
            bool first = true;
            const auto flush = [&](bool last) {
                if (first || last) {
                    const int e = 2 * group + (first ? 0 : 1);
                    ends[e * GL + gl] = acc;
                    if (gl == 0) {
                        end_row[e] = cur;
                    }
                } else {
                    float4 a = table[cur * GL + gl];
                    a.x += acc.x;
                    a.y += acc.y;
                    a.z += acc.z;
                    a.w += acc.w;
                    table[cur * GL + gl] = a;
                }
            };
            for (int p = p0; p < p1; p += kUnroll) {
                Raw<T, 4> v[kUnroll];
                int k[kUnroll];
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    const int q = min(p + u, p1 - 1);
                    k[u] = skey[q];
                    v[u] = load_raw<T, 4>(src + (long long)stok[q] * C);
                }
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    if (p + u < p1) {
                        if (k[u] != cur) {
                            flush(false);
                            first = false;
                            cur = k[u];
                            acc = make_float4(0.f, 0.f, 0.f, 0.f);
                        }
                        float y[4];
                        unpack_raw<T, 4>(v[u], y);
                        acc.x += y[0];
                        acc.y += y[1];
                        acc.z += y[2];
                        acc.w += y[3];
                    }
                }
            }
            flush(true);
        }
        __syncthreads();
        // the ranges' ends, sorted by row: the first entry of a row adds them up
        for (int e = group; e < 2 * kGroups; e += kGroups) {
            const int row = end_row[e];
            int prev = -1;
            for (int q = e - 1; q >= 0 && prev < 0; --q) {
                prev = end_row[q];
            }
            if (row < 0 || prev == row) {
                continue;
            }
            float4 a = table[row * GL + gl];
            for (int q = e; q < 2 * kGroups && (end_row[q] == row || end_row[q] < 0); ++q) {
                if (end_row[q] == row) {
                    const float4 b = ends[q * GL + gl];
                    a.x += b.x;
                    a.y += b.y;
                    a.z += b.z;
                    a.w += b.w;
                }
            }
            table[row * GL + gl] = a;
        }
        __syncthreads();
    }
    __syncthreads();
    if (on) {
        for (int row = group; row < V; row += kGroups) {
            *reinterpret_cast<float4*>(partial + ((long long)blockIdx.x * V + row) * C + col) =
                table[row * GL + gl];
        }
    }
}

// The CTAs' sums in order: four channels a thread, kReduceSegs threads over the CTAs.
constexpr int kReduceSegs = 16;

__global__ void __launch_bounds__(32 * kReduceSegs)
    embed_local_reduce_kernel(const float4* partial, int parts, int total4, float scale,
                              float4* dtable) {
    wait_before();
    __shared__ float4 sh[kReduceSegs][32];
    const int r = threadIdx.x & 31, seg = threadIdx.x >> 5, i = blockIdx.x * 32 + r;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < total4) {
#pragma unroll 10
        for (int p = seg; p < parts; p += kReduceSegs) {
            const float4 v = partial[(long long)p * total4 + i];
            s.x += v.x;
            s.y += v.y;
            s.z += v.z;
            s.w += v.w;
        }
    }
    sh[seg][r] = s;
    __syncthreads();
    if (seg == 0 && i < total4) {
#pragma unroll
        for (int k = 1; k < kReduceSegs; ++k) {
            s.x += sh[k][r].x;
            s.y += sh[k][r].y;
            s.z += sh[k][r].z;
            s.w += sh[k][r].w;
        }
        dtable[i] = make_float4(s.x * scale, s.y * scale, s.z * scale, s.w * scale);
    }
}

struct BwdPlan {
    bool local;
    int lanes, parts;  // local: lanes of a token, CTAs a slab
    long long per;     // tokens a CTA
    int passes, bits, nblocks;
    int slabs, chunks, len, vec;
    size_t off_present, off_counts, off_totals, off_keys[2], off_toks[2], off_partial, bytes;
};

size_t round256(size_t n) {
    return (n + 255) & ~size_t(255);
}

// Everything the backward does follows from T, V, C and the channel vector. False: too large.
bool plan_bwd(int64_t T, int64_t V, int64_t C, int vec, BwdPlan& p) {
    if (T >= (int64_t(1) << 31) - kSortItems || V >= (int64_t(1) << 31) - 1 ||
        C >= (int64_t(1) << 31)) {
        return false;
    }
    p.lanes = C <= 32 ? 8 : C <= 64 ? 16 : 32;
    // Where a CTA's table of sums and its tokens' sort fit shared memory, us (local / sorted): T
    // 589824, V 65, C 128 41 / 75, clipped offsets (nearly all of one row) 42 / 175; T 262144: V 23,
    // C 256 35 / 50, V 256, C 128 25 / 39; T 512, V 23, C 256 10 / 12; T 16384, V 250, C 1024 24 / 24.
    // (a grid has at most 65535 slabs)
    const int64_t local_slabs = (C + 4 * p.lanes - 1) / (4 * p.lanes);
    p.local = vec >= 4 && V <= kLocalThreads && local_slabs <= 65535 &&
              local_smem((int)V, p.lanes).bytes <= kLocalSmem;
    if (p.local) {
        p.slabs = (int)local_slabs;
        // a CTA an SM, of at least 512 tokens
        const int64_t want = std::max<int64_t>(1, kSms / p.slabs);
        p.per = std::max<int64_t>(512, (T + want - 1) / want);
        p.parts = (int)((T + p.per - 1) / p.per);
        p.off_partial = 0;
        p.bytes = round256((size_t)p.parts * V * C * 4);
        return true;
    }
    int width = 1;
    while ((int64_t(1) << width) <= V) {
        ++width;  // V itself is a key
    }
    p.passes = (width + kMaxDigit - 1) / kMaxDigit;
    p.bits = (width + p.passes - 1) / p.passes;
    p.nblocks = (int)((T + kSortItems - 1) / kSortItems);
    p.vec = vec;
    p.slabs = (int)((C + 32 * p.vec - 1) / (32 * p.vec));
    // chunks: enough warps to fill the machine (48 a SM), of at least 16 pairs
    const int64_t want = std::max<int64_t>(1, 48 * kSms / p.slabs);
    p.len = (int)std::max<int64_t>(16, (T + want - 1) / want);
    p.chunks = (int)((T + p.len - 1) / p.len);
    size_t at = 0;
    const auto take = [&](size_t n) {
        const size_t o = at;
        at += round256(n);
        return o;
    };
    p.off_present = take((size_t)V);
    p.off_counts = take((size_t)p.nblocks * (size_t(1) << p.bits) * 4);
    p.off_totals = take((size_t(1) << p.bits) * 4);
    for (int i = 0; i < 2; ++i) {
        p.off_keys[i] = take((size_t)T * 4);
        p.off_toks[i] = take((size_t)T * 4);
    }
    p.off_partial = take((size_t)p.chunks * 2 * (size_t)C * 4);
    p.bytes = at;
    return true;
}

template <typename T, typename Id, int GL>
cudaError_t launch_embed_local(cudaStream_t s, const void* ids, const void* dout, float* dtable,
                               int64_t n, int64_t V, int64_t C, float scale, float* partial,
                               const BwdPlan& p) {
    auto kern = embed_local_kernel<T, Id, GL>;
    static bool done[kMaxDevices] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev >= kMaxDevices || !done[dev])) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kLocalSmem);
        if (e == cudaSuccess && dev < kMaxDevices) {
            done[dev] = true;
        }
    }
    if (e != cudaSuccess) {
        return e;
    }
    kern<<<dim3(p.parts, p.slabs), kLocalThreads, local_smem((int)V, GL).bytes, s>>>(
        static_cast<const Id*>(ids), static_cast<const T*>(dout), partial, n, (int)V, (int)C,
        p.per);
    const int total4 = (int)(V * C / 4);
    e = cudaGetLastError();
    return e != cudaSuccess
               ? e
               : launch_behind(embed_local_reduce_kernel, (total4 + 31) / 32, 32 * kReduceSegs, 0,
                               s, reinterpret_cast<const float4*>(partial), p.parts, total4,
                               scale, reinterpret_cast<float4*>(dtable));
}

template <typename T, typename Id>
cudaError_t launch_embed_bwd(cudaStream_t s, const void* ids, const void* dout, float* dtable,
                             int64_t n, int64_t V, int64_t C, float scale, uint8_t* ws,
                             const BwdPlan& p) {
    if (p.local) {
        float* partial = reinterpret_cast<float*>(ws + p.off_partial);
        return p.lanes == 8    ? launch_embed_local<T, Id, 8>(s, ids, dout, dtable, n, V, C, scale,
                                                              partial, p)
               : p.lanes == 16 ? launch_embed_local<T, Id, 16>(s, ids, dout, dtable, n, V, C,
                                                               scale, partial, p)
                               : launch_embed_local<T, Id, 32>(s, ids, dout, dtable, n, V, C,
                                                               scale, partial, p);
    }
    int* counts = reinterpret_cast<int*>(ws + p.off_counts);
    int* totals = reinterpret_cast<int*>(ws + p.off_totals);
    unsigned* keys[2];
    int* toks[2];
    for (int i = 0; i < 2; ++i) {
        keys[i] = reinterpret_cast<unsigned*>(ws + p.off_keys[i]);
        toks[i] = reinterpret_cast<int*>(ws + p.off_toks[i]);
    }
    float* partial = reinterpret_cast<float*>(ws + p.off_partial);
    // A table that is small beside the tokens is cleared whole: marking costs 0.05 to 0.1 ns a
    // token, since its blocks meet on the same rows, a clear 1 ns each 4 KB.
    const bool clear = V * C <= 64 * n;
    uint8_t* present = clear ? nullptr : ws + p.off_present;
    cudaError_t e = clear ? cudaMemsetAsync(dtable, 0, (size_t)(V * C) * 4, s)
                          : cudaMemsetAsync(present, 0, (size_t)V, s);
    if (e != cudaSuccess) {
        return e;
    }
    // the rows without a token in equal shares, one for every kernel after the first but the scans
    const int shares = 2 * p.passes;
    int share = 0;
    const auto next_share = [&] {
        ZeroShare z{};
        z.present = present;
        z.dtable = dtable;
        z.row0 = (int)(V * share / shares / 32 * 32);
        ++share;
        z.row1 = share == shares ? (int)V : (int)(V * share / shares / 32 * 32);
        z.C = (int)C;
        z.vec = p.vec > 1;
        z.blocks = clear ? 0 : std::min(8 * kSms, (z.row1 - z.row0 + 31) / 32);
        return z;
    };
    const int bins = 1 << p.bits;
    int cur = 0;
    for (int pass = 0; pass < p.passes; ++pass) {
        const int shift = pass * p.bits;
        if (pass == 0) {
            sort_count_kernel<Id><<<p.nblocks, kSortThreads, 0, s>>>(
                static_cast<const Id*>(ids), (int)n, (unsigned)V, shift, p.bits, counts,
                p.nblocks, present, ZeroShare{});
        } else {
            const ZeroShare z = next_share();
            launch_behind(sort_count_kernel<unsigned>, p.nblocks + z.blocks, kSortThreads, 0, s,
                          keys[cur], (int)n, (unsigned)V, shift, p.bits, counts, p.nblocks, nullptr,
                          z);
        }
        const int scanned = p.nblocks > kFewBlocks;
        if (scanned) {
            launch_behind(sort_scan_kernel, (bins + kSortWarps - 1) / kSortWarps, kSortThreads, 0,
                          s, counts, totals, bins, p.nblocks);
        }
        const ZeroShare z = next_share();
        if (pass == 0) {
            launch_behind(sort_scatter_kernel<Id, true>, p.nblocks + z.blocks, kSortThreads, 0, s,
                          static_cast<const Id*>(ids), nullptr, (int)n, (unsigned)V, shift, p.bits,
                          counts, totals, p.nblocks, scanned, keys[cur], toks[cur], z);
        } else {
            launch_behind(sort_scatter_kernel<unsigned, false>, p.nblocks + z.blocks, kSortThreads,
                          0, s, keys[cur], toks[cur], (int)n, (unsigned)V, shift, p.bits, counts,
                          totals, p.nblocks, scanned, keys[cur ^ 1], toks[cur ^ 1], z);
            cur ^= 1;
        }
    }
    const int64_t items = (int64_t)p.chunks * p.slabs;
    const unsigned sum_grid = (unsigned)((items + kSumWarps - 1) / kSumWarps);
    const ZeroShare z = next_share();
    const auto sum = [&](auto tag) {
        constexpr int VEC = decltype(tag)::value;
        launch_behind(embed_sum_kernel<T, VEC>, sum_grid + z.blocks, kSumThreads, 0, s, keys[cur],
                      toks[cur], static_cast<const T*>(dout), dtable, partial, (int)n, (unsigned)V,
                      (int)C, p.slabs, p.chunks, p.len, (int)sum_grid, scale, z);
        if (p.chunks > 1) {
            constexpr int JVEC = VEC == 1 ? 1 : 4;  // narrower slabs: more blocks for a long row
            const int slabs = (int)((C + 32 * JVEC - 1) / (32 * JVEC));
            const int64_t joins = (int64_t)p.chunks * slabs;
            launch_behind(embed_join_kernel<JVEC>, (unsigned)((joins + kSumWarps - 1) / kSumWarps),
                          kSumThreads, 0, s, keys[cur], dtable, partial, (int)n, (unsigned)V,
                          (int)C, slabs, p.chunks, p.len, scale);
        }
    };
    if (p.vec == 8) {
        if constexpr (sizeof(T) == 2) {
            sum(std::integral_constant<int, 8>{});
        }
    } else if (p.vec == 4) {
        sum(std::integral_constant<int, 4>{});
    } else {
        sum(std::integral_constant<int, 1>{});
    }
    return cudaGetLastError();
}

int check_sizes(const char* who, int64_t T, int64_t V, int64_t C) {
    int64_t a = 0, b = 0;
    if (T < 0 || V < 0 || C < 0) {
        return fail(kInvalidArgument, std::string(who) + ": sizes must be non-negative");
    }
    if (C >= (int64_t(1) << 31) || __builtin_mul_overflow(T, C * 4, &a) ||
        __builtin_mul_overflow(V, C * 4, &b)) {
        return fail(kInvalidArgument, std::string(who) + ": sizes overflow");
    }
    return kOk;
}

}  // namespace
}  // namespace cflk

using namespace cflk;

extern "C" int cflk_embed(void* stream, int table_dtype, int out_dtype, int ids_64,
                          const void* ids, const void* table, void* out, int64_t T, int64_t V,
                          int64_t C, float scale) {
    clear_error();
    const auto known = [](int d) { return d == kF16 || d == kBF16 || d == kF32; };
    if (!known(table_dtype) || !known(out_dtype) ||
        (table_dtype != out_dtype && table_dtype != kF32)) {
        return fail(kInvalidArgument,
                    "embed: table must be f16, bf16 or f32, out the table's type (or any of the "
                    "three for an f32 table)");
    }
    if (ids_64 != 0 && ids_64 != 1) {
        return fail(kInvalidArgument, "embed: ids are int32 (ids_64 0) or int64 (1)");
    }
    const int rc = check_sizes("embed", T, V, C);
    if (rc != kOk) {
        return rc;
    }
    if (T == 0 || C == 0) {
        return kOk;
    }
    if (ids == nullptr || out == nullptr || (V > 0 && table == nullptr)) {
        return fail(kInvalidArgument, "embed: null buffer");
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (V == 0) {  // no row to read: zeros
        const cudaError_t e = cudaMemsetAsync(out, 0, (size_t)T * (size_t)C * (out_dtype == kF32 ? 4 : 2), s);
        return e == cudaSuccess ? kOk
                                : fail(kInternal, std::string("embed: ") + cudaGetErrorString(e));
    }
    const auto run = [&](auto ti, auto to) -> cudaError_t {
        using TI = decltype(ti);
        using TO = decltype(to);
        return ids_64 ? launch_embed<TI, TO, long long>(s, ids, table, out, T, V, C, scale)
                      : launch_embed<TI, TO, int>(s, ids, table, out, T, V, C, scale);
    };
    const cudaError_t e = table_dtype == kF16    ? run(__half{}, __half{})
                          : table_dtype == kBF16 ? run(__nv_bfloat16{}, __nv_bfloat16{})
                          : out_dtype == kF16    ? run(float{}, __half{})
                          : out_dtype == kBF16   ? run(float{}, __nv_bfloat16{})
                                                 : run(float{}, float{});
    if (e != cudaSuccess) {
        return fail(kInternal, std::string("embed launch: ") + cudaGetErrorString(e));
    }
    return kOk;
}

extern "C" int cflk_embed_bwd_workspace_size(int64_t T, int64_t V, int64_t C, size_t* bytes) {
    clear_error();
    const int rc = check_sizes("embed_bwd", T, V, C);
    if (rc != kOk) {
        return rc;
    }
    if (bytes == nullptr) {
        return fail(kInvalidArgument, "embed_bwd: null size");
    }
    *bytes = 0;
    if (T == 0 || V == 0 || C == 0) {
        return kOk;
    }
    // whichever vector the type and the buffers' alignment take
    for (const int vec : {1, 4, 8}) {
        BwdPlan p;
        if (!plan_bwd(T, V, C, vec, p)) {
            return fail(kInvalidArgument, "embed_bwd: T and V must be below 2^31");
        }
        *bytes = std::max(*bytes, p.bytes);
    }
    return kOk;
}

extern "C" int cflk_embed_bwd(void* stream, int dtype, int ids_64, const void* ids,
                              const void* dout, float* dtable, int64_t T, int64_t V, int64_t C,
                              float scale, void* workspace, size_t ws_bytes) {
    clear_error();
    if (dtype != kF16 && dtype != kBF16 && dtype != kF32) {
        return fail(kInvalidArgument, "embed_bwd: dout must be f16, bf16 or f32");
    }
    if (ids_64 != 0 && ids_64 != 1) {
        return fail(kInvalidArgument, "embed_bwd: ids are int32 (ids_64 0) or int64 (1)");
    }
    const int rc = check_sizes("embed_bwd", T, V, C);
    if (rc != kOk) {
        return rc;
    }
    if (V == 0 || C == 0) {
        return kOk;
    }
    if (dtable == nullptr || (T > 0 && (ids == nullptr || dout == nullptr))) {
        return fail(kInvalidArgument, "embed_bwd: null buffer");
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (T == 0) {
        const cudaError_t e = cudaMemsetAsync(dtable, 0, (size_t)V * (size_t)C * 4, s);
        return e == cudaSuccess
                   ? kOk
                   : fail(kInternal, std::string("embed_bwd: ") + cudaGetErrorString(e));
    }
    // eight or four channels a lane (16 bytes of dout and 32 of dtable, or half) where the rows
    // allow it
    const auto fits = [&](int v) {
        const size_t bytes = (size_t)v * (dtype == kF32 ? 4 : 2);
        return C % v == 0 && reinterpret_cast<uintptr_t>(dout) % bytes == 0 &&
               reinterpret_cast<uintptr_t>(dtable) % (4 * v) == 0;
    };
    // (eight only where it leaves no more of the last slab's lanes idle)
    const bool wide = (C + 255) / 256 * 2 <= (C + 127) / 128;
    const int vec = dtype != kF32 && fits(8) && wide ? 8 : fits(4) ? 4 : 1;
    BwdPlan p;
    if (!plan_bwd(T, V, C, vec, p)) {
        return fail(kInvalidArgument, "embed_bwd: T and V must be below 2^31");
    }
    if (workspace == nullptr || ws_bytes < p.bytes ||
        reinterpret_cast<uintptr_t>(workspace) % 256 != 0) {
        return fail(kInvalidArgument,
                    "embed_bwd: workspace below cflk_embed_bwd_workspace_size or not 256-byte "
                    "aligned");
    }
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const auto run = [&](auto tag) -> cudaError_t {
        using T_ = decltype(tag);
        return ids_64 ? launch_embed_bwd<T_, long long>(s, ids, dout, dtable, T, V, C, scale, ws, p)
                      : launch_embed_bwd<T_, int>(s, ids, dout, dtable, T, V, C, scale, ws, p);
    };
    const cudaError_t e = dtype == kF16    ? run(__half{})
                          : dtype == kBF16 ? run(__nv_bfloat16{})
                                           : run(float{});
    if (e != cudaSuccess) {
        return fail(kInternal, std::string("embed_bwd launch: ") + cudaGetErrorString(e));
    }
    return kOk;
}
