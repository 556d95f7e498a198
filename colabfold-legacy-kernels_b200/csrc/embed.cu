// Embedding lookup with scaling and its gradient by sorted tokens.
//
//   forward   out[t] = scale * table[ids[t]]        (a row of zeros for an id outside [0, V))
//   backward  dtable[v] = scale * sum over t with ids[t] = v of dout[t], float32
//
// Both are bound by HBM: the forward by the T output rows, the backward by the T rows of dout and
// the V float32 rows it writes. The backward sorts (id, token) pairs by id (a stable radix sort:
// the tokens of one id stay in order), cuts the sorted list into equal chunks so that an id with
// many tokens is spread over many warps, and adds the chunks' partial sums in the order of the
// list: no float atomics, the same bits every run.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "capi_internal.h"
#include "cflk_b200.h"
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
// remainder, so the loop divides nothing.
template <typename TI, typename TO, typename Id, int VEC>
__global__ void __launch_bounds__(kFwdThreads)
    embed_kernel(const Id* __restrict__ ids, const TI* __restrict__ table, TO* __restrict__ out,
                 long long T, long long V, int cv, float scale) {
    const long long stride = (long long)gridDim.x * kFwdThreads;
    const long long first = (long long)blockIdx.x * kFwdThreads + threadIdx.x;
    const long long drow = stride / cv;
    const int dcol = (int)(stride - drow * cv);
    long long row = first / cv;
    int col = (int)(first - row * cv);
    while (row < T) {
        long long r[kFwdUnroll], id[kFwdUnroll];
        int c[kFwdUnroll];
#pragma unroll
        for (int u = 0; u < kFwdUnroll; ++u) {
            r[u] = row;
            c[u] = col;
            id[u] = row < T ? (long long)ids[row] : -1;
            row += drow;
            col += dcol;
            if (col >= cv) {
                col -= cv;
                ++row;
            }
        }
        float v[kFwdUnroll][VEC];
#pragma unroll
        for (int u = 0; u < kFwdUnroll; ++u) {
            const bool ok = id[u] >= 0 && id[u] < V;
            if (ok) {
                load_vec<TI, VEC>(table + (id[u] * cv + c[u]) * VEC, v[u]);
            }
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
            V, (int)cv, scale);
    } else {
        embed_kernel<TI, TO, Id, 1><<<grid, kFwdThreads, 0, s>>>(
            static_cast<const Id*>(ids), static_cast<const TI*>(table), static_cast<TO*>(out), T,
            V, (int)cv, scale);
    }
    return cudaGetLastError();
}

// ------------------------------------------------------------------------------------------
// backward: stable radix sort of (id, token)
// ------------------------------------------------------------------------------------------
constexpr int kSortThreads = 256, kSortWarps = kSortThreads / 32, kSortRounds = 4;
constexpr int kSortItems = kSortThreads * kSortRounds;  // a block's consecutive pairs
constexpr int kMaxDigit = 9;                            // bits of a pass

// An id outside [0, V) sorts as V, behind every row.
template <typename Id>
__device__ __forceinline__ unsigned sort_key(const Id* ids, long long t, unsigned V) {
    const long long id = (long long)ids[t];
    return id >= 0 && id < (long long)V ? (unsigned)id : V;
}

// counts[digit][block]
template <typename Key>
__global__ void __launch_bounds__(kSortThreads)
    sort_count_kernel(const Key* __restrict__ keys, int T, unsigned V, int shift, int bits,
                      int* __restrict__ counts, int nblocks) {
    __shared__ int hist[1 << kMaxDigit];
    const int bins = 1 << bits;
    for (int i = threadIdx.x; i < bins; i += kSortThreads) {
        hist[i] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortRounds; ++j) {
        const long long t = (long long)blockIdx.x * kSortItems + j * kSortThreads + threadIdx.x;
        if (t < T) {
            atomicAdd(&hist[(sort_key(keys, t, V) >> shift) & (bins - 1)], 1);
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
    sort_scan_kernel(int* __restrict__ counts, int* __restrict__ totals, int bins, int nblocks) {
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

// Each block puts its pairs at their places. Warp w owns the block's pairs [w 32 kSortRounds,
// (w + 1) 32 kSortRounds) in rounds of 32: a pair's rank among the warp's of its digit is the
// digit's running count plus the lower lanes of the round with the same digit, so equal digits
// keep their order. FIRST: the pairs are (ids[t], t).
template <typename Key, bool FIRST>
__global__ void __launch_bounds__(kSortThreads)
    sort_scatter_kernel(const Key* __restrict__ keys, const int* __restrict__ toks, int T,
                        unsigned V, int shift, int bits, const int* __restrict__ counts,
                        const int* __restrict__ totals, int nblocks, unsigned* __restrict__ okeys,
                        int* __restrict__ otoks) {
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
    const int t0 = d0 < bins ? totals[d0] : 0, t1 = d0 + 1 < bins ? totals[d0 + 1] : 0;
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
        base[d0] = before + counts[(long long)d0 * nblocks + blockIdx.x];
    }
    if (d0 + 1 < bins) {
        base[d0 + 1] = before + t0 + counts[(long long)(d0 + 1) * nblocks + blockIdx.x];
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
constexpr int kSumThreads = 256, kSumWarps = kSumThreads / 32, kSumUnroll = 8;

// A warp sums chunk `c` of the sorted list (len pairs) over one slab of 32 VEC channels. Rows
// whose pairs all lie in the chunk are written; the sum of a row that began before the chunk goes
// to partial[c][0], that of a row that began in it and goes on after it to partial[c][1].
template <typename T, int VEC>
__global__ void __launch_bounds__(kSumThreads)
    embed_sum_kernel(const unsigned* __restrict__ keys, const int* __restrict__ toks,
                     const T* __restrict__ dout, float* __restrict__ dtable,
                     float* __restrict__ partial, int n, unsigned V, int C, int slabs, int chunks,
                     int len, float scale) {
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * kSumWarps + (threadIdx.x >> 5);
    if (item >= (long long)chunks * slabs) {
        return;
    }
    const int c = (int)(item / slabs), slab = (int)(item - (long long)c * slabs);
    const int col = (slab * 32 + lane) * VEC;
    const bool on = col < C;
    const int p0 = c * len, p1 = min(p0 + len, n);
    const unsigned prev = p0 > 0 ? keys[p0 - 1] : 0xffffffffu;
    const unsigned next = p1 < n ? keys[p1] : 0xffffffffu;
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
    for (int p = p0; p < p1; p += kSumUnroll) {
        unsigned k[kSumUnroll];
        float v[kSumUnroll][VEC];
#pragma unroll
        for (int u = 0; u < kSumUnroll; ++u) {
            k[u] = p + u < p1 ? keys[p + u] : V;
        }
#pragma unroll
        for (int u = 0; u < kSumUnroll; ++u) {
            if (k[u] < V && on) {
                load_vec<T, VEC>(dout + (long long)toks[p + u] * C + col, v[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < kSumUnroll; ++u) {
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

// Rows that cross a chunk's end, by the warp of the chunk they begin in: its part and the
// following chunks' in order.
template <int VEC>
__device__ __forceinline__ void join_row(const unsigned* keys, float* dtable,
                                         const float* partial, int n, unsigned V, int C, int c,
                                         int slab, int len, float scale) {
    const int lane = threadIdx.x & 31, col = (slab * 32 + lane) * VEC;
    const long long end = (long long)(c + 1) * len;
    if (end >= n) {
        return;
    }
    const unsigned row = keys[end - 1];
    const bool began_here = c == 0 || keys[(long long)c * len - 1] != row;
    if (row >= V || keys[end] != row || !began_here || col >= C) {
        return;
    }
    // the row's last chunk: the one that holds the last pair with its key
    long long lo = end, hi = n;  // keys[lo] == row, keys[hi] != row (or past the end)
    while (hi - lo > 1) {
        const long long mid = (lo + hi) >> 1;
        if (keys[mid] == row) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    const int last = (int)(lo / len);
    float acc[VEC];
    load_vec<float, VEC>(partial + ((long long)c * 2 + 1) * C + col, acc);
    for (int q = c + 1; q <= last; q += 8) {
        float v[8][VEC];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (q + u <= last) {
                load_vec<float, VEC>(partial + (long long)(q + u) * 2 * C + col, v[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (q + u <= last) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    acc[i] += v[u][i];
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        acc[i] *= scale;
    }
    store_vec<float, VEC>(dtable + (long long)row * C + col, acc);
}

// The rows that cross chunks (the first chunks * slabs warps) and, by every warp, the rows
// without a token: 32 rows a step, each lane looks its row up in the sorted keys.
template <int VEC>
__global__ void __launch_bounds__(kSumThreads)
    embed_finish_kernel(const unsigned* __restrict__ keys, float* __restrict__ dtable,
                        const float* __restrict__ partial, int n, unsigned V, int C, int slabs,
                        int chunks, int len, float scale) {
    const int lane = threadIdx.x & 31;
    const long long warp = (long long)blockIdx.x * kSumWarps + (threadIdx.x >> 5);
    const long long warps = (long long)gridDim.x * kSumWarps;
    for (long long item = warp; item < (long long)chunks * slabs; item += warps) {
        const int c = (int)(item / slabs);
        join_row<VEC>(keys, dtable, partial, n, V, C, c, (int)(item - (long long)c * slabs), len,
                      scale);
    }
    for (long long r0 = warp * 32; r0 < (long long)V; r0 += warps * 32) {
        const long long row = r0 + lane;
        bool empty = row < (long long)V;
        if (empty) {
            int lo = 0, hi = n;  // first place with keys >= row
            while (lo < hi) {
                const int mid = (int)(((long long)lo + hi) >> 1);
                if (keys[mid] < (unsigned)row) {
                    lo = mid + 1;
                } else {
                    hi = mid;
                }
            }
            empty = lo >= n || keys[lo] != (unsigned)row;
        }
        unsigned todo = __ballot_sync(0xffffffffu, empty);
        float zero[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            zero[i] = 0.f;
        }
        while (todo != 0) {
            const int r = __ffs(todo) - 1;
            todo &= todo - 1;
            float* dst = dtable + (r0 + r) * C;
            for (int col = lane * VEC; col < C; col += 32 * VEC) {
                store_vec<float, VEC>(dst + col, zero);
            }
        }
    }
}

struct BwdPlan {
    int passes, bits, nblocks;
    int slabs, chunks, len, vec;
    size_t off_counts, off_totals, off_keys[2], off_toks[2], off_partial, bytes;
};

size_t round256(size_t n) {
    return (n + 255) & ~size_t(255);
}

// Everything the backward does follows from T, V, C and the channel vector. False: too large.
bool plan_bwd(int64_t T, int64_t V, int64_t C, bool vec, BwdPlan& p) {
    if (T >= (int64_t(1) << 31) - kSortItems || V >= (int64_t(1) << 31) - 1 ||
        C >= (int64_t(1) << 31)) {
        return false;
    }
    int width = 1;
    while ((int64_t(1) << width) <= V) {
        ++width;  // V itself is a key
    }
    p.passes = (width + kMaxDigit - 1) / kMaxDigit;
    p.bits = (width + p.passes - 1) / p.passes;
    p.nblocks = (int)((T + kSortItems - 1) / kSortItems);
    p.vec = vec ? 4 : 1;
    p.slabs = (int)((C + 32 * p.vec - 1) / (32 * p.vec));
    // chunks: enough warps to fill the machine (16 a SM), at least 8 pairs each
    const int64_t want = std::max<int64_t>(1, 16 * kSms / p.slabs);
    p.len = (int)std::max<int64_t>(8, (T + want - 1) / want);
    p.chunks = (int)((T + p.len - 1) / p.len);
    size_t at = 0;
    const auto take = [&](size_t n) {
        const size_t o = at;
        at += round256(n);
        return o;
    };
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

template <typename T, typename Id>
cudaError_t launch_embed_bwd(cudaStream_t s, const void* ids, const void* dout, float* dtable,
                             int64_t n, int64_t V, int64_t C, float scale, uint8_t* ws,
                             const BwdPlan& p) {
    int* counts = reinterpret_cast<int*>(ws + p.off_counts);
    int* totals = reinterpret_cast<int*>(ws + p.off_totals);
    unsigned* keys[2];
    int* toks[2];
    for (int i = 0; i < 2; ++i) {
        keys[i] = reinterpret_cast<unsigned*>(ws + p.off_keys[i]);
        toks[i] = reinterpret_cast<int*>(ws + p.off_toks[i]);
    }
    float* partial = reinterpret_cast<float*>(ws + p.off_partial);
    const int bins = 1 << p.bits;
    int cur = 0;
    for (int pass = 0; pass < p.passes; ++pass) {
        const int shift = pass * p.bits;
        if (pass == 0) {
            sort_count_kernel<Id><<<p.nblocks, kSortThreads, 0, s>>>(
                static_cast<const Id*>(ids), (int)n, (unsigned)V, shift, p.bits, counts,
                p.nblocks);
        } else {
            sort_count_kernel<unsigned><<<p.nblocks, kSortThreads, 0, s>>>(
                keys[cur], (int)n, (unsigned)V, shift, p.bits, counts, p.nblocks);
        }
        sort_scan_kernel<<<(bins + kSortWarps - 1) / kSortWarps, kSortThreads, 0, s>>>(
            counts, totals, bins, p.nblocks);
        if (pass == 0) {
            sort_scatter_kernel<Id, true><<<p.nblocks, kSortThreads, 0, s>>>(
                static_cast<const Id*>(ids), nullptr, (int)n, (unsigned)V, shift, p.bits, counts,
                totals, p.nblocks, keys[cur], toks[cur]);
        } else {
            sort_scatter_kernel<unsigned, false><<<p.nblocks, kSortThreads, 0, s>>>(
                keys[cur], toks[cur], (int)n, (unsigned)V, shift, p.bits, counts, totals,
                p.nblocks, keys[cur ^ 1], toks[cur ^ 1]);
            cur ^= 1;
        }
    }
    const int64_t items = (int64_t)p.chunks * p.slabs;
    const unsigned sum_grid = (unsigned)((items + kSumWarps - 1) / kSumWarps);
    const unsigned fin_grid = (unsigned)std::min<int64_t>(
        4 * kSms, std::max<int64_t>(sum_grid, (V + 32 * kSumWarps - 1) / (32 * kSumWarps)));
    if (p.vec == 4) {
        embed_sum_kernel<T, 4><<<sum_grid, kSumThreads, 0, s>>>(
            keys[cur], toks[cur], static_cast<const T*>(dout), dtable, partial, (int)n,
            (unsigned)V, (int)C, p.slabs, p.chunks, p.len, scale);
        embed_finish_kernel<4><<<fin_grid, kSumThreads, 0, s>>>(
            keys[cur], dtable, partial, (int)n, (unsigned)V, (int)C, p.slabs, p.chunks, p.len,
            scale);
    } else {
        embed_sum_kernel<T, 1><<<sum_grid, kSumThreads, 0, s>>>(
            keys[cur], toks[cur], static_cast<const T*>(dout), dtable, partial, (int)n,
            (unsigned)V, (int)C, p.slabs, p.chunks, p.len, scale);
        embed_finish_kernel<1><<<fin_grid, kSumThreads, 0, s>>>(
            keys[cur], dtable, partial, (int)n, (unsigned)V, (int)C, p.slabs, p.chunks, p.len,
            scale);
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
    BwdPlan a, b;
    if (!plan_bwd(T, V, C, false, a) || !plan_bwd(T, V, C, true, b)) {
        return fail(kInvalidArgument, "embed_bwd: T and V must be below 2^31");
    }
    *bytes = std::max(a.bytes, b.bytes);  // whichever the buffers' alignment takes
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
    // four channels a lane (8 or 16 bytes of dout, 16 of dtable) when the rows allow it
    const size_t want = dtype == kF32 ? 16 : 8;
    const bool vec = C % 4 == 0 && reinterpret_cast<uintptr_t>(dout) % want == 0 &&
                     aligned16(dtable);
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
