// The global norm of many gradient tensors, and clipping by it.
//
//   sumsq = sum of g^2 over all tensors
//   norm = scale * sqrt(sumsq);  out = g * scale * min(1, max_norm / (norm + eps))
//
// `scale` takes a loss scale out. Bound by HBM: every gradient is read once for the norm, read
// again (out of L2 where all of them fit) and written once for the clip. Two launches: the first
// leaves one float64 sum a block, the second adds those in a fixed order in every block (about
// 9 KB out of L2) and scales. Neither has atomics, so a call's bits depend on its tensors' sizes,
// alignment and values only. Tensors are cut into chunks of kChunk elements and the blocks take
// equal ranges of them, so a thousand small tensors and one large one spread alike; the table of
// tensors travels as a kernel parameter (no copy, nothing to keep alive on the host), kTable tensors
// a launch. A block's clip goes backwards through the chunks: it finds what its norm read last still
// in L2.
//
// 300 M bf16 elements clipped into float32: norm 114 us (5.3 TB/s), clip 318 us (600 MB read, 1.2 GB
// written, 5.7 TB/s). 93 M elements in 384 tensors, half of them 16-bit, in place: 58 and 93 us.
// 16 tensors of 300000 elements in all: 4 and 5 us, the launches.
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

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kBlocksPerSm = 4;    // at most 64 registers a thread: all resident at once
constexpr int kBlocks = 148 * kBlocksPerSm;
constexpr int kChunk = 16384;        // elements
constexpr int kTable = 900;          // tensors a launch: 32 KB of kernel parameters at most
constexpr int kSmallTable = 64;      // and of a call of few, whose parameters cost less to pass
constexpr float kInfF = __builtin_huge_valf();
constexpr int kUnroll = 4;           // 16-byte loads a thread keeps in flight
constexpr int kSumUnroll = 8;

template <int N>
struct Table {
    int n;
    int chunks;
    const void* src[N];
    void* dst[N];
    long long numel[N];
    int first[N];              // the tensor's first chunk
    uint8_t type[N];           // source type, destination type << 4
};
static_assert(sizeof(Table<kTable>) <= 32000, "kernel parameters");

// the tensor that holds chunk c: the last with first <= c (tensors without elements have none)
template <int N>
__device__ __forceinline__ int find_tensor(const Table<N>& t, int c) {
    int lo = 0, hi = t.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= c) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    return lo;
}

// elements before the first 16-byte boundary
template <typename T>
__device__ __forceinline__ int head_of(const void* p, long long numel) {
    const int off = (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T);
    return numel < off ? (int)numel : off;
}

__device__ __forceinline__ double block_sum(double x) {
    __shared__ double part[kWarps];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, d);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
        part[threadIdx.x >> 5] = x;
    }
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        s += part[w];
    }
    return s;
}

// The sum of a vector's squares: in float32 (three roundings at most on a square's way, 3 2^-24
// relative; bf16's and f16's squares are exact), then widened, one conversion for 4 or 8 elements: a
// conversion each would bound the kernel (300 M bf16 elements 132 us, so 114). A sum that left float32's normal range is taken again in
// float64: squares overflow float32 from 2^64 on and lose bits below 2^-63.
template <typename T>
__device__ __forceinline__ double vector_sumsq(const Raw<T, 16 / (int)sizeof(T)>& r) {
    constexpr int V = 16 / (int)sizeof(T);
    float y[V];
    unpack_raw<T, V>(r, y);
    float s = 0.f;
    if constexpr (V == 8) {
        const float a = fmaf(y[1], y[1], y[0] * y[0]), b = fmaf(y[3], y[3], y[2] * y[2]);
        const float c = fmaf(y[5], y[5], y[4] * y[4]), d = fmaf(y[7], y[7], y[6] * y[6]);
        s = (a + b) + (c + d);
    } else {
        s = fmaf(y[1], y[1], y[0] * y[0]) + fmaf(y[3], y[3], y[2] * y[2]);
    }
    if (s >= 0x1p-90f && s < kInfF) {
        return (double)s;
    }
    double t = 0.0;
#pragma unroll 1
    for (int k = 0; k < V; ++k) {
        float x = y[0];  // a select, not an index into local memory
#pragma unroll
        for (int q = 1; q < V; ++q) {
            x = q == k ? y[q] : x;
        }
        t = fma((double)x, (double)x, t);
    }
    return t;
}

template <typename T>
__device__ __forceinline__ double chunk_sumsq(const T* p, long long numel, int at_chunk) {
    constexpr int V = 16 / (int)sizeof(T);
    const int head = head_of<T>(p, numel);
    const long long body = (numel - head) / V * V;  // whole 16-byte vectors
    // the unaligned ends, fewer than V elements each, with the first chunk
    float end0 = 0.f, end1 = 0.f;
    if (at_chunk == 0 && threadIdx.x < V) {
        const int i = threadIdx.x;
        end0 = i < head ? Elem<T>::to_f(p[i]) : 0.f;
        end1 = i < numel - head - body ? Elem<T>::to_f(p[head + body + i]) : 0.f;
    }
    double acc = 0.0;
    const T* q = p + head;
    const long long b = (long long)at_chunk * kChunk;
    const long long e = b + kChunk < body ? b + kChunk : body;
    for (long long i = b + threadIdx.x * V; i < e; i += (long long)kThreads * V * kSumUnroll) {
        Raw<T, V> v[kSumUnroll];
#pragma unroll
        for (int u = 0; u < kSumUnroll; ++u) {
            const long long j = i + (long long)u * kThreads * V;
            v[u] = load_raw<T, V>(q + (j < e ? j : i));
        }
#pragma unroll
        for (int u = 0; u < kSumUnroll; ++u) {
            if (i + (long long)u * kThreads * V < e) {
                acc += vector_sumsq<T>(v[u]);
            }
        }
    }
    return acc + fma((double)end0, (double)end0, (double)end1 * end1);
}

// The chunks of block `b`: a contiguous range, so that a block looks its first tensor up once.
template <int N>
__device__ __forceinline__ void block_range(const Table<N>& t, int& c0, int& c1) {
    c0 = (int)((long long)t.chunks * blockIdx.x / gridDim.x);
    c1 = (int)((long long)t.chunks * (blockIdx.x + 1) / gridDim.x);
}

template <int N>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    sumsq_kernel(const __grid_constant__ Table<N> t, double* __restrict__ partial) {
    double acc = 0.0;
    int c0, c1;
    block_range(t, c0, c1);
    int i = find_tensor(t, c0);
    for (int c = c0; c < c1; ++c) {
        while (i + 1 < t.n && t.first[i + 1] <= c) {
            ++i;
        }
        const int at = c - t.first[i];
        const int type = t.type[i] & 15;
        const void* p = t.src[i];
        const long long n = t.numel[i];
        acc += type == kF32   ? chunk_sumsq(static_cast<const float*>(p), n, at)
               : type == kF16 ? chunk_sumsq(static_cast<const __half*>(p), n, at)
                              : chunk_sumsq(static_cast<const __nv_bfloat16*>(p), n, at);
    }
    const double s = block_sum(acc);
    if (threadIdx.x == 0) {
        partial[blockIdx.x] = s;
    }
}

// partial[0..n) in a fixed order, the same in every block
__device__ __forceinline__ double sum_partials(const double* partial, int n) {
    double x = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        x += partial[i];
    }
    return block_sum(x);
}

__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    sumsq_final_kernel(const double* __restrict__ partial, int n, double* __restrict__ sumsq) {
    const double s = sum_partials(partial, n);
    if (threadIdx.x == 0) {
        *sumsq = s;
    }
}

template <typename TI, typename TO>
__device__ __forceinline__ void chunk_scale(const TI* p, TO* o, long long numel, int at_chunk,
                                            float by) {
    // vectors of 16 bytes of the wider type, so both sides move whole ones
    constexpr int V = 16 / (int)(sizeof(TI) > sizeof(TO) ? sizeof(TI) : sizeof(TO));
    const int head = head_of<TO>(o, numel);
    // both reach their boundary at the same element, else one element a thread
    const bool vec = (reinterpret_cast<uintptr_t>(p + head) & (sizeof(TI) * V - 1)) == 0;
    const int h = vec ? head : 0;
    const long long body = vec ? (numel - h) / V * V : numel;
    if (at_chunk == 0 && vec) {
        const long long tail = numel - h - body;
        const int i = threadIdx.x;
        if (i < h) {
            o[i] = Elem<TO>::from_f(Elem<TI>::to_f(p[i]) * by);
        }
        if (i < tail) {
            const long long j = h + body + i;
            o[j] = Elem<TO>::from_f(Elem<TI>::to_f(p[j]) * by);
        }
    }
    const TI* q = p + h;
    TO* r = o + h;
    const long long b = (long long)at_chunk * kChunk;
    const long long e = b + kChunk < body ? b + kChunk : body;
    if (vec) {
        for (long long i = b + threadIdx.x * V; i < e; i += (long long)kThreads * V * kUnroll) {
            Raw<TI, V> v[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const long long j = i + (long long)u * kThreads * V;
                v[u] = load_raw<TI, V>(q + (j < e ? j : i));
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const long long j = i + (long long)u * kThreads * V;
                if (j < e) {
                    float y[V];
                    unpack_raw<TI, V>(v[u], y);
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        y[k] *= by;
                    }
                    store_vec<TO, V>(r + j, y);
                }
            }
        }
    } else {
        for (long long i = b + threadIdx.x; i < e; i += kThreads) {
            r[i] = Elem<TO>::from_f(Elem<TI>::to_f(q[i]) * by);
        }
    }
}

// `partial`: the sums of cflk_grad_clip's first launch, or one sumsq (n 1).
template <int N>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    clip_kernel(const __grid_constant__ Table<N> t, const double* __restrict__ partial, int n,
                float max_norm, float eps, float scale, float* __restrict__ norm_out) {
    const double sumsq = sum_partials(partial, n);
    const float norm = (float)(sqrt(sumsq) * fabs((double)scale));
    // a NaN norm stays a NaN factor
    const float ratio = max_norm / (norm + eps);
    const float by = (ratio >= 1.f ? 1.f : ratio) * scale;
    if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out != nullptr) {
        *norm_out = norm;
    }
    // backwards: what the norm's kernel read last is what L2 still holds
    int c0, c1;
    block_range(t, c0, c1);
    int i = c1 > c0 ? find_tensor(t, c1 - 1) : 0;
    for (int c = c1 - 1; c >= c0; --c) {
        while (t.first[i] > c) {
            --i;
        }
        const int at = c - t.first[i];
        const int ti = t.type[i] & 15, to = t.type[i] >> 4;
        const long long m = t.numel[i];
        if (by == 1.f && t.src[i] == t.dst[i]) {
            continue;  // in place and nothing to change
        }
        if (ti == kF32) {
            chunk_scale(static_cast<const float*>(t.src[i]), static_cast<float*>(t.dst[i]), m, at,
                        by);
        } else if (ti == kF16) {
            const __half* p = static_cast<const __half*>(t.src[i]);
            if (to == kF32) {
                chunk_scale(p, static_cast<float*>(t.dst[i]), m, at, by);
            } else {
                chunk_scale(p, static_cast<__half*>(t.dst[i]), m, at, by);
            }
        } else {
            const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(t.src[i]);
            if (to == kF32) {
                chunk_scale(p, static_cast<float*>(t.dst[i]), m, at, by);
            } else {
                chunk_scale(p, static_cast<__nv_bfloat16*>(t.dst[i]), m, at, by);
            }
        }
    }
}

// the tensors from `at` on that one launch takes; the index after them
template <int N>
int64_t fill_table(Table<N>& t, int64_t at, int64_t n, const void* const* src, void* const* dst,
                   const int64_t* numel, const int* src_dtype, const int* dst_dtype) {
    t.n = 0;
    t.chunks = 0;
    for (; at < n && t.n < N; ++at) {
        if (numel[at] == 0) {
            continue;
        }
        const int64_t c = (numel[at] + kChunk - 1) / kChunk;
        const int i = t.n++;
        t.src[i] = src[at];
        t.dst[i] = dst != nullptr ? dst[at] : nullptr;
        t.numel[i] = numel[at];
        t.first[i] = t.chunks;
        t.type[i] = (uint8_t)(src_dtype[at] | (dst_dtype != nullptr ? dst_dtype[at] << 4 : 0));
        t.chunks += (int)c;
    }
    return at;
}

int check_tensors(const char* who, int64_t n, const void* const* src, void* const* dst,
                  bool with_dst, const int64_t* numel, const int* src_dtype,
                  const int* dst_dtype) {
    const auto bad = [&](const char* what) {
        return fail(kInvalidArgument, std::string(who) + ": " + what);
    };
    if (n < 0) {
        return bad("the number of tensors must be non-negative");
    }
    if (n > 0 && (src == nullptr || numel == nullptr || src_dtype == nullptr ||
                  (with_dst && (dst == nullptr || dst_dtype == nullptr)))) {
        return bad("null table");
    }
    const auto known = [](int d) { return d == kF16 || d == kBF16 || d == kF32; };
    int64_t chunks = 0;  // a launch counts them in 32 bits, and the workspace the launches by n
    for (int64_t i = 0; i < n; ++i) {
        if (numel[i] < 0 || numel[i] >= (int64_t(1) << 44)) {
            return bad("a tensor's elements must be non-negative and below 2^44");
        }
        if (!known(src_dtype[i]) ||
            (with_dst && dst_dtype[i] != src_dtype[i] && dst_dtype[i] != kF32)) {
            return bad("gradients are f16, bf16 or f32, outputs their type or f32");
        }
        if (numel[i] == 0) {
            continue;
        }
        chunks += (numel[i] + kChunk - 1) / kChunk;
        if (chunks >= (int64_t(1) << 31)) {
            return bad("the tensors hold 2^45 elements or more together");
        }
        const size_t es = src_dtype[i] == kF32 ? 4 : 2;
        if (src[i] == nullptr || reinterpret_cast<uintptr_t>(src[i]) % es != 0) {
            return bad("a tensor's pointer is null or not aligned to its type");
        }
        if (with_dst) {
            const size_t ed = dst_dtype[i] == kF32 ? 4 : 2;
            if (dst[i] == nullptr || reinterpret_cast<uintptr_t>(dst[i]) % ed != 0) {
                return bad("a tensor's pointer is null or not aligned to its type");
            }
            // in place each element is read and written by one thread; otherwise nothing orders them
            const uintptr_t a = reinterpret_cast<uintptr_t>(src[i]);
            const uintptr_t b = reinterpret_cast<uintptr_t>(dst[i]);
            const size_t m = (size_t)numel[i];
            if ((a != b || es != ed) && a < b + m * ed && b < a + m * es) {
                return bad("an output overlaps its gradient without being it");
            }
        }
    }
    return kOk;
}

// The launches of the sum; their number of partials in `parts`.
template <int N>
cudaError_t launch_sumsq(cudaStream_t s, int64_t n, const void* const* grads,
                         const int64_t* numel, const int* dtypes, double* partial, int& parts) {
    parts = 0;
    Table<N> t;
    for (int64_t at = 0; at < n;) {
        at = fill_table(t, at, n, grads, nullptr, numel, dtypes, nullptr);
        if (t.n == 0) {
            break;
        }
        const int grid = std::min(t.chunks, kBlocks);
        sumsq_kernel<<<grid, kThreads, 0, s>>>(t, partial + parts);
        parts += grid;
    }
    return cudaGetLastError();
}

template <int N>
cudaError_t launch_clip(cudaStream_t s, int64_t n, const void* const* grads, void* const* outs,
                        const int64_t* numel, const int* dtypes, const int* out_dtypes,
                        const double* partial, int parts, float max_norm, float eps, float scale,
                        float* norm) {
    Table<N> t;
    int64_t at = 0;
    do {
        at = fill_table(t, at, n, grads, outs, numel, dtypes, out_dtypes);
        // the first launch writes the norm, even with no tensor to scale
        if (t.n > 0 || norm != nullptr) {
            clip_kernel<<<std::max(1, std::min(t.chunks, kBlocks)), kThreads, 0, s>>>(
                t, partial, parts, max_norm, eps, scale, norm);
        }
        norm = nullptr;
    } while (at < n);
    return cudaGetLastError();
}

}  // namespace
}  // namespace cflk

using namespace cflk;

extern "C" int cflk_grad_workspace_size(int64_t n, size_t* bytes) {
    clear_error();
    if (n < 0 || n >= (int64_t(1) << 40) || bytes == nullptr) {
        return fail(kInvalidArgument, "grad_norm: the number of tensors must be non-negative");
    }
    *bytes = (size_t)std::max<int64_t>(1, (n + kTable - 1) / kTable) * kBlocks * sizeof(double);
    return kOk;
}

namespace {

int check_workspace(const char* who, int64_t n, const void* ws, size_t ws_bytes) {
    size_t need = 0;
    const int rc = cflk_grad_workspace_size(n, &need);
    if (rc != kOk) {
        return rc;
    }
    if (ws == nullptr || ws_bytes < need || reinterpret_cast<uintptr_t>(ws) % 8 != 0) {
        return fail(kInvalidArgument, std::string(who) +
                                          ": workspace below cflk_grad_workspace_size or not "
                                          "8-byte aligned");
    }
    return kOk;
}

}  // namespace

extern "C" int cflk_grad_sumsq(void* stream, int64_t n, const void* const* grads,
                               const int64_t* numel, const int* dtypes, double* sumsq,
                               void* workspace, size_t ws_bytes) {
    clear_error();
    int rc = check_tensors("grad_norm", n, grads, nullptr, false, numel, dtypes, nullptr);
    if (rc != kOk) {
        return rc;
    }
    if (sumsq == nullptr) {
        return fail(kInvalidArgument, "grad_norm: null buffer");
    }
    rc = check_workspace("grad_norm", n, workspace, ws_bytes);
    if (rc != kOk) {
        return rc;
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    double* partial = static_cast<double*>(workspace);
    int parts = 0;
    cudaError_t e = (n <= kSmallTable ? launch_sumsq<kSmallTable> : launch_sumsq<kTable>)(
        s, n, grads, numel, dtypes, partial, parts);
    if (e == cudaSuccess) {
        sumsq_final_kernel<<<1, kThreads, 0, s>>>(partial, parts, sumsq);
        e = cudaGetLastError();
    }
    if (e != cudaSuccess) {
        return fail(kInternal, std::string("grad_norm launch: ") + cudaGetErrorString(e));
    }
    return kOk;
}

extern "C" int cflk_grad_clip(void* stream, int64_t n, const void* const* grads,
                              void* const* outs, const int64_t* numel, const int* dtypes,
                              const int* out_dtypes, const double* sumsq, float max_norm,
                              float eps, float scale, float* norm, void* workspace,
                              size_t ws_bytes) {
    clear_error();
    int rc = check_tensors("grad_clip", n, grads, outs, true, numel, dtypes, out_dtypes);
    if (rc != kOk) {
        return rc;
    }
    if (!(max_norm >= 0.f) || !(eps >= 0.f) || !(scale > 0.f)) {
        return fail(kInvalidArgument,
                    "grad_clip: max_norm and eps must be non-negative, scale positive");
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    const double* partial = sumsq;
    int parts = 1;
    if (sumsq == nullptr) {
        rc = check_workspace("grad_clip", n, workspace, ws_bytes);
        if (rc != kOk) {
            return rc;
        }
        e = (n <= kSmallTable ? launch_sumsq<kSmallTable> : launch_sumsq<kTable>)(
            s, n, grads, numel, dtypes, static_cast<double*>(workspace), parts);
        partial = static_cast<const double*>(workspace);
    }
    if (e == cudaSuccess) {
        e = (n <= kSmallTable ? launch_clip<kSmallTable> : launch_clip<kTable>)(
            s, n, grads, outs, numel, dtypes, out_dtypes, partial, parts, max_norm, eps,
                        scale, norm);
    }
    if (e != cudaSuccess) {
        return fail(kInternal, std::string("grad_clip launch: ") + cudaGetErrorString(e));
    }
    return kOk;
}
