// Status codes, dtype codes and the last-error message shared by the C-ABI entry points.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <string>

namespace cflk {

// return codes of every entry point (the XLA FFI handler maps them to ffi::Error kinds)
enum Status : int { kOk = 0, kInvalidArgument = 1, kInternal = 2 };
// element type of the 16-bit buffers (kF32 only where an entry point says so)
enum DType : int { kF16 = 0, kBF16 = 1, kF32 = 2 };

constexpr int kMaxDevices = 64;

// record msg as this thread's last error and return code
int fail(int code, const std::string& msg);
void clear_error();

// each translation unit's device status word (bounded waits that gave up), read and cleared
unsigned read_and_clear_status_fwd();
unsigned read_and_clear_status_bwd();
unsigned read_and_clear_status_fused();
unsigned read_and_clear_status_gemm();
unsigned read_and_clear_status_opm();
unsigned read_and_clear_status_xent();
unsigned read_and_clear_status_head();
unsigned read_and_clear_status_few();

// VoltaOpmOuter fused at C = E = 32 (the caller has validated the sizes); the workspace holds
// wT laid out chunk by chunk (F * 2 KB)
int opm_outer_fused(void* stream, int dtype, const void* left, const void* right, const void* wT,
                    void* out, int64_t B, int64_t D, int64_t F, void* workspace,
                    size_t ws_bytes);

// The linear softmax cross entropy of heads of few classes (the caller has validated the buffers):
// whether the sizes fit, its workspace, and the forward or backward
struct HeadCall {
    cudaStream_t stream;
    int dtype, labels_64;
    const void *x, *w, *bias, *labels;
    const float *lse_in, *dloss;
    float *loss, *lse;
    void *dx, *dw, *dbias;
    int64_t T, V, C;
    void* workspace;
};
bool xent_head_fits(int64_t V, int64_t C, bool bwd);
size_t xent_head_workspace(int64_t T, int64_t V, int64_t C, bool bwd);
cudaError_t xent_head(const HeadCall& c, bool bwd, bool& map_ok);
// the forward of a few tokens
bool xent_few_fits(int64_t T);
size_t xent_few_workspace();
cudaError_t xent_few(const HeadCall& c, bool& map_ok);

// VoltaGdp through the tile GEMM (widths the resident-weight row-tile kernel does not take)
int gdp_general(void* stream, int dtype, const void* x, const void* wp, const void* bp,
                const void* wg, const void* bg, const void* mask, void* out, int64_t M,
                int64_t K, int64_t N, int64_t activation);

}  // namespace cflk
