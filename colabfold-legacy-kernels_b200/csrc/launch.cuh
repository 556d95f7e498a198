// A kernel launched behind another of the same call: its blocks are put on the machine while the
// one before it still runs (from the moment all of that one's blocks have begun and called
// begin_next), and start their work when all of it has finished and its writes can be seen (after
// wait_before). That takes the launch and the draining of the kernel before out of a chain's time.
//
// Calls in a stream, us, so / by plain launches: gradient of 16384 tokens of 50001 rows of 1024
// channels (six kernels) 74 / 80, cross entropy of 4095 tokens and 32001 classes and its gradients
// (twelve) 455 / 468, of 4 tokens (two) 17.2 / 18.0. Clipping, whose second kernel finds in L2
// what the first one read, keeps plain launches (384 tensors of 242000 float32 elements 187 / 179,
// 300 M bf16 elements 437 / 414, 0.3 M 8.0 / 7.8): blocks that begin where others end are no
// longer on the SM of the block that read their range.
//
// Such a kernel can be at work while the one before it still writes what it will read, so only the
// caller's own inputs are __restrict__ in it: on memory that a kernel of the call writes, that word
// would let the compiler move accesses above wait_before or load them as data that never changes.
#pragma once

#include <cuda_runtime.h>

namespace cflk {

// First statement of a kernel launched by launch_behind. Without effect in one launched otherwise.
__device__ __forceinline__ void wait_before() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// In a kernel that another of the same call follows.
__device__ __forceinline__ void begin_next() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <typename T>
struct Same {
    using type = T;
};

template <typename... P>
cudaError_t launch_behind(void (*kern)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                          const typename Same<P>::type&... args) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    void* at[] = {const_cast<void*>(static_cast<const void*>(&args))...};
    return cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kern), at);
}

}  // namespace cflk
