// overlap.cuh -- launches whose blocks are set up while the kernel before them in
// the stream ends. Such a kernel calls prior_kernels_done() in every thread before it
// touches global memory: until then the writes of earlier kernels may be missing, and
// memory that they read may not be written. Its loads are plain ones: a read-only load
// (__ldg, a __restrict__ pointer to const) says that the data does not change while the
// kernel runs, which is not so before the wait, and the compiler may move it ahead.
// What the kernels before the one before wrote may be read without the wait, if every
// block of the kernel before has waited in its turn (merge_kernel in decode_q8.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace ann {

__device__ __forceinline__ void prior_kernels_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A load that stays behind prior_kernels_done() (both are volatile) and that ordinary
// stores before it in the program do not hold up: for inputs that the kernel does not write.
__device__ __forceinline__ uint32_t load_input(uint32_t const* p) {
    uint32_t v;
    asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ float load_input(float const* p) {
    return __uint_as_float(load_input(reinterpret_cast<uint32_t const*>(p)));
}

inline cudaLaunchAttribute overlapping() {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    return attr;
}

// One such launch; the error, if any, is the thread's last one.
template <typename... P, typename... A>
void launch_overlapping(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream, A... args) {
    cudaLaunchAttribute attr = overlapping();
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

}  // namespace ann
