// Launch helpers: the counter shared by all host wrappers (defined in
// gemm_tcgen05.cu) and launches that overlap their set-up with the kernel before.
#pragma once

namespace h3 {

void note_launch();

#ifdef __CUDACC__
// A kernel launched this way may be resident before the stream's previous
// kernel has ended; it must call wait_for_prior() in every thread before it
// touches memory that earlier work reads or writes.  The set-up before that call
// (barriers, TMEM, the work list) then costs nothing between kernels.
template <typename... P, typename... A>
inline void launch_overlapped(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                              A&&... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = 1;
  cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);
}

// Returns once all earlier work of the stream is complete and visible.
__device__ __forceinline__ void wait_for_prior() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
#endif

}  // namespace h3
