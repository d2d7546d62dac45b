// Launches that may begin before the kernel ahead of them in the stream has ended
// (programmatic dependent launch): the launch itself, and whatever a kernel does before
// pdl_wait() (ptx.cuh), overlap that kernel's end. Every kernel launched so calls pdl_wait()
// before its first access to global memory that another kernel may write or still read.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>

#include <initializer_list>

namespace da3b {

// cluster: CTAs a cluster along x (1: none). A launch that fails leaves no error behind for
// cudaGetLastError, which the next call would take for its own.
template <typename... Params, typename... Args>
cudaError_t launch_pdl(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s,
                       unsigned cluster, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
  if (e != cudaSuccess) cudaGetLastError();
  return e;
}

// Whether kernels can use these buffers: memory of the current device, or managed or pinned
// memory (null is passed over). Anything else (pageable host memory, another device's) would
// fault in the kernel instead of failing here. Asked of the driver, which answers for one
// attribute in 40 ns, a fraction of the time that the runtime's query of all of them takes.
bool usable_here(std::initializer_list<const void*> buffers);

// Multiprocessors of a device (asked once).
int sm_count(int dev);

// Largest count of rows or columns: rounding up to a tile stays inside 32 bits.
constexpr int kMostCount = 0x7fffff00;

}  // namespace da3b
