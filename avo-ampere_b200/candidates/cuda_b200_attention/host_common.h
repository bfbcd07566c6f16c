// Host-side helpers of the library's translation units (defined in attn_abi.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace avo_b200 {
namespace host {

// Pipeline-wait limit of the kernels in nanoseconds (AVO_B200_WATCHDOG_MS).
unsigned long long watchdog_limit();
// Test hook AVO_B200_TEST_SKIP_LOAD: the copy each CTA's producer leaves out, or -1.
int skip_load();
// AVO_B200_OK if the current device is a B200 (checked once per device); its SM count.
int device(int* sm_count);
// TMA map of a contiguous bf16 [heads, rows, 128] tensor: boxes of 64 columns x 128 rows,
// 128-byte swizzle, rows past the end read as zero.
int encode(CUtensorMap* map, const void* base, int rows, int heads);

inline bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// A launch that may start while the previous work in its stream finishes (programmatic
// dependent launch): the kernel waits with griddepcontrol.wait before it touches global
// memory, or, where it reads nothing that the previous kernel writes, before it ends.
template <typename... Params, typename... Args>
bool launch_early(void (*kernel)(Params...), unsigned grid, unsigned threads, size_t smem, cudaStream_t stream,
                  Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, static_cast<Args&&>(args)...) == cudaSuccess) return true;
  (void)cudaGetLastError();
  return false;
}

}  // namespace host
}  // namespace avo_b200
