// Host-side helpers shared by the entry points that live beside their kernels (defined in api.cu).
#pragma once
#include <cstdio>
#include <cuda.h>
#include <cuda_runtime.h>

#include "cuda_llm_b200.h"

namespace b200 {

void set_error_message(const char* msg);
int check_current_device();  // CUDA_LLM_OK on an sm_100 device
int current_sm_count();

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn tensor_map_encoder();

inline int refuse(int code, const char* msg) {
  set_error_message(msg);
  return code;
}
inline int cuda_result(cudaError_t e, const char* where) {
  if (e == cudaSuccess) return CUDA_LLM_OK;
  char msg[192];
  snprintf(msg, sizeof(msg), "%s: %s", where, cudaGetErrorString(e));
  set_error_message(msg);
  return CUDA_LLM_ECUDA;
}

// Whether no two of the rows [n0][n1] of `width` elements, addressed by two strides, share an element.
inline bool rows_apart(long long st0, long long n0, long long st1, long long n1, long long width) {
  if (n0 <= 1) return n1 <= 1 || st1 >= width;
  if (n1 <= 1) return st0 >= width;
  const bool first = st0 <= st1;  // which index steps over the shorter distance
  return first ? st0 >= width && st1 >= st0 * (n0 - 1) + width : st1 >= width && st0 >= st1 * (n1 - 1) + width;
}

// Raises a kernel's dynamic shared memory limit once per device (`configured`: a static array of 64 of the caller).
inline cudaError_t allow_shared_memory(const void* kern, int bytes, int* configured) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && configured[dev])) return e;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) configured[dev] = 1;
  return e;
}

}  // namespace b200
