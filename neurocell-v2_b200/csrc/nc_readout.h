// nc_readout.h -- workspace layout and kernels of the linear readout's cross-entropy.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "neurocell_b200.h"

namespace nc {

// What the kernels of one call read.  `features` (rows, dim), `weight` (classes, dim) and
// `bias` (classes, may be null) hold the call's element type.
struct CeArgs {
  const void* features;
  const void* weight;
  const void* bias;
  const int32_t* labels;
  int rows, dim, classes;
  int ignore_index;
  int reduction;
};

// A row that takes part: every label but ignore_index.  A label outside [0, classes) takes
// part with a NaN log-sum-exp, so that its loss and the gradients read NaN.
__device__ __forceinline__ bool ce_kept(const CeArgs& a, int row) {
  return a.labels[row] != a.ignore_index;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void store_as(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_as(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

}  // namespace nc
