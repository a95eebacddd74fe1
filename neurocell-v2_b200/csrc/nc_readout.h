// nc_readout.h -- workspace layout and kernels of the linear readout's cross-entropy.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
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
  int32_t* status;   // the workspace's status word (nc_workspace_status)
};

// What the gradient kernels read of the loss's own gradient, and where the results go.
struct CeGrads {
  const float* lse;
  const float* g_loss;
  void* features;
  void* weight;
  void* bias;
};

// The tensor-core path (nc_readout_tc.cu).  `ws` bytes from ce_tc_bytes; prepare() first.
size_t ce_tc_bytes(const nc_linear_ce* d, bool grad);
// `grad`: the workspace is one of a gradient.  g_loss: the loss's own gradient, or null for 1.
nc_status ce_tc_prepare(const nc_linear_ce* d, const CeArgs& a, bool grad, const float* g_loss, char* ws,
                        cudaStream_t st);
// lse and row losses (rows), and their sum or mean into `loss` unless that is null.
nc_status ce_tc_value(const nc_linear_ce* d, const CeArgs& a, bool grad, float* lse, float* row_loss, float* loss,
                      char* ws, cudaStream_t st);
nc_status ce_tc_grad(const nc_linear_ce* d, const CeArgs& a, const CeGrads& g, char* ws, cudaStream_t st);

inline size_t pad256(size_t n) { return (n + 255) / 256 * 256; }

// A row that takes part: every label but ignore_index.  A label outside [0, classes) takes
// part with a NaN log-sum-exp, so that its loss and the gradients read NaN.
__device__ __forceinline__ bool ce_kept(const CeArgs& a, int row) {
  return a.labels[row] != a.ignore_index;
}

// Running (maximum, sum of exp) merges.  A maximum of -inf carries a sum of 0, or NaN when
// a NaN was seen.
__device__ __forceinline__ float2 lse_merge(float2 x, float2 y) {
  const float m = fmaxf(x.x, y.x);
  const float sx = x.x == -INFINITY ? x.y : x.y * expf(x.x - m);
  const float sy = y.x == -INFINITY ? y.y : y.y * expf(y.x - m);
  return make_float2(m, sx + sy);
}

// A row's log-sum-exp and loss from the merged pair.  The loss is not taken from the log-sum-exp:
// rounded to float32 that has lost what the other classes add to a large logit.  The gradients do
// go by the log-sum-exp, which is NaN where its rounding would put them off by more than an eighth (and
// where no class is left).  Labels outside the classes, other than ignore_index, make both NaN.
__device__ __forceinline__ void finish_row(const CeArgs& a, int row, float2 x, const float* zlabel, float* lse,
                                           float* row_loss) {
  const int label = a.labels[row];
  const bool in = label >= 0 && label < a.classes;
  const float l = logf(x.y);
  const float sum = x.x + l;
  lse[row] = in && fabsf((sum - x.x) - l) <= 0.125f ? sum : NAN;
  row_loss[row] = label == a.ignore_index ? 0.f : in ? x.x - zlabel[row] + l : NAN;
}

// Rows that take part, counted by a whole block (every thread gets the count).
__device__ __forceinline__ int count_kept(const CeArgs& a) {
  __shared__ int total;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  int n = 0;
  for (int i = threadIdx.x; i < a.rows; i += blockDim.x) n += ce_kept(a, i);
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) atomicAdd(&total, n);
  __syncthreads();
  return total;
}

// Sums v[i] over the lanes.  Each step halves the values a lane keeps while more than one
// is left, so 64 values take 62 shuffles instead of 320; afterwards a lane holds
// max(1, N / 32) sums, from value *first on (equal on the lanes that share it).
template <int N>
__device__ __forceinline__ void warp_sums(float (&v)[N], int lane, int* first) {
  int n = N, at = 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (i < n) {
          const float send = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
      }
      at += up ? n : 0;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
  *first = at;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void store_as(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_as(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

}  // namespace nc
