// nc_readout.cu -- softmax cross-entropy of a linear readout over a large vocabulary, with
// its gradients, without the (rows, classes) logits in memory.
//
//   z = f w^T + b,  lse_n = log sum_v exp z_nv,  loss_n = lse_n - z_n,label
//   dz = g_n (exp(z - lse) - onehot),  df = dz w,  dw = dz^T f,  db = sum_n dz
//
// The value keeps one running (maximum, sum) per row and block of classes; the gradient
// computes the logits of a block of classes again and multiplies them out while they are
// on chip.
#include <math.h>

#include "nc_common.cuh"
#include "nc_errors.h"
#include "nc_readout.h"

namespace nc {

namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kRowDimChunk = 1024;   // features staged in shared memory at a time
constexpr int kRowTile = 4;          // classes a warp takes together

template <int VEC, typename T>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = to_f32(p[0]);
  } else if constexpr (sizeof(T) == 4) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
  } else {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(q.x << 16), v[1] = __uint_as_float(q.x & 0xffff0000u);
    v[2] = __uint_as_float(q.y << 16), v[3] = __uint_as_float(q.y & 0xffff0000u);
  }
}

template <int VEC, typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    store_as(p, v[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
    uint2 q;
    q.x = *reinterpret_cast<uint32_t*>(&lo);
    q.y = *reinterpret_cast<uint32_t*>(&hi);
    *reinterpret_cast<uint2*>(p) = q;
  }
}

// Logits of the row group [row0, row0 + RN) and the classes [v0, v0 + vb) into
// z[r * vb + v] (no bias); vb is a multiple of kRowWarps * kRowTile.  A warp takes kRowTile classes at a time, its lanes split the
// dimension; the group's features are in shared memory, where one 16-byte read serves
// kRowTile * 4 products.  Rows that are ignored or past the end read as zeros; classes past the end
// repeat the last one and are dropped by the caller.
template <typename T, int RN, int VEC>
__device__ void group_logits(const CeArgs& a, int row0, int v0, int vb, float* hs, float* z) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* f = static_cast<const T*>(a.features);
  const T* w = static_cast<const T*>(a.weight);
  const int chunks = (a.dim + kRowDimChunk - 1) / kRowDimChunk;
  const int pitch = min(a.dim, kRowDimChunk);
  for (int vp = 0; vp < vb; vp += kRowWarps * kRowTile) {
    float acc[kRowTile * RN];
#pragma unroll
    for (int i = 0; i < kRowTile * RN; ++i) acc[i] = 0.f;
    const int vw = vp + warp * kRowTile;
    for (int c = 0; c < chunks; ++c) {
      const int d0 = c * kRowDimChunk, len = min(kRowDimChunk, a.dim - d0);
      if (chunks > 1 || vp == 0) {
        __syncthreads();
        for (int i = tid * VEC; i < RN * len; i += kRowThreads * VEC) {
          const int r = i / len, d = i - r * len, row = row0 + r;
          float v[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[e] = 0.f;
          if (row < a.rows && ce_kept(a, row)) load_vec<VEC>(f + (size_t)row * a.dim + d0 + d, v);
#pragma unroll
          for (int e = 0; e < VEC; ++e) hs[r * pitch + d + e] = v[e];
        }
        __syncthreads();
      }
      const T* wr[kRowTile];
#pragma unroll
      for (int j = 0; j < kRowTile; ++j)
        wr[j] = w + (size_t)min(v0 + vw + j, a.classes - 1) * a.dim + d0;
#pragma unroll 2
      for (int d = lane * VEC; d < len; d += 32 * VEC) {
        float x[kRowTile][VEC];
#pragma unroll
        for (int j = 0; j < kRowTile; ++j) load_vec<VEC>(wr[j] + d, x[j]);
#pragma unroll
        for (int r = 0; r < RN; ++r) {
          float h[VEC];
          load_vec<VEC>(hs + r * pitch + d, h);
#pragma unroll
          for (int j = 0; j < kRowTile; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[j * RN + r] = fmaf(x[j][e], h[e], acc[j * RN + r]);
        }
      }
    }
    int first;
    warp_sums(acc, lane, &first);
#pragma unroll
    for (int i = 0; i < (kRowTile * RN + 31) / 32; ++i) {
      const int k = first + i;
      z[(k % RN) * vb + vw + k / RN] = acc[i];
    }
  }
  __syncthreads();
}

// grid (class blocks, row groups): the block's (maximum, sum) of each row, and the label's
// logit where the block holds it.
template <typename T, int RN, int VEC>
__global__ void __launch_bounds__(kRowThreads) ce_rows_value_kernel(CeArgs a, int vb, int blocks,
                                                                    float2* __restrict__ part,
                                                                    float* __restrict__ zlabel) {
  extern __shared__ __align__(16) float sm[];
  float* hs = sm;
  float* z = sm + RN * min(a.dim, kRowDimChunk);
  const int v0 = blockIdx.x * vb, row0 = blockIdx.y * RN;
  pdl_enter();
  group_logits<T, RN, VEC>(a, row0, v0, vb, hs, z);
  const T* bias = static_cast<const T*>(a.bias);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = min(vb, a.classes - v0);
  for (int r = warp; r < RN && row0 + r < a.rows; r += kRowWarps) {
    const int row = row0 + r, label = a.labels[row];
    float m = -INFINITY;
    for (int v = lane; v < n; v += 32) {
      const float x = z[r * vb + v] + (bias ? to_f32(bias[v0 + v]) : 0.f);
      z[r * vb + v] = x;
      m = fmaxf(m, x);
      if (v0 + v == label) zlabel[row] = x;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float s = 0.f;
    for (int v = lane; v < n; v += 32) {
      const float x = z[r * vb + v];
      s += x == -INFINITY ? 0.f : expf(x - m);
    }
    s = warp_sum(s);
    if (lane == 0) part[(size_t)row * blocks + blockIdx.x] = make_float2(m, s);
  }
}

// One warp per row: the blocks' pairs merged in a fixed order, the row's loss.
__global__ void ce_finish_rows_kernel(CeArgs a, int blocks, const float2* __restrict__ part,
                                      const float* __restrict__ zlabel, float* __restrict__ lse,
                                      float* __restrict__ row_loss) {
  pdl_enter();
  const int row = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= a.rows) return;
  float2 x = make_float2(-INFINITY, 0.f);
  for (int i = lane; i < blocks; i += 32) x = lse_merge(x, part[(size_t)row * blocks + i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float2 y = make_float2(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o));
    x = lse_merge(x, y);
  }
  if (lane != 0) return;
  finish_row(a, row, x, zlabel, lse, row_loss);
}

// One block: the sum or mean of the row losses, in a fixed order.
__global__ void __launch_bounds__(1024) ce_sum_kernel(CeArgs a, const float* __restrict__ row_loss,
                                                      float* __restrict__ loss) {
  pdl_enter();
  __shared__ double red[32];
  const int n = count_kept(a);
  double s = 0.0;
  for (int i = threadIdx.x; i < a.rows; i += blockDim.x) s += row_loss[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t += red[i];
    loss[0] = (float)(a.reduction == NC_REDUCE_MEAN ? t / (double)max(n, 1) : t);
  }
}

// Gradients of one block of classes over all rows.  The logits of each row group are
// computed again and left as p = g_n (exp(z - lse) - onehot) in shared memory; then the
// threads own columns d: dw[v] = sum_n p f[n] (8 classes in registers) and the block's part
// of df[n] = sum_v p w[v] (a row group in registers), written to its own slot.
template <typename T, int RN, int VEC>
__global__ void __launch_bounds__(kRowThreads) ce_rows_grad_kernel(
    CeArgs a, int vb, int slots_per_block, int td, const float* __restrict__ lse,
    const float* __restrict__ g_loss, T* __restrict__ g_weight, T* __restrict__ g_bias,
    float* __restrict__ df_part) {
  extern __shared__ __align__(16) float sm[];
  const int rows_pad = (a.rows + RN - 1) / RN * RN;
  float* p = sm;                          // (rows_pad, vb)
  float* hs = sm + rows_pad * vb;
  const int v0 = blockIdx.x * vb, tid = threadIdx.x;
  const T* bias = static_cast<const T*>(a.bias);
  pdl_enter();
  float scale = 1.f;
  if (a.reduction == NC_REDUCE_MEAN) scale = 1.f / (float)max(count_kept(a), 1);
  for (int row0 = 0; row0 < a.rows; row0 += RN) {
    float* z = p + row0 * vb;
    group_logits<T, RN, VEC>(a, row0, v0, vb, hs, z);
    for (int i = tid; i < RN * vb; i += kRowThreads) {
      const int r = i / vb, v = v0 + i - r * vb, row = row0 + r;
      float x = 0.f;
      if (row < a.rows && v < a.classes && ce_kept(a, row)) {
        const float g = g_loss ? g_loss[a.reduction == NC_REDUCE_NONE ? row : 0] * scale : scale;
        x = z[i] + (bias ? to_f32(bias[v]) : 0.f);
        x = g * (expf(x - lse[row]) - (v == a.labels[row] ? 1.f : 0.f));
      }
      z[i] = x;
    }
    __syncthreads();
  }
  if (g_bias) {
    for (int v = tid; v < vb && v0 + v < a.classes; v += kRowThreads) {
      float s = 0.f;
      for (int n = 0; n < a.rows; ++n) s += p[n * vb + v];
      store_as(g_bias + v0 + v, s);
    }
  }
  const T* f = static_cast<const T*>(a.features);
  const T* w = static_cast<const T*>(a.weight);
  const int nd = (a.dim + VEC - 1) / VEC, dt = tid & (td - 1), vg = tid / td, groups = kRowThreads / td;
  if (g_weight) {
    for (int dv = dt; dv < nd; dv += td) {
      for (int v8 = vg * 8; v8 < vb && v0 + v8 < a.classes; v8 += groups * 8) {
        float acc[8][VEC];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[j][e] = 0.f;
        for (int n = 0; n < a.rows; ++n) {
          if (!ce_kept(a, n)) continue;   // its features may hold anything
          float h[VEC], q[8];
          load_vec<VEC>(f + (size_t)n * a.dim + dv * VEC, h);
          *reinterpret_cast<float4*>(q) = *reinterpret_cast<const float4*>(p + n * vb + v8);
          *reinterpret_cast<float4*>(q + 4) = *reinterpret_cast<const float4*>(p + n * vb + v8 + 4);
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[j][e] = fmaf(q[j], h[e], acc[j][e]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (v0 + v8 + j < a.classes) store_vec<VEC>(g_weight + (size_t)(v0 + v8 + j) * a.dim + dv * VEC, acc[j]);
      }
    }
  }
  if (!df_part || vg >= slots_per_block) return;
  float* out = df_part + ((size_t)blockIdx.x * slots_per_block + vg) * a.rows * a.dim;
  for (int row0 = 0; row0 < a.rows; row0 += RN) {
    for (int dv = dt; dv < nd; dv += td) {
      float acc[RN][VEC];
#pragma unroll
      for (int r = 0; r < RN; ++r)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[r][e] = 0.f;
      for (int v4 = vg * 4; v4 < vb; v4 += slots_per_block * 4) {
        float x[4][VEC];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          load_vec<VEC>(w + (size_t)min(v0 + v4 + j, a.classes - 1) * a.dim + dv * VEC, x[j]);
#pragma unroll
        for (int r = 0; r < RN; ++r) {
          const float4 q = *reinterpret_cast<const float4*>(p + (row0 + r) * vb + v4);
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            acc[r][e] += q.x * x[0][e] + q.y * x[1][e] + q.z * x[2][e] + q.w * x[3][e];
        }
      }
#pragma unroll
      for (int r = 0; r < RN; ++r)
        if (row0 + r < a.rows) store_vec<VEC>(out + (size_t)(row0 + r) * a.dim + dv * VEC, acc[r]);
    }
  }
}

// df: the slots' parts summed in order.
template <typename T>
__global__ void ce_sum_parts_kernel(const float* __restrict__ part, int64_t n, int slots, T* __restrict__ out) {
  pdl_enter();
  const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
#pragma unroll 4
  for (int k = 0; k < slots; ++k) s += part[(size_t)k * n + i];
  store_as(out + i, s);
}

struct RowsPlan {
  int rn, vec, vb, blocks, groups, td, slots;
  size_t smem_value, smem_grad;
};

int pow2_at_least(int x) {
  int p = 1;
  while (p < x) p *= 2;
  return p;
}

// `vec`: elements per load, 4 or 1.  A plan of 1 never has more slots than one of 4.
RowsPlan rows_plan(const nc_linear_ce* d, int vec) {
  RowsPlan r;
  r.rn = d->rows <= 1 ? 1 : d->rows <= 4 ? 4 : d->rows <= 8 ? 8 : 16;
  r.groups = (d->rows + r.rn - 1) / r.rn;
  // two blocks of classes per SM, within the shared memory that the gradient's p takes
  const int rows_pad = r.groups * r.rn;
  const int even = ((d->classes + 295) / 296 + 31) / 32 * 32;
  const int fit = (int)(96 * 1024 / (4 * (size_t)rows_pad)) / 32 * 32;
  r.vb = even < 32 ? 32 : even;
  if (r.vb > 256) r.vb = 256;
  if (r.vb > fit) r.vb = fit < 32 ? 32 : fit;
  r.blocks = (d->classes + r.vb - 1) / r.vb;
  r.vec = vec;
  const int nd = d->dim / r.vec;
  r.td = pow2_at_least(nd < kRowThreads ? nd : kRowThreads);
  const int groups = kRowThreads / r.td, most = r.vb / 4;
  r.slots = groups < most ? groups : most;
  const size_t hs = (size_t)r.rn * (d->dim < kRowDimChunk ? d->dim : kRowDimChunk) * 4;
  r.smem_value = hs + (size_t)r.rn * r.vb * 4;
  r.smem_grad = hs + (size_t)rows_pad * r.vb * 4;
  return r;
}

// Few rows: the row-group kernels, which read the weight once as it is.  From kRowsMost on
// the tensor cores.
constexpr int kRowsMost = 32;
bool on_tensor_cores(const nc_linear_ce* d) { return d->rows > kRowsMost; }

struct CeLayout {
  size_t status, row_loss, part, zlabel, df_part, tc, total;
};

CeLayout ce_layout(const nc_linear_ce* d, bool grad) {
  CeLayout L{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += pad256(bytes);
    return o;
  };
  L.status = take(4);
  if (d->rows > 0) {   // else nothing is launched
    L.row_loss = take((size_t)d->rows * 4);
    if (on_tensor_cores(d)) {
      L.tc = take(ce_tc_bytes(d, grad));
    } else {
      const RowsPlan r = rows_plan(d, d->dim % 4 == 0 ? 4 : 1);
      L.part = take((size_t)d->rows * r.blocks * sizeof(float2));
      L.zlabel = take((size_t)d->rows * 4);
      if (grad) L.df_part = take((size_t)r.blocks * r.slots * d->rows * d->dim * 4);
    }
  }
  L.total = at;
  return L;
}

nc_status check_desc(const nc_linear_ce* d) {
  if (!d) return set_error(NC_ERR_INVALID, "nc_linear_ce descriptor is null");
  if (d->rows < 0 || d->dim < 1 || d->classes < 1)
    return set_error(NC_ERR_INVALID, "bad readout shape (rows %d, dim %d, classes %d)", d->rows, d->dim, d->classes);
  if (d->dtype != NC_F32 && d->dtype != NC_BF16) return set_error(NC_ERR_INVALID, "unknown dtype %d", d->dtype);
  if (d->reduction < NC_REDUCE_MEAN || d->reduction > NC_REDUCE_NONE)
    return set_error(NC_ERR_INVALID, "unknown reduction %d", d->reduction);
  if (d->ignore_index >= 0 && d->ignore_index < d->classes)
    return set_error(NC_ERR_INVALID, "ignore_index %d is one of the %d classes", d->ignore_index, d->classes);
  return NC_OK;
}

// Pointers of elements of the call's type: not null, on an element's boundary.
nc_status check_elems(const nc_linear_ce* d, const void* p, const char* name) {
  if (!p) return set_error(NC_ERR_INVALID, "%s is null", name);
  const size_t size = d->dtype == NC_BF16 ? 2 : 4;
  if (reinterpret_cast<uintptr_t>(p) % size != 0)
    return set_error(NC_ERR_INVALID, "%s is not %zu-byte aligned", name, size);
  return NC_OK;
}

nc_status check_ws(const void* ws, size_t have, size_t need) {
  if (!ws || reinterpret_cast<uintptr_t>(ws) % 256 != 0)
    return set_error(NC_ERR_WORKSPACE, "workspace is null or not 256-byte aligned");
  if (have < need) return set_error(NC_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", have, need);
  return NC_OK;
}

CeArgs make_args(const nc_linear_ce* d, const void* f, const void* w, const void* b, const int32_t* labels) {
  CeArgs a;
  a.features = f, a.weight = w, a.bias = b, a.labels = labels;
  a.rows = d->rows, a.dim = d->dim, a.classes = d->classes;
  a.ignore_index = d->ignore_index, a.reduction = d->reduction;
  return a;
}

template <typename K>
nc_status allow_smem(K kernel, size_t bytes) {
  if (bytes > 48 * 1024)
    NC_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  return NC_OK;
}

template <typename T, int RN, int VEC>
nc_status launch_rows_value(const CeArgs& a, const RowsPlan& r, float2* part, float* zlabel, cudaStream_t st) {
  auto k = ce_rows_value_kernel<T, RN, VEC>;
  NC_CHECK(allow_smem(k, r.smem_value));
  PdlLaunch l(dim3(r.blocks, r.groups), dim3(kRowThreads), r.smem_value, st);
  NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, k, a, r.vb, r.blocks, part, zlabel));
  return launch_check("ce_rows_value_kernel launch");
}

template <typename T, int RN, int VEC>
nc_status launch_rows_grad(const CeArgs& a, const RowsPlan& r, const float* lse, const float* g_loss, void* gw,
                           void* gb, float* df_part, cudaStream_t st) {
  auto k = ce_rows_grad_kernel<T, RN, VEC>;
  NC_CHECK(allow_smem(k, r.smem_grad));
  PdlLaunch l(dim3(r.blocks), dim3(kRowThreads), r.smem_grad, st);
  NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, k, a, r.vb, r.slots, r.td, lse, g_loss, static_cast<T*>(gw),
                                   static_cast<T*>(gb), df_part));
  return launch_check("ce_rows_grad_kernel launch");
}

// Calls fn<T, RN, VEC>::run for the call's element type, row group and vector width.
#define NC_ROWS_DISPATCH(FN, ...)                                                     \
  do {                                                                                \
    if (bf16) {                                                                       \
      if (r.vec == 4) {                                                               \
        return r.rn == 1   ? FN<__nv_bfloat16, 1, 4>(__VA_ARGS__)                     \
               : r.rn == 4 ? FN<__nv_bfloat16, 4, 4>(__VA_ARGS__)                     \
               : r.rn == 8 ? FN<__nv_bfloat16, 8, 4>(__VA_ARGS__)                     \
                           : FN<__nv_bfloat16, 16, 4>(__VA_ARGS__);                   \
      }                                                                               \
      return r.rn == 1   ? FN<__nv_bfloat16, 1, 1>(__VA_ARGS__)                       \
             : r.rn == 4 ? FN<__nv_bfloat16, 4, 1>(__VA_ARGS__)                       \
             : r.rn == 8 ? FN<__nv_bfloat16, 8, 1>(__VA_ARGS__)                       \
                         : FN<__nv_bfloat16, 16, 1>(__VA_ARGS__);                     \
    }                                                                                 \
    if (r.vec == 4) {                                                                 \
      return r.rn == 1   ? FN<float, 1, 4>(__VA_ARGS__)                               \
             : r.rn == 4 ? FN<float, 4, 4>(__VA_ARGS__)                               \
             : r.rn == 8 ? FN<float, 8, 4>(__VA_ARGS__)                               \
                         : FN<float, 16, 4>(__VA_ARGS__);                             \
    }                                                                                 \
    return r.rn == 1   ? FN<float, 1, 1>(__VA_ARGS__)                                 \
           : r.rn == 4 ? FN<float, 4, 1>(__VA_ARGS__)                                 \
           : r.rn == 8 ? FN<float, 8, 1>(__VA_ARGS__)                                 \
                       : FN<float, 16, 1>(__VA_ARGS__);                               \
  } while (0)

nc_status rows_value(bool bf16, const CeArgs& a, const RowsPlan& r, float2* part, float* zlabel, cudaStream_t st) {
  NC_ROWS_DISPATCH(launch_rows_value, a, r, part, zlabel, st);
}

nc_status rows_grad(bool bf16, const CeArgs& a, const RowsPlan& r, const float* lse, const float* g_loss, void* gw,
                    void* gb, float* df_part, cudaStream_t st) {
  NC_ROWS_DISPATCH(launch_rows_grad, a, r, lse, g_loss, gw, gb, df_part, st);
}

// Vector loads need rows and base addresses on multiples of four elements.
int vec_of(const nc_linear_ce* d, const void* p, const void* q, const void* out) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out);
  return d->dim % 4 == 0 && at % (d->dtype == NC_BF16 ? 8 : 16) == 0 ? 4 : 1;
}

// lse and row losses, then the reduced loss.  `grad`: the layout of the workspace.
nc_status value(const nc_linear_ce* d, const CeArgs& a, bool grad, float* loss, float* lse, char* ws, cudaStream_t st) {
  const CeLayout L = ce_layout(d, grad);
  const bool none = d->reduction == NC_REDUCE_NONE;
  float* row_loss = none ? loss : reinterpret_cast<float*>(ws + L.row_loss);
  if (on_tensor_cores(d)) return ce_tc_value(d, a, grad, lse, row_loss, none ? nullptr : loss, ws + L.tc, st);
  {
    const RowsPlan r = rows_plan(d, vec_of(d, a.features, a.weight, nullptr));
    float2* part = reinterpret_cast<float2*>(ws + L.part);
    float* zlabel = reinterpret_cast<float*>(ws + L.zlabel);
    NC_CHECK(rows_value(d->dtype == NC_BF16, a, r, part, zlabel, st));
    PdlLaunch l(dim3((d->rows + 3) / 4), dim3(128), 0, st);
    NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ce_finish_rows_kernel, a, r.blocks, (const float2*)part,
                                     (const float*)zlabel, lse, row_loss));
    NC_CHECK(launch_check("ce_finish_rows_kernel launch"));
  }
  if (none) return NC_OK;
  PdlLaunch l(dim3(1), dim3(1024), 0, st);
  NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ce_sum_kernel, a, (const float*)row_loss, loss));
  return launch_check("ce_sum_kernel launch");
}

nc_status gradients(const nc_linear_ce* d, const CeArgs& a, const CeGrads& g, char* ws, cudaStream_t st) {
  const CeLayout L = ce_layout(d, true);
  if (on_tensor_cores(d)) return ce_tc_grad(d, a, g, ws + L.tc, st);
  const bool bf16 = d->dtype == NC_BF16;
  const RowsPlan r = rows_plan(d, vec_of(d, a.features, a.weight, g.weight));
  float* df_part = g.features ? reinterpret_cast<float*>(ws + L.df_part) : nullptr;
  NC_CHECK(rows_grad(bf16, a, r, g.lse, g.g_loss, g.weight, g.bias, df_part, st));
  if (!g.features) return NC_OK;
  const int64_t n = (int64_t)d->rows * d->dim;
  PdlLaunch l(dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st);
  const int slots = r.blocks * r.slots;
  if (bf16)
    NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ce_sum_parts_kernel<__nv_bfloat16>, (const float*)df_part, n, slots,
                                     static_cast<__nv_bfloat16*>(g.features)));
  else
    NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ce_sum_parts_kernel<float>, (const float*)df_part, n, slots,
                                     static_cast<float*>(g.features)));
  return launch_check("ce_sum_parts_kernel launch");
}

nc_status check_inputs(const nc_linear_ce* d, const void* features, const void* weight, const void* bias,
                       const int32_t* labels, const float* lse) {
  NC_CHECK(check_elems(d, features, "features"));
  NC_CHECK(check_elems(d, weight, "weight"));
  if (bias) NC_CHECK(check_elems(d, bias, "bias"));
  NC_CHECK(check_ptr(labels, "labels"));
  return check_ptr(lse, "lse");
}

nc_status check_grads(const nc_linear_ce* d, const void* g_features, const void* g_weight, const void* g_bias) {
  if (g_features) NC_CHECK(check_elems(d, g_features, "g_features"));
  if (g_weight) NC_CHECK(check_elems(d, g_weight, "g_weight"));
  if (g_bias) NC_CHECK(check_elems(d, g_bias, "g_bias"));
  return NC_OK;
}

// No rows: a loss of 0 and gradients of 0.
nc_status no_rows(const nc_linear_ce* d, float* loss, void* g_weight, void* g_bias, cudaStream_t st) {
  const size_t size = d->dtype == NC_BF16 ? 2 : 4;
  if (loss && d->reduction != NC_REDUCE_NONE) NC_CUDA_CHECK(cudaMemsetAsync(loss, 0, 4, st));
  if (g_weight) NC_CUDA_CHECK(cudaMemsetAsync(g_weight, 0, (size_t)d->classes * d->dim * size, st));
  if (g_bias) NC_CUDA_CHECK(cudaMemsetAsync(g_bias, 0, (size_t)d->classes * size, st));
  clear_error();
  return NC_OK;
}

}  // namespace

}  // namespace nc

using namespace nc;

extern "C" {

size_t nc_linear_ce_workspace_bytes(const nc_linear_ce* desc, int32_t grad) {
  if (check_desc(desc) != NC_OK) return 0;
  return ce_layout(desc, grad != 0).total;
}

nc_status nc_linear_ce_forward(const nc_linear_ce* desc, const void* features, const void* weight,
                               const void* bias, const int32_t* labels, float* loss, float* lse, void* d_ws,
                               size_t ws_bytes, void* stream) {
  NC_CHECK(check_desc(desc));
  NC_CHECK(check_ptr(loss, "loss"));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (desc->rows == 0) return no_rows(desc, loss, nullptr, nullptr, st);
  NC_CHECK(check_inputs(desc, features, weight, bias, labels, lse));
  NC_CHECK(check_ws(d_ws, ws_bytes, ce_layout(desc, false).total));
  char* ws = static_cast<char*>(d_ws);
  const CeArgs a = make_args(desc, features, weight, bias, labels);
  if (on_tensor_cores(desc)) NC_CHECK(ce_tc_prepare(desc, a, false, nullptr, ws + ce_layout(desc, false).tc, st));
  NC_CHECK(value(desc, a, false, loss, lse, ws, st));
  clear_error();
  return NC_OK;
}

nc_status nc_linear_ce_backward(const nc_linear_ce* desc, const void* features, const void* weight,
                                const void* bias, const int32_t* labels, const float* lse, const float* g_loss,
                                void* g_features, void* g_weight, void* g_bias, void* d_ws, size_t ws_bytes,
                                void* stream) {
  NC_CHECK(check_desc(desc));
  NC_CHECK(check_grads(desc, g_features, g_weight, g_bias));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (desc->rows == 0) return no_rows(desc, nullptr, g_weight, g_bias, st);
  NC_CHECK(check_inputs(desc, features, weight, bias, labels, lse));
  if (g_loss) NC_CHECK(check_ptr(g_loss, "g_loss"));
  NC_CHECK(check_ws(d_ws, ws_bytes, ce_layout(desc, true).total));
  char* ws = static_cast<char*>(d_ws);
  const CeArgs a = make_args(desc, features, weight, bias, labels);
  if (on_tensor_cores(desc)) NC_CHECK(ce_tc_prepare(desc, a, true, g_loss, ws + ce_layout(desc, true).tc, st));
  const CeGrads g{lse, g_loss, g_features, g_weight, g_bias};
  NC_CHECK(gradients(desc, a, g, ws, st));
  clear_error();
  return NC_OK;
}

nc_status nc_linear_ce_value_and_grad(const nc_linear_ce* desc, const void* features, const void* weight,
                                      const void* bias, const int32_t* labels, float* loss, float* lse,
                                      void* g_features, void* g_weight, void* g_bias, void* d_ws, size_t ws_bytes,
                                      void* stream) {
  NC_CHECK(check_desc(desc));
  NC_CHECK(check_ptr(loss, "loss"));
  NC_CHECK(check_grads(desc, g_features, g_weight, g_bias));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (desc->rows == 0) return no_rows(desc, loss, g_weight, g_bias, st);
  NC_CHECK(check_inputs(desc, features, weight, bias, labels, lse));
  NC_CHECK(check_ws(d_ws, ws_bytes, ce_layout(desc, true).total));
  char* ws = static_cast<char*>(d_ws);
  const CeArgs a = make_args(desc, features, weight, bias, labels);
  if (on_tensor_cores(desc)) NC_CHECK(ce_tc_prepare(desc, a, true, nullptr, ws + ce_layout(desc, true).tc, st));
  NC_CHECK(value(desc, a, true, loss, lse, ws, st));
  const CeGrads g{lse, nullptr, g_features, g_weight, g_bias};
  NC_CHECK(gradients(desc, a, g, ws, st));
  clear_error();
  return NC_OK;
}

}  // extern "C"
