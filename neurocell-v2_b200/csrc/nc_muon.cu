// nc_muon.cu -- orthogonalisation of matrices by Newton-Schulz products, and the update of
// parameters by orthogonalised momentum.
//
//   X0 = x / (|x|_F + eps);  steps times: A = X X^T, X <- a X + (b A + c A^2) X
//
// on the short side (A = X^T X, X <- a X + X (b A + c A^2) when rows > cols).  Every
// singular value s of x goes through s <- a s + b s^3 + c s^5; the singular vectors stay.
// The norm is summed in float64: the iteration magnifies an error of the scale of X0 up to
// about a hundred times.
#include <cooperative_groups.h>
#include <math.h>

#include "nc_common.cuh"
#include "nc_errors.h"
#include "nc_readout.h"
#include "nc_tc.cuh"

namespace nc {

namespace {

constexpr int kNormThreads = 256;
constexpr int kNormPer = 16;   // elements a thread of the momentum / norm pass takes

struct MuonArgs {
  float beta;
  int nesterov;
};

__device__ __forceinline__ double block_sum_f64(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t += red[i];
  return t;
}

// grid (blocks, batch).  Sum of squares of x per block; with `momentum`: m = beta m + x,
// and the sum is of u = x + beta m (nesterov) or m, written to `u`.
template <typename T>
__global__ void __launch_bounds__(kNormThreads) ns_norm_kernel(const T* __restrict__ x, float* __restrict__ momentum,
                                                               MuonArgs mu, int64_t n, float* __restrict__ u,
                                                               double* __restrict__ part,
                                                               int32_t* __restrict__ status) {
  __shared__ double red[kNormThreads / 32];
  pdl_enter();
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *status = 0;
  const size_t base = (size_t)blockIdx.y * n;
  const int64_t i0 = (int64_t)blockIdx.x * kNormThreads * kNormPer + threadIdx.x;
  double s = 0.0;
#pragma unroll 4
  for (int k = 0; k < kNormPer; ++k) {
    const int64_t i = i0 + (int64_t)k * kNormThreads;
    if (i >= n) break;
    float v = to_f32(x[base + i]);
    if (momentum) {
      const float m = fmaf(mu.beta, momentum[base + i], v);
      momentum[base + i] = m;
      v = mu.nesterov ? fmaf(mu.beta, m, v) : m;
      u[base + i] = v;
    }
    s += (double)v * v;
  }
  s = block_sum_f64(s, red);
  if (threadIdx.x == 0) part[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = s;
}

// ---- short sides up to 64: one cluster per matrix ------------------------------------------
// The CTAs of a cluster hold slices of the long side in shared memory for all steps, as
// X[l][i] (i along the short side, padded to S).  A step: every CTA adds up its slice's part
// of A = X X^T, the cluster sums the parts (each CTA its share of A, read from and written to
// the others' shared memory), and every CTA updates its slice, Y = A X, X <- a X + b Y + c A Y,
// which needs no other slice and no A^2.  The momentum, the norm and the final update are in
// the same launch, so the cost is the two cluster barriers of a step and the FMAs, 3 S^2 per
// column of a slice.
constexpr int kSmallThreads = 256;
constexpr size_t kSmallSmem = 200 * 1024;

struct SmallArgs {
  const void* x;
  float* momentum;
  float* params;
  void* out;
  int rows, cols, slice;    // slice: columns of the long side per CTA, whole 4s
  int steps;
  float a, b, c;
  double eps;
  MuonArgs mu;
  float decay, step;
  int32_t* status;
};

template <int S>
__host__ __device__ constexpr size_t small_smem(int slice) {
  return (size_t)(2 * slice * (S + 4) + 4096 + S * (S + 4)) * 4;
}

// out[l][i..i+3] for 4 columns l: sum over k of A[k][i] in[l][k].
template <int S>
__device__ __forceinline__ void small_product(const float* A, const float* in, int i, float (&acc)[4][4]) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[q][e] = 0.f;
#pragma unroll 4
  for (int k = 0; k < S; k += 4) {
    float m[4][4], v[4][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) *reinterpret_cast<float4*>(m[e]) = *reinterpret_cast<const float4*>(A + (k + e) * (S + 4) + i);
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<float4*>(v[q]) = *reinterpret_cast<const float4*>(in + q * (S + 4) + k);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[q][r] = fmaf(m[e][r], v[q][e], acc[q][r]);
  }
}

template <int S, typename T>
__global__ void __launch_bounds__(kSmallThreads) ns_small_kernel(SmallArgs p) {
  namespace cg = cooperative_groups;
  constexpr int kPitch = S + 4, kPer = S / 4, kCell = kPer * kPer;   // threads of one S x S product
  constexpr int kGroups = kSmallThreads / kCell;                     // that split the slice's columns
  extern __shared__ __align__(16) float sm[];
  __shared__ double red[kSmallThreads / 32], total;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank(), tid = threadIdx.x;
  float* X = sm;
  float* Y = X + p.slice * kPitch;
  float* part = Y + p.slice * kPitch;   // (kGroups, S, S)
  float* A = part + 4096;               // (S, pitch)
  const bool tall = p.rows > p.cols;
  const int s = tall ? p.cols : p.rows, len = tall ? p.rows : p.cols;
  const int l0 = rank * p.slice;
  const size_t base = (size_t)(blockIdx.x / ranks) * p.rows * p.cols;
  pdl_enter();
  if (blockIdx.x == 0 && tid == 0) *p.status = 0;

  // the source in the order of its memory; momentum in passing
  const T* x = static_cast<const T*>(p.x) + base;
  double sum = 0.0;
  for (int e = tid; e < p.slice * S; e += kSmallThreads) {
    const int l = tall ? e / S : e % p.slice, i = tall ? e % S : e / p.slice;
    float v = 0.f;
    if (i < s && l0 + l < len) {
      const size_t o = tall ? (size_t)(l0 + l) * p.cols + i : (size_t)i * p.cols + l0 + l;
      v = to_f32(x[o]);
      if (p.momentum) {
        const float m = fmaf(p.mu.beta, p.momentum[base + o], v);
        p.momentum[base + o] = m;
        v = p.mu.nesterov ? fmaf(p.mu.beta, m, v) : m;
      }
    }
    X[l * kPitch + i] = v;
    sum += (double)v * v;
  }
  sum = block_sum_f64(sum, red);
  if (tid == 0) total = sum;
  cluster.sync();
  double norm = 0.0;
  for (int r = 0; r < ranks; ++r) norm += *cluster.map_shared_rank(&total, r);
  const double inv = 1.0 / (sqrt(norm) + p.eps);
  for (int e = tid; e < p.slice * S; e += kSmallThreads) {
    const int o = e / S * kPitch + e % S;
    X[o] = (float)((double)X[o] * inv);
  }
  __syncthreads();

  const int cell = tid % kCell, group = tid / kCell;
  const int ti = cell % kPer * 4, tj = cell / kPer * 4;
  const int share = S * S / ranks;   // elements of A that this CTA sums
  for (int step = 0; step < p.steps; ++step) {
    float acc[4][4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[q][e] = 0.f;
#pragma unroll 4
    for (int l = group; l < p.slice; l += kGroups) {
      float u[4], v[4];
      *reinterpret_cast<float4*>(u) = *reinterpret_cast<const float4*>(X + l * kPitch + ti);
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(X + l * kPitch + tj);
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[q][e] = fmaf(v[q], u[e], acc[q][e]);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<float4*>(part + group * S * S + (tj + q) * S + ti) =
          make_float4(acc[q][0], acc[q][1], acc[q][2], acc[q][3]);
    if constexpr (kGroups > 1) {
      __syncthreads();
      for (int e = tid; e < S * S; e += kSmallThreads) {
        float v = part[e];
#pragma unroll
        for (int g = 1; g < kGroups; ++g) v += part[g * S * S + e];
        part[e] = v;
      }
    }
    cluster.sync();
    for (int e = rank * share + tid; e < (rank + 1) * share; e += kSmallThreads) {
      float v = 0.f;
#pragma unroll 8
      for (int r = 0; r < ranks; ++r) v += cluster.map_shared_rank(part, r)[e];
      const int o = e / S * kPitch + e % S;
#pragma unroll 8
      for (int r = 0; r < ranks; ++r) cluster.map_shared_rank(A, r)[o] = v;
    }
    cluster.sync();
    for (int t = tid; t < p.slice / 4 * kPer; t += kSmallThreads) {
      const int i = t % kPer * 4, l = t / kPer * 4;
      small_product<S>(A, X + l * kPitch, i, acc);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<float4*>(Y + (l + q) * kPitch + i) = make_float4(acc[q][0], acc[q][1], acc[q][2], acc[q][3]);
    }
    __syncthreads();
    for (int t = tid; t < p.slice / 4 * kPer; t += kSmallThreads) {
      const int i = t % kPer * 4, l = t / kPer * 4;
      small_product<S>(A, Y + l * kPitch, i, acc);
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int o = (l + q) * kPitch + i + e;
          X[o] = fmaf(p.a, X[o], fmaf(p.b, Y[o], p.c * acc[q][e]));
        }
    }
    __syncthreads();
  }
  T* out = static_cast<T*>(p.out) + base;
  for (int e = tid; e < p.slice * S; e += kSmallThreads) {
    const int l = tall ? e / S : e % p.slice, i = tall ? e % S : e / p.slice;
    if (i >= s || l0 + l >= len) continue;
    const size_t o = tall ? (size_t)(l0 + l) * p.cols + i : (size_t)i * p.cols + l0 + l;
    const float v = X[l * kPitch + i];
    if (p.params)
      p.params[base + o] = p.params[base + o] * p.decay - p.step * v;
    else
      store_as(out + o, v);
  }
  cluster.sync();   // no CTA leaves while another may still read its shared memory
}

// CTAs per cluster and columns per CTA; `fits`: within shared memory.
struct SmallPlan {
  int pad, ranks, slice;
  bool fits;
};

SmallPlan small_plan(const nc_newton_schulz* d) {
  const int s = d->rows < d->cols ? d->rows : d->cols, len = d->rows < d->cols ? d->cols : d->rows;
  SmallPlan r{};
  r.pad = s <= 16 ? 16 : s <= 32 ? 32 : 64;
  r.ranks = len > 28 ? 8 : len > 12 ? 4 : len > 4 ? 2 : 1;
  r.slice = ((len + r.ranks - 1) / r.ranks + 3) / 4 * 4;
  const size_t need = r.pad == 16 ? small_smem<16>(r.slice) : r.pad == 32 ? small_smem<32>(r.slice) : small_smem<64>(r.slice);
  r.fits = s <= 64 && need <= kSmallSmem;
  return r;
}

template <int S, typename T>
nc_status launch_small(const SmallArgs& a, const SmallPlan& r, int batch, cudaStream_t st) {
  auto k = ns_small_kernel<S, T>;
  const size_t smem = small_smem<S>(r.slice);
  NC_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = r.ranks, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(r.ranks * batch), cfg.blockDim = dim3(kSmallThreads);
  cfg.dynamicSmemBytes = smem, cfg.stream = st, cfg.attrs = attr, cfg.numAttrs = 2;
  NC_CUDA_CHECK(cudaLaunchKernelEx(&cfg, k, a));
  return launch_check("ns_small_kernel launch");
}

// ---- products on the tensor cores --------------------------------------------------------
// X, A = X X^T and b A + c A^2 are kept as two float16 planes each (nc_tc.cuh), scaled by
// 2^12: |entries| stay below 16 while the singular values do, and an entry of 2^-26 still has
// its 11 bits in the high plane.
constexpr float kPlaneScale = 4096.f, kPlaneInv = 1.f / 4096.f;

struct Planes {   // (batch, plane, rows, pitch)
  __half* p;
  int pitch;
  int64_t plane;
};

// X0 of one matrix as planes.
template <typename T>
__global__ void __launch_bounds__(kNormThreads) ns_split_kernel(const T* __restrict__ x, int64_t n, int cols, int parts,
                                                                const double* __restrict__ part, double eps,
                                                                Planes out) {
  __shared__ double red[kNormThreads / 32];
  pdl_enter();
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += kNormThreads) s += part[(size_t)blockIdx.y * parts + i];
  s = block_sum_f64(s, red);
  const double inv = 1.0 / (sqrt(s) + eps);
  const size_t base = (size_t)blockIdx.y * n;
  __half* hi = out.p + (size_t)blockIdx.y * 2 * out.plane;
  const int64_t i0 = (int64_t)blockIdx.x * kNormThreads * kNormPer + threadIdx.x;
#pragma unroll 4
  for (int k = 0; k < kNormPer; ++k) {
    const int64_t i = i0 + (int64_t)k * kNormThreads;
    if (i >= n) break;
    const int r = (int)i / cols, c = (int)i - r * cols;
    uint16_t h, l;
    tc::split_f16((float)((double)to_f32(x[base + i]) * inv) * kPlaneScale, &h, &l);
    const size_t o = (size_t)r * out.pitch + c;
    hi[o] = __ushort_as_half(h);
    hi[out.plane + o] = __ushort_as_half(l);
  }
}

enum NsMode { kGram, kPoly, kUpdate, kFinal };

// 16 values of both planes, added up (still scaled).
__device__ __forceinline__ void load_planes(const Planes& s, size_t o, float (&v)[16]) {
  uint32_t h[8], l[8];
  tc::load_v8(s.p + o, h);
  tc::load_v8(s.p + s.plane + o, l);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 a = __half22float2(*reinterpret_cast<__half2*>(&h[i]));
    const float2 b = __half22float2(*reinterpret_cast<__half2*>(&l[i]));
    v[2 * i] = a.x + b.x, v[2 * i + 1] = a.y + b.y;
  }
}

// Epilogue of the three products of a step, on scaled values:
//   gram: A = acc;  poly: b A + c acc;  update: a X + acc;  final: the same, to the caller
template <int MODE, typename T>
struct NsEpilogue {
  Planes src, dst;   // same shape: A for poly, X for update
  int m, n;
  float mul, add;    // value = mul acc + add src
  T* out;            // final: the result (rows, cols), or
  float* params;     // params <- decay params - step result
  float decay, step;
  bool wide;         // rows of out or params start on 32 bytes

  template <int HALF>
  __device__ __forceinline__ int begin(const tc::Tile&, int, int, float*) const {
    return 0;
  }
  template <int HALF>
  __device__ __forceinline__ void run(int, const tc::Tile& x, int row, int col, float (&acc)[HALF]) const {
    if (row >= m) return;
    const size_t base = (size_t)x.batch * 2 * src.plane + (size_t)row * src.pitch;
    const bool mirror = (MODE == kGram || MODE == kPoly) && x.n0 > x.m0;
#pragma unroll
    for (int j = 0; j < HALF; j += 16) {
      if (col + j >= n) break;
      float v[16];
      if constexpr (MODE == kGram) {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = acc[j + e] * mul;
      } else {
        load_planes(src, base + col + j, v);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = fmaf(acc[j + e], mul, v[e] * add);
      }
      if constexpr (MODE == kFinal) {
        const size_t o = ((size_t)x.batch * m + row) * n + col + j;
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] *= kPlaneInv;
        if (params) {
          if (wide && col + j + 16 <= n) {
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
              uint32_t q[8];
              tc::load_v8(params + o + e, q);
#pragma unroll
              for (int i = 0; i < 8; ++i) q[i] = __float_as_uint(__uint_as_float(q[i]) * decay - step * v[e + i]);
              tc::store_v8(params + o + e, q);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (col + j + e < n) params[o + e] = params[o + e] * decay - step * v[e];
          }
        } else if (wide && col + j + 16 <= n) {
          uint32_t q[8];
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
#pragma unroll
              for (int i = 0; i < 8; ++i) q[i] = __float_as_uint(v[e + i]);
              tc::store_v8(out + o + e, q);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
              q[i] = *reinterpret_cast<const uint32_t*>(&b);
            }
            tc::store_v8(out + o, q);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (col + j + e < n) store_as(out + o + e, v[e]);
        }
      } else {
        uint32_t h[8], l[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) tc::split_f16x2(v[2 * i], v[2 * i + 1], &h[i], &l[i]);
        __half* d = dst.p + base + col + j;
        tc::store_v8(d, h);
        tc::store_v8(d + dst.plane, l);
        if (mirror) {   // lanes hold consecutive rows: the transposed store is contiguous over them
          __half* t = dst.p + (size_t)x.batch * 2 * dst.plane + row;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (col + j + i >= n) break;
            const size_t o = (size_t)(col + j + i) * dst.pitch;
            t[o] = __ushort_as_half((uint16_t)(h[i / 2] >> (16 * (i & 1))));
            t[o + dst.plane] = __ushort_as_half((uint16_t)(l[i / 2] >> (16 * (i & 1))));
          }
        }
      }
    }
  }
};

int norm_blocks(int64_t n) { return (int)((n + kNormThreads * kNormPer - 1) / (kNormThreads * kNormPer)); }

// k-tiles (of 64) that one accumulator takes before it is added to the registers.
constexpr int kNsChunk = 1;
constexpr int kNsTile = 128;

// Short sides up to 64 whose slices fit take one cluster per matrix, the others the tensor
// cores.
bool on_tensor_cores(const nc_newton_schulz* d) { return !small_plan(d).fits; }

int plane_pitch(int cols) { return (cols + 63) / 64 * 64; }

struct NsLayout {
  size_t status, part, u, x, y, gram, poly, total;
};

NsLayout ns_layout(const nc_newton_schulz* d) {
  NsLayout L{};
  const size_t n = (size_t)d->rows * d->cols, s = d->rows < d->cols ? d->rows : d->cols;
  const size_t x = (size_t)d->rows * plane_pitch(d->cols), g = s * plane_pitch((int)s);   // two float16 planes each
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += pad256(bytes);
    return o;
  };
  L.status = take(4);
  if (!on_tensor_cores(d)) {
    L.total = at;
    return L;
  }
  L.part = take((size_t)d->batch * norm_blocks(n) * 8);
  L.u = take(d->batch * n * 4);
  L.x = take(d->batch * x * 4);
  L.y = take(d->batch * x * 4);
  L.gram = take(d->batch * g * 4);
  L.poly = take(d->batch * g * 4);
  L.total = at;
  return L;
}

nc_status check_desc(const nc_newton_schulz* d) {
  if (!d) return set_error(NC_ERR_INVALID, "nc_newton_schulz descriptor is null");
  if (d->batch < 0 || d->rows < 1 || d->cols < 1)
    return set_error(NC_ERR_INVALID, "bad matrices (batch %d, rows %d, cols %d)", d->batch, d->rows, d->cols);
  if (d->dtype != NC_F32 && d->dtype != NC_BF16) return set_error(NC_ERR_INVALID, "unknown dtype %d", d->dtype);
  if (d->steps < 0 || d->steps > 64) return set_error(NC_ERR_INVALID, "steps %d is not in 0..64", d->steps);
  if (!(d->eps >= 0.f)) return set_error(NC_ERR_INVALID, "eps is negative or NaN");
  if (d->batch > 65535 || (int64_t)d->rows * d->cols > INT32_MAX)
    return set_error(NC_ERR_UNSUPPORTED, "more than 65535 matrices, or more than 2^31 - 1 elements in one");
  return NC_OK;
}

nc_status check_ws(const void* ws, size_t have, size_t need) {
  if (!ws || reinterpret_cast<uintptr_t>(ws) % 256 != 0)
    return set_error(NC_ERR_WORKSPACE, "workspace is null or not 256-byte aligned");
  if (have < need) return set_error(NC_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", have, need);
  return NC_OK;
}

// No steps: X0 as it is.
template <typename T>
__global__ void __launch_bounds__(256) ns_store_kernel(Planes x, int rows, int cols, T* __restrict__ out,
                                                       float* __restrict__ params, float decay, float step) {
  pdl_enter();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * cols) return;
  const size_t s = (size_t)blockIdx.y * 2 * x.plane + (size_t)(i / cols) * x.pitch + i % cols;
  const size_t o = (size_t)blockIdx.y * rows * cols + i;
  const float v = (__half2float(x.p[s]) + __half2float(x.p[x.plane + s])) * kPlaneInv;
  if (params)
    params[o] = params[o] * decay - step * v;
  else
    store_as(out + o, v);
}

template <int MODE, typename T>
nc_status tensor_product(const nc_newton_schulz* d, const Planes& A, bool a_mn, const Planes& B, bool b_mn, int m, int n,
                         int k, const NsEpilogue<MODE, T>& epi, int32_t* status, cudaStream_t st) {
  tc::Problem p{};
  p.m = m, p.n = n, p.k = k, p.batch = d->batch, p.splits = 1, p.chunk = kNsChunk;
  tc::set_tiles<kNsTile, 1>(&p);
  p.symmetric = MODE == kGram || MODE == kPoly;
  p.status = status;
  NC_CHECK((tc::make_operand<2, kNsTile, 1>(&p, true, A.p, a_mn, m, k, A.pitch, A.plane, d->batch, 2 * A.plane)));
  NC_CHECK((tc::make_operand<2, kNsTile, 1>(&p, false, B.p, b_mn, n, k, B.pitch, B.plane, d->batch, 2 * B.plane)));
  return tc::launch_product<2, kNsTile, 1>(p, epi, st, "Newton-Schulz product launch");
}

template <typename T>
nc_status run_tensor(const nc_newton_schulz* d, const T* x, const float* u, const double* part, T* out, float* params,
                     float decay, float step, char* ws, const NsLayout& L, cudaStream_t st) {
  const int64_t n = (int64_t)d->rows * d->cols;
  const int nb = norm_blocks(n), s = d->rows < d->cols ? d->rows : d->cols;
  const bool tall = d->rows > d->cols;
  int32_t* status = reinterpret_cast<int32_t*>(ws + L.status);
  auto planes = [&](size_t o, int rows, int cols) {
    Planes q;
    q.p = reinterpret_cast<__half*>(ws + o), q.pitch = plane_pitch(cols), q.plane = (int64_t)rows * q.pitch;
    return q;
  };
  Planes X = planes(L.x, d->rows, d->cols), Y = planes(L.y, d->rows, d->cols);
  const Planes G = planes(L.gram, s, s), Q = planes(L.poly, s, s);
  {
    PdlLaunch l(dim3(nb, d->batch), dim3(kNormThreads), 0, st);
    if (u)
      NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ns_split_kernel<float>, u, n, d->cols, nb, part, (double)d->eps, X));
    else
      NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ns_split_kernel<T>, x, n, d->cols, nb, part, (double)d->eps, X));
    NC_CHECK(launch_check("ns_split_kernel launch"));
  }
  if (d->steps == 0) {
    PdlLaunch l(dim3((unsigned)((n + 255) / 256), d->batch), dim3(256), 0, st);
    NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ns_store_kernel<T>, X, d->rows, d->cols, out, params, decay, step));
    return launch_check("ns_store_kernel launch");
  }
  const void* to = params ? static_cast<void*>(params) : static_cast<void*>(out);
  const size_t size = params ? 4 : sizeof(T);
  const bool wide = reinterpret_cast<uintptr_t>(to) % 32 == 0 && (size_t)d->cols * size % 32 == 0;
  for (int k = 0; k < d->steps; ++k) {
    NsEpilogue<kGram, T> g{};
    g.src = g.dst = G, g.m = g.n = s, g.mul = kPlaneInv;
    NC_CHECK(tensor_product(d, X, tall, X, tall, s, s, tall ? d->rows : d->cols, g, status, st));
    NsEpilogue<kPoly, T> q{};
    q.src = G, q.dst = Q, q.m = q.n = s, q.mul = d->c * kPlaneInv, q.add = d->b;
    NC_CHECK(tensor_product(d, G, false, G, false, s, s, s, q, status, st));
    // rows <= cols: (b A + c A^2) X, X with its own index contiguous; else X (b A + c A^2)
    const Planes &A = tall ? X : Q, &B = tall ? Q : X;
    if (k + 1 < d->steps) {
      NsEpilogue<kUpdate, T> e{};
      e.src = X, e.dst = Y, e.m = d->rows, e.n = d->cols, e.mul = kPlaneInv, e.add = d->a;
      NC_CHECK(tensor_product(d, A, false, B, !tall, d->rows, d->cols, s, e, status, st));
      const Planes t = X;
      X = Y, Y = t;
    } else {
      NsEpilogue<kFinal, T> e{};
      e.src = X, e.m = d->rows, e.n = d->cols, e.mul = kPlaneInv, e.add = d->a;
      e.out = out, e.params = params, e.decay = decay, e.step = step, e.wide = wide;
      NC_CHECK(tensor_product(d, A, false, B, !tall, d->rows, d->cols, s, e, status, st));
    }
  }
  return NC_OK;
}

// From the source x (or x and momentum) to the orthogonalised matrix; `out` or `params`.
template <typename T>
nc_status run(const nc_newton_schulz* d, const T* x, float* momentum, MuonArgs mu, T* out, float* params, float decay,
              float step, void* d_ws, cudaStream_t st) {
  const NsLayout L = ns_layout(d);
  char* ws = static_cast<char*>(d_ws);
  int32_t* status = reinterpret_cast<int32_t*>(ws + L.status);
  if (!on_tensor_cores(d)) {
    const SmallPlan r = small_plan(d);
    const SmallArgs a{x,    momentum, params, out,  d->rows, d->cols, r.slice, d->steps,
                      d->a, d->b,     d->c,   d->eps, mu,      decay,   step,    status};
    return r.pad == 16   ? launch_small<16, T>(a, r, d->batch, st)
           : r.pad == 32 ? launch_small<32, T>(a, r, d->batch, st)
                         : launch_small<64, T>(a, r, d->batch, st);
  }
  float* u = reinterpret_cast<float*>(ws + L.u);
  double* part = reinterpret_cast<double*>(ws + L.part);
  const int64_t n = (int64_t)d->rows * d->cols;
  PdlLaunch l(dim3(norm_blocks(n), d->batch), dim3(kNormThreads), 0, st);
  NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ns_norm_kernel<T>, x, momentum, mu, n, u, part, status));
  NC_CHECK(launch_check("ns_norm_kernel launch"));
  return run_tensor(d, x, momentum ? u : nullptr, part, out, params, decay, step, ws, L, st);
}

}  // namespace

}  // namespace nc

using namespace nc;

extern "C" {

size_t nc_newton_schulz_workspace_bytes(const nc_newton_schulz* desc) {
  if (check_desc(desc) != NC_OK) return 0;
  return ns_layout(desc).total;
}

nc_status nc_orthogonalize(const nc_newton_schulz* desc, const void* x, void* out, void* d_ws, size_t ws_bytes,
                           void* stream) {
  NC_CHECK(check_desc(desc));
  if (desc->batch == 0) {
    clear_error();
    return NC_OK;
  }
  const bool bf16 = desc->dtype == NC_BF16;
  if (!x || !out) return set_error(NC_ERR_INVALID, "x or out is null");
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) % (bf16 ? 2 : 4) != 0)
    return set_error(NC_ERR_INVALID, "x or out is not on an element's boundary");
  NC_CHECK(check_ws(d_ws, ws_bytes, ns_layout(desc).total));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const MuonArgs mu{};
  if (bf16)
    NC_CHECK(run(desc, static_cast<const __nv_bfloat16*>(x), nullptr, mu, static_cast<__nv_bfloat16*>(out), nullptr,
                 1.f, 0.f, d_ws, st));
  else
    NC_CHECK(run(desc, static_cast<const float*>(x), nullptr, mu, static_cast<float*>(out), nullptr, 1.f, 0.f, d_ws,
                 st));
  clear_error();
  return NC_OK;
}

nc_status nc_muon_update(const nc_newton_schulz* desc, float* params, const float* grads, float* momentum, float lr,
                         float beta, int32_t nesterov, float weight_decay, void* d_ws, size_t ws_bytes, void* stream) {
  NC_CHECK(check_desc(desc));
  if (desc->dtype != NC_F32) return set_error(NC_ERR_INVALID, "nc_muon_update takes float32");
  if (desc->batch == 0) {
    clear_error();
    return NC_OK;
  }
  NC_CHECK(check_ptr(params, "params"));
  NC_CHECK(check_ptr(grads, "grads"));
  NC_CHECK(check_ptr(momentum, "momentum"));
  if (params == momentum || params == grads || momentum == grads)
    return set_error(NC_ERR_INVALID, "params, grads and momentum must be different buffers");
  NC_CHECK(check_ws(d_ws, ws_bytes, ns_layout(desc).total));
  const MuonArgs mu{beta, nesterov};
  const double tall = (double)desc->rows / desc->cols;
  const float step = (float)((double)lr * sqrt(tall > 1.0 ? tall : 1.0));
  NC_CHECK(run<float>(desc, grads, momentum, mu, nullptr, params, (float)(1.0 - (double)lr * weight_decay), step, d_ws,
                      reinterpret_cast<cudaStream_t>(stream)));
  clear_error();
  return NC_OK;
}

}  // extern "C"
