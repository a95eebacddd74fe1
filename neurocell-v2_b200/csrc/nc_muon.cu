// nc_muon.cu -- orthogonalisation of matrices by Newton-Schulz products, and the update of
// parameters by orthogonalised momentum.
//
//   X0 = x / (|x|_F + eps);  steps times: A = X X^T, X <- a X + (b A + c A^2) X
//
// on the short side (A = X^T X, X <- a X + X (b A + c A^2) when rows > cols).  Every
// singular value s of x goes through s <- a s + b s^3 + c s^5; the singular vectors stay.
// The norm is summed in float64: the iteration magnifies an error of the scale of X0 up to
// about a hundred times.
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

// X0 of one matrix; every block sums the matrix's parts again, in the same order.
template <typename T>
__global__ void __launch_bounds__(kNormThreads) ns_scale_kernel(const T* __restrict__ x, int64_t n, int parts,
                                                                const double* __restrict__ part, double eps,
                                                                float* __restrict__ out) {
  __shared__ double red[kNormThreads / 32];
  pdl_enter();
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += kNormThreads) s += part[(size_t)blockIdx.y * parts + i];
  s = block_sum_f64(s, red);
  const double inv = 1.0 / (sqrt(s) + eps);
  const size_t base = (size_t)blockIdx.y * n;
  const int64_t i0 = (int64_t)blockIdx.x * kNormThreads * kNormPer + threadIdx.x;
#pragma unroll 4
  for (int k = 0; k < kNormPer; ++k) {
    const int64_t i = i0 + (int64_t)k * kNormThreads;
    if (i >= n) break;
    out[base + i] = (float)((double)to_f32(x[base + i]) * inv);
  }
}

// One product of batched matrices, out = alpha A B + beta C: 64 x 64 tiles of float32 in
// registers (4 x 4 per thread).  Element (i, k) of A is at i * a_i + k * a_k, and so on.
struct Product {
  const float *A, *B, *C;
  float* out;
  int m, n, k;
  int64_t a_i, a_k, b_k, b_j, stride_a, stride_b, stride_c;   // C and out: row-major (m, n)
  float alpha, beta;
};

__global__ void __launch_bounds__(256) ns_product_kernel(Product p) {
  __shared__ float as[16][64 + 4], bs[16][64 + 4];
  pdl_enter();
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64, tid = threadIdx.x;
  const float* A = p.A + (size_t)blockIdx.z * p.stride_a;
  const float* B = p.B + (size_t)blockIdx.z * p.stride_b;
  const int tx = tid & 15, ty = tid >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < p.k; k0 += 16) {
    __syncthreads();
    for (int e = tid; e < 16 * 64; e += 256) {
      // the thread order follows the operand's contiguous direction
      const int ka = p.a_k == 1 ? e & 15 : e >> 6, ia = p.a_k == 1 ? e >> 4 : e & 63;
      as[ka][ia] = k0 + ka < p.k && i0 + ia < p.m ? A[(i0 + ia) * p.a_i + (k0 + ka) * p.a_k] : 0.f;
      const int kb = p.b_k == 1 ? e & 15 : e >> 6, jb = p.b_k == 1 ? e >> 4 : e & 63;
      bs[kb][jb] = k0 + kb < p.k && j0 + jb < p.n ? B[(k0 + kb) * p.b_k + (j0 + jb) * p.b_j] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = as[k][ty * 4 + e], y[e] = bs[k][tx * 4 + e];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][c] = fmaf(x[r], y[c], acc[r][c]);
    }
  }
  const size_t base = (size_t)blockIdx.z * p.stride_c;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int i = i0 + ty * 4 + r, j = j0 + tx * 4 + c;
      if (i >= p.m || j >= p.n) continue;
      const size_t o = base + (size_t)i * p.n + j;
      p.out[o] = p.alpha * acc[r][c] + (p.C ? p.beta * p.C[o] : 0.f);
    }
}

// out = X in the caller's type, or with `params`: p <- decay p - step X.
template <typename T>
__global__ void ns_store_kernel(const float* __restrict__ x, int64_t n, T* __restrict__ out, float* __restrict__ params,
                                float decay, float step) {
  pdl_enter();
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  if (params)
    params[i] = params[i] * decay - step * x[i];
  else
    store_as(out + i, x[i]);
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
  __device__ __forceinline__ void run(const tc::Tile& x, int row, int col, float (&acc)[HALF]) const {
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
        for (int i = 0; i < 8; ++i) {
          uint16_t h0, l0, h1, l1;
          tc::split_f16(v[2 * i], &h0, &l0);
          tc::split_f16(v[2 * i + 1], &h1, &l1);
          h[i] = h0 | (uint32_t)h1 << 16, l[i] = l0 | (uint32_t)l1 << 16;
        }
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

// k-tiles (of 32) that one accumulator takes before it is added to the registers.
constexpr int kNsChunk = 2;
constexpr int kNsTile = 128;

// The tensor cores from a short side of 65 on; below, one 64 x 64 float32 tile holds A.
bool on_tensor_cores(const nc_newton_schulz* d) { return d->rows > 64 && d->cols > 64 && d->steps > 0; }

int plane_pitch(int cols) { return (cols + 63) / 64 * 64; }

struct NsLayout {
  size_t status, part, u, x, y, gram, poly, total;
};

NsLayout ns_layout(const nc_newton_schulz* d) {
  NsLayout L{};
  const size_t n = (size_t)d->rows * d->cols, s = d->rows < d->cols ? d->rows : d->cols;
  // float32 (rows, cols), or two planes of float16 with padded rows
  const bool tensor = on_tensor_cores(d);
  const size_t x = tensor ? (size_t)d->rows * plane_pitch(d->cols) : n, g = tensor ? s * plane_pitch((int)s) : s * s;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += pad256(bytes);
    return o;
  };
  L.status = take(4);
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

nc_status product(const Product& p, int batch, cudaStream_t st) {
  PdlLaunch l(dim3((p.n + 63) / 64, (p.m + 63) / 64, batch), dim3(256), 0, st);
  NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ns_product_kernel, p));
  return launch_check("ns_product_kernel launch");
}

template <int MODE, typename T>
nc_status tensor_product(const nc_newton_schulz* d, const Planes& A, bool a_mn, const Planes& B, bool b_mn, int m, int n,
                         int k, const NsEpilogue<MODE, T>& epi, int32_t* status, cudaStream_t st) {
  tc::Problem p{};
  p.m = m, p.n = n, p.k = k, p.batch = d->batch, p.splits = 1, p.chunk = kNsChunk;
  p.tiles_m = (m + tc::kBM - 1) / tc::kBM, p.tiles_n = (n + kNsTile - 1) / kNsTile;
  p.symmetric = MODE == kGram || MODE == kPoly;
  p.status = status;
  NC_CHECK((tc::make_operand<2, kNsTile>(&p, true, A.p, a_mn, m, k, A.pitch, A.plane, d->batch, 2 * A.plane)));
  NC_CHECK((tc::make_operand<2, kNsTile>(&p, false, B.p, b_mn, n, k, B.pitch, B.plane, d->batch, 2 * B.plane)));
  return tc::launch_product<2, kNsTile>(p, epi, st, "Newton-Schulz product launch");
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
  auto f32 = [&](size_t o) { return reinterpret_cast<float*>(ws + o); };
  double* part = reinterpret_cast<double*>(ws + L.part);
  const int64_t n = (int64_t)d->rows * d->cols;
  const int nb = norm_blocks(n), s = d->rows < d->cols ? d->rows : d->cols;
  {
    PdlLaunch l(dim3(nb, d->batch), dim3(kNormThreads), 0, st);
    NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ns_norm_kernel<T>, x, momentum, mu, n, f32(L.u), part,
                                     reinterpret_cast<int32_t*>(ws + L.status)));
    NC_CHECK(launch_check("ns_norm_kernel launch"));
  }
  if (on_tensor_cores(d))
    return run_tensor(d, x, momentum ? f32(L.u) : nullptr, part, out, params, decay, step, ws, L, st);
  float *X = f32(L.x), *Y = f32(L.y);
  {
    PdlLaunch l(dim3(nb, d->batch), dim3(kNormThreads), 0, st);
    if (momentum)
      NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ns_scale_kernel<float>, (const float*)f32(L.u), n, nb,
                                       (const double*)part, (double)d->eps, X));
    else
      NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ns_scale_kernel<T>, x, n, nb, (const double*)part, (double)d->eps, X));
    NC_CHECK(launch_check("ns_scale_kernel launch"));
  }
  const bool tall = d->rows > d->cols;
  const int64_t ss = (int64_t)s * s;
  for (int k = 0; k < d->steps; ++k) {
    Product g{};   // Gram matrix of the short side
    g.A = X, g.B = X, g.out = f32(L.gram), g.m = s, g.n = s, g.k = tall ? d->rows : d->cols;
    g.a_i = tall ? 1 : d->cols, g.a_k = tall ? d->cols : 1, g.b_k = g.a_k, g.b_j = g.a_i;
    g.stride_a = g.stride_b = n, g.stride_c = ss, g.alpha = 1.f;
    NC_CHECK(product(g, d->batch, st));
    Product q{};   // b A + c A^2
    q.A = q.B = q.C = f32(L.gram), q.out = f32(L.poly), q.m = q.n = q.k = s;
    q.a_i = q.b_k = s, q.a_k = q.b_j = 1, q.stride_a = q.stride_b = q.stride_c = ss, q.alpha = d->c, q.beta = d->b;
    NC_CHECK(product(q, d->batch, st));
    Product u{};   // a X + (b A + c A^2) X
    u.m = d->rows, u.n = d->cols, u.k = s, u.C = X, u.out = Y, u.alpha = 1.f, u.beta = d->a, u.stride_c = n;
    u.A = tall ? X : f32(L.poly), u.B = tall ? f32(L.poly) : X;
    u.a_i = s, u.a_k = 1, u.b_k = d->cols, u.b_j = 1;
    u.stride_a = tall ? n : ss, u.stride_b = tall ? ss : n;
    NC_CHECK(product(u, d->batch, st));
    float* t = X;
    X = Y, Y = t;
  }
  const int64_t all = n * d->batch;
  PdlLaunch l(dim3((unsigned)((all + 255) / 256)), dim3(256), 0, st);
  NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ns_store_kernel<T>, (const float*)X, all, out, params, decay, step));
  return launch_check("ns_store_kernel launch");
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
