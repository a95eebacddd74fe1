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

// ---- short sides up to 64: one cluster per matrix ------------------------------------------
// The CTAs of a cluster hold slices of the long side in shared memory for all steps, as
// X[l][i] (i along the short side, padded to S).  A step: every CTA adds up its slice's part
// of A = X X^T, the cluster sums the parts (each CTA its share of A, read from and written to
// the others' shared memory), and every CTA updates its slice, which needs no other slice:
//   narrow slices (up to S):  Y = A X,  X <- a X + b Y + c A Y       2 S^2 FMAs a column
//   wide ones:  Q = b A + c A^2 in every CTA (S^3),  X <- a X + Q X  S^2 a column
// The momentum, the norm and the final update are in the same launch, so the cost is the two
// cluster barriers of a step and the FMAs: three 62 x 62 grids take 24 us for five steps, 32 x 3969
// on 16 CTAs 43 us.
constexpr int kSmallThreads = 512;
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
struct Small {
  static constexpr int kPitch = S + 4, kPer = S / 4, kCell = kPer * kPer;   // threads of one S x S product
  static constexpr int kGroups = kSmallThreads / kCell;                     // that split the slice's columns
  static constexpr int kParts = kGroups * S * S > S * kPitch ? kGroups * S * S : S * kPitch;   // Q fits too
  static_assert(kCell <= kSmallThreads, "a thread takes 4 x 4 of A");
};

template <int S>
__host__ __device__ constexpr size_t small_smem(int slice) {
  return (size_t)(2 * slice * Small<S>::kPitch + Small<S>::kParts + S * Small<S>::kPitch) * 4;
}

// N columns l of sum over k of A[k][i..i+3] in[l][k].
template <int S, int N>
__device__ __forceinline__ void small_product(const float* A, const float* in, int i, float (&acc)[N][4]) {
  constexpr int kPitch = Small<S>::kPitch;
#pragma unroll
  for (int q = 0; q < N; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[q][e] = 0.f;
#pragma unroll 4
  for (int k = 0; k < S; k += 4) {
    float m[4][4], v[N][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) *reinterpret_cast<float4*>(m[e]) = *reinterpret_cast<const float4*>(A + (k + e) * kPitch + i);
#pragma unroll
    for (int q = 0; q < N; ++q) *reinterpret_cast<float4*>(v[q]) = *reinterpret_cast<const float4*>(in + q * kPitch + k);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int q = 0; q < N; ++q)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[q][r] = fmaf(m[e][r], v[q][e], acc[q][r]);
  }
}

// put(l, i, sums) for all columns l of `count` and rows i..i+3 of A in: by threads of 4 columns
// each, or where those would be few, of one.
template <int S, typename Put>
__device__ __forceinline__ void small_products(const float* A, const float* in, int count, Put put) {
  constexpr int kPer = Small<S>::kPer, kPitch = Small<S>::kPitch;
  if (count * kPer <= 2 * kSmallThreads) {
    for (int t = threadIdx.x; t < count * kPer; t += kSmallThreads) {
      const int i = t % kPer * 4, l = t / kPer;
      float acc[1][4];
      small_product<S, 1>(A, in + l * kPitch, i, acc);
      put(l, i, acc[0]);
    }
  } else {
    for (int t = threadIdx.x; t < count / 4 * kPer; t += kSmallThreads) {
      const int i = t % kPer * 4, l = t / kPer * 4;
      float acc[4][4];
      small_product<S, 4>(A, in + l * kPitch, i, acc);
#pragma unroll
      for (int q = 0; q < 4; ++q) put(l + q, i, acc[q]);
    }
  }
}

template <int S, typename T>
__global__ void __launch_bounds__(kSmallThreads) ns_small_kernel(SmallArgs p) {
  namespace cg = cooperative_groups;
  constexpr int kPitch = Small<S>::kPitch, kPer = Small<S>::kPer, kCell = Small<S>::kCell, kGroups = Small<S>::kGroups;
  extern __shared__ __align__(16) float sm[];
  __shared__ double red[kSmallThreads / 32], total;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank(), tid = threadIdx.x;
  float* X = sm;
  float* Y = X + p.slice * kPitch;
  float* part = Y + p.slice * kPitch;       // (kGroups, S, S)
  float* A = part + Small<S>::kParts;       // (S, pitch)
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
    auto put4 = [](float* at, float x, float y, float z, float w) {
      *reinterpret_cast<float4*>(at) = make_float4(x, y, z, w);
    };
    if (p.slice <= S) {
      small_products<S>(A, X, p.slice, [&](int l, int i, float (&v)[4]) { put4(Y + l * kPitch + i, v[0], v[1], v[2], v[3]); });
      __syncthreads();
      small_products<S>(A, Y, p.slice, [&](int l, int i, float (&v)[4]) {
        float* x = X + l * kPitch + i;
        const float* y = Y + l * kPitch + i;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(p.a, x[e], fmaf(p.b, y[e], p.c * v[e]));
        put4(x, v[0], v[1], v[2], v[3]);
      });
    } else {
      // A is symmetric, so its rows serve as columns; the parts' place takes Q (its readers have
      // passed the cluster's barrier)
      float* Q = part;
      small_products<S>(A, A, S, [&](int l, int i, float (&v)[4]) {
        const float* x = A + l * kPitch + i;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(p.b, x[e], p.c * v[e]);
        put4(Q + l * kPitch + i, v[0], v[1], v[2], v[3]);
      });
      __syncthreads();
      small_products<S>(Q, X, p.slice, [&](int l, int i, float (&v)[4]) {
        const float* x = X + l * kPitch + i;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(p.a, x[e], v[e]);
        put4(Y + l * kPitch + i, v[0], v[1], v[2], v[3]);
      });
      float* t = X;
      X = Y, Y = t;
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
  r.ranks = len > 1024 ? 16 : len > 28 ? 8 : len > 12 ? 4 : len > 4 ? 2 : 1;
  r.slice = ((len + r.ranks - 1) / r.ranks + 3) / 4 * 4;
  const size_t need = r.pad == 16 ? small_smem<16>(r.slice) : r.pad == 32 ? small_smem<32>(r.slice) : small_smem<64>(r.slice);
  r.fits = s <= 64 && need <= kSmallSmem;
  return r;
}

template <int S, typename T>
nc_status launch_small(const SmallArgs& a, const SmallPlan& r, int batch, cudaStream_t st) {
  auto k = ns_small_kernel<S, T>;
  const size_t smem = small_smem<S>(r.slice);
  NC_CHECK(allow_smem((const void*)k, smem));
  if (r.ranks > 8) NC_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
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

// ---- longer short sides: products on the tensor cores --------------------------------------
// X, A = X X^T and Q = b A + c A^2 are kept as two float16 planes each (nc_tc.cuh), scaled by
// 2^12: |entries| stay below 16 while the singular values do, and an entry of 2^-26 still has
// its 11 bits in the high plane.
//
// Bound by shared memory where matrices are large: per k-tile a 128 x 128 tile's three products
// read 96 KB of operands and the copies write 64 KB, 1250 cycles at 128 bytes a cycle (768 on the
// tensor pipe alone); a k-tile takes about 1400.
//
// All steps are one cooperative launch: a product of such sizes takes a few microseconds, and
// a launch, its set-up of tensor memory and its first loads as much again.  Between products
// the grid meets (cooperative_groups); the symmetric ones compute the tiles on and above the
// diagonal and store them twice; a product with fewer tiles than SMs is split along k, its
// float32 parts summed in order by the whole grid.  2001 x 513 takes 280 us (18 a product, mostly
// meetings, split sums, fill and drain), three 1024 x 1024 updates 455 us, three
// 256 x 256 on a cluster each 133 us.
constexpr float kPlaneScale = 4096.f, kPlaneInv = 1.f / 4096.f;
constexpr int kNsChunk = 1;  // k-tiles (of 64) per accumulator: Gram sums of one sign show the additions' truncation
constexpr int kNsCols = 32;  // columns of an epilogue thread
// Where matrices have many tiles: 128 x 128, the whole grid on all matrices (pairs of CTAs on
// 256 x 128 took 146 cycles for a product of 16 k that one CTA does in 115 on its half).  Where
// they have few: 128 x 64 and a cluster of 8 or 16 on each matrix.
template <bool CLUSTER>
struct NsTile {
  static constexpr int kBN = CLUSTER ? 64 : 128, kWarps = CLUSTER ? 8 : 16;
};
template <bool CLUSTER>
using NsEngine = tc::Engine<2, NsTile<CLUSTER>::kBN, 1, NsTile<CLUSTER>::kWarps>;
static_assert(NsEngine<true>::COLS == kNsCols && NsEngine<false>::COLS == kNsCols, "the epilogue is written for 32");

struct Planes {   // (batch, plane, rows, pitch)
  __half* p;
  int pitch;
  int64_t plane;
};

enum NsProduct { kGram, kPoly, kUpdate };

constexpr int kCluster = 8, kLargeCluster = 16;   // CTAs
constexpr int kLargeClusters = 7;                 // that run at a time

struct NsArgs {
  // X and its next value, A and Q as operands a and b: with k contiguous, or by rows of k
  CUtensorMap k_a[2], k_b[2], rows_a[2], rows_b[2], gram_a, gram_b, poly_a, poly_b;
  Planes X[2], G, Q;
  const void* x;
  float* momentum;
  float* params;
  void* out;
  double* norms;    // (batch, CTAs) parts of the squared norms
  float4* parts;    // of split products
  int64_t parts_each;   // of one matrix, where clusters work on one each
  int batch, rows, cols, steps;
  int splits[3];
  int vec;              // cols are whole 4s and the tensors start on 16 bytes
  float a, b, c;
  double eps;
  MuonArgs mu;
  float decay, step;
  int32_t* status;
  int first;            // of the call's launches: clears the status
};

// The transposed store of 32 rows (a lane each) and 32 columns: through the warp's patch, as 32
// rows of 64 bytes.  `rows`, `cols`: how many of them exist; what lies behind a row's end is
// padding.
__device__ __forceinline__ void store_mirrored(uint8_t* patch, __half* p, int64_t pitch, int rows, int cols,
                                               const uint32_t (&v)[16]) {
  const int lane = threadIdx.x & 31, odd = lane & 1;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    // pairs of lanes exchange: an even one gets both rows of column 2 i, an odd one of 2 i + 1
    const uint32_t other = __shfl_xor_sync(0xffffffffu, v[i], 1);
    const uint32_t two = odd ? __byte_perm(other, v[i], 0x7632) : __byte_perm(v[i], other, 0x5410);
    *reinterpret_cast<uint32_t*>(patch + (2 * i + odd) * 64 + (lane >> 1) * 4) = two;
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = i * 8 + (lane >> 2), q = lane & 3;
    if (c < cols && 8 * q < rows)
      *reinterpret_cast<uint4*>(p + c * pitch + 8 * q) = *reinterpret_cast<const uint4*>(patch + c * 64 + 16 * q);
  }
}

// acc += add times a row's 32 values of one plane, in 16-byte pieces at `at(i)`.
template <typename At>
__device__ __forceinline__ void add_row(At at, float add, float (&acc)[32]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 w = *reinterpret_cast<const uint4*>(at(i));
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[e]));
      acc[8 * i + 2 * e] = fmaf(add, f.x, acc[8 * i + 2 * e]);
      acc[8 * i + 2 * e + 1] = fmaf(add, f.y, acc[8 * i + 2 * e + 1]);
    }
  }
}

// acc += add times 32 rows and 32 columns of both planes in global memory.
__device__ __forceinline__ void add_planes(uint8_t* patch, const Planes& s, size_t at, int rows, int cols, float add,
                                           float (&acc)[32]) {
  const int lane = threadIdx.x & 31, q = lane & 3;
  uint4 v[2][4];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + (lane >> 2);
      v[k][i] = r < rows && 8 * q < cols ? *reinterpret_cast<const uint4*>(s.p + k * s.plane + at + (size_t)r * s.pitch + 8 * q)
                                         : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) *tc::patch_at<32>(patch, i * 8 + (lane >> 2), q) = v[k][i];
    __syncwarp();
    add_row([&](int i) { return tc::patch_at<32>(patch, lane, i); }, add, acc);
  }
}

// Result of a product for 32 rows from row0 on and 32 columns from col on, on scaled values:
// mul acc + add (A or X), to planes (and mirrored), or (last) unscaled to the caller.  `prior`:
// 64 columns of A or X in shared memory (Engine::extra), or null to take them from global memory.
template <typename T>
__device__ __forceinline__ void ns_store(const NsArgs& p, NsProduct product, int k, bool last, const tc::Tile& x,
                                         int row0, int col, uint8_t* patch, const uint8_t* prior, float (&acc)[32]) {
  const Planes& dst = product == kGram ? p.G : product == kPoly ? p.Q : p.X[(k + 1) & 1];
  const int s = min(p.rows, p.cols), m = product == kUpdate ? p.rows : s, n = product == kUpdate ? p.cols : s;
  const int lane = threadIdx.x & 31, rows = min(32, m - row0), cols = min(32, n - col);
  const size_t at = (size_t)x.batch * 2 * dst.plane + (size_t)row0 * dst.pitch + col;
  const float mul = product == kPoly ? p.c * kPlaneInv : kPlaneInv, add = product == kPoly ? p.b : p.a;
  // symmetric results: what lies right of the diagonal's square goes left of it too
  const bool mirror = product != kUpdate && col >= x.m0 + tc::kBM;
  if (rows <= 0 || cols <= 0) return;   // the same for the whole warp
#pragma unroll
  for (int j = 0; j < 32; ++j) acc[j] *= mul;
  if (product != kGram && prior) {
    const int r = row0 - x.m0 + lane, c = (col - x.n0) % 64 / 8;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      add_row([&](int i) { return prior + h * (tc::kBM * 128) + r * 128 + (((c + i) ^ (r & 7)) << 4); }, add, acc);
  } else if (product != kGram) {
    add_planes(patch, product == kPoly ? p.G : p.X[k & 1], at, rows, cols, add, acc);
  }
  if (!last) {
    __half* d = dst.p + at;
    __half* t = dst.p + (size_t)x.batch * 2 * dst.plane + (size_t)col * dst.pitch + row0;
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {   // a plane, and what it leaves for the next
      uint32_t v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const __half2 w = __floats2half2_rn(acc[2 * i], acc[2 * i + 1]);
        const float2 b = __half22float2(w);
        acc[2 * i] -= b.x, acc[2 * i + 1] -= b.y;
        v[i] = *reinterpret_cast<const uint32_t*>(&w);
      }
      tc::patch_store<32>(patch, v, reinterpret_cast<uint16_t*>(d), dst.pitch, rows, (cols + 7) / 8);
      if (mirror) store_mirrored(patch, t, dst.pitch, rows, cols, v);
      d += dst.plane, t += dst.plane;
    }
    return;
  }
  // 16 columns at a time, two rows per access
  float* f = reinterpret_cast<float*>(patch);
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; ++j) f[lane * 16 + (j ^ (lane & 15))] = acc[16 * g + j] * kPlaneInv;
    __syncwarp();
    const int c = lane & 15;
    if (16 * g + c < cols) {
      const size_t o = ((size_t)x.batch * m + row0) * n + col + 16 * g + c;
#pragma unroll 8
      for (int r = lane >> 4; r < rows; r += 2) {
        const float v = f[r * 16 + (c ^ (r & 15))];
        if (p.params)
          p.params[o + (size_t)r * n] = p.params[o + (size_t)r * n] * p.decay - p.step * v;
        else
          store_as(static_cast<T*>(p.out) + o + (size_t)r * n, v);
      }
    }
  }
}

// Product f of a step on `batch` matrices.  gram: the short side's rows of X against themselves;
// poly: A A; update: Q X, or X Q.
template <bool CLUSTER>
__device__ __forceinline__ tc::Problem ns_problem(const NsArgs& p, int f, int batch) {
  const bool tall = p.rows > p.cols;
  const int s = tall ? p.cols : p.rows, len = tall ? p.rows : p.cols;
  tc::Problem q;
  q.m = f == kUpdate ? p.rows : s, q.n = f == kUpdate ? p.cols : s, q.k = f == kGram ? len : s;
  q.a_mn = f == kGram && tall, q.b_mn = f == kGram ? tall : f == kUpdate && !tall;
  tc::set_tiles<NsTile<CLUSTER>::kBN, 1>(&q);
  q.batch = batch, q.splits = p.splits[f], q.symmetric = f != kUpdate, q.chunk = kNsChunk, q.bf16 = 0;
  q.a_k0 = q.b_k0 = q.b_n0 = 0;
  return q;
}
// Whether the result is added to a tile that comes through the pipeline.
__device__ __forceinline__ bool wants_prior(const tc::Problem& q, int f) { return f != kGram && q.splits == 1; }

// Four consecutive elements, or as many as `left`.
template <typename T>
__device__ __forceinline__ void load4(const T* p, bool vec, int left, float (&v)[4]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p);
    } else {
      const uint2 q = *reinterpret_cast<const uint2*>(p);
      v[0] = __uint_as_float(q.x << 16), v[1] = __uint_as_float(q.x & 0xffff0000u);
      v[2] = __uint_as_float(q.y << 16), v[3] = __uint_as_float(q.y & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < left ? to_f32(p[j]) : 0.f;
  }
}
__device__ __forceinline__ void store4(float* p, bool vec, int left, const float (&v)[4]) {
  if (vec) {
    *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = v[j];
  }
}

template <typename T, bool CLUSTER>
__global__ void __launch_bounds__(NsEngine<CLUSTER>::C::kThreads, 1) ns_kernel(const __grid_constant__ NsArgs p) {
  using E = NsEngine<CLUSTER>;
  constexpr int kWarps = E::kEpiWarps, kThreads = E::C::kThreads, kBN = NsTile<CLUSTER>::kBN;
  extern __shared__ __align__(1024) uint8_t raw[];
  __shared__ tc::Shared<2, kBN, 1, kWarps> sh;
  __shared__ double red[kThreads / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (p.first && blockIdx.x == 0 && tid == 0) *p.status = 0;
  E e(raw, &sh, p.status);
  // The CTAs that work together: the whole grid on all matrices, or a cluster on one.
  const int size = CLUSTER ? (int)tc::cluster_size() : gridDim.x, rank = CLUSTER ? (int)tc::cluster_rank() : blockIdx.x;
  const int b0 = CLUSTER ? blockIdx.x / size : 0, batch = CLUSTER ? 1 : p.batch;
  // Everything stored so far is there for every CTA's loads, plain ones and tensor copies.
  auto meet = [&] {
    __threadfence();
    asm volatile("fence.proxy.async;" ::: "memory");
    if constexpr (CLUSTER)
      tc::cluster_sync();
    else
      cooperative_groups::this_grid().sync();
    asm volatile("fence.proxy.async;" ::: "memory");
  };
  auto tile = [&](const tc::Problem& q, int t) {
    tc::Tile x = tc::problem_tile<kBN, 1>(q, t, 0);
    x.batch += b0;
    return x;
  };
  const int64_t n = (int64_t)p.rows * p.cols;
  const int quads = (p.cols + 3) / 4;   // four columns at a time
  const int64_t all = (int64_t)p.rows * quads;

  // momentum, and each CTA's part of the squared norms
  for (int b = b0; b < b0 + batch; ++b) {
    double sum = 0.0;
#pragma unroll 2
    for (int64_t i = (int64_t)rank * kThreads + tid; i < all; i += (int64_t)size * kThreads) {
      const int r = (int)((uint32_t)i / (uint32_t)quads), c = 4 * ((int)i - r * quads), left = p.cols - c;
      const size_t o = (size_t)b * n + (size_t)r * p.cols + c;
      float u[4];
      load4(static_cast<const T*>(p.x) + o, p.vec, left, u);
      if (p.momentum) {
        float m[4];
        load4(p.momentum + o, p.vec, left, m);
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = fmaf(p.mu.beta, m[j], u[j]);
        store4(p.momentum + o, p.vec, left, m);
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = p.mu.nesterov ? fmaf(p.mu.beta, m[j], u[j]) : m[j];
      }
      double s = 0.0;
#pragma unroll
      for (int j = 0; j < 4; ++j) s += (double)u[j] * u[j];
      sum += s;
    }
    __syncthreads();   // red of the last matrix has been read
    sum = block_sum_f64(sum, red);
    if (tid == 0) p.norms[(size_t)b * size + rank] = sum;
  }
  meet();
  // X0 as planes; every CTA adds up a matrix's parts, in order
  for (int b = b0; b < b0 + batch; ++b) {
    double sum = 0.0;
    for (int j = tid; j < size; j += kThreads) sum += p.norms[(size_t)b * size + j];
    __syncthreads();
    sum = block_sum_f64(sum, red);
    const double inv = 1.0 / (sqrt(sum) + p.eps);
    __half* hi = p.X[0].p + (size_t)b * 2 * p.X[0].plane;
#pragma unroll 2
    for (int64_t i = (int64_t)rank * kThreads + tid; i < all; i += (int64_t)size * kThreads) {
      const int r = (int)((uint32_t)i / (uint32_t)quads), c = 4 * ((int)i - r * quads), left = p.cols - c;
      const size_t o = (size_t)b * n + (size_t)r * p.cols + c;
      float u[4];
      load4(static_cast<const T*>(p.x) + o, p.vec, left, u);
      if (p.momentum) {
        float m[4];
        load4(p.momentum + o, p.vec, left, m);
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = p.mu.nesterov ? fmaf(p.mu.beta, m[j], u[j]) : m[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = (float)((double)u[j] * inv) * kPlaneScale;
      uint32_t h[2], l[2];
      tc::split_f16x2(u[0], u[1], &h[0], &l[0]);
      tc::split_f16x2(u[2], u[3], &h[1], &l[1]);
      __half* to = hi + (size_t)r * p.X[0].pitch + c;   // the padding behind a row takes the rest
      *reinterpret_cast<uint2*>(to) = make_uint2(h[0], h[1]);
      *reinterpret_cast<uint2*>(to + p.X[0].plane) = make_uint2(l[0], l[1]);
    }
  }
  meet();

  // The roles go through the products each in a loop of its own.
  if (warp == kWarps) {
    for (int k = 0; k < p.steps; ++k) {
#pragma unroll 1
      for (int f = kGram; f <= kUpdate; ++f) {
        const tc::Problem q = ns_problem<CLUSTER>(p, f, batch);
        const bool tall = p.rows > p.cols;
        const int w = k & 1;
        const CUtensorMap* ma = f == kGram ? (tall ? &p.rows_a[w] : &p.k_a[w]) : f == kPoly ? &p.gram_a : tall ? &p.k_a[w] : &p.poly_a;
        const CUtensorMap* mb = f == kGram ? (tall ? &p.rows_b[w] : &p.k_b[w]) : f == kPoly ? &p.gram_b : tall ? &p.poly_b : &p.rows_b[w];
        const int tiles = tc::problem_tiles<kBN, 1>(q);
        if (lane == 0) {
          for (int t = rank; t < tiles && e.ok; t += size) {
            const tc::Tile x = tile(q, t);
            e.load(q, ma, mb, x);
            if (wants_prior(q, f)) e.load_extra(f == kPoly ? &p.gram_a : &p.k_a[w], x);
          }
        }
        __syncwarp();
        meet();
        if (q.splits > 1) meet();
      }
    }
  } else if (warp == kWarps + 1) {
    for (int k = 0; k < p.steps; ++k) {
#pragma unroll 1
      for (int f = kGram; f <= kUpdate; ++f) {
        const tc::Problem q = ns_problem<CLUSTER>(p, f, batch);
        const int tiles = tc::problem_tiles<kBN, 1>(q);
        for (int t = rank; t < tiles && e.ok; t += size) {
          e.multiply(q, tile(q, t));
          if (wants_prior(q, f)) e.skip_extra();
        }
        meet();
        if (q.splits > 1) meet();
      }
    }
  } else {
    float4* const parts = p.parts + (size_t)b0 * p.parts_each;
    for (int k = 0; k < p.steps; ++k) {
#pragma unroll 1
      for (int f = kGram; f <= kUpdate; ++f) {
        const tc::Problem q = ns_problem<CLUSTER>(p, f, batch);
        const bool last = f == kUpdate && k + 1 == p.steps;
        // The tiles of this CTA; then, where a product was split, a second pass in which each warp
        // of the group adds up the parts of one warp's rows and columns, `whole` tiles apart.
        const int tiles = tc::problem_tiles<kBN, 1>(q), whole = tiles / q.splits;
        for (int pass = 0; pass < (q.splits > 1 ? 2 : 1); ++pass) {
          const int begin = pass == 0 ? rank : rank * kWarps + warp, end = pass == 0 ? tiles : whole * kWarps;
          for (int w = begin; w < end && e.ok; w += pass == 0 ? size : size * kWarps) {
            const int t = pass == 0 ? w : w / kWarps, part = pass == 0 ? warp : w % kWarps;
            const tc::Tile x = tile(q, t);
            float acc[kNsCols];
            const uint8_t* prior = nullptr;
            if (pass == 0) {
              e.collect(q, x, acc);
              if (!e.ok) break;
              if (q.splits > 1) {
                float4* o = parts + ((size_t)t * kWarps + warp) * (kNsCols * 8) + lane;
#pragma unroll
                for (int j = 0; j < kNsCols / 4; ++j)
                  o[j * 32] = make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]);
                continue;
              }
              if (wants_prior(q, f)) prior = e.extra();
              if (!e.ok) break;
            } else {
#pragma unroll
              for (int j = 0; j < kNsCols; ++j) acc[j] = 0.f;
              for (int g = 0; g < q.splits; ++g) {
                const float4* o = parts + ((size_t)(t + g * whole) * kWarps + part) * (kNsCols * 8) + lane;
                float4 v[kNsCols / 4];
#pragma unroll
                for (int j = 0; j < kNsCols / 4; ++j) v[j] = __ldcg(o + j * 32);
#pragma unroll
                for (int j = 0; j < kNsCols / 4; ++j)
                  acc[4 * j] += v[j].x, acc[4 * j + 1] += v[j].y, acc[4 * j + 2] += v[j].z, acc[4 * j + 3] += v[j].w;
              }
            }
            ns_store<T>(p, (NsProduct)f, k, last, x, x.m0 + 32 * (part & 3), x.n0 + (part >> 2) * kNsCols, e.patch, prior,
                        acc);
            if (prior) e.extra_done();
          }
          meet();
        }
      }
    }
  }
  if (p.steps == 0) {   // X0 as it is
    for (int64_t w = b0 * n + rank * (int64_t)kThreads + tid; w < n * (b0 + batch); w += (int64_t)size * kThreads) {
      const int64_t b = w / n, i = w - b * n;
      const size_t o = (size_t)b * 2 * p.X[0].plane + (size_t)(i / p.cols) * p.X[0].pitch + i % p.cols;
      const float v = (__half2float(p.X[0].p[o]) + __half2float(p.X[0].p[p.X[0].plane + o])) * kPlaneInv;
      if (p.params)
        p.params[w] = p.params[w] * p.decay - p.step * v;
      else
        store_as(static_cast<T*>(p.out) + w, v);
    }
  }
  e.finish();
}

// Short sides up to 64 whose slices fit take one cluster per matrix, the others the tensor
// cores.
bool on_tensor_cores(const nc_newton_schulz* d) { return !small_plan(d).fits; }

int plane_pitch(int cols) { return (cols + 63) / 64 * 64; }

// Splits of a product along k: as many as shorten the k-tiles of the busiest of `at_once` workers
// by more than the sum costs (an extra meeting and a pass over the parts, about 8 k-tiles' time).
int choose_splits(int64_t tiles, int k, int at_once) {
  auto ceil_div = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
  const int64_t kt = ceil_div(k, tc::kBK);
  int64_t best = ceil_div(tiles, at_once) * kt;
  int splits = 1;
  for (int s = 2; s <= 32 && s <= kt; ++s) {
    const int64_t cost = ceil_div(tiles * s, at_once) * ceil_div(kt, s) + 8 + s / 4;
    if (cost < best) best = cost, splits = s;
  }
  return splits;
}

// Planes (and so matrices) of one launch; more matrices go by several launches on the same
// workspace. 64000 x 65 x 520 would take 23 GB at once; a launch's start and end are about 170 us
// beside several milliseconds.
constexpr size_t kLaunchBytes = (size_t)1 << 30;

struct NsLayout {
  size_t status, norms, x, y, gram, poly, parts, total;
  int cluster;   // CTAs of one, or 0
  int batch;   // matrices of a launch
  int splits[3], blocks;
  int64_t parts_each;
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
  // A meeting of a cluster takes half of the grid's, and a smaller tile's stores are sooner done.  Five
  // steps of one matrix, us on a cluster of 8, of 16 and on the grid: 8 times 256 x 256 (8 tiles) 122, -
  // and 226; 128 x 1024 (16) 133, 114 and 199; 256 x 512 (16) 151, 130 and 213; 384 x 384 (18) 226, 159 and
  // 219; 128 x 2048 (32) 178, 141 and 203; 200 x 1500 (48) -, 196 and 219; 512 x 512 (32) 360, 240 and
  // 241; 512 x 600 (40) -, 280 and 249.  So a cluster of 16 where its rounds of tiles come to at most
  // 16 k-tiles.  Not for many matrices, as 7 clusters of 16 or some 14 of 8 run at a time while the
  // grid shares all tiles: 20 times 128 x 128 176 on clusters of 8 and 214 on the grid, 36 times 260
  // and 253; 16 times 256 x 512 303 and 263.
  const auto tiles_of = [](int64_t m, int64_t n, int wide) { return ((m + 127) / 128) * ((n + wide - 1) / wide); };
  const int64_t narrow = tiles_of(d->rows, d->cols, 64);
  const int64_t deep = (narrow + kLargeCluster - 1) / kLargeCluster * ((s + tc::kBK - 1) / tc::kBK);
  const bool large = narrow <= 4 * kLargeCluster && deep <= 16 && d->batch <= kLargeClusters;
  L.cluster = narrow <= kCluster && d->batch <= 20          ? kCluster
              : large                                       ? kLargeCluster
              : narrow <= 2 * kCluster && d->batch <= 14 ? kCluster
                                                         : 0;
  const size_t most_batch = kLaunchBytes / (8 * (x + g)) + 1;
  L.batch = (size_t)d->batch < most_batch ? d->batch : (int)most_batch;
  tc::Problem q{};
  q.m = q.n = (int)s, q.batch = L.cluster ? 1 : L.batch, q.splits = 1, q.symmetric = 1;
  if (L.cluster)
    tc::set_tiles<64, 1>(&q);
  else
    tc::set_tiles<128, 1>(&q);
  const int64_t triangle = L.cluster ? tc::problem_tiles<64, 1>(q) : tc::problem_tiles<128, 1>(q);
  const int64_t whole = tiles_of(d->rows, d->cols, L.cluster ? 64 : 128) * q.batch;
  const int64_t count[3] = {triangle, triangle, whole};
  const int depth[3] = {d->rows < d->cols ? d->cols : d->rows, (int)s, (int)s};
  const int tile = 128 * (L.cluster ? 64 : 128);
  int64_t most = 1, parts = 0;
  for (int f = 0; f < 3; ++f) {
    L.splits[f] = choose_splits(count[f], depth[f], L.cluster ? L.cluster : 148);
    const int64_t all = count[f] * L.splits[f];
    if (all > most) most = all;
    if (L.splits[f] > 1 && all > parts) parts = all;
  }
  L.parts_each = parts * tile / 4;
  // as many CTAs as any product keeps busy, or as share the element-wise passes well
  int64_t blocks = (int64_t)(L.batch * n / 4096);
  if (most > blocks) blocks = most;
  L.blocks = L.cluster ? L.cluster * L.batch : (int)(blocks < 148 ? blocks : 148);
  L.norms = take((size_t)L.batch * (L.cluster ? L.cluster : L.blocks) * 8);
  L.x = take(L.batch * x * 4);
  L.y = take(L.batch * x * 4);
  L.gram = take(L.batch * g * 4);
  L.poly = take(L.batch * g * 4);
  L.parts = take((size_t)L.parts_each * (L.cluster ? L.batch : 1) * 16);
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
  if (d->batch > 65535 || (int64_t)d->rows * d->cols > 1 << 30)
    return set_error(NC_ERR_UNSUPPORTED, "more than 65535 matrices, or more than 2^30 elements in one");
  return NC_OK;
}

nc_status check_ws(const void* ws, size_t have, size_t need) {
  if (!ws || reinterpret_cast<uintptr_t>(ws) % 256 != 0)
    return set_error(NC_ERR_WORKSPACE, "workspace is null or not 256-byte aligned");
  if (have < need) return set_error(NC_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", have, need);
  return NC_OK;
}

template <typename T>
nc_status run_tensor(const nc_newton_schulz* d, const T* x, float* momentum, MuonArgs mu, T* out, float* params,
                     float decay, float step, char* ws, const NsLayout& L, cudaStream_t st) {
  const int s = d->rows < d->cols ? d->rows : d->cols;
  auto planes = [&](size_t o, int rows, int cols) {
    Planes q;
    q.p = reinterpret_cast<__half*>(ws + o), q.pitch = plane_pitch(cols), q.plane = (int64_t)rows * q.pitch;
    return q;
  };
  NsArgs a{};
  a.X[0] = planes(L.x, d->rows, d->cols), a.X[1] = planes(L.y, d->rows, d->cols);
  a.G = planes(L.gram, s, s), a.Q = planes(L.poly, s, s);
  // operands with k contiguous (a box has as many of the own index as a CTA's tile), or by rows of
  // k (boxes of 64 by 64)
  const int a_rows = 128, b_rows = L.cluster ? 64 : 128;
  auto map = [&](CUtensorMap* m, const Planes& q, int rows, int cols, int box) {
    return tc::make_map(m, q.p, false, 2, cols, rows, q.pitch, q.plane, L.batch, 2 * q.plane, 64, box);
  };
  for (int i = 0; i < 2; ++i) {
    NC_CHECK(map(&a.k_a[i], a.X[i], d->rows, d->cols, a_rows));
    NC_CHECK(map(&a.k_b[i], a.X[i], d->rows, d->cols, b_rows));
    NC_CHECK(map(&a.rows_a[i], a.X[i], d->rows, d->cols, tc::kBK));
    a.rows_b[i] = a.rows_a[i];
  }
  NC_CHECK(map(&a.gram_a, a.G, s, s, a_rows));
  NC_CHECK(map(&a.gram_b, a.G, s, s, b_rows));
  NC_CHECK(map(&a.poly_a, a.Q, s, s, a_rows));
  NC_CHECK(map(&a.poly_b, a.Q, s, s, b_rows));
  a.norms = reinterpret_cast<double*>(ws + L.norms), a.parts = reinterpret_cast<float4*>(ws + L.parts);
  a.parts_each = L.parts_each;
  a.rows = d->rows, a.cols = d->cols, a.steps = d->steps;
  for (int f = 0; f < 3; ++f) a.splits[f] = L.splits[f];
  a.vec = d->cols % 4 == 0 && (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(momentum)) % 16 == 0;
  a.a = d->a, a.b = d->b, a.c = d->c, a.eps = d->eps, a.mu = mu, a.decay = decay, a.step = step;
  a.status = reinterpret_cast<int32_t*>(ws + L.status);
  auto k = L.cluster ? ns_kernel<T, true> : ns_kernel<T, false>;
  const int smem = L.cluster ? NsEngine<true>::C::kSmem : NsEngine<false>::C::kSmem;
  NC_CHECK(allow_smem((const void*)k, smem));
  if (L.cluster > 8) NC_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  if (L.cluster) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = L.cluster, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  } else {
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
  }
  cfg.blockDim = dim3(L.cluster ? NsEngine<true>::C::kThreads : NsEngine<false>::C::kThreads);
  cfg.dynamicSmemBytes = smem, cfg.stream = st, cfg.attrs = attr, cfg.numAttrs = 1;
  const size_t n = (size_t)d->rows * d->cols;
  for (int b = 0; b < d->batch; b += L.batch) {
    a.batch = d->batch - b < L.batch ? d->batch - b : L.batch;
    a.x = x + b * n, a.momentum = momentum ? momentum + b * n : nullptr;
    a.params = params ? params + b * n : nullptr, a.out = out ? out + b * n : nullptr;
    a.first = b == 0;
    cfg.gridDim = dim3((unsigned)(L.cluster ? L.cluster * a.batch : L.blocks));
    NC_CUDA_CHECK(cudaLaunchKernelEx(&cfg, k, a));
    NC_CHECK(launch_check("ns_kernel launch"));
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
  return run_tensor(d, x, momentum, mu, out, params, decay, step, ws, L, st);
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
  const size_t bytes = (size_t)desc->batch * desc->rows * desc->cols * (bf16 ? 2 : 4);
  if ((x != out && overlap(x, bytes, out, bytes)) || overlap(x, bytes, d_ws, ws_bytes) ||
      overlap(out, bytes, d_ws, ws_bytes))
    return set_error(NC_ERR_INVALID, "x, out and the workspace overlap (out may only be x itself)");
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
  const size_t bytes = (size_t)desc->batch * desc->rows * desc->cols * 4;
  if (overlap(params, bytes, momentum, bytes) || overlap(params, bytes, grads, bytes) ||
      overlap(momentum, bytes, grads, bytes))
    return set_error(NC_ERR_INVALID, "params, grads and momentum must be different buffers");
  NC_CHECK(check_ws(d_ws, ws_bytes, ns_layout(desc).total));
  if (overlap(params, bytes, d_ws, ws_bytes) || overlap(momentum, bytes, d_ws, ws_bytes) ||
      overlap(grads, bytes, d_ws, ws_bytes))
    return set_error(NC_ERR_INVALID, "the workspace overlaps params, grads or momentum");
  const MuonArgs mu{beta, nesterov};
  const double tall = (double)desc->rows / desc->cols;
  const float step = (float)((double)lr * sqrt(tall > 1.0 ? tall : 1.0));
  NC_CHECK(run<float>(desc, grads, momentum, mu, nullptr, params, (float)(1.0 - (double)lr * weight_decay), step, d_ws,
                      reinterpret_cast<cudaStream_t>(stream)));
  clear_error();
  return NC_OK;
}

}  // extern "C"
