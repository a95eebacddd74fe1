// nc_readout.cu -- softmax cross-entropy of a linear readout over a large vocabulary, with
// its gradients, without the (rows, classes) logits in memory.
//
//   z = f w^T + b,  lse_n = log sum_v exp z_nv,  loss_n = lse_n - z_n,label
//   dz = g_n (exp(z - lse) - onehot),  df = dz w,  dw = dz^T f,  db = sum_n dz
//
// The value keeps one running (maximum, sum) per row and block of classes; the gradient
// computes the logits of a block of classes again and multiplies them out while they are
// on chip.
//
// Few rows (here): a CTA streams its share of the weight through shared memory once, in chunks
// that bulk copies bring while it works on the one before, and everything a chunk is needed
// for happens there.  Bound by reading the weight (and writing its gradient): one float32 row
// x 1024 x 50000 is scored in 40 us (5.1 TB/s, 79 % of a copy's rate).  With more rows the FFMAs
// and their shared memory reads take over: value and gradients of 8 rows take 201 us, 0.6 GB at
// 3.1 TB/s (from global memory without the copies 240 us).  More rows: nc_readout_tc.cu.
#include <math.h>

#include <initializer_list>

#include "nc_common.cuh"
#include "nc_errors.h"
#include "nc_readout.h"
#include "nc_tc.cuh"

namespace nc {

namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kRowDim = 4 * kRowThreads;       // most columns: four a thread
constexpr int kRowBuffers = 2, kRowChunk = 64;   // most classes of a chunk
constexpr size_t kRowChunkBytes = 64 * 1024;   // two in flight cover the memory's latency
constexpr int kRowsMost = 16, kRowsMostBf16 = 4;
constexpr int kRowStats = 512;                 // logits a row collects before its statistics take them in

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

template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
  } else {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
    __stcs(reinterpret_cast<uint2*>(p),
           make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi)));
  }
}

// What the streaming kernels share.  chunk: classes per chunk; chunks: of all classes.
struct RowArgs {
  CeArgs a;
  int chunk, chunks;
  int bulk;           // the weight starts on 16 bytes
};

// The stream of this CTA's chunks [c0, c1) of the weight.
template <typename T>
struct RowStream {
  const RowArgs& r;
  uint8_t* ring;
  uint32_t bars;
  int* abort;
  int c0, c1;
  bool ok = true;

  __device__ __forceinline__ RowStream(const RowArgs& args, uint8_t* buffers, uint64_t* barriers, int* flag)
      : r(args), ring(buffers), bars(tc::smem_addr(barriers)), abort(flag) {
    c0 = (int)((int64_t)r.chunks * blockIdx.x / gridDim.x), c1 = (int)((int64_t)r.chunks * (blockIdx.x + 1) / gridDim.x);
    if (threadIdx.x == 0) {
      for (int i = 0; i < kRowBuffers; ++i) tc::bar_init(bars + 8 * i, 1);
      *abort = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
  }
  __device__ __forceinline__ int classes(int c) const { return min(r.chunk, r.a.classes - c * r.chunk); }
  __device__ __forceinline__ const T* at(int c) const {
    return static_cast<const T*>(r.a.weight) + (size_t)c * r.chunk * r.a.dim;
  }
  __device__ __forceinline__ T* buffer(int c) const {
    return reinterpret_cast<T*>(ring + (size_t)((c - c0) % kRowBuffers) * r.chunk * r.a.dim * sizeof(T));
  }
  // This thread's class of chunk c: its bias, asked for a chunk ahead of its use.
  __device__ __forceinline__ float bias(int c) const {
    const T* b = static_cast<const T*>(r.a.bias);
    return b && c < c1 && (int)threadIdx.x < classes(c) ? to_f32(b[(size_t)c * r.chunk + threadIdx.x]) : 0.f;
  }
  __device__ __forceinline__ uint32_t bytes(int c) const { return (uint32_t)(classes(c) * r.a.dim * sizeof(T)); }
  // Thread 0 asks for chunk c; its buffer is free.
  __device__ __forceinline__ void ask(int c) const {
    if (!r.bulk || c >= c1 || threadIdx.x != 0) return;
    const uint32_t bar = bars + 8 * ((c - c0) % kRowBuffers), n = bytes(c) & ~15u;
    tc::bar_expect(bar, n);
    if (n > 0)
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                       tc::smem_addr(buffer(c))),
                   "l"(at(c)), "r"(n), "r"(bar)
                   : "memory");
  }
  // The whole CTA: chunk c is in its buffer.  Chunks start on 16 bytes; what a last one has
  // behind whole 16s, and chunks of a weight that does not start so, are loaded here.
  __device__ __forceinline__ bool wait(int c) {
    const int i = c - c0;
    if (r.bulk) ok = tc::bar_wait(bars + 8 * (i % kRowBuffers), i / kRowBuffers & 1, abort, r.a.status);
    const int n = classes(c) * r.a.dim, from = r.bulk ? (int)((bytes(c) & ~15u) / sizeof(T)) : 0;
    T* to = buffer(c);
    for (int e = from + threadIdx.x; e < n; e += kRowThreads) to[e] = at(c)[e];
    ok = __syncthreads_and(ok);
    return ok;
  }
  // After an abort: the copies in flight land before the CTA ends.
  __device__ __forceinline__ void drain(int c) const {
    if (ok || !r.bulk || threadIdx.x != 0) return;
    for (int k = c; k < min(c + kRowBuffers, c1); ++k)
      for (int j = 0; j < tc::kWaitLimit && !tc::bar_try(bars + 8 * ((k - c0) % kRowBuffers), (k - c0) / kRowBuffers & 1); ++j) {
      }
  }
};

// The features in shared memory, zeros for rows that take no part or do not exist.
template <typename T, int RN>
__device__ __forceinline__ void stage_features(const CeArgs& a, float* hs) {
  const T* f = static_cast<const T*>(a.features);
  for (int i = threadIdx.x; i < RN * a.dim; i += kRowThreads) {
    const int row = i / a.dim;
    hs[i] = row < a.rows && ce_kept(a, row) ? to_f32(f[i]) : 0.f;
  }
}

// Logits (no bias) of the chunk's classes: put(v, r, z).  A warp takes VT classes at a time, its
// lanes split the columns; a 16-byte read of the features serves 4 VT products.  Classes past
// `n` read what the buffer holds and are not put.
template <typename T, int RN, int VEC, int VT, typename Put>
__device__ __forceinline__ void chunk_logits(const T* w, const float* hs, int dim, int n, Put put) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int v0 = warp * VT; v0 < n; v0 += kRowWarps * VT) {
    float acc[VT * RN];
#pragma unroll
    for (int i = 0; i < VT * RN; ++i) acc[i] = 0.f;
#pragma unroll 2
    for (int d = lane * VEC; d < dim; d += 32 * VEC) {
      float x[VT][VEC];
#pragma unroll
      for (int j = 0; j < VT; ++j) load_vec<VEC>(w + min(v0 + j, n - 1) * dim + d, x[j]);
#pragma unroll
      for (int r = 0; r < RN; ++r) {
        float h[VEC];
        load_vec<VEC>(hs + r * dim + d, h);
#pragma unroll
        for (int j = 0; j < VT; ++j)
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[j * RN + r] = fmaf(x[j][e], h[e], acc[j * RN + r]);
      }
    }
    int first;
    warp_sums(acc, lane, &first);
#pragma unroll
    for (int i = 0; i < (VT * RN + 31) / 32; ++i) {
      const int k = first + i, v = v0 + k / RN;
      if (v < n) put(v, k % RN, acc[i]);
    }
  }
}

// Each CTA's (maximum, sum) of every row, and the label's logit where it has it.
template <typename T, int RN, int VEC, int VT>
__global__ void __launch_bounds__(kRowThreads) ce_rows_value_kernel(const RowArgs args, float2* __restrict__ part,
                                                                    float* __restrict__ zlabel) {
  extern __shared__ __align__(128) uint8_t raw[];
  __shared__ __align__(8) uint64_t bars[kRowBuffers];
  __shared__ int flag;
  __shared__ float bias[kRowChunk];
  const CeArgs& a = args.a;
  float* hs = reinterpret_cast<float*>(raw + kRowBuffers * (size_t)args.chunk * a.dim * sizeof(T));
  float* z = hs + RN * a.dim;   // (RN, kRowStats)
  RowStream<T> s(args, raw, bars, &flag);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kMine = (RN + kRowWarps - 1) / kRowWarps;   // rows whose statistics a warp keeps
  float2 mine[kMine];
#pragma unroll
  for (int k = 0; k < kMine; ++k) mine[k] = make_float2(-INFINITY, 0.f);
  pdl_enter();
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
  for (int c = s.c0; c < s.c0 + kRowBuffers; ++c) s.ask(c);
  stage_features<T, RN>(a, hs);
  int held = 0, base = s.c0 * args.chunk;   // classes base .. base + held - 1 are in z
  int c = s.c0;
  float next = s.bias(c);
  for (; c < s.c1; ++c) {
    if (threadIdx.x < kRowChunk) bias[threadIdx.x] = next;
    next = s.bias(c + 1);
    if (!s.wait(c)) break;
    const int n = s.classes(c);
    chunk_logits<T, RN, VEC, VT>(s.buffer(c), hs, a.dim, n,
                                 [&](int v, int r, float x) { z[r * kRowStats + held + v] = x + bias[v]; });
    __syncthreads();
    s.ask(c + kRowBuffers);
    held += n;
    if (held + args.chunk <= kRowStats && c + 1 < s.c1) continue;
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int r = warp + k * kRowWarps;
      if (r >= a.rows || r >= RN) continue;
      const int label = a.labels[r];
      float m = -INFINITY;
      for (int v = lane; v < held; v += 32) {
        const float x = z[r * kRowStats + v];
        m = fmaxf(m, x);
        if (base + v == label) zlabel[r] = x;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      float t = 0.f;
      for (int v = lane; v < held; v += 32) {
        const float x = z[r * kRowStats + v];
        t += x == -INFINITY ? 0.f : expf(x - m);
      }
      mine[k] = lse_merge(mine[k], make_float2(m, warp_sum(t)));
    }
    base += held, held = 0;
    __syncthreads();
  }
  s.drain(c);
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    const int r = warp + k * kRowWarps;
    if (lane == 0 && r < RN && r < a.rows) part[(size_t)r * gridDim.x + blockIdx.x] = mine[k];
  }
}

// One block, a warp a row: the CTAs' pairs merged in a fixed order, the rows' losses, and their
// sum or mean into `loss` unless that is null.
__global__ void __launch_bounds__(512) ce_rows_finish_kernel(CeArgs a, int blocks, const float2* __restrict__ part,
                                                             const float* __restrict__ zlabel, float* __restrict__ lse,
                                                             float* row_loss, float* __restrict__ loss) {
  pdl_enter();
  const int row = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (row < a.rows) {
    float2 x = make_float2(-INFINITY, 0.f);
    for (int i = lane; i < blocks; i += 32) x = lse_merge(x, part[(size_t)row * blocks + i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float2 y = make_float2(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o));
      x = lse_merge(x, y);
    }
    if (lane == 0) finish_row(a, row, x, zlabel, lse, row_loss);
  }
  __syncthreads();
  if (!loss || threadIdx.x != 0) return;
  double t = 0.0;
  int kept = 0;
  for (int i = 0; i < a.rows; ++i) t += row_loss[i], kept += ce_kept(a, i);
  loss[0] = (float)(a.reduction == NC_REDUCE_MEAN ? t / (double)max(kept, 1) : t);
}

// Gradients.  Of each chunk the logits again, left as p = g_n (exp(z - lse) - onehot); then a thread
// owns four columns (a sum over classes needs no other thread until the end), with the features'
// and df's in registers for all rows, and goes through
// the classes: dw[v] = sum_n p f[n] is stored, df[n] += p w[v] stays.  Where the columns need
// fewer threads (td of them), groups of td share the classes and meet at the end.
template <typename T, int RN, int VEC, int VT>
__global__ void __launch_bounds__(kRowThreads) ce_rows_grad_kernel(
    const RowArgs args, int td, const float* __restrict__ lse, const float* __restrict__ g_loss, T* __restrict__ g_weight,
    T* __restrict__ g_bias, float* __restrict__ df_part) {
  extern __shared__ __align__(128) uint8_t raw[];
  __shared__ __align__(8) uint64_t bars[kRowBuffers];
  __shared__ int flag;
  __shared__ float bias[kRowChunk];
  __shared__ float row_g[RN], row_lse[RN];
  __shared__ int row_label[RN];
  const CeArgs& a = args.a;
  float* hs = reinterpret_cast<float*>(raw + kRowBuffers * (size_t)args.chunk * a.dim * sizeof(T));
  float* p = hs + RN * a.dim;   // (chunk, RN)
  RowStream<T> s(args, raw, bars, &flag);
  const int tid = threadIdx.x;
  pdl_enter();
  if (blockIdx.x == 0 && tid == 0) *a.status = 0;
  for (int c = s.c0; c < s.c0 + kRowBuffers; ++c) s.ask(c);
  if (tid < RN) {
    int kept = 0;
    for (int i = 0; i < a.rows; ++i) kept += ce_kept(a, i);
    const bool in = tid < a.rows && ce_kept(a, tid);
    const float g = g_loss && in ? g_loss[a.reduction == NC_REDUCE_NONE ? tid : 0] : 1.f;
    row_g[tid] = !in ? 0.f : a.reduction == NC_REDUCE_MEAN ? g / (float)max(kept, 1) : g;
    row_lse[tid] = in ? lse[tid] : 0.f;
    row_label[tid] = in ? a.labels[tid] : -1;
  }
  stage_features<T, RN>(a, hs);
  __syncthreads();
  const int dt = tid % td, group = tid / td, groups = kRowThreads / td;
  int col[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) col[e] = VEC == 4 ? 4 * dt + e : dt + e * td;
  float h[RN][4], acc[RN][4];
#pragma unroll
  for (int r = 0; r < RN; ++r)
#pragma unroll
    for (int e = 0; e < 4; ++e) h[r][e] = col[e] < a.dim ? hs[r * a.dim + col[e]] : 0.f, acc[r][e] = 0.f;
  int c = s.c0;
  float next = s.bias(c);
  for (; c < s.c1; ++c) {
    if (tid < kRowChunk) bias[tid] = next;
    next = s.bias(c + 1);
    if (!s.wait(c)) break;
    const int n = s.classes(c), v0 = c * args.chunk;
    const T* w = s.buffer(c);
    chunk_logits<T, RN, VEC, VT>(w, hs, a.dim, n, [&](int v, int r, float x) { p[v * RN + r] = x; });
    __syncthreads();
    for (int i = tid; i < n * RN; i += kRowThreads) {
      const int v = i / RN, r = i % RN;
      const float x = p[i] + bias[v];
      p[i] = row_g[r] == 0.f ? 0.f : row_g[r] * (expf(x - row_lse[r]) - (v0 + v == row_label[r] ? 1.f : 0.f));
    }
    __syncthreads();
    if (g_bias) {
      for (int v = tid; v < n; v += kRowThreads) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < RN; ++r) t += p[v * RN + r];
        store_as(g_bias + v0 + v, t);
      }
    }
    if (col[0] < a.dim) {
#pragma unroll 2
      for (int v = group; v < n; v += groups) {
        static_assert(RN == 1 || RN % 4 == 0, "rows come in fours");
        float x[4], out[4] = {0.f, 0.f, 0.f, 0.f};
        alignas(16) float q[RN];
        if constexpr (VEC == 4) {
          load_vec<4>(w + v * a.dim + col[0], x);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = col[e] < a.dim ? to_f32(w[v * a.dim + col[e]]) : 0.f;
        }
        if constexpr (RN % 4 == 0) {
#pragma unroll
          for (int r = 0; r < RN; r += 4) *reinterpret_cast<float4*>(q + r) = *reinterpret_cast<const float4*>(p + v * RN + r);
        } else {
          q[0] = p[v];
        }
#pragma unroll
        for (int r = 0; r < RN; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            out[e] = fmaf(q[r], h[r][e], out[e]);
            acc[r][e] = fmaf(q[r], x[e], acc[r][e]);
          }
        if (g_weight) {
          T* o = g_weight + (size_t)(v0 + v) * a.dim;
          if constexpr (VEC == 4) {
            store4(o + col[0], out);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col[e] < a.dim) store_as(o + col[e], out[e]);
          }
        }
      }
    }
    __syncthreads();
    s.ask(c + kRowBuffers);
  }
  s.drain(c);
  if (!df_part) return;
  // the groups' sums, in order; the ring's place is free
  float* sum = reinterpret_cast<float*>(raw);   // (groups, RN, 4 td)
  if (groups > 1) {
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RN; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[(group * RN + r) * 4 * td + e * td + dt] = acc[r][e];
    __syncthreads();
    for (int i = tid; i < RN * 4 * td; i += kRowThreads) {
      const int r = i / (4 * td), k = i % (4 * td), d = VEC == 4 ? k % td * 4 + k / td : k % td + k / td * td;
      float t = 0.f;
      for (int g = 0; g < groups; ++g) t += sum[g * RN * 4 * td + i];
      if (r < a.rows && d < a.dim) df_part[((size_t)blockIdx.x * a.rows + r) * a.dim + d] = t;
    }
  } else {
#pragma unroll
    for (int r = 0; r < RN; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (r < a.rows && col[e] < a.dim) df_part[((size_t)blockIdx.x * a.rows + r) * a.dim + col[e]] = acc[r][e];
  }
}

// df: the CTAs' parts, 8 threads an element, in a fixed order; 0 in rows that take no part, whatever
// the weight (0 times an infinity) and g_loss hold.
template <typename T>
__global__ void __launch_bounds__(256) ce_sum_parts_kernel(CeArgs a, const float* __restrict__ part, int n, int slots,
                                                           T* __restrict__ out) {
  __shared__ float sm[8][32];
  pdl_enter();
  const int i = blockIdx.x * 32 + threadIdx.x % 32, g = threadIdx.x / 32;
  float s = 0.f;
  if (i < n) {
#pragma unroll 4
    for (int k = g; k < slots; k += 8) s += part[(size_t)k * n + i];
  }
  sm[g][threadIdx.x % 32] = s;
  __syncthreads();
  if (g != 0 || i >= n) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) s += sm[k][threadIdx.x];
  store_as(out + i, ce_kept(a, i / a.dim) ? s : 0.f);
}

struct RowsPlan {
  int rn, vec, vt, chunk, chunks, blocks, td;
  size_t smem_value, smem_grad;
};

int pow2_at_least(int x) {
  int p = 1;
  while (p < x) p *= 2;
  return p;
}

// `vec`: columns per load, 4 or 1.
RowsPlan rows_plan(const nc_linear_ce* d, int vec) {
  RowsPlan r;
  r.rn = d->rows <= 1 ? 1 : d->rows <= 4 ? 4 : d->rows <= 8 ? 8 : 16;
  r.vec = vec;
  const size_t row = (size_t)d->dim * (d->dtype == NC_BF16 ? 2 : 4);
  r.chunk = kRowChunk;   // 16 classes of up to 4 KB fit a buffer
  while (r.chunk > 16 && (r.chunk * row > kRowChunkBytes || d->classes < r.chunk * 148)) r.chunk /= 2;
  r.vt = r.chunk >= 32 ? 4 : 2;
  r.chunks = (d->classes + r.chunk - 1) / r.chunk;
  r.blocks = r.chunks < 148 ? r.chunks : 148;
  r.td = pow2_at_least((d->dim + 3) / 4);
  const size_t ring = kRowBuffers * r.chunk * row, hs = (size_t)r.rn * d->dim * 4, sums = (size_t)r.rn * 4 * kRowThreads * 4;
  r.smem_value = ring + hs + (size_t)r.rn * kRowStats * 4;
  r.smem_grad = ring + hs + (size_t)r.rn * r.chunk * 4;
  if (r.smem_grad < sums) r.smem_grad = sums;   // the groups' sums of df
  return r;
}

// Few rows take the streaming kernels, which read the weight as it is; from then on the tensor
// cores are faster.  In bfloat16 they need no planes of the weight and win from
// 5 rows on.  Value and gradients of rows x 1024 x 50000: float32 16 rows 325 us here, 17 rows
// 367 us there; bfloat16 4 rows 130 us here, 5 rows 190 and 16 rows 174 us there.
bool on_tensor_cores(const nc_linear_ce* d) {
  return d->dim > kRowDim || d->rows > (d->dtype == NC_BF16 ? kRowsMostBf16 : kRowsMost);
}

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
      const RowsPlan r = rows_plan(d, 1);
      L.part = take((size_t)d->rows * r.blocks * sizeof(float2));
      L.zlabel = take((size_t)d->rows * 4);
      if (grad) L.df_part = take((size_t)r.blocks * d->rows * d->dim * 4);
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
  // what tile counts, block counts (int) and the tensor maps' strides (40 bits) hold
  const int64_t side = 1 << 24, rows = d->rows, dim = d->dim, classes = d->classes;
  if (rows > side || dim > side || classes > side || rows * classes > (int64_t)1 << 44 ||
      rows * dim > (int64_t)1 << 38 || classes * dim > (int64_t)1 << 38)
    return set_error(NC_ERR_UNSUPPORTED, "readout too large (rows %d, dim %d, classes %d)", d->rows, d->dim, d->classes);
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

CeArgs make_args(const nc_linear_ce* d, const void* f, const void* w, const void* b, const int32_t* labels, char* ws) {
  CeArgs a;
  a.features = f, a.weight = w, a.bias = b, a.labels = labels;
  a.rows = d->rows, a.dim = d->dim, a.classes = d->classes;
  a.ignore_index = d->ignore_index, a.reduction = d->reduction;
  a.status = reinterpret_cast<int32_t*>(ws);   // the layout's first word
  return a;
}

// What a call of the streaming kernels takes along.
struct RowsCall {
  RowArgs args;
  RowsPlan r;
  cudaStream_t st;
  // value
  float2* part;
  float* zlabel;
  // gradient
  const CeGrads* g;
  float* df_part;
};

template <typename T, int RN, int VEC, int VT>
nc_status launch_rows(const RowsCall& c) {
  if (!c.g) {
    auto k = ce_rows_value_kernel<T, RN, VEC, VT>;
    NC_CHECK(allow_smem((const void*)k, c.r.smem_value));
    PdlLaunch l(dim3(c.r.blocks), dim3(kRowThreads), c.r.smem_value, c.st);
    NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, k, c.args, c.part, c.zlabel));
    return launch_check("ce_rows_value_kernel launch");
  }
  auto k = ce_rows_grad_kernel<T, RN, VEC, VT>;
  NC_CHECK(allow_smem((const void*)k, c.r.smem_grad));
  PdlLaunch l(dim3(c.r.blocks), dim3(kRowThreads), c.r.smem_grad, c.st);
  NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, k, c.args, c.r.td, c.g->lse, c.g->g_loss, static_cast<T*>(c.g->weight),
                                   static_cast<T*>(c.g->bias), c.df_part));
  return launch_check("ce_rows_grad_kernel launch");
}

template <typename T, int RN>
nc_status launch_rows_of(const RowsCall& c) {
  if (c.r.vec == 1) return c.r.vt == 2 ? launch_rows<T, RN, 1, 2>(c) : launch_rows<T, RN, 1, 4>(c);
  return c.r.vt == 2 ? launch_rows<T, RN, 4, 2>(c) : launch_rows<T, RN, 4, 4>(c);
}

template <typename T>
nc_status launch_rows_as(const RowsCall& c) {
  return c.r.rn == 1   ? launch_rows_of<T, 1>(c)
         : c.r.rn == 4 ? launch_rows_of<T, 4>(c)
         : c.r.rn == 8 ? launch_rows_of<T, 8>(c)
                       : launch_rows_of<T, 16>(c);
}

// Vector loads and stores need rows and base addresses on multiples of four elements.
RowsCall rows_call(const nc_linear_ce* d, const CeArgs& a, const void* g_weight, cudaStream_t st) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.weight) | reinterpret_cast<uintptr_t>(g_weight);
  RowsCall c{};
  c.r = rows_plan(d, d->dim % 4 == 0 && at % (d->dtype == NC_BF16 ? 8 : 16) == 0 ? 4 : 1);
  c.args = RowArgs{a, c.r.chunk, c.r.chunks, reinterpret_cast<uintptr_t>(a.weight) % 16 == 0};
  c.st = st;
  return c;
}

// lse and row losses, then the reduced loss.  `grad`: the layout of the workspace.
nc_status value(const nc_linear_ce* d, const CeArgs& a, bool grad, float* loss, float* lse, char* ws, cudaStream_t st) {
  const CeLayout L = ce_layout(d, grad);
  const bool none = d->reduction == NC_REDUCE_NONE;
  float* row_loss = none ? loss : reinterpret_cast<float*>(ws + L.row_loss);
  if (on_tensor_cores(d)) return ce_tc_value(d, a, grad, lse, row_loss, none ? nullptr : loss, ws + L.tc, st);
  RowsCall c = rows_call(d, a, nullptr, st);
  c.part = reinterpret_cast<float2*>(ws + L.part), c.zlabel = reinterpret_cast<float*>(ws + L.zlabel);
  NC_CHECK(d->dtype == NC_BF16 ? launch_rows_as<__nv_bfloat16>(c) : launch_rows_as<float>(c));
  PdlLaunch l(dim3(1), dim3(512), 0, st);
  NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ce_rows_finish_kernel, a, c.r.blocks, (const float2*)c.part,
                                   (const float*)c.zlabel, lse, row_loss, none ? (float*)nullptr : loss));
  return launch_check("ce_rows_finish_kernel launch");
}

nc_status gradients(const nc_linear_ce* d, const CeArgs& a, const CeGrads& g, char* ws, cudaStream_t st) {
  const CeLayout L = ce_layout(d, true);
  if (on_tensor_cores(d)) return ce_tc_grad(d, a, g, ws + L.tc, st);
  RowsCall c = rows_call(d, a, g.weight, st);
  c.g = &g, c.df_part = g.features ? reinterpret_cast<float*>(ws + L.df_part) : nullptr;
  const bool bf16 = d->dtype == NC_BF16;
  NC_CHECK(bf16 ? launch_rows_as<__nv_bfloat16>(c) : launch_rows_as<float>(c));
  if (!g.features) return NC_OK;
  const int n = d->rows * d->dim;
  PdlLaunch l(dim3((n + 31) / 32), dim3(256), 0, st);
  if (bf16)
    NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ce_sum_parts_kernel<__nv_bfloat16>, a, (const float*)c.df_part, n, c.r.blocks,
                                     static_cast<__nv_bfloat16*>(g.features)));
  else
    NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ce_sum_parts_kernel<float>, a, (const float*)c.df_part, n, c.r.blocks,
                                     static_cast<float*>(g.features)));
  return launch_check("ce_sum_parts_kernel launch");
}

// What the value and the gradient share, once before either.
nc_status prepare(const nc_linear_ce* d, const CeArgs& a, bool grad, const float* g_loss, char* ws, cudaStream_t st) {
  const CeLayout L = ce_layout(d, grad);
  return on_tensor_cores(d) ? ce_tc_prepare(d, a, grad, g_loss, ws + L.tc, st) : NC_OK;
}

nc_status check_inputs(const nc_linear_ce* d, const void* features, const void* weight, const void* bias,
                       const int32_t* labels, const float* lse) {
  NC_CHECK(check_elems(d, features, "features"));
  NC_CHECK(check_elems(d, weight, "weight"));
  if (bias) NC_CHECK(check_elems(d, bias, "bias"));
  if (d->dtype == NC_BF16 && d->dim % 8 == 0 && reinterpret_cast<uintptr_t>(weight) % 16 != 0)
    return set_error(NC_ERR_INVALID, "a bfloat16 weight with a dim of whole 8s must start on 16 bytes");
  NC_CHECK(check_ptr(labels, "labels"));
  return check_ptr(lse, "lse");
}

nc_status check_grads(const nc_linear_ce* d, const void* g_features, const void* g_weight, const void* g_bias) {
  if (g_features) NC_CHECK(check_elems(d, g_features, "g_features"));
  if (g_weight) NC_CHECK(check_elems(d, g_weight, "g_weight"));
  if (g_bias) NC_CHECK(check_elems(d, g_bias, "g_bias"));
  return NC_OK;
}

// A buffer of a call.
struct Span {
  const void* p;
  size_t bytes;
  const char* name;
};

// Refuses what is written where something else of the call lies: the pieces of the gradient
// products read their inputs while earlier pieces' results are stored.
nc_status check_apart(std::initializer_list<Span> written, std::initializer_list<Span> read) {
  for (const Span* x = written.begin(); x != written.end(); ++x) {
    for (const Span* y = x + 1; y != written.end(); ++y)
      if (overlap(x->p, x->bytes, y->p, y->bytes))
        return set_error(NC_ERR_INVALID, "%s and %s overlap", x->name, y->name);
    for (const Span& y : read)
      if (overlap(x->p, x->bytes, y.p, y.bytes))
        return set_error(NC_ERR_INVALID, "%s and %s overlap", x->name, y.name);
  }
  return NC_OK;
}

// Bytes of the call's buffers.
struct Sizes {
  size_t features, weight, bias, rows, loss;
  explicit Sizes(const nc_linear_ce* d) {
    const size_t size = d->dtype == NC_BF16 ? 2 : 4;
    features = size * d->rows * d->dim, weight = size * d->classes * d->dim, bias = size * d->classes;
    rows = (size_t)d->rows * 4, loss = d->reduction == NC_REDUCE_NONE ? rows : 4;
  }
};

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
  const Sizes n(desc);
  NC_CHECK(check_apart({{loss, n.loss, "loss"}, {lse, n.rows, "lse"}, {d_ws, ws_bytes, "the workspace"}},
                       {{features, n.features, "features"}, {weight, n.weight, "weight"}, {bias, n.bias, "bias"},
                        {labels, n.rows, "labels"}}));
  char* ws = static_cast<char*>(d_ws);
  const CeArgs a = make_args(desc, features, weight, bias, labels, ws);
  NC_CHECK(prepare(desc, a, false, nullptr, ws, st));
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
  const Sizes n(desc);
  NC_CHECK(check_apart({{g_features, n.features, "g_features"}, {g_weight, n.weight, "g_weight"},
                        {g_bias, n.bias, "g_bias"}, {d_ws, ws_bytes, "the workspace"}},
                       {{features, n.features, "features"}, {weight, n.weight, "weight"}, {bias, n.bias, "bias"},
                        {labels, n.rows, "labels"}, {lse, n.rows, "lse"}, {g_loss, n.loss, "g_loss"}}));
  char* ws = static_cast<char*>(d_ws);
  const CeArgs a = make_args(desc, features, weight, bias, labels, ws);
  NC_CHECK(prepare(desc, a, true, g_loss, ws, st));
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
  const Sizes n(desc);
  NC_CHECK(check_apart({{loss, n.loss, "loss"}, {lse, n.rows, "lse"}, {g_features, n.features, "g_features"},
                        {g_weight, n.weight, "g_weight"}, {g_bias, n.bias, "g_bias"},
                        {d_ws, ws_bytes, "the workspace"}},
                       {{features, n.features, "features"}, {weight, n.weight, "weight"}, {bias, n.bias, "bias"},
                        {labels, n.rows, "labels"}}));
  char* ws = static_cast<char*>(d_ws);
  const CeArgs a = make_args(desc, features, weight, bias, labels, ws);
  NC_CHECK(prepare(desc, a, true, nullptr, ws, st));
  NC_CHECK(value(desc, a, true, loss, lse, ws, st));
  const CeGrads g{lse, nullptr, g_features, g_weight, g_bias};
  NC_CHECK(gradients(desc, a, g, ws, st));
  clear_error();
  return NC_OK;
}

}  // extern "C"
