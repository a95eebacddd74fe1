// nc_readout_tc.cu -- the readout's cross-entropy on the tensor cores (nc_tc.cuh).
//
//   value:     z tile = features weight^T; the epilogue keeps each row's (maximum, sum of exp)
//              over its half of the tile's classes, and the label's logit.
//   gradient:  the classes go by in pieces.  A piece's logits are computed again and their
//              epilogue writes dz = f_n (exp(z - lse) - onehot) as 16-bit planes; two
//              products read them soon after, dw = dz^T features (whole for the piece) and df
//              += dz weight (split over the piece's classes, parts summed in order at the end).
//              A piece's dz takes up to 160 MB beside 126 MB of L2 (2048 x 512 x 32768: 134 MB),
//              so part of it comes from memory again; pieces that fit L2 measured slower.
//
// float32 operands are two float16 planes each, scaled by a power of two that brings the
// tensor's largest finite value to [2^13, 2^14): an entry down to 2^-18 of it keeps float32's
// precision, smaller ones an absolute error of 2^-38 of it.  bfloat16 operands are used as
// they are, and dz is rounded to bfloat16 (2^-9 of an entry, as the products read it); their sums
// leave the accumulator every 128 k-tiles, logits every 32 (tc::kLongChunk).
// Bound by the tensor pipe where rows, dim and classes are large: 2048 x 512 x 32768 in float32
// takes 0.80 ms in a burst and 0.94 ms at the power cap (880 TFLOP/s of 16-bit products), 4096 x
// 1024 x 50000 in bfloat16 1.50 and 1.69 ms (993 TFLOP/s); the value alone of 4096 x 1024 x 50000
// takes 0.32 ms (1320 TFLOP/s). The tensor pipe is active 60 % of the value's time (2048 x 1024 x
// 16384 in bfloat16), 49 of dz's, 49 of dw's, 54 of df's; warps wait for their accumulators (long
// scoreboard).  Small calls are bound by nine dependent launches: 128 x 8 x 256
// 39 us as a graph.
//
// f_n = g_n / max |g| lies in [-1, 1], and dz has a fixed scale of 2^15: 22 bits down to 2^-18 (the low
// plane's smallest step is 2^-24), an absolute error of 2^-40 below. A class that is improbable in
// every row (p of 1e-11) therefore keeps one digit of its weight gradient.
#include <math.h>

#include "nc_readout.h"
#include "nc_tc.cuh"

namespace nc {

namespace {

constexpr int kPrepThreads = 256;
constexpr int kMaxBlocks = 296;        // blocks of the largest-value pass, per tensor
constexpr float kDzScale = 32768.f;    // dz planes hold dz 2^15 (|dz| <= 1)
constexpr int kChunk = 3;              // k-tiles (of 64) per accumulator beside float32 operands
constexpr int kLogitChunk = 32;        // of bfloat16 logits: the loss is float32 (see tc::kLongChunk)
constexpr size_t kPieceBytes = 160u << 20;  // most that dz of one piece takes
constexpr int kMaxSplits = 48;

// Device scalars of a call.
struct Scales {
  float w, w_inv, f, f_inv;   // 2^e and 2^-e of weight and features
  float g;                    // max |g_n|
  int kept;                   // rows that take part
  int blocks_done;            // of the value's last kernel
};

struct Plan {
  bool grad, bf16, copy_w;
  int pitch;                  // of the planes of features and weight
  int rows_pad;               // rows, whole 256s
  int classes_pad;            // classes, whole 256s
  int slots;                  // half tiles of classes
  int piece, pieces;          // classes per piece (whole 256s)
  // CTA pairs on 256 x 256 tiles, or one CTA on 128 x 128: the value's product, dz's, dw's, df's
  bool pair, pair_dz, pair_w, pair_f;
  int splits;                 // of df over a piece's classes
  size_t scales, max_part, w, f, bias, part, zlabel, fac, dz, df_part, db_part, total;
};

// Time of a product (m, n) over `depth` k-tiles, as 20ths of a pair's k-tile: its rounds of tiles
// over the SMs, each with a fixed part (fill, drain, epilogue) and its k-tiles.  The constants are
// fitted to the value's products of 512 .. 4096 rows, 256 .. 1024 columns and 4096 .. 16384 classes: a
// round of pairs takes 4.5 + 0.87 kt us in float32 and 1.8 + 0.4 kt (5 at least, the epilogue's) in
// bfloat16, one of single CTAs 1.5 + 0.8 kt and 1.2 + 0.34 kt.  So pairs win where there are many rounds (1024 x 512 x
// 16384: 67 us and 76), single CTAs where tiles are few (333 x 512 x 10007: 41 us and 37).
// dz's epilogue beside float32 operands (`dz`: both planes of 128 columns a thread) costs a pair
// more: 1024 x 512 x 16384 takes 245 us with pairs there and 233 without, 4096 x 1024 x 50000 4.3 ms
// and 4.6.
int64_t product_time(int64_t m, int64_t n, int64_t depth, bool pair, bool bf16, bool dz = false) {
  const int64_t side = pair ? 256 : 128, at = pair ? 74 : 148;
  const int64_t rounds = (((m + side - 1) / side) * ((n + side - 1) / side) + at - 1) / at;
  if (bf16) return rounds * (pair ? (depth > 8 ? 90 + 20 * depth : 250) : 60 + 17 * depth);
  return rounds * (pair ? (dz ? 300 : 100) + 20 * depth : (dz ? 64 : 34) + 18 * depth);
}

bool pairs_win(int64_t m, int64_t n, int64_t depth, bool bf16, bool dz = false) {
  return product_time(m, n, depth, true, bf16, dz) < product_time(m, n, depth, false, bf16, dz);
}

// Pieces, splits and tiles by product_time.
// 2048 x 512 x 32768 in float32: five pieces of 26 tiles of 256 classes, which fit L2, leave a
// third of the pairs idle in dw and take 949 us; the choice here takes 760 to 780. Splits keep SMs busy
// in df where it has few tiles: 333 x 128 x 10007 (all by pairs) took 79 us with them priced at the
// traffic of their parts, 87 us at a flat 4 k-tiles each (which left df to 18 CTAs).
void choose_pieces(const nc_linear_ce* d, int planes, Plan* p) {
  auto ceil_div = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
  const int bk = 64;
  const int tiles = p->classes_pad / 256;
  const size_t tile_bytes = (size_t)p->rows_pad * 256 * 2 * planes;
  int64_t most = (int64_t)(kPieceBytes / tile_bytes);
  if (most < 1) most = 1;
  const int64_t fewest = ceil_div(tiles, most);
  const int64_t launch = 240;   // a launch's start and end
  int64_t best = INT64_MAX;
  for (int64_t pieces = fewest; pieces < fewest + 4 && pieces <= tiles; ++pieces) {
    const int64_t t = ceil_div(tiles, pieces), classes = 256 * t;
    const bool pair_dz = pairs_win(d->rows, classes, ceil_div(d->dim, bk), p->bf16, true);
    const bool pair_w = pairs_win(classes, d->dim, ceil_div(d->rows, bk), p->bf16);
    const int64_t one = product_time(d->rows, classes, ceil_div(d->dim, bk), pair_dz, p->bf16, true) +
                        product_time(classes, d->dim, ceil_div(d->rows, bk), pair_w, p->bf16) + 3 * launch;
    for (int splits = 1; splits <= kMaxSplits && splits <= t; ++splits) {
      const int64_t depth = ceil_div(t * (256 / bk), splits);
      for (int pair_f = 0; pair_f < 2; ++pair_f) {
        // splits as rows of tiles; a split's part of df is written and read once: about a k-tile
        // for 250,000 elements
        const int64_t side = pair_f ? 256 : 128;
        const int64_t all = (one + product_time(ceil_div(d->rows, side) * side * splits, d->dim, depth, pair_f, p->bf16)) *
                                ceil_div(tiles, t) +
                            10 * splits * ((int64_t)d->rows * p->pitch / 250000 + 1);
        if (all < best) {
          best = all, p->piece = (int)classes, p->splits = splits;
          p->pair_dz = pair_dz, p->pair_w = pair_w, p->pair_f = pair_f;
        }
      }
    }
  }
  p->pieces = (int)ceil_div(tiles, p->piece / 256);
}

Plan make_plan(const nc_linear_ce* d, bool grad) {
  Plan p{};
  p.grad = grad;
  p.bf16 = d->dtype == NC_BF16;
  p.copy_w = !p.bf16 || d->dim % 8 != 0;   // else the weight is read where it is
  p.pitch = (d->dim + 7) / 8 * 8;
  p.rows_pad = (d->rows + 255) / 256 * 256;
  p.classes_pad = (d->classes + 255) / 256 * 256;
  p.pair = pairs_win(d->rows, d->classes, (d->dim + 63) / 64, p.bf16);
  const int tile = p.pair ? 256 : 128;
  p.slots = (d->classes + tile - 1) / tile * 2;
  const int planes = p.bf16 ? 1 : 2;
  choose_pieces(d, planes, &p);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += pad256(bytes);
    return o;
  };
  p.scales = take(sizeof(Scales));
  p.max_part = take(2 * kMaxBlocks * 4);
  if (p.copy_w) p.w = take((size_t)d->classes * p.pitch * 2 * planes);
  p.f = take((size_t)d->rows * p.pitch * 2 * planes);
  p.bias = take((size_t)p.classes_pad * 4);
  p.part = take((size_t)p.slots * p.rows_pad * sizeof(float2));
  p.zlabel = take((size_t)d->rows * 4);
  if (grad) {
    p.fac = take((size_t)d->rows * 4);
    p.dz = take((size_t)p.rows_pad * p.piece * 2 * planes);
    p.df_part = take((size_t)p.splits * d->rows * p.pitch * 4);
    p.db_part = take((size_t)(p.rows_pad / 32) * p.classes_pad * 4);
  }
  p.total = at;
  return p;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// ---- preparation ---------------------------------------------------------------------------

// Largest finite magnitude per block: blocks [0, kMaxBlocks) of the weight, the rest of the
// features' rows that take part.
__global__ void __launch_bounds__(kPrepThreads) ce_max_kernel(CeArgs a, float* __restrict__ part) {
  __shared__ float red[kPrepThreads / 32];
  pdl_enter();
  const bool of_w = blockIdx.x < kMaxBlocks;
  const float* x = static_cast<const float*>(of_w ? a.weight : a.features);
  const int64_t n = (int64_t)(of_w ? a.classes : a.rows) * a.dim;
  const int64_t step = (int64_t)kMaxBlocks * kPrepThreads, i0 = (blockIdx.x % kMaxBlocks) * kPrepThreads + threadIdx.x;
  float m = 0.f;
  auto see = [&](float v) {
    v = fabsf(v);
    if (v <= 3.402823466e38f) m = fmaxf(m, v);   // not NaN, not an infinity
  };
  if (of_w && n % 4 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0) {
    const float4* x4 = reinterpret_cast<const float4*>(x);
#pragma unroll 4
    for (int64_t i = i0; i < n / 4; i += step) {
      const float4 v = x4[i];
      see(v.x), see(v.y), see(v.z), see(v.w);
    }
  } else {
    for (int64_t i = i0; i < n; i += step)
      if (of_w || ce_kept(a, (int)(i / a.dim))) see(x[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kPrepThreads / 32; ++i) m = fmaxf(m, red[i]);
    part[blockIdx.x] = m;
  }
}

// Exponent e of the scale: largest value x 2^e in [2^13, 2^14), within what float32 holds.
__device__ __forceinline__ int scale_exponent(float largest) {
  if (largest == 0.f) return 0;
  const int e = 13 - ((int)(__float_as_uint(largest) >> 23) - 127);
  return min(e, 120);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Eight values of a row as 16-bit planes (or bfloat16, or float32 -> bfloat16-wide copies).
template <typename T>
__device__ __forceinline__ void put8(const T* src, int left, bool wide, float scale, bool bf16, uint16_t* out,
                                     int64_t plane) {
  float v[8];
  if (wide && left >= 8) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      const uint4 q = *reinterpret_cast<const uint4*>(src);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? to_f32(src[i]) : 0.f;
  }
  uint16_t h[8], l[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (bf16)
      h[i] = __bfloat16_as_ushort(__float2bfloat16_rn(v[i]));
    else
      tc::split_f16(v[i] * scale, &h[i], &l[i]);
  }
  *reinterpret_cast<uint4*>(out) =
      make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
  if (!bf16)
    *reinterpret_cast<uint4*>(out + plane) =
        make_uint4(l[0] | l[1] << 16, l[2] | l[3] << 16, l[4] | l[5] << 16, l[6] | l[7] << 16);
}

// By one block: how many rows take part, f_n = g_n / max |g| of every row (0 where it takes
// no part) and max |g|.
__device__ void row_factors(const CeArgs& a, const float* g_loss, float* fac, Scales* scales) {
  __shared__ float red[kPrepThreads / 32];
  const int n = count_kept(a);
  if (threadIdx.x == 0) scales->kept = n;
  if (!fac) return;
  const bool each = a.reduction == NC_REDUCE_NONE && g_loss;
  const float all = (g_loss && !each ? g_loss[0] : 1.f) / (a.reduction == NC_REDUCE_MEAN ? (float)max(n, 1) : 1.f);
  float m = fabsf(all);
  if (each) {
    m = 0.f;
    for (int i = threadIdx.x; i < a.rows; i += kPrepThreads)
      if (ce_kept(a, i)) m = fmaxf(m, fabsf(g_loss[i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int i = 0; i < kPrepThreads / 32; ++i) m = fmaxf(m, red[i]);
  }
  for (int i = threadIdx.x; i < a.rows; i += kPrepThreads) {
    const float g = each ? g_loss[i] : all;
    fac[i] = !ce_kept(a, i) ? 0.f : m > 0.f ? g / m : g;   // else g is 0 or NaN
  }
  if (threadIdx.x == 0) scales->g = m;
}

// Features, bias and (copy_w) weight in the products' form; the last block the row factors.  Rows that take no part become
// zeros; the bias of the classes past the end is -inf.
template <typename T>
__global__ void __launch_bounds__(kPrepThreads) ce_planes_kernel(CeArgs a, int copy_w, int pitch, int classes_pad,
                                                                 int wide_w, int wide_f,
                                                                 const float* __restrict__ max_part, Scales* scales,
                                                                 uint16_t* __restrict__ w,
                                                                 uint16_t* __restrict__ f, float* __restrict__ bias,
                                                                 const float* __restrict__ g_loss,
                                                                 float* __restrict__ fac) {
  constexpr bool bf16 = sizeof(T) == 2;
  __shared__ float red[2][kPrepThreads / 32];
  pdl_enter();
  if (blockIdx.x == gridDim.x - 1) {
    row_factors(a, g_loss, fac, scales);
    return;
  }
  float sw = 1.f, sf = 1.f;
  if constexpr (!bf16) {
    float m[2] = {0.f, 0.f};
    for (int k = 0; k < 2; ++k) {
      for (int i = threadIdx.x; i < kMaxBlocks; i += kPrepThreads) m[k] = fmaxf(m[k], max_part[k * kMaxBlocks + i]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m[k] = fmaxf(m[k], __shfl_xor_sync(0xffffffffu, m[k], o));
      if ((threadIdx.x & 31) == 0) red[k][threadIdx.x >> 5] = m[k];
    }
    __syncthreads();
    for (int k = 0; k < 2; ++k) {
      m[k] = red[k][0];
      for (int i = 1; i < kPrepThreads / 32; ++i) m[k] = fmaxf(m[k], red[k][i]);
    }
    sw = pow2(scale_exponent(m[0])), sf = pow2(scale_exponent(m[1]));
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    scales->w = sw, scales->f = sf, scales->w_inv = 1.f / sw, scales->f_inv = 1.f / sf;
    scales->blocks_done = 0;
    *a.status = 0;
  }
  const int64_t step = (int64_t)(gridDim.x - 1) * kPrepThreads, i0 = (int64_t)blockIdx.x * kPrepThreads + threadIdx.x;
  const int per = pitch / 8;
  const int64_t nf = (int64_t)a.rows * per, nw = copy_w ? (int64_t)a.classes * per : 0;
  for (int64_t i = i0; i < nf; i += step) {
    const int row = (int)(i / per), c = (int)(i - (int64_t)row * per) * 8;
    const T* src = static_cast<const T*>(a.features) + (size_t)row * a.dim + c;
    put8<T>(src, ce_kept(a, row) ? a.dim - c : 0, wide_f, sf, bf16, f + (size_t)row * pitch + c,
            (int64_t)a.rows * pitch);
  }
  for (int64_t i = i0; i < classes_pad; i += step)
    bias[i] = i >= a.classes ? -INFINITY : a.bias ? to_f32(static_cast<const T*>(a.bias)[i]) : 0.f;
#pragma unroll 2
  for (int64_t i = i0; i < nw; i += step) {
    const int row = (int)(i / per), c = (int)(i - (int64_t)row * per) * 8;
    const T* src = static_cast<const T*>(a.weight) + (size_t)row * a.dim + c;
    put8<T>(src, a.dim - c, wide_w, sw, bf16, w + (size_t)row * pitch + c, (int64_t)a.classes * pitch);
  }
}

// ---- value ---------------------------------------------------------------------------------

// 2^t, and e^d.  The hardware's 2^t is good to 2 ulp; exp_near() adds what rounding d log2(e)
// lost, so that large |d| keep float32's precision.  d is at least -200 (e^d is 0 there).
__device__ __forceinline__ float exp2_fast(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f, kLog2eLow = (float)(1.4426950408889634 - (double)1.4426950408889634f);
__device__ __forceinline__ float exp_fast(float d) { return exp2_fast(d * kLog2e); }
__device__ __forceinline__ float exp_near(float d) {
  const float t = d * kLog2e, r = fmaf(d, kLog2eLow, fmaf(d, kLog2e, -t)), e = exp2_fast(t);
  return fmaf(e, r * 0.69314718f, e);
}

// The tile's bias into the warp's scratch.
template <int COLS>
__device__ __forceinline__ void stage_bias(const float* bias, float* scratch) {
  const int lane = threadIdx.x & 31;
  if constexpr (COLS == 128)
    reinterpret_cast<float4*>(scratch)[lane] = reinterpret_cast<const float4*>(bias)[lane];
  else
    reinterpret_cast<float2*>(scratch)[lane] = reinterpret_cast<const float2*>(bias)[lane];
}

struct ValueEpilogue {
  CeArgs a;
  const Scales* scales;
  const float* bias;
  float2* part;      // (slots, rows_pad)
  float* zlabel;
  int rows_pad;

  struct State {
    float sw, sf;
    int label;            // within the half tile, or out of it
    const float* bias;
  };
  template <int COLS>
  __device__ __forceinline__ State begin(const tc::Tile&, int row, int col, uint8_t* patch) const {
    stage_bias<COLS>(bias + col, reinterpret_cast<float*>(patch));
    return State{scales->w_inv, scales->f_inv, row < a.rows ? a.labels[row] - col : -1, reinterpret_cast<const float*>(patch)};
  }
  template <int COLS>
  __device__ __forceinline__ void run(const State& st, const tc::Tile&, int row, int col, float (&z)[COLS]) const {
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < COLS; j += 4) {
      const float4 q = *reinterpret_cast<const float4*>(st.bias + j);
      const float b[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        z[j + e] = fmaf(z[j + e] * st.sw, st.sf, b[e]);
        m[e] = fmaxf(m[e], z[j + e]);
      }
    }
    const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), base = top == -INFINITY ? 0.f : top;
    const bool mine = st.label >= 0 && st.label < COLS;
    float zl = 0.f;
    if (__any_sync(0xffffffffu, mine)) {
#pragma unroll
      for (int j = 0; j < COLS; ++j)
        if (j == st.label) zl = z[j];
    }
#pragma unroll
    for (int j = 0; j < COLS; ++j) s[j & 3] += exp_fast(z[j] - base);
    if (row >= a.rows) return;
    part[(size_t)(col / COLS) * rows_pad + row] = make_float2(top, (s[0] + s[1]) + (s[2] + s[3]));
    if (mine) zlabel[row] = zl;
  }
};

// 32 rows per block, a lane each; the warps split the slots and meet in shared memory.  The
// last block to finish adds up the row losses (in order, whichever block that is), except
// with NC_REDUCE_NONE.
__global__ void __launch_bounds__(1024) ce_finish_kernel(CeArgs a, int slots, int rows_pad,
                                                         const float2* __restrict__ part,
                                                         const float* __restrict__ zlabel, Scales* scales,
                                                         float* __restrict__ lse, float* __restrict__ row_loss,
                                                         float* __restrict__ loss) {
  __shared__ float2 sm[32][32];
  __shared__ double red[32];
  __shared__ bool last;
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x * 32 + lane;
  float2 x = make_float2(-INFINITY, 0.f);
#pragma unroll 4
  for (int s = warp; s < slots; s += 32) x = lse_merge(x, part[(size_t)s * rows_pad + row]);
  sm[warp][lane] = x;
  __syncthreads();
  x = sm[lane][warp];   // a warp per row now
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    x = lse_merge(x, make_float2(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o)));
  if (lane == 0 && blockIdx.x * 32 + warp < a.rows) finish_row(a, blockIdx.x * 32 + warp, x, zlabel, lse, row_loss);
  if (!loss) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(&scales->blocks_done, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double s = 0.0;
  for (int i = threadIdx.x; i < a.rows; i += 1024) s += *((volatile const float*)row_loss + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) red[warp] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int i = 0; i < 32; ++i) t += red[i];
    loss[0] = (float)(a.reduction == NC_REDUCE_MEAN ? t / (double)max(scales->kept, 1) : t);
  }
}

// ---- gradient ------------------------------------------------------------------------------

template <bool BF16>
struct DzEpilogue {   // its sums for db cost 8 % of a call in bfloat16 (4096 x 1024 x 50000)
  CeArgs a;
  const Scales* scales;
  const float* bias;
  const float* lse;
  const float* fac;
  uint16_t* dz;        // (planes, rows, piece)
  float* db_part;      // (rows_pad / 32, classes_pad) or null
  int v0, piece, classes_pad;

  struct State {
    float sw, sf, f, lse;
    int label;
    uint8_t* patch;   // the bias first
  };
  template <int COLS>
  __device__ __forceinline__ State begin(const tc::Tile&, int row, int col, uint8_t* patch) const {
    stage_bias<COLS>(bias + v0 + col, reinterpret_cast<float*>(patch));
    const bool in = row < a.rows;
    float f = in ? fac[row] : 0.f, l = in ? lse[row] : 0.f;
    if (f == 0.f)
      l = INFINITY;          // p = 0
    else if (!(l > -INFINITY))
      f = NAN, l = 0.f;      // a bad label, no class left, or NaN among the logits
    return State{scales->w_inv, scales->f_inv, f, l, in ? a.labels[row] - v0 - col : -1, patch};
  }
  template <int COLS>
  __device__ __forceinline__ void run(const State& st, const tc::Tile&, int row, int col, float (&z)[COLS]) const {
#pragma unroll
    for (int j = 0; j < COLS; j += 4) {
      const float4 q = *reinterpret_cast<const float4*>(st.patch + 4 * j);
      const float b[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float d = fmaxf(fmaf(z[j + e] * st.sw, st.sf, b[e]) - st.lse, -200.f);
        z[j + e] = st.f * (BF16 ? exp_fast(d) : exp_near(d));
      }
    }
    if (__any_sync(0xffffffffu, st.label >= 0 && st.label < COLS)) {
#pragma unroll
      for (int j = 0; j < COLS; ++j)
        if (j == st.label) z[j] -= st.f;
    }
    const int lane = threadIdx.x & 31, rows = min(32, a.rows - (row - lane));
    uint16_t* out = dz + (size_t)(row - lane) * piece + col;
#pragma unroll
    for (int j = 0; j < COLS; j += 64) {
#pragma unroll
      for (int k = 0; k < (BF16 ? 1 : 2); ++k) {   // a plane at a time
        uint32_t v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float x = z[j + 2 * i], y = z[j + 2 * i + 1];
          if constexpr (BF16) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
            v[i] = *reinterpret_cast<const uint32_t*>(&b);
          } else {
            uint32_t h, lo;
            tc::split_f16x2(x * kDzScale, y * kDzScale, &h, &lo);
            v[i] = k == 0 ? h : lo;
          }
        }
        tc::patch_store<64>(st.patch, v, out + (size_t)k * a.rows * piece + j, piece, rows, 8);
      }
    }
    if (db_part) {
      int first;
      warp_sums(z, lane, &first);
      float* o = db_part + (size_t)(row / 32) * classes_pad + v0 + col + first;
#pragma unroll
      for (int i = 0; i < COLS / 32; ++i) o[i] = z[i];
    }
  }
};

// dw of a piece, written once.
template <typename T>
struct WeightEpilogue {
  const Scales* scales;
  T* out;          // of the piece's first class
  int classes, dim;
  bool wide;       // rows on 16 bytes
  struct State {
    float scale, g;
    uint8_t* patch;
  };
  template <int COLS>
  __device__ __forceinline__ State begin(const tc::Tile&, int, int, uint8_t* patch) const {
    return State{scales->f_inv * (sizeof(T) == 4 ? 1.f / kDzScale : 1.f), scales->g, patch};
  }
  template <int COLS>
  __device__ __forceinline__ void run(const State& st, const tc::Tile&, int row, int col, float (&v)[COLS]) const {
    const int lane = threadIdx.x & 31, row0 = row - lane, rows = min(32, classes - row0);
    if (rows <= 0) return;
    constexpr int kGroup = sizeof(T) == 4 ? 32 : 64;   // columns in 128 bytes
#pragma unroll
    for (int j = 0; j < COLS; j += kGroup) {
      if (col + j >= dim) break;
      const int cols = min(kGroup, dim - col - j);
#pragma unroll
      for (int e = 0; e < kGroup; ++e) v[j + e] = v[j + e] * st.scale * st.g;   // a power of two first: exact
      if (wide) {
        T* o = out + (size_t)row0 * dim + col + j;
        if constexpr (sizeof(T) == 4) {
          tc::patch_store_f32(st.patch, v + j, o, dim, rows, cols / 4, false);
        } else {
          uint32_t q[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[j + 2 * i], v[j + 2 * i + 1]);
            q[i] = *reinterpret_cast<const uint32_t*>(&b);
          }
          tc::patch_store<64>(st.patch, q, reinterpret_cast<uint16_t*>(o), dim, rows, cols / 8);
        }
      } else if (row < classes) {
        T* o = out + (size_t)row * dim + col + j;
#pragma unroll
        for (int e = 0; e < kGroup; ++e)
          if (e < cols) store_as(o + e, v[j + e]);
      }
    }
  }
};

// df of a piece and split, added to that split's part (one CTA owns an element).
struct FeatureEpilogue {
  const Scales* scales;
  float* part;     // (splits, rows, pitch); the pitch is whole 8s
  int rows, dim, pitch, first;
  float mul;
  struct State {
    float scale;
    uint8_t* patch;
  };
  template <int COLS>
  __device__ __forceinline__ State begin(const tc::Tile&, int, int, uint8_t* patch) const {
    return State{scales->w_inv * mul, patch};
  }
  template <int COLS>
  __device__ __forceinline__ void run(const State& st, const tc::Tile& x, int row, int col, float (&v)[COLS]) const {
    const int lane = threadIdx.x & 31, row0 = row - lane, count = min(32, rows - row0);
    if (count <= 0) return;
    float* o = part + ((size_t)x.split * rows + row0) * pitch + col;
#pragma unroll
    for (int j = 0; j < COLS; j += 32) {
      if (col + j >= pitch) break;
#pragma unroll
      for (int e = 0; e < 32; ++e) v[j + e] *= st.scale;
      tc::patch_store_f32(st.patch, v + j, o + j, pitch, count, min(8, (pitch - col - j) / 4), !first);
    }
  }
};

// df: the splits' parts in order; 0 in rows that take no part, whatever the weight (0 times an
// infinity) and g_loss hold.
template <typename T>
__global__ void __launch_bounds__(256) ce_features_kernel(CeArgs a, const float* __restrict__ part, int splits,
                                                          int pitch, const Scales* __restrict__ scales,
                                                          T* __restrict__ out) {
  pdl_enter();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)a.rows * a.dim) return;
  const int row = (int)(i / a.dim), c = (int)(i - (int64_t)row * a.dim);
  float s = 0.f;
#pragma unroll 8
  for (int k = 0; k < splits; ++k) s += part[((size_t)k * a.rows + row) * pitch + c];
  store_as(out + i, ce_kept(a, row) ? s * scales->g : 0.f);
}

template <typename T>
__global__ void __launch_bounds__(256) ce_bias_kernel(const float* __restrict__ part, int groups, int classes,
                                                      int classes_pad, const Scales* __restrict__ scales,
                                                      T* __restrict__ out) {
  pdl_enter();
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v >= classes) return;
  float s = 0.f;
#pragma unroll 8
  for (int k = 0; k < groups; ++k) s += part[(size_t)k * classes_pad + v];
  store_as(out + v, s * scales->g);
}

// ---- launches ------------------------------------------------------------------------------

template <typename T>
struct Call {
  static constexpr int PL = sizeof(T) == 2 ? 1 : 2;
  const nc_linear_ce* d;
  const CeArgs& a;
  Plan p;
  char* ws;
  cudaStream_t st;

  template <typename U>
  U* at(size_t o) const {
    return reinterpret_cast<U*>(ws + o);
  }
  Scales* scales() const { return at<Scales>(p.scales); }

  template <int BN, int CG, int EW>
  tc::Problem problem(int m, int n, int k, int splits) const {
    tc::Problem q{};
    q.m = m, q.n = n, q.k = k, q.batch = 1, q.splits = splits, q.bf16 = p.bf16;
    tc::set_tiles<BN, CG>(&q);
    q.chunk = PL == 1 ? tc::kLongChunk : kChunk;
    q.status = a.status;
    return q;
  }

  // Operands: rows of features or weight (k = dim contiguous), or with their columns as the
  // own index and rows as k.
  template <int BN, int CG, int EW>
  nc_status features_op(tc::Problem* q, bool is_a, bool by_column) const {
    return tc::make_operand<PL, BN, CG, EW>(q, is_a, at<void>(p.f), by_column, by_column ? d->dim : d->rows,
                                    by_column ? d->rows : d->dim, p.pitch, (int64_t)d->rows * p.pitch, 1,
                                    (int64_t)PL * d->rows * p.pitch);
  }
  template <int BN, int CG, int EW>
  nc_status weight_op(tc::Problem* q, bool by_column) const {
    const void* base = p.copy_w ? at<void>(p.w) : a.weight;
    const int pitch = p.copy_w ? p.pitch : d->dim;
    return tc::make_operand<PL, BN, CG, EW>(q, false, base, by_column, by_column ? d->dim : d->classes,
                                    by_column ? d->classes : d->dim, pitch, (int64_t)d->classes * pitch, 1,
                                    (int64_t)PL * d->classes * pitch);
  }
  template <int BN, int CG, int EW>
  nc_status dz_op(tc::Problem* q, bool by_column) const {
    return tc::make_operand<PL, BN, CG, EW>(q, true, at<void>(p.dz), by_column, by_column ? p.piece : d->rows,
                                    by_column ? d->rows : p.piece, p.piece, (int64_t)d->rows * p.piece, 1,
                                    (int64_t)PL * d->rows * p.piece);
  }

  nc_status prepare(const float* g_loss) const {
    if (PL == 2) {
      PdlLaunch l(dim3(2 * kMaxBlocks), dim3(kPrepThreads), 0, st);
      NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ce_max_kernel, a, at<float>(p.max_part)));
      NC_CHECK(launch_check("ce_max_kernel launch"));
    }
    const int64_t items = ((int64_t)d->rows + (p.copy_w ? d->classes : 0)) * (p.pitch / 8);
    int64_t blocks = (items + kPrepThreads - 1) / kPrepThreads;
    if (blocks > 148 * 16) blocks = 148 * 16;
    PdlLaunch l(dim3((unsigned)blocks + 1), dim3(kPrepThreads), 0, st);
    const int even = d->dim % 8 == 0;
    NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ce_planes_kernel<T>, a, (int)p.copy_w, p.pitch, p.classes_pad,
                                     (int)(even && aligned16(a.weight)), (int)(even && aligned16(a.features)),
                                     (const float*)at<float>(p.max_part), scales(), at<uint16_t>(p.w),
                                     at<uint16_t>(p.f), at<float>(p.bias), g_loss,
                                     p.grad ? at<float>(p.fac) : nullptr));
    return launch_check("ce_planes_kernel launch");
  }

  template <int BN, int CG, int EW>
  nc_status value_product() const {
    tc::Problem q = problem<BN, CG, EW>(d->rows, d->classes, d->dim, 1);
    NC_CHECK((features_op<BN, CG, EW>(&q, true, false)));
    NC_CHECK((weight_op<BN, CG, EW>(&q, false)));
    if (PL == 1) q.chunk = kLogitChunk;
    const ValueEpilogue e{a, scales(), at<float>(p.bias), at<float2>(p.part), at<float>(p.zlabel), p.rows_pad};
    return tc::launch_product<PL, BN, CG, EW>(q, e, st, "readout value product launch");
  }

  nc_status value(float* lse, float* row_loss, float* loss) const {
    NC_CHECK(p.pair ? (value_product<256, 2, 8>()) : (value_product<128, 1, 8>()));
    PdlLaunch l(dim3((d->rows + 31) / 32), dim3(1024), 0, st);
    NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ce_finish_kernel, a, p.slots, p.rows_pad,
                                     (const float2*)at<float2>(p.part), (const float*)at<float>(p.zlabel), scales(),
                                     lse, row_loss, loss));
    return launch_check("ce_finish_kernel launch");
  }

  template <int BN, int CG, int EW>
  nc_status dz_product(const CeGrads& g, int v0, int width) const {
    tc::Problem q = problem<BN, CG, EW>(d->rows, width, d->dim, 1);
    NC_CHECK((features_op<BN, CG, EW>(&q, true, false)));
    NC_CHECK((weight_op<BN, CG, EW>(&q, false)));
    q.b_n0 = v0;
    if (PL == 1) q.chunk = kLogitChunk;
    const DzEpilogue<PL == 1> e{a,     scales(), at<float>(p.bias), g.lse,  at<float>(p.fac), at<uint16_t>(p.dz),
                                g.bias ? at<float>(p.db_part) : nullptr, v0, p.piece, p.classes_pad};
    return tc::launch_product<PL, BN, CG, EW>(q, e, st, "readout logit gradient launch");
  }

  template <int BN, int CG, int EW>
  nc_status weight_product(const CeGrads& g, int v0, int classes) const {
    tc::Problem q = problem<BN, CG, EW>(classes, d->dim, d->rows, 1);
    NC_CHECK((dz_op<BN, CG, EW>(&q, true)));
    NC_CHECK((features_op<BN, CG, EW>(&q, false, true)));
    T* out = static_cast<T*>(g.weight) + (size_t)v0 * d->dim;
    const bool wide = reinterpret_cast<uintptr_t>(out) % 16 == 0 && (size_t)d->dim * sizeof(T) % 16 == 0;
    const WeightEpilogue<T> e{scales(), out, classes, d->dim, wide};
    return tc::launch_product<PL, BN, CG, EW>(q, e, st, "readout weight gradient launch");
  }

  template <int BN, int CG, int EW>
  nc_status feature_product(const CeGrads& g, int v0, int width) const {
    tc::Problem q = problem<BN, CG, EW>(d->rows, d->dim, width, p.splits);
    NC_CHECK((dz_op<BN, CG, EW>(&q, false)));
    NC_CHECK((weight_op<BN, CG, EW>(&q, true)));
    q.b_k0 = v0;
    const FeatureEpilogue e{scales(), at<float>(p.df_part), d->rows, d->dim, p.pitch, v0 == 0,
                            PL == 1 ? 1.f : 1.f / kDzScale};
    return tc::launch_product<PL, BN, CG, EW>(q, e, st, "readout feature gradient launch");
  }

  nc_status gradients(const CeGrads& g) const {
    for (int k = 0; k < p.pieces; ++k) {
      const int v0 = k * p.piece;
      // the last piece may be shorter; `width` is whole tiles
      const int width = p.classes_pad - v0 < p.piece ? p.classes_pad - v0 : p.piece;
      const int classes = d->classes - v0 < width ? d->classes - v0 : width;
      NC_CHECK(p.pair_dz ? (dz_product<256, 2, 8>(g, v0, width)) : (dz_product<128, 1, 8>(g, v0, width)));
      if (g.weight)
        NC_CHECK(p.pair_w ? (weight_product<256, 2, 8>(g, v0, classes)) : (weight_product<128, 1, 8>(g, v0, classes)));
      if (g.features)
        NC_CHECK(p.pair_f ? (feature_product<256, 2, 8>(g, v0, width)) : (feature_product<128, 1, 8>(g, v0, width)));
    }
    if (g.features) {
      const int64_t n = (int64_t)d->rows * d->dim;
      PdlLaunch l(dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st);
      NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ce_features_kernel<T>, a, (const float*)at<float>(p.df_part), p.splits,
                                       p.pitch, (const Scales*)scales(),
                                       static_cast<T*>(g.features)));
      NC_CHECK(launch_check("ce_features_kernel launch"));
    }
    if (g.bias) {
      PdlLaunch l(dim3((d->classes + 255) / 256), dim3(256), 0, st);
      NC_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, ce_bias_kernel<T>, (const float*)at<float>(p.db_part), (d->rows + 31) / 32,
                                       d->classes, p.classes_pad, (const Scales*)scales(), static_cast<T*>(g.bias)));
      NC_CHECK(launch_check("ce_bias_kernel launch"));
    }
    return NC_OK;
  }
};

}  // namespace

size_t ce_tc_bytes(const nc_linear_ce* d, bool grad) { return make_plan(d, grad).total; }

#define NC_TC_CALL(GRAD, WHAT)                                                                       \
  const Plan plan = make_plan(d, GRAD);                                                              \
  return plan.bf16 ? Call<__nv_bfloat16>{d, a, plan, ws, st}.WHAT : Call<float>{d, a, plan, ws, st}.WHAT

nc_status ce_tc_prepare(const nc_linear_ce* d, const CeArgs& a, bool grad, const float* g_loss, char* ws,
                        cudaStream_t st) {
  NC_TC_CALL(grad, prepare(g_loss));
}

nc_status ce_tc_value(const nc_linear_ce* d, const CeArgs& a, bool grad, float* lse, float* row_loss, float* loss,
                      char* ws, cudaStream_t st) {
  NC_TC_CALL(grad, value(lse, row_loss, loss));
}

nc_status ce_tc_grad(const nc_linear_ce* d, const CeArgs& a, const CeGrads& g, char* ws, cudaStream_t st) {
  NC_TC_CALL(true, gradients(g));
}

}  // namespace nc
