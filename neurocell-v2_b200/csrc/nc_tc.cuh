// nc_tc.cuh -- products of 16-bit matrices on the tensor cores (tcgen05, accumulators in
// tensor memory), with the caller's epilogue on float32 accumulators in registers.
//
// float32 operands come as two float16 planes: x s = hi + lo with hi = fp16(x s) and
// lo = fp16(x s - hi), s a power of two.  A product takes lo hi + hi lo + hi hi; what is left
// out (lo lo) and the rounding of lo are 2^-24 and 2^-23 of a factor, so the result is as
// exact as float32 multiplications, for three 16-bit products (three bfloat16 planes would
// take six).  bfloat16 operands are one plane and one product.
//
// The tensor core adds in float32 but not to nearest, which shows in long sums; the accumulator is
// therefore drained every `chunk` k-tiles into float32 registers (added to nearest there) while
// the other half of tensor memory takes the next chunk.  One plane has long chunks (kLongChunk),
// and most of its products are one.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "nc_common.cuh"
#include "nc_errors.h"

namespace nc {
namespace tc {

constexpr int kBM = 128;            // rows of a tile per CTA: one tensor-memory lane each
constexpr int kBK = 64;             // k of a stage: a swizzled row of 128 bytes (rows of 64 took products 6 % longer)
// The tensor core adds toward zero: where a chunk's terms share a sign (the diagonal of a Gram
// matrix) the sum of a k-tile comes out short by about 2^-22 of itself.  Given back, the
// orthogonalised 96 x 4000 matrix is off by 1.3e-6 instead of 1.7e-6.
constexpr float kRestore = 1.f + 2.3841858e-7f;
// k-tiles per accumulator of one plane.  A sum of one sign comes out short by about 4e-7 of itself per
// k-tile of its accumulator: 5e-5 here, a fortieth of a bfloat16 rounding (2^20 terms in one
// accumulator: 6.5e-3).
constexpr int kLongChunk = 128;
#ifndef NC_TC_WAIT_LIMIT
#define NC_TC_WAIT_LIMIT (1 << 20)
#endif
constexpr int kWaitLimit = NC_TC_WAIT_LIMIT; // polls of a bounded wait (a test lets them run out sooner)

// One product of (batched) matrices, D (m, n) = A (m, k) B (n, k)^T.  An operand is stored
// either with k contiguous, or (a_mn, b_mn) with its own row index contiguous.
struct Problem {
  CUtensorMap a, b;
  int m, n, k;
  int a_mn, b_mn;
  int tiles_m, tiles_n, batch, splits;   // splits of k; tiles run over m first
  int symmetric;                         // D is symmetric: tiles below the diagonal are left out
  int chunk;                             // k-tiles per accumulator
  int bf16;
  int a_k0, b_k0, b_n0;                  // offsets into the stored operands
  int32_t* status;                       // set to 1 when a bounded wait gives up
};

struct Tile {
  int m0, n0, batch, split;
  int kt0, kt1;   // k-tiles [kt0, kt1)
};

// CG = 2: two CTAs on two SMs work on one tile of 256 rows.  Each loads its 128 rows of A and
// half of B; the products read both halves.  Shared memory bounds a product of one CTA (a
// 128 x 256 tile writes and reads 192 bytes a cycle for 128 that it can take); the pair needs
// 128.
//
// EW epilogue warps (the first of the CTA), EW / 4 side by side on the columns of each lane quarter.
template <int PL, int BN, int CG, int EW>
struct Config {
  static constexpr int kBRows = BN / CG;   // of B in one CTA
  static constexpr int kA = PL * kBM * kBK * 2, kB = PL * kBRows * kBK * 2;
  static constexpr int kCols = BN * 4 / EW;               // of an epilogue thread
  static constexpr int kPiece = kCols < 64 ? kCols : 64;  // 16-bit values of a row in a warp's patch
  static constexpr int kPatch = 32 * kPiece * 2;
  static constexpr int kThreads = 32 * (EW + 2);
  // Accumulators in turn: all that 512 columns of tensor memory hold, up to 4.  A drain takes
  // about 2000 cycles from the last product to the freed accumulator (of a pair), more than a
  // k-tile's products on a narrow tile.
  static constexpr int kAccs = BN >= 256 ? 2 : 4;
  static constexpr int kExtras = (BN + 63) / 64;          // stages of an extra tile (load_extra)
  static constexpr int kStage = kA + kB;
  static constexpr int kStages = 192 * 1024 / kStage;
  static constexpr int kSmem = kStages * kStage + EW * kPatch;   // the stages first, on 1024 bytes
};

// Symmetric D, tiles `high` times as high as wide: those with column index j >= high i hold all
// on and above the diagonal, row i of them tiles_n - high i.
__host__ __device__ inline int symmetric_tiles(const Problem& p, int high) {
  return p.tiles_m * p.tiles_n - high * (p.tiles_m * (p.tiles_m - 1) / 2);
}
template <int BN, int CG>
__host__ __device__ inline int problem_tiles(const Problem& p) {
  return (p.symmetric ? symmetric_tiles(p, kBM * CG / BN) : p.tiles_m * p.tiles_n) * p.batch * p.splits;
}

// `rank`: of the CTA in its pair.
template <int BN, int CG>
__device__ __forceinline__ Tile problem_tile(const Problem& p, int t, int rank) {
  Tile x;
  int mn;
  if (p.symmetric) {
    constexpr int high = kBM * CG / BN;
    const int per = symmetric_tiles(p, high);
    mn = t % per;
    t /= per;
    int i = 0;
    for (; mn >= p.tiles_n - high * i; ++i) mn -= p.tiles_n - high * i;
    x.m0 = i * kBM * CG + rank * kBM, x.n0 = (high * i + mn) * BN;
  } else {
    const int per = p.tiles_m * p.tiles_n;
    mn = t % per;
    t /= per;
    x.m0 = mn % p.tiles_m * kBM * CG + rank * kBM, x.n0 = mn / p.tiles_m * BN;
  }
  x.batch = t % p.batch, x.split = t / p.batch;
  const int kt = (p.k + kBK - 1) / kBK;
  x.kt0 = (int)((int64_t)kt * x.split / p.splits), x.kt1 = (int)((int64_t)kt * (x.split + 1) / p.splits);
  return x;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The same barrier in another CTA of the cluster.
__device__ __forceinline__ uint32_t remote_addr(uint32_t bar, uint32_t cta) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(bar), "r"(cta));
  return r;
}
__device__ __forceinline__ void bar_arrive_remote(uint32_t bar, uint32_t cta) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote_addr(bar, cta)) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return n;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}

// Bounded wait.  Giving up (here or in another warp of the CTA) sets the abort flag and the
// caller's status word; every role then leaves its loop.  Lanes poll on their own and may
// differ in the outcome: a whole warp takes it by warp_wait().
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* abort, int32_t* status) {
  for (int i = 0; i < kWaitLimit; ++i) {
    if (bar_try(bar, parity)) return true;
    if (*abort) return false;
  }
  *abort = 1;
  *status = 1;
  return false;
}
// By a whole warp: true on every lane, or (where any of them gave up) false on every lane.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort, int32_t* status) {
  // the usual case without a loop: three 1024 x 1024 updates take 455 us, with bar_wait() alone 496
  if (__all_sync(0xffffffffu, bar_try(bar, parity))) return true;
  return __all_sync(0xffffffffu, bar_wait(bar, parity, abort, status));
}

// A box into this CTA's shared memory; its bytes count on `bar`, for a pair the first CTA's.
template <int CG>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c3) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(0), "r"(c3)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(0), "r"(c3)
        : "memory");
}

template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}
// One arrival on `bar` (in both CTAs of the pair that starts with CTA `lead`) when the products
// issued so far are done.
template <int CG>
__device__ __forceinline__ void mma_commit(uint32_t bar, uint32_t lead) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)(3u << lead))
        : "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t slot, int columns) {
  if constexpr (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t tmem, int columns) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 lanes (the wait belongs to the same statement, so that no use
// of the registers moves above it).
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(addr)
      : "memory");
}

// Shared-memory matrix descriptors: in the low word the start address and the leading byte
// offset, in the high word the stride byte offset (16-byte units), descriptor version 1 and
// the swizzle mode (2: rows of 128 bytes).  k contiguous: 8-row groups 1024 bytes apart, 16
// values of k 32 bytes.  Own index contiguous: blocks of 64 of it `block` bytes apart, each k
// 128 bytes, 8-k groups 1024 bytes apart, 16 values of k 2048 bytes.
constexpr uint32_t kDescHigh = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, bool mn, uint32_t block) {
  return (addr & 0x3ffff) >> 4 | (mn ? block >> 4 : 1u) << 16;   // a cluster address holds the CTA above
}
__device__ __forceinline__ uint64_t desc(uint32_t low) { return (uint64_t)kDescHigh << 32 | low; }

// One lane of a whole warp (always the same one).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p;
}

// 16-bit planes of a float32 value that was scaled to float16's range.
__device__ __forceinline__ void split_f16(float x, uint16_t* hi, uint16_t* lo) {
  const __half h = __float2half_rn(x);
  const __half l = __float2half_rn(x - __half2float(h));
  *hi = __half_as_ushort(h), *lo = __half_as_ushort(l);
}

// Two of them, packed.
__device__ __forceinline__ void split_f16x2(float x, float y, uint32_t* hi, uint32_t* lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 b = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - b.x, y - b.y);
  *hi = *reinterpret_cast<const uint32_t*>(&h), *lo = *reinterpret_cast<const uint32_t*>(&l);
}

// An epilogue thread holds a row, so that its own global accesses would touch 32 rows at a
// time (a 128-byte line each: they took most of an epilogue).  The warp's patch of shared
// memory, 32 rows of W 16-bit values, turns them: the 16-byte pieces of a row are placed so
// that neither the rows of a piece nor the pieces of a row meet in a bank.
template <int W>
__device__ __forceinline__ uint4* patch_at(uint8_t* patch, int r, int q) {
  const int turn = W == 64 ? r & 7 : r >> 1 & 3;
  return reinterpret_cast<uint4*>(patch + r * 2 * W + ((q ^ turn) << 4));
}

// Rows [0, rows) of W 16-bit values, one per lane in `v` (W / 2 words), to p + row * pitch; the
// first 8 * pieces values of each.  p and pitch on 16 bytes.
template <int W>
__device__ __forceinline__ void patch_store(uint8_t* patch, const uint32_t* v, uint16_t* p, int64_t pitch, int rows,
                                            int pieces) {
  constexpr int kPer = W / 8;   // lanes a row
  const int lane = threadIdx.x & 31, q = lane % kPer;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    *patch_at<W>(patch, lane, i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = i * (32 / kPer) + lane / kPer;
    if (r < rows && q < pieces) *reinterpret_cast<uint4*>(p + r * pitch + 8 * q) = *patch_at<W>(patch, r, q);
  }
}

// The same for rows of 32 float32 values (a patch of 128-byte rows), stored or added to what is
// there; the first 4 * pieces of each.
__device__ __forceinline__ void patch_store_f32(uint8_t* patch, const float* v, float* p, int64_t pitch, int rows,
                                                int pieces, bool add) {
  const int lane = threadIdx.x & 31, q = lane & 7;
  float4 old[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = i * 4 + (lane >> 3);
    old[i] = add && r < rows && q < pieces ? *reinterpret_cast<const float4*>(p + r * pitch + 4 * q)
                                           : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i)
    *reinterpret_cast<float4*>(patch_at<64>(patch, lane, i)) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = i * 4 + (lane >> 3);
    const float4 x = *reinterpret_cast<const float4*>(patch_at<64>(patch, r, q));
    if (r < rows && q < pieces)
      *reinterpret_cast<float4*>(p + r * pitch + 4 * q) =
          make_float4(old[i].x + x.x, old[i].y + x.y, old[i].z + x.z, old[i].w + x.w);
  }
}

// What a CTA's warps share beside the stages.
template <int PL, int BN, int CG, int EW>
struct Shared {
  uint64_t bars[2 * Config<PL, BN, CG, EW>::kStages + 2 * Config<PL, BN, CG, EW>::kAccs + 1 + 2 * Config<PL, BN, CG, EW>::kExtras];
  uint32_t tmem_slot;
  int abort, extra_readers[Config<PL, BN, CG, EW>::kExtras];
};

// One warp's view of the pipeline: the loading warp fills stages, the multiplying warp (of a
// pair's first CTA) turns them into accumulators, the epilogue warps collect those.  Each
// role keeps its own place; the places advance over tiles and over products alike.
template <int PL, int BN, int CG, int EW>
struct Engine {
  using C = Config<PL, BN, CG, EW>;
  static constexpr int BK = kBK, COLS = C::kCols, kEpiWarps = EW;
  static constexpr uint32_t a_block = C::kA / (kBM / 64), b_block = C::kB / (C::kBRows / 64);
  static_assert(C::kBRows >= 64, "operands by columns come in blocks of 64");

  uint32_t stages, bar0, tmem;
  uint8_t *base, *patch;   // of the stages, and of this epilogue warp
  int* extra_readers;
  volatile int* abort;
  int32_t* status;
  int rank;        // in the pair
  uint32_t lead;   // the pair's first CTA in the cluster
  // stage and its phase (loader and multiplier), accumulator and its phase (multiplier; the
  // epilogue's is ph); the epilogue's own stage and the phase of extra tiles
  int s = 0, buf = 0, issued = 0, extras = 0, es = 0;
  uint32_t ph, aph = 1, eph = 0;
  bool ok = true;

  __device__ __forceinline__ uint32_t full(int i) const { return bar0 + 8 * i; }
  __device__ __forceinline__ uint32_t empty(int i) const { return bar0 + 8 * (C::kStages + i); }
  __device__ __forceinline__ uint32_t acc_full(int i) const { return bar0 + 8 * (2 * C::kStages + i); }
  __device__ __forceinline__ uint32_t acc_empty(int i) const { return bar0 + 8 * (2 * C::kStages + C::kAccs + i); }
  __device__ __forceinline__ uint32_t drain() const { return bar0 + 8 * (2 * C::kStages + 2 * C::kAccs); }
  __device__ __forceinline__ uint32_t extra_full(int i) const { return bar0 + 8 * (2 * C::kStages + 2 * C::kAccs + 1 + i); }
  __device__ __forceinline__ uint32_t extra_read(int i) const { return extra_full(C::kExtras + i); }

  // By the whole CTA, before it reads anything that an earlier kernel wrote.  `raw`: the dynamic
  // shared memory, on 1024 bytes.
  __device__ __forceinline__ Engine(uint8_t* raw, Shared<PL, BN, CG, EW>* sh, int32_t* status_word) {
    stages = smem_addr(raw);
    base = raw;
    patch = base + C::kStages * C::kStage + (threadIdx.x >> 5) * C::kPatch;
    extra_readers = sh->extra_readers;
    bar0 = smem_addr(sh->bars);
    abort = &sh->abort;
    status = status_word;
    const uint32_t cta = CG == 1 ? 0 : cluster_rank();
    rank = cta & 1, lead = cta & ~1u;
    const int warp = threadIdx.x >> 5;
    ph = warp == kEpiWarps;   // the loader starts on empty stages
    if (threadIdx.x == 0) {
      for (int i = 0; i < C::kStages; ++i) bar_init(full(i), 1), bar_init(empty(i), 1);
      for (int i = 0; i < C::kAccs; ++i) bar_init(acc_full(i), 1), bar_init(acc_empty(i), kEpiWarps * CG);
      bar_init(drain(), 1);
      for (int i = 0; i < C::kExtras; ++i) bar_init(extra_full(i), 1), bar_init(extra_read(i), 1), sh->extra_readers[i] = 0;
      sh->abort = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kEpiWarps + 1) tmem_alloc<CG>(smem_addr(&sh->tmem_slot), C::kAccs * BN);
    fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    fence_after();
    tmem = sh->tmem_slot;
  }

  // One thread of the loading warp: the k-tiles of a tile.
  __device__ __forceinline__ void load(const Problem& p, const CUtensorMap* a, const CUtensorMap* b, const Tile& x) {
    for (int kt = x.kt0; kt < x.kt1 && ok; ++kt) {
      if (!(ok = bar_wait(empty(s), ph, abort, status))) return;
      if (rank == 0) bar_expect(full(s), C::kStage * CG);
      const uint32_t bar = CG == 1 ? full(s) : remote_addr(full(s), lead);
      const uint32_t at = stages + s * C::kStage;
      const int ka = p.a_k0 + kt * BK, kb = p.b_k0 + kt * BK, nb = p.b_n0 + x.n0 + rank * C::kBRows;
      if (p.a_mn) {
#pragma unroll
        for (int i = 0; i < kBM / 64; ++i) tma_load<CG>(at + i * a_block, a, bar, x.m0 + 64 * i, ka, x.batch);
      } else {
        tma_load<CG>(at, a, bar, ka, x.m0, x.batch);
      }
      if (p.b_mn) {
#pragma unroll
        for (int i = 0; i < C::kBRows / 64; ++i)
          tma_load<CG>(at + C::kA + i * b_block, b, bar, nb + 64 * i, kb, x.batch);
      } else {
        tma_load<CG>(at + C::kA, b, bar, kb, nb, x.batch);
      }
      if (issued < C::kStages) ++issued;
      if (++s == C::kStages) s = 0, ph ^= 1;
    }
  }

  // Behind a tile's k-tiles, what the epilogue wants of a stored matrix: this CTA's rows of the
  // tile, both planes, a stage for every 64 columns.  It lands in this CTA (of a pair too) on
  // barriers of its own; the multiplying warp steps over it with skip_extra(), the epilogue
  // takes it with extra() and extra_done().  The next tile's waits until all warps have read this
  // one: with fewer k-tiles than stages it could land first, and a slow warp would miss a phase.
  __device__ __forceinline__ void load_extra(const CUtensorMap* m, const Tile& x) {
    constexpr int bytes = PL * kBM * 128;
    static_assert(bytes <= C::kStage, "64 columns fit a stage");
#pragma unroll
    for (int i = 0; i < C::kExtras; ++i) {
      if (!ok || !(ok = bar_wait(extra_read(i), (extras / C::kExtras & 1) ^ 1, abort, status))) return;
      if (!(ok = bar_wait(empty(s), ph, abort, status))) return;
      bar_expect(extra_full(i), bytes);
      tma_load<1>(stages + s * C::kStage, m, extra_full(i), x.n0 + 64 * i, x.m0, x.batch);
      ++extras;
      if (rank == 0) bar_arrive(full(s));   // keeps the stage's phases in step
      if (issued < C::kStages) ++issued;
      if (++s == C::kStages) s = 0, ph ^= 1;
    }
  }
  __device__ __forceinline__ void skip_extra() {
#pragma unroll
    for (int i = 0; i < C::kExtras; ++i)
      if (++s == C::kStages) s = 0, ph ^= 1;
  }

  // The multiplying warp, whole: what it computes is the same on all lanes and stays in
  // uniform registers, and one lane issues (issuing from a lane's own branch cost about 150
  // cycles a product, more than a 128-wide one takes).
  __device__ __forceinline__ void multiply(const Problem& p, const Tile& x) {
    // accumulator float32; operand types; which operands have their own index contiguous
    const uint32_t idesc = 1u << 4 | (p.bf16 ? 1u << 7 | 1u << 10 : 0u) | (p.a_mn ? 1u << 15 : 0u) |
                           (p.b_mn ? 1u << 16 : 0u) | (uint32_t)(BN >> 3) << 17 | (uint32_t)(kBM * CG >> 4) << 24;
    const uint32_t a_plane = (p.a_mn ? a_block / PL : C::kA / PL) >> 4, b_plane = (p.b_mn ? b_block / PL : C::kB / PL) >> 4;
    const uint32_t a_step = p.a_mn ? 2048 >> 4 : 32 >> 4, b_step = p.b_mn ? 2048 >> 4 : 32 >> 4;
    const uint32_t a0 = desc_low(stages, p.a_mn, a_block), b0 = desc_low(stages + C::kA, p.b_mn, b_block);
    for (int c0 = x.kt0; c0 < x.kt1; c0 += p.chunk) {
      if (!(ok = warp_wait(acc_empty(buf), aph, abort, status))) return;
      fence_after();
      const uint32_t d = tmem + buf * BN;
      const int c1 = min(c0 + p.chunk, x.kt1);
      for (int kt = c0; kt < c1; ++kt) {
        if (!(ok = warp_wait(full(s), ph, abort, status))) return;
        fence_after();
        const uint32_t a = a0 + s * (C::kStage >> 4), b = b0 + s * (C::kStage >> 4);
        if (elect_one()) {
          // low parts first, while the accumulator is small
          constexpr int kProducts = PL == 1 ? 1 : 3;
#pragma unroll
          for (int q = 0; q < kProducts; ++q) {
            const int pa = PL == 1 ? 0 : (q == 0 ? 1 : 0), pb = PL == 1 ? 0 : (q == 1 ? 1 : 0);
#pragma unroll
            for (int ks = 0; ks < BK / 16; ++ks)
              mma<CG>(d, desc(a + pa * a_plane + ks * a_step), desc(b + pb * b_plane + ks * b_step), idesc,
                      kt > c0 || q > 0 || ks > 0);
          }
          mma_commit<CG>(empty(s), lead);
          if (kt + 1 == c1) mma_commit<CG>(acc_full(buf), lead);
        }
        __syncwarp();
        if (++s == C::kStages) s = 0, ph ^= 1;
      }
      if (++buf == C::kAccs) buf = 0, aph ^= 1;
    }
  }

  // An epilogue warp: the sums of its 32 rows and COLS columns.  DRAIN: of several chunks; one alone
  // (one plane) needs no second set of registers.
  template <bool DRAIN = PL == 2>
  __device__ __forceinline__ void collect(const Problem& p, const Tile& x, float (&acc)[COLS]) {
    const int warp = threadIdx.x >> 5;
    const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (warp >> 2) * COLS;
#pragma unroll
    for (int i = 0; i < COLS; ++i) acc[i] = 0.f;
    for (int c0 = x.kt0; c0 < x.kt1; c0 += p.chunk) {
      if (!__all_sync(0xffffffffu, ok && bar_wait(acc_full(buf), ph, abort, status))) {
        ok = false;
        return;
      }
      fence_after();
#pragma unroll
      for (int i = 0; i < COLS; i += 32) {
        float v[32];
        tmem_load(lanes + buf * BN + i, v);
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[i + j] = DRAIN ? fmaf(v[j], PL == 1 ? 1.f : kRestore, acc[i + j]) : v[j];
      }
      fence_before();
      if ((threadIdx.x & 31) == 0) {
        if constexpr (CG == 1)
          bar_arrive(acc_empty(buf));
        else
          bar_arrive_remote(acc_empty(buf), lead);
      }
      __syncwarp();
      if (++buf == C::kAccs) buf = 0, ph ^= 1;
    }
    es = (es + x.kt1 - x.kt0) % C::kStages;
  }

  // An epilogue warp, after collect(): the stage of its columns' 64 (null after an abort): plane,
  // row, 128 bytes in 16-byte pieces q ^ (row & 7).  Every epilogue warp calls extra_done() when it
  // has read its part; the last of a stage's readers frees it.
  __device__ __forceinline__ const uint8_t* extra() {
    const int i = (threadIdx.x >> 7) * COLS / 64;
    if (!__all_sync(0xffffffffu, ok && bar_wait(extra_full(i), eph, abort, status))) {
      ok = false;
      return nullptr;
    }
    const int at = es + i;
    return base + (at >= C::kStages ? at - C::kStages : at) * C::kStage;
  }
  __device__ __forceinline__ void extra_done() {
    const int i = (threadIdx.x >> 7) * COLS / 64, at = es + i;
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
      __threadfence_block();
      constexpr int readers = EW / C::kExtras;
      if (atomicAdd(extra_readers + i, 1) % readers == readers - 1) {
        bar_arrive(empty(at >= C::kStages ? at - C::kStages : at));
        bar_arrive(extra_read(i));
      }
    }
    eph ^= 1;
    es += C::kExtras;
    if (es >= C::kStages) es -= C::kStages;
  }

  // At the end, by the whole CTA.
  __device__ __forceinline__ void finish() {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == kEpiWarps && lane == 0 && (!ok || *abort)) {
      // the copies in flight land before the CTA (or the pair) ends
      for (int i = 0; i < issued && rank == 0; ++i) {
        if (s-- == 0) s = C::kStages - 1, ph ^= 1;
        for (int j = 0; j < kWaitLimit && !bar_try(full(s), ph ^ 1); ++j) {
        }
      }
      for (int i = 0; i < C::kExtras; ++i) {
        const int n = (extras + C::kExtras - 1 - i) / C::kExtras;   // copies on this barrier
        for (int j = 0; j < kWaitLimit && n > 0 && !bar_try(extra_full(i), (n - 1) & 1); ++j) {
        }
      }
    }
    if (warp == kEpiWarps + 1 && rank == 0) {
      // every product has finished before tensor memory is given back
      if (elect_one()) mma_commit<CG>(drain(), lead);
      for (int j = 0; j < kWaitLimit && !bar_try(drain(), 0); ++j) {
      }
    }
    __syncthreads();
    // a pair ends together: each reads the other's shared memory and signals its barriers
    if constexpr (CG == 2) cluster_sync();
    if (warp == kEpiWarps + 1) {
      fence_after();
      tmem_free<CG>(tmem, C::kAccs * BN);
    }
  }
};

// The kernel of one product: the first EW warps epilogue, the next loads, the last multiplies;
// persistent over tiles.  Epi::run(state, tile, row, col, acc) gets COLS consecutive columns of a row as
// float32 sums; Epi::begin(tile, row, col, patch) runs before the wait for them and returns the
// state.
template <int PL, int BN, int CG, int EW, class Epi, bool DRAIN>
__global__ void __launch_bounds__(32 * (EW + 2), 1) product_kernel(const __grid_constant__ Problem p, const Epi epi) {
  using E = Engine<PL, BN, CG, EW>;
  extern __shared__ __align__(1024) uint8_t raw[];
  __shared__ Shared<PL, BN, CG, EW> sh;
  E e(raw, &sh, p.status);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = blockIdx.x / CG, stride = gridDim.x / CG, tiles = problem_tiles<BN, CG>(p);
  pdl_enter();
  if (warp == EW) {
    if (lane == 0)
      for (int t = first; t < tiles && e.ok; t += stride) e.load(p, &p.a, &p.b, problem_tile<BN, CG>(p, t, e.rank));
  } else if (warp == EW + 1) {
    if (e.rank == 0)
      for (int t = first; t < tiles && e.ok; t += stride) e.multiply(p, problem_tile<BN, CG>(p, t, 0));
  } else {
    for (int t = first; t < tiles && e.ok; t += stride) {
      const Tile x = problem_tile<BN, CG>(p, t, e.rank);
      const int row = x.m0 + 32 * (warp & 3) + lane, col = x.n0 + (warp >> 2) * E::COLS;
      __syncwarp();   // the last tile's readers of the patch are done
      const auto state = epi.template begin<E::COLS>(x, row, col, e.patch);
      __syncwarp();
      float acc[E::COLS];
      e.template collect<DRAIN>(p, x, acc);
      if (e.ok) epi.template run<E::COLS>(state, x, row, col, acc);
    }
  }
  __syncwarp();
  e.finish();
}

// Tensor map of a stored matrix (inner contiguous, `outer` rows `pitch` elements apart, planes
// `plane` elements apart, batches `per_batch` apart); box of (box_inner, box_outer) per plane.
nc_status make_map(CUtensorMap* map, const void* base, bool bf16, int planes, int inner, int outer, int64_t pitch,
                   int64_t plane, int batch, int64_t per_batch, int box_inner, int box_outer);

int sm_count();

// The two operands' maps: `mn` says that the operand's own index (extent `own`) is contiguous.
template <int PL, int BN, int CG, int EW>
nc_status make_operand(Problem* p, bool is_a, const void* base, bool mn, int own, int k, int64_t pitch, int64_t plane,
                       int batch, int64_t per_batch) {
  using C = Config<PL, BN, CG, EW>;
  (is_a ? p->a_mn : p->b_mn) = mn;
  const int rows = is_a ? kBM : C::kBRows;
  return mn ? make_map(is_a ? &p->a : &p->b, base, p->bf16, PL, own, k, pitch, plane, batch, per_batch, 64, kBK)
            : make_map(is_a ? &p->a : &p->b, base, p->bf16, PL, k, own, pitch, plane, batch, per_batch, kBK, rows);
}

// Tiles that cover (m, n).
template <int BN, int CG>
__host__ __device__ inline void set_tiles(Problem* p) {
  p->tiles_m = (p->m + kBM * CG - 1) / (kBM * CG), p->tiles_n = (p->n + BN - 1) / BN;
}

template <int PL, int BN, int CG, int EW, class Epi>
nc_status launch_product(const Problem& p, const Epi& epi, cudaStream_t st, const char* what) {
  auto k = product_kernel<PL, BN, CG, EW, Epi, true>;
  if constexpr (PL == 1) {
    const int kt = (p.k + kBK - 1) / kBK;
    if ((kt + p.splits - 1) / p.splits <= p.chunk) k = product_kernel<PL, BN, CG, EW, Epi, false>;
  }
  constexpr int smem = Config<PL, BN, CG, EW>::kSmem;
  NC_CHECK(allow_smem((const void*)k, smem));
  const int tiles = problem_tiles<BN, CG>(p), most = sm_count() / CG;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((tiles < most ? tiles : most) * CG), cfg.blockDim = dim3(32 * (EW + 2));
  cfg.dynamicSmemBytes = smem, cfg.stream = st, cfg.attrs = attr, cfg.numAttrs = CG == 1 ? 1 : 2;
  NC_CUDA_CHECK(cudaLaunchKernelEx(&cfg, k, p, epi));
  return launch_check(what);
}

}  // namespace tc
}  // namespace nc
