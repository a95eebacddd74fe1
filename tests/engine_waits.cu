// The tensor-core engine with a loading warp that loads nothing: the waits of the multiplying
// and of the epilogue warps run out.  Built by test_gpu_engine_waits.py with a small
// NC_TC_WAIT_LIMIT.
#include <cuda_runtime.h>

#include "nc_tc.cuh"

namespace {

using namespace nc;

template <int PL, int BN, int CG, int EW>
__global__ void __launch_bounds__(32 * (EW + 2), 1) starved_kernel(const __grid_constant__ tc::Problem p, int* left) {
  using E = tc::Engine<PL, BN, CG, EW>;
  extern __shared__ __align__(1024) uint8_t raw[];
  __shared__ tc::Shared<PL, BN, CG, EW> sh;
  E e(raw, &sh, p.status);
  const int warp = threadIdx.x >> 5;
  if (warp == EW + 1) {
    if (e.rank == 0) e.multiply(p, tc::problem_tile<BN, CG>(p, 0, 0));
  } else if (warp < EW) {
    float acc[E::COLS];
    e.collect(p, tc::problem_tile<BN, CG>(p, 0, e.rank), acc);
  }
  __syncwarp();
  if (!e.ok) atomicAdd(left, 1);
  e.finish();
}

template <int PL, int BN, int CG, int EW>
int starve(int* out) {
  int* dev = nullptr;
  cudaError_t err = cudaMalloc(&dev, 8);
  if (err != cudaSuccess) return err;
  err = cudaMemset(dev, 0, 8);
  tc::Problem p{};
  p.m = 128 * CG, p.n = BN, p.k = 256, p.tiles_m = p.tiles_n = p.batch = p.splits = 1, p.chunk = 2;
  p.status = dev;
  auto k = starved_kernel<PL, BN, CG, EW>;
  constexpr int smem = tc::Config<PL, BN, CG, EW>::kSmem;
  if (err == cudaSuccess) err = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(CG), cfg.blockDim = dim3(32 * (EW + 2));
  cfg.dynamicSmemBytes = smem, cfg.attrs = attr, cfg.numAttrs = 1;
  if (err == cudaSuccess) err = cudaLaunchKernelEx(&cfg, k, p, dev + 1);
  if (err == cudaSuccess) err = cudaMemcpy(out, dev, 8, cudaMemcpyDeviceToHost);
  const cudaError_t freed = cudaFree(dev);
  return err == cudaSuccess ? freed : err;
}

}  // namespace

// out[0]: the status word, out[1]: threads whose role gave up.
extern "C" int starved_engine(int pair, int* out) {
  return pair ? starve<1, 256, 2, 8>(out) : starve<2, 128, 1, 16>(out);
}
