// nc_tc.cu -- host side of the tensor-core products: tensor maps.
#include "nc_tc.cuh"

namespace nc {
namespace tc {

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

nc_status make_map(CUtensorMap* map, const void* base, bool bf16, int planes, int inner, int outer, int64_t pitch,
                   int64_t plane, int batch, int64_t per_batch, int box_inner, int box_outer) {
  EncodeFn fn = encode_fn();
  if (!fn) return set_error(NC_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t dims[4] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)planes, (cuuint64_t)batch};
  const cuuint64_t strides[3] = {(cuuint64_t)pitch * 2, (cuuint64_t)plane * 2, (cuuint64_t)per_batch * 2};
  const cuuint32_t box[4] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer, (cuuint32_t)planes, 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  const CUresult r =
      fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base),
         dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(NC_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for %d x %d, pitch %lld", (int)r, outer, inner,
                     (long long)pitch);
  return NC_OK;
}

int sm_count() {
  static thread_local int dev_seen = -1, sms = 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev != dev_seen) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 1) return 148;
    dev_seen = dev;
  }
  return sms;
}

}  // namespace tc
}  // namespace nc
