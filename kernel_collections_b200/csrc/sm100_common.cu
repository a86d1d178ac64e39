// Host-side pieces shared by the sm_100a kernels: the tensor-map encoder and the status clear.
#include "sm100_common.cuh"

namespace xkv {
namespace sm100 {

__global__ void clear_status_kernel(int* status) {
  if (threadIdx.x < 64) status[threadIdx.x] = 0;
}

EncodeTiledFn get_encode() {
  // looked up once; a second thread waits for the first one's answer
  static const EncodeTiledFn fn = []() -> EncodeTiledFn {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeTiledFn>(p);
    cudaGetLastError();
    return nullptr;
  }();
  return fn;
}

bool encode_tiled_16bit(CUtensorMap* m, int dtype, int rank, const void* ptr, const cuuint64_t* dims,
                        const cuuint64_t* strides, const cuuint32_t* box) {
  EncodeTiledFn fn = get_encode();
  if (!fn) return false;
  cuuint32_t es[5] = {1, 1, 1, 1, 1};
  const CUtensorMapDataType dt = dtype == XKV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  for (int again = 0; again < 2; ++again) {
    const CUresult r = fn(m, dt, (cuuint32_t)rank, const_cast<void*>(ptr), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS) return true;
    // a host thread that has made no CUDA call of its own has no context yet: setting its device gives it one
    int dev = 0;
    if ((r != CUDA_ERROR_INVALID_CONTEXT && r != CUDA_ERROR_NOT_INITIALIZED) || cudaGetDevice(&dev) != cudaSuccess ||
        cudaSetDevice(dev) != cudaSuccess) {
      cudaGetLastError();
      return false;
    }
  }
  return false;
}

}  // namespace sm100
}  // namespace xkv
