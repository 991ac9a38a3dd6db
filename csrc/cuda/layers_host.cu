// Host side shared by the layer operators: tensor maps, the status word, device facts.
#include <mutex>

#include "tcgen05.cuh"

namespace hipress {
namespace {

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                            const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

Encode encoder() {   // looked up in the driver, so that nothing links against it
  static const Encode f = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (told(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q)) ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (Encode)p;
  }();
  return f;
}

constexpr int kDevices = 64;

// Two warps at a barrier that nobody arrives at: the first gives up after `limit`, the second, which
// would wait for kWaitNs, because the first has.
__global__ void wait_probe(uint64_t limit, uint64_t* took, uint32_t* status) {
  __shared__ uint64_t bar;
  __shared__ Guard guard;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    mbar_init_fence();
    guard.gave_up = 0;
    guard.status = status;
  }
  __syncthreads();
  const uint64_t start = global_timer_ns();
  const bool came = threadIdx.x < 32 ? guard_wait(&bar, 0, guard, 0x90000, limit) : guard_wait(&bar, 0, guard, 0x90001);
  if (threadIdx.x % 32 == 0) took[threadIdx.x / 32] = came ? 0 : global_timer_ns() - start;
}

}  // namespace

bool tensor_map(CUtensorMap* m, const void* base, int type, int rank, const uint64_t* sizes, const uint64_t* strides_bytes,
                const uint32_t* box) {
  const Encode f = encoder();
  if (!f) return false;
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  cuuint64_t size[5], stride[5];
  for (int i = 0; i < rank; ++i) {
    size[i] = sizes[i] ? sizes[i] : 1;
    if (i) stride[i - 1] = strides_bytes[i - 1];
  }
  const CUtensorMapDataType t = type == HP_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                : type == HP_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  auto encode = [&] {
    return f(m, t, (cuuint32_t)rank, (void*)base, size, stride, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  if (encode() == CUDA_SUCCESS) return true;
  // a thread that has not used the device yet (autograd's, in its first backward pass) has no context
  int dev = 0;
  if (told(cudaGetDevice(&dev)) || told(cudaSetDevice(dev))) return false;
  return encode() == CUDA_SUCCESS;
}

uint32_t* layer_status(int* rc) {
  static uint32_t* words[kDevices] = {};
  static std::mutex lock;
  int dev = 0;
  *rc = told(cudaGetDevice(&dev));
  if (*rc) return nullptr;
  if (dev >= kDevices) {
    *rc = HP_ERR_BAD_ARG;
    return nullptr;
  }
  std::lock_guard<std::mutex> hold(lock);
  if (!words[dev]) {   // pinned for good, 64 bytes
    void* p = nullptr;
    *rc = told(cudaHostAlloc(&p, 64, cudaHostAllocMapped | cudaHostAllocPortable));
    if (*rc) return nullptr;
    *(volatile uint32_t*)p = 0;
    words[dev] = (uint32_t*)p;
  }
  volatile uint32_t* w = words[dev];
  if (*w) {
    *w = 0;
    *rc = HP_ERR_TIMEOUT;
    return nullptr;
  }
  return words[dev];
}

int layer_sms() {
  static int sms[kDevices] = {};
  int dev = 0, n = 0;
  if (told(cudaGetDevice(&dev)) || dev >= kDevices) return 1;
  if (!sms[dev]) {
    if (told(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev))) return 1;
    sms[dev] = n;
  }
  return sms[dev];
}

}  // namespace hipress

extern "C" int hp_cuda_layer_wait_probe(uint64_t limit_ns, uint64_t* took, void* stream) {
  using namespace hipress;
  if (!took || limit_ns > kWaitNs) return HP_ERR_BAD_ARG;
  int rc;
  uint32_t* status = layer_status(&rc);
  if (rc) return rc;
  wait_probe<<<1, 64, 0, (cudaStream_t)stream>>>(limit_ns, took, status);
  return cudaGetLastError();
}
