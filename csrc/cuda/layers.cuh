// What the layer operators' kernels share: element types, reductions inside a warp or CTA.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "hipress/capi.h"
#include "hipress/layers.h"
#include "hipress/per_device.h"

namespace hipress {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// two values in one register
template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
  return *(const uint32_t*)&v;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
  const __half2 v = __floats2half2_rn(x, y);
  return *(const uint32_t*)&v;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {   // the upper half of a float
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*(const __half2*)&v);
}

// A choice that is made when a generic function is compiled
struct Yes {
  __device__ constexpr operator bool() const { return true; }
};
struct No {
  __device__ constexpr operator bool() const { return false; }
};

// Two values at a time: half the instructions.
struct F2 {
  float x, y;
};
__device__ __forceinline__ uint64_t bits(F2 v) {
  return (uint64_t)__float_as_uint(v.y) << 32 | __float_as_uint(v.x);
}
__device__ __forceinline__ F2 f2(uint64_t v) { return {__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))}; }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
  return f2(d);
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)));
  return f2(d);
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)));
  return f2(d);
}

// 16 bytes of elements, in 32 bits
template <typename T>
constexpr int kPiece = 16 / sizeof(T);
template <typename T>
__device__ __forceinline__ void unpack(uint4 raw, float (&v)[kPiece<T>]) {
  const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<T>(r[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void unpack<float>(uint4 raw, float (&v)[4]) {
  v[0] = __uint_as_float(raw.x), v[1] = __uint_as_float(raw.y), v[2] = __uint_as_float(raw.z), v[3] = __uint_as_float(raw.w);
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&v)[kPiece<T>]) {
  return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}
template <>
__device__ __forceinline__ uint4 pack<float>(const float (&v)[4]) {
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}

// element i of an array whose type is known at run time (uniform over the launch)
__device__ __forceinline__ float load_any(const void* p, int64_t i, int type) {
  return type == HP_F32 ? ((const float*)p)[i]
                        : type == HP_BF16 ? to_f(((const __nv_bfloat16*)p)[i]) : to_f(((const __half*)p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int64_t i, float v, int type) {
  if (type == HP_F32) ((float*)p)[i] = v;
  else if (type == HP_BF16) ((__nv_bfloat16*)p)[i] = from_f<__nv_bfloat16>(v);
  else ((__half*)p)[i] = from_f<__half>(v);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// sum over the CTA, the same value in every thread; `part` holds 32 floats
__device__ __forceinline__ float cta_sum(float v, float* part) {
  v = warp_sum(v);
  __syncthreads();   // part may still be read from the sum before
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < (int)(blockDim.x + 31) / 32; ++i) s += part[i];
  return s;
}

// A kernel that may be started while the one in front of it in the stream still runs: its CTAs set
// up barriers, tensor memory and tensor maps meanwhile, and wait for the end of the one in front
// (and of what that has waited for) before they touch memory.  Kernels launched by launch_behind()
// call both; the plain norm kernels are launched the ordinary way and neither start early nor let others.
__device__ __forceinline__ void dependents_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_kernel_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The code that is returned for a call of the runtime.  The runtime keeps it as well, for whoever asks next
// about a launch of their own: that is taken back.
inline int told(cudaError_t rc) {
  if (rc != cudaSuccess) cudaGetLastError();
  return rc;
}

template <typename... Params, typename... Args>
int launch(bool early, void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = early ? 1 : 0;
  return told(cudaLaunchKernelEx(&cfg, kernel, Params(args)...));
}
template <typename... Params, typename... Args>
int launch_behind(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, const Args&... args) {
  return launch(true, kernel, grid, block, smem, s, args...);
}

// Lets the kernel have `smem` bytes of dynamic shared memory on the current device.  `done` is the
// kernel's own.
template <typename K>
int allow_shared_memory(PerDevice& done, K kernel, int smem) {
  int dev = 0, value;
  if (const int rc = told(cudaGetDevice(&dev))) return rc;
  return done.get(dev, [&](int* v) {
    *v = 1;
    return told(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  }, &value);
}

inline bool type_ok(int64_t t) { return t >= HP_F32 && t <= HP_F16; }

}  // namespace hipress
