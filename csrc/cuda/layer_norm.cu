// Layer norm, forward and backward.
#include "layers.cuh"

namespace hipress {
namespace {

template <typename T>
__global__ void __launch_bounds__(256) norm_forward_kernel(const __grid_constant__ HpNormForward a) {
  __shared__ float part[32];
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.ldx;
  const T* r = a.residual ? (const T*)a.residual + row * a.ldr : nullptr;
  T* y = (T*)a.y + row * a.cols;
  T* z = a.z ? (T*)a.z + row * a.cols : nullptr;
  auto value = [&](int64_t i) { return r ? to_f(from_f<T>(to_f(x[i]) + to_f(r[i]))) : to_f(x[i]); };
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < a.cols; i += blockDim.x) s += value(i);
  const float mean = cta_sum(s, part) / (float)a.cols;
  s = 0.f;
  for (int64_t i = threadIdx.x; i < a.cols; i += blockDim.x) {
    const float d = value(i) - mean;
    s = fmaf(d, d, s);
  }
  const float rstd = 1.f / sqrtf(cta_sum(s, part) / (float)a.cols + (float)a.eps);
  for (int64_t i = threadIdx.x; i < a.cols; i += blockDim.x) {
    const float v = value(i);
    float o = (v - mean) * rstd;
    if (a.weight) o *= load_any(a.weight, i, (int)a.wtype);
    if (a.bias) o += load_any(a.bias, i, (int)a.wtype);
    y[i] = from_f<T>(o);
    if (z) z[i] = from_f<T>(v);
  }
  if (threadIdx.x == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) norm_dx_kernel(const __grid_constant__ HpNormBackward a) {
  __shared__ float part[32];
  const int64_t row = blockIdx.x;
  const T* z = (const T*)a.z + row * a.ldz;
  const T* dy = (const T*)a.dy + row * a.lddy;
  const T* dz = a.dz ? (const T*)a.dz + row * a.lddz : nullptr;
  T* dx = (T*)a.dx + row * a.cols;
  const float mean = a.mean[row], rstd = a.rstd[row];
  auto grad = [&](int64_t i) { return a.weight ? to_f(dy[i]) * load_any(a.weight, i, (int)a.wtype) : to_f(dy[i]); };
  float s1 = 0.f, s2 = 0.f;
  for (int64_t i = threadIdx.x; i < a.cols; i += blockDim.x) {
    const float g = grad(i);
    s1 += g;
    s2 = fmaf(g, (to_f(z[i]) - mean) * rstd, s2);
  }
  s1 = cta_sum(s1, part) / (float)a.cols;
  s2 = cta_sum(s2, part) / (float)a.cols;
  for (int64_t i = threadIdx.x; i < a.cols; i += blockDim.x) {
    const float h = (to_f(z[i]) - mean) * rstd;
    float d = rstd * (grad(i) - s1 - h * s2);
    if (dz) d += to_f(dz[i]);
    dx[i] = from_f<T>(d);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) norm_dw_kernel(const __grid_constant__ HpNormBackward a) {
  __shared__ float sw[8][33], sb[8][33];
  const int64_t col = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float w = 0.f, b = 0.f;
  if (col < a.cols)
    for (int64_t r = threadIdx.y; r < a.rows; r += 8) {
      const float d = to_f(((const T*)a.dy)[r * a.lddy + col]);
      w = fmaf(d, (to_f(((const T*)a.z)[r * a.ldz + col]) - a.mean[r]) * a.rstd[r], w);
      b += d;
    }
  sw[threadIdx.y][threadIdx.x] = w;
  sb[threadIdx.y][threadIdx.x] = b;
  __syncthreads();
  if (threadIdx.y == 0 && col < a.cols) {
    for (int i = 1; i < 8; ++i) w += sw[i][threadIdx.x], b += sb[i][threadIdx.x];
    if (a.dweight) store_any(a.dweight, col, w, (int)a.wtype);
    if (a.dbias) store_any(a.dbias, col, b, (int)a.wtype);
  }
}

template <typename T>
int forward(const HpNormForward& a, cudaStream_t s) {
  norm_forward_kernel<T><<<(unsigned)a.rows, 256, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T>
int backward(const HpNormBackward& a, cudaStream_t s) {
  if (a.dx && a.rows) norm_dx_kernel<T><<<(unsigned)a.rows, 256, 0, s>>>(a);
  if (a.dweight || a.dbias) norm_dw_kernel<T><<<(unsigned)((a.cols + 31) / 32), dim3(32, 8), 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace hipress

using namespace hipress;

extern "C" int hp_cuda_norm_forward(const HpNormForward* a, void* stream) {
  if (!a || a->rows < 0 || a->cols < 1 || a->rows > INT32_MAX || !type_ok(a->type) || !type_ok(a->wtype) ||
      (a->residual && !a->z))
    return HP_ERR_BAD_ARG;
  if (!a->rows) return 0;
  cudaStream_t s = (cudaStream_t)stream;
  return a->type == HP_F32 ? forward<float>(*a, s)
                           : a->type == HP_BF16 ? forward<__nv_bfloat16>(*a, s) : forward<__half>(*a, s);
}

extern "C" int hp_cuda_norm_backward(const HpNormBackward* a, void* stream) {
  if (!a || a->rows < 0 || a->cols < 1 || a->rows > INT32_MAX || !type_ok(a->type) || !type_ok(a->wtype))
    return HP_ERR_BAD_ARG;
  cudaStream_t s = (cudaStream_t)stream;
  return a->type == HP_F32 ? backward<float>(*a, s)
                           : a->type == HP_BF16 ? backward<__nv_bfloat16>(*a, s) : backward<__half>(*a, s);
}

extern "C" uint64_t hp_cuda_norm_workspace(int64_t, int64_t, int64_t) { return 0; }
