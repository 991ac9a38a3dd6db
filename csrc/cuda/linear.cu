// The matrix product with bias, activation and residual in its epilogue, and what its
// backward pass needs besides two more products.
#include "activation.cuh"

namespace hipress {
namespace {

constexpr int kTile = 64, kDepth = 16;

template <typename T, int ACT>
__global__ void __launch_bounds__(256) product_kernel(const __grid_constant__ HpProduct a) {
  __shared__ float sa[kDepth][kTile + 1], sb[kDepth][kTile + 1];
  const int64_t m0 = (int64_t)blockIdx.y * kTile, n0 = (int64_t)blockIdx.x * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < a.k; k0 += kDepth) {
    for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
      const int ka = a.a_kmajor ? i % kDepth : i / kTile, ra = a.a_kmajor ? i / kDepth : i % kTile;
      const int64_t m = m0 + ra, k = k0 + ka;
      sa[ka][ra] = m < a.m && k < a.k ? to_f(((const T*)a.a)[a.a_kmajor ? m * a.lda + k : k * a.lda + m]) : 0.f;
      const int kb = a.b_kmajor ? i % kDepth : i / kTile, rb = a.b_kmajor ? i / kDepth : i % kTile;
      const int64_t n = n0 + rb, l = k0 + kb;
      sb[kb][rb] = n < a.n && l < a.k ? to_f(((const T*)a.b)[a.b_kmajor ? n * a.ldb + l : l * a.ldb + n]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty + 16 * i], sb[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m >= a.m || n >= a.n) continue;
      float p = acc[i][j];
      if (a.bias) p += load_any(a.bias, n, (int)a.btype);
      if (a.pre) ((T*)a.pre)[m * a.ldy + n] = from_f<T>(p);
      p = activate<ACT>(p);
      if (a.residual) p += to_f(((const T*)a.residual)[m * a.ldr + n]);
      store_any(a.y, m * a.ldy + n, p, (int)a.ytype);
    }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256) slope_kernel(const __grid_constant__ HpSlope a) {
  __shared__ float sums[8][33];
  const int64_t col = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (col < a.cols)
    for (int64_t r = threadIdx.y; r < a.rows; r += 8) {
      float g = to_f(((const T*)a.dy)[r * a.lddy + col]);
      if (ACT != HP_ACT_NONE) g *= slope<ACT>(to_f(((const T*)a.pre)[r * a.ldpre + col]));
      if (a.g) ((T*)a.g)[r * a.ldg + col] = from_f<T>(g);
      s += g;
    }
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && col < a.cols && a.dbias) {
    for (int i = 1; i < 8; ++i) s += sums[i][threadIdx.x];
    store_any(a.dbias, col, s, (int)a.btype);
  }
}

template <typename T>
int product(const HpProduct& a, cudaStream_t s) {
  const dim3 grid((unsigned)((a.n + kTile - 1) / kTile), (unsigned)((a.m + kTile - 1) / kTile));
  switch (a.act) {
    case HP_ACT_NONE: product_kernel<T, HP_ACT_NONE><<<grid, 256, 0, s>>>(a); break;
    case HP_ACT_RELU: product_kernel<T, HP_ACT_RELU><<<grid, 256, 0, s>>>(a); break;
    case HP_ACT_GELU: product_kernel<T, HP_ACT_GELU><<<grid, 256, 0, s>>>(a); break;
    default: product_kernel<T, HP_ACT_GELU_TANH><<<grid, 256, 0, s>>>(a); break;
  }
  return cudaGetLastError();
}

template <typename T>
int slopes(const HpSlope& a, cudaStream_t s) {
  const unsigned grid = (unsigned)((a.cols + 31) / 32);
  const dim3 block(32, 8);
  switch (a.act) {
    case HP_ACT_NONE: slope_kernel<T, HP_ACT_NONE><<<grid, block, 0, s>>>(a); break;
    case HP_ACT_RELU: slope_kernel<T, HP_ACT_RELU><<<grid, block, 0, s>>>(a); break;
    case HP_ACT_GELU: slope_kernel<T, HP_ACT_GELU><<<grid, block, 0, s>>>(a); break;
    default: slope_kernel<T, HP_ACT_GELU_TANH><<<grid, block, 0, s>>>(a); break;
  }
  return cudaGetLastError();
}

}  // namespace
}  // namespace hipress

using namespace hipress;

extern "C" int hp_cuda_product(const HpProduct* a, void* stream) {
  if (!a || a->m < 0 || a->n < 0 || a->k < 0 || a->m > INT32_MAX / 2 || a->n > INT32_MAX / 2 || a->k > INT32_MAX / 2 ||
      (a->type != HP_BF16 && a->type != HP_F16) || !type_ok(a->ytype) || !type_ok(a->btype) || a->act < 0 ||
      a->act > HP_ACT_GELU_TANH)
    return HP_ERR_BAD_ARG;
  if (!a->m || !a->n) return 0;
  cudaStream_t s = (cudaStream_t)stream;
  return a->type == HP_BF16 ? product<__nv_bfloat16>(*a, s) : product<__half>(*a, s);
}

extern "C" uint64_t hp_cuda_product_workspace(int64_t, int64_t, int64_t) { return 0; }

extern "C" int hp_cuda_slope(const HpSlope* a, void* stream) {
  if (!a || a->rows < 0 || a->cols < 0 || (a->type != HP_BF16 && a->type != HP_F16) || !type_ok(a->btype) ||
      a->act < 0 || a->act > HP_ACT_GELU_TANH || (a->rows && a->cols && a->act && !a->pre))
    return HP_ERR_BAD_ARG;
  if (!a->cols) return 0;
  cudaStream_t s = (cudaStream_t)stream;
  return a->type == HP_BF16 ? slopes<__nv_bfloat16>(*a, s) : slopes<__half>(*a, s);
}

extern "C" uint64_t hp_cuda_slope_workspace(int64_t, int64_t, int64_t) { return 0; }
