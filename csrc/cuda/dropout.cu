// Dropout of any tensor, with a residual: y = kept ? x / share : 0 (+ residual).
//
// Bound: the traffic, x (residual) in and y out; a word of random bits takes about 130 instructions for
// 32 elements, and is made while the loads are under way.  A warp has 1024 elements, 32 words: each lane
// makes one word, and a shuffle hands its bits to the lanes whose pieces of 16 bytes they are of, so that
// loads and stores stay side by side.
#include "philox.cuh"

namespace hipress {
namespace {

constexpr int kChunk = 1024, kThreads = 256;

template <typename T, bool ALIGNED>
__device__ __forceinline__ void take(const T* from, int64_t i, int64_t n, float (&v)[kPiece<T>]) {
  constexpr int V = kPiece<T>;
  if (ALIGNED && i + V <= n) {
    unpack<T>(*(const uint4*)(from + i), v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = i + j < n ? to_f(from[i + j]) : 0.f;
  }
}

template <typename T, bool ALIGNED, bool RESIDUAL>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const __grid_constant__ HpDrop a, const __grid_constant__ Drop d) {
  constexpr int V = kPiece<T>, PIECES = kChunk / 32 / V;
  const int lane = threadIdx.x & 31;
  const int64_t chunk = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5, first = chunk * kChunk;
  dependents_may_start();
  wait_for_kernel_before();
  if (first >= a.n) return;
  const T *x = (const T*)a.x, *r = (const T*)a.residual;
  float v[PIECES][V], u[RESIDUAL ? PIECES : 1][V];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    take<T, ALIGNED>(x, first + (i * 32 + lane) * V, a.n, v[i]);
    if (RESIDUAL) take<T, ALIGNED>(r, first + (i * 32 + lane) * V, a.n, u[i]);
  }
  const uint32_t mine = kept_word(d, drop_key(d), (uint64_t)(chunk * 32 + lane));
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const uint32_t bits = __shfl_sync(0xffffffffu, mine, (i * 32 + lane) * V / 32) >> (lane * V & 31);
    const int64_t at = first + (i * 32 + lane) * V;
    float y[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      y[j] = bits >> j & 1 ? v[i][j] * d.up : 0.f;
      if (RESIDUAL) y[j] += u[i][j];
    }
    T* to = (T*)a.y + at;
    if (at + V <= a.n) *(uint4*)to = pack<T>(y);
    else
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (at + j < a.n) to[j] = from_f<T>(y[j]);
  }
}

template <typename T>
int run(const HpDrop& a, const Drop& d, cudaStream_t s) {
  const int64_t ctas = (a.n + kChunk * (kThreads / 32) - 1) / (kChunk * (kThreads / 32));
  if (ctas > INT32_MAX) return HP_ERR_TOO_LARGE;
  const bool aligned = ((uintptr_t)a.x | (uintptr_t)a.residual) % 16 == 0;
  const auto kernel = a.residual ? (aligned ? dropout_kernel<T, true, true> : dropout_kernel<T, false, true>)
                                 : (aligned ? dropout_kernel<T, true, false> : dropout_kernel<T, false, false>);
  return launch_behind(kernel, (unsigned)ctas, kThreads, 0, s, a, d);
}

}  // namespace
}  // namespace hipress

using namespace hipress;

extern "C" int hp_cuda_dropout(const HpDrop* a, void* stream) {
  Drop d;
  if (!a || a->n < 0 || !type_ok(a->type) || (uintptr_t)a->y % 16 || !drop_of(&d, a->drop)) return HP_ERR_BAD_ARG;
  if (!a->n) return 0;
  cudaStream_t s = (cudaStream_t)stream;
  return a->type == HP_F32 ? run<float>(*a, d, s) : a->type == HP_BF16 ? run<__nv_bfloat16>(*a, d, s) : run<__half>(*a, d, s);
}
