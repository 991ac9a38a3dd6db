// Attention, forward, and backward from recomputed probabilities.
#include "layers.cuh"

namespace hipress {
namespace {

constexpr int kWarps = 4, kMaxDim = 128;

__device__ __forceinline__ bool sees(const HpAttention& a, int64_t b, int64_t i, int64_t j) {
  return j < a.sk && (!a.causal || j <= i + a.sk - a.sq) && (!a.key_mask || a.key_mask[b * a.mask_b + j]);
}

template <typename T>
__device__ __forceinline__ float dot(const float* x, const T* y, int d) {
  float s = 0.f;
  for (int i = 0; i < d; ++i) s = fmaf(x[i], to_f(y[i]), s);
  return s;
}

// One warp for each query row; the lanes share the keys of a chunk, then the dimensions.
template <typename T>
__global__ void __launch_bounds__(32 * kWarps) attention_forward_kernel(const __grid_constant__ HpAttention a) {
  __shared__ float sq[kWarps][kMaxDim];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, d = (int)a.dim;
  const int64_t i = (int64_t)blockIdx.x * kWarps + w, h = blockIdx.y, b = blockIdx.z, hk = h / (a.heads / a.kv_heads);
  if (i >= a.sq) return;
  const T* q = (const T*)a.q + b * a.q_b + i * a.q_s + h * a.q_h;
  const T* k = (const T*)a.k + b * a.k_b + hk * a.k_h;
  const T* v = (const T*)a.v + b * a.v_b + hk * a.v_h;
  for (int c = lane; c < d; c += 32) sq[w][c] = to_f(q[c]);
  __syncwarp();
  float top = -INFINITY, sum = 0.f, acc[kMaxDim / 32] = {};
  for (int64_t j0 = 0; j0 < a.sk; j0 += 32) {
    const bool see = sees(a, b, i, j0 + lane);
    const float x = see ? dot(sq[w], k + (j0 + lane) * a.k_s, d) * (float)a.scale : -INFINITY;
    float m = x;
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (!__any_sync(0xffffffffu, see)) continue;
    m = fmaxf(m, top);
    const float keep = expf(top - m), p = see ? expf(x - m) : 0.f;
    sum = fmaf(sum, keep, p);   // each lane its own keys
    for (int c = 0; c < kMaxDim / 32; ++c) acc[c] *= keep;
    for (int l = 0; l < 32; ++l) {
      const float pl = __shfl_sync(0xffffffffu, p, l);
      if (pl == 0.f) continue;
      for (int c = 0; c < kMaxDim / 32; ++c)
        if (32 * c + lane < d) acc[c] = fmaf(pl, to_f(v[(j0 + l) * a.v_s + 32 * c + lane]), acc[c]);
    }
    top = m;
  }
  sum = warp_sum(sum);
  T* o = (T*)a.o + b * a.o_b + i * a.o_s + h * a.o_h;
  for (int c = 0; c < kMaxDim / 32; ++c)
    if (32 * c + lane < d) o[32 * c + lane] = from_f<T>(sum != 0.f ? acc[c] / sum : 0.f);
  if (lane == 0) a.lse[(b * a.heads + h) * a.sq + i] = sum != 0.f ? top + logf(sum) : -INFINITY;
}

// rows of d_o against rows of o: [batch, heads, sq]
template <typename T>
__global__ void __launch_bounds__(32 * kWarps) attention_delta_kernel(const __grid_constant__ HpAttention a) {
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t i = (int64_t)blockIdx.x * kWarps + w, h = blockIdx.y, b = blockIdx.z;
  if (i >= a.sq) return;
  const T* o = (const T*)a.o + b * a.o_b + i * a.o_s + h * a.o_h;
  const T* g = (const T*)a.d_o + b * a.do_b + i * a.do_s + h * a.do_h;
  float s = 0.f;
  for (int c = lane; c < a.dim; c += 32) s = fmaf(to_f(o[c]), to_f(g[c]), s);
  s = warp_sum(s);
  if (lane == 0) a.delta[(b * a.heads + h) * a.sq + i] = s;
}

template <typename T>
__global__ void __launch_bounds__(32 * kWarps) attention_dq_kernel(const __grid_constant__ HpAttention a) {
  __shared__ float sq[kWarps][kMaxDim], sg[kWarps][kMaxDim];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, d = (int)a.dim;
  const int64_t i = (int64_t)blockIdx.x * kWarps + w, h = blockIdx.y, b = blockIdx.z, hk = h / (a.heads / a.kv_heads);
  if (i >= a.sq) return;
  const T* q = (const T*)a.q + b * a.q_b + i * a.q_s + h * a.q_h;
  const T* g = (const T*)a.d_o + b * a.do_b + i * a.do_s + h * a.do_h;
  const T* k = (const T*)a.k + b * a.k_b + hk * a.k_h;
  const T* v = (const T*)a.v + b * a.v_b + hk * a.v_h;
  for (int c = lane; c < d; c += 32) sq[w][c] = to_f(q[c]), sg[w][c] = to_f(g[c]);
  __syncwarp();
  const int64_t at = (b * a.heads + h) * a.sq + i;
  const float lse = a.lse[at], delta = a.delta[at];
  float acc[kMaxDim / 32] = {};
  for (int64_t j0 = 0; j0 < a.sk; j0 += 32) {
    const int64_t j = j0 + lane;
    float ds = 0.f;
    const bool see = sees(a, b, i, j);
    if (see) {
      const float p = expf(dot(sq[w], k + j * a.k_s, d) * (float)a.scale - lse);
      ds = p * (dot(sg[w], v + j * a.v_s, d) - delta);
    }
    for (unsigned left = __ballot_sync(0xffffffffu, see); left; left &= left - 1) {
      const int l = __ffs(left) - 1;
      const float dl = __shfl_sync(0xffffffffu, ds, l);
      for (int c = 0; c < kMaxDim / 32; ++c)
        if (32 * c + lane < d) acc[c] = fmaf(dl, to_f(k[(j0 + l) * a.k_s + 32 * c + lane]), acc[c]);
    }
  }
  T* o = (T*)a.dq + b * a.dq_b + i * a.dq_s + h * a.dq_h;
  for (int c = 0; c < kMaxDim / 32; ++c)
    if (32 * c + lane < d) o[32 * c + lane] = from_f<T>(acc[c] * (float)a.scale);
}

// One warp for each key row: the lanes share the queries of a chunk, of every head that reads it.
template <typename T>
__global__ void __launch_bounds__(32 * kWarps) attention_dkv_kernel(const __grid_constant__ HpAttention a) {
  __shared__ float sk[kWarps][kMaxDim], sv[kWarps][kMaxDim];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, d = (int)a.dim;
  const int64_t j = (int64_t)blockIdx.x * kWarps + w, hk = blockIdx.y, b = blockIdx.z, group = a.heads / a.kv_heads;
  if (j >= a.sk) return;
  const T* k = (const T*)a.k + b * a.k_b + j * a.k_s + hk * a.k_h;
  const T* v = (const T*)a.v + b * a.v_b + j * a.v_s + hk * a.v_h;
  for (int c = lane; c < d; c += 32) sk[w][c] = to_f(k[c]), sv[w][c] = to_f(v[c]);
  __syncwarp();
  float dk[kMaxDim / 32] = {}, dv[kMaxDim / 32] = {};
  for (int64_t h = hk * group; h < (hk + 1) * group; ++h) {
    const T* q = (const T*)a.q + b * a.q_b + h * a.q_h;
    const T* g = (const T*)a.d_o + b * a.do_b + h * a.do_h;
    for (int64_t i0 = 0; i0 < a.sq; i0 += 32) {
      const int64_t i = i0 + lane, at = (b * a.heads + h) * a.sq + i;
      float p = 0.f, ds = 0.f;
      const bool see = i < a.sq && sees(a, b, i, j);
      if (see) {
        p = expf(dot(sk[w], q + i * a.q_s, d) * (float)a.scale - a.lse[at]);
        ds = p * (dot(sv[w], g + i * a.do_s, d) - a.delta[at]);
      }
      for (unsigned left = __ballot_sync(0xffffffffu, see); left; left &= left - 1) {
        const int l = __ffs(left) - 1;
        const float pl = __shfl_sync(0xffffffffu, p, l), dl = __shfl_sync(0xffffffffu, ds, l);
        for (int c = 0; c < kMaxDim / 32; ++c)
          if (32 * c + lane < d) {
            dv[c] = fmaf(pl, to_f(g[(i0 + l) * a.do_s + 32 * c + lane]), dv[c]);
            dk[c] = fmaf(dl, to_f(q[(i0 + l) * a.q_s + 32 * c + lane]), dk[c]);
          }
      }
    }
  }
  T* ok = (T*)a.dk + b * a.dk_b + j * a.dk_s + hk * a.dk_h;
  T* ov = (T*)a.dv + b * a.dv_b + j * a.dv_s + hk * a.dv_h;
  for (int c = 0; c < kMaxDim / 32; ++c)
    if (32 * c + lane < d) {
      ok[32 * c + lane] = from_f<T>(dk[c] * (float)a.scale);
      ov[32 * c + lane] = from_f<T>(dv[c]);
    }
}

bool args_ok(const HpAttention* a) {
  return a && a->batch >= 0 && a->batch <= 65535 && a->sq >= 0 && a->sk >= 0 && a->sq <= INT32_MAX / 2 &&
         a->sk <= INT32_MAX / 2 && a->kv_heads >= 1 && a->heads >= 1 && a->heads <= 65535 &&
         a->heads % a->kv_heads == 0 && a->dim >= 8 && a->dim <= kMaxDim && a->dim % 8 == 0 &&
         (a->type == HP_BF16 || a->type == HP_F16);
}

template <typename T>
int forward(const HpAttention& a, cudaStream_t s) {
  const dim3 grid((unsigned)((a.sq + kWarps - 1) / kWarps), (unsigned)a.heads, (unsigned)a.batch);
  attention_forward_kernel<T><<<grid, 32 * kWarps, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T>
int backward(const HpAttention& a, cudaStream_t s) {
  const dim3 grid((unsigned)((a.sq + kWarps - 1) / kWarps), (unsigned)a.heads, (unsigned)a.batch);
  const dim3 keys((unsigned)((a.sk + kWarps - 1) / kWarps), (unsigned)a.kv_heads, (unsigned)a.batch);
  if (a.sq) {
    attention_delta_kernel<T><<<grid, 32 * kWarps, 0, s>>>(a);
    attention_dq_kernel<T><<<grid, 32 * kWarps, 0, s>>>(a);
  }
  if (a.sk) attention_dkv_kernel<T><<<keys, 32 * kWarps, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace hipress

using namespace hipress;

extern "C" int hp_cuda_attention_forward(const HpAttention* a, void* stream) {
  if (!args_ok(a)) return HP_ERR_BAD_ARG;
  if (!a->batch || !a->sq) return 0;
  cudaStream_t s = (cudaStream_t)stream;
  return a->type == HP_BF16 ? forward<__nv_bfloat16>(*a, s) : forward<__half>(*a, s);
}

extern "C" int hp_cuda_attention_backward(const HpAttention* a, void* stream) {
  if (!args_ok(a)) return HP_ERR_BAD_ARG;
  if (!a->batch) return 0;
  cudaStream_t s = (cudaStream_t)stream;
  return a->type == HP_BF16 ? backward<__nv_bfloat16>(*a, s) : backward<__half>(*a, s);
}
