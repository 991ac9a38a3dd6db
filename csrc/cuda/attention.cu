// Attention, forward, and backward from recomputed probabilities.
#include "activation.cuh"
#include "tcgen05.cuh"

namespace hipress {
namespace {

constexpr int kB = 128;                 // queries and keys of a tile
constexpr uint32_t kPanel = kB * 128;   // bytes of 64 columns of a tile

__device__ __forceinline__ uint32_t staged(int r, int b) { return (uint32_t)(r * 128 + (b ^ ((r & 7) << 4))); }

// 2^x for the softmax is exp2_fast(); what a masked score becomes
constexpr float kNone = -INFINITY;

// Which of a tile's 128 columns a row may see, a bit each.
struct Seen {
  uint32_t w[4];
};
// columns lo .. hi-1 of the tile
__device__ __forceinline__ Seen seen_between(int lo, int hi) {
  Seen s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int a = min(max(lo - 32 * i, 0), 32), b = min(max(hi - 32 * i, 0), 32);
    const uint32_t below_b = b == 32 ? 0xffffffffu : (1u << b) - 1, below_a = a == 32 ? 0xffffffffu : (1u << a) - 1;
    s.w[i] = below_b & ~below_a;
  }
  return s;
}

// By a whole warp: the mask's bits of keys k0 .. k0+127 of one sequence, all in every lane.
__device__ __forceinline__ Seen mask_bits(const uint8_t* mask, int64_t k0, int64_t sk) {
  Seen s;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t k = k0 + 32 * i + lane;
    s.w[i] = __ballot_sync(0xffffffffu, k < sk && mask[k]);
  }
  return s;
}

struct Maps {
  CUtensorMap q, k, v, o, d_o, dq, dk, dv;
};
struct Launch {
  Maps map;
  HpAttention p;
  float c;             // |scale| log2(e)
  int negative;        // scale < 0
  uint32_t* status;
};

// ---------------------------------------------------------------------- forward
// A CTA has QT tiles of 128 queries of one head and walks over the keys, 128 at a time: scores
// S = q k^T into tensor memory, one thread a row for the softmax, probabilities back over the
// scores, O += P v.  While one tile's rows are at work the other's products run.  The sums keep a
// running maximum; the results so far are scaled anew only when it rises by more than 2^8 (the
// factor that 32-bit sums and 16-bit probabilities bear easily).  Bound: 2^x, 16 a cycle and SM.
template <int DP, int QT>
struct Forward {
  static constexpr int kPanels = DP / 64, kTile = kPanels * (int)kPanel, kStages = DP == 64 && QT == 2 ? 4 : 2;
  static constexpr int kThreads = 64 + 128 * QT;
  static constexpr int kSmem = QT * kTile + kStages * 2 * kTile + 1024 + 1024;
  static constexpr int kTmem = QT == 2 ? 512 : 256;
};
struct ForwardBars {
  uint64_t q_full, k_full[4], v_full[4], k_empty[4], v_empty[4], mask_full[4], s_full[2], p_full[2], o_full[2], drain;
  Seen seen[4];
  uint32_t tmem;
  Guard guard;
};

template <typename T, int DP, int QT>
__global__ void __launch_bounds__(64 + 128 * QT, QT == 1 ? 2 : 1) attention_forward_tiles(const __grid_constant__ Launch l) {
  using F = Forward<DP, QT>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sq = smem;
  uint8_t* skv = smem + QT * F::kTile;   // stages of k and v
  ForwardBars& bar = *(ForwardBars*)(skv + F::kStages * 2 * F::kTile);
  const HpAttention& p = l.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the tiles with the most keys first, where the mask is causal
  const int qt = (int)gridDim.x - 1 - (int)blockIdx.x, h = blockIdx.y, b = blockIdx.z, hk = h / (int)(p.heads / p.kv_heads);
  const int q0 = qt * kB * QT, sk = (int)p.sk, shift = (int)(p.sk - p.sq);
  // key tiles of each query tile
  int n[QT], most = 0;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int last = min(q0 + (t + 1) * kB, (int)p.sq) - 1;   // its last query
    const int keys = q0 + t * kB >= p.sq ? 0 : p.causal ? min(sk, max(0, last + shift + 1)) : sk;
    n[t] = (keys + kB - 1) / kB;
    most = max(most, n[t]);
  }
  if (threadIdx.x == 0) {
    mbar_init(&bar.q_full, 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bar.k_full[i], 1), mbar_init(&bar.v_full[i], 1), mbar_init(&bar.k_empty[i], 1), mbar_init(&bar.v_empty[i], 1);
      mbar_init(&bar.mask_full[i], 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&bar.s_full[i], 1), mbar_init(&bar.p_full[i], 128), mbar_init(&bar.o_full[i], 1);
    mbar_init(&bar.drain, 1);
    mbar_init_fence();
    bar.guard.gave_up = 0;
    bar.guard.status = l.status;
  }
  if (warp == 1) tmem_alloc<1>(&bar.tmem, F::kTmem);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = bar.tmem, tmem_o = tmem + QT * 128;   // scores, then results
  Guard& g = bar.guard;
  const bool masked = p.key_mask != nullptr;

  if (warp == 0) {
    // k and v of key tile j into stage j; the mask's bits beside them
    int waits = 0;   // copies to wait for should the CTA give up
    if (lane == 0 && most) {
      tma_prefetch(&l.map.k);
      tma_prefetch(&l.map.v);
      mbar_expect_tx(&bar.q_full, QT * F::kTile);
      for (int t = 0; t < QT; ++t)
        for (int i = 0; i < F::kPanels; ++i)
          tma_load_4d(sq + t * F::kTile + i * kPanel, &l.map.q, 64 * i, h, q0 + t * kB, b, &bar.q_full);
    }
    for (int j = 0; j < most; ++j) {
      const int s = j % F::kStages;
      const uint32_t ph = (j / F::kStages) & 1;
      uint8_t* k = skv + s * 2 * F::kTile;
      if (!guard_wait(&bar.k_empty[s], ph ^ 1, g, 0x10001)) break;
      if (lane == 0) {
        mbar_expect_tx(&bar.k_full[s], F::kTile);
        for (int i = 0; i < F::kPanels; ++i) tma_load_4d(k + i * kPanel, &l.map.k, 64 * i, hk, j * kB, b, &bar.k_full[s]);
      }
      // whoever reads the bits gives probabilities before the product that frees v
      if (!guard_wait(&bar.v_empty[s], ph ^ 1, g, 0x10003)) break;
      if (masked) {
        const Seen m = mask_bits(p.key_mask + b * p.mask_b, (int64_t)j * kB, sk);
        if (lane == 0) bar.seen[s] = m, mbar_arrive(&bar.mask_full[s]);
      }
      if (lane == 0) {
        mbar_expect_tx(&bar.v_full[s], F::kTile);
        for (int i = 0; i < F::kPanels; ++i)
          tma_load_4d(k + F::kTile + i * kPanel, &l.map.v, 64 * i, hk, j * kB, b, &bar.v_full[s]);
      }
      waits = j + 1;
    }
    __syncwarp();
    if (g.gave_up && lane == 0 && most) {   // nothing may land once the CTA is gone
      mbar_wait_bounded(&bar.q_full, 0, kWaitNs, g.status, HP_STATUS_TIMEOUT | 0x10004);
      for (int j = max(0, waits - F::kStages); j < waits; ++j) {
        mbar_wait_bounded(&bar.k_full[j % F::kStages], (j / F::kStages) & 1, kWaitNs, g.status, HP_STATUS_TIMEOUT | 0x10005);
        mbar_wait_bounded(&bar.v_full[j % F::kStages], (j / F::kStages) & 1, kWaitNs, g.status, HP_STATUS_TIMEOUT | 0x10006);
      }
      if (waits < most)   // the k of a tile whose v was not fetched
        mbar_wait_bounded(&bar.k_full[waits % F::kStages], (waits / F::kStages) & 1, kWaitNs / 64, g.status, HP_STATUS_TIMEOUT | 0x10007);
    }
  } else if (warp == 1) {
    if (lane == 0 && most) {
      const bool bf = p.type == HP_BF16;
      const uint32_t id_s = mma_idesc(128, 128, bf, true, true) | (l.negative ? kNegateA : 0);
      const uint32_t id_o = mma_idesc(128, DP, bf, true, false);
      bool ok = guard_wait(&bar.q_full, 0, g, 0x20001);
      auto scores = [&](int t, int j) {   // S_t = q_t k_j^T
        const int s = j % F::kStages;
        const uint32_t a = smem_u32(sq + t * F::kTile), k = smem_u32(skv + s * 2 * F::kTile);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
          const uint32_t at = (i / 4) * kPanel + (i % 4) * 32;
          mma_ss<1>(tmem + t * 128, mma_desc(a + at, 16, 1024), mma_desc(k + at, 16, 1024), id_s, i > 0);
        }
        mma_commit<1>(&bar.s_full[t]);
      };
      for (int j = 0; j <= most && ok; ++j) {   // scores of tile j, results of tile j - 1
        if (j < most) ok = guard_wait(&bar.k_full[j % F::kStages], (j / F::kStages) & 1, g, 0x20002);
        if (j > 0 && ok) ok = guard_wait(&bar.v_full[(j - 1) % F::kStages], ((j - 1) / F::kStages) & 1, g, 0x20003);
        tmem_fence_after();
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          if (!ok) break;
          if (j > 0 && j - 1 < n[t]) {
            ok = guard_wait(&bar.p_full[t], (j - 1) & 1, g, 0x20004);
            if (!ok) break;
            tmem_fence_after();
            const uint32_t v = smem_u32(skv + ((j - 1) % F::kStages) * 2 * F::kTile + F::kTile);
#pragma unroll
            for (int i = 0; i < kB / 16; ++i)
              mma_ts(tmem_o + t * DP, tmem + t * 128 + i * 8, mma_desc(v + i * 2048, kPanel, 1024), id_o, j > 1 || i > 0);
            mma_commit<1>(&bar.o_full[t]);
          }
          if (j < n[t]) scores(t, j);
        }
        if (j > 0) mma_commit<1>(&bar.v_empty[(j - 1) % F::kStages]);
        if (j < most) mma_commit<1>(&bar.k_empty[j % F::kStages]);
      }
      mma_commit<1>(&bar.drain);
    }
  } else {
    const int t = (warp - 2) >> 2, quad = warp & 3, r = 32 * quad + lane;   // one row to a thread
    const int row = q0 + t * kB + r, nt = QT == 1 ? n[0] : (t ? n[QT - 1] : n[0]);
    const uint32_t lanes = (uint32_t)(32 * quad) << 16, ts = tmem + t * 128 + lanes, to = tmem_o + t * DP + lanes;
    const int sees = p.causal ? min(sk, row + shift + 1) : sk;   // keys this row sees but for the mask
    float m = kNone, sum = 0.f;
    bool ok = true;
    for (int j = 0; j < nt; ++j) {
      const int s = j % F::kStages;
      Seen seen;
      bool whole = sees >= (j + 1) * kB;
      if (masked) {
        if (!guard_wait(&bar.mask_full[s], (j / F::kStages) & 1, g, 0x30001)) { ok = false; break; }
        seen = bar.seen[s];
        const bool all = (seen.w[0] & seen.w[1] & seen.w[2] & seen.w[3]) == 0xffffffffu;
        if (!all) {
          // no probability is left where a key is masked, but a product with what it holds would be
          // no number if that is none: its v counts as zero (rows behind the last key already do).
          // Each tile sees to it before it gives its probabilities.
          if (!guard_wait(&bar.v_full[s], (j / F::kStages) & 1, g, 0x30002)) { ok = false; break; }
          if (!(seen.w[quad] >> lane & 1)) {
            uint4* v = (uint4*)(skv + s * 2 * F::kTile + F::kTile + r * 128);
#pragma unroll
            for (int i = 0; i < F::kPanels; ++i)
#pragma unroll
              for (int k = 0; k < 8; ++k) v[i * (kPanel / 16) + k] = make_uint4(0, 0, 0, 0);
          }
          fence_async_shared();
        }
        whole = whole && all;
      }
      if (!__all_sync(0xffffffffu, whole)) {
        const Seen mine = seen_between(0, sees - j * kB);
#pragma unroll
        for (int i = 0; i < 4; ++i) seen.w[i] = masked ? seen.w[i] & mine.w[i] : mine.w[i];
        whole = false;
      }
      if (!guard_wait(&bar.s_full[t], j & 1, g, 0x30003)) { ok = false; break; }
      // the product before these scores is done too; every phase is waited for, so that none is mistaken
      if (j > 0 && !guard_wait(&bar.o_full[t], (j - 1) & 1, g, 0x30004)) { ok = false; break; }
      tmem_fence_after();
      float top = kNone;
#pragma unroll
      for (int c = 0; c < kB; c += 32) {
        uint32_t x[32];
        tmem_ld32(ts + c, x);
        tmem_wait_ld();
        if (whole) {
#pragma unroll
          for (int i = 0; i < 32; ++i) top = fmaxf(top, __uint_as_float(x[i]));
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) top = fmaxf(top, seen.w[c / 32] >> i & 1 ? __uint_as_float(x[i]) : kNone);
        }
      }
      top = top == kNone ? kNone : top * l.c;   // 0 times infinity otherwise
      if (__any_sync(0xffffffffu, top > m + 8.f || (m == kNone && top != kNone))) {
        const float now = fmaxf(m, top), keep = now == kNone ? 1.f : exp2_fast(m - now);
        sum *= keep;
        m = now;
        if (j > 0) {
#pragma unroll
          for (int c = 0; c < DP; c += 32) {
            uint32_t o[32];
            tmem_ld32(to + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
            tmem_st32(to + c, o);
          }
          tmem_wait_st();
        }
      }
      const float base = m == kNone ? 0.f : -m;
#pragma unroll
      for (int c = 0; c < kB; c += 32) {
        uint32_t x[32], y[16];
        tmem_ld32(ts + c, x);
        tmem_wait_ld();
        float e[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          e[i] = exp2_fast(fmaf(__uint_as_float(x[i]), l.c, base));
          if (!whole) e[i] = seen.w[c / 32] >> i & 1 ? e[i] : 0.f;
        }
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 32; ++i) part[i & 3] += e[i];
        sum += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = pack2<T>(e[2 * i], e[2 * i + 1]);
        tmem_st16(ts + c / 2, y);
      }
      tmem_wait_st();
      tmem_fence_before();
      mbar_arrive(&bar.p_full[t]);
    }
    const bool some = sum != 0.f;   // NaN too
    const float inv = some ? 1.f / sum : 0.f;
    if (row < p.sq) p.lse[(b * p.heads + h) * p.sq + row] = some ? (m + log2f(sum)) * 0.6931471805599453f : kNone;
    if (ok && nt) ok = guard_wait(&bar.o_full[t], (nt - 1) & 1, g, 0x30005);
    else if (ok && most) ok = guard_wait(&bar.q_full, 0, g, 0x30006);   // the copy into the space used below
    tmem_fence_after();
    // the rows leave through the space of their queries, which all products have read
    if (ok && q0 + t * kB < p.sq) {
#pragma unroll
      for (int i = 0; i < F::kPanels; ++i) {
        uint8_t* to_smem = sq + t * F::kTile + i * kPanel + 32 * quad * 128;
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          uint32_t o[32];
          if (nt) {
            tmem_ld32(to + 64 * i + c, o);
            tmem_wait_ld();
          }
          float v[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] = nt && some ? __uint_as_float(o[k]) * inv : 0.f;
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            *(uint4*)(to_smem + staged(lane, 2 * (c + k))) =
                make_uint4(pack2<T>(v[k], v[k + 1]), pack2<T>(v[k + 2], v[k + 3]), pack2<T>(v[k + 4], v[k + 5]),
                           pack2<T>(v[k + 6], v[k + 7]));
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) tma_store_4d(&l.map.o, to_smem, 64 * i, h, q0 + t * kB + 32 * quad, b), tma_store_commit();
      }
      if (lane == 0) tma_store_wait_read<0>();
    }
    tmem_fence_before();
  }
  __syncwarp();
  __syncthreads();
  if (warp == 1 && most) {
    if (lane == 0) {
      g.gave_up = 0;
      guard_wait(&bar.drain, 0, g, 0x60001);
    }
    __syncwarp();
  }
  tmem_fence_after();
  if (warp == 1) tmem_free<1>(tmem, F::kTmem);
}

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

// [batch, length, heads, dim] in boxes of 64 columns and `rows` rows of one head
bool head_map(CUtensorMap* m, const void* base, const HpAttention& a, int64_t length, int64_t heads, int64_t sb, int64_t ss,
              int64_t sh, uint32_t rows) {
  auto pitch = [](int64_t n, int64_t stride) { return (uint64_t)(n > 1 ? 2 * stride : 16); };   // of one there is no next
  const uint64_t size[4] = {(uint64_t)a.dim, (uint64_t)heads, (uint64_t)length, (uint64_t)a.batch};
  const uint64_t strides[3] = {pitch(heads, sh), pitch(length, ss), pitch(a.batch, sb)};
  const uint32_t box[4] = {64, 1, rows, 1};
  return tensor_map(m, base, (int)a.type, 4, size, strides, box);
}

int prepare(Launch& l, const HpAttention& a) {
  int rc;
  l.status = layer_status(&rc);
  l.p = a;
  l.c = (float)(a.scale < 0 ? -a.scale : a.scale) * kLog2e;
  l.negative = a.scale < 0;
  return rc;
}

template <typename T, int DP, int QT>
int forward_tiles(const Launch& l, cudaStream_t s) {
  using F = Forward<DP, QT>;
  static const cudaError_t allowed =
      cudaFuncSetAttribute(attention_forward_tiles<T, DP, QT>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem);
  if (allowed != cudaSuccess) return allowed;
  const dim3 grid((unsigned)((l.p.sq + kB * QT - 1) / (kB * QT)), (unsigned)l.p.heads, (unsigned)l.p.batch);
  attention_forward_tiles<T, DP, QT><<<grid, F::kThreads, F::kSmem, s>>>(l);
  return cudaGetLastError();
}

template <typename T>
int forward(const HpAttention& a, cudaStream_t s) {
  Launch l;
  if (const int rc = prepare(l, a)) return rc;
  if (!head_map(&l.map.q, a.q, a, a.sq, a.heads, a.q_b, a.q_s, a.q_h, kB) ||
      !head_map(&l.map.k, a.sk ? a.k : a.q, a, a.sk, a.kv_heads, a.k_b, a.k_s, a.k_h, kB) ||
      !head_map(&l.map.v, a.sk ? a.v : a.q, a, a.sk, a.kv_heads, a.v_b, a.v_s, a.v_h, kB) ||
      !head_map(&l.map.o, a.o, a, a.sq, a.heads, a.o_b, a.o_s, a.o_h, 32))
    return HP_ERR_BAD_ARG;
  const bool two = a.sq > kB;
  if (a.dim <= 64) return two ? forward_tiles<T, 64, 2>(l, s) : forward_tiles<T, 64, 1>(l, s);
  return two ? forward_tiles<T, 128, 2>(l, s) : forward_tiles<T, 128, 1>(l, s);
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
