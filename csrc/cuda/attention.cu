// Attention, forward, and backward from recomputed probabilities.
#include <type_traits>

#include "activation.cuh"
#include "tcgen05.cuh"

namespace hipress {
namespace {

constexpr int kB = 128;                 // queries and keys of a tile
constexpr int kMaxDim = 128;
constexpr uint32_t kPanel = kB * 128;   // bytes of 64 columns of a tile

__device__ __forceinline__ uint32_t staged(int r, int b) { return (uint32_t)(r * 128 + (b ^ ((r & 7) << 4))); }

// 2^x for the softmax is exp2_fast(); what a masked score becomes
constexpr float kNone = -INFINITY;

// Two values at a time: half the instructions for what is not 2^x.
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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

struct Yes {
  __device__ constexpr operator bool() const { return true; }
};
struct No {
  __device__ constexpr operator bool() const { return false; }
};

// Which of a tile's columns a row may see, a bit each.
template <int COLS>
struct Seen {
  uint32_t w[COLS / 32];
  __device__ __forceinline__ bool all() const {
    uint32_t a = w[0];
#pragma unroll
    for (int i = 1; i < COLS / 32; ++i) a &= w[i];
    return a == 0xffffffffu;
  }
  __device__ __forceinline__ bool none() const {
    uint32_t a = w[0];
#pragma unroll
    for (int i = 1; i < COLS / 32; ++i) a |= w[i];
    return a == 0;
  }
};
// columns lo .. hi-1 of the tile
template <int COLS>
__device__ __forceinline__ Seen<COLS> seen_between(int lo, int hi) {
  Seen<COLS> s;
#pragma unroll
  for (int i = 0; i < COLS / 32; ++i) {
    const int a = min(max(lo - 32 * i, 0), 32), b = min(max(hi - 32 * i, 0), 32);
    const uint32_t below_b = b == 32 ? 0xffffffffu : (1u << b) - 1, below_a = a == 32 ? 0xffffffffu : (1u << a) - 1;
    s.w[i] = below_b & ~below_a;
  }
  return s;
}

// By a whole warp: the mask's bits of keys from k0 on of one sequence, all in every lane.
template <int COLS>
__device__ __forceinline__ Seen<COLS> mask_bits(const uint8_t* mask, int64_t k0, int64_t sk) {
  Seen<COLS> s;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < COLS / 32; ++i) {
    const int64_t k = k0 + 32 * i + lane;
    s.w[i] = __ballot_sync(0xffffffffu, k < sk && mask[k]);
  }
  return s;
}

// By the whole CTA: one more than the last key that a sequence's mask lets see.
__device__ __forceinline__ int visible_keys(const uint8_t* mask, int sk, int* shared) {
  if (threadIdx.x == 0) *shared = 0;
  __syncthreads();
  int last = 0;
  for (int k = threadIdx.x; k < sk; k += blockDim.x)
    if (mask[k]) last = k + 1;
#pragma unroll
  for (int o = 16; o; o >>= 1) last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
  if ((threadIdx.x & 31) == 0) atomicMax(shared, last);
  __syncthreads();
  return *shared;
}

struct Maps {
  CUtensorMap q, k, v, o, d_o, dq, dk, dv;
  CUtensorMap q64, k64, v64, do64;   // in boxes of 64 rows
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
// scores, O += P v.  While some rows are at work another tile's or another CTA's products run.  The
// sums keep a running maximum; the results so far are scaled anew only when it rises by more than 2^8
// (the factor that 32-bit sums and 16-bit probabilities bear easily).  Bound: 2^x, 16 a cycle and SM.
//   <64, 1>        two CTAs an SM.  Four tiles of queries against 64 keys at a time in one CTA that has
//                  the SM alone took 0.9 to 1.07 times as long where the SMs were full (64 x 300 tokens
//                  of 16 heads: 95 against 106 us, 1 x 8192 of 16, causal: both 207) and up to twice as
//                  long where not (1 x 4096 of 16, causal: 111 against 64)
//   <128, 1>, <128, 2>   tensor memory holds the results of two CTAs, or of one CTA's two tiles, which
//                  share the keys they fetch
//   SHORT          up to 128 queries and keys: one tile each, nothing to walk over.  Results take the
//                  half of the scores' columns that the probabilities leave, so that four CTAs fit
//                  an SM and hide one another's latency
template <int DP, int QT, bool SHORT>
struct Forward {
  static constexpr int kPanels = DP / 64, kTile = kPanels * (int)kPanel;   // bytes
  // two stages of keys; four warps that fetch and issue, one for each tile, and four for each tile's
  // rows; the former give registers to the latter
  static constexpr int kStages = SHORT ? 1 : 2, kThreads = 128 + 128 * QT, kPerSm = SHORT ? 4 : QT == 1 ? 2 : 1;
  static constexpr int kAtStart = SHORT ? 64 : QT == 1 ? 128 : 168;
  static constexpr int kFew = SHORT ? 64 : 72, kMany = SHORT ? 64 : QT == 1 ? 184 : 216;
  static_assert(kFew + QT * kMany <= (1 + QT) * kAtStart, "more registers than the CTA has");
  static constexpr int kSmem = QT * kTile + kStages * 2 * kTile + 1024 + 1024;
  static constexpr int kTmem = SHORT ? 128 : QT == 1 ? 256 : 512;
  // columns: scores of each tile, results, probabilities.  Where there is room these have columns of
  // their own, and the next scores need not wait for the product that reads them
  static constexpr bool kApart = !SHORT && DP == 64;
  static constexpr uint32_t kO = SHORT ? 64 : QT * kB, kP = kApart ? kB + DP : 0;
};
struct ForwardBars {
  uint64_t q_full, k_full[2], v_full[2], k_empty[2], v_empty[2], mask_full[2], s_full[2], s_free[2], p_full[2], o_full[2], drain;
  Seen<kB> seen[2];
  uint32_t tmem;
  int keys;
  Guard guard;
};

template <typename T, int DP, int QT, bool SHORT>
__global__ void __launch_bounds__((Forward<DP, QT, SHORT>::kThreads), (Forward<DP, QT, SHORT>::kPerSm))
attention_forward_tiles(const __grid_constant__ Launch l) {
  using F = Forward<DP, QT, SHORT>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sq = smem;
  uint8_t* skv = smem + QT * F::kTile;   // stages of k and v
  ForwardBars& bar = *(ForwardBars*)(skv + F::kStages * 2 * F::kTile);
  const HpAttention& p = l.p;
  const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  // of all heads first the tiles with the most keys, where the mask is causal
  const int qt = (int)gridDim.y - 1 - (int)blockIdx.y, h = blockIdx.x % (int)p.heads, b = blockIdx.x / (int)p.heads;
  const int hk = h / (int)(p.heads / p.kv_heads);
  const int q0 = qt * kB * QT, shift = (int)(p.sk - p.sq);
  const bool masked = p.key_mask != nullptr;
  const uint8_t* mask = masked ? p.key_mask + b * p.mask_b : nullptr;
  wait_for_kernel_before();
  const int sk = !SHORT && masked && p.sk > kB ? visible_keys(mask, (int)p.sk, &bar.keys) : (int)p.sk;
  // key tiles of a query tile: up to the last that its last query sees
  auto tiles_of = [&](int t) {
    const int first = q0 + t * kB, last = min(first + kB, (int)p.sq) - 1;
    const int keys = first >= p.sq ? 0 : p.causal ? min(sk, max(0, last + shift + 1)) : sk;
    return (keys + kB - 1) / kB;
  };
  int most = 0;
#pragma unroll
  for (int t = 0; t < QT; ++t) most = max(most, tiles_of(t));
  if (threadIdx.x == 0) {
    mbar_init(&bar.q_full, 1);
    for (int i = 0; i < F::kStages; ++i) {
      mbar_init(&bar.k_full[i], 1), mbar_init(&bar.v_full[i], 1), mbar_init(&bar.mask_full[i], 1);
      mbar_init(&bar.k_empty[i], QT), mbar_init(&bar.v_empty[i], QT);
    }
    for (int i = 0; i < QT; ++i) {
      mbar_init(&bar.s_full[i], 1), mbar_init(&bar.s_free[i], 128);
      mbar_init(&bar.p_full[i], 128), mbar_init(&bar.o_full[i], 1);
    }
    mbar_init(&bar.drain, QT);
    mbar_init_fence();
    bar.guard.gave_up = 0;
    bar.guard.status = l.status;
  }
  if (warp == 1) tmem_alloc<1>(&bar.tmem, F::kTmem);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  dependents_may_start();
  const uint32_t tmem = uniform(bar.tmem), tmem_o = tmem + F::kO;
  Guard& g = bar.guard;

  if (warp < 4) {
    if (F::kFew < F::kMany) fewer_registers<F::kFew>();
    if (warp == 0) {
      // k and v of key tile j into stage j; the mask's bits beside them
      int waits = 0;   // copies to wait for should the CTA give up
      if (lane == 0 && most) {
        tma_prefetch(&l.map.k);
        tma_prefetch(&l.map.v);
        mbar_expect_tx(&bar.q_full, QT * F::kTile);
#pragma unroll 1
        for (int i = 0; i < QT * F::kPanels; ++i)
          tma_load_4d(sq + i * kPanel, &l.map.q, 64 * (i % F::kPanels), h, q0 + i / F::kPanels * kB, b, &bar.q_full);
      }
      int s = 0;
      uint32_t ph = 0;
      for (int j = 0; j < most; ++j) {
        uint8_t* k = skv + s * 2 * F::kTile;
        if (!guard_wait(&bar.k_empty[s], ph ^ 1, g, 0x10001)) break;
        if (lane == 0) {
          mbar_expect_tx(&bar.k_full[s], F::kTile);
          for (int i = 0; i < F::kPanels; ++i) tma_load_4d(k + i * kB * 128, &l.map.k, 64 * i, hk, j * kB, b, &bar.k_full[s]);
        }
        // whoever reads the bits gives probabilities before the product that frees v
        if (!guard_wait(&bar.v_empty[s], ph ^ 1, g, 0x10003)) break;
        if (masked) {
          const Seen<kB> m = mask_bits<kB>(mask, (int64_t)j * kB, sk);
          if (lane == 0) bar.seen[s] = m, mbar_arrive(&bar.mask_full[s]);
        }
        if (lane == 0) {
          mbar_expect_tx(&bar.v_full[s], F::kTile);
          for (int i = 0; i < F::kPanels; ++i)
            tma_load_4d(k + F::kTile + i * kB * 128, &l.map.v, 64 * i, hk, j * kB, b, &bar.v_full[s]);
        }
        waits = j + 1;
        if (++s == F::kStages) s = 0, ph ^= 1;
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
    } else if (warp <= QT) {
      if (most) {
        const int t = warp - 1, tiles = tiles_of(t);   // each for its own tile
        const uint32_t leader = elect_one();
        const bool bf = p.type == HP_BF16;
        const uint32_t id_s = mma_idesc(128, kB, bf, true, true) | (l.negative ? kNegateA : 0);
        const uint32_t id_o = mma_idesc(128, DP, bf, true, false);
        bool ok = warp_wait(&bar.q_full, 0, g, 0x20001);
        auto scores = [&](int s) {   // S_t = q_t k^T of the stage
          const uint64_t a = mma_desc(smem_u32(sq + t * F::kTile), 16, 1024), k = mma_desc(smem_u32(skv + s * 2 * F::kTile), 16, 1024);
#pragma unroll
          for (int i = 0; i < DP / 16; ++i)
            mma_ss<1>(leader, tmem + t * kB, a + ((i / 4) * kPanel + (i % 4) * 32) / 16, k + ((i / 4) * kB * 128 + (i % 4) * 32) / 16, id_s, i > 0);
          mma_commit<1>(leader, &bar.s_full[t]);
        };
        auto results = [&](int s, bool add) {   // O_t += P_t v
          const uint64_t v = mma_desc(smem_u32(skv + s * 2 * F::kTile + F::kTile), kB * 128, 1024);
#pragma unroll
          for (int i = 0; i < kB / 16; ++i)
            mma_ts(leader, tmem_o + t * DP, tmem + F::kP + t * kB + i * 8, v + i * 128, id_o, add || i > 0);
          mma_commit<1>(leader, &bar.o_full[t]);
        };
        int s = 0, s_before = 0;
        uint32_t ph = 0, ph_before = 0;
        for (int j = 0; j <= most && ok; ++j) {   // scores of tile j, results of tile j - 1
          if (j < most) ok = warp_wait(&bar.k_full[s], ph, g, 0x20002);
          if (F::kApart && j < tiles && ok) {   // scores as soon as the last ones have been read
            if (j > 0) ok = warp_wait(&bar.s_free[t], (j - 1) & 1, g, 0x20005);
            tmem_fence_after();
            if (ok) scores(s);
          }
          if (F::kApart && ok && j < most) mma_commit<1>(leader, &bar.k_empty[s]);
          if (j > 0 && ok) ok = warp_wait(&bar.v_full[s_before], ph_before, g, 0x20003);
          tmem_fence_after();
          if (j > 0 && j - 1 < tiles && ok) {
            ok = warp_wait(&bar.p_full[t], (j - 1) & 1, g, 0x20004);
            tmem_fence_after();
            if (ok) results(s_before, j > 1);
          }
          if (!F::kApart && j < tiles && ok) scores(s);   // over the probabilities just used
          if (j > 0) mma_commit<1>(leader, &bar.v_empty[s_before]);
          if (!F::kApart && j < most) mma_commit<1>(leader, &bar.k_empty[s]);
          s_before = s, ph_before = ph;
          if (++s == F::kStages) s = 0, ph ^= 1;
        }
        mma_commit<1>(leader, &bar.drain);
      }
    }
  } else {
    if (F::kFew < F::kMany) more_registers<F::kMany>();
    const int t = (warp - 4) >> 2, quad = warp & 3, r = 32 * quad + lane;   // one row to a thread
    const int row = q0 + t * kB + r, nt = tiles_of(t);
    const uint32_t lanes = (uint32_t)(32 * quad) << 16, ts = tmem + t * kB + lanes, to = tmem_o + t * DP + lanes;
    const uint32_t tp = tmem + F::kP + t * kB + lanes;
    const int sees = p.causal ? min(sk, row + shift + 1) : sk;   // keys this row sees but for the mask
    float m = kNone, sum = 0.f;
    bool ok = true;
    int s = 0;
    uint32_t ph = 0;
    for (int j = 0; j < nt; ++j) {
      Seen<kB> seen;
      bool whole = sees >= (j + 1) * kB;
      if (masked) {
        if (!guard_wait(&bar.mask_full[s], ph, g, 0x30001)) { ok = false; break; }
        seen = bar.seen[s];
        const bool all = seen.all();
        if (!all) {
          // no probability is left where a key is masked, but a product with what it holds would be
          // no number if that is none: its v counts as zero (rows behind the last key already do).
          // Each tile sees to it before it gives its probabilities.
          if (!guard_wait(&bar.v_full[s], ph, g, 0x30002)) { ok = false; break; }
          if (!(seen.w[quad] >> lane & 1)) {
            uint4* v = (uint4*)(skv + s * 2 * F::kTile + F::kTile + r * 128);
#pragma unroll
            for (int i = 0; i < F::kPanels; ++i)
#pragma unroll
              for (int k = 0; k < 8; ++k) v[i * kB * 8 + k] = make_uint4(0, 0, 0, 0);
          }
          fence_async_shared();
        }
        whole = whole && all;
      }
      if (!__all_sync(0xffffffffu, whole)) {
        const Seen<kB> mine = seen_between<kB>(0, sees - j * kB);
#pragma unroll
        for (int i = 0; i < kB / 32; ++i) seen.w[i] = masked ? seen.w[i] & mine.w[i] : mine.w[i];
        whole = false;
      }
      if (++s == F::kStages) s = 0, ph ^= 1;
      if (!guard_wait(&bar.s_full[t], j & 1, g, 0x30003)) { ok = false; break; }
      tmem_fence_after();
      // a row of scores stays in registers where those suffice, else it is read twice, in steps
      constexpr int kStep = SHORT ? 16 : 32, kHeld = SHORT ? kStep : kB;
      uint32_t x[kHeld];
      auto read = [&](int c, uint32_t* to) {
        if constexpr (SHORT) tmem_ld16(ts + c, *(uint32_t(*)[16])to);
        else tmem_ld32(ts + c, *(uint32_t(*)[32])to);
      };
      float part[4] = {kNone, kNone, kNone, kNone};
      if (!SHORT) {
#pragma unroll
        for (int c = 0; c < kB; c += kStep) read(c, x + c % kHeld);
        tmem_wait_ld();
        if (F::kApart) {
          tmem_fence_before();
          mbar_arrive(&bar.s_free[t]);
        }
      }
      auto highest = [&](auto all) {   // tiles that are seen whole test no bits
#pragma unroll
        for (int c = 0; c < kB; c += kStep) {
          if (SHORT) {
            read(c, x);
            tmem_wait_ld();
          }
#pragma unroll
          for (int i = 0; i < kStep; i += 2) {
            const float v = __uint_as_float(x[(c + i) % kHeld]), w = __uint_as_float(x[(c + i + 1) % kHeld]);
            const uint32_t two = all ? 3 : seen.w[c / 32] >> (c % 32 + i) & 3;
            float& top = part[i / 2 & 3];
            top = max3(top, all || (two & 1) ? v : kNone, all || (two & 2) ? w : kNone);
          }
        }
      };
      if (whole) highest(Yes());
      else highest(No());
      float top = max3(fmaxf(part[0], part[1]), part[2], part[3]);
      top = top == kNone ? kNone : top * l.c;   // 0 times infinity otherwise
      // the product of the last tile's probabilities: awaited before its results are scaled or its
      // probabilities replaced, and once a tile, so that no phase of the barrier is mistaken.  Where
      // scores and probabilities share columns these scores have come after it.
      bool behind = j > 0;
      auto settle = [&] {
        if (!behind) return true;
        behind = false;
        const bool done = guard_wait(&bar.o_full[t], (j - 1) & 1, g, 0x30004);
        tmem_fence_after();
        return done;
      };
      if (__any_sync(0xffffffffu, top > m + 8.f || (m == kNone && top != kNone))) {
        const float now = fmaxf(m, top), keep = now == kNone ? 1.f : exp2_fast(m - now);
        sum *= keep;
        m = now;
        if (j > 0) {
          if (!settle()) { ok = false; break; }
#pragma unroll 1
          for (int c = 0; c < DP; c += 16) {   // rare, and the scores hold most registers
            uint32_t o[16];
            tmem_ld16(to + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
            tmem_st16(to + c, o);
          }
          tmem_wait_st();
        }
      }
      const float base = m == kNone ? 0.f : -m;
      F2 sums[2] = {{0.f, 0.f}, {0.f, 0.f}};
      uint32_t y[SHORT ? kStep / 2 : kB / 2];   // packed; all of a row before the first is stored, where registers allow
      auto probabilities = [&](auto all) {
#pragma unroll
        for (int c = 0; c < kB; c += kStep) {
          uint32_t* to_y = SHORT ? y : y + c / 2;
          if (SHORT) {
            read(c, x);
            tmem_wait_ld();
          }
#pragma unroll
          for (int i = 0; i < kStep; i += 2) {
            const F2 z = fma2({__uint_as_float(x[(c + i) % kHeld]), __uint_as_float(x[(c + i + 1) % kHeld])}, {l.c, l.c}, {base, base});
            F2 e = {exp2_fast(z.x), exp2_fast(z.y)};
            if (!all) {
              const uint32_t two = seen.w[c / 32] >> (c % 32 + i);
              e.x = two & 1 ? e.x : 0.f, e.y = two & 2 ? e.y : 0.f;
            }
            sums[i / 2 & 1] = add2(sums[i / 2 & 1], e);
            to_y[i / 2] = pack2<T>(e.x, e.y);
          }
          if constexpr (SHORT) tmem_st8(tp + c / 2, *(const uint32_t(*)[8])y);
        }
      };
      if (whole) probabilities(Yes());
      else probabilities(No());
      sum += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
      if (!settle()) { ok = false; break; }
      if constexpr (!SHORT) {
#pragma unroll
        for (int c = 0; c < kB; c += 32) tmem_st16(tp + c / 2, *(const uint32_t(*)[16])(y + c / 2));
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
#pragma unroll 1
      for (int i = 0; i < F::kPanels; ++i) {
        uint8_t* to_smem = sq + t * F::kTile + i * kPanel + 32 * quad * 128;
#pragma unroll 1
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

// --------------------------------------------------------------------- backward
// What the backward pass wants of every query: the logarithm of its softmax sum to base 2, and its
// row of d_o against its row of o (delta); both negative.  [batch, heads] blocks of kRowWords words
// for each row, rows rounded up to 128: all lse, all delta, then for products (see below) tiles of
// 64 rows, first -lse / c of each row in three parts that add up to it and have 11 bits each, then
// -delta likewise.  The fourth word of such a row meets a zero in the product and is used otherwise:
// in the first tile what dS of this row is multiplied by (2^..), in the second, for the first of the
// rows that a CTA of attention_rows() has, the exponent of the largest of them.  Behind the last row,
// and where a row saw nothing, lse is so large that every probability comes out as zero.
constexpr int kRowWords = 10, kPass = 64;
constexpr float kNever = 1e35f;

// In fp16 probabilities and dS = P (dP - delta) would leave the type's range downwards where rows are
// long or d_o is small: P is 1 / keys on average, and below 2^-25 nothing is left.  Both are therefore
// held times powers of two that the results' scale takes out again.  P, which is 1 at most, times
// 2^kUpP: all its bits down to 2^-24, and room for the 2^6 that scores near 2^26 may be off by, whose 32
// bits no longer hold the digits behind the point; what is beyond stops at the largest number.  dS times 2^(1 - m), with m the exponent of |d_o|: of the query's own row for dq, of the
// largest row for dk, whose sum runs over the queries.  It is less than 2 |v| then (P (1 - P) is 1/4
// at most, and |dP - dP'| at most 2 |d_o| |v|), which fits for |v| up to 32752.  Bfloat16 has the
// exponents of 32 bits and needs none of this.
template <typename T>
constexpr bool kNarrow = std::is_same<T, __half>::value;
template <typename T>
constexpr int kUpP = kNarrow<T> ? 10 : 0;
template <typename T>
__device__ __forceinline__ uint32_t pack_p(float x, float y) {   // probabilities
  if constexpr (kNarrow<T>) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
  } else {
    return pack2<T>(x, y);
  }
}
constexpr int kNoRow = -1000;   // exponent of a row of zeros, or of one that is not finite
// m from the sum of a row's squares
__device__ __forceinline__ int row_exponent(float squares) {
  const uint32_t bits = __float_as_uint(squares);
  return squares > 0.f && bits < 0x7f800000u ? ((int)(bits >> 23) - 127) >> 1 : kNoRow;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // e normal
__device__ __forceinline__ int ds_up(int exponent) { return exponent == kNoRow ? 0 : 1 - exponent; }
__host__ __device__ __forceinline__ int64_t padded(int64_t rows) { return (rows + kB - 1) / kB * kB; }

__device__ __forceinline__ float4 three_parts(float v) {
  auto upper = [](float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); };
  const float hi = upper(v), mid = upper(v - hi), lo = upper(v - hi - mid);
  return make_float4(hi, mid, lo, 0.f);
}

// delta is made from the result as the forward pass rounded it, o in 32 bits being kept by nobody: one
// error for a whole row of dS.  With it fp16 dq and dk of short rows are off by up to 2.3 times what
// a result is that is rounded once.
template <typename T, int LANES>   // that share a row, 16 bytes each
__global__ void __launch_bounds__(256) attention_rows(const __grid_constant__ HpAttention a, float c) {
  const int lane = threadIdx.x % LANES;
  const int64_t i = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES, h = blockIdx.y, b = blockIdx.z;
  const int64_t rows = padded(a.sq);
  dependents_may_start();
  wait_for_kernel_before();   // the CTAs' rows add up to `rows`
  float s = 0.f, lse = -INFINITY, squares = 0.f;
  if (i < a.sq) {
    if (8 * lane < a.dim) {
      float o[8], g[8];
      unpack<T>(*(const uint4*)((const T*)a.o + b * a.o_b + i * a.o_s + h * a.o_h + 8 * lane), o);
      unpack<T>(*(const uint4*)((const T*)a.d_o + b * a.do_b + i * a.do_s + h * a.do_h + 8 * lane), g);
#pragma unroll
      for (int k = 0; k < 8; ++k) s = fmaf(o[k], g[k], s);
      if (kNarrow<T>)
#pragma unroll
        for (int k = 0; k < 8; ++k) squares = fmaf(g[k], g[k], squares);
    }
    if (lane == 0) lse = a.lse[(b * a.heads + h) * a.sq + i] * kLog2e;
  }
#pragma unroll
  for (int k = LANES / 2; k; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
  int up = 0, largest = kNoRow;
  if constexpr (kNarrow<T>) {
    __shared__ int most[8];
#pragma unroll
    for (int k = LANES / 2; k; k >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, k);
    const int e = row_exponent(squares), of_warp = __reduce_max_sync(0xffffffffu, e);
    up = ds_up(e);
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = of_warp;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; ++k) largest = max(largest, most[k]);
  }
  if (lane == 0) {
    float* out = a.delta + (b * a.heads + h) * kRowWords * rows;
    float4* parts = (float4*)(out + 2 * rows) + i / kPass * 2 * kPass + i % kPass;
    const bool none = lse == -INFINITY;
    out[i] = none ? -kNever : (float)up - lse;
    out[rows + i] = -s;
    float4 first = none ? make_float4(-kNever, 0.f, 0.f, 0.f) : three_parts(((float)kUpP<T> - lse) / c), second = three_parts(-s);
    if (kNarrow<T>) first.w = power_of_two(up), second.w = (float)largest;
    parts[0] = first;
    parts[kPass] = second;
  }
}

// Two kinds of CTA, each with a tile of 128 rows that stays and tiles of 64 that pass by:
//   keys     k, v stay; q, d_o pass.  S^T = k q^T, dP^T = v d_o^T; dv += P^T d_o, dk += dS^T q
//   queries  q, d_o stay; k, v pass.  S = q k^T, dP = d_o v^T; dq += dS k
// with P = 2^(c S - lse) and dS = P (dP - delta).  Computing S and dP for each kind costs two
// products of seven more than one kernel that adds its parts of dq up in memory, and saves
// those additions, their 32-bit buffer and their order, which would differ from run to run.
// P and dS go back to tensor memory over S, as the left operands, in the inputs' type: products of 16
// bits run at twice the rate of tf32's, from half the memory.  Two groups of four warps, a row
// to a thread, take the tiles by turns, so that what one waits for (fetch, store, products) goes on
// behind the other's 2^x: with tiles of 128 that both groups shared, 2600 cycles passed for each
// where its products take 1000.  With keys, lse and delta go by the column: read from shared memory,
// a value for each element, they took half of the rows' time (and of the memory that the products
// read).  One more product for each of S and dP adds them: ones, three for each row, by the three
// parts of -lse / c and -delta.  Tensor memory holds S and dP of three tiles, or of two where the
// results of keys with more than 64 dimensions take half of it.
template <int DP>
struct Backward {
  static constexpr int kPanels = DP / 64, kTile = kPanels * (int)kPanel, kPassed = kPanels * kPass * 128;   // bytes
  static constexpr int kStages = DP == 64 ? 8 : 4;   // even: a stage is always the same group's
  // four warps that fetch and issue, eight for the rows; the former give registers to the latter
  static constexpr int kThreads = 128 + 256, kAtStart = 168, kFew = 72, kMany = 216;
  static_assert(kFew + 2 * kMany <= 3 * kAtStart, "more registers than the CTA has");
  static constexpr int kOnes = 2 * kB * 16, kParts = 2 * kPass * 16;   // bytes: [2][128 rows][4], a stage's [2][64][4]
  static constexpr int kSmem = 2 * kTile + kStages * (2 * kPassed + kParts) + 2 * kOnes + 1024 + 1024;
  // columns: tile j's S (later P, dS) at kBuffer times its buffer, dP kPass further on; the results
  static constexpr uint32_t kBuffer = 2 * kPass, kAcc1 = DP == 64 ? 384 : 256, kAcc2 = DP == 64 ? 448 : 384;
};
struct BackwardBars {
  uint64_t stay_full, in_full[8], in_empty[8], mask_full[8], s_full[6], s_free[3], p_full[3], acc_full;
  Seen<kPass> seen[8];
  uint32_t tmem;
  int keys;       // or the largest row's exponent
  Guard guard;
};

// By the whole CTA: the exponent of the largest row of d_o among rows from `first` on, of `heads` heads.
template <int DP>
__device__ __forceinline__ int largest_row(const float* delta, int heads, int64_t first, int64_t rows, int* shared) {
  constexpr int kRows = 256 / (DP / 8);   // of a CTA of attention_rows(), which kPass is a multiple of
  if (threadIdx.x == 0) *shared = kNoRow;
  __syncthreads();
  int e = kNoRow;
  for (int h = 0; h < heads; ++h)
    for (int64_t i = first + (int64_t)threadIdx.x * kRows; i < rows; i += (int64_t)blockDim.x * kRows)
      e = max(e, (int)delta[h * kRowWords * rows + 2 * rows + (i / kPass * 2 * kPass + kPass + i % kPass) * 4 + 3]);
  e = __reduce_max_sync(0xffffffffu, e);
  if ((threadIdx.x & 31) == 0) atomicMax(shared, e);
  __syncthreads();
  return *shared;
}

template <typename T, int DP>
__global__ void __launch_bounds__(384, 1) attention_backward_tiles(const __grid_constant__ Launch l) {
  using F = Backward<DP>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  uint8_t* stay = smem;
  uint8_t* pass = smem + 2 * F::kTile;
  uint8_t* parts = pass + F::kStages * 2 * F::kPassed;   // a stage's -lse / c and -delta
  uint8_t* ones = parts + F::kStages * F::kParts;        // for the former, for the latter
  BackwardBars& bar = *(BackwardBars*)(ones + 2 * F::kOnes);
  const HpAttention& p = l.p;
  const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int nq = (int)((p.sq + kB - 1) / kB), nk = (int)((p.sk + kB - 1) / kB), group = (int)(p.heads / p.kv_heads);
  const int sk = (int)p.sk, shift = (int)(p.sk - p.sq);
  // Of all heads first the tiles with the most to do: under a causal mask the first keys and the
  // last queries, side by side where there are as many of both; else keys first, which with shared
  // heads have more to do.
  const int hk = (int)(p.kv_heads * p.batch), hq = (int)(p.heads * p.batch);
  int id = blockIdx.x, head, tile;
  bool keys;
  if (nq == nk) {
    tile = id / (hk + hq), id %= hk + hq;
    keys = id < hk;
    if (!keys) id -= hk, tile = nq - 1 - tile;
  } else {
    keys = id < nk * hk;
    if (!keys) id -= nk * hk;
    tile = keys ? id / hk : nq - 1 - id / hq;
    id %= keys ? hk : hq;
  }
  const int heads = keys ? (int)p.kv_heads : (int)p.heads, b = id / heads;
  head = id % heads;
  const int r0 = tile * kB;           // first row that stays
  const uint8_t* mask = p.key_mask ? p.key_mask + b * p.mask_b : nullptr;
  const bool masked = mask != nullptr;
  wait_for_kernel_before();
  // tiles that pass: queries from `first` on, of each head of the group in turn; or keys up to the last seen
  int first = 0, count;
  if (keys) {
    if (p.causal) first = max(0, r0 - shift) / kPass;
    count = max(0, (int)((p.sq + kPass - 1) / kPass) - first);
    if (masked && mask_bits<kB>(mask, r0, sk).none()) count = 0;
  } else {
    int see = masked && sk > kPass ? visible_keys(mask, sk, &bar.keys) : sk;
    if (p.causal) see = min(see, max(0, min(r0 + kB, (int)p.sq) + shift));
    count = (see + kPass - 1) / kPass;
  }
  const int n = keys ? count * group : count;
  int up = 0;   // dS is held times 2^up, for keys
  if (kNarrow<T> && keys && n)
    up = ds_up(largest_row<DP>(p.delta + ((int64_t)b * p.heads + head * group) * kRowWords * padded(p.sq), group, (int64_t)first * kPass,
                               padded(p.sq), &bar.keys));
  const int buffers = DP == 64 || !keys ? 3 : 2, turns = buffers == 3 ? 6 : 2;   // a turn is one group's, of one buffer
  if (threadIdx.x == 0) {
    mbar_init(&bar.stay_full, 1);
    for (int i = 0; i < F::kStages; ++i) mbar_init(&bar.in_full[i], 1), mbar_init(&bar.in_empty[i], 1), mbar_init(&bar.mask_full[i], 1);
    for (int i = 0; i < 6; ++i) mbar_init(&bar.s_full[i], 2);
    for (int i = 0; i < 3; ++i) mbar_init(&bar.s_free[i], 1), mbar_init(&bar.p_full[i], 128);
    mbar_init(&bar.acc_full, 3);
    mbar_init_fence();
    bar.guard.gave_up = 0;
    bar.guard.status = l.status;
  }
  if (warp == 1) tmem_alloc<1>(&bar.tmem, 512);
  if (keys)   // [which][four k][row]: three ones where the parts are that it adds
    for (int i = threadIdx.x; i < 4 * kB; i += blockDim.x) {
      const float one = i / (2 * kB) == i / kB % 2 ? 1.f : 0.f;
      ((float4*)ones)[i] = make_float4(one, one, one, 0.f);
    }
  fence_async_shared();
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  dependents_may_start();
  const uint32_t tmem = uniform(bar.tmem);
  Guard& g = bar.guard;

  if (warp < 4) {
    fewer_registers<F::kFew>();
    if (warp == 0) {
      const uint32_t bytes = 2 * F::kPassed + (keys ? F::kParts : 0);
      const int64_t rows = padded(p.sq);
      int waits = 0;
      if (lane == 0 && n) {
        mbar_expect_tx(&bar.stay_full, 2 * F::kTile);
        for (int i = 0; i < F::kPanels; ++i) {
          tma_load_4d(stay + i * kPanel, keys ? &l.map.k : &l.map.q, 64 * i, head, r0, b, &bar.stay_full);
          tma_load_4d(stay + F::kTile + i * kPanel, keys ? &l.map.v : &l.map.d_o, 64 * i, head, r0, b, &bar.stay_full);
        }
      }
      int s = 0, h = keys ? head * group : head / group, at = first;
      uint32_t ph = 0;
      for (int j = 0; j < n; ++j) {
        if (!guard_wait(&bar.in_empty[s], ph ^ 1, g, 0x11001)) break;
        if (lane == 0) {
          uint8_t* to = pass + s * 2 * F::kPassed;
          mbar_expect_tx(&bar.in_full[s], bytes);
          for (int i = 0; i < F::kPanels; ++i) {
            tma_load_4d(to + i * kPass * 128, keys ? &l.map.q64 : &l.map.k64, 64 * i, h, at * kPass, b, &bar.in_full[s]);
            tma_load_4d(to + F::kPassed + i * kPass * 128, keys ? &l.map.do64 : &l.map.v64, 64 * i, h, at * kPass, b, &bar.in_full[s]);
          }
          if (keys)
            bulk_load(parts + s * F::kParts, p.delta + (b * p.heads + h) * kRowWords * rows + 2 * rows + at * (F::kParts / 4), F::kParts,
                      &bar.in_full[s]);
        }
        if (!keys && masked) {
          const Seen<kPass> m = mask_bits<kPass>(mask, (int64_t)j * kPass, sk);
          if (lane == 0) bar.seen[s] = m, mbar_arrive(&bar.mask_full[s]);
        }
        waits = j + 1;
        if (++at == first + count) at = first, ++h;   // the next head of the group
        if (++s == F::kStages) s = 0, ph ^= 1;
      }
      __syncwarp();
      if (g.gave_up && lane == 0 && n) {   // nothing may land once the CTA is gone
        mbar_wait_bounded(&bar.stay_full, 0, kWaitNs, g.status, HP_STATUS_TIMEOUT | 0x11002);
        for (int j = max(0, waits - F::kStages); j < waits; ++j)
          mbar_wait_bounded(&bar.in_full[j % F::kStages], (j / F::kStages) & 1, kWaitNs, g.status, HP_STATUS_TIMEOUT | 0x11003);
      }
    } else {
      // one warp issues S, one dP, one the results: each product takes as long to issue as to run, and more
      if (n) {
        const uint32_t leader = elect_one();
        const bool bf = p.type == HP_BF16;
        const uint32_t id_s = mma_idesc(128, kPass, bf, true, true) | (l.negative ? kNegateA : 0);
        const uint32_t id_dp = mma_idesc(128, kPass, bf, true, true), id_acc = mma_idesc(128, DP, bf, true, false);
        auto in = [&](int s) { return smem_u32(pass + s * 2 * F::kPassed); };
        auto wide = [&](uint32_t d, uint32_t x, uint32_t y, uint32_t id) {   // rows by rows, over the dimensions
          const uint64_t dx = mma_desc(x, 16, 1024), dy = mma_desc(y, 16, 1024);
#pragma unroll
          for (int i = 0; i < DP / 16; ++i)
            mma_ss<1>(leader, d, dx + ((i / 4) * kPanel + (i % 4) * 32) / 16, dy + ((i / 4) * kPass * 128 + (i % 4) * 32) / 16, id, i > 0);
        };
        auto deep = [&](uint32_t d, uint32_t x, uint32_t y, bool add) {      // P or dS, over the tile's columns
          const uint64_t dy = mma_desc(y, kPass * 128, 1024);
#pragma unroll
          for (int i = 0; i < kPass / 16; ++i) mma_ts(leader, d, x + i * 8, dy + i * 128, id_acc, add || i > 0);
        };
        int s = 0, q = 0, turn = 0;
        uint32_t ph = 0, round = 0;   // of the stages, of the buffers
        bool ok = true;
        if (warp != 2) {
          const bool of_dp = warp == 3;
          const uint32_t a = smem_u32(stay) + (of_dp ? F::kTile : 0), id_w = of_dp ? id_dp : id_s;
          ok = warp_wait(&bar.stay_full, 0, g, 0x21002);
          for (int j = 0; j < n && ok; ++j) {
            ok = warp_wait(&bar.in_full[s], ph, g, 0x21001) && warp_wait(&bar.s_free[q], round ^ 1, g, 0x21005);
            if (!ok) break;
            tmem_fence_after();
            const uint32_t d = tmem + F::kBuffer * q + (of_dp ? kPass : 0);
            wide(d, a, in(s) + (of_dp ? F::kPassed : 0), id_w);
            if (keys)
              mma_tf32(leader, d, mma_desc_plain(smem_u32(ones) + (of_dp ? F::kOnes : 0), kB * 16, 128),
                       mma_desc_plain(smem_u32(parts + s * F::kParts), kPass * 16, 128), mma_idesc_tf32(128, kPass), true);
            mma_commit<1>(leader, &bar.s_full[turn]);
            if (++s == F::kStages) s = 0, ph ^= 1;
            if (++q == buffers) q = 0, round ^= 1;
            if (++turn == turns) turn = 0;
          }
        } else {
          for (int j = 0; j < n; ++j) {
            if (!warp_wait(&bar.p_full[q], round, g, 0x21003)) break;
            tmem_fence_after();
            const uint32_t x = tmem + F::kBuffer * q;
            if (keys) deep(tmem + F::kAcc1, x, in(s) + F::kPassed, j > 0);
            deep(tmem + F::kAcc2, x + kPass / 2, in(s), j > 0);
            mma_commit<1>(leader, &bar.s_free[q]);
            mma_commit<1>(leader, &bar.in_empty[s]);   // S and dP of this tile are behind p_full
            if (++s == F::kStages) s = 0;
            if (++q == buffers) q = 0, round ^= 1;
          }
        }
        mma_commit<1>(leader, &bar.acc_full);
      }
    }
  } else {
    more_registers<F::kMany>();
    const int quad = warp & 3, half = (warp - 4) >> 2, r = 32 * quad + lane, row = r0 + r;
    const uint32_t lanes = (uint32_t)(32 * quad) << 16;
    float lse = 0.f, delta = 0.f;   // of a query that stays, negative
    float ds_scale = kNarrow<T> ? power_of_two(keys ? up : 0) : 1.f;   // what dS is held times: a query's own
    const float of_p = kNarrow<T> ? power_of_two(up - kUpP<T>) : 1.f;  // the same of keys where P is held times 2^kUpP
    bool mine = true;               // a key that stays is seen at all
    if (keys) {
      mine = row < sk && (!masked || mask[row]);
    } else {
      const float* from = p.delta + (b * p.heads + head) * kRowWords * padded(p.sq) + row;
      lse = from[0], delta = from[padded(p.sq)];
      if (kNarrow<T>) ds_scale = (from - row)[2 * padded(p.sq) + (row / kPass * 2 * kPass + row % kPass) * 4 + 3];
    }
    const int sees = p.causal ? min(sk, row + shift + 1) : sk;
    bool ok = true;
    // of tile j: stage, buffer, turn, and place among its head's tiles
    int s = half, q = half, turn = half, place = half;
    uint32_t ph = 0, round = 0;
    auto advance = [&] {
      s += 2, q += 2, turn += 2, place += 2;
      if (s >= F::kStages) s -= F::kStages, ph ^= 1;
      if (q >= buffers) q -= buffers;
      if (turn >= turns) turn -= turns, round ^= 1;
      while (place >= count) place -= count;
    };
    if (n && place >= count) place -= count;   // a head of one tile
    for (int j = half; j < n; j += 2, advance()) {
      Seen<kPass> seen;
      bool whole;
      if (keys) {
        const int from = p.causal ? row - shift - (first + place) * kPass : 0;   // its first query in this tile
        whole = mine && from <= 0;
        if (!__all_sync(0xffffffffu, whole)) {
          seen = seen_between<kPass>(mine ? from : kPass, kPass);
          whole = false;
        }
      } else {
        whole = sees >= (j + 1) * kPass;
        if (masked) {
          if (!guard_wait(&bar.mask_full[s], ph, g, 0x31001)) { ok = false; break; }
          seen = bar.seen[s];
          const bool all = seen.all();
          if (!all) {   // what a masked key holds is left out of dq: its k counts as zero
            if (!guard_wait(&bar.in_full[s], ph, g, 0x31002)) { ok = false; break; }
            if (r < kPass && !(seen.w[quad & 1] >> lane & 1)) {
              uint4* k = (uint4*)(pass + s * 2 * F::kPassed + r * 128);
#pragma unroll
              for (int i = 0; i < F::kPanels; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) k[i * kPass * 8 + e] = make_uint4(0, 0, 0, 0);
            }
            fence_async_shared();
          }
          whole = whole && all;
        }
        if (!__all_sync(0xffffffffu, whole)) {
          const Seen<kPass> up_to = seen_between<kPass>(0, sees - j * kPass);
#pragma unroll
          for (int i = 0; i < kPass / 32; ++i) seen.w[i] = masked ? seen.w[i] & up_to.w[i] : up_to.w[i];
          whole = false;
        }
      }
      if (!guard_wait(&bar.s_full[turn], round, g, 0x31003)) { ok = false; break; }
      tmem_fence_after();
      const uint32_t at = tmem + lanes + F::kBuffer * q;
      uint32_t x[kPass], y[kPass];
#pragma unroll
      for (int c = 0; c < kPass; c += 32) {
        tmem_ld32(at + c, *(uint32_t(*)[32])(x + c));
        tmem_ld32(at + kPass + c, *(uint32_t(*)[32])(y + c));
      }
      tmem_wait_ld();
      auto gradients = [&](auto all, auto of_keys) {   // packed P into x, dS into y
#pragma unroll
        for (int i = 0; i < kPass; i += 2) {
          const F2 v = {__uint_as_float(x[i]), __uint_as_float(x[i + 1])}, u = {__uint_as_float(y[i]), __uint_as_float(y[i + 1])};
          const F2 z = of_keys ? mul2(v, {l.c, l.c}) : fma2(v, {l.c, l.c}, {lse, lse});
          F2 pr = {exp2_fast(z.x), exp2_fast(z.y)};
          F2 ds = mul2(kNarrow<T> && of_keys ? mul2(pr, {of_p, of_p}) : pr, of_keys ? u : add2(u, {delta, delta}));
          if (!all) {
            const uint32_t two = seen.w[i / 32] >> (i % 32);
            if (!(two & 1)) pr.x = ds.x = 0.f;
            if (!(two & 2)) pr.y = ds.y = 0.f;
          }
          if (of_keys) x[i / 2] = pack_p<T>(pr.x, pr.y);
          y[i / 2] = pack2<T>(ds.x, ds.y);
        }
      };
      if (keys) {
        if (whole) gradients(Yes(), Yes());
        else gradients(No(), Yes());
#pragma unroll
        for (int c = 0; c < kPass / 2; c += 16) tmem_st16(at + c, *(const uint32_t(*)[16])(x + c));
      } else {
        if (whole) gradients(Yes(), No());
        else gradients(No(), No());
      }
#pragma unroll
      for (int c = 0; c < kPass / 2; c += 16) tmem_st16(at + kPass / 2 + c, *(const uint32_t(*)[16])(y + c));
      tmem_wait_st();
      tmem_fence_before();
      mbar_arrive(&bar.p_full[q]);
    }
    if (ok && n) ok = guard_wait(&bar.acc_full, 0, g, 0x31006);
    tmem_fence_after();
    // results leave through the space of what stayed: panels of 64 columns, by turns of the two groups
    const int64_t length = keys ? p.sk : p.sq;
    if (ok && r0 < length)
      for (int job = half; job < (keys ? 2 : 1) * F::kPanels; job += 2) {
        const bool is_v = keys && job < F::kPanels;   // dv first, then dk; or dq alone
        const int panel = job % F::kPanels;
        const uint32_t from = tmem + lanes + (is_v ? F::kAcc1 : F::kAcc2) + 64 * panel;
        const float scale = is_v ? 1.f / (float)(1 << kUpP<T>) : (float)p.scale / ds_scale;
        uint8_t* to = stay + job * kPanel + 32 * quad * 128;
#pragma unroll 1
        for (int c = 0; c < 64; c += 32) {
          uint32_t o[32];
          if (n) {
            tmem_ld32(from + c, o);
            tmem_wait_ld();
          }
          float v[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] = n ? __uint_as_float(o[k]) * scale : 0.f;
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            *(uint4*)(to + staged(lane, 2 * (c + k))) =
                make_uint4(pack2<T>(v[k], v[k + 1]), pack2<T>(v[k + 2], v[k + 3]), pack2<T>(v[k + 4], v[k + 5]),
                           pack2<T>(v[k + 6], v[k + 7]));
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) {
          tma_store_4d(keys ? (is_v ? &l.map.dv : &l.map.dk) : &l.map.dq, to, 64 * panel, head, r0 + 32 * quad, b);
          tma_store_commit();
        }
      }
    if (lane == 0) tma_store_wait_read<0>();
    tmem_fence_before();
  }
  __syncwarp();
  __syncthreads();
  if (warp == 1 && n) {
    if (lane == 0) {
      g.gave_up = 0;
      guard_wait(&bar.acc_full, 0, g, 0x60002);
    }
    __syncwarp();
  }
  tmem_fence_after();
  if (warp == 1) tmem_free<1>(tmem, 512);
}

// Up to 128 queries and keys of up to 64 dimensions: everything of one head in one CTA, S and dP once,
// and nothing left for another kernel.  Rows are keys: S^T and dP^T as above; P^T goes back to tensor
// memory, dS^T into shared memory, where it is the left operand of dk (along its rows) and of dq
// (across them).  dv and dk take dP's columns, dq those of S.  Two CTAs fit an SM.  Bound: the
// latency of one pass from fetch to store, not the traffic.
struct ShortBars {
  uint64_t kq_full, vo_full, s_full, dp_full, rows_full, p_full, acc_full, out_full;
  float lse[kB], delta[kB];
  uint32_t tmem;
  int largest;    // exponent of the largest row of d_o
  Guard guard;
};
constexpr int kShortSmem = 6 * (int)kPanel + 2048 + 1024;

template <typename T>
__global__ void __launch_bounds__(320, 2) attention_backward_short(const __grid_constant__ Launch l) {
  extern __shared__ uint8_t raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  uint8_t *sk_ = smem, *sq_ = smem + kPanel, *sv_ = smem + 2 * kPanel, *sg_ = smem + 3 * kPanel;
  uint8_t* sds = smem + 4 * kPanel;   // dS^T: two panels of 64 queries; o before that
  ShortBars& bar = *(ShortBars*)(smem + 6 * kPanel);
  const HpAttention& p = l.p;
  const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int h = blockIdx.x % (int)p.heads, b = blockIdx.x / (int)p.heads;
  const int sq = (int)p.sq, sk = (int)p.sk, shift = sk - sq;
  if (threadIdx.x == 0) {
    mbar_init(&bar.kq_full, 1), mbar_init(&bar.vo_full, 1), mbar_init(&bar.s_full, 1), mbar_init(&bar.dp_full, 1);
    mbar_init(&bar.rows_full, 128), mbar_init(&bar.p_full, 256), mbar_init(&bar.acc_full, 1), mbar_init(&bar.out_full, 256);
    mbar_init_fence();
    bar.guard.gave_up = 0;
    bar.guard.status = l.status;
    bar.largest = kNoRow;
    wait_for_kernel_before();
    mbar_expect_tx(&bar.kq_full, 2 * kPanel);
    tma_load_4d(sk_, &l.map.k, 0, h, 0, b, &bar.kq_full);
    tma_load_4d(sq_, &l.map.q, 0, h, 0, b, &bar.kq_full);
    mbar_expect_tx(&bar.vo_full, 3 * kPanel);
    tma_load_4d(sv_, &l.map.v, 0, h, 0, b, &bar.vo_full);
    tma_load_4d(sg_, &l.map.d_o, 0, h, 0, b, &bar.vo_full);
    tma_load_4d(sds, &l.map.o, 0, h, 0, b, &bar.vo_full);
  }
  if (warp == 1) tmem_alloc<1>(&bar.tmem, 256);
  wait_for_kernel_before();
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  dependents_may_start();
  const uint32_t tmem = uniform(bar.tmem);
  Guard& g = bar.guard;
  if (warp == 1) {
    const uint32_t leader = elect_one();
    const bool bf = p.type == HP_BF16;
    const uint32_t id_s = mma_idesc(128, 128, bf, true, true), id = mma_idesc(128, 64, bf, true, false);
    auto desc = [&](uint8_t* x) { return mma_desc(smem_u32(x), kPanel, 1024); };
    bool ok = warp_wait(&bar.kq_full, 0, g, 0x22001);
    if (ok) {
#pragma unroll
      for (int i = 0; i < 4; ++i) mma_ss<1>(leader, tmem, desc(sk_) + i * 2, desc(sq_) + i * 2, id_s | (l.negative ? kNegateA : 0), i > 0);
      mma_commit<1>(leader, &bar.s_full);
      ok = warp_wait(&bar.vo_full, 0, g, 0x22002);
    }
    if (ok) {
#pragma unroll
      for (int i = 0; i < 4; ++i) mma_ss<1>(leader, tmem + 128, desc(sv_) + i * 2, desc(sg_) + i * 2, id_s, i > 0);
      mma_commit<1>(leader, &bar.dp_full);
      ok = warp_wait(&bar.p_full, 0, g, 0x22003);
      tmem_fence_after();
    }
    if (ok) {
#pragma unroll
      for (int i = 0; i < 8; ++i) mma_ts(leader, tmem + 128, tmem + (i / 2) * 32 + (i % 2) * 8, desc(sg_) + i * 128, id, i > 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) mma_ss<1>(leader, tmem + 192, desc(sds) + (i / 4) * (kPanel / 16) + (i % 4) * 2, desc(sq_) + i * 128, id, i > 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) mma_ss<1>(leader, tmem, desc(sds) + i * 128, desc(sk_) + i * 128, mma_idesc(128, 64, bf, false, false), i > 0);
    }
    mma_commit<1>(leader, &bar.acc_full);
  } else if (warp >= 2) {
    const int quad = warp & 3, half = (warp - 2) >> 2, r = 32 * quad + lane;   // a key, half of the queries
    const uint32_t lanes = (uint32_t)(32 * quad) << 16;
    const bool there = r < sk, mine = there && (!p.key_mask || p.key_mask[b * p.mask_b + r]);
    bool ok = true;
    if (half == 0) {   // lse and delta, negative, of query r
      const float lse = r < sq ? p.lse[(b * p.heads + h) * p.sq + r] : -INFINITY;
      ok = guard_wait(&bar.vo_full, 0, g, 0x32001);
      float d = 0.f, squares = 0.f;
#pragma unroll
      for (int c = 0; c < 128; c += 16) {
        float x[8], y[8];
        unpack<T>(*(const uint4*)(sg_ + staged(r, c)), x);
        unpack<T>(*(const uint4*)(sds + staged(r, c)), y);
#pragma unroll
        for (int i = 0; i < 8; ++i) d = fmaf(x[i], y[i], d);
        if (kNarrow<T>)
#pragma unroll
          for (int i = 0; i < 8; ++i) squares = fmaf(x[i], x[i], squares);
      }
      bar.lse[r] = lse == -INFINITY ? -INFINITY : (float)kUpP<T> - lse * kLog2e;
      bar.delta[r] = -d;
      if (kNarrow<T>) {
        const int e = __reduce_max_sync(0xffffffffu, row_exponent(squares));
        if (lane == 0) atomicMax(&bar.largest, e);
      }
      mbar_arrive(&bar.rows_full);
    }
    const int from = p.causal ? r - shift : 0;   // the first query that sees this key
    bool whole = mine && from <= 0;
    Seen<kB> seen;
    if (!__all_sync(0xffffffffu, whole)) {
      seen = seen_between<kB>(mine ? from : kB, kB);
      whole = false;
    }
    ok = ok && guard_wait(&bar.rows_full, 0, g, 0x32002) && guard_wait(&bar.s_full, 0, g, 0x32003) &&
         guard_wait(&bar.dp_full, 0, g, 0x32004);
    tmem_fence_after();
    // one factor for all of dS, which dk and dq are both made from
    const int up = kNarrow<T> && ok ? ds_up(bar.largest) : 0;
    const float of_p = power_of_two(up - kUpP<T>);
    if (ok) {
      if (there && !mine && half == 0)   // what a masked key holds is left out of dq: it counts as zero
#pragma unroll
        for (int c = 0; c < 8; ++c) *((uint4*)(sk_ + r * 128) + c) = make_uint4(0, 0, 0, 0);
      auto gradients = [&](auto all) {
#pragma unroll 1
        for (int c = 64 * half; c < 64 * half + 64; c += 32) {
          const uint32_t bits_of = all ? 0xffffffffu : c < 64 ? (c < 32 ? seen.w[0] : seen.w[1]) : (c < 96 ? seen.w[2] : seen.w[3]);
          uint32_t x[32], y[32];
          tmem_ld32(tmem + lanes + c, x);
          tmem_ld32(tmem + lanes + 128 + c, y);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 ls = *(const float4*)(bar.lse + c + i), de = *(const float4*)(bar.delta + c + i);
            const float lv[4] = {ls.x, ls.y, ls.z, ls.w}, dv[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
              const F2 z = fma2({__uint_as_float(x[i + k]), __uint_as_float(x[i + k + 1])}, {l.c, l.c}, {lv[k], lv[k + 1]});
              F2 pr = {exp2_fast(z.x), exp2_fast(z.y)};
              F2 ds = mul2(kNarrow<T> ? mul2(pr, {of_p, of_p}) : pr, add2({__uint_as_float(y[i + k]), __uint_as_float(y[i + k + 1])}, {dv[k], dv[k + 1]}));
              if (!all) {
                const uint32_t two = bits_of >> (i + k);
                if (!(two & 1)) pr.x = ds.x = 0.f;
                if (!(two & 2)) pr.y = ds.y = 0.f;
              }
              x[(i + k) / 2] = pack_p<T>(pr.x, pr.y);
              y[(i + k) / 2] = pack2<T>(ds.x, ds.y);
            }
          }
          tmem_st16(tmem + lanes + c, *(const uint32_t(*)[16])x);
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *(uint4*)(sds + half * kPanel + staged(r, 2 * (c % 64) + 4 * i)) = make_uint4(y[i], y[i + 1], y[i + 2], y[i + 3]);
        }
      };
      if (whole) gradients(Yes());
      else gradients(No());
      tmem_wait_st();
      fence_async_shared();
      tmem_fence_before();
      mbar_arrive(&bar.p_full);
      ok = guard_wait(&bar.acc_full, 0, g, 0x32005);
      tmem_fence_after();
    }
    // dv (first group) or dk, and half of dq's columns; through the space of v, q and d_o
    auto emit = [&](uint32_t from_col, float scale, uint8_t* to, int col) {
      uint32_t o[32];
      tmem_ld32(tmem + lanes + from_col, o);
      tmem_wait_ld();
#pragma unroll
      for (int k = 0; k < 32; k += 8) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[e] = pack2<T>(__uint_as_float(o[k + 2 * e]) * scale, __uint_as_float(o[k + 2 * e + 1]) * scale);
        *(uint4*)(to + staged(r, 2 * (col + k))) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    };
    if (ok) {
      const float scale = (float)p.scale * power_of_two(-up);
      uint8_t* to = half ? sq_ : sv_;
#pragma unroll 1
      for (int c = 0; c < 64; c += 32) emit(128 + 64 * half + c, half ? scale : 1.f / (float)(1 << kUpP<T>), to, c);
      emit(32 * half, scale, sg_, 32 * half);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) {
        tma_store_4d(half ? &l.map.dk : &l.map.dv, to + 32 * quad * 128, 0, h, 32 * quad, b);
        tma_store_commit();
      }
    }
    mbar_arrive(&bar.out_full);
    if (ok && half == 0 && guard_wait(&bar.out_full, 0, g, 0x32006) && lane == 0) {
      tma_store_4d(&l.map.dq, sg_ + 32 * quad * 128, 0, h, 32 * quad, b);
      tma_store_commit();
    }
    if (lane == 0) tma_store_wait_read<0>();
    tmem_fence_before();
  }
  __syncwarp();
  __syncthreads();
  if (warp == 1) {
    if (lane == 0) {
      if (g.gave_up) {   // nothing may land, and no product run, once the CTA is gone
        mbar_wait_bounded(&bar.kq_full, 0, kWaitNs, g.status, HP_STATUS_TIMEOUT | 0x12001);
        mbar_wait_bounded(&bar.vo_full, 0, kWaitNs, g.status, HP_STATUS_TIMEOUT | 0x12002);
      }
      g.gave_up = 0;
      guard_wait(&bar.acc_full, 0, g, 0x60003);
    }
    __syncwarp();
  }
  tmem_fence_after();
  if (warp == 1) tmem_free<1>(tmem, 256);
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
  // Without any scale every score counts as much: a small one does the same, and can be divided by.
  l.c = (float)(a.scale < 0 ? -a.scale : a.scale) * kLog2e;
  if (l.c < 1e-20f) l.c = 1e-20f;
  l.negative = a.scale < 0;
  return rc;
}

template <typename T, int DP, int QT, bool SHORT = false>
int forward_tiles(Launch& l, cudaStream_t s) {
  using F = Forward<DP, QT, SHORT>;
  const auto kernel = attention_forward_tiles<T, DP, QT, SHORT>;
  static PerDevice allowed;
  if (const int rc = allow_shared_memory(allowed, kernel, F::kSmem)) return rc;
  const HpAttention& a = l.p;
  if (!head_map(&l.map.q, a.q, a, a.sq, a.heads, a.q_b, a.q_s, a.q_h, kB) ||
      !head_map(&l.map.k, a.sk ? a.k : a.q, a, a.sk, a.kv_heads, a.k_b, a.k_s, a.k_h, kB) ||
      !head_map(&l.map.v, a.sk ? a.v : a.q, a, a.sk, a.kv_heads, a.v_b, a.v_s, a.v_h, kB) ||
      !head_map(&l.map.o, a.o, a, a.sq, a.heads, a.o_b, a.o_s, a.o_h, 32))
    return HP_ERR_BAD_ARG;
  if (a.heads * a.batch > INT32_MAX) return HP_ERR_TOO_LARGE;
  const dim3 grid((unsigned)(a.heads * a.batch), (unsigned)((a.sq + kB * QT - 1) / (kB * QT)));
  if (grid.y > 65535) return HP_ERR_TOO_LARGE;
  return launch_behind(kernel, grid, F::kThreads, F::kSmem, s, l);
}

template <typename T>
int forward(const HpAttention& a, cudaStream_t s) {
  Launch l;
  if (const int rc = prepare(l, a)) return rc;
  if (a.dim <= 64)
    return a.sq <= kB && a.sk <= kB ? forward_tiles<T, 64, 1, true>(l, s) : forward_tiles<T, 64, 1>(l, s);
  // Two tiles of queries in a CTA pay once there are more tiles than SMs, and twice as many where the
  // mask makes them uneven.  One tile a CTA against two, in us, bfloat16, 148 SMs:
  //   1 x 1024, 8 heads: 20 to 26           1 x 2048, 16 heads, causal: 38 to 43
  //   1 x 2048, 12 heads: 66 to 46          1 x 2048, 24 heads, causal: 57 to 44
  const int64_t tiles = (a.sq + kB - 1) / kB * a.heads * a.batch;
  const bool two = a.sq > kB && tiles > (a.causal ? 2 : 1) * layer_sms();
  return two ? forward_tiles<T, 128, 2>(l, s) : forward_tiles<T, 128, 1>(l, s);
}

template <typename T>
int backward_short(const Launch& l, cudaStream_t s) {
  const auto kernel = attention_backward_short<T>;
  static PerDevice allowed;
  if (const int rc = allow_shared_memory(allowed, kernel, kShortSmem)) return rc;
  if (l.p.heads * l.p.batch > INT32_MAX) return HP_ERR_TOO_LARGE;
  return launch_behind(kernel, (unsigned)(l.p.heads * l.p.batch), 320, kShortSmem, s, l);
}

template <typename T, int DP>
int backward_tiles(const Launch& l, cudaStream_t s) {
  using F = Backward<DP>;
  static PerDevice allowed;
  if (const int rc = allow_shared_memory(allowed, attention_backward_tiles<T, DP>, F::kSmem)) return rc;
  const HpAttention& a = l.p;
  const int64_t nq = (a.sq + kB - 1) / kB, nk = (a.sk + kB - 1) / kB, tiles = (nk * a.kv_heads + nq * a.heads) * a.batch;
  if (tiles > INT32_MAX) return HP_ERR_TOO_LARGE;
  if (a.sq) {
    constexpr int kLanes = DP / 8;
    if (const int rc = launch_behind(attention_rows<T, kLanes>, dim3((unsigned)(padded(a.sq) / (256 / kLanes)), (unsigned)a.heads, (unsigned)a.batch),
                                     256, 0, s, a, l.c))
      return rc;
  }
  return launch_behind(attention_backward_tiles<T, DP>, (unsigned)tiles, F::kThreads, F::kSmem, s, l);
}

template <typename T>
int backward(const HpAttention& a, cudaStream_t s) {
  if (!a.sq && !a.sk) return 0;
  Launch l;
  if (const int rc = prepare(l, a)) return rc;
  const void* some = a.sq ? a.q : a.k;   // an address for tensors without elements, of which nothing is read
  auto map = [&](CUtensorMap* m, const void* base, bool key, int64_t sb, int64_t ss, int64_t sh, uint32_t rows) {
    const int64_t length = key ? a.sk : a.sq;
    return head_map(m, length ? base : some, a, length, key ? a.kv_heads : a.heads, sb, ss, sh, rows);
  };
  if (!map(&l.map.q, a.q, false, a.q_b, a.q_s, a.q_h, kB) || !map(&l.map.k, a.k, true, a.k_b, a.k_s, a.k_h, kB) ||
      !map(&l.map.v, a.v, true, a.v_b, a.v_s, a.v_h, kB) || !map(&l.map.d_o, a.d_o, false, a.do_b, a.do_s, a.do_h, kB) ||
      !map(&l.map.dq, a.dq, false, a.dq_b, a.dq_s, a.dq_h, 32) || !map(&l.map.dk, a.dk, true, a.dk_b, a.dk_s, a.dk_h, 32) ||
      !map(&l.map.dv, a.dv, true, a.dv_b, a.dv_s, a.dv_h, 32) ||
      !map(&l.map.o, a.o, false, a.o_b, a.o_s, a.o_h, kB) ||
      !map(&l.map.q64, a.q, false, a.q_b, a.q_s, a.q_h, kPass) || !map(&l.map.k64, a.k, true, a.k_b, a.k_s, a.k_h, kPass) ||
      !map(&l.map.v64, a.v, true, a.v_b, a.v_s, a.v_h, kPass) || !map(&l.map.do64, a.d_o, false, a.do_b, a.do_s, a.do_h, kPass))
    return HP_ERR_BAD_ARG;
  if (a.dim <= 64 && a.sq <= kB && a.sk <= kB && a.heads == a.kv_heads && a.sq && a.sk) return backward_short<T>(l, s);
  return a.dim <= 64 ? backward_tiles<T, 64>(l, s) : backward_tiles<T, 128>(l, s);
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
