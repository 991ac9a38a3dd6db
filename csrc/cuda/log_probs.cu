// Log probabilities of one token in each row of logits, the entropy of the row and its likeliest tokens,
// in one pass over the logits; the gradient in a second one.
//
// A thread keeps the largest logit so far m, the sum s of exp(x - m) and the sum e of z 2^z, with z = (x - m)
// log2(e): then log p = x - m - log s, and the entropy is log s - ln 2 e / s; a large m has cancelled in both
// already, and logits at the type's lowest value stay apart from -inf.  Bound: the traffic; 2^z takes 16 a
// cycle and SM, which is as long as 16-bit logits take to arrive.  A thread fetches its own pieces ahead into
// shared memory (cp.async), so that what is in flight costs no registers and no barrier.
//
// The likeliest tokens need no second pass.  The k-th largest of the maxima of 32 groups of threads is no larger
// than the k-th largest value, so what is smaller than it is none of the k.  It is taken from batches 0, 1, 2, 4,
// 8 .. of pieces, and pieces that hold what is not smaller, a few dozen as a rule, go to a list.  In the end their
// values are looked at once more, and those that count put in order.  Values are compared together with their
// place, so that of equals the first counts and a row of equal values does not flood the list; should it
// overflow, or a value be no number, the row is read again once for each of the k.
#include "activation.cuh"
#include "tcgen05.cuh"

namespace hipress {
namespace {

constexpr int kBatch = 4, kMostTop = 32;   // pieces of 16 bytes that a thread takes at a time
constexpr int kLong = 128;                 // threads of a long row
constexpr float kLn2 = 0.6931471805599453f;
// Rows of G = 32 threads: CTAs of eight, which go from row to row
template <int G>
constexpr int kCta = G == 32 ? 256 : G;
template <int G>
constexpr int kPerSm = G == 32 ? 3 : 8;    // CTAs to an SM
template <int G>
constexpr int kAhead = 2;    // batches of a thread in shared memory

// Values and their places in one order: larger values first, then lower places.  Zero: nothing.
__device__ __forceinline__ uint64_t key_of(float v, int col) {
  const uint32_t u = v != v ? 0x7fc00000u : __float_as_uint(v + 0.f);   // -0 is 0, a NaN the largest of all
  return (uint64_t)(u ^ ((int)u < 0 ? 0xffffffffu : 0x80000000u)) << 32 | ~(uint32_t)col;
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u ^ ((int)u < 0 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int place_of(uint64_t key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }

// The sums over some of a row's values.
struct Sums {
  float m, s, e;
  __device__ __forceinline__ void raise(float to) {   // the largest value
    const float d = fmaxf(m - to, -1e4f) * kLog2e, f = exp2_fast(d);   // of -inf the sums are zero, or NaN
    e = f * fmaf(d, s, e), s *= f, m = to;
  }
};
__device__ __forceinline__ Sums joined(Sums x, Sums y) {
  const float m = fmaxf(x.m, y.m);
  x.raise(m), y.raise(m);
  return {m, x.s + y.s, x.e + y.e};
}
__device__ __forceinline__ Sums of_warp(Sums v) {
  float m = v.m;
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  v.raise(m);
#pragma unroll
  for (int o = 16; o; o >>= 1) v.s += __shfl_xor_sync(0xffffffffu, v.s, o), v.e += __shfl_xor_sync(0xffffffffu, v.e, o);
  return v;
}

template <typename T>
__device__ __forceinline__ uint32_t none16() {
  if constexpr (sizeof(T) == 2) return pack2<T>(-INFINITY, -INFINITY);
  else return 0;
}

// One row (or part of it) in pieces of 16 bytes, cut at their boundaries; what is outside reads as -inf.
template <typename T>
struct Row {
  static constexpr int V = kPiece<T>;
  const T* x;
  int vocab, phase, pieces;
  __device__ __forceinline__ Row(const void* logits, int row, int64_t inner, int64_t ld_outer, int64_t ld, int64_t cols) {
    x = (const T*)logits;
    if (row < inner) {
      x += row * ld;
    } else {
      const uint32_t o = (uint32_t)row / (uint32_t)inner;
      x += o * ld_outer + (row - o * inner) * ld;
    }
    vocab = (int)cols;
    phase = (int)((uintptr_t)x / sizeof(T) % V);
    pieces = (vocab + phase + V - 1) / V;
  }
  __device__ __forceinline__ bool whole(int p, int end) const {
    const int col = p * V - phase;
    return p < end && col >= 0 && col + V <= vocab;
  }
  static __device__ __forceinline__ uint4 nothing() {
    const uint32_t none = sizeof(T) == 4 ? 0xff800000u : none16<T>();
    return make_uint4(none, none, none, none);
  }
  // the first or the last piece, one element at a time
  static __device__ __noinline__ uint4 end_piece(const T* x, int col, int vocab) {
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = col + j >= 0 && col + j < vocab ? to_f(x[col + j]) : -INFINITY;
    return pack<T>(v);
  }
  __device__ __forceinline__ uint4 piece(int p, int end) const {
    const int col = p * V - phase;
    return p >= end ? nothing() : whole(p, end) ? *(const uint4*)(x + col) : end_piece(x, col, vocab);
  }
  // N pieces, `step` apart, into shared memory some time, `stride` apart; none from `end` on.  What a piece holds
  // outside the row comes with it, where that is the logits' memory (`span` bytes from `base` on).
  template <int N>
  __device__ __forceinline__ void fetch(uint4* to, int stride, int p, int step, int end, const void* base, int64_t span) const {
    const int col = p * V - phase;
    if (col >= 0 && col + ((N - 1) * step + 1) * V <= vocab && p + (N - 1) * step < end) {
      const uint4* from = (const uint4*)(x + col);
#pragma unroll
      for (int i = 0; i < N; ++i) copy_ahead(to + i * stride, from + i * step);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = col + i * step * V;
        if (p + i * step >= end) break;
        const int64_t at = (const uint8_t*)(x + c) - (const uint8_t*)base;
        if (at >= 0 && at + 16 <= span) copy_ahead(to + i * stride, x + c);
        else to[i * stride] = end_piece(x, c, vocab);
      }
    }
  }
  static __device__ __forceinline__ void copy_ahead(uint4* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
  }
  // a piece with -inf in place of what lies in front of the row, or from column `limit` on
  __device__ __forceinline__ uint4 inside(uint4 raw, int p, int limit) const {
    const int col = p * V - phase;
    if (col >= 0 && col + V <= limit) return raw;
    uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      auto in = [&](int j) { return col + j >= 0 && col + j < limit; };
      if constexpr (sizeof(T) == 4) {
        w[i] = in(i) ? w[i] : 0xff800000u;
      } else {
        const uint32_t none = none16<T>();
        w[i] = (in(2 * i) ? w[i] & 0xffffu : none & 0xffffu) | (in(2 * i + 1) ? w[i] & 0xffff0000u : none & 0xffff0000u);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// The largest of a piece; a NaN is none
template <typename T>
__device__ __forceinline__ float highest(uint4 v);
template <>
__device__ __forceinline__ float highest<float>(uint4 v) {
  return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
}
template <typename T2>
__device__ __forceinline__ T2 highest2(uint4 v) {
  return __hmax2(__hmax2(*(T2*)&v.x, *(T2*)&v.y), __hmax2(*(T2*)&v.z, *(T2*)&v.w));
}
template <>
__device__ __forceinline__ float highest<__nv_bfloat16>(uint4 v) {
  const float2 f = __bfloat1622float2(highest2<__nv_bfloat162>(v));
  return fmaxf(f.x, f.y);
}
template <>
__device__ __forceinline__ float highest<__half>(uint4 v) {
  const float2 f = __half22float2(highest2<__half2>(v));
  return fmaxf(f.x, f.y);
}
// Where z 2^z is wanted: no z is infinite, and one whose 2^z is zero may be any other such.  NaN stays.
__device__ __forceinline__ float finite(float z) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(z), "f"(-1e4f));
  return y;
}

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return n;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(n));
  return n;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// the address of the first CTA's `p`
__device__ __forceinline__ uint32_t first_cta(const void* p) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_u32(p)));
  return at;
}
__device__ __forceinline__ void store_there(uint32_t at, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}
__device__ __forceinline__ void store_there(uint32_t at, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}

constexpr int kMostSplit = 8;   // CTAs that share a row

// What G threads that share a row keep of its largest values.
template <int G>
struct Largest {
  static constexpr int kGroups = 32, kList = G == 32 ? 256 : 1024, kKeys = G == 32 ? 256 : 512;
  alignas(16) uint64_t group[kGroups];
  uint64_t least, best[kMostTop], found[G / 32], keys[kKeys];
  int list[kList], n, left;   // pieces; of what they hold
};

template <int G>
__device__ __forceinline__ void group_sync() {
  if (G == 32) __syncwarp();
  else __syncthreads();
}

// The k-th largest of the groups' maxima; `t` in the row's threads
template <int G>
__device__ __forceinline__ uint64_t least_of(Largest<G>& l, uint64_t best, int k, int t) {
  constexpr int kShare = G / Largest<G>::kGroups, kEach = Largest<G>::kGroups / kShare;   // threads to a group, keys to each
#pragma unroll
  for (int o = 1; o < kShare; o *= 2) best = larger(best, __shfl_xor_sync(0xffffffffu, best, o));
  const int g = t / kShare, part = t % kShare;
  if (part == 0) l.group[g] = best;
  group_sync<G>();
  int above = 0;
#pragma unroll 8
  for (int i = 0; i < kEach; i += 2) {
    const ulonglong2 g2 = *(const ulonglong2*)(l.group + part * kEach + i);
    above += (int)(g2.x > best) + (int)(g2.y > best);
  }
#pragma unroll
  for (int o = 1; o < kShare; o *= 2) above += __shfl_xor_sync(0xffffffffu, above, o);
  if (above == k - 1 && part == 0) l.least = best;   // one group's, or all those that have none
  group_sync<G>();
  return l.least;
}

// `n` keys into the k largest of them, in order; zeros where there are fewer
template <int G>
__device__ __forceinline__ void in_order(const uint64_t* keys, int n, uint64_t* best, int k, int t) {
  if (t < k) best[t] = 0;
  group_sync<G>();
  for (int i = t; i < n; i += G) {
    const uint64_t mine = keys[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += keys[j] > mine;
    if (mine && above < k) best[above] = mine;
  }
  group_sync<G>();
}

template <typename T, int G, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(kCta<G>, kPerSm<G>) log_probs_kernel(const __grid_constant__ HpLogProbs a) {
  constexpr int V = kPiece<T>, kThreads = kCta<G>, kRows = kThreads / G;
  extern __shared__ uint4 fetched[];   // [kAhead][kBatch][threads]
  __shared__ Sums part[G / 32], parts[kMostSplit];
  __shared__ uint64_t others[TOP && G != 32 ? kMostSplit * kMostTop : 1];
  __shared__ Largest<G> largest[TOP ? kRows : 1];
  __shared__ float losses[kRows][2];
  const int t = threadIdx.x % G, lane = threadIdx.x & 31, k = (int)a.top;
  const int split = G == 32 ? 1 : (int)cluster_size(), rank = split > 1 ? (int)cluster_rank() : 0;
  const int64_t start = G == 32 ? (int64_t)blockIdx.x * kRows + threadIdx.x / G : blockIdx.x / split, step = (int64_t)gridDim.x * kRows;
  Largest<G>& l = largest[TOP ? threadIdx.x / G : 0];
  dependents_may_start();
  if (split > 1) cluster_arrive();   // whose shared memory is written has started
  wait_for_kernel_before();
  auto row_at = [&](int64_t row) { return Row<T>(a.logits, (int)row, a.inner, a.ld_outer, a.ld, a.vocab); };
  float loss = 0.f, count = 0.f;
  int64_t token = start < a.rows ? a.tokens[start] : a.ignored;

  // what is fetched: batch after batch of a row's pieces from `from` to `to`, then of the next row's
  Row<T> ahead = row_at(start < a.rows ? start : 0);
  const int each = (ahead.pieces + split - 1) / split, first = rank * each;
  // rows of which nothing is wanted are left out where a CTA has one row
  const bool read = start < a.rows && (G == 32 || ENTROPY || TOP || token != a.ignored);
  int64_t row_ahead = start;
  int from = first, to = read ? min(first + each, ahead.pieces) : 0;
  uint4* into = fetched + threadIdx.x;
  const int64_t last_outer = (a.rows - 1) / a.inner, last_inner = (a.rows < a.inner ? a.rows : a.inner) - 1,
                span = (last_outer * a.ld_outer + last_inner * a.ld + a.vocab) * (int64_t)sizeof(T);
  auto next_slot = [&](uint4* slot) {
    slot += kBatch * kThreads;
    return slot == fetched + threadIdx.x + kAhead<G> * kBatch * kThreads ? fetched + threadIdx.x : slot;
  };
  auto fetch = [&] {
    if (from < to) ahead.template fetch<kBatch>(into, kThreads, from + t, G, to, a.logits, span);
    asm volatile("cp.async.commit_group;" ::: "memory");
    into = next_slot(into);
    from += G * kBatch;
    if (G == 32 && from >= to && row_ahead < a.rows) {
      row_ahead += step;
      if (row_ahead < a.rows) ahead = row_at(row_ahead), from = 0, to = ahead.pieces;
    }
  };
  Row<T> r = ahead;
  int end = to;
#pragma unroll
  for (int i = 0; i < kAhead<G>; ++i) fetch();
  uint4* slot = fetched + threadIdx.x;

  for (int64_t row = start; G != 32 || row < a.rows; row += step) {
    const bool there = G == 32 || row < a.rows;
    if (G == 32 && row != start) r = row_at(row), end = r.pieces;
    int64_t token_after = a.ignored;
    if (G == 32 && row + step < a.rows) token_after = a.tokens[row + step];
    const bool inside = token != a.ignored && token >= 0 && token < r.vocab;
    const float at_token = t == 0 && inside ? to_f(r.x[token]) : 0.f;   // on its way while the row is read
    if (TOP) {
      if (t == 0) l.n = l.left = 0, l.least = 0;
      group_sync<G>();
    }
    Sums sum = {-INFINITY, 0.f, 0.f};
    uint64_t best = 0, least = 0;
    float high = -INFINITY, bar = -INFINITY;   // the thread's largest value; that of `least`
    int turn = 0;
    for (int p = first, batch = 0; p < end; p += G * kBatch, ++batch) {   // the same for all threads of a row
      uint4 raw[kBatch];
      float top[kBatch];
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead<G> - 1) : "memory");
#pragma unroll
      for (int i = 0; i < kBatch; ++i) raw[i] = slot[i * kThreads];
      slot = next_slot(slot);
      // the row's ends: pieces that lie across them, and pieces that are not there
      const int limit = min(r.vocab, end * V - r.phase);
      const bool edge = (p == 0 && r.phase) || (p + G * kBatch) * V - r.phase > limit;
      if (edge)
#pragma unroll
        for (int i = 0; i < kBatch; ++i) raw[i] = r.inside(raw[i], p + t + i * G, limit);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) top[i] = highest<T>(raw[i]);
      const float now = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      // the sums bear values that are larger by a few powers of two: raised is seldom more than once
      if (now > sum.m + 8.f || sum.m == -INFINITY) sum.raise(fmaxf(now, sum.m));
      if (TOP) {
        if (batch == 0 && p + t < end) {   // the first of the places that hold the largest value
          int at = max((p + t) * V - r.phase, 0);
#pragma unroll
          for (int i = kBatch - 1; i >= 0; --i)
            if (top[i] == now && now != -INFINITY) {
              float v[V];
              unpack<T>(raw[i], v);
#pragma unroll
              for (int j = V - 1; j >= 0; --j)
                if (v[j] == now) at = (p + t + i * G) * V - r.phase + j;
            }
          best = key_of(now, at);
          high = now;
        }
        high = fmaxf(high, now);
      }
      fetch();   // where this thread alone has read, and has what it read
      const float minus = sum.m == -INFINITY ? 0.f : -sum.m;
      F2 s, e;
      auto add_up = [&](auto infinite) {
        s = e = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          if (infinite && p + i * G >= end) break;   // of no thread's
          float v[V];
          unpack<T>(raw[i], v);
#pragma unroll
          for (int j = 0; j < V; j += 2) {
            F2 z = mul2(add2({v[j], v[j + 1]}, {minus, minus}), {kLog2e, kLog2e});
            if (infinite) z = {finite(z.x), finite(z.y)};
            const F2 x = {exp2_fast(z.x), exp2_fast(z.y)};
            s = add2(s, x);
            if (ENTROPY) e = fma2(x, z, e);
          }
        }
      };
      if (edge) {
        add_up(Yes());
      } else {
        add_up(No());
        if (ENTROPY && !(e.x + e.y > -INFINITY)) add_up(Yes());   // zero times an infinity, or a NaN of the logits'
      }
      sum.s += s.x + s.y, sum.e += e.x + e.y;
      if (TOP) {
        if (batch == turn) {   // batches 0, 1, 2, 4, 8 ..
          turn = turn ? 2 * turn : 1;
          if (high > value_of(best) || !best) best = high == -INFINITY ? best : key_of(high, -1);   // wherever it is
          least = least_of<G>(l, best, k, t);
          bar = least ? value_of(least) : -INFINITY;
        }
        if (now >= bar) {
          const uint32_t place = ~(uint32_t)least;   // of equal values the first count; all, where no place is known
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const int q = p + t + i * G;
            if (q < end && (top[i] > bar || (top[i] == bar && (uint32_t)max(q * V - r.phase, 0) <= place))) {
              const int at = atomicAdd(&l.n, 1);
              if (at < Largest<G>::kList) l.list[at] = q;
            }
          }
        }
      }
    }
    // a NaN is no maximum and in no list, but in the sum
    sum = of_warp(sum);
    if (G != 32) {
      if (lane == 0) part[threadIdx.x / 32] = sum;
      __syncthreads();
      if (TOP || threadIdx.x < 32) {
        sum = part[lane % (G / 32)];
        float m = sum.m;
#pragma unroll
        for (int o = G / 64; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        sum.raise(m);
#pragma unroll
        for (int o = G / 64; o; o >>= 1)
          sum.s += __shfl_xor_sync(0xffffffffu, sum.s, o), sum.e += __shfl_xor_sync(0xffffffffu, sum.e, o);
      }
    }
    if (TOP) {
      group_sync<G>();
      const int n = l.n;
      bool listed = n <= Largest<G>::kList && sum.s == sum.s;
      if (listed) {
        if (n > 16) {   // the first ones were let in by lower bars
          if (high > value_of(best)) best = key_of(high, -1);
          least = least_of<G>(l, best, k, t);
        }
        for (int i = t; i < n; i += G) {
          const int q = l.list[i];
          float v[V];
          unpack<T>(r.piece(q, end), v);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int col = q * V - r.phase + j;
            const uint64_t key = key_of(v[j], col);
            if (key >= least && col >= 0 && col < r.vocab) {
              const int at = atomicAdd(&l.left, 1);
              if (at < Largest<G>::kKeys) l.keys[at] = key;
            }
          }
        }
        group_sync<G>();
        listed = l.left <= Largest<G>::kKeys;
      }
      if (listed) {
        in_order<G>(l.keys, l.left, l.best, k, t);
      } else {
        uint64_t last = ~0ull;
        for (int i = 0; i < k; ++i) {
          uint64_t next = 0;
          for (int p = first + t; p < end; p += G) {
            float v[V];
            unpack<T>(r.piece(p, end), v);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const int col = p * V - r.phase + j;
              const uint64_t key = key_of(v[j], col);
              if (col >= 0 && col < r.vocab && key < last) next = larger(next, key);
            }
          }
#pragma unroll
          for (int o = 16; o; o >>= 1) next = larger(next, __shfl_xor_sync(0xffffffffu, next, o));
          group_sync<G>();
          if (lane == 0) l.found[t / 32] = next;
          group_sync<G>();
          for (int w = 0; w < G / 32; ++w) next = larger(next, l.found[w]);
          if (t == 0) l.best[i] = next;
          last = next;
        }
        group_sync<G>();
      }
    }
    if (split > 1) {
      cluster_wait();
      if (threadIdx.x == 0) {
        const uint32_t to = first_cta(&parts[rank]);
        store_there(to, sum.m), store_there(to + 4, sum.s), store_there(to + 8, sum.e);
      }
      if (TOP && G != 32 && t < k) store_there(first_cta(&others[rank * k + t]), l.best[t]);
      cluster_arrive();
      cluster_wait();
      if (rank) return;
      sum = parts[0];
      for (int i = 1; i < split; ++i) sum = joined(sum, parts[i]);
      if (TOP && G != 32) in_order<G>(others, split * k, l.best, k, t);
    }
    const bool none = sum.s == 0.f;   // nothing above -inf
    const float lns = none ? 0.f : logf(sum.s);
    auto log_p = [&](float v) { return none ? -INFINITY : (v - sum.m) - lns; };
    float lp = 0.f;
    if (t == 0 && there) {
      if (token != a.ignored) lp = inside ? log_p(at_token) : NAN;
      if (a.log_probs) a.log_probs[row] = lp;
      *(float2*)(a.stats + 2 * row) = make_float2(sum.m, lns);
      if (ENTROPY) a.entropy[row] = none ? 0.f : fmaf(-kLn2, sum.e / sum.s, lns);
      if (token != a.ignored) loss -= lp, count += 1.f;
    }
    if (TOP && there && t < k) {
      a.top_log_probs[row * k + t] = log_p(value_of(l.best[t]));
      a.top_tokens[row * k + t] = place_of(l.best[t]);
    }
    if (G != 32) break;
    token = token_after;
  }
  if (a.loss) {
    if (t == 0) losses[threadIdx.x / G][0] = loss, losses[threadIdx.x / G][1] = count;
    __syncthreads();
    if (threadIdx.x < 2) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < kRows; ++i) s += losses[i][threadIdx.x];
      ((float*)a.workspace)[2 * (int64_t)(blockIdx.x / split) + threadIdx.x] = s;
    }
  }
}

// The parts' losses and rows, added in their order by one CTA, in 64 bits; their mean or sum.
__global__ void __launch_bounds__(1024) loss_kernel(const float2* parts, int64_t n, float* loss, float* count, int summed) {
  __shared__ double sums[2][32];
  dependents_may_start();
  wait_for_kernel_before();
  double s = 0., c = 0.;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < n; i += 1024) {
    const float2 v = parts[i];
    s += v.x, c += v.y;
  }
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), c += __shfl_xor_sync(0xffffffffu, c, o);
    if (pass) break;
    if ((threadIdx.x & 31) == 0) sums[0][threadIdx.x / 32] = s, sums[1][threadIdx.x / 32] = c;
    __syncthreads();
    s = sums[0][threadIdx.x & 31], c = sums[1][threadIdx.x & 31];
  }
  if (threadIdx.x == 0) {
    *loss = (float)(summed ? s : s / c);   // of no rows the mean is no number
    *count = (float)c;
  }
}

// dx = g (1 at the token - p) - h p (log p + entropy).  Pieces go by the boundaries of the result; logits that
// lie otherwise are read element by element.  A row's batches are shared by `chunks` CTAs, which fetch one ahead.
template <typename T, int G, bool ENTROPY>
__global__ void __launch_bounds__(256, 4) log_probs_backward_kernel(const __grid_constant__ HpLogProbsBackward a, int chunks) {
  constexpr int V = kPiece<T>, kRows = 256 / G;
  const int t = threadIdx.x % G;
  const int64_t row = (int64_t)(blockIdx.x / chunks) * kRows + threadIdx.x / G;
  const int chunk = blockIdx.x % chunks;
  dependents_may_start();
  wait_for_kernel_before();
  if (row >= a.rows) return;
  const Row<T> in(a.logits, (int)row, a.inner, a.ld_outer, a.ld, a.vocab), out(a.dlogits, (int)row, a.rows, 0, a.vocab, a.vocab);
  const int64_t token = a.tokens[row];
  float g = token == a.ignored || !a.dlog_probs ? 0.f : a.dlog_probs[a.one ? 0 : row];
  if (g != 0.f && a.count) g /= *a.count;
  if (a.negative) g = -g;
  const float h = ENTROPY ? a.dentropy[row] : 0.f, m = a.stats[2 * row], log2s = a.stats[2 * row + 1] * kLog2e;
  if (token != a.ignored && (token < 0 || token >= in.vocab)) g = NAN;
  const bool some = (g != 0.f || h != 0.f) && m != -INFINITY, alike = in.phase == out.phase;
  // p times by + hz z, z = log2 p
  const float hz = h * -kLn2, by = ENTROPY ? fmaf(-h, a.entropy[row], -g) : -g;
  const int mine = g != 0.f && token >= 0 && token < in.vocab ? (int)token : -V;
  T* to = (T*)a.dlogits + row * a.vocab;
  auto take = [&](uint4 (&raw)[kBatch], int p) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int col = (p + i * G + t) * V - out.phase;
      if (!some || col >= out.vocab) {
        raw[i] = make_uint4(0, 0, 0, 0);
      } else if (alike && col >= 0 && col + V <= out.vocab) {
        raw[i] = *(const uint4*)(in.x + col);
      } else {
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = col + j >= 0 && col + j < out.vocab ? to_f(in.x[col + j]) : 0.f;
        raw[i] = pack<T>(v);
      }
    }
  };
  uint4 next[kBatch];
  take(next, chunk * G * kBatch);
  for (int p = chunk * G * kBatch; p < out.pieces; p += chunks * G * kBatch) {
    uint4 raw[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) raw[i] = next[i];
    if (p + chunks * G * kBatch < out.pieces) take(next, p + chunks * G * kBatch);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int col = (p + i * G + t) * V - out.phase;
      if (col >= out.vocab) break;
      float v[V];
      unpack<T>(raw[i], v);
      if (some) {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
          F2 z = fma2(add2({v[j], v[j + 1]}, {-m, -m}), {kLog2e, kLog2e}, {-log2s, -log2s});
          if (ENTROPY) z = {finite(z.x), finite(z.y)};
          const F2 x = mul2({exp2_fast(z.x), exp2_fast(z.y)}, ENTROPY ? fma2(z, {hz, hz}, {by, by}) : F2{by, by});
          v[j] = x.x, v[j + 1] = x.y;
        }
        const int at = mine - col;
        if (at >= 0 && at < V)
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (j == at) v[j] += g;
      }
      if (col >= 0 && col + V <= out.vocab) {
        *(uint4*)(to + col) = pack<T>(v);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (col + j >= 0 && col + j < out.vocab) to[col + j] = from_f<T>(v[j]);
      }
    }
  }
}

// Rows of about this many pieces have a warp each, and longer ones too where there are enough of them.  A warp
// against a CTA, us, 16 bits, forward (backward): 100000 x 1024 92 against 378 (backward), 100000 x 1100 131 against 304, 20000 x
// 5000 with 10 alternatives 103 against 144 (69 against 115), 8192 x 32000 107 against 88.
constexpr int kWarpPieces = 128;

template <typename T, int G, bool ENTROPY, bool TOP>
int forward_of(const HpLogProbs& a, int split, cudaStream_t s) {
  int64_t ctas = a.rows * split;
  if (G == 32) {
    const int64_t most = (int64_t)kPerSm<G> * layer_sms(), all = (a.rows + 7) / 8;
    ctas = all < most ? all : most;
  }
  if (ctas > INT32_MAX) return HP_ERR_TOO_LARGE;
  const int space = kAhead<G> * kBatch * kCta<G> * 16;
  static PerDevice allowed;
  if (const int rc = allow_shared_memory(allowed, log_probs_kernel<T, G, ENTROPY, TOP>, space)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = (unsigned)ctas, cfg.blockDim = kCta<G>, cfg.dynamicSmemBytes = space, cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)split, at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = split > 1 ? 2 : 1;
  if (const int rc = told(cudaLaunchKernelEx(&cfg, log_probs_kernel<T, G, ENTROPY, TOP>, a))) return rc;
  if (!a.loss) return 0;
  return launch_behind(loss_kernel, 1, 1024, 0, s, (const float2*)a.workspace, ctas / split, a.loss, a.count, (int)a.summed);
}

template <typename T>
int64_t most_pieces(int64_t vocab) {
  return (vocab + 2 * kPiece<T> - 2) / kPiece<T>;
}

template <typename T>
int forward(const HpLogProbs& a, cudaStream_t s) {
  const int64_t pieces = most_pieces<T>(a.vocab);
#define BY_USE(G, split)                                                                                       \
  a.entropy ? (a.top ? forward_of<T, G, true, true>(a, split, s) : forward_of<T, G, true, false>(a, split, s)) \
            : (a.top ? forward_of<T, G, false, true>(a, split, s) : forward_of<T, G, false, false>(a, split, s))
  if (pieces <= kWarpPieces + 1 || (pieces <= 8 * kWarpPieces && a.rows >= 16 * kPerSm<32> * layer_sms())) return BY_USE(32, 1);
  // Few rows are shared by up to eight CTAs, as long as each has a batch: until six are on their way for each SM
  // instead of four, 300 x 128000 bf16 takes 22 us instead of 29.
  int split = 1;
  while (split < kMostSplit && a.rows * split < 6 * layer_sms() && pieces > split * kLong * kBatch) split *= 2;
  return BY_USE(kLong, split);
#undef BY_USE
}

template <typename T, int G, bool ENTROPY>
int backward_of(const HpLogProbsBackward& a, cudaStream_t s) {
  // CTAs that a row takes: enough for four to an SM, a batch each at least
  int64_t chunks = 1;
  if (G != 32) {
    const int64_t most = (most_pieces<T>(a.vocab) + G * kBatch - 1) / (G * kBatch), want = (4 * layer_sms() + a.rows - 1) / a.rows;
    chunks = want < most ? want : most;
  }
  const int64_t ctas = G == 32 ? (a.rows + 7) / 8 : a.rows * chunks;
  if (ctas > INT32_MAX) return HP_ERR_TOO_LARGE;
  return launch_behind(log_probs_backward_kernel<T, G, ENTROPY>, (unsigned)ctas, 256, 0, s, a, (int)chunks);
}
template <typename T>
int backward(const HpLogProbsBackward& a, cudaStream_t s) {
  if (most_pieces<T>(a.vocab) <= 2 * kWarpPieces || (most_pieces<T>(a.vocab) <= 16 * kWarpPieces && a.rows >= 32 * layer_sms()))
    return a.dentropy ? backward_of<T, 32, true>(a, s) : backward_of<T, 32, false>(a, s);
  return a.dentropy ? backward_of<T, 256, true>(a, s) : backward_of<T, 256, false>(a, s);
}

bool sizes_ok(int64_t rows, int64_t inner, int64_t vocab, int64_t type) {
  return rows >= 0 && rows <= INT32_MAX && inner >= 1 && vocab >= 1 && vocab <= 1 << 30 && type_ok(type);
}

}  // namespace
}  // namespace hipress

using namespace hipress;

#define BY_TYPE(fn) a->type == HP_F32 ? fn<float>(*a, s) : a->type == HP_BF16 ? fn<__nv_bfloat16>(*a, s) : fn<__half>(*a, s)

extern "C" int hp_cuda_log_probs(const HpLogProbs* a, void* stream) {
  if (!a || !sizes_ok(a->rows, a->inner, a->vocab, a->type) || a->top < 0 || a->top > kMostTop || a->top > a->vocab ||
      (a->loss && (!a->count || (a->rows && !a->workspace))))
    return HP_ERR_BAD_ARG;
  cudaStream_t s = (cudaStream_t)stream;
  if (!a->rows)
    return a->loss ? launch_behind(loss_kernel, 1, 1024, 0, s, (const float2*)nullptr, (int64_t)0, a->loss, a->count, (int)a->summed) : 0;
  return BY_TYPE(forward);
}

extern "C" uint64_t hp_cuda_log_probs_workspace(int64_t rows) { return (uint64_t)rows * 8; }

extern "C" int hp_cuda_log_probs_backward(const HpLogProbsBackward* a, void* stream) {
  if (!a || !sizes_ok(a->rows, a->inner, a->vocab, a->type) || (a->dentropy && !a->entropy) || (uintptr_t)a->dlogits % 16)
    return HP_ERR_BAD_ARG;
  if (!a->rows) return 0;
  cudaStream_t s = (cudaStream_t)stream;
  return BY_TYPE(backward);
}
