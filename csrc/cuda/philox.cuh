// Which elements a dropout keeps, as a function of the seed, the call's number and the element's
// place: nothing is stored, and the backward pass makes the same bits again.
//
// Elements go by words of 32.  Word w has 16 random words, the results of Philox4x32 (Salmon, Moraes, Dror
// and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) for the counters (w, site, 0 .. 3), w in
// two words, under the seed as its key.  Bit i of the j-th of them is bit j of a number u of 16 bits for
// the word's element i, which is kept where u >= 2^16 - t, so with a probability of t / 2^16.  Seven rounds:
// the fewest that pass all of the paper's tests; its ten cost 1.4 times as much.
//
// The 32 comparisons of a word are made at once, a bit of t at a time from the lowest on: where it is set the
// upper bits decide for 1 or leave it as it is, r | m, else for 0, r & m.  Both are the majority of r, m
// and the bit of t, one instruction for 32 elements.  Zeros of t below its lowest one decide nothing: where the
// upper four bits are all there is (p = 1/2, 1/4 ..), only the last call is made.
#pragma once
#include "layers.cuh"

namespace hipress {

struct Drop {
  const int64_t* seed_at;
  int64_t seed;
  uint32_t site, first;    // the first call whose bits of t are not all zero
  uint32_t bit[16];        // bits of t, all ones or zeros
  float up, share;         // 2^16 / t, t / 2^16
};

// false where the numbers are out of range
inline bool drop_of(Drop* d, const HpDropout& a) {
  if (a.keep < 1 || a.keep > 65535 || a.site < 0 || a.site > 0xffffffffll) return false;
  d->seed_at = a.seed_at, d->seed = a.seed, d->site = (uint32_t)a.site;
  d->first = 0;
  while (!(a.keep >> (4 * d->first) & 15)) ++d->first;
  for (int i = 0; i < 16; ++i) d->bit[i] = a.keep >> i & 1 ? 0xffffffffu : 0u;
  d->up = 65536.f / (float)a.keep;
  d->share = (float)a.keep / 65536.f;
  return true;
}

struct Key {
  uint32_t lo, hi;
};
// By a whole warp.  The compiler knows that it is the same in all threads, and keeps the rounds' keys in
// uniform registers: added up in each thread they were an eighth of the instructions of a dropped attention.
__device__ __forceinline__ Key drop_key(const Drop& d) {
  const int64_t s = d.seed_at ? *d.seed_at : d.seed;
  return {__shfl_sync(0xffffffffu, (uint32_t)s, 0), __shfl_sync(0xffffffffu, (uint32_t)(s >> 32), 0)};
}

__device__ __forceinline__ uint4 philox_round(uint4 c, Key k) {
  const uint64_t a = (uint64_t)c.x * 0xD2511F53u, b = (uint64_t)c.z * 0xCD9E8D57u;
  return make_uint4((uint32_t)(b >> 32) ^ c.y ^ k.lo, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ k.hi, (uint32_t)a);
}
// N counters round by round, side by side: one alone is a chain of fourteen instructions, each of which waits
// for the last.
template <int N>
__device__ __forceinline__ void philox(uint4 (&c)[N], Key k) {
#pragma unroll
  for (int i = 0; i < 7; ++i) {
#pragma unroll
    for (int n = 0; n < N; ++n) c[n] = philox_round(c[n], k);
    k.lo += 0x9E3779B9u, k.hi += 0xBB67AE85u;
  }
}

__device__ __forceinline__ uint32_t majority(uint32_t a, uint32_t b, uint32_t c) { return (a & b) | (c & (a | b)); }

__device__ __forceinline__ uint32_t majority4(uint4 r, uint32_t m, const uint32_t* bit) {
  return majority(r.w, majority(r.z, majority(r.y, majority(r.x, m, bit[0]), bit[1]), bit[2]), bit[3]);
}

// The bits of words w: set where an element is kept.
template <int N>
__device__ __forceinline__ void kept_words(const Drop& d, Key k, const uint64_t (&w)[N], uint32_t (&m)[N]) {
  auto counter = [&](int n, uint32_t call) { return make_uint4((uint32_t)w[n], (uint32_t)(w[n] >> 32), d.site, call); };
  if (d.first == 3) {
    uint4 c[N];
#pragma unroll
    for (int n = 0; n < N; ++n) c[n] = counter(n, 3);
    philox(c, k);
#pragma unroll
    for (int n = 0; n < N; ++n) m[n] = majority4(c[n], 0, d.bit + 12);
  } else {
    uint4 c[4 * N];
#pragma unroll
    for (int n = 0; n < 4 * N; ++n) c[n] = counter(n / 4, n % 4);
    philox(c, k);
#pragma unroll
    for (int n = 0; n < N; ++n) m[n] = 0;
#pragma unroll
    for (int n = 0; n < 4 * N; ++n) m[n / 4] = majority4(c[n], m[n / 4], d.bit + 4 * (n % 4));
  }
}
__device__ __forceinline__ uint32_t kept_word(const Drop& d, Key k, uint64_t w) {
  const uint64_t ws[1] = {w};
  uint32_t m[1];
  kept_words<1>(d, k, ws, m);
  return m[0];
}

}  // namespace hipress
