// The matrix product with bias, activation and residual in its epilogue, and what its
// backward pass needs besides two more products.
#include "activation.cuh"
#include "column_sums.cuh"
#include "tcgen05.cuh"

namespace hipress {
namespace {


template <int BYTES>
struct Word;
template <>
struct Word<16> { using type = uint4; };
template <>
struct Word<4> { using type = uint32_t; };
template <>
struct Word<2> { using type = uint16_t; };

// ------------------------------------------------------------------- the product
// A persistent kernel of specialised warps: one thread fetches tiles (TMA), one issues the
// matrix products, others empty the accumulators.  Two accumulators in tensor memory: the
// next tile's products run while the last one's results are written.
//   CG  CTAs that share a tile: 1, or 2 (each holds half of both operands and 128 rows of results)
//   BN  columns of a tile; it has 128 CG rows
constexpr int kBK = 64;            // k of a stage: one line of the swizzle
constexpr int kStaging = 4096;     // a warp's buffer: 32 rows of 128 bytes

template <int CG, int BN>
struct Shape {
  static constexpr int kRowsB = BN / CG;
  static constexpr int kBytesA = 128 * 128, kBytesB = kRowsB * 128, kStage = kBytesA + kBytesB;
  static constexpr int kStages = kStage <= 24576 ? 6 : 4;
  // Warps that empty an accumulator, each 32 rows of 64 columns: with 256 columns sixteen, since two
  // to a scheduler took twice as long over GELU as the products of 1024 k take.  Staging for them:
  // two buffers each, or one where they are sixteen.
  static constexpr int kEpiWarps = BN / 16, kCols = 64, kBuffers = kEpiWarps > 8 ? 1 : 2;
  static constexpr int kThreads = 32 * (2 + kEpiWarps);
  static constexpr int kSmem = kStages * kStage + kEpiWarps * (kBuffers * kStaging + kCols * 4) + 512 + 1024;
  static constexpr int kTmem = 2 * BN;
  // A pair allocates on two SMs.  Two pairs that shared both could each hold what the other waits for on
  // its second SM, so that no SM may have room for two: half of its 228 KB.
  static_assert(CG == 1 || kSmem > 114 * 1024, "two pairs of CTAs fit an SM");
};

struct Launch {
  CUtensorMap a, b, y, pre;  // y: the partial sums where k is split
  HpProduct p;
  int64_t ldp;               // pitch of the partial sums
  int tiles_m, tiles_n, kblocks, splits;
  int vec_y, vec_r;          // bytes of an aligned access to y and pre, to the residual
  uint32_t* status;
};

struct Bars {
  uint64_t full[8], empty[8], acc_full[2], acc_empty[2], drain;
  uint32_t tmem;
  Guard guard;
};

struct Unit {
  int m0, n0, k0, k1, split;
};
// Tiles in groups of 16 rows of tiles, so that those at work together share their operands in L2.
__device__ __forceinline__ Unit unit_of(const Launch& l, int u, int bm, int bn) {
  Unit w;
  w.split = u % l.splits;
  const int t = u / l.splits, group = 16 * l.tiles_n, g = t / group, first = 16 * g;
  const int rows = min(16, l.tiles_m - first), in = t - g * group;
  w.m0 = (first + in % rows) * bm;
  w.n0 = (in / rows) * bn;
  w.k0 = (int)((int64_t)l.kblocks * w.split / l.splits);
  w.k1 = (int)((int64_t)l.kblocks * (w.split + 1) / l.splits);
  return w;
}

// byte `b` of row `r` of a warp's staging rows, as the 128-byte swizzle of a TMA store has it
__device__ __forceinline__ uint32_t staged(int r, int b) { return (uint32_t)(r * 128 + (b ^ ((r & 7) << 4))); }

// A warp's 32 staged rows of 128 bytes to rows that TMA cannot address: V bytes an access.
// Rows below `rows` and bytes below `width` only.
template <int V>
__device__ __forceinline__ void store_rows(const uint8_t* s, uint8_t* g, int64_t pitch, int rows, int width, int lane) {
  using Raw = typename Word<V>::type;
#pragma unroll 1
  for (int r = 0; r < rows; ++r)
#pragma unroll
    for (int b = lane * V; b < 128; b += 32 * V) {
      const uint8_t* at = s + staged(r, b);
      uint8_t* to = g + r * pitch + b;
      if (b + V <= width) *(Raw*)to = *(const Raw*)at;
      else if (V == 4 && b + 2 <= width) *(uint16_t*)to = *(const uint16_t*)at;
    }
}
__device__ __noinline__ void store_ragged(int vec, const uint8_t* s, uint8_t* g, int64_t pitch, int rows, int width, int lane) {
  if (vec >= 4) store_rows<4>(s, g, pitch, rows, width, lane);
  else store_rows<2>(s, g, pitch, rows, width, lane);
}

// Emptied staging rows leave through a tensor map, or by plain stores where y has no 16-byte
// rows.  Two buffers take turns, where there are two.
template <int BUFFERS>
struct Out {
  uint8_t* base;
  int turn;
  __device__ __forceinline__ uint8_t* buffer() const { return base + turn * kStaging; }
  // before the buffer is filled: what was stored from it has been read
  __device__ __forceinline__ void ready(int lane) const {
    if (lane == 0) tma_store_wait_read<BUFFERS - 1>();
    __syncwarp();
  }
  __device__ __forceinline__ void send(const Launch& l, const CUtensorMap& map, void* plain, int64_t pitch, int bytes,
                                       int row0, int col0, int split, int lane) {
    const HpProduct& p = l.p;
    if (l.vec_y == 16) {
      fence_async_shared();
      __syncwarp();
      if (lane == 0) {
        if (row0 < p.m && col0 < p.n) tma_store_3d(&map, buffer(), col0, row0, split);
        tma_store_commit();
      }
    } else {
      __syncwarp();
      const int64_t rows = p.m - row0, width = (p.n - col0) * bytes;
      if (rows > 0 && width > 0)
        store_ragged(l.vec_y, buffer(), (uint8_t*)plain + (row0 * pitch + col0) * bytes, pitch * bytes,
                     rows < 32 ? (int)rows : 32, width < 128 ? (int)width : 128, lane);
      __syncwarp();
    }
    turn = (turn + 1) % BUFFERS;
  }
};

template <int ACT, int N>
__device__ __forceinline__ void activate_all(float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = activate<ACT>(v[i]);
}
template <int N>
__device__ __forceinline__ void activate_all(int act, float (&v)[N]) {
  if (act == HP_ACT_RELU) activate_all<HP_ACT_RELU>(v);
  else if (act == HP_ACT_GELU) activate_all<HP_ACT_GELU>(v);
  else if (act == HP_ACT_GELU_TANH) activate_all<HP_ACT_GELU_TANH>(v);
}

// Sixteen pairs of residuals of one row, zeros where there are none.
template <typename T>
__device__ __forceinline__ void load_residual(const Launch& l, int row, int col, uint32_t (&r)[16]) {
  const HpProduct& p = l.p;
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = 0;
  if (!p.residual || row >= p.m) return;
  const T* from = (const T*)p.residual + row * p.ldr + col;
  if (l.vec_r == 16 && col + 32 <= p.n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 q = *(const uint4*)(from + 8 * i);
      r[4 * i] = q.x, r[4 * i + 1] = q.y, r[4 * i + 2] = q.z, r[4 * i + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t lo = col + 2 * i < p.n ? *(const uint16_t*)(from + 2 * i) : 0;
      const uint32_t hi = col + 2 * i + 1 < p.n ? *(const uint16_t*)(from + 2 * i + 1) : 0;
      r[i] = lo | hi << 16;
    }
  }
}

template <typename T, int CG, int BN>
__global__ void __launch_bounds__(Shape<CG, BN>::kThreads, 1) product_kernel(const __grid_constant__ Launch l) {
  using S = Shape<CG, BN>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  uint8_t* staging = smem + S::kStages * S::kStage;
  float* biases = (float*)(staging + S::kEpiWarps * S::kBuffers * kStaging);   // [kEpiWarps][kCols]
  Bars& bar = *(Bars*)(biases + S::kEpiWarps * S::kCols);
  const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  const HpProduct& p = l.p;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(&bar.full[i], 1), mbar_init(&bar.empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&bar.acc_full[i], 1), mbar_init(&bar.acc_empty[i], CG * S::kEpiWarps);
    mbar_init(&bar.drain, 1);
    mbar_init_fence();
    bar.guard.gave_up = 0;
    bar.guard.status = l.status;
    tma_prefetch(&l.a);
    tma_prefetch(&l.b);
    if (l.vec_y == 16) tma_prefetch(&l.y);
  }
  if (warp == 1) tmem_alloc<CG>(&bar.tmem, S::kTmem);
  tmem_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();   // the other CTA's barriers are there
  tmem_fence_after();
  const uint32_t tmem = uniform(bar.tmem);
  dependents_may_start();
  wait_for_kernel_before();
  Guard& g = bar.guard;
  const int units = l.tiles_m * l.tiles_n * l.splits, step = gridDim.x / CG, first = blockIdx.x / CG;

  if (warp == 0) {
    if (elect_one()) {
      int s = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t full0 = CG == 2 ? cluster_addr(&bar.full[0], 0) : 0;
      for (int u = first; u < units && ok; u += step) {
        const Unit w = unit_of(l, u, 128 * CG, BN);
        const int ma = w.m0 + 128 * (int)rank, nb = w.n0 + S::kRowsB * (int)rank;
        for (int kb = w.k0; kb < w.k1; ++kb) {
          if (!guard_wait(&bar.empty[s], phase ^ 1, g, 0x10000)) {
            ok = false;
            break;
          }
          uint8_t* a = smem + s * S::kStage;
          uint8_t* b = a + S::kBytesA;
          if (rank == 0) mbar_expect_tx(&bar.full[s], CG * S::kStage);
          auto load = [&](uint8_t* to, const CUtensorMap* map, int x, int y) {
            if (CG == 2) tma_load_2d_pair(to, map, x, y, full0 + 8 * s);
            else tma_load_2d(to, map, x, y, &bar.full[s]);
          };
          const int k = kb * kBK;
          if (p.a_kmajor) load(a, &l.a, k, ma);
          else
            for (int i = 0; i < 2; ++i) load(a + 8192 * i, &l.a, ma + 64 * i, k);
          if (p.b_kmajor) load(b, &l.b, k, nb);
          else
            for (int i = 0; i < S::kRowsB / 64; ++i) load(b + 8192 * i, &l.b, nb + 64 * i, k);
          ++issued;
          if (++s == S::kStages) s = 0, phase ^= 1;
        }
      }
      // every copy has landed before the CTA may end (the products wait for them too, unless they gave up)
      if (!ok && rank == 0) {
        g.gave_up = 0;   // these waits are for copies alone
        for (int i = 0; i < S::kStages && i < issued; ++i) {
          const int q = (s + S::kStages - 1 - i) % S::kStages, lap = (issued - 1 - i) / S::kStages;
          guard_wait(&bar.full[q], lap & 1, g, 0x40000);
        }
        g.gave_up = 1;
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t leader = elect_one();
      const uint32_t idesc = mma_idesc(128 * CG, BN, p.type == HP_BF16, p.a_kmajor, p.b_kmajor);
      const uint32_t lead_a = p.a_kmajor ? 16 : 8192, lead_b = p.b_kmajor ? 16 : 8192;
      const uint32_t step_a = p.a_kmajor ? 2 : 128, step_b = p.b_kmajor ? 2 : 128;   // 16 k further on, 16 bytes to a unit
      int s = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = first; u < units && ok; u += step, ++it) {
        const Unit w = unit_of(l, u, 128 * CG, BN);
        const int acc = it & 1;
        if (!warp_wait(&bar.acc_empty[acc], ((it >> 1) & 1) ^ 1, g, 0x20000)) break;
        tmem_fence_after();
        for (int kb = w.k0; kb < w.k1; ++kb) {
          if (!warp_wait(&bar.full[s], phase, g, 0x30000)) {
            ok = false;
            break;
          }
          tmem_fence_after();
          const uint64_t a = mma_desc(smem_u32(smem + s * S::kStage), lead_a, 1024);
          const uint64_t b = mma_desc(smem_u32(smem + s * S::kStage + S::kBytesA), lead_b, 1024);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)
            mma_ss<CG>(leader, tmem + acc * BN, a + k * step_a, b + k * step_b, idesc, kb > w.k0 || k > 0);
          mma_commit<CG>(leader, &bar.empty[s]);
          if (++s == S::kStages) s = 0, phase ^= 1;
        }
        if (ok) mma_commit<CG>(leader, &bar.acc_full[acc]);
      }
      mma_commit<CG>(leader, &bar.drain);
    }
  } else {
    const int e = warp - 2, quad = warp & 3, half = e >> 2;
    const int base = half * S::kCols;          // this warp's columns of a tile
    const bool raw = l.splits > 1 || p.ytype == HP_F32;   // the sums as they are, in 32 bits
    Out<S::kBuffers> out = {staging + e * S::kBuffers * kStaging, 0};
    int it = 0;
    for (int u = first; u < units; u += step, ++it) {
      const Unit w = unit_of(l, u, 128 * CG, BN);
      const int acc = it & 1, row0 = w.m0 + 128 * (int)rank + 32 * quad, col = w.n0 + base;
      const uint32_t from = tmem + acc * BN + base + ((uint32_t)(32 * quad) << 16);
      auto release = [&] {   // the accumulator has been read
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (CG == 2) mbar_arrive_cluster(cluster_addr(&bar.acc_empty[acc], 0));
          else mbar_arrive(&bar.acc_empty[acc]);
        }
      };
      if (raw) {
        if (!guard_wait(&bar.acc_full[acc], (it >> 1) & 1, g, 0x50000)) break;
        tmem_fence_after();
#pragma unroll 1
        for (int c = 0; c < S::kCols; c += 32) {
          uint32_t r[32];
          tmem_ld32(from + c, r);
          out.ready(lane);
          tmem_wait_ld();
          if (c + 32 == S::kCols) release();
          uint8_t* to = out.buffer();
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *(uint4*)(to + staged(lane, 4 * i)) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
          out.send(l, l.y, p.y, p.ldy, 4, row0, col + c, w.split, lane);
        }
        continue;
      }
      // bias and the first residuals come while the products still run
      float* bias = biases + e * S::kCols;
      if (p.bias)
        for (int i = lane; i < S::kCols; i += 32) bias[i] = col + i < p.n ? load_any(p.bias, col + i, (int)p.btype) : 0.f;
      uint32_t next[16];
      load_residual<T>(l, row0 + lane, col, next);
      if (!guard_wait(&bar.acc_full[acc], (it >> 1) & 1, g, 0x50000)) break;
      tmem_fence_after();
      __syncwarp();
#pragma unroll 1
      for (int c = 0; c < S::kCols; c += 64) {
        uint32_t y[32];
#pragma unroll
        for (int h = 0; h < 64; h += 32) {
          uint32_t r[32], res[16];
          tmem_ld32(from + c + h, r);
#pragma unroll
          for (int i = 0; i < 16; ++i) res[i] = next[i];
          if (c + h + 32 < S::kCols) load_residual<T>(l, row0 + lane, col + c + h + 32, next);
          if (h == 0) out.ready(lane);
          tmem_wait_ld();
          if (c + h + 32 == S::kCols) release();
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
          if (p.bias)
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 b = *(const float4*)(bias + c + h + i);
              v[i] += b.x, v[i + 1] += b.y, v[i + 2] += b.z, v[i + 3] += b.w;
            }
          if (p.pre) {
            uint8_t* to = out.buffer();
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              *(uint4*)(to + staged(lane, 2 * (h + i))) =
                  make_uint4(pack2<T>(v[i], v[i + 1]), pack2<T>(v[i + 2], v[i + 3]), pack2<T>(v[i + 4], v[i + 5]),
                             pack2<T>(v[i + 6], v[i + 7]));
          }
          activate_all(p.act, v);
          if (p.residual)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 q = unpack2<T>(res[i]);
              v[2 * i] += q.x, v[2 * i + 1] += q.y;
            }
#pragma unroll
          for (int i = 0; i < 16; ++i) y[h / 2 + i] = pack2<T>(v[2 * i], v[2 * i + 1]);
        }
        if (p.pre) {
          out.send(l, l.pre, p.pre, p.ldy, 2, row0, col + c, 0, lane);
          out.ready(lane);
        }
        uint8_t* to = out.buffer();
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *(uint4*)(to + staged(lane, 4 * i)) = make_uint4(y[i], y[i + 1], y[i + 2], y[i + 3]);
        out.send(l, l.y, p.y, p.ldy, 2, row0, col + c, 0, lane);
      }
    }
    if (lane == 0) tma_store_wait_read<0>();   // before the shared memory goes
  }
  __syncwarp();
  __syncthreads();
  if (warp == 1) {
    if (lane == 0) {   // the products have ended, also those nobody waits for
      g.gave_up = 0;
      guard_wait(&bar.drain, 0, g, 0x60000);
    }
    __syncwarp();
  }
  tmem_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();   // neither CTA's memory goes while the other's products read it
  tmem_fence_after();
  if (warp == 1) tmem_free<CG>(tmem, S::kTmem);
}

// y from the partial sums of the splits (none: of a product without k), added in their order
template <typename T>
__global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ Launch l) {
  const HpProduct& p = l.p;
  const int64_t quads = l.ldp / 4, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  dependents_may_start();
  wait_for_kernel_before();
  if (at >= p.m * quads) return;
  const int64_t m = at / quads, n = at % quads * 4;
  float v[4] = {};
  const float* part = (const float*)p.workspace + m * l.ldp + n;
  for (int s = 0; s < l.splits; ++s) {
    const float4 q = *(const float4*)(part + (int64_t)s * p.m * l.ldp);
    v[0] += q.x, v[1] += q.y, v[2] += q.z, v[3] += q.w;
  }
  const int cols = (int)min((int64_t)4, p.n - n);
  for (int i = 0; i < cols; ++i) {
    if (p.bias) v[i] += load_any(p.bias, n + i, (int)p.btype);
    if (p.pre) ((T*)p.pre)[m * p.ldy + n + i] = from_f<T>(v[i]);
  }
  activate_all(p.act, v);
  for (int i = 0; i < cols; ++i) {
    if (p.residual) v[i] += to_f(((const T*)p.residual)[m * p.ldr + n + i]);
    store_any(p.y, m * p.ldy + n + i, v[i], (int)p.ytype);
  }
}

struct Choice {
  int cg, bn, splits;
};

// Which kernel, and into how many parts k is split: the least of an estimate in SM cycles.  Pairs
// of CTAs with 256 columns are the fastest where there are tiles enough (4096 x 4096 x 1024: 41 us,
// against 43, 45 and 66 with 256 x 128, 128 x 128 and 128 x 64); the small tiles where few would
// leave SMs idle (1024 x 1024 x 4096: 35, 25, 29, 23), and parts of k where even those do (512 x
// 512 x 32768: 128 x 64 alone 116, in four parts 46; in eight with 256 x 128 40).
Choice choose(int64_t m, int64_t n, int64_t kblocks, int sms) {
  const struct {
    int cg, bn;
    double stage;   // cycles of 64 k
  } kinds[] = {{2, 256, 540}, {2, 128, 340}, {1, 128, 350}, {1, 64, 240}};
  Choice best = {1, 128, 1};
  double least = 1e30;
  for (const auto& c : kinds) {
    const int64_t tiles = ((m + 128 * c.cg - 1) / (128 * c.cg)) * ((n + c.bn - 1) / c.bn), slots = sms / c.cg;
    for (int64_t s = 1; s <= 64 && s <= kblocks; s = s < 4 ? s + 1 : s + s / 2) {
      const int64_t rounds = (tiles * s + slots - 1) / slots;
      const int64_t per = (kblocks + s - 1) / s;
      double t = rounds * (per * c.stage + 300.0) + 3000.0 + c.bn * 10.0;
      if (s > 1) t += 4000.0 + (double)m * n * (2 * s) * 4 / 3000.0;   // the partial sums, and one more launch
      if (t < least) least = t, best = {c.cg, c.bn, (int)s};
    }
  }
  return best;
}

int64_t pitch4(int64_t n) { return (n + 3) / 4 * 4; }

template <typename T, int CG, int BN>
int run_product(Launch& l, int sms, cudaStream_t s) {
  using S = Shape<CG, BN>;
  const HpProduct& p = l.p;
  const uint32_t box_k[2] = {kBK, 128}, box_m[2] = {64, kBK};
  const uint32_t box_kb[2] = {kBK, (uint32_t)S::kRowsB};
  auto map = [&](CUtensorMap* t, const void* base, int64_t rows, int64_t ld, bool kmajor, const uint32_t* box) {
    const uint64_t size[2] = {(uint64_t)(kmajor ? p.k : rows), (uint64_t)(kmajor ? rows : p.k)};
    const uint64_t pitch[1] = {size[1] > 1 ? 2 * (uint64_t)ld : 16};   // of one line there is no next
    return tensor_map(t, base, (int)p.type, 2, size, pitch, box);
  };
  if (!map(&l.a, p.a, p.m, p.lda, p.a_kmajor, p.a_kmajor ? box_k : box_m) ||
      !map(&l.b, p.b, p.n, p.ldb, p.b_kmajor, p.b_kmajor ? box_kb : box_m))
    return HP_ERR_BAD_ARG;
  if (l.vec_y == 16) {
    const bool split = l.splits > 1, wide = split || p.ytype == HP_F32;
    const uint64_t e = wide ? 4 : 2, row = e * (uint64_t)(split ? l.ldp : p.ldy);
    const uint64_t size[3] = {(uint64_t)p.n, (uint64_t)p.m, (uint64_t)l.splits};
    const uint64_t pitch[2] = {p.m > 1 ? row : 16, p.m > 1 ? row * (uint64_t)p.m : split ? row : 16};
    const uint32_t box[3] = {(uint32_t)(128 / e), 32, 1};
    if (!tensor_map(&l.y, split ? p.workspace : p.y, wide ? HP_F32 : (int)p.type, 3, size, pitch, box) ||
        (p.pre && !split && !tensor_map(&l.pre, p.pre, (int)p.type, 3, size, pitch, box)))
      return HP_ERR_BAD_ARG;
  }
  static PerDevice allowed;
  if (const int rc = allow_shared_memory(allowed, product_kernel<T, CG, BN>, S::kSmem)) return rc;
  l.tiles_m = (int)((p.m + 128 * CG - 1) / (128 * CG));
  l.tiles_n = (int)((p.n + BN - 1) / BN);
  const int64_t units = (int64_t)l.tiles_m * l.tiles_n * l.splits;
  if (units > INT32_MAX / 2) return HP_ERR_TOO_LARGE;
  const int64_t slots = sms / CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(CG * (units < slots ? units : slots)));
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return told(cudaLaunchKernelEx(&cfg, product_kernel<T, CG, BN>, l));
}

int alignment(const void* p, int64_t pitch_bytes) {
  const uint64_t v = (uint64_t)(uintptr_t)p | (uint64_t)pitch_bytes;
  return v % 16 == 0 ? 16 : v % 4 == 0 ? 4 : 2;
}

template <typename T>
int product(const HpProduct& a, cudaStream_t s) {
  Launch l;
  int rc;
  l.status = layer_status(&rc);
  if (rc) return rc;
  const int sms = layer_sms();
  l.p = a;
  l.ldp = pitch4(a.n);
  l.kblocks = (int)((a.k + kBK - 1) / kBK);
  const int e = a.ytype == HP_F32 ? 4 : 2;
  l.vec_y = alignment(a.y, a.ldy * e);
  if (a.pre && alignment(a.pre, a.ldy * 2) < l.vec_y) l.vec_y = alignment(a.pre, a.ldy * 2);
  l.vec_r = alignment(a.residual, a.ldr * 2);
  l.splits = 0;
  if (a.k) {
    const Choice c = choose(a.m, a.n, l.kblocks, sms);
    l.splits = c.splits;
    if (l.splits > 1) l.vec_y = 16;   // the partial sums' rows
    rc = c.cg == 2 ? (c.bn == 256 ? run_product<T, 2, 256>(l, sms, s) : run_product<T, 2, 128>(l, sms, s))
                   : (c.bn == 128 ? run_product<T, 1, 128>(l, sms, s) : run_product<T, 1, 64>(l, sms, s));
    if (rc) return rc;
    if (l.splits == 1) return 0;
  }
  const int64_t quads = a.m * (l.ldp / 4);
  if (quads > (int64_t)INT32_MAX * 128) return HP_ERR_TOO_LARGE;
  return launch_behind(finish_kernel<T>, (unsigned)((quads + 255) / 256), 256, 0, s, l);
}

// --------------------------------------------------- the gradient before the activation
// g = dy act'(pre) and the sums of its columns, in one pass over dy and pre: traffic bound.  pre is kept
// in 16 bits, half the traffic of both passes, and g rounded to them, since products take no others.  A
// thread has V columns (16 bytes where all rows lie on that boundary, else 4 or 2) and the rows
// of its warp; the CTA's eight warps add up their sums, and leave one row of partial sums.
constexpr int kSlopeWarps = 8;

template <typename T, int ACT, int V>
__global__ void __launch_bounds__(32 * kSlopeWarps) slope_kernel(const __grid_constant__ HpSlope a) {
  using Raw = typename Word<2 * V>::type;
  __shared__ float sums[kSlopeWarps][32 * V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t col = ((int64_t)blockIdx.x * 32 + lane) * V, step = (int64_t)gridDim.y * kSlopeWarps;
  float s[V] = {};
  dependents_may_start();
  wait_for_kernel_before();
  auto put = [&](int64_t row, Raw dy, Raw pre) {
    T* d = (T*)&dy;
    const T* q = (const T*)&pre;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float g = to_f(d[j]);
      if (ACT != HP_ACT_NONE) g *= slope<ACT>(to_f(q[j]));
      s[j] += g;
      d[j] = from_f<T>(g);
    }
    if (a.g) *(Raw*)((T*)a.g + row * a.ldg + col) = dy;
  };
  if (col + V <= a.cols) {
    int64_t row = (int64_t)blockIdx.y * kSlopeWarps + warp;
    const T* dy = (const T*)a.dy + col;
    const T* pre = (const T*)a.pre + col;
    constexpr int kAhead = 4;
    for (; row + (kAhead - 1) * step < a.rows; row += kAhead * step) {
      Raw d[kAhead], q[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        d[i] = *(const Raw*)(dy + (row + i * step) * a.lddy);
        if (ACT != HP_ACT_NONE) q[i] = *(const Raw*)(pre + (row + i * step) * a.ldpre);
        else q[i] = d[i];
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) put(row + i * step, d[i], q[i]);
    }
    for (; row < a.rows; row += step) {
      const Raw d = *(const Raw*)(dy + row * a.lddy);
      put(row, d, ACT != HP_ACT_NONE ? *(const Raw*)(pre + row * a.ldpre) : d);
    }
  } else if (V > 1 && col < a.cols) {   // the row ends inside this thread's columns
    for (int64_t row = (int64_t)blockIdx.y * kSlopeWarps + warp; row < a.rows; row += step)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (col + j < a.cols) {
          float g = to_f(((const T*)a.dy)[row * a.lddy + col + j]);
          if (ACT != HP_ACT_NONE) g *= slope<ACT>(to_f(((const T*)a.pre)[row * a.ldpre + col + j]));
          s[j] += g;
          if (a.g) ((T*)a.g)[row * a.ldg + col + j] = from_f<T>(g);
        }
  }
  if (!a.dbias) return;
#pragma unroll
  for (int j = 0; j < V; ++j) sums[warp][j * 32 + lane] = s[j];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * V; i += 32 * kSlopeWarps) {
    const int64_t c = (int64_t)blockIdx.x * 32 * V + (i % 32) * V + i / 32;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kSlopeWarps; ++w) t += sums[w][i];
    if (c < a.cols) ((float*)a.workspace)[(int64_t)blockIdx.y * a.cols + c] = t;
  }
}

constexpr int kSlopeParts = 256;   // rows of partial sums at most

template <typename T, int ACT, int V>
int slopes(const HpSlope& a, cudaStream_t s) {
  const int64_t wide = (a.cols + 32 * V - 1) / (32 * V);
  // four CTAs to an SM; at least four rows to a warp, so that the sums stay few
  int64_t high = ((int64_t)layer_sms() * 4 + wide - 1) / wide, most = (a.rows + 4 * kSlopeWarps - 1) / (4 * kSlopeWarps);
  if (high > most) high = most;
  if (high > kSlopeParts) high = kSlopeParts;
  if (high < 1) high = 1;
  const int rc = launch_behind(slope_kernel<T, ACT, V>, dim3((unsigned)wide, (unsigned)high), 32 * kSlopeWarps, 0, s, a);
  if (rc || !a.dbias) return rc;
  return column_sums((const float*)a.workspace, (int)high, a.cols, a.cols, a.dbias, nullptr, (int)a.btype, s);
}
template <typename T, int ACT>
int slopes(const HpSlope& a, cudaStream_t s) {
  int v = alignment(a.dy, 2 * a.lddy);
  if (ACT != HP_ACT_NONE && alignment(a.pre, 2 * a.ldpre) < v) v = alignment(a.pre, 2 * a.ldpre);
  if (a.g && alignment(a.g, 2 * a.ldg) < v) v = alignment(a.g, 2 * a.ldg);
  return v == 16 ? slopes<T, ACT, 8>(a, s) : v == 4 ? slopes<T, ACT, 2>(a, s) : slopes<T, ACT, 1>(a, s);
}
template <typename T>
int slopes(const HpSlope& a, cudaStream_t s) {
  switch (a.act) {
    case HP_ACT_NONE: return slopes<T, HP_ACT_NONE>(a, s);
    case HP_ACT_RELU: return slopes<T, HP_ACT_RELU>(a, s);
    case HP_ACT_GELU: return slopes<T, HP_ACT_GELU>(a, s);
    default: return slopes<T, HP_ACT_GELU_TANH>(a, s);
  }
}

}  // namespace
}  // namespace hipress

using namespace hipress;

extern "C" int hp_cuda_product(const HpProduct* a, void* stream) {
  if (!a || a->m < 0 || a->n < 0 || a->k < 0 || a->m > INT32_MAX / 2 || a->n > INT32_MAX / 2 || a->k > INT32_MAX / 2 ||
      (a->type != HP_BF16 && a->type != HP_F16) || (a->ytype != a->type && a->ytype != HP_F32) || !type_ok(a->btype) ||
      a->act < 0 || a->act > HP_ACT_GELU_TANH ||
      (a->ytype == HP_F32 && (a->bias || a->act || a->residual || a->pre)))
    return HP_ERR_BAD_ARG;
  if (!a->m || !a->n) return 0;
  cudaStream_t s = (cudaStream_t)stream;
  return a->type == HP_BF16 ? product<__nv_bfloat16>(*a, s) : product<__half>(*a, s);
}

extern "C" uint64_t hp_cuda_product_workspace(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const Choice c = choose(m, n, (k + kBK - 1) / kBK, layer_sms());
  return c.splits > 1 ? (uint64_t)c.splits * m * pitch4(n) * 4 : 0;
}

extern "C" int hp_cuda_slope(const HpSlope* a, void* stream) {
  if (!a || a->rows < 0 || a->cols < 0 || (a->type != HP_BF16 && a->type != HP_F16) || !type_ok(a->btype) ||
      a->act < 0 || a->act > HP_ACT_GELU_TANH || (a->rows && a->cols && a->act && !a->pre))
    return HP_ERR_BAD_ARG;
  if (!a->cols) return 0;
  cudaStream_t s = (cudaStream_t)stream;
  return a->type == HP_BF16 ? slopes<__nv_bfloat16>(*a, s) : slopes<__half>(*a, s);
}

extern "C" uint64_t hp_cuda_slope_workspace(int64_t, int64_t cols) { return (uint64_t)kSlopeParts * cols * 4; }
