// Layer norm, forward and backward.
//
// No operand is used twice outside its row, so the bound is the traffic: x (residual) in, y (z)
// out; z and dy (dz) in, dx out.  A row is read once and stays in registers, in 32 bits, for its
// mean, the sum of its squared deviations and the result.
#include "column_sums.cuh"
#include "tcgen05.cuh"

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
  const float rstd = rsqrtf(cta_sum(s, part) / (float)a.cols + (float)a.eps);
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

// ------------------------------------------------------------- rows through shared memory
// NW warps share a row, each thread CH pieces of 16 bytes of it.  Whole rows are fetched ahead by
// bulk copies into a ring of `depth` slots, so that what is in flight does not cost registers;
// a thread keeps its columns from row to row, and with them the weights and (backward) the sums
// of the weights' gradients.  With plain loads into registers the forward pass of 65536 x 1024
// bf16 took 69 to 86 us, however many rows were loaded ahead.
//
// Rows whose first element is not on a 16-byte boundary (RAGGED) are cut at the boundaries all
// the same: the pieces start `phase` elements ahead of the row, and what is outside the row is
// cleared.  The phase goes by the row modulo the elements of a piece, and the rows of one group
// of warps are a multiple of eight apart, so that its columns stay the same.  The first and the
// last row have no neighbour to be read along with them: their ends are loaded element by element.
template <typename T, bool RAGGED>
struct Piece {
  static constexpr int V = kPiece<T>, kBits = 8 * sizeof(T);
  int first;   // column of its first element
  __device__ __forceinline__ bool whole(int cols) const {
    return RAGGED ? first >= 0 && first + V <= cols : first < cols;
  }
  __device__ __forceinline__ bool has(int j, int cols) const {
    return RAGGED ? first + j >= 0 && first + j < cols : first < cols;
  }
  // from a slot whose first 16 bytes hold the row's first element; zeros outside the row
  __device__ __forceinline__ uint4 take(const uint8_t* slot, int cols, int phase) const {
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (first >= cols) return raw;
    raw = *(const uint4*)(slot + (first + phase) * (int)sizeof(T));
    if (RAGGED && !whole(cols)) {
      // a row is at least a piece long: it either begins or ends in this one
      const int cut = kBits * (first < 0 ? -first : V + first - cols);   // bits to clear, 0 < cut < 128
      const uint64_t all = ~(uint64_t)0;
      uint64_t lo = raw.x | (uint64_t)raw.y << 32, hi = raw.z | (uint64_t)raw.w << 32;
      if (first < 0) {
        lo &= cut < 64 ? all << cut : 0;
        if (cut > 64) hi &= all << (cut - 64);
      } else {
        hi &= cut < 64 ? all >> cut : 0;
        if (cut > 64) lo &= all >> (cut - 64);
      }
      raw = make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
    }
    return raw;
  }
  __device__ __forceinline__ void store(T* row, int cols, uint4 raw) const {
    if (whole(cols)) {
      *(uint4*)(row + first) = raw;
      return;
    }
    if (!RAGGED || first >= cols) return;
    // 8, 4 and 2 bytes from the row's side of the boundary on, each on a boundary of its own
    uint8_t* at = (uint8_t*)(row + first);
    const int n = (int)sizeof(T) * (first < 0 ? V + first : cols - first);   // bytes, 0 < n < 16
    if (first < 0) {
      if (n & 8) *(uint2*)(at + 8) = make_uint2(raw.z, raw.w);
      if (n & 4) *(uint32_t*)(at + 12 - (n & 8)) = n & 8 ? raw.y : raw.w;
      const int e = (n & 12) == 12 ? 0 : (n & 12) == 8 ? 1 : (n & 12) == 4 ? 2 : 3;   // the word that is cut
      if (n & 2) *(uint16_t*)(at + 4 * e + 2) = (uint16_t)((e < 2 ? (e ? raw.y : raw.x) : (e == 2 ? raw.z : raw.w)) >> 16);
    } else {
      if (n & 8) *(uint2*)at = make_uint2(raw.x, raw.y);
      if (n & 4) *(uint32_t*)(at + (n & 8)) = n & 8 ? raw.z : raw.x;
      const int e = n >> 2;
      if (n & 2) *(uint16_t*)(at + 4 * e) = (uint16_t)(e < 2 ? (e ? raw.y : raw.x) : (e == 2 ? raw.z : raw.w));
    }
  }
};

constexpr int kMostSlots = 8;
template <int NW>
constexpr int kThreadsOf = 32 * (NW == 1 ? 4 : NW);
template <int NW>
constexpr int kGroupsOf = kThreadsOf<NW> / (32 * NW);

// CTAs that an SM is to hold: 16 to 20 warps, with the 96 to 128 registers that two pieces take.
// A CTA goes through its rows one at a time, and what a row takes hardly depends on its length, so
// more CTAs are better until the ring of each gets too short.
template <int NW>
constexpr int kCtasOf = NW == 1 ? 4 : NW == 3 ? 6 : NW <= 5 ? 4 : NW == 6 ? 3 : NW <= 10 ? 2 : 1;

// Backward, where three tensors fill the ring: one CTA of ten warps instead of two took 89 us
// instead of 97 for 8192 x 5000 fp16, but 134 instead of 110 for the ragged rows of 8191 x 4999
// (their ends cost latency); of eight warps 74 instead of 64 for 8192 x 4096.
template <int NW, bool RAGGED>
constexpr int kCtasBack = NW == 3 ? 4 + RAGGED : NW == 4 ? 3 : NW == 5 || NW == 6 || NW == 10 ? kCtasOf<NW> - !RAGGED : kCtasOf<NW>;

// A row of weights in 32 bits, in shared memory: pieces of four, so that lanes read next to
// each other (a piece's first half here, its second half `half` further on).  Threads whose rows start at
// different phases (groups of one warp, RAGGED) each need other columns and read global memory.
template <typename T, bool RAGGED, int NW>
struct Weights {
  static constexpr int V = kPiece<T>;
  static constexpr bool kShared = !RAGGED || kGroupsOf<NW> == 1;
  const void* global;
  int type, half;
  float none;
  float4* shared;
  __device__ __forceinline__ void place(const void* p, int t, float otherwise, int cols, int phase, float4* space) {
    global = p, type = t, none = otherwise, shared = space;
    half = (cols + phase + V - 1) / V;
    if (!kShared || !p) return;
    for (int i = threadIdx.x; i < half * V; i += blockDim.x) {
      const int c = i - phase;
      const float v = c >= 0 && c < cols ? load_any(p, c, type) : 0.f;
      ((float*)(shared + (i % V / 4) * half + i / V))[i % 4] = v;
    }
  }
  __device__ __forceinline__ void get(Piece<T, RAGGED> c, int cols, int phase, float (&v)[V]) const {
    if (!global) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = none;
    } else if (kShared) {
      const int piece = c.first < cols ? (c.first + phase) / V : 0;
#pragma unroll
      for (int q = 0; q < V / 4; ++q) {
        const float4 f = shared[q * half + piece];
        v[4 * q] = f.x, v[4 * q + 1] = f.y, v[4 * q + 2] = f.z, v[4 * q + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = c.has(j, cols) ? load_any(global, c.first + j, type) : 0.f;
    }
  }
};

// Sums over the NW warps that share a row, of N values together behind one barrier.
template <int NW, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (&part)[N][16], int warp) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (NW == 1) return;
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) part[i][warp] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v[i] += part[i][w];
  }
}

// After row_sums(): all threads of a row have read its slot, which may be filled again.  Where the
// sums went through a barrier they have; shuffles alone order no memory, least of all reads whose
// values the sums do not take.
template <int NW>
__device__ __forceinline__ void slot_read() {
  if (NW == 1) __syncwarp();
}

// From here on `raw` is taken apart anew: the compiler would keep the 32-bit values instead,
// twice the registers.
__device__ __forceinline__ void forget(uint4& raw) {
  asm volatile("" : "+r"(raw.x), "+r"(raw.y), "+r"(raw.z), "+r"(raw.w));
}

// The ring of one group of warps: in a slot one row of each of the tensors that are read together.
template <typename T, int N, bool RAGGED>
struct Ring {
  const T* base[N];
  int64_t pitch[N];
  int n;                    // tensors there are; a slot has their rows one behind the other
  int64_t rows;
  uint8_t* slots;
  uint64_t* full;
  int cols, depth, bytes;   // bytes of one row in a slot
  bool leader;
  uint32_t waited, pending; // a bit for each slot: the phase its barrier is in; a copy is on its way
  __device__ __forceinline__ bool alone(int64_t row) const { return RAGGED && (row == 0 || row + 1 >= rows); }
  __device__ __forceinline__ uint8_t* slot(int s, int i) const { return slots + (s * n + i) * bytes; }
  // once nobody reads slot s any more
  __device__ __forceinline__ void fetch(int64_t row, int s) {
    if (!leader || row >= rows) return;
    uint32_t total = 0, size[N];
    uintptr_t from[N];
    const int in = alone(row) ? 15 : 0;   // only the pieces that lie inside the row
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i >= n) continue;
      const uintptr_t p = (uintptr_t)(base[i] + row * pitch[i]), end = p + cols * sizeof(T);
      from[i] = (p + in) & ~(uintptr_t)15;
      size[i] = (uint32_t)(((end + 15 - in) & ~(uintptr_t)15) - from[i]);
      total += size[i];
    }
    mbar_expect_tx(&full[s], total);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i >= n || (RAGGED && !size[i])) continue;
      const int ahead = RAGGED ? (int)(from[i] - ((uintptr_t)(base[i] + row * pitch[i]) & ~(uintptr_t)15)) : 0;
      bulk_load(slot(s, i) + ahead, (const void*)from[i], size[i], &full[s]);
    }
    pending |= 1u << s;
  }
  __device__ __forceinline__ void wait(int s, Guard& g) {
    if (!guard_wait(&full[s], waited >> s & 1, g, 0x70000)) return;
    waited ^= 1u << s;
    pending &= ~(1u << s);
  }
  // what fetch() left out of them
  template <int NW>
  __device__ __forceinline__ void fill_ends(int64_t row, int s, int phase, int t) {
    constexpr int V = kPiece<T>;
    const int head = (V - phase) % V, tail = (phase + cols) % V;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i >= n) continue;
      const T* from = base[i] + row * pitch[i];
      T* to = (T*)slot(s, i) + phase;
      if (t < head) to[t] = from[t];
      if (t < tail) to[cols - 1 - t] = from[cols - 1 - t];
    }
    fence_async_shared();   // a copy will follow into the same slot
    if (NW == 1) __syncwarp();
    else __syncthreads();
  }
  // before the CTA ends after a wait that ran out: the copies that are still on their way
  __device__ __forceinline__ void drain(Guard& g) {
    if (!leader) return;
    for (int s = 0; s < depth; ++s)
      if (pending >> s & 1) mbar_wait_bounded(&full[s], waited >> s & 1, kWaitNs, g.status, HP_STATUS_TIMEOUT | 0x80000);
  }
};

// What a kernel of rows starts with: barriers, the ring, the first rows on their way.
template <typename T, int NW, int N, bool RAGGED>
__device__ __forceinline__ void start_ring(Ring<T, N, RAGGED>& ring, uint8_t* space, uint64_t (*full)[kMostSlots], Guard& guard,
                                           uint32_t* status, int64_t first, int64_t step) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < kGroupsOf<NW> * kMostSlots; ++i) mbar_init(&full[0][0] + i, 1);
    mbar_init_fence();
    guard.gave_up = 0;
    guard.status = status;
  }
  __syncthreads();
  dependents_may_start();
  wait_for_kernel_before();
  const int group = threadIdx.x / (32 * NW);
  ring.slots = space + group * ring.depth * ring.n * ring.bytes;
  ring.full = full[group];
  ring.leader = threadIdx.x % (32 * NW) == 0;
  ring.waited = ring.pending = 0;
  for (int s = 0; s < ring.depth; ++s) ring.fetch(first + s * step, s);
}

template <typename T, int NW, int CH, bool RAGGED>
__global__ void __launch_bounds__(kThreadsOf<NW>, NW == 1 && CH > 2 ? 3 : kCtasOf<NW>)
norm_forward_rows(const __grid_constant__ HpNormForward a, int depth, int slot_bytes, int ring_bytes, uint32_t* status) {
  constexpr int V = kPiece<T>, kGroups = kGroupsOf<NW>;
  extern __shared__ __align__(128) uint8_t space[];
  __shared__ float part[2][1][16];
  __shared__ uint64_t full[kGroups][kMostSlots];
  __shared__ Guard guard;
  const int cols = (int)a.cols, t = threadIdx.x % (32 * NW), warp = t >> 5;
  const int64_t first = (int64_t)blockIdx.x * kGroups + threadIdx.x / (32 * NW), step = (int64_t)gridDim.x * kGroups;
  const bool sum_in_front = a.residual != nullptr;
  Ring<T, 2, RAGGED> ring;
  ring.base[0] = (const T*)a.x, ring.base[1] = (const T*)a.residual;
  ring.pitch[0] = a.ldx, ring.pitch[1] = a.ldr;
  ring.n = sum_in_front ? 2 : 1;
  ring.rows = a.rows, ring.cols = cols, ring.depth = depth, ring.bytes = slot_bytes;
  start_ring<T, NW>(ring, space, full, guard, status, first, step);
  const int phase = RAGGED ? (int)(((uintptr_t)((const T*)a.x + first * a.ldx) / sizeof(T)) % V) : 0;
  Piece<T, RAGGED> c[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) c[i].first = (t + i * 32 * NW) * V - phase;
  Weights<T, RAGGED, NW> weight, bias;
  weight.place(a.weight, (int)a.wtype, 1.f, cols, phase, (float4*)(space + ring_bytes));
  bias.place(a.bias, (int)a.wtype, 0.f, cols, phase, (float4*)(space + ring_bytes) + weight.half * (V / 4));
  __syncthreads();
  constexpr bool kHold = NW == 1 || CH <= 2;   // in registers
  float held[kHold ? CH : 1][2][V];
#pragma unroll
  for (int i = 0; kHold && i < CH; ++i) weight.get(c[i], cols, phase, held[i][0]), bias.get(c[i], cols, phase, held[i][1]);
  const float inv = 1.f / (float)cols;
  int s = 0;
  for (int64_t row = first; row < a.rows; row += step) {
    uint4 raw[CH];
    ring.wait(s, guard);
    if (ring.alone(row)) ring.template fill_ends<NW>(row, s, phase, t);
    auto piece = [&](int i, int k) { return c[i].take(ring.slot(s, k), cols, phase); };
    // a row stays packed as it came; to take it apart costs an instruction for an element
    float sum[1] = {0.f};
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      raw[i] = piece(i, 0);
      float v[V];
      unpack<T>(raw[i], v);
      if (sum_in_front) {
        float r[V];
        unpack<T>(piece(i, 1), r);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] += r[j];
        raw[i] = pack<T>(v);   // the sum as it is stored is what is normalised
        unpack<T>(raw[i], v);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) sum[0] += v[j];
    }
    row_sums<NW>(sum, part[0], warp);
    slot_read<NW>();
    if (!guard.gave_up) ring.fetch(row + depth * step, s);
    if (++s == depth) s = 0;
    const float mean = sum[0] * inv;
    // up to two pieces of a thread stay taken apart from here on, more would not fit the registers
    constexpr bool kKeep = NW > 1 && CH <= 2;
    float d[kKeep ? CH : 1][V];
    auto apart = [&](int i, float (&e)[V]) {
      forget(raw[i]);
      unpack<T>(raw[i], e);
#pragma unroll
      for (int j = 0; j < V; ++j) e[j] -= mean;
    };
    sum[0] = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float(&e)[V] = d[kKeep ? i : 0];
      apart(i, e);
      if (sum_in_front) c[i].store((T*)a.z + row * a.cols, cols, raw[i]);
      if (c[i].whole(cols)) {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[0] = fmaf(e[j], e[j], sum[0]);
      } else if (RAGGED && c[i].first < cols) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c[i].has(j, cols)) sum[0] = fmaf(e[j], e[j], sum[0]);
      }
    }
    row_sums<NW>(sum, part[1], warp);
    const float rstd = rsqrtf(sum[0] * inv + (float)a.eps);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float(&e)[V] = d[kKeep ? i : 0];
      if (!kKeep) apart(i, e);
      float(&w)[2][V] = held[kHold ? i : 0];
      if (!kHold) weight.get(c[i], cols, phase, w[0]), bias.get(c[i], cols, phase, w[1]);
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = fmaf(e[j] * rstd, w[0][j], w[1][j]);
      c[i].store((T*)a.y + row * a.cols, cols, pack<T>(y));
    }
    if (t == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
  if (guard.gave_up) ring.drain(guard);
}

template <typename T, int NW, int CH, bool RAGGED>
__global__ void __launch_bounds__(kThreadsOf<NW>, NW == 1 && CH > 1 ? (CH == 4 ? 2 : 3) : kCtasBack<NW, RAGGED>)
norm_backward_rows(const __grid_constant__ HpNormBackward a, int depth, int slot_bytes, int ring_bytes, uint32_t* status) {
  constexpr int V = kPiece<T>, kGroups = kGroupsOf<NW>;
  extern __shared__ __align__(128) uint8_t space[];
  __shared__ float part[2][2][16];
  __shared__ uint64_t full[kGroups][kMostSlots];
  __shared__ Guard guard;
  const int cols = (int)a.cols, t = threadIdx.x % (32 * NW), warp = t >> 5, group = threadIdx.x / (32 * NW);
  const int64_t first = (int64_t)blockIdx.x * kGroups + group, step = (int64_t)gridDim.x * kGroups;
  const bool more = a.dz != nullptr;
  Ring<T, 3, RAGGED> ring;
  ring.base[0] = (const T*)a.z, ring.base[1] = (const T*)a.dy, ring.base[2] = (const T*)a.dz;
  ring.pitch[0] = a.ldz, ring.pitch[1] = a.lddy, ring.pitch[2] = a.lddz;
  ring.n = more ? 3 : 2;
  ring.rows = a.rows, ring.cols = cols, ring.depth = depth, ring.bytes = slot_bytes;
  start_ring<T, NW>(ring, space, full, guard, status, first, step);
  const int phase = RAGGED ? (int)(((uintptr_t)((const T*)a.z + first * a.ldz) / sizeof(T)) % V) : 0;
  Piece<T, RAGGED> c[CH];
  float dw[CH][V], db[CH][V];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    c[i].first = (t + i * 32 * NW) * V - phase;
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.f;
  }
  Weights<T, RAGGED, NW> weight;
  weight.place(a.weight, (int)a.wtype, 1.f, cols, phase, (float4*)(space + ring_bytes));
  __syncthreads();
  // the sums take the registers; what is left holds the weights of short rows
  constexpr bool kHold = NW <= 4;
  float held[CH][V];
  if (kHold)
#pragma unroll
    for (int i = 0; i < CH; ++i) weight.get(c[i], cols, phase, held[i]);
  auto weights = [&](int i, float (&w)[V]) {
    if (!kHold) {
      weight.get(c[i], cols, phase, w);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] = held[i][j];
    }
  };
  const float inv = 1.f / (float)cols;
  int s = 0, turn = 0;
  float mean_next = first < a.rows ? a.mean[first] : 0.f, rstd_next = first < a.rows ? a.rstd[first] : 0.f;
  for (int64_t row = first; row < a.rows; row += step, turn ^= 1) {
    uint4 zr[CH], gr[CH], ur[CH];
    const float mean = mean_next, rstd = rstd_next;
    if (row + step < a.rows) mean_next = a.mean[row + step], rstd_next = a.rstd[row + step];
    ring.wait(s, guard);
    if (ring.alone(row)) ring.template fill_ends<NW>(row, s, phase, t);
    auto piece = [&](int i, int k) { return c[i].take(ring.slot(s, k), cols, phase); };
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float z[V], g[V], w[V];
      weights(i, w);
      zr[i] = piece(i, 0), gr[i] = piece(i, 1);
      if (more) ur[i] = piece(i, 2);
      unpack<T>(zr[i], z);
      unpack<T>(gr[i], g);   // zeros outside the row
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float h = (z[j] - mean) * rstd, gw = g[j] * w[j];
        dw[i][j] = fmaf(g[j], h, dw[i][j]);
        db[i][j] += g[j];
        sum[0] += gw;
        sum[1] = fmaf(gw, h, sum[1]);
      }
    }
    row_sums<NW>(sum, part[turn], warp);
    slot_read<NW>();
    if (!guard.gave_up) ring.fetch(row + depth * step, s);
    if (++s == depth) s = 0;
    if (!a.dx) continue;
    // rstd (g w - mean(g w) - h mean(g w h)), with h = (z - mean) rstd
    const float s1 = -sum[0] * inv * rstd, s2 = sum[1] * inv * rstd * rstd;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float z[V], g[V], d[V], up[V], w[V];
      weights(i, w);
      forget(zr[i]);
      forget(gr[i]);
      unpack<T>(zr[i], z);
      unpack<T>(gr[i], g);
      if (more) unpack<T>(ur[i], up);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        d[j] = fmaf(mean - z[j], s2, fmaf(g[j], w[j] * rstd, s1));
        if (more) d[j] += up[j];
      }
      c[i].store((T*)a.dx + row * a.cols, cols, pack<T>(d));
    }
  }
  if (guard.gave_up) ring.drain(guard);
  if (!a.dweight && !a.dbias) return;
  float* out = (float*)a.workspace + (int64_t)blockIdx.x * 2 * cols;
  if constexpr (kGroups == 1) {
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c[i].has(j, cols)) out[c[i].first + j] = dw[i][j], out[cols + c[i].first + j] = db[i][j];
  } else {
    // every group its own sums, a thread's next to its neighbours'; then by columns
    float* joint = (float*)space;   // the ring is done with
    const int pieces = 32 * NW * CH, most = kGroups * V * pieces;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int at = (group * V + j) * pieces + t + i * 32 * NW;
        joint[at] = dw[i][j], joint[most + at] = db[i][j];
      }
    __syncthreads();
    for (int e = threadIdx.x; e < cols; e += blockDim.x) {
      float sw = 0.f, sb = 0.f;
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        const int64_t row = (int64_t)blockIdx.x * kGroups + k;
        const int at = e + (RAGGED ? (int)(((uintptr_t)((const T*)a.z + row * a.ldz) / sizeof(T)) % V) : 0);
        const int q = (k * V + at % V) * pieces + at / V;
        sw += joint[q], sb += joint[most + q];
      }
      out[e] = sw, out[cols + e] = sb;
    }
  }
}

// How many warps share a row of so many columns, and how many pieces a thread has; 0 where a row
// does not fit.  Two pieces a thread and as many warps as that takes: three pieces in eight warps
// needed 242 us for forward and backward of 8191 x 4999 fp16, two in ten 194.  Where rows start
// anywhere, one piece more than the row's length takes.  Of one warp's rows three pieces
// instead of four: 65536 x 768 forward 53 to 44 us in bf16, with a residual in fp16 67 to 70.
struct Split {
  int warps, pieces;
};
template <typename T>
Split split_of(int64_t cols, bool ragged) {
  if (ragged && cols < kPiece<T>) return {0, 0};   // a row's boundaries would reach beyond its neighbours
  const int64_t n = (cols + kPiece<T> - 1) / kPiece<T> + (ragged ? 1 : 0);
  if (n <= 32) return {1, 1};
  if (n <= 64) return {1, 2};
  if (n <= 96) return {1, 3};
  if (n <= 128) return {1, 4};
  for (int warps : {3, 4, 5, 6, 8, 10, 12, 16})
    if (n <= 64 * warps) return {warps, 2};
  if (n <= 1536) return {16, 3};
  if (n <= 2048) return {16, 4};
  return {0, 0};
}

// Rows cut alike: whether every tensor's rows lie alike with regard to 16-byte boundaries, and
// whether they all begin and end on one.  The length counts for itself: padded rows begin on a
// boundary whatever it is, and where no dense result is among the tensors it shows nowhere else.
struct Rows {
  uintptr_t phase;
  int64_t pitch;
  bool alike = true, any = false;
  int size;
  int64_t end;
  Rows(int bytes, int64_t cols) : size(bytes), end(cols * bytes % 16) {}
  void add(const void* p, int64_t ld) {
    if (!p) return;
    const uintptr_t f = (uintptr_t)p % 16;
    const int64_t l = ld * size % 16;
    if (any && (f != phase || l != pitch)) alike = false;
    phase = f, pitch = l, any = true;
  }
  bool ragged() const { return phase != 0 || pitch != 0 || end != 0; }
};

constexpr int kMostCtas = 1024;   // rows of partial sums

// CTAs for `rows` rows, `groups` at once in each: at most `per_sm` to an SM and kMostCtas; where
// rows start anywhere a multiple of eight, which keeps a group's rows alike
unsigned ctas_for(int64_t rows, int groups, int per_sm, bool ragged) {
  int64_t n = (rows + groups - 1) / groups, most = (int64_t)layer_sms() * per_sm;
  if (most > kMostCtas) most = kMostCtas;
  if (ragged) n = (n + 7) / 8 * 8, most = most < 8 ? 8 : most / 8 * 8;
  return (unsigned)(n < most ? n : most);
}

// Shared memory of a CTA at most: what an SM has, divided by the CTAs it is meant to hold.  The
// weights take their part of it, the ring the rest; when the ring is done with, its space holds
// the groups' sums.
constexpr int space_of(int ctas) { return 216 / ctas * 1024; }

struct RingSize {
  int slot, depth, ring, bytes;
};
template <typename T, int NW, int CH, bool RAGGED>
RingSize ring_size(int space, int64_t cols, int tensors, int weights, bool sums) {
  RingSize r;
  r.slot = (int)((cols * sizeof(T) + (RAGGED ? 30 : 0) + 15) / 16 * 16);
  const int set = kGroupsOf<NW> * tensors * r.slot;
  const int w = Weights<T, RAGGED, NW>::kShared ? weights * (int)((cols + 2 * kPiece<T>) * 4) : 0;
  r.depth = (space - w) / set;
  if (r.depth > kMostSlots) r.depth = kMostSlots;
  r.ring = r.depth * set;   // whole pieces, as the weights behind it want
  r.bytes = r.ring + w;
  const int joint = sums && kGroupsOf<NW> > 1 ? kGroupsOf<NW> * 2 * kPiece<T> * 32 * NW * CH * 4 : 0;
  if (r.bytes < joint) r.bytes = joint;
  return r;
}

// CTAs of the kernel that an SM of the current device holds, with the largest ring; `known` is the kernel's own
template <typename K>
int resident(PerDevice& known, K kernel, int threads, int smem, int* ctas) {
  int dev = 0;
  if (const int rc = told(cudaGetDevice(&dev))) return rc;
  return known.get(dev, [&](int* n) {
    if (const int rc = told(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem))) return rc;
    const int rc = told(cudaOccupancyMaxActiveBlocksPerMultiprocessor(n, kernel, threads, smem));
    if (*n < 1) *n = 1;
    return rc;
  }, ctas);
}

template <typename T, int NW, int CH, bool RAGGED>
int forward_rows(const HpNormForward& a, uint32_t* status, cudaStream_t s) {
  static PerDevice known;
  int per_sm;
  if (const int rc = resident(known, norm_forward_rows<T, NW, CH, RAGGED>, kThreadsOf<NW>, space_of(kCtasOf<NW>), &per_sm)) return rc;
  const RingSize r = ring_size<T, NW, CH, RAGGED>(space_of(kCtasOf<NW>), a.cols, a.residual ? 2 : 1, 2, false);
  return launch_behind(norm_forward_rows<T, NW, CH, RAGGED>, ctas_for(a.rows, kGroupsOf<NW>, per_sm, RAGGED), kThreadsOf<NW>,
                       r.bytes, s, a, r.depth, r.slot, r.ring, status);
}
template <typename T, int NW, int CH, bool RAGGED>
int backward_rows(const HpNormBackward& a, uint32_t* status, cudaStream_t s) {
  static PerDevice known;
  int per_sm;
  if (const int rc = resident(known, norm_backward_rows<T, NW, CH, RAGGED>, kThreadsOf<NW>, space_of(kCtasBack<NW, RAGGED>), &per_sm))
    return rc;
  const RingSize r = ring_size<T, NW, CH, RAGGED>(space_of(kCtasBack<NW, RAGGED>), a.cols, a.dz ? 3 : 2, 1, true);
  const unsigned grid = ctas_for(a.rows, kGroupsOf<NW>, per_sm, RAGGED);
  const int rc = launch_behind(norm_backward_rows<T, NW, CH, RAGGED>, grid, kThreadsOf<NW>, r.bytes, s, a, r.depth, r.slot,
                               r.ring, status);
  if (rc || (!a.dweight && !a.dbias)) return rc;
  return column_sums((const float*)a.workspace, (int)grid, 2 * a.cols, a.cols, a.dweight, a.dbias, (int)a.wtype, s);
}

#define BY_SPLIT(call)                          \
  switch (p.warps * 8 + p.pieces) {             \
    case 1 * 8 + 1: return call(1, 1);          \
    case 1 * 8 + 2: return call(1, 2);          \
    case 1 * 8 + 3: return call(1, 3);          \
    case 1 * 8 + 4: return call(1, 4);          \
    case 3 * 8 + 2: return call(3, 2);          \
    case 4 * 8 + 2: return call(4, 2);          \
    case 5 * 8 + 2: return call(5, 2);          \
    case 6 * 8 + 2: return call(6, 2);          \
    case 8 * 8 + 2: return call(8, 2);          \
    case 10 * 8 + 2: return call(10, 2);        \
    case 12 * 8 + 2: return call(12, 2);        \
    case 16 * 8 + 2: return call(16, 2);        \
    case 16 * 8 + 3: return call(16, 3);        \
    case 16 * 8 + 4: return call(16, 4);        \
    default: break;                             \
  }

template <typename T>
int forward(const HpNormForward& a, cudaStream_t s) {
  Rows r(sizeof(T), a.cols);
  r.add(a.x, a.ldx);
  r.add(a.residual, a.ldr);
  r.add(a.y, a.cols);
  r.add(a.z, a.cols);
  if (r.alike) {
    const Split p = split_of<T>(a.cols, r.ragged());
    int rc;
    uint32_t* status = layer_status(&rc);
    if (rc) return rc;
#define CALL(nw, ch) r.ragged() ? forward_rows<T, nw, ch, true>(a, status, s) : forward_rows<T, nw, ch, false>(a, status, s)
    BY_SPLIT(CALL)
#undef CALL
  }
  norm_forward_kernel<T><<<(unsigned)a.rows, 256, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T>
int backward(const HpNormBackward& a, cudaStream_t s) {
  Rows r(sizeof(T), a.cols);
  r.add(a.z, a.ldz);
  r.add(a.dy, a.lddy);
  r.add(a.dz, a.lddz);
  r.add(a.dx, a.cols);
  if (r.alike && a.rows) {
    const Split p = split_of<T>(a.cols, r.ragged());
    int rc;
    uint32_t* status = layer_status(&rc);
    if (rc) return rc;
#define CALL(nw, ch) r.ragged() ? backward_rows<T, nw, ch, true>(a, status, s) : backward_rows<T, nw, ch, false>(a, status, s)
    BY_SPLIT(CALL)
#undef CALL
  }
  if (a.dx && a.rows) norm_dx_kernel<T><<<(unsigned)a.rows, 256, 0, s>>>(a);
  if (a.dweight || a.dbias) norm_dw_kernel<T><<<(unsigned)((a.cols + 31) / 32), dim3(32, 8), 0, s>>>(a);
  return cudaGetLastError();
}

template <typename A>
bool types_ok(const A& a) {
  return type_ok(a.type) && (a.wtype == HP_F32 || a.wtype == a.type);
}

}  // namespace
}  // namespace hipress

using namespace hipress;

#define BY_TYPE(fn) a->type == HP_F32 ? fn<float>(*a, s) : a->type == HP_BF16 ? fn<__nv_bfloat16>(*a, s) : fn<__half>(*a, s)

extern "C" int hp_cuda_norm_forward(const HpNormForward* a, void* stream) {
  if (!a || a->rows < 0 || a->cols < 1 || a->rows > INT32_MAX || !types_ok(*a) || (a->residual && !a->z))
    return HP_ERR_BAD_ARG;
  if (!a->rows) return 0;
  cudaStream_t s = (cudaStream_t)stream;
  return BY_TYPE(forward);
}

extern "C" int hp_cuda_norm_backward(const HpNormBackward* a, void* stream) {
  if (!a || a->rows < 0 || a->cols < 1 || a->rows > INT32_MAX || !types_ok(*a)) return HP_ERR_BAD_ARG;
  cudaStream_t s = (cudaStream_t)stream;
  return BY_TYPE(backward);
}

extern "C" uint64_t hp_cuda_norm_workspace(int64_t rows, int64_t cols) {
  const int64_t ctas = rows + 8 < kMostCtas ? rows + 8 : kMostCtas;
  return (uint64_t)ctas * 2 * cols * 4;
}
