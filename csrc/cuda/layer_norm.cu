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

// ------------------------------------------------------------- rows in registers
// NW warps share a row, each thread CH pieces of 16 bytes of it.  A thread keeps its columns
// from row to row, and with them the weights and (backward) the sums of the weights' gradients.
// Rows whose first element is not on a 16-byte boundary are cut at the boundaries all the
// same: the pieces start `phase` elements ahead of the row, and what is outside the row is left
// out.  The phase goes by the row modulo the elements of a piece, and the rows of one group
// of warps are that far apart, so that its columns stay the same.
// The columns that a thread's piece covers.  Unless RAGGED a piece is in the row or behind it.
template <typename T, bool RAGGED>
struct Piece {
  static constexpr int V = kPiece<T>, kBits = 8 * sizeof(T);
  int first;
  __device__ __forceinline__ bool whole(int cols) const {
    return RAGGED ? first >= 0 && first + V <= cols : first < cols;
  }
  __device__ __forceinline__ bool has(int j, int cols) const {
    return RAGGED ? first + j >= 0 && first + j < cols : first < cols;
  }
  __device__ __forceinline__ void load_weights(const void* p, int type, int cols, float none, float (&v)[V]) const {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = p && has(j, cols) ? load_any(p, first + j, type) : none;
  }
  // Zeros outside the row.  A piece at an end of it: where the rows next to this one are there
  // (`inner`; and no row is shorter than a piece) it is loaded whole and what is not the row's
  // is cleared; else it goes element by element, shifted through its 128 bits: few registers
  // for what few threads do.
  __device__ __forceinline__ uint4 load(const T* row, int cols, bool there, bool inner) const {
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (!there) return raw;
    if (whole(cols)) return __ldg((const uint4*)(row + first));
    if (!RAGGED || first >= cols) return raw;
    T* v = (T*)&raw;
    if (inner && cols >= V) {
      raw = __ldg((const uint4*)(row + first));
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (!has(j, cols)) v[j] = from_f<T>(0.f);
      return raw;
    }
    uint64_t lo = 0, hi = 0;
#pragma unroll 1
    for (int j = 0; j < V; ++j) {
      T e = from_f<T>(0.f);
      if (has(j, cols)) e = row[first + j];
      const uint64_t bits = sizeof(T) == 4 ? *(const uint32_t*)&e : *(const uint16_t*)&e;
      lo = lo >> kBits | hi << (64 - kBits);
      hi = hi >> kBits | bits << (64 - kBits);
    }
    return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
  }
  __device__ __forceinline__ void store(T* row, int cols, bool there, uint4 raw) const {
    if (!there) return;
    if (whole(cols)) {
      *(uint4*)(row + first) = raw;
      return;
    }
    if (!RAGGED || first >= cols) return;
    uint64_t lo = raw.x | (uint64_t)raw.y << 32, hi = raw.z | (uint64_t)raw.w << 32;
#pragma unroll 1
    for (int j = 0; j < V; ++j) {
      if (has(j, cols)) {
        if (sizeof(T) == 4) ((uint32_t*)row)[first + j] = (uint32_t)lo;
        else ((uint16_t*)row)[first + j] = (uint16_t)lo;
      }
      lo = lo >> kBits | hi << (64 - kBits);
      hi >>= kBits;
    }
  }
};

// Sums over the NW warps that share a row, of N values together behind one barrier; `part` is
// theirs until the barrier after the next.
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

// From here on `raw` is taken apart anew: the compiler would keep the 32-bit values instead,
// twice the registers.
__device__ __forceinline__ void forget(uint4& raw) {
  asm volatile("" : "+r"(raw.x), "+r"(raw.y), "+r"(raw.z), "+r"(raw.w));
}

template <int NW>
constexpr int kThreadsOf = 32 * (NW < 4 ? 4 : NW);

// Rows that a group of warps takes at once: their loads are in flight together and their sums
// share the shuffles' and barriers' latency.
template <int CH>
constexpr int kAtOnce = CH == 1 ? 4 : CH == 2 ? 2 : 1;

template <typename T, int NW, int CH, bool RAGGED>
__global__ void __launch_bounds__(kThreadsOf<NW>, NW <= 4 ? (CH == 1 ? 7 : 4) : NW == 8 ? (CH == 2 ? 3 : 2) : 1)
norm_forward_rows(const __grid_constant__ HpNormForward a) {
  constexpr int V = kPiece<T>, kGroups = kThreadsOf<NW> / (32 * NW), R = kAtOnce<CH>;
  __shared__ float part[2][R][16];
  const int cols = (int)a.cols, t = threadIdx.x % (32 * NW), warp = t >> 5;
  const int64_t first = (int64_t)blockIdx.x * kGroups + threadIdx.x / (32 * NW), step = (int64_t)gridDim.x * kGroups;
  if (first >= a.rows) return;   // the whole CTA where it shares a row
  const int phase = RAGGED ? (int)(((uintptr_t)((const T*)a.x + first * a.ldx) / sizeof(T)) % V) : 0;
  Piece<T, RAGGED> c[CH];
  float w[CH][V], b[CH][V];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    c[i].first = (t + i * 32 * NW) * V - phase;
    c[i].load_weights(a.weight, (int)a.wtype, cols, 1.f, w[i]);
    c[i].load_weights(a.bias, (int)a.wtype, cols, 0.f, b[i]);
  }
  const float inv = 1.f / (float)cols;
  for (int64_t row0 = first; row0 < a.rows; row0 += R * step) {
    uint4 raw[R][CH], res[R][CH];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t row = row0 + k * step;
      const bool there = row < a.rows, inner = row > 0 && row + 1 < a.rows;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        raw[k][i] = c[i].load((const T*)a.x + row * a.ldx, cols, there, inner);
        if (a.residual) res[k][i] = c[i].load((const T*)a.residual + row * a.ldr, cols, there, inner);
      }
    }
    // a row stays packed as it came; to take it apart costs an instruction for an element, and half
    // the registers are half the warps
    float s[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      s[k] = 0.f;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        float v[V];
        unpack<T>(raw[k][i], v);
        if (a.residual) {
          float r[V];
          unpack<T>(res[k][i], r);
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] += r[j];
          raw[k][i] = pack<T>(v);   // the sum as it is stored is what is normalised
          unpack<T>(raw[k][i], v);
          c[i].store((T*)a.z + (row0 + k * step) * a.cols, cols, row0 + k * step < a.rows, raw[k][i]);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) s[k] += v[j];
      }
    }
    row_sums<NW>(s, part[0], warp);
    float mean[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      mean[k] = s[k] * inv;
      s[k] = 0.f;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        float v[V];
        forget(raw[k][i]);
        unpack<T>(raw[k][i], v);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = v[j] - mean[k];
          if (c[i].has(j, cols)) s[k] = fmaf(d, d, s[k]);
        }
      }
    }
    row_sums<NW>(s, part[1], warp);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t row = row0 + k * step;
      const float rstd = 1.f / sqrtf(s[k] * inv + (float)a.eps);
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        float v[V];
        forget(raw[k][i]);
        unpack<T>(raw[k][i], v);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = fmaf((v[j] - mean[k]) * rstd, w[i][j], b[i][j]);
        c[i].store((T*)a.y + row * a.cols, cols, row < a.rows, pack<T>(v));
      }
      if (t == 0 && row < a.rows) {
        a.mean[row] = mean[k];
        a.rstd[row] = rstd;
      }
    }
  }
}

template <typename T, int NW, int CH, bool RAGGED>
__global__ void __launch_bounds__(kThreadsOf<NW>, NW <= 4 ? (CH == 1 ? 5 : 3) : NW == 8 ? (CH == 2 ? 2 : 1) : 1)
norm_backward_rows(const __grid_constant__ HpNormBackward a) {
  constexpr int V = kPiece<T>, kGroups = kThreadsOf<NW> / (32 * NW), R = CH >= 3 || NW == 16 ? 1 : 2;
  __shared__ float part[2][2 * R][16];
  extern __shared__ float joint[];   // [2 cols], where several rows are at work in a CTA
  const int cols = (int)a.cols, t = threadIdx.x % (32 * NW), warp = t >> 5, group = threadIdx.x / (32 * NW);
  const int64_t first = (int64_t)blockIdx.x * kGroups + group, step = (int64_t)gridDim.x * kGroups;
  const int phase = RAGGED ? (int)(((uintptr_t)((const T*)a.z + first * a.ldz) / sizeof(T)) % V) : 0;
  Piece<T, RAGGED> c[CH];
  float w[CH][V], dw[CH][V], db[CH][V];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    c[i].first = (t + i * 32 * NW) * V - phase;
    c[i].load_weights(a.weight, (int)a.wtype, cols, 1.f, w[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.f;
  }
  dependents_may_start();
  const float inv = 1.f / (float)cols;
  int turn = 0;
  for (int64_t row0 = first; row0 < a.rows; row0 += R * step, turn ^= 1) {
    uint4 zr[R][CH], gr[R][CH], ur[R][CH];
    float mean[R], rstd[R], s[2 * R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t row = row0 + k * step;
      const bool there = row < a.rows, inner = row > 0 && row + 1 < a.rows;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        zr[k][i] = c[i].load((const T*)a.z + row * a.ldz, cols, there, inner);
        gr[k][i] = c[i].load((const T*)a.dy + row * a.lddy, cols, there, inner);
        if (a.dz) ur[k][i] = c[i].load((const T*)a.dz + row * a.lddz, cols, there, inner);
      }
      mean[k] = there ? a.mean[row] : 0.f, rstd[k] = there ? a.rstd[row] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        float z[V], g[V];
        unpack<T>(zr[k][i], z);
        unpack<T>(gr[k][i], g);   // zeros outside the row
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float h = (z[j] - mean[k]) * rstd[k], gw = g[j] * w[i][j];
          dw[i][j] = fmaf(g[j], h, dw[i][j]);
          db[i][j] += g[j];
          s1 += gw;
          s2 = fmaf(gw, h, s2);
        }
      }
      s[2 * k] = s1, s[2 * k + 1] = s2;
    }
    if (!a.dx) continue;
    row_sums<NW>(s, part[turn], warp);   // one barrier a turn: the halves take turns
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t row = row0 + k * step;
      // rstd (g w - mean(g w) - h mean(g w h)), with h = (z - mean) rstd
      const float s1 = -s[2 * k] * inv * rstd[k], s2 = s[2 * k + 1] * inv * rstd[k] * rstd[k];
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        float z[V], g[V], d[V], up[V];
        forget(zr[k][i]);
        forget(gr[k][i]);
        unpack<T>(zr[k][i], z);
        unpack<T>(gr[k][i], g);
        if (a.dz) unpack<T>(ur[k][i], up);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          d[j] = fmaf(mean[k] - z[j], s2, fmaf(g[j], w[i][j] * rstd[k], s1));
          if (a.dz) d[j] += up[j];
        }
        c[i].store((T*)a.dx + row * a.cols, cols, row < a.rows, pack<T>(d));
      }
    }
  }
  if (!a.dweight && !a.dbias) return;
  float* out = (float*)a.workspace + (int64_t)blockIdx.x * 2 * cols;
  if constexpr (kGroups == 1) {
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c[i].has(j, cols)) out[c[i].first + j] = dw[i][j], out[cols + c[i].first + j] = db[i][j];
  } else {
    for (int k = 0; k < kGroups; ++k) {   // one row's warps after the other
      if (group == k)
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (c[i].has(j, cols)) {
              float* at = joint + c[i].first + j;
              at[0] = k ? at[0] + dw[i][j] : dw[i][j];
              at[cols] = k ? at[cols] + db[i][j] : db[i][j];
            }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * cols; i += blockDim.x) out[i] = joint[i];
  }
}

// How many warps share a row of so many columns, and how many pieces a thread has; 0 where a row
// does not fit.  One piece more than the row's length takes, where rows start anywhere.
struct Split {
  int warps, pieces;
};
template <typename T>
Split split_of(int64_t cols, bool ragged) {
  const int64_t n = (cols + kPiece<T> - 1) / kPiece<T> + (ragged ? 1 : 0);
  if (n <= 32) return {1, 1};
  if (n <= 64) return {1, 2};
  if (n <= 128) return {4, 1};
  if (n <= 256) return {4, 2};
  if (n <= 512) return {8, 2};
  if (n <= 768) return {8, 3};
  if (n <= 1024) return {16, 2};
  if (n <= 2048) return {16, 4};
  return {0, 0};
}

// Rows cut alike: whether every tensor's rows lie alike with regard to 16-byte boundaries, and
// whether they all begin on one.
struct Rows {
  uintptr_t phase;
  int64_t pitch;
  bool alike = true, any = false;
  int size;
  explicit Rows(int bytes) : size(bytes) {}
  void add(const void* p, int64_t ld) {
    if (!p) return;
    const uintptr_t f = (uintptr_t)p % 16;
    const int64_t l = ld * size % 16;
    if (any && (f != phase || l != pitch)) alike = false;
    phase = f, pitch = l, any = true;
  }
  bool ragged() const { return phase != 0 || pitch != 0; }
};

constexpr int kMostCtas = 1024;   // rows of partial sums

template <typename K>
int resident(K kernel, int threads, int smem) {
  int n = 1;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess || n < 1) n = 1;
  return n;
}

// CTAs for `rows` rows, `groups` at once in each: at most `per_sm` to an SM and kMostCtas; where
// rows start anywhere a multiple of eight, which keeps a group's rows alike
unsigned ctas_for(int64_t rows, int groups, int per_sm, bool ragged) {
  int64_t n = (rows + groups - 1) / groups, most = (int64_t)layer_sms() * per_sm;
  if (most > kMostCtas) most = kMostCtas;
  if (ragged) n = (n + 7) / 8 * 8, most = most < 8 ? 8 : most / 8 * 8;
  return (unsigned)(n < most ? n : most);
}

template <typename T, int NW, int CH, bool RAGGED>
int forward_rows(const HpNormForward& a, cudaStream_t s) {
  constexpr int kThreads = kThreadsOf<NW>, kGroups = kThreads / (32 * NW);
  static const int per_sm = resident(norm_forward_rows<T, NW, CH, RAGGED>, kThreads, 0);
  norm_forward_rows<T, NW, CH, RAGGED><<<ctas_for(a.rows, kGroups, per_sm, RAGGED), kThreads, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T, int NW, int CH, bool RAGGED>
int backward_rows(const HpNormBackward& a, cudaStream_t s) {
  constexpr int kThreads = kThreadsOf<NW>, kGroups = kThreads / (32 * NW);
  const int smem = kGroups > 1 ? (int)(8 * a.cols) : 0;
  static const int per_sm = resident(norm_backward_rows<T, NW, CH, RAGGED>, kThreads, kGroups > 1 ? 8 * 32 * CH * kPiece<T> : 0);
  const unsigned grid = ctas_for(a.rows, kGroups, per_sm, RAGGED);
  norm_backward_rows<T, NW, CH, RAGGED><<<grid, kThreads, smem, s>>>(a);
  const int rc = cudaGetLastError();
  if (rc || (!a.dweight && !a.dbias)) return rc;
  return column_sums((const float*)a.workspace, (int)grid, 2 * a.cols, a.cols, a.dweight, a.dbias, (int)a.wtype, s);
}

#define BY_SPLIT(call)                          \
  switch (p.warps * 8 + p.pieces) {             \
    case 1 * 8 + 1: return call(1, 1);          \
    case 1 * 8 + 2: return call(1, 2);          \
    case 4 * 8 + 1: return call(4, 1);          \
    case 4 * 8 + 2: return call(4, 2);          \
    case 8 * 8 + 2: return call(8, 2);          \
    case 8 * 8 + 3: return call(8, 3);          \
    case 16 * 8 + 2: return call(16, 2);        \
    case 16 * 8 + 4: return call(16, 4);        \
    default: break;                             \
  }

template <typename T>
int forward(const HpNormForward& a, cudaStream_t s) {
  Rows r(sizeof(T));
  r.add(a.x, a.ldx);
  r.add(a.residual, a.ldr);
  r.add(a.y, a.cols);
  r.add(a.z, a.cols);
  if (r.alike) {
    const Split p = split_of<T>(a.cols, r.ragged());
#define CALL(nw, ch) r.ragged() ? forward_rows<T, nw, ch, true>(a, s) : forward_rows<T, nw, ch, false>(a, s)
    BY_SPLIT(CALL)
#undef CALL
  }
  norm_forward_kernel<T><<<(unsigned)a.rows, 256, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T>
int backward(const HpNormBackward& a, cudaStream_t s) {
  Rows r(sizeof(T));
  r.add(a.z, a.ldz);
  r.add(a.dy, a.lddy);
  r.add(a.dz, a.lddz);
  r.add(a.dx, a.cols);
  if (r.alike && a.rows) {
    const Split p = split_of<T>(a.cols, r.ragged());
#define CALL(nw, ch) r.ragged() ? backward_rows<T, nw, ch, true>(a, s) : backward_rows<T, nw, ch, false>(a, s)
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

extern "C" uint64_t hp_cuda_norm_workspace(int64_t rows, int64_t cols, int64_t) {
  const int64_t ctas = rows + 8 < kMostCtas ? rows + 8 : kMostCtas;
  return (uint64_t)ctas * 2 * cols * 4;
}
