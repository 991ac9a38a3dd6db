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
template <typename T>
constexpr int kPiece = 16 / sizeof(T);

template <typename T>
struct Piece {   // which columns a thread's piece covers
  int first;
  __device__ __forceinline__ bool whole(int cols) const { return first >= 0 && first + kPiece<T> <= cols; }
  __device__ __forceinline__ bool has(int j, int cols) const { return first + j >= 0 && first + j < cols; }
};

// A piece at an end of the row goes element by element, shifted through its 128 bits: few
// registers for what few threads do.
template <typename T>
__device__ __forceinline__ uint4 load_piece(const T* row, Piece<T> c, int cols) {
  if (c.whole(cols)) return __ldg((const uint4*)(row + c.first));
  uint64_t lo = 0, hi = 0;
  constexpr int kBits = 8 * sizeof(T);
  if (c.first < cols)
#pragma unroll 1
    for (int j = 0; j < kPiece<T>; ++j) {
      T v = from_f<T>(0.f);
      if (c.has(j, cols)) v = row[c.first + j];
      uint64_t bits = 0;
      if (sizeof(T) == 4) bits = *(const uint32_t*)&v;
      else bits = *(const uint16_t*)&v;
      lo = lo >> kBits | hi << (64 - kBits);
      hi = hi >> kBits | bits << (64 - kBits);
    }
  return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}
template <typename T>
__device__ __forceinline__ void store_piece(T* row, Piece<T> c, int cols, const float (&v)[kPiece<T>]) {
  uint4 raw;
  T* t = (T*)&raw;
#pragma unroll
  for (int j = 0; j < kPiece<T>; ++j) t[j] = from_f<T>(v[j]);
  if (c.whole(cols)) {
    *(uint4*)(row + c.first) = raw;
    return;
  }
  uint64_t lo = raw.x | (uint64_t)raw.y << 32, hi = raw.z | (uint64_t)raw.w << 32;
  constexpr int kBits = 8 * sizeof(T);
  if (c.first < cols)
#pragma unroll 1
    for (int j = 0; j < kPiece<T>; ++j) {
      if (c.has(j, cols)) {
        if (sizeof(T) == 4) ((uint32_t*)row)[c.first + j] = (uint32_t)lo;
        else ((uint16_t*)row)[c.first + j] = (uint16_t)lo;
      }
      lo = lo >> kBits | hi << (64 - kBits);
      hi >>= kBits;
    }
}
template <typename T>
__device__ __forceinline__ void unpack(uint4 raw, float (&v)[kPiece<T>]) {
  const T* t = (const T*)&raw;
#pragma unroll
  for (int j = 0; j < kPiece<T>; ++j) v[j] = to_f(t[j]);
}

// sums over the NW warps that share a row; `part` [2][16] floats, used in turn
template <int NW>
__device__ __forceinline__ float row_sum(float v, float* part, int warp) {
  v = warp_sum(v);
  if (NW == 1) return v;
  if ((threadIdx.x & 31) == 0) part[warp] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) s += part[i];
  return s;
}

template <int NW>
constexpr int kThreadsOf = 32 * (NW < 4 ? 4 : NW);

template <typename T, typename W, int NW, int CH>
__global__ void __launch_bounds__(kThreadsOf<NW>, NW <= 4 ? 4 : NW == 8 ? 2 : 1) norm_forward_rows(const __grid_constant__ HpNormForward a, int ragged) {
  constexpr int V = kPiece<T>, kGroups = kThreadsOf<NW> / (32 * NW);
  __shared__ float part[2][16];
  const int cols = (int)a.cols, t = threadIdx.x % (32 * NW), warp = t >> 5;
  const int64_t first = (int64_t)blockIdx.x * kGroups + threadIdx.x / (32 * NW), step = (int64_t)gridDim.x * kGroups;
  if (first >= a.rows) return;   // the whole CTA where it shares a row
  const int phase = ragged ? (int)(((uintptr_t)((const T*)a.x + first * a.ldx) / sizeof(T)) % V) : 0;
  Piece<T> c[CH];
  float w[CH][V], b[CH][V];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    c[i].first = (t + i * 32 * NW) * V - phase;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w[i][j] = a.weight && c[i].has(j, cols) ? to_f(((const W*)a.weight)[c[i].first + j]) : 1.f;
      b[i][j] = a.bias && c[i].has(j, cols) ? to_f(((const W*)a.bias)[c[i].first + j]) : 0.f;
    }
  }
  const float inv = 1.f / (float)cols;
  uint4 raw[CH], res[CH];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      raw[i] = load_piece((const T*)a.x + row * a.ldx, c[i], cols);
      if (a.residual) res[i] = load_piece((const T*)a.residual + row * a.ldr, c[i], cols);
    }
  };
  constexpr bool kAhead = CH <= 2;   // with more pieces the registers do not suffice
  if (kAhead) fetch(first);
  for (int64_t row = first; row < a.rows; row += step) {
    if (!kAhead) fetch(row);
    float v[CH][V], s = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      unpack<T>(raw[i], v[i]);
      if (a.residual) {
        float r[V];
        unpack<T>(res[i], r);
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = to_f(from_f<T>(v[i][j] + r[j]));
        store_piece((T*)a.z + row * a.cols, c[i], cols, v[i]);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) s += v[i][j];
    }
    if (kAhead && row + step < a.rows) fetch(row + step);   // on its way while this row is summed
    const float mean = row_sum<NW>(s, part[0], warp) * inv;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const bool whole = c[i].whole(cols);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = v[i][j] - mean;
        v[i][j] = d;
        if (whole || c[i].has(j, cols)) s = fmaf(d, d, s);
      }
    }
    const float rstd = 1.f / sqrtf(row_sum<NW>(s, part[1], warp) * inv + (float)a.eps);
    T* y = (T*)a.y + row * a.cols;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = fmaf(v[i][j] * rstd, w[i][j], b[i][j]);
      store_piece(y, c[i], cols, v[i]);
    }
    if (t == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

template <typename T, typename W, int NW, int CH>
__global__ void __launch_bounds__(kThreadsOf<NW>, NW <= 4 ? 4 : NW == 8 ? 2 : 1) norm_backward_rows(const __grid_constant__ HpNormBackward a, int ragged) {
  constexpr int V = kPiece<T>, kGroups = kThreadsOf<NW> / (32 * NW);
  __shared__ float part[4][16];
  extern __shared__ float joint[];   // [2 cols], where several rows are at work in a CTA
  const int cols = (int)a.cols, t = threadIdx.x % (32 * NW), warp = t >> 5, group = threadIdx.x / (32 * NW);
  const int64_t first = (int64_t)blockIdx.x * kGroups + group, step = (int64_t)gridDim.x * kGroups;
  const int phase =
      ragged ? (int)(((uintptr_t)((const T*)a.z + first * a.ldz) / sizeof(T)) % V) : 0;
  Piece<T> c[CH];
  float w[CH][V], dw[CH][V], db[CH][V];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    c[i].first = (t + i * 32 * NW) * V - phase;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w[i][j] = a.weight && c[i].has(j, cols) ? to_f(((const W*)a.weight)[c[i].first + j]) : 1.f;
      dw[i][j] = db[i][j] = 0.f;
    }
  }
  dependents_may_start();
  const float inv = 1.f / (float)cols;
  int turn = 0;
  uint4 zn[CH], gn[CH];
  float mean_next = 0.f, rstd_next = 0.f;
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      zn[i] = load_piece((const T*)a.z + row * a.ldz, c[i], cols);
      gn[i] = load_piece((const T*)a.dy + row * a.lddy, c[i], cols);
    }
    mean_next = a.mean[row], rstd_next = a.rstd[row];
  };
  constexpr bool kAhead = CH <= 2;   // with more pieces the registers do not suffice
  if (kAhead && first < a.rows) fetch(first);
  for (int64_t row = first; row < a.rows; row += step, turn ^= 2) {
    if (!kAhead) fetch(row);
    uint4 zr[CH], gr[CH];
    const float mean = mean_next, rstd = rstd_next;
#pragma unroll
    for (int i = 0; i < CH; ++i) zr[i] = zn[i], gr[i] = gn[i];
    if (row + step < a.rows) fetch(row + step);   // on its way while this row is summed
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float z[V], g[V];
      unpack<T>(zr[i], z);
      unpack<T>(gr[i], g);   // zeros outside the row
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float h = (z[j] - mean) * rstd, gw = g[j] * w[i][j];
        dw[i][j] = fmaf(g[j], h, dw[i][j]);
        db[i][j] += g[j];
        s1 += gw;
        s2 = fmaf(gw, h, s2);
      }
    }
    if (!a.dx) continue;
    if (NW == 1) {
      s1 = warp_sum(s1), s2 = warp_sum(s2);
    } else {   // both sums behind one barrier; the next row's go to the other half
      s1 = warp_sum(s1), s2 = warp_sum(s2);
      if ((threadIdx.x & 31) == 0) part[turn][warp] = s1, part[turn + 1][warp] = s2;
      __syncthreads();
      s1 = s2 = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) s1 += part[turn][i], s2 += part[turn + 1][i];
    }
    s1 *= inv, s2 *= inv;
    T* dx = (T*)a.dx + row * a.cols;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float z[V], g[V], d[V], up[V];
      unpack<T>(zr[i], z);
      unpack<T>(gr[i], g);
      if (a.dz) unpack<T>(load_piece((const T*)a.dz + row * a.lddz, c[i], cols), up);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float h = (z[j] - mean) * rstd;
        d[j] = rstd * (fmaf(g[j], w[i][j], -s1) - h * s2);
        if (a.dz) d[j] += up[j];
      }
      store_piece(dx, c[i], cols, d);
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

template <typename T, typename W, int NW, int CH>
int forward_rows(const HpNormForward& a, bool ragged, cudaStream_t s) {
  constexpr int kThreads = kThreadsOf<NW>, kGroups = kThreads / (32 * NW);
  static const int per_sm = resident(norm_forward_rows<T, W, NW, CH>, kThreads, 0);
  norm_forward_rows<T, W, NW, CH><<<ctas_for(a.rows, kGroups, per_sm, ragged), kThreads, 0, s>>>(a, ragged);
  return cudaGetLastError();
}
template <typename T, typename W, int NW, int CH>
int backward_rows(const HpNormBackward& a, bool ragged, cudaStream_t s) {
  constexpr int kThreads = kThreadsOf<NW>, kGroups = kThreads / (32 * NW);
  const int smem = kGroups > 1 ? (int)(8 * a.cols) : 0;
  static const int per_sm = resident(norm_backward_rows<T, W, NW, CH>, kThreads, kGroups > 1 ? 8 * 32 * CH * kPiece<T> : 0);
  const unsigned grid = ctas_for(a.rows, kGroups, per_sm, ragged);
  norm_backward_rows<T, W, NW, CH><<<grid, kThreads, smem, s>>>(a, ragged);
  if (!a.dweight && !a.dbias) return cudaGetLastError();
  const int rc = cudaGetLastError();
  return rc ? rc : column_sums((const float*)a.workspace, (int)grid, 2 * a.cols, a.cols, a.dweight, a.dbias, (int)a.wtype, s);
}

#define BY_SPLIT(call)                          \
  switch (p.warps * 8 + p.pieces) {             \
    case 1 * 8 + 1: return call(1, 1);          \
    case 1 * 8 + 2: return call(1, 2);          \
    case 4 * 8 + 1: return call(4, 1);          \
    case 4 * 8 + 2: return call(4, 2);          \
    case 8 * 8 + 2: return call(8, 2);          \
    case 16 * 8 + 2: return call(16, 2);        \
    case 16 * 8 + 4: return call(16, 4);        \
    default: break;                             \
  }

template <typename T, typename W>
int forward(const HpNormForward& a, cudaStream_t s) {
  Rows r(sizeof(T));
  r.add(a.x, a.ldx);
  r.add(a.residual, a.ldr);
  r.add(a.y, a.cols);
  r.add(a.z, a.cols);
  if (r.alike) {
    const Split p = split_of<T>(a.cols, r.ragged());
#define CALL(nw, ch) forward_rows<T, W, nw, ch>(a, r.ragged(), s)
    BY_SPLIT(CALL)
#undef CALL
  }
  norm_forward_kernel<T><<<(unsigned)a.rows, 256, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T, typename W>
int backward(const HpNormBackward& a, cudaStream_t s) {
  Rows r(sizeof(T));
  r.add(a.z, a.ldz);
  r.add(a.dy, a.lddy);
  r.add(a.dz, a.lddz);
  r.add(a.dx, a.cols);
  if (r.alike && a.rows) {
    const Split p = split_of<T>(a.cols, r.ragged());
#define CALL(nw, ch) backward_rows<T, W, nw, ch>(a, r.ragged(), s)
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

#define BY_TYPE(fn)                                                                              \
  a->type == HP_F32    ? fn<float, float>(*a, s)                                                 \
  : a->type == HP_BF16 ? (a->wtype == HP_F32 ? fn<__nv_bfloat16, float>(*a, s)                   \
                                             : fn<__nv_bfloat16, __nv_bfloat16>(*a, s))          \
                       : (a->wtype == HP_F32 ? fn<__half, float>(*a, s) : fn<__half, __half>(*a, s))

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
