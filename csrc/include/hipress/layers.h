// C ABI of the layer operators: layer norm, the matrix product with an epilogue and
// attention.  Every function takes a structure of its arguments and the stream.
//
// Return values as in capi.h.  Kernels that wait (for copies or matrix products of their
// own CTA) bound every wait but that for room in tensor memory, which the CTAs that hold it end
// (tcgen05.cuh says why); one that expired is reported by the next call on that device with
// HP_ERR_TIMEOUT.
#pragma once
#include <stdint.h>

#define HP_ERR_TIMEOUT (-4)  // an earlier kernel gave up on one of its waits: its results are invalid

// element types
#define HP_F32 0
#define HP_BF16 1
#define HP_F16 2

// activations of HpProduct and HpSlope
#define HP_ACT_NONE 0
#define HP_ACT_RELU 1
#define HP_ACT_GELU 2       // p Phi(p)
#define HP_ACT_GELU_TANH 3  // its tanh form

#ifdef __cplusplus
extern "C" {
#endif

// z = x (+ residual, rounded to the type); y = (z - mean) rstd weight + bias, by rows of
// `cols` elements.  Outputs are dense; inputs have a pitch in elements.
typedef struct {
  const void* x;
  const void* residual;  // or NULL
  const void* weight;    // or NULL (1)
  const void* bias;      // or NULL (0)
  void* y;
  void* z;               // the sum, only with a residual
  float* mean;           // [rows]
  float* rstd;           // [rows]
  int64_t rows, cols, ldx, ldr;
  int64_t type, wtype;   // of x, residual, y, z; of weight and bias
  double eps;
} HpNormForward;
int hp_cuda_norm_forward(const HpNormForward* a, void* stream);

// dx (the gradient of z), dweight and dbias
typedef struct {
  const void* z;
  const void* dy;
  const void* dz;        // gradient that reaches z on another way, or NULL
  const void* weight;
  const float* mean;
  const float* rstd;
  void* dx;              // or NULL
  void* dweight;         // or NULL
  void* dbias;           // or NULL
  void* workspace;       // hp_cuda_norm_workspace(rows, cols) bytes
  int64_t rows, cols, ldz, lddy, lddz;
  int64_t type, wtype;
} HpNormBackward;
int hp_cuda_norm_backward(const HpNormBackward* a, void* stream);
uint64_t hp_cuda_norm_workspace(int64_t rows, int64_t cols);

// One product out[m, n] = sum_k a(m, k) b(n, k) with its epilogue: p = out + bias;
// y = act(p) + residual.  An operand is stored along k (kmajor 1: row m, pitch lda) or along
// its own index (kmajor 0: row k, pitch lda); both bases and pitches on 16-byte boundaries.  y
// has the operands' type, or is in 32 bits, without an epilogue.
typedef struct {
  const void* a;
  const void* b;
  const void* bias;      // [n] or NULL
  const void* residual;  // [m, n] or NULL
  void* y;               // [m, n], pitch ldy
  void* pre;             // p, where the backward pass needs it; pitch ldy; or NULL
  void* workspace;       // hp_cuda_product_workspace(m, n, k) bytes
  int64_t m, n, k;
  int64_t lda, ldb, ldy, ldr;
  int64_t a_kmajor, b_kmajor;
  int64_t type, ytype, btype;  // of a, b, residual and pre; of y; of bias
  int64_t act;
} HpProduct;
int hp_cuda_product(const HpProduct* a, void* stream);
uint64_t hp_cuda_product_workspace(int64_t m, int64_t n, int64_t k);

// g = dy act'(pre), with a pitch of its own, and dbias = its sums over the rows.  Without an
// activation and with g NULL only the sums.
typedef struct {
  const void* dy;
  const void* pre;
  void* g;
  void* dbias;           // or NULL
  void* workspace;       // hp_cuda_slope_workspace(rows, cols) bytes
  int64_t rows, cols, lddy, ldpre, ldg;
  int64_t type, btype, act;
} HpSlope;
int hp_cuda_slope(const HpSlope* a, void* stream);
uint64_t hp_cuda_slope_workspace(int64_t rows, int64_t cols);

// Attention, forward (o, lse) and backward (dq, dk, dv from d_o, o and lse).  Tensors are
// [batch, length, heads, dim] with the last axis dense; strides in elements.
typedef struct {
  const void *q, *k, *v;
  void* o;
  float* lse;               // [batch, heads, sq], natural logarithm
  const uint8_t* key_mask;  // [batch, sk], nonzero: may be seen; or NULL
  const void* d_o;
  void *dq, *dk, *dv;
  float* delta;             // backward: workspace, [batch, heads, 10, sq rounded up to 128]
  int64_t batch, sq, sk, heads, kv_heads, dim;
  int64_t q_b, q_s, q_h, k_b, k_s, k_h, v_b, v_s, v_h, o_b, o_s, o_h, do_b, do_s, do_h;
  int64_t dq_b, dq_s, dq_h, dk_b, dk_s, dk_h, dv_b, dv_s, dv_h;
  int64_t mask_b;
  int64_t type, causal;
  double scale;
} HpAttention;
int hp_cuda_attention_forward(const HpAttention* a, void* stream);
int hp_cuda_attention_backward(const HpAttention* a, void* stream);

// A wait of the layer operators' kind that runs out after `limit_ns`, and one beside it, which then
// ends too; the nanoseconds that each took to two words of device memory.  For tests.
int hp_cuda_layer_wait_probe(uint64_t limit_ns, uint64_t* took, void* stream);

#ifdef __cplusplus
}
#endif
