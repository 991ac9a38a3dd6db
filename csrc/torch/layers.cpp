// PyTorch binding of the layer operators on CUDA tensors: extension module `_layers`.
//
// Autograd nodes in C++: a layer norm of one sentence takes 8 us on the GPU, and as a Python
// autograd.Function it took 120 us on the host, forward and backward.  Arguments have been
// checked by the caller (hipress_b200/ops/layers.py); what is done here is layout (rows, pitches,
// copies where tiles cannot be fetched), allocation and the calls of the CUDA library, whose
// functions bind() hands over.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/utils/pybind.h>

#include "hipress/capi.h"
#include "hipress/layers.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library {
  int (*norm_forward)(const HpNormForward*, void*);
  int (*norm_backward)(const HpNormBackward*, void*);
  uint64_t (*norm_workspace)(int64_t, int64_t);
  int (*product)(const HpProduct*, void*);
  uint64_t (*product_workspace)(int64_t, int64_t, int64_t);
  int (*slope)(const HpSlope*, void*);
  uint64_t (*slope_workspace)(int64_t, int64_t);
  int (*attention_forward)(const HpAttention*, void*);
  int (*attention_backward)(const HpAttention*, void*);
  const char* (*error_string)(int);
} lib;

const struct {
  const char* name;
  void** slot;
} kSymbols[] = {{"hp_cuda_norm_forward", (void**)&lib.norm_forward},
                {"hp_cuda_norm_backward", (void**)&lib.norm_backward},
                {"hp_cuda_norm_workspace", (void**)&lib.norm_workspace},
                {"hp_cuda_product", (void**)&lib.product},
                {"hp_cuda_product_workspace", (void**)&lib.product_workspace},
                {"hp_cuda_slope", (void**)&lib.slope},
                {"hp_cuda_slope_workspace", (void**)&lib.slope_workspace},
                {"hp_cuda_attention_forward", (void**)&lib.attention_forward},
                {"hp_cuda_attention_backward", (void**)&lib.attention_backward},
                {"hp_cuda_error_string", (void**)&lib.error_string}};

void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, ": ", lib.error_string(rc), " (", rc, ")"); }

int type_of(at::ScalarType t) { return t == at::kFloat ? HP_F32 : t == at::kBFloat16 ? HP_BF16 : HP_F16; }
int type_of(const Tensor& t) { return t.defined() ? type_of(t.scalar_type()) : HP_F32; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
Tensor scratch(uint64_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
using Maybe = std::optional<Tensor>;
Tensor get(const Maybe& t) { return t ? *t : Tensor(); }
bool wanted(const Tensor& t) { return t.defined() && t.requires_grad(); }
// Whether a node is needed.  Tangents (forward mode) are refused: a tensor may have one without
// requiring a gradient, and would lose it.
template <typename... Ts>
bool differentiable(const char* what, const Ts&... t) {
  TORCH_CHECK(!((t.defined() && t._fw_grad(0).defined()) || ...), what, ": forward mode differentiation is not supported");
  return at::GradMode::is_enabled() && (wanted(t) || ...);
}
// Whether an argument of a node wants its gradient.  A node counts the tensors that are there:
// `present` has a bit for each tensor argument.
bool wants(AutogradContext* ctx, int64_t present, int i) {
  int edge = 0;
  for (int k = 0; k < i; ++k) edge += present >> k & 1;
  return (present >> i & 1) && ctx->needs_input_grad(edge);
}
// A backward pass whose results have no graph.  Where one is wanted (create_graph) they say so when they
// are differentiated by what they were made from (the inputs, and the gradients that came in), whether
// or not these gradients have a graph themselves.  What is handed on unchanged keeps the graph that it has.
variable_list first_order(variable_list (*gradients)(AutogradContext*, const variable_list&), AutogradContext* ctx,
                          const variable_list& grads) {
  variable_list out;
  {
    at::NoGradGuard guard;
    out = gradients(ctx, grads);
  }
  if (!at::GradMode::is_enabled()) return out;
  torch::autograd::edge_list made_from = torch::autograd::get_current_node()->next_edges();
  for (const Tensor& g : grads)
    if (wanted(g)) made_from.push_back(torch::autograd::impl::gradient_edge(g));
  const auto refused = std::make_shared<torch::autograd::Error>("a gradient of a layer operator cannot be differentiated",
                                                                std::move(made_from));
  for (Tensor& g : out) {
    bool same = !g.defined();
    for (const Tensor& x : grads) same = same || (x.defined() && g.is_same(x));
    if (!same) torch::autograd::set_history(g = g.detach(), refused);
  }
  return out;
}

// A saved tensor as it comes back.  Hooks may have kept it elsewhere, and return it in strides of
// their own, so that whoever takes it lays it out anew; what the kernels read must still be all there.
Tensor kept(const Tensor& t, const Tensor& grad, at::ScalarType type, at::IntArrayRef sizes, const char* what) {
  TORCH_CHECK(t.defined() && t.device() == grad.device() && t.scalar_type() == type && t.sizes() == sizes, what,
              ": a saved tensor came back as another");
  return t;
}

// As a matrix whose rows are dense; a copy only where there is no such view.
Tensor rows_of(const Tensor& x) {
  int64_t rows = 1;   // counted: of no elements they cannot be divided by the columns
  for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
  Tensor m = x.dim() == 2 ? x : x.reshape({rows, x.size(-1)});
  return m.stride(1) == 1 || m.size(1) == 1 ? m : m.contiguous();
}
// of one row there is no second to be reached, and its stride may be anything
int64_t pitch(const Tensor& m) { return !m.defined() ? 0 : m.size(0) > 1 ? m.stride(0) : m.size(1); }

// ------------------------------------------------------------------ layer norm
struct Norm {
  Tensor y, z, kept, stats;   // kept: what was normalised, for the backward pass
};

Norm norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, double eps) {
  Norm n;
  const Tensor x2 = rows_of(x), r2 = residual.defined() ? rows_of(residual) : residual, w = dense(weight), b = dense(bias);
  n.y = at::empty(x.sizes(), x.options());
  if (residual.defined()) n.z = at::empty(x.sizes(), x.options());
  n.stats = at::empty({2, x2.size(0)}, x.options().dtype(at::kFloat));
  HpNormForward a = {};
  a.x = ptr(x2), a.residual = ptr(r2), a.weight = ptr(w), a.bias = ptr(b), a.y = ptr(n.y), a.z = ptr(n.z);
  a.mean = (float*)ptr(n.stats), a.rstd = a.mean + x2.size(0);
  a.rows = x2.size(0), a.cols = x2.size(1), a.ldx = pitch(x2), a.ldr = pitch(r2);
  a.type = type_of(x), a.wtype = type_of(w.defined() ? w : b), a.eps = eps;
  check(lib.norm_forward(&a, stream()), "layer_norm");
  // the result itself, of which autograd knows that it is one; a view of it would hold its node, which
  // holds the view
  n.kept = n.z.defined() ? n.z : x.dim() == 2 ? x2 : x2.view(x.sizes());
  return n;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& w, const Maybe& b, const Maybe& r, double eps) {
    const Tensor weight = get(w), bias = get(b), residual = get(r);
    ctx->saved_data["present"] = (int64_t)(1 | weight.defined() << 1 | bias.defined() << 2 | residual.defined() << 3);
    Norm n = norm_forward(x, weight, bias, residual, eps);
    ctx->save_for_backward({n.kept, weight, n.stats});
    ctx->saved_data["sizes"] = x.sizes();
    ctx->saved_data["type"] = (int64_t)(weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : at::kFloat);
    ctx->set_materialize_grads(false);
    return n.z.defined() ? variable_list{n.y, n.z} : variable_list{n.y};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return first_order(gradients, ctx, grads);
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor dy = grads[0], dz = grads.size() > 1 ? grads[1] : Tensor(), any = dy.defined() ? dy : dz;
    if (!any.defined()) return variable_list(5);
    c10::cuda::CUDAGuard guard(any.device());
    const int64_t present = ctx->saved_data["present"].toInt();
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    const Tensor z = rows_of(kept(saved[0], any, any.scalar_type(), sizes, "layer_norm"));
    const bool need_x = wants(ctx, present, 0), need_w = wants(ctx, present, 1), need_b = wants(ctx, present, 2),
               need_r = wants(ctx, present, 3);
    const int64_t rows = z.size(0), cols = z.size(1);
    const auto wide = z.options().dtype((at::ScalarType)ctx->saved_data["type"].toInt());
    const Tensor stats = dense(kept(saved[2], any, at::kFloat, {2, rows}, "layer_norm"));
    const Tensor weight = present & 2 ? dense(kept(saved[1], any, wide.dtype().toScalarType(), {cols}, "layer_norm")) : Tensor();
    if (!dy.defined())   // only the sum was used further on
      return {need_x ? dz : Tensor(), need_w ? at::zeros({cols}, wide) : Tensor(), need_b ? at::zeros({cols}, wide) : Tensor(),
              need_r ? dz : Tensor(), Tensor()};
    const Tensor g = rows_of(dy), up = dz.defined() ? rows_of(dz) : dz;
    Tensor dx, dw, db, ws;
    if (need_x || need_r) dx = at::empty(sizes, z.options());
    if (need_w) dw = at::empty({cols}, wide);
    if (need_b) db = at::empty({cols}, wide);
    if (need_w || need_b) ws = scratch(lib.norm_workspace(rows, cols), z);
    HpNormBackward a = {};
    a.z = ptr(z), a.dy = ptr(g), a.dz = ptr(up), a.weight = ptr(weight);
    a.mean = (const float*)ptr(stats), a.rstd = a.mean + rows;
    a.dx = ptr(dx), a.dweight = ptr(dw), a.dbias = ptr(db), a.workspace = ptr(ws);
    a.rows = rows, a.cols = cols, a.ldz = pitch(z), a.lddy = pitch(g), a.lddz = pitch(up);
    a.type = type_of(z), a.wtype = type_of(wide.dtype().toScalarType());
    check(lib.norm_backward(&a, stream()), "layer_norm backward");
    return {need_x ? dx : Tensor(), dw, db, need_r ? dx : Tensor(), Tensor()};
  }
};

std::pair<Tensor, Maybe> layer_norm(const Tensor& x, const Maybe& weight, const Maybe& bias, const Maybe& residual, double eps) {
  c10::cuda::CUDAGuard guard(x.device());
  const Tensor w = get(weight), b = get(bias), r = get(residual);
  if (differentiable("layer_norm", x, w, b, r)) {
    variable_list out = LayerNorm::apply(x, weight, bias, residual, eps);
    return {out[0], out.size() > 1 ? Maybe(out[1]) : Maybe()};
  }
  Norm n = norm_forward(x, w, b, r, eps);
  return {n.y, n.z.defined() ? Maybe(n.z) : Maybe()};
}

// ---------------------------------------------------------------------- linear
// Whether tiles of a matrix can be fetched: rows on 16-byte boundaries.
bool tiled(const Tensor& m) {
  return m.stride(1) == 1 && (uintptr_t)m.data_ptr() % 16 == 0 && (m.size(0) <= 1 || m.stride(0) % 8 == 0);
}
Tensor operand(const Tensor& m, at::ScalarType type) {
  if (m.scalar_type() == type && tiled(m)) return m;
  return at::empty({m.size(0), (m.size(1) + 7) / 8 * 8}, m.options().dtype(type)).narrow(1, 0, m.size(1)).copy_(m);
}

Tensor product(const Tensor& a, const Tensor& b, int64_t m, int64_t n, int64_t k, bool a_k, bool b_k, at::IntArrayRef sizes,
               at::ScalarType type, const Tensor& bias = {}, const Tensor& residual = {}, const Tensor& pre = {}, int act = 0) {
  const Tensor y = at::empty(sizes, a.options().dtype(type)), ws = scratch(lib.product_workspace(m, n, k), a);
  HpProduct p = {};
  p.a = ptr(a), p.b = ptr(b), p.bias = ptr(bias), p.residual = ptr(residual), p.y = ptr(y), p.pre = ptr(pre);
  p.workspace = ptr(ws), p.m = m, p.n = n, p.k = k, p.lda = pitch(a), p.ldb = pitch(b), p.ldy = n, p.ldr = pitch(residual);
  p.a_kmajor = a_k, p.b_kmajor = b_k, p.type = type_of(a), p.ytype = type_of(type), p.btype = type_of(bias), p.act = act;
  check(lib.product(&p, stream()), "linear");
  return y;
}

struct Product {
  Tensor y, x, w, pre;
};
Product linear_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, int64_t act, bool keep) {
  Product f;
  const Tensor x2 = rows_of(x), r2 = residual.defined() ? rows_of(residual) : residual;
  const int64_t m = x2.size(0), k = x2.size(1), n = weight.size(0);
  f.x = operand(x2, x.scalar_type());
  f.w = operand(weight, x.scalar_type());
  if (act && keep) f.pre = at::empty({m, n}, x.options());
  std::vector<int64_t> sizes = x.sizes().vec();
  sizes.back() = n;
  f.y = product(f.x, f.w, m, n, k, true, true, sizes, x.scalar_type(), dense(bias), r2, f.pre, (int)act);
  return f;
}

struct Linear : torch::autograd::Function<Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& b, const Maybe& r, int64_t act) {
    const Tensor bias = get(b), residual = get(r);
    ctx->saved_data["present"] = (int64_t)(3 | bias.defined() << 2 | residual.defined() << 3);
    Product f = linear_forward(x, weight, bias, residual, act, true);
    ctx->save_for_backward({f.x, f.w, f.pre});
    ctx->saved_data["act"] = act;
    ctx->saved_data["sizes"] = x.sizes();
    ctx->saved_data["wtype"] = (int64_t)weight.scalar_type();
    ctx->saved_data["btype"] = (int64_t)(bias.defined() ? bias.scalar_type() : at::kFloat);
    return f.y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return first_order(gradients, ctx, grads);
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    c10::cuda::CUDAGuard guard(grads[0].device());
    const Tensor dy = rows_of(grads[0]);
    const int64_t m = dy.size(0), n = dy.size(1), act = ctx->saved_data["act"].toInt();
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    const int64_t k = sizes.back();
    const auto type = dy.scalar_type();
    const Tensor x = operand(kept(saved[0], dy, type, {m, k}, "linear"), type);
    const Tensor w = operand(kept(saved[1], dy, type, {n, k}, "linear"), type);
    const Tensor pre = act ? rows_of(kept(saved[2], dy, type, {m, n}, "linear")) : Tensor();
    const int64_t present = ctx->saved_data["present"].toInt();
    const bool need_x = wants(ctx, present, 0), need_w = wants(ctx, present, 1), need_b = wants(ctx, present, 2);
    Tensor g = dy, dx, dw, db;
    // rows that a tile copy cannot start at are laid out anew, as is what an activation changes
    const bool anew = act || !tiled(dy);
    if (anew) g = at::empty({m, (n + 7) / 8 * 8}, x.options()).narrow(1, 0, n);
    if (anew || need_b) {
      const auto btype = (at::ScalarType)ctx->saved_data["btype"].toInt();
      if (need_b) db = at::empty({n}, x.options().dtype(btype));
      const Tensor ws = need_b ? scratch(lib.slope_workspace(m, n), x) : Tensor();
      HpSlope a = {};
      a.dy = ptr(dy), a.pre = ptr(pre), a.g = anew ? ptr(g) : nullptr, a.dbias = ptr(db), a.workspace = ptr(ws);
      a.rows = m, a.cols = n, a.lddy = pitch(dy), a.ldpre = pitch(pre), a.ldg = pitch(g);
      a.type = type_of(x), a.btype = type_of(btype), a.act = act;
      check(lib.slope(&a, stream()), "linear backward");
    }
    if (need_x) dx = product(g, w, m, k, n, true, false, sizes, type);
    if (need_w) dw = product(g, x, n, k, m, false, false, {n, k}, (at::ScalarType)ctx->saved_data["wtype"].toInt());
    return {dx, dw, db, wants(ctx, present, 3) ? grads[0] : Tensor(), Tensor()};
  }
};

Tensor linear(const Tensor& x, const Tensor& weight, const Maybe& bias, const Maybe& residual, int64_t act) {
  c10::cuda::CUDAGuard guard(x.device());
  const Tensor b = get(bias), r = get(residual);
  if (differentiable("linear", x, weight, b, r)) return Linear::apply(x, weight, bias, residual, act);
  return linear_forward(x, weight, b, r, act, false).y;
}

// ------------------------------------------------------------------- attention
// The tensor itself where tiles of it can be fetched (the last axis dense, everything on 16-byte
// boundaries), else a copy.
Tensor tileable(const Tensor& x) {
  const auto s = x.strides();
  if (s[3] == 1 && (uintptr_t)x.data_ptr() % 16 == 0 && (s[0] | s[1] | s[2]) % 8 == 0 && s[0] > 0 && s[1] > 0 && s[2] > 0) return x;
  return x.clone(at::MemoryFormat::Contiguous);
}
void put(const Tensor& x, int64_t& b, int64_t& s, int64_t& h) { b = x.stride(0), s = x.stride(1), h = x.stride(2); }

HpAttention block(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse, const Tensor& mask,
                  bool causal, double scale) {
  HpAttention a = {};
  a.q = ptr(q), a.k = ptr(k), a.v = ptr(v), a.o = ptr(o), a.lse = (float*)ptr(lse), a.key_mask = (const uint8_t*)ptr(mask);
  a.batch = q.size(0), a.sq = q.size(1), a.sk = k.size(1), a.heads = q.size(2), a.kv_heads = k.size(2), a.dim = q.size(3);
  put(q, a.q_b, a.q_s, a.q_h), put(k, a.k_b, a.k_s, a.k_h), put(v, a.v_b, a.v_s, a.v_h), put(o, a.o_b, a.o_s, a.o_h);
  a.mask_b = mask.defined() ? mask.stride(0) : 0;
  a.type = type_of(q), a.causal = causal, a.scale = scale;
  return a;
}
Tensor mask_rows(const Tensor& mask) { return !mask.defined() || mask.stride(1) == 1 ? mask : mask.contiguous(); }

std::pair<Tensor, Tensor> attention_forward(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& mask0, bool causal,
                                            double scale) {
  const Tensor o = at::empty(q0.sizes(), q0.options());
  const Tensor lse = at::empty({q0.size(0), q0.size(2), q0.size(1)}, q0.options().dtype(at::kFloat));
  const Tensor q = tileable(q0), k = tileable(k0), v = tileable(v0), mask = mask_rows(mask0);
  const HpAttention a = block(q, k, v, o, lse, mask, causal, scale);
  check(lib.attention_forward(&a, stream()), "attention");
  return {o, lse};
}
void attention_backward(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& o0, const Tensor& lse0, const Tensor& do0,
                        const Tensor& mask0, bool causal, double scale, const Tensor& dq, const Tensor& dk, const Tensor& dv) {
  const Tensor q = tileable(q0), k = tileable(k0), v = tileable(v0), o = tileable(o0), d_o = tileable(do0), lse = dense(lse0),
               mask = mask_rows(mask0);
  const Tensor delta = at::empty({q.size(0), q.size(2), 10, (q.size(1) + 127) / 128 * 128}, q.options().dtype(at::kFloat));
  HpAttention a = block(q, k, v, o, lse, mask, causal, scale);
  a.d_o = ptr(d_o), a.dq = ptr(dq), a.dk = ptr(dk), a.dv = ptr(dv), a.delta = (float*)ptr(delta);
  put(d_o, a.do_b, a.do_s, a.do_h), put(dq, a.dq_b, a.dq_s, a.dq_h), put(dk, a.dk_b, a.dk_s, a.dk_h), put(dv, a.dv_b, a.dv_s, a.dv_h);
  check(lib.attention_backward(&a, stream()), "attention backward");
}

void keep(AutogradContext* ctx, bool causal, double scale, const Tensor& lse) {
  ctx->saved_data["causal"] = causal;
  ctx->saved_data["scale"] = scale;
  ctx->mark_non_differentiable({lse});
  ctx->set_materialize_grads(false);
}

// o, lse and the mask, if there is one, as they come back
void kept_results(const Tensor& o, const Tensor& lse, const Tensor& mask, const Tensor& d_o, int64_t keys, const char* what) {
  kept(o, d_o, d_o.scalar_type(), d_o.sizes(), what);
  kept(lse, d_o, at::kFloat, {d_o.size(0), d_o.size(2), d_o.size(1)}, what);
  if (mask.defined()) kept(mask, d_o, at::kBool, {d_o.size(0), keys}, what);
}

struct Attention : torch::autograd::Function<Attention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& m,
                               bool causal, double scale) {
    const Tensor mask = get(m);
    auto [o, lse] = attention_forward(q, k, v, mask, causal, scale);
    ctx->save_for_backward({q, k, v, o, lse, mask});
    keep(ctx, causal, scale, lse);
    return {o, lse};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return first_order(gradients, ctx, grads);
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(6);
    if (!grads[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    c10::cuda::CUDAGuard guard(grads[0].device());
    const Tensor& d_o = grads[0];
    const int64_t keys = s[1].dim() == 4 ? s[1].size(1) : 0, heads = s[1].dim() == 4 && s[1].size(2) ? s[1].size(2) : 1;
    TORCH_CHECK(d_o.size(2) % heads == 0, "attention: a saved tensor came back as another");
    kept(s[0], d_o, d_o.scalar_type(), d_o.sizes(), "attention");
    for (int i = 1; i < 3; ++i) kept(s[i], d_o, d_o.scalar_type(), {d_o.size(0), keys, heads, d_o.size(3)}, "attention");
    kept_results(s[3], s[4], s[5], d_o, keys, "attention");
    for (int i = 0; i < 3; ++i) out[i] = at::empty(s[i].sizes(), s[i].options());
    attention_backward(s[0], s[1], s[2], s[3], s[4], grads[0], s[5], ctx->saved_data["causal"].toBool(),
                       ctx->saved_data["scale"].toDouble(), out[0], out[1], out[2]);
    for (int i = 0; i < 3; ++i)
      if (!ctx->needs_input_grad(i)) out[i] = Tensor();
    return out;
  }
};

struct SelfAttention : torch::autograd::Function<SelfAttention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& qkv, const Maybe& m, bool causal, double scale) {
    const Tensor mask = get(m);
    auto [o, lse] = attention_forward(qkv.select(2, 0), qkv.select(2, 1), qkv.select(2, 2), mask, causal, scale);
    ctx->save_for_backward({qkv, o, lse, mask});
    keep(ctx, causal, scale, lse);
    return {o, lse};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return first_order(gradients, ctx, grads);
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    c10::cuda::CUDAGuard guard(grads[0].device());
    const auto size = grads[0].sizes();
    const Tensor qkv = kept(s[0], grads[0], grads[0].scalar_type(), {size[0], size[1], 3, size[2], size[3]}, "self_attention");
    kept_results(s[1], s[2], s[3], grads[0], size[1], "self_attention");
    const Tensor d = at::empty(qkv.sizes(), qkv.options());
    attention_backward(qkv.select(2, 0), qkv.select(2, 1), qkv.select(2, 2), s[1], s[2], grads[0], s[3],
                       ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(), d.select(2, 0), d.select(2, 1),
                       d.select(2, 2));
    out[0] = d;
    return out;
  }
};

std::pair<Tensor, Tensor> attention(const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& mask, bool causal, double scale) {
  c10::cuda::CUDAGuard guard(q.device());
  if (differentiable("attention", q, k, v)) {
    variable_list out = Attention::apply(q, k, v, mask, causal, scale);
    return {out[0], out[1]};
  }
  return attention_forward(q, k, v, get(mask), causal, scale);
}
std::pair<Tensor, Tensor> self_attention(const Tensor& qkv, const Maybe& mask, bool causal, double scale) {
  c10::cuda::CUDAGuard guard(qkv.device());
  if (differentiable("self_attention", qkv)) {
    variable_list out = SelfAttention::apply(qkv, mask, causal, scale);
    return {out[0], out[1]};
  }
  return attention_forward(qkv.select(2, 0), qkv.select(2, 1), qkv.select(2, 2), get(mask), causal, scale);
}

std::vector<std::string> symbols() {
  std::vector<std::string> s;
  for (const auto& k : kSymbols) s.push_back(k.name);
  return s;
}
void bind(const std::unordered_map<std::string, uintptr_t>& addresses) {
  for (const auto& k : kSymbols) *k.slot = (void*)addresses.at(k.name);
}

}  // namespace

PYBIND11_MODULE(_layers, m) {
  using release = pybind11::call_guard<pybind11::gil_scoped_release>;   // a full launch queue blocks
  m.def("symbols", symbols, "symbol names bind() takes");
  m.def("bind", bind, "bind({symbol: address}): the CUDA library to call");
  m.def("layer_norm", layer_norm, release(), "(x, weight, bias, residual, eps) -> (y, z or None)");
  m.def("linear", linear, release(), "(x, weight, bias, residual, activation) -> y");
  m.def("attention", attention, release(), "(q, k, v, key_mask, causal, scale) -> (o, lse)");
  m.def("self_attention", self_attention, release(), "(qkv, key_mask, causal, scale) -> (o, lse)");
}
