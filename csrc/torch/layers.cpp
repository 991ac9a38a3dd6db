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
  int (*dropout)(const HpDrop*, void*);
  int (*norm_forward)(const HpNormForward*, void*);
  int (*norm_backward)(const HpNormBackward*, void*);
  uint64_t (*norm_workspace)(int64_t, int64_t);
  int (*product)(const HpProduct*, void*);
  uint64_t (*product_workspace)(int64_t, int64_t, int64_t);
  int (*slope)(const HpSlope*, void*);
  uint64_t (*slope_workspace)(int64_t, int64_t);
  int (*attention_forward)(const HpAttention*, void*);
  int (*attention_backward)(const HpAttention*, void*);
  int (*log_probs)(const HpLogProbs*, void*);
  uint64_t (*log_probs_workspace)(int64_t);
  int (*log_probs_backward)(const HpLogProbsBackward*, void*);
  const char* (*error_string)(int);
} lib;

const struct {
  const char* name;
  void** slot;
} kSymbols[] = {{"hp_cuda_dropout", (void**)&lib.dropout},
                {"hp_cuda_norm_forward", (void**)&lib.norm_forward},
                {"hp_cuda_norm_backward", (void**)&lib.norm_backward},
                {"hp_cuda_norm_workspace", (void**)&lib.norm_workspace},
                {"hp_cuda_product", (void**)&lib.product},
                {"hp_cuda_product_workspace", (void**)&lib.product_workspace},
                {"hp_cuda_slope", (void**)&lib.slope},
                {"hp_cuda_slope_workspace", (void**)&lib.slope_workspace},
                {"hp_cuda_attention_forward", (void**)&lib.attention_forward},
                {"hp_cuda_attention_backward", (void**)&lib.attention_backward},
                {"hp_cuda_log_probs", (void**)&lib.log_probs},
                {"hp_cuda_log_probs_workspace", (void**)&lib.log_probs_workspace},
                {"hp_cuda_log_probs_backward", (void**)&lib.log_probs_backward},
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

// Which elements a dropout keeps.  The seed is a number, or a tensor of one that is read when a kernel
// runs; the backward pass wants the same, and autograd sees to it that nobody has changed it in between.
struct Random {
  Tensor seed_at;
  int64_t seed = 0, site = 0, keep = 0;
  Random() = default;
  Random(const Maybe& at, int64_t number, int64_t site_of, int64_t keep_of)
      : seed_at(get(at)), seed(number), site(site_of), keep(keep_of) {}
  HpDropout args() const { return {seed_at.defined() ? (const int64_t*)seed_at.data_ptr() : nullptr, seed, site, keep}; }
  void save(AutogradContext* ctx) const {
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["site"] = site;
    ctx->saved_data["keep"] = keep;
    ctx->saved_data["moving"] = seed_at.defined();
  }
  // as save() has left it, with the tensor as it comes back
  static Random kept_in(AutogradContext* ctx, const Tensor& at, const Tensor& grad, const char* what) {
    Random r;
    r.keep = ctx->saved_data["keep"].toInt();
    if (!r.keep) return r;
    r.seed = ctx->saved_data["seed"].toInt(), r.site = ctx->saved_data["site"].toInt();
    if (ctx->saved_data["moving"].toBool()) {
      TORCH_CHECK(at.defined() && at.device() == grad.device() && at.scalar_type() == at::kLong && at.numel() == 1, what,
                  ": a saved tensor came back as another");
      r.seed_at = at;
    }
    return r;
  }
};

// As a matrix whose rows are dense; a copy only where there is no such view.
Tensor rows_of(const Tensor& x) {
  int64_t rows = 1;   // counted: of no elements they cannot be divided by the columns
  for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
  Tensor m = x.dim() == 2 ? x : x.reshape({rows, x.size(-1)});
  return m.stride(1) == 1 || m.size(1) == 1 ? m : m.contiguous();
}
// of one row there is no second to be reached, and its stride may be anything
int64_t pitch(const Tensor& m) { return !m.defined() ? 0 : m.size(0) > 1 ? m.stride(0) : m.size(1); }

// --------------------------------------------------------------------- dropout
Tensor drop(const Tensor& x0, const Tensor& residual0, const Random& random) {
  const Tensor x = dense(x0), residual = dense(residual0), y = at::empty(x.sizes(), x.options());
  const HpDrop a = {ptr(x), ptr(residual), ptr(y), x.numel(), type_of(x), random.args()};
  check(lib.dropout(&a, stream()), "dropout");
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& r, const Random& random) {
    const Tensor residual = get(r);
    ctx->saved_data["present"] = (int64_t)(1 | residual.defined() << 1);
    random.save(ctx);
    ctx->save_for_backward({random.seed_at});
    return drop(x, residual, random);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return first_order(gradients, ctx, grads);
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const int64_t present = ctx->saved_data["present"].toInt();
    c10::cuda::CUDAGuard guard(grads[0].device());
    Tensor dx;
    if (wants(ctx, present, 0))
      dx = drop(grads[0], Tensor(), Random::kept_in(ctx, ctx->get_saved_variables()[0], grads[0], "dropout"));
    return {dx, wants(ctx, present, 1) ? grads[0] : Tensor(), Tensor()};
  }
};

Tensor dropout(const Tensor& x, const Maybe& residual, const Maybe& seed_at, int64_t seed, int64_t site, int64_t keep) {
  c10::cuda::CUDAGuard guard(x.device());
  const Random random(seed_at, seed, site, keep);
  const Tensor r = get(residual);
  if (differentiable("dropout", x, r)) return Dropout::apply(x, residual, random);
  return drop(x, r, random);
}

// ------------------------------------------------------------------ layer norm
struct Norm {
  Tensor y, z, kept, stats;   // kept: what was normalised, for the backward pass
};

Norm norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, double eps,
                  const Random& random) {
  Norm n;
  Tensor x2 = rows_of(x), r2 = residual.defined() ? rows_of(residual) : residual;
  if (random.keep) x2 = x2.contiguous(), r2 = r2.contiguous();
  const Tensor w = dense(weight), b = dense(bias);
  n.y = at::empty(x.sizes(), x.options());
  if (residual.defined()) n.z = at::empty(x.sizes(), x.options());
  n.stats = at::empty({2, x2.size(0)}, x.options().dtype(at::kFloat));
  HpNormForward a = {};
  a.x = ptr(x2), a.residual = ptr(r2), a.weight = ptr(w), a.bias = ptr(b), a.y = ptr(n.y), a.z = ptr(n.z);
  a.mean = (float*)ptr(n.stats), a.rstd = a.mean + x2.size(0);
  a.rows = x2.size(0), a.cols = x2.size(1), a.ldx = pitch(x2), a.ldr = pitch(r2);
  a.type = type_of(x), a.wtype = type_of(w.defined() ? w : b), a.eps = eps, a.drop = random.args();
  check(lib.norm_forward(&a, stream()), "layer_norm");
  // the result itself, of which autograd knows that it is one; a view of it would hold its node, which
  // holds the view
  n.kept = n.z.defined() ? n.z : x.dim() == 2 ? x2 : x2.view(x.sizes());
  return n;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& w, const Maybe& b, const Maybe& r, double eps,
                               const Random& random) {
    const Tensor weight = get(w), bias = get(b), residual = get(r);
    ctx->saved_data["present"] = (int64_t)(1 | weight.defined() << 1 | bias.defined() << 2 | residual.defined() << 3);
    Norm n = norm_forward(x, weight, bias, residual, eps, random);
    ctx->save_for_backward({n.kept, weight, n.stats, random.seed_at});
    random.save(ctx);
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
    if (!any.defined()) return variable_list(6);
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
    const Random random = Random::kept_in(ctx, saved[3], any, "layer_norm");
    if (!dy.defined())   // only the sum was used further on
      return {!need_x ? Tensor() : random.keep ? drop(dz, Tensor(), random) : dz, need_w ? at::zeros({cols}, wide) : Tensor(),
              need_b ? at::zeros({cols}, wide) : Tensor(), need_r ? dz : Tensor(), Tensor(), Tensor()};
    const Tensor g = rows_of(dy), up = dz.defined() ? rows_of(dz) : dz;
    Tensor dx, dropped, dw, db, ws;
    if (random.keep ? need_r : need_x || need_r) dx = at::empty(sizes, z.options());
    if (random.keep && need_x) dropped = at::empty(sizes, z.options());
    if (need_w) dw = at::empty({cols}, wide);
    if (need_b) db = at::empty({cols}, wide);
    if (need_w || need_b) ws = scratch(lib.norm_workspace(rows, cols), z);
    HpNormBackward a = {};
    a.z = ptr(z), a.dy = ptr(g), a.dz = ptr(up), a.weight = ptr(weight);
    a.mean = (const float*)ptr(stats), a.rstd = a.mean + rows;
    a.dx = ptr(dx), a.dweight = ptr(dw), a.dbias = ptr(db), a.workspace = ptr(ws);
    a.rows = rows, a.cols = cols, a.ldz = pitch(z), a.lddy = pitch(g), a.lddz = pitch(up);
    a.type = type_of(z), a.wtype = type_of(wide.dtype().toScalarType());
    // of neither gradient nothing is dropped
    if (dx.defined() || dropped.defined()) a.dropped = ptr(dropped), a.drop = random.args();
    check(lib.norm_backward(&a, stream()), "layer_norm backward");
    return {!need_x ? Tensor() : random.keep ? dropped : dx, dw, db, need_r ? dx : Tensor(), Tensor(), Tensor()};
  }
};

std::pair<Tensor, Maybe> layer_norm(const Tensor& x, const Maybe& weight, const Maybe& bias, const Maybe& residual, double eps,
                                    const Maybe& seed_at, int64_t seed, int64_t site, int64_t keep) {
  c10::cuda::CUDAGuard guard(x.device());
  const Random random(seed_at, seed, site, keep);
  const Tensor w = get(weight), b = get(bias), r = get(residual);
  if (differentiable("layer_norm", x, w, b, r)) {
    variable_list out = LayerNorm::apply(x, weight, bias, residual, eps, random);
    return {out[0], out.size() > 1 ? Maybe(out[1]) : Maybe()};
  }
  Norm n = norm_forward(x, w, b, r, eps, random);
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
                  bool causal, double scale, const Random& random) {
  HpAttention a = {};
  a.q = ptr(q), a.k = ptr(k), a.v = ptr(v), a.o = ptr(o), a.lse = (float*)ptr(lse), a.key_mask = (const uint8_t*)ptr(mask);
  a.batch = q.size(0), a.sq = q.size(1), a.sk = k.size(1), a.heads = q.size(2), a.kv_heads = k.size(2), a.dim = q.size(3);
  put(q, a.q_b, a.q_s, a.q_h), put(k, a.k_b, a.k_s, a.k_h), put(v, a.v_b, a.v_s, a.v_h), put(o, a.o_b, a.o_s, a.o_h);
  a.mask_b = mask.defined() ? mask.stride(0) : 0;
  a.type = type_of(q), a.causal = causal, a.scale = scale, a.drop = random.args();
  return a;
}
Tensor mask_rows(const Tensor& mask) { return !mask.defined() || mask.stride(1) == 1 ? mask : mask.contiguous(); }

std::pair<Tensor, Tensor> attention_forward(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& mask0, bool causal,
                                            double scale, const Random& random) {
  const Tensor o = at::empty(q0.sizes(), q0.options());
  const Tensor lse = at::empty({q0.size(0), q0.size(2), q0.size(1)}, q0.options().dtype(at::kFloat));
  const Tensor q = tileable(q0), k = tileable(k0), v = tileable(v0), mask = mask_rows(mask0);
  const HpAttention a = block(q, k, v, o, lse, mask, causal, scale, random);
  check(lib.attention_forward(&a, stream()), "attention");
  return {o, lse};
}
void attention_backward(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& o0, const Tensor& lse0, const Tensor& do0,
                        const Tensor& mask0, bool causal, double scale, const Random& random, const Tensor& dq, const Tensor& dk,
                        const Tensor& dv) {
  const Tensor q = tileable(q0), k = tileable(k0), v = tileable(v0), o = tileable(o0), d_o = tileable(do0), lse = dense(lse0),
               mask = mask_rows(mask0);
  const Tensor delta = at::empty({q.size(0), q.size(2), 10, (q.size(1) + 127) / 128 * 128}, q.options().dtype(at::kFloat));
  HpAttention a = block(q, k, v, o, lse, mask, causal, scale, random);
  a.d_o = ptr(d_o), a.dq = ptr(dq), a.dk = ptr(dk), a.dv = ptr(dv), a.delta = (float*)ptr(delta);
  put(d_o, a.do_b, a.do_s, a.do_h), put(dq, a.dq_b, a.dq_s, a.dq_h), put(dk, a.dk_b, a.dk_s, a.dk_h), put(dv, a.dv_b, a.dv_s, a.dv_h);
  check(lib.attention_backward(&a, stream()), "attention backward");
}

void keep(AutogradContext* ctx, bool causal, double scale, const Random& random, const Tensor& lse) {
  random.save(ctx);
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
                               bool causal, double scale, const Random& random) {
    const Tensor mask = get(m);
    auto [o, lse] = attention_forward(q, k, v, mask, causal, scale, random);
    ctx->save_for_backward({q, k, v, o, lse, mask, random.seed_at});
    keep(ctx, causal, scale, random, lse);
    return {o, lse};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return first_order(gradients, ctx, grads);
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(7);
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
                       ctx->saved_data["scale"].toDouble(), Random::kept_in(ctx, s[6], d_o, "attention"), out[0], out[1], out[2]);
    for (int i = 0; i < 3; ++i)
      if (!ctx->needs_input_grad(i)) out[i] = Tensor();
    return out;
  }
};

struct SelfAttention : torch::autograd::Function<SelfAttention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& qkv, const Maybe& m, bool causal, double scale, const Random& random) {
    const Tensor mask = get(m);
    auto [o, lse] = attention_forward(qkv.select(2, 0), qkv.select(2, 1), qkv.select(2, 2), mask, causal, scale, random);
    ctx->save_for_backward({qkv, o, lse, mask, random.seed_at});
    keep(ctx, causal, scale, random, lse);
    return {o, lse};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return first_order(gradients, ctx, grads);
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(5);
    if (!grads[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    c10::cuda::CUDAGuard guard(grads[0].device());
    const auto size = grads[0].sizes();
    const Tensor qkv = kept(s[0], grads[0], grads[0].scalar_type(), {size[0], size[1], 3, size[2], size[3]}, "self_attention");
    kept_results(s[1], s[2], s[3], grads[0], size[1], "self_attention");
    const Tensor d = at::empty(qkv.sizes(), qkv.options());
    attention_backward(qkv.select(2, 0), qkv.select(2, 1), qkv.select(2, 2), s[1], s[2], grads[0], s[3],
                       ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(),
                       Random::kept_in(ctx, s[4], grads[0], "self_attention"), d.select(2, 0), d.select(2, 1), d.select(2, 2));
    out[0] = d;
    return out;
  }
};

std::pair<Tensor, Tensor> attention(const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& mask, bool causal, double scale,
                                    const Maybe& seed_at, int64_t seed, int64_t site, int64_t keep) {
  c10::cuda::CUDAGuard guard(q.device());
  const Random random(seed_at, seed, site, keep);
  if (differentiable("attention", q, k, v)) {
    variable_list out = Attention::apply(q, k, v, mask, causal, scale, random);
    return {out[0], out[1]};
  }
  return attention_forward(q, k, v, get(mask), causal, scale, random);
}
std::pair<Tensor, Tensor> self_attention(const Tensor& qkv, const Maybe& mask, bool causal, double scale, const Maybe& seed_at,
                                         int64_t seed, int64_t site, int64_t keep) {
  c10::cuda::CUDAGuard guard(qkv.device());
  const Random random(seed_at, seed, site, keep);
  if (differentiable("self_attention", qkv)) {
    variable_list out = SelfAttention::apply(qkv, mask, causal, scale, random);
    return {out[0], out[1]};
  }
  return attention_forward(qkv.select(2, 0), qkv.select(2, 1), qkv.select(2, 2), get(mask), causal, scale, random);
}

// ----------------------------------------------------------- log probabilities
// Logits as rows of two strides: row r at (r / inner) outer + (r % inner) ld.  A copy only where
// there are more, or the columns are not side by side.
struct LogitRows {
  Tensor x;
  int64_t rows = 1, inner = 1, outer = 0, ld = 0, vocab;
  explicit LogitRows(const Tensor& t) : x(t), vocab(t.size(-1)) {
    if (!settle()) x = t.contiguous(), settle();
  }
  bool settle() {
    if (vocab > 1 && x.stride(-1) != 1) return false;
    rows = 1;
    for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
    inner = 1, outer = ld = vocab;
    int level = 0;   // of strides found, from the last axis on
    int64_t reach = 0;
    for (int64_t i = x.dim() - 2; i >= 0 && rows; --i) {
      if (x.size(i) == 1) continue;
      if (level == 0) ld = x.stride(i), inner = x.size(i), reach = ld * inner, level = 1;
      else if (x.stride(i) == reach && level == 1) inner *= x.size(i), reach *= x.size(i);
      else if (level == 1) outer = x.stride(i), reach = outer * x.size(i), level = 2;
      else if (x.stride(i) == reach) reach *= x.size(i);
      else return false;
    }
    return true;
  }
};

struct LogProbs {
  Tensor log_probs, entropy, top_log_probs, top_tokens, stats, loss, count;
};
LogProbs log_probs_forward(const Tensor& logits, const Tensor& tokens, int64_t ignored, int64_t top, bool entropy, bool loss, bool summed) {
  LogProbs f;
  const LogitRows x(logits);
  const Tensor t = dense(tokens);
  const auto wide = logits.options().dtype(at::kFloat);
  const auto sizes = logits.sizes().slice(0, logits.dim() - 1);
  HpLogProbs a = {};
  if (!loss) f.log_probs = at::empty(sizes, wide);
  if (entropy) f.entropy = at::empty(sizes, wide);
  if (top) {
    std::vector<int64_t> more = sizes.vec();
    more.push_back(top);
    f.top_log_probs = at::empty(more, wide), f.top_tokens = at::empty(more, logits.options().dtype(at::kLong));
  }
  f.stats = at::empty({x.rows, 2}, wide);
  Tensor ws;
  if (loss) f.loss = at::empty({}, wide), f.count = at::empty({}, wide), ws = scratch(lib.log_probs_workspace(x.rows), logits);
  a.logits = ptr(x.x), a.tokens = (const int64_t*)ptr(t), a.log_probs = (float*)ptr(f.log_probs), a.entropy = (float*)ptr(f.entropy);
  a.top_log_probs = (float*)ptr(f.top_log_probs), a.top_tokens = (int64_t*)ptr(f.top_tokens), a.stats = (float*)ptr(f.stats);
  a.loss = (float*)ptr(f.loss), a.count = (float*)ptr(f.count), a.workspace = ptr(ws);
  a.rows = x.rows, a.inner = x.inner, a.vocab = x.vocab, a.ld_outer = x.outer, a.ld = x.ld;
  a.type = type_of(logits), a.top = top, a.ignored = ignored, a.summed = summed;
  check(lib.log_probs(&a, stream()), loss ? "cross_entropy" : "token_log_probs");
  return f;
}
Tensor log_probs_backward(const Tensor& logits, const Tensor& tokens, const Tensor& stats, const Tensor& entropy, const Tensor& dlogp,
                          const Tensor& dentropy, const Tensor& count, int64_t ignored, bool loss) {
  const LogitRows x(logits);
  const Tensor t = dense(tokens), g = dense(dlogp), h = dense(dentropy), st = dense(stats), e = dense(entropy),
               d = at::empty(logits.sizes(), logits.options());
  HpLogProbsBackward a = {};
  a.logits = ptr(x.x), a.tokens = (const int64_t*)ptr(t), a.stats = (const float*)ptr(st), a.entropy = (const float*)ptr(e);
  a.dlog_probs = (const float*)ptr(g), a.dentropy = (const float*)ptr(h), a.count = (const float*)ptr(count), a.dlogits = ptr(d);
  a.rows = x.rows, a.inner = x.inner, a.vocab = x.vocab, a.ld_outer = x.outer, a.ld = x.ld;
  a.type = type_of(logits), a.ignored = ignored, a.one = loss, a.negative = loss;
  check(lib.log_probs_backward(&a, stream()), loss ? "cross_entropy backward" : "token_log_probs backward");
  return d;
}

// the logits, tokens and statistics that a node has kept, as they come back
void kept_rows(const variable_list& s, at::ScalarType type, at::IntArrayRef sizes, const Tensor& any, const char* what) {
  int64_t rows = 1;
  for (size_t i = 0; i + 1 < sizes.size(); ++i) rows *= sizes[i];
  kept(s[0], any, type, sizes, what);
  kept(s[1], any, at::kLong, sizes.slice(0, sizes.size() - 1), what);
  kept(s[2], any, at::kFloat, {rows, 2}, what);
}

struct TokenLogProbs : torch::autograd::Function<TokenLogProbs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, int64_t ignored, int64_t top, bool entropy) {
    LogProbs f = log_probs_forward(logits, tokens, ignored, top, entropy, false, false);
    ctx->save_for_backward({logits, tokens, f.stats, f.entropy});
    ctx->saved_data["ignored"] = ignored;
    ctx->saved_data["entropy"] = entropy;
    ctx->saved_data["type"] = (int64_t)logits.scalar_type();
    ctx->saved_data["sizes"] = logits.sizes();
    ctx->set_materialize_grads(false);
    variable_list out{f.log_probs};
    if (entropy) out.push_back(f.entropy);
    if (top) {
      ctx->mark_non_differentiable({f.top_log_probs, f.top_tokens});
      out.push_back(f.top_log_probs), out.push_back(f.top_tokens);
    }
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return first_order(gradients, ctx, grads);
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(5);
    const bool entropy = ctx->saved_data["entropy"].toBool();
    const Tensor dlogp = grads[0], dentropy = entropy ? grads[1] : Tensor(), any = dlogp.defined() ? dlogp : dentropy;
    if (!any.defined()) return out;
    c10::cuda::CUDAGuard guard(any.device());
    const auto s = ctx->get_saved_variables();
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    kept_rows(s, (at::ScalarType)ctx->saved_data["type"].toInt(), sizes, any, "token_log_probs");
    if (dentropy.defined()) kept(s[3], any, at::kFloat, at::IntArrayRef(sizes).slice(0, sizes.size() - 1), "token_log_probs");
    out[0] = log_probs_backward(s[0], s[1], s[2], dentropy.defined() ? s[3] : Tensor(), dlogp, dentropy, Tensor(),
                                ctx->saved_data["ignored"].toInt(), false);
    return out;
  }
};

struct CrossEntropy : torch::autograd::Function<CrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, int64_t ignored, bool summed) {
    LogProbs f = log_probs_forward(logits, labels, ignored, 0, false, true, summed);
    ctx->save_for_backward({logits, labels, f.stats, f.count});
    ctx->saved_data["ignored"] = ignored;
    ctx->saved_data["summed"] = summed;
    ctx->saved_data["type"] = (int64_t)logits.scalar_type();
    ctx->saved_data["sizes"] = logits.sizes();
    return f.loss;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return first_order(gradients, ctx, grads);
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    c10::cuda::CUDAGuard guard(grads[0].device());
    const auto s = ctx->get_saved_variables();
    kept_rows(s, (at::ScalarType)ctx->saved_data["type"].toInt(), ctx->saved_data["sizes"].toIntVector(), grads[0], "cross_entropy");
    kept(s[3], grads[0], at::kFloat, {}, "cross_entropy");
    return {log_probs_backward(s[0], s[1], s[2], Tensor(), grads[0], Tensor(), ctx->saved_data["summed"].toBool() ? Tensor() : s[3],
                               ctx->saved_data["ignored"].toInt(), true),
            Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Maybe, Maybe, Maybe> token_log_probs(const Tensor& logits, const Tensor& tokens, int64_t ignored, int64_t top, bool entropy) {
  c10::cuda::CUDAGuard guard(logits.device());
  if (differentiable("token_log_probs", logits)) {
    variable_list out = TokenLogProbs::apply(logits, tokens, ignored, top, entropy);
    const size_t tops = entropy ? 2 : 1;
    return {out[0], entropy ? Maybe(out[1]) : Maybe(), top ? Maybe(out[tops]) : Maybe(), top ? Maybe(out[tops + 1]) : Maybe()};
  }
  LogProbs f = log_probs_forward(logits, tokens, ignored, top, entropy, false, false);
  return {f.log_probs, entropy ? Maybe(f.entropy) : Maybe(), top ? Maybe(f.top_log_probs) : Maybe(), top ? Maybe(f.top_tokens) : Maybe()};
}
Tensor cross_entropy(const Tensor& logits, const Tensor& labels, int64_t ignored, bool summed) {
  c10::cuda::CUDAGuard guard(logits.device());
  if (differentiable("cross_entropy", logits)) return CrossEntropy::apply(logits, labels, ignored, summed);
  return log_probs_forward(logits, labels, ignored, 0, false, true, summed).loss;
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
  m.def("dropout", dropout, release(), "(x, residual, seed tensor, seed, site, keep) -> y");
  m.def("layer_norm", layer_norm, release(), "(x, weight, bias, residual, eps, seed tensor, seed, site, keep) -> (y, z or None)");
  m.def("linear", linear, release(), "(x, weight, bias, residual, activation) -> y");
  m.def("attention", attention, release(), "(q, k, v, key_mask, causal, scale, seed tensor, seed, site, keep) -> (o, lse)");
  m.def("self_attention", self_attention, release(), "(qkv, key_mask, causal, scale, seed tensor, seed, site, keep) -> (o, lse)");
  m.def("token_log_probs", token_log_probs, release(),
        "(logits, tokens, ignored, top, entropy) -> (log probabilities, entropy, top log probabilities, top tokens)");
  m.def("cross_entropy", cross_entropy, release(), "(logits, labels, ignored, summed) -> loss");
}
