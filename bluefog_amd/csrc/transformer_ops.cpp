// Copyright 2026. Licensed under the Apache License, Version 2.0.
//
// Torch side of the transformer training operators: argument checks, strides,
// workspaces, and the autograd nodes. The nodes are C++ so that a small call
// costs microseconds and the backward pass runs without the interpreter. The
// operators are known to torch's dispatcher, so that a trace records a call of
// theirs and not the allocation that it returns.

#include <torch/extension.h>

#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <optional>

#include "transformer_kernels.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int code_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return 0;
    case at::kHalf:
      return 2;
    case at::kBFloat16:
      return 3;
    default:
      TORCH_CHECK_TYPE(false, "bluefog_amd transformer kernels support f32/f16/bf16, got ",
                       t.scalar_type());
  }
}

hipStream_t stream_of(const Tensor& t) {
  return at::hip::getCurrentHIPStream(t.device().index()).stream();
}

void check(hipError_t e, const char* what) {
  TORCH_CHECK(e == hipSuccess, "bluefog_amd ", what, ": ", hipGetErrorString(e));
}

// Torch may leave a negation to whoever reads the memory (the imaginary part of a
// conjugate): a copy then.
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

// Saved tensors as the kernels read them: hooks may bring back the same values in
// another layout (torch.autograd.graph.saved_tensors_hooks).
Tensor dense(const Tensor& t) { return !t.defined() || t.is_contiguous() ? t : t.contiguous(); }

// A fake tensor, or one whose storage was freed, is a GPU tensor with nowhere to
// read: a kernel would fault.
void with_memory(const char* what, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->numel() || t->const_data_ptr(), "bluefog_amd ", what,
                                " needs tensors with memory: no fake ones, none whose storage was freed");
}

// The kernels take no tangents along: the derivative would silently be lost.
void no_tangents(const char* what, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), "bluefog_amd ", what,
                                " has no forward-mode derivative");
}

// The kernels' results have no graph of their own: a second derivative
// through them would silently be zero.
void once_only(const char* what, const Tensor& grad) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "bluefog_amd ", what,
              " is differentiable once: create_graph=True is not supported");
  no_tangents(what, {&grad});
}

BfDropout dropout_args(const Tensor& seed_tensor, int64_t seed, int64_t offset,
                       double p) {
  BfDropout d{};
  d.seed_ptr = seed_tensor.defined() ? seed_tensor.const_data_ptr<int64_t>() : nullptr;
  d.seed = static_cast<uint64_t>(seed);
  d.offset = static_cast<uint32_t>(offset);
  const int64_t t = static_cast<int64_t>(p * 65536 + 0.5);
  d.threshold = static_cast<uint32_t>(t < 65535 ? t : 65535);
  d.scale = static_cast<float>(65536.0 / (65536.0 - d.threshold));
  return d;
}

void check_dropout(const Tensor& like, const Tensor& seed, int64_t offset, double p) {
  TORCH_CHECK_VALUE(p >= 0 && p < 1, "dropout probability has to be in [0, 1), got ", p);
  TORCH_CHECK_VALUE(offset >= 0 && offset <= 0xFFFFFFFFll, "offset has to be in [0, 2^32), got ", offset);
  if (!seed.defined()) return;
  TORCH_CHECK_VALUE(seed.scalar_type() == at::kLong && seed.numel() == 1 && seed.device() == like.device(),
                    "seed has to be an int or one int64 on the input's device");
}

bool any_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------

// Whether rows and heads of t are dense along the last dimension, rows are
// less than 2^22 values apart (a tile's places fit 32 bits) and, where a head
// fills whole 16-byte accesses, start on one. Other tensors are copied, dense
// ones that start elsewhere too: a copy is cheaper than element-wise reads by
// every tile. Dense rows, of at most 65535 heads of 128, fit as well.
Tensor readable(const Tensor& t) {
  const int64_t e = t.element_size(), d = t.size(2);
  bool ok = (t.stride(2) == 1 || d == 1) && (t.size(0) == 1 || t.stride(0) <= 1 << 22);
  if (d * e % 16 == 0) {
    ok = ok && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
    for (int i = 0; i < 2; ++i) ok = ok && (t.size(i) == 1 || t.stride(i) * e % 16 == 0);
  }
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

BfAttnArgs attn_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu, const Tensor& table,
                     double scale, bool causal, const BfDropout& drop) {
  BfAttnArgs a{};
  a.q = q.const_data_ptr();
  a.k = k.const_data_ptr();
  a.v = v.const_data_ptr();
  a.cu = cu.const_data_ptr<int>();
  a.table = table.defined() ? table.const_data_ptr<int>() : nullptr;
  a.seqs = static_cast<int>(cu.numel()) - 1;
  a.rows = static_cast<int>(q.size(0));
  a.heads = static_cast<int>(q.size(1));
  a.kv_heads = static_cast<int>(k.size(1));
  a.dim = static_cast<int>(q.size(2));
  a.q_row = q.stride(0), a.q_head = q.stride(1);
  a.k_row = k.stride(0), a.k_head = k.stride(1);
  a.v_row = v.stride(0), a.v_head = v.stride(1);
  a.scale = static_cast<float>(scale);
  a.causal = causal;
  a.vec = q.size(2) * q.element_size() % 16 == 0;
  a.drop = drop;
  return a;
}

Tensor attn_partial(BfAttnArgs& a, const at::TensorOptions& f32) {
  const long n = bf_attn_partial_floats(&a);
  if (n == 0) return Tensor();
  Tensor t = at::empty({n}, f32);
  a.partial = t.data_ptr<float>();
  return t;
}

Tensor attn_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu,
                    double scale, bool causal, const BfDropout& drop, Tensor* lse, Tensor* rest, Tensor* kept_table) {
  c10::DeviceGuard guard(q.device());
  Tensor out = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
  if (lse) *lse = at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat));
  if (rest && q.scalar_type() != at::kFloat) *rest = at::empty(out.sizes(), q.options());
  if (out.numel() == 0) return out;
  with_memory("packed_attention", {&out});  // a mode may make new tensors fake
  BfAttnArgs a = attn_args(q, k, v, cu, Tensor(), scale, causal, drop);
  Tensor table;
  if (const int n = bf_attn_table_ints(&a)) {
    table = at::empty({n}, cu.options());
    a.table = table.data_ptr<int>();
    check(bf_attn_table(&a, table.data_ptr<int>(), stream_of(q)), "packed_attention");
  }
  if (kept_table) *kept_table = table;
  a.o = out.data_ptr();
  a.lse = lse ? lse->data_ptr<float>() : nullptr;
  a.rest = rest && rest->defined() ? rest->data_ptr() : nullptr;
  a.key_slices = bf_attn_key_slices(&a, code_of(q));
  a.query_slices = 1;
  const Tensor partial = attn_partial(a, q.options().dtype(at::kFloat));
  check(bf_attn_fwd(&a, code_of(q), stream_of(q)), "packed_attention");
  return out;
}

struct PackedAttention : torch::autograd::Function<PackedAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const Tensor& cu, const std::optional<Tensor>& seed_tensor, double scale,
                        bool causal, double p, int64_t seed, int64_t offset) {
    Tensor lse, rest, table;
    const Tensor st = seed_tensor.value_or(Tensor());
    Tensor out = attn_forward(q, k, v, cu, scale, causal, dropout_args(st, seed, offset, p), &lse, &rest, &table);
    ctx->save_for_backward({q, k, v, cu, st, out, lse, rest, table});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("packed_attention", grads[0]);
    variable_list none(10);
    if (!grads[0].defined()) return none;
    const variable_list s = ctx->get_saved_variables();
    with_memory("packed_attention backward", {&s[0], &s[1], &s[2], &s[3], &s[4], &s[5], &s[6], &s[7], &s[8], &grads[0]});
    const Tensor q = readable(s[0]), k = readable(s[1]), v = readable(s[2]), cu = dense(s[3]), &seed_tensor = s[4];
    const Tensor out = dense(s[5]), lse = dense(s[6]), rest = dense(s[7]), table = dense(s[8]);
    c10::DeviceGuard guard(q.device());
    const bool need_dkv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    const Tensor dout = readable(plain(grads[0]));
    Tensor dq = at::empty(out.sizes(), out.options());
    Tensor dk = at::empty(k.sizes(), k.options(), at::MemoryFormat::Contiguous);
    Tensor dv = at::empty(v.sizes(), v.options(), at::MemoryFormat::Contiguous);
    with_memory("packed_attention backward", {&dq});
    if (out.numel()) {
      Tensor delta = at::empty(lse.sizes(), lse.options());
      BfAttnArgs a = attn_args(q, k, v, cu, table, ctx->saved_data["scale"].toDouble(),
                               ctx->saved_data["causal"].toBool(),
                               dropout_args(seed_tensor, ctx->saved_data["seed"].toInt(),
                                            ctx->saved_data["offset"].toInt(),
                                            ctx->saved_data["p"].toDouble()));
      a.out = out.const_data_ptr();
      a.rest = rest.defined() ? const_cast<void*>(rest.const_data_ptr()) : nullptr;
      a.dout = dout.const_data_ptr();
      a.do_row = dout.stride(0), a.do_head = dout.stride(1);
      a.lse = lse.data_ptr<float>();
      a.delta = delta.data_ptr<float>();
      a.dq = dq.data_ptr();
      a.dk = dk.data_ptr();
      a.dv = dv.data_ptr();
      a.key_slices = bf_attn_key_slices(&a, code_of(q));
      a.query_slices = need_dkv ? bf_attn_query_slices(&a, code_of(q)) : 1;
      const Tensor partial = attn_partial(a, lse.options());
      check(bf_attn_bwd(&a, code_of(q), need_dkv, stream_of(q)), "packed_attention backward");
    }
    none[0] = dq, none[1] = dk, none[2] = dv;
    return none;
  }
};

Tensor packed_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu,
                        double scale, bool causal, double p, const std::optional<Tensor>& seed_tensor,
                        int64_t seed, int64_t offset) {
  const Tensor st = seed_tensor.value_or(Tensor());
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "q, k and v have to be [tokens, heads, dim]");
  TORCH_CHECK_VALUE(q.is_cuda() && k.device() == q.device() && v.device() == q.device() && cu.device() == q.device(),
                    "q, k, v and cu_seqlens have to be on one GPU");
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                   "q, k and v have to be of one type");
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(2) == q.size(2),
                    "shapes of q, k and v do not match");
  TORCH_CHECK_VALUE(q.size(2) >= 1 && q.size(2) <= 128, "head dimensions of 1 to 128 are supported, got ", q.size(2));
  TORCH_CHECK_VALUE(k.size(1) >= 1 && q.size(1) >= 1 && q.size(1) % k.size(1) == 0 && q.size(1) <= 65535,
                    "the number of query heads has to be a multiple of the key/value heads");
  TORCH_CHECK_VALUE(q.size(0) <= 0x7FFF0000ll, "too many tokens");
  TORCH_CHECK_TYPE(cu.scalar_type() == at::kInt, "cu_seqlens has to be int32");
  TORCH_CHECK_VALUE(cu.dim() == 1 && cu.numel() >= 1 && cu.is_contiguous(), "cu_seqlens has to be a dense vector");
  TORCH_CHECK_VALUE(cu.numel() <= 1 << 24, "too many sequences");
  TORCH_CHECK_VALUE(static_cast<float>(scale) > 0 && std::isfinite(static_cast<float>(scale)),
                    "scale has to be positive and finite in 32 bits, got ", scale);
  check_dropout(q, st, offset, p);
  const int code = code_of(q);
  const bool grad = any_grad({&q, &k, &v});
  BfAttnArgs size{};
  size.seqs = static_cast<int>(cu.numel()) - 1, size.rows = static_cast<int>(q.size(0)), size.dim = static_cast<int>(q.size(2));
  size.heads = static_cast<int>(q.size(1)), size.kv_heads = static_cast<int>(k.size(1));
  TORCH_CHECK_VALUE(bf_attn_fits(&size, code, grad), "too many sequences or tokens for ", q.size(1), " heads: ", cu.numel() - 1,
                    " sequences, ", q.size(0), " tokens");
  with_memory("packed_attention", {&q, &k, &v, &cu, &st});
  no_tangents("packed_attention", {&q, &k, &v});
  const Tensor rq = readable(plain(q)), rk = readable(plain(k)), rv = readable(plain(v));
  if (grad) return PackedAttention::apply(rq, rk, rv, cu, seed_tensor, scale, causal, p, seed, offset);
  return attn_forward(rq, rk, rv, cu, scale, causal, dropout_args(st, seed, offset, p), nullptr, nullptr, nullptr);
}

// ---------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------

// t as rows of its last dimension: the tensor to read (a copy where its rows
// are not dense or not one stride apart) and that stride
std::pair<Tensor, int64_t> as_rows(const Tensor& t) {
  const int64_t n = t.dim(), width = t.size(n - 1);
  if (t.is_contiguous()) return {t, width};
  bool ok = t.stride(n - 1) == 1 || width == 1;
  int64_t inner = -1, stride = width;  // innermost dimension of rows
  for (int64_t i = n - 2; i >= 0 && ok; --i) {
    if (t.size(i) == 1) continue;
    if (inner < 0) stride = t.stride(i);
    else ok = t.stride(i) == t.stride(inner) * t.size(inner);
    inner = i;
  }
  if (ok) return {t, stride};
  return {t.contiguous(), width};
}

BfNormArgs norm_args(const Tensor& x, const Tensor& weight, const Tensor& bias,
                     double eps, const BfDropout& drop) {
  BfNormArgs a{};
  a.width = static_cast<int>(x.size(-1));
  a.rows = x.numel() / a.width;
  a.weight = weight.defined() ? weight.const_data_ptr() : nullptr;
  a.bias = bias.defined() ? bias.const_data_ptr() : nullptr;
  const Tensor& w = weight.defined() ? weight : bias;
  a.weight_f32 = !w.defined() || w.scalar_type() == at::kFloat;
  a.eps = static_cast<float>(eps);
  a.drop = drop;
  return a;
}

Tensor norm_forward(const Tensor& x, const Tensor& r, const Tensor& weight, const Tensor& bias,
                    double eps, const BfDropout& drop, Tensor* mean, Tensor* rstd) {
  c10::DeviceGuard guard(x.device());
  const Tensor& kind = r.defined() ? r : x;
  Tensor y = at::empty(x.sizes(), kind.options(), at::MemoryFormat::Contiguous);
  BfNormArgs a = norm_args(x, weight, bias, eps, drop);
  if (mean) {
    *mean = at::empty({a.rows}, x.options().dtype(at::kFloat));
    *rstd = at::empty({a.rows}, x.options().dtype(at::kFloat));
    a.mean = mean->data_ptr<float>();
    a.rstd = rstd->data_ptr<float>();
  }
  if (a.rows == 0) return y;
  with_memory("layer_norm", {&y});  // a mode may make new tensors fake
  const auto [rx, x_row] = as_rows(x);
  a.x = rx.const_data_ptr(), a.x_row = x_row;
  Tensor hold;
  if (r.defined()) {
    const auto [rr, r_row] = as_rows(r);
    hold = rr;
    a.r = rr.const_data_ptr(), a.r_row = r_row;
  }
  a.y = y.data_ptr();
  check(bf_norm_fwd(&a, code_of(x), code_of(kind), stream_of(x)), "layer_norm");
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  using Optional = std::optional<Tensor>;

  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Optional& residual, const Optional& weight_,
                        const Optional& bias_, const Optional& seed_tensor, double eps, double p,
                        int64_t seed, int64_t offset) {
    const Tensor none;
    const Tensor r = residual.value_or(none), weight = weight_.value_or(none), bias = bias_.value_or(none),
                 st = seed_tensor.value_or(none);
    Tensor mean, rstd;
    Tensor y = norm_forward(x, r, weight, bias, eps, dropout_args(st, seed, offset, p), &mean, &rstd);
    ctx->save_for_backward({x, r, weight, bias, st, mean, rstd});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("layer_norm", grads[0]);
    variable_list got(9);
    if (!grads[0].defined()) return got;
    const variable_list s = ctx->get_saved_variables();
    with_memory("layer_norm backward", {&s[0], &s[1], &s[2], &s[3], &s[4], &s[5], &s[6], &grads[0]});
    const Tensor &x = s[0], &r = s[1], &seed_tensor = s[4];
    const Tensor weight = dense(s[2]), bias = dense(s[3]), mean = dense(s[5]), rstd = dense(s[6]);
    c10::DeviceGuard guard(x.device());
    BfNormArgs a = norm_args(x, weight, bias, ctx->saved_data["eps"].toDouble(),
                             dropout_args(seed_tensor, ctx->saved_data["seed"].toInt(),
                                          ctx->saved_data["offset"].toInt(), ctx->saved_data["p"].toDouble()));
    const Tensor& kind = r.defined() ? r : x;
    const auto dense = at::MemoryFormat::Contiguous;
    // an absent tensor has no edge
    const int r_edge = 1, w_edge = r_edge + r.defined(), b_edge = w_edge + weight.defined();
    if (ctx->needs_input_grad(0)) got[0] = at::empty(x.sizes(), x.options(), dense);
    if (r.defined() && ctx->needs_input_grad(r_edge)) {
      // without dropout both branches of the join have the same gradient
      const bool same = !a.drop.threshold && got[0].defined() && r.scalar_type() == x.scalar_type();
      got[1] = same ? got[0] : at::empty(r.sizes(), r.options(), dense);
    }
    if (weight.defined() && ctx->needs_input_grad(w_edge)) got[2] = at::empty_like(weight);
    if (bias.defined() && ctx->needs_input_grad(b_edge)) got[3] = at::empty_like(bias);
    with_memory("layer_norm backward", {&got[0], &got[1], &got[2], &got[3]});
    if (a.rows == 0) {
      for (int i = 2; i < 4; ++i)
        if (got[i].defined()) got[i].zero_();
      return got;
    }
    const auto [rx, x_row] = as_rows(x);
    const auto [rdy, dy_row] = as_rows(plain(grads[0]));
    a.x = rx.const_data_ptr(), a.x_row = x_row;
    a.dy = rdy.const_data_ptr(), a.dy_row = dy_row;
    Tensor hold;
    if (r.defined()) {
      const auto [rr, r_row] = as_rows(r);
      hold = rr;
      a.r = rr.const_data_ptr(), a.r_row = r_row;
    }
    a.mean = mean.data_ptr<float>();
    a.rstd = rstd.data_ptr<float>();
    a.dx = got[0].defined() ? got[0].data_ptr() : nullptr;
    a.dr = got[1].defined() && !got[1].is_same(got[0]) ? got[1].data_ptr() : nullptr;
    a.dweight = got[2].defined() ? got[2].data_ptr() : nullptr;
    a.dbias = got[3].defined() ? got[3].data_ptr() : nullptr;
    Tensor partial;
    if (a.dweight || a.dbias) {
      partial = at::empty({bf_norm_partial_floats(a.rows, a.width)},
                          x.options().dtype(at::kFloat));
      a.partial = partial.data_ptr<float>();
    }
    check(bf_norm_bwd(&a, code_of(x), code_of(kind), stream_of(x)), "layer_norm backward");
    return got;
  }
};

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps,
                  const std::optional<Tensor>& residual, double p, const std::optional<Tensor>& seed_tensor,
                  int64_t seed, int64_t offset) {
  Tensor r = residual.value_or(Tensor());
  const Tensor st = seed_tensor.value_or(Tensor());
  Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 1 << 26,
                    "layer_norm needs a GPU tensor with a last dimension of 1 to 2^26");
  code_of(x);
  for (const Tensor* t : {&w, &b}) {
    if (!t->defined()) continue;
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == x.size(-1) && t->device() == x.device(),
                      "weight and bias have to be vectors of the last dimension");
    TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat || t->scalar_type() == x.scalar_type(),
                     "weight and bias have to be f32 or of the input's type");
  }
  TORCH_CHECK_TYPE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(),
                   "weight and bias have to be of one type");
  if (r.defined()) {
    TORCH_CHECK_VALUE(r.sizes() == x.sizes() && r.device() == x.device(), "residual has to have the input's shape");
    TORCH_CHECK_TYPE(r.scalar_type() == at::kFloat || r.scalar_type() == x.scalar_type(),
                     "residual has to be f32 or of the input's type");
  }
  TORCH_CHECK_VALUE((eps == 0 || static_cast<float>(eps) > 0) && std::isfinite(static_cast<float>(eps)),
                    "eps has to be finite and not negative, in 32 bits, got ", eps);
  check_dropout(x, st, offset, p);
  with_memory("layer_norm", {&x, &r, &w, &b, &st});
  no_tangents("layer_norm", {&x, &r, &w, &b});
  const bool grad = any_grad({&x, &r, &w, &b});
  const Tensor in = plain(x);
  r = plain(r);
  if (w.defined()) w = plain(w).contiguous();
  if (b.defined()) b = plain(b).contiguous();
  if (grad) {
    const auto given = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    return LayerNorm::apply(in, given(r), given(w), given(b), given(st), eps, p, seed, offset);
  }
  return norm_forward(in, r, w, b, eps, dropout_args(st, seed, offset, p), nullptr, nullptr);
}

// ---------------------------------------------------------------------------
// dropout
// ---------------------------------------------------------------------------

Tensor masked(const Tensor& x, const BfDropout& d) {
  c10::DeviceGuard guard(x.device());
  const Tensor in = x.contiguous();
  Tensor y = at::empty(in.sizes(), in.options(), at::MemoryFormat::Contiguous);
  with_memory("counter_dropout", {&in, &y});
  if (in.numel())
    check(bf_dropout(y.data_ptr(), in.const_data_ptr(), in.numel(), code_of(in), &d, stream_of(in)),
          "counter_dropout");
  return y;
}

struct CounterDropout : torch::autograd::Function<CounterDropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& seed_tensor,
                        double p, int64_t seed, int64_t offset) {
    const Tensor st = seed_tensor.value_or(Tensor());
    ctx->save_for_backward({st});
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    return masked(x, dropout_args(st, seed, offset, p));
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("counter_dropout", grads[0]);
    variable_list got(5);
    if (!grads[0].defined()) return got;
    const Tensor seed_tensor = ctx->get_saved_variables()[0];
    with_memory("counter_dropout backward", {&seed_tensor});
    got[0] = masked(plain(grads[0]), dropout_args(seed_tensor, ctx->saved_data["seed"].toInt(),
                                           ctx->saved_data["offset"].toInt(), ctx->saved_data["p"].toDouble()));
    return got;
  }
};

Tensor counter_dropout(const Tensor& x, double p, const std::optional<Tensor>& seed_tensor, int64_t seed,
                       int64_t offset) {
  const Tensor st = seed_tensor.value_or(Tensor());
  TORCH_CHECK_VALUE(x.is_cuda(), "counter_dropout needs a GPU tensor");
  check_dropout(x, st, offset, p);
  code_of(x);
  TORCH_CHECK_VALUE(x.numel() <= bf_dropout_most(), "counter_dropout takes at most ", bf_dropout_most(), " values, got ", x.numel());
  with_memory("counter_dropout", {&x, &st});
  no_tangents("counter_dropout", {&x});
  const bool grad = any_grad({&x});
  if (grad) return CounterDropout::apply(plain(x), seed_tensor, p, seed, offset);
  return masked(plain(x), dropout_args(st, seed, offset, p));
}

// the operator `name` as torch's dispatcher calls it, with F's arguments
template <auto F>
struct Dispatched;
template <typename... Args, Tensor (*F)(Args...)>
struct Dispatched<F> {
  static void bind(py::module& m, const char* name, const char* doc) {
    const auto op =
        c10::Dispatcher::singleton().findSchemaOrThrow((std::string("bluefog_amd::") + name).c_str(), "").typed<Tensor(Args...)>();
    m.def(name, [op](Args... args) { return op.call(args...); }, py::call_guard<py::gil_scoped_release>(), doc);
  }
};

}  // namespace

TORCH_LIBRARY(bluefog_amd, m) {
  m.def("packed_attention(Tensor q, Tensor k, Tensor v, Tensor cu_seqlens, float scale, bool causal, float dropout_p, "
        "Tensor? seed_tensor, int seed, int offset) -> Tensor", &packed_attention);
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, Tensor? residual, float dropout_p, "
        "Tensor? seed_tensor, int seed, int offset) -> Tensor", &layer_norm);
  m.def("counter_dropout(Tensor x, float p, Tensor? seed_tensor, int seed, int offset) -> Tensor", &counter_dropout);
}

void bf_register_transformer_ops(py::module& m) {
  Dispatched<&packed_attention>::bind(m, "packed_attention", "softmax(scale q k^T) v inside packed sequences");
  Dispatched<&layer_norm>::bind(m, "layer_norm", "LayerNorm(residual + dropout(x))");
  Dispatched<&counter_dropout>::bind(m, "counter_dropout", "x * keep / (1 - p), the mask from a counter");
}
