// Bindings of the rotary, tree-attention and logits operators (see serve_ops.h).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <tuple>
#include <utility>
#include <vector>

#include "check.h"
#include "serve_ops.h"
#include "types.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

int code_of(const Tensor& t, const char* n) {
  switch (t.scalar_type()) {
    case torch::kFloat: return cob::kF32;
    case torch::kHalf: return cob::kF16;
    case torch::kBFloat16: return cob::kBF16;
    default: COB_CHECK(false, n, ": unsupported dtype ", std::string(c10::toString(t.scalar_type())));
  }
  return -1;
}

void ok(cudaError_t e, const char* what) { COB_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e)); }

cudaStream_t cur() { return at::cuda::getCurrentCUDAStream(); }

// what the kernels read through its pointer is the tensor's value: no pending negation, no memory given back (a sharded
// parameter between its uses) or never there
void has_memory(const Tensor& t, const char* n) {
  constexpr c10::DispatchKeySet kOther({c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor});
  const c10::TensorImpl* impl = t.unsafeGetTensorImpl();
  COB_CHECK(t.layout() == torch::kStrided && !(impl->key_set() & kOther).has_any(kOther) &&
                (t.numel() == 0 || impl->unsafe_storage().nbytes() > 0),
            n, " must be a strided tensor with memory of its values (a negated view: resolve_neg() first)");
}
void on_device(const Tensor& t, const char* n, const Tensor& ref) {
  COB_CHECK(t.is_cuda() && t.device() == ref.device(), n, " must be a CUDA tensor on the device of the first operand");
  has_memory(t, n);
}

// contiguous tensor of one type on the reference's device
void dense(const Tensor& t, const char* n, torch::ScalarType ty, const Tensor& ref) {
  on_device(t, n, ref);
  COB_CHECK(t.scalar_type() == ty, n, " must be ", std::string(c10::toString(ty)));
  COB_CHECK(t.is_contiguous(), n, " must be contiguous");
}

// the bytes that a tensor's elements reach
struct Span {
  uintptr_t lo = 0, hi = 0;
  Span() = default;
  explicit Span(const Tensor* t) {
    if (!t || t->numel() == 0) return;
    lo = reinterpret_cast<uintptr_t>(t->const_data_ptr());
    int64_t last = t->numel() - 1;
    if (!t->is_contiguous()) {
      const auto n = t->sizes(), s = t->strides();
      last = 0;
      for (size_t i = 0; i < n.size(); ++i) last += (n[i] - 1) * s[i];
    }
    hi = lo + (last + 1) * t->element_size();
  }
  bool meets(const Span& o) const { return lo < o.hi && o.lo < hi; }
};
bool overlap(const Tensor& a, const Tensor& b) { return Span(&a).meets(Span(&b)); }
// what a call writes lies apart from what it reads, and from whatever else it writes
void apart(std::initializer_list<const Tensor*> written, std::initializer_list<const Tensor*> read, const char* what) {
  Span w[4];
  int n = 0;
  for (const Tensor* t : written) {
    w[n] = Span(t);
    for (int i = 0; i < n; ++i) COB_CHECK(!w[n].meets(w[i]), what);
    ++n;
  }
  for (const Tensor* t : read) {
    const Span r(t);
    for (int i = 0; i < n; ++i) COB_CHECK(!w[i].meets(r), what);
  }
}
const Tensor* given(const OptTensor& t) { return t.has_value() ? &*t : nullptr; }

// an output that writes every element once: no dimension folded onto itself
void writable(const Tensor& t, const char* n) {
  long long span = 1;
  // strides, from the smallest, must step over everything below them
  std::vector<std::pair<long long, long long>> d;
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) d.emplace_back(t.stride(i), t.size(i));
  std::sort(d.begin(), d.end());
  for (auto& x : d) {
    COB_CHECK(x.first >= span, n, " overlaps itself (expanded or overlapping strides)");
    span = x.first * (x.second - 1) + span;
  }
}

// a caller's tensor that a kernel writes: autograd must see that a value saved for a backward pass has changed (tensors
// of inference mode have no version)
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Derivatives that are not formed must not be lost silently: operands of calls without a backward pass take no gradient
// (while gradients are recorded), and none of the calls takes a forward-mode tangent.
void no_tangent(const char* op, std::initializer_list<const Tensor*> operands) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : operands) COB_CHECK(!t || !t->_fw_grad(0).defined(), op, " has no forward-mode derivative");
}
void constants(const char* op, std::initializer_list<const Tensor*> operands) {
  if (torch::GradMode::is_enabled())
    for (const Tensor* t : operands)
      COB_CHECK(!t || !t->requires_grad(), op, " forms no gradient: call it under torch.no_grad(), or with detached operands");
  no_tangent(op, operands);
}

struct Tables {
  int max_pos, rot;
};
Tables tables(const Tensor& cos_t, const Tensor& sin_t, int64_t D, const Tensor& ref) {
  dense(cos_t, "cos", torch::kFloat, ref);
  dense(sin_t, "sin", torch::kFloat, ref);
  COB_CHECK(cos_t.dim() == 2 && cos_t.sizes() == sin_t.sizes(), "cos and sin must be [max_pos, rotary_dim / 2]");
  COB_CHECK(cos_t.size(0) >= 1 && cos_t.size(0) < (1ll << 31), "cos and sin need between 1 and 2^31 - 1 positions");
  const int64_t rot = 2 * cos_t.size(1);
  COB_CHECK(rot >= 2 && rot <= D, "rotary_dim (2 x the tables' columns) must be between 2 and head_dim, got ", rot,
            " for head_dim ", D);
  COB_CHECK(!cos_t.requires_grad() && !sin_t.requires_grad(), "cos and sin are constants: no gradient is formed");
  // rows of a multiple of four angles are read four at a time
  for (const auto* t : {&cos_t, &sin_t})
    COB_CHECK(cos_t.size(1) % 4 || reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0, "cos and sin must be 16-byte aligned");
  return {(int)cos_t.size(0), (int)rot};
}

void head_dim_ok(int64_t D) {
  COB_CHECK(D >= 2 && D <= 512 && D % 2 == 0, "head_dim must be even and at most 512, got ", D);
}

// components contiguous (a copy where they are not)
Tensor unit_last(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

// [N, H, D] or [B, S, H, D]
cob::HeadView view_of(const Tensor& t) {
  cob::HeadView v;
  v.p = t.data_ptr();
  const bool four = t.dim() == 4;
  v.sb = four ? t.stride(0) : 0;
  v.ss = t.stride(four ? 1 : 0);
  v.sh = t.stride(four ? 2 : 1);
  v.heads = (int)t.size(four ? 2 : 1);
  return v;
}

void rows_of(const Tensor& x, const Tensor& pos, cob::RotaryParams& p) {
  const bool four = x.dim() == 4;
  p.batch = four ? (int)x.size(0) : 1;
  p.seq = (int)x.size(four ? 1 : 0);
  on_device(pos, "positions", x);
  COB_CHECK(pos.scalar_type() == torch::kInt, "positions must be int32");
  if (pos.dim() == 1) {
    COB_CHECK(pos.size(0) == p.seq, "positions must be [seq] or [batch, seq] of the operand");
    p.pos_sb = 0;
    p.pos_ss = pos.stride(0);
  } else {
    COB_CHECK(four && pos.dim() == 2 && pos.size(0) == p.batch && pos.size(1) == p.seq,
              "positions must be [seq] or [batch, seq] of the operand");
    p.pos_sb = pos.stride(0);
    p.pos_ss = pos.stride(1);
  }
  p.pos = pos.data_ptr<int32_t>();
}

void operand_ok(const Tensor& x, const char* n) {
  COB_CHECK(x.is_cuda(), n, " must be a CUDA tensor");
  has_memory(x, n);
  COB_CHECK(x.dim() == 3 || x.dim() == 4, n, " must be [tokens, heads, head_dim] or [batch, seq, heads, head_dim]");
  code_of(x, n);
  head_dim_ok(x.size(-1));
  for (int64_t i = 0; i < x.dim(); ++i) COB_CHECK(x.size(i) < (1ll << 31), n, " has a dimension past 2^31");
  COB_CHECK(x.size(-2) <= (1 << 24), n, " has more than 2^24 heads");  // (sums of heads stay in 32 bits)
}

Tensor py_rotary(Tensor x, Tensor positions, Tensor cos_t, Tensor sin_t, bool interleaved, bool inverse, OptTensor out) {
  operand_ok(x, "x");
  constants("rotary", {&x, given(out)});
  cob::RotaryParams p;
  const Tables t = tables(cos_t, sin_t, x.size(-1), x);
  rows_of(x, positions, p);
  Tensor y;
  if (out.has_value()) {
    y = *out;
    on_device(y, "out", x);
    COB_CHECK(y.sizes() == x.sizes() && y.scalar_type() == x.scalar_type() && (y.stride(-1) == 1 || y.numel() == 0),
              "out must have x's shape and type, components contiguous");
    writable(y, "out");
    const bool in_place = y.data_ptr() == x.data_ptr() && y.strides() == x.strides();
    COB_CHECK(in_place || !overlap(x, y), "out must be x itself or lie in memory of its own");
    apart({&y}, {&positions, &cos_t, &sin_t}, "out must lie in memory of its own: it overlaps an input");
  }
  const c10::cuda::CUDAGuard g(x.device());
  if (!out.has_value()) y = torch::empty(x.sizes(), x.options().requires_grad(false));
  if (x.numel() == 0) return y;
  const Tensor xc = unit_last(x);
  p.in[0] = view_of(xc);
  p.out[0] = view_of(y);
  p.cos_t = cos_t.data_ptr<float>();
  p.sin_t = sin_t.data_ptr<float>();
  p.max_pos = t.max_pos;
  p.rot = t.rot;
  p.D = (int)x.size(-1);
  p.interleaved = interleaved;
  p.inverse = inverse;
  p.dtype = code_of(x, "x");
  ok(cob::rotary_forward(p, cur()), "rotary");
  if (out.has_value()) written(y);
  return y;
}

// y = R x; the gradient of a rotation is the rotation back (itself differentiable)
struct RotaryFn : public torch::autograd::Function<RotaryFn> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, Tensor x, Tensor positions, Tensor cos_t, Tensor sin_t,
                        bool interleaved, bool inverse) {
    ctx->save_for_backward({positions, cos_t, sin_t});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    return py_rotary(x, positions, cos_t, sin_t, interleaved, inverse, c10::nullopt);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list dy) {
    const auto s = ctx->get_saved_variables();
    const Tensor dx = RotaryFn::apply(dy[0], s[0], s[1], s[2], ctx->saved_data["interleaved"].toBool(),
                                      !ctx->saved_data["inverse"].toBool());
    return {dx, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor py_rotary_autograd(Tensor x, Tensor positions, Tensor cos_t, Tensor sin_t, bool interleaved, bool inverse) {
  no_tangent("rotary", {&x});
  return RotaryFn::apply(x, positions, cos_t, sin_t, interleaved, inverse);
}

void weights_ok(const Tensor& wq, const Tensor& wk, const Tensor& x, cob::RotaryParams& p) {
  for (const auto* w : {&wq, &wk}) {
    on_device(*w, "norm weight", x);
    COB_CHECK(w->dim() == 1 && w->size(0) == x.size(-1) && w->is_contiguous(), "norm weights must be contiguous [head_dim]");
    COB_CHECK(w->scalar_type() == wq.scalar_type() &&
                  (w->scalar_type() == torch::kFloat || w->scalar_type() == x.scalar_type()),
              "norm weights must both be float32 or both of the operands' type");
  }
  p.w[0] = wq.data_ptr();
  p.w[1] = wk.data_ptr();
  p.w_f32 = wq.scalar_type() == torch::kFloat;
}

void pair_ok(const Tensor& q, const Tensor& k) {
  operand_ok(q, "q");
  operand_ok(k, "k");
  on_device(k, "k", q);
  COB_CHECK(q.dim() == k.dim() && q.scalar_type() == k.scalar_type() && q.size(-1) == k.size(-1) &&
                q.size(0) == k.size(0) && (q.dim() == 3 || q.size(1) == k.size(1)),
            "q and k must agree in type, rows and head_dim");
}

std::tuple<Tensor, Tensor> py_qk_norm_rotary(Tensor q, Tensor k, Tensor wq, Tensor wk, Tensor positions, Tensor cos_t,
                                             Tensor sin_t, double eps, bool interleaved) {
  pair_ok(q, k);
  constants("qk_norm_rotary", {&q, &k, &wq, &wk});
  cob::RotaryParams p;
  const Tables t = tables(cos_t, sin_t, q.size(-1), q);
  rows_of(q, positions, p);
  weights_ok(wq, wk, q, p);
  const c10::cuda::CUDAGuard g(q.device());
  Tensor yq = torch::empty(q.sizes(), q.options().requires_grad(false));
  Tensor yk = torch::empty(k.sizes(), k.options().requires_grad(false));
  if (q.numel() + k.numel() == 0) return {yq, yk};
  const Tensor qc = unit_last(q), kc = unit_last(k);
  p.in[0] = view_of(qc);
  p.in[1] = view_of(kc);
  p.out[0] = view_of(yq);
  p.out[1] = view_of(yk);
  p.cos_t = cos_t.data_ptr<float>();
  p.sin_t = sin_t.data_ptr<float>();
  p.max_pos = t.max_pos;
  p.rot = t.rot;
  p.D = (int)q.size(-1);
  p.eps = (float)eps;
  p.interleaved = interleaved;
  p.dtype = code_of(q, "q");
  ok(cob::rotary_forward(p, cur()), "qk_norm_rotary");
  return {yq, yk};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> py_qk_norm_rotary_backward(Tensor dq, Tensor dk, Tensor q, Tensor k,
                                                                      Tensor wq, Tensor wk, Tensor positions,
                                                                      Tensor cos_t, Tensor sin_t, double eps,
                                                                      bool interleaved) {
  pair_ok(q, k);
  no_tangent("qk_norm_rotary_backward", {&dq, &dk, &q, &k, &wq, &wk});
  on_device(dq, "dq", q);
  on_device(dk, "dk", q);
  COB_CHECK(dq.sizes() == q.sizes() && dk.sizes() == k.sizes() && dq.scalar_type() == q.scalar_type() &&
                dk.scalar_type() == q.scalar_type(),
            "gradients must have the operands' shapes and type");
  cob::RotaryParams p;
  const Tables t = tables(cos_t, sin_t, q.size(-1), q);
  rows_of(q, positions, p);
  weights_ok(wq, wk, q, p);
  const c10::cuda::CUDAGuard g(q.device());
  Tensor gq = torch::empty(q.sizes(), q.options().requires_grad(false));
  Tensor gk = torch::empty(k.sizes(), k.options().requires_grad(false));
  if (q.numel() == 0 || k.numel() == 0) {
    COB_CHECK(q.numel() + k.numel() == 0, "q and k must both have rows and heads, or neither");
    return {gq, gk, torch::zeros_like(wq), torch::zeros_like(wk)};
  }
  Tensor gwq = torch::empty(wq.sizes(), wq.options().requires_grad(false));
  Tensor gwk = torch::empty(wk.sizes(), wk.options().requires_grad(false));
  const Tensor qc = unit_last(q), kc = unit_last(k), dqc = unit_last(dq), dkc = unit_last(dk);
  p.in[0] = view_of(qc);
  p.in[1] = view_of(kc);
  p.grad[0] = view_of(dqc);
  p.grad[1] = view_of(dkc);
  p.out[0] = view_of(gq);
  p.out[1] = view_of(gk);
  p.cos_t = cos_t.data_ptr<float>();
  p.sin_t = sin_t.data_ptr<float>();
  p.max_pos = t.max_pos;
  p.rot = t.rot;
  p.D = (int)q.size(-1);
  p.eps = (float)eps;
  p.interleaved = interleaved;
  p.dtype = code_of(q, "q");
  // the blocks' partial weight gradients: memory of this call (or of the graph that captures it)
  Tensor ws = torch::empty({cob::rotary_backward_blocks(p), q.size(-1)}, wq.options().dtype(torch::kFloat).requires_grad(false));
  ok(cob::rotary_norm_backward(p, ws.data_ptr<float>(), gwq.data_ptr(), gwk.data_ptr(), cur()), "qk_norm_rotary backward");
  return {gq, gk, gwq, gwk};
}

struct QkNormRotaryFn : public torch::autograd::Function<QkNormRotaryFn> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, Tensor q, Tensor k, Tensor wq,
                                                Tensor wk, Tensor positions, Tensor cos_t, Tensor sin_t, double eps,
                                                bool interleaved) {
    ctx->save_for_backward({q, k, wq, wk, positions, cos_t, sin_t});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    auto y = py_qk_norm_rotary(q, k, wq, wk, positions, cos_t, sin_t, eps, interleaved);
    return {std::get<0>(y), std::get<1>(y)};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list dy) {
    COB_CHECK(!torch::GradMode::is_enabled(), "qk_norm_rotary: gradients of its gradients are not formed");
    const auto s = ctx->get_saved_variables();
    auto g = py_qk_norm_rotary_backward(dy[0], dy[1], s[0], s[1], s[2], s[3], s[4], s[5], s[6],
                                        ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool());
    return {std::get<0>(g), std::get<1>(g), std::get<2>(g), std::get<3>(g), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> py_qk_norm_rotary_autograd(Tensor q, Tensor k, Tensor wq, Tensor wk, Tensor positions,
                                                      Tensor cos_t, Tensor sin_t, double eps, bool interleaved) {
  no_tangent("qk_norm_rotary", {&q, &k, &wq, &wk});
  auto y = QkNormRotaryFn::apply(q, k, wq, wk, positions, cos_t, sin_t, eps, interleaved);
  return {y[0], y[1]};
}

// caches [num_blocks, nkv, 16, D] and block tables [batch, max_blocks]
void cache_ok(const Tensor& k, const Tensor& v, const Tensor& bt, const Tensor& ref, int64_t nkv, int64_t D, int64_t batch) {
  for (const auto* c : {&k, &v}) {
    dense(*c, c == &k ? "k_cache" : "v_cache", ref.scalar_type(), ref);
    COB_CHECK(c->dim() == 4 && c->size(0) >= 1 && c->size(1) == nkv && c->size(2) == 16 && c->size(3) == D,
              "caches must be [num_blocks, ", nkv, ", 16, ", D, "]");
    COB_CHECK(reinterpret_cast<uintptr_t>(c->data_ptr()) % 16 == 0, "caches must be 16-byte aligned");
  }
  COB_CHECK(k.size(0) == v.size(0), "k_cache and v_cache must have the same number of blocks");
  COB_CHECK(k.size(0) * nkv * 16 < (1ll << 31), "a cache holds at most 2^31 - 1 head rows");
  dense(bt, "block_tables", torch::kInt, ref);
  COB_CHECK(bt.dim() == 2 && bt.size(0) == batch && bt.size(1) >= 1 && bt.size(1) <= (1 << 26),
            "block_tables must be [batch, max_blocks], at most 2^26 pages a sequence");
}

void lens_ok(const Tensor& t, const char* n, int64_t batch, const Tensor& ref) {
  dense(t, n, torch::kInt, ref);
  COB_CHECK(t.dim() == 1 && t.size(0) == batch, n, " must be int32 [batch]");
}

void py_qk_norm_rotary_append(Tensor qkv, Tensor positions, Tensor cos_t, Tensor sin_t, Tensor block_tables,
                              Tensor starts, Tensor q_out, Tensor k_cache, Tensor v_cache, int64_t nq, int64_t nkv,
                              OptTensor wq, OptTensor wk, double eps, OptTensor lens, OptTensor bias, bool interleaved) {
  COB_CHECK(qkv.is_cuda() && (qkv.dim() == 2 || qkv.dim() == 3), "qkv must be a CUDA tensor [batch, seq, width] or [batch * seq, width]");
  has_memory(qkv, "qkv");
  code_of(qkv, "qkv");
  constants("qk_norm_rotary_append_kv", {&qkv, &q_out, &k_cache, &v_cache, given(wq), given(wk), given(bias)});
  COB_CHECK(nq >= 1 && nkv >= 1 && nq <= (1 << 24) && nkv <= (1 << 24), "nq and nkv must be positive, at most 2^24");
  on_device(starts, "starts", qkv);
  const int64_t B = starts.numel(), W = qkv.size(-1), n = nq + 2 * nkv;
  COB_CHECK(W % n == 0, "qkv's rows must hold nq + 2 nkv heads");
  const int64_t D = W / n;
  head_dim_ok(D);
  lens_ok(starts, "starts", B, qkv);
  const bool three = qkv.dim() == 3;
  COB_CHECK(three ? qkv.size(0) == B : (B == 0 ? qkv.size(0) == 0 : qkv.size(0) % B == 0), "qkv's rows must be starts.numel() x seq");
  const int64_t S = three ? qkv.size(1) : (B ? qkv.size(0) / B : 0);
  COB_CHECK(B < (1ll << 31) && S < (1ll << 31), "too many rows");
  COB_CHECK(qkv.stride(-1) == 1 || qkv.numel() == 0, "qkv's last dimension must be contiguous");
  const Tables t = tables(cos_t, sin_t, D, qkv);
  dense(positions, "positions", torch::kInt, qkv);
  const bool per_row = positions.dim() == 2 ? positions.size(0) == B && positions.size(1) == S
                                            : positions.dim() == 1 && positions.size(0) == B * S;
  COB_CHECK(per_row || (positions.dim() == 1 && positions.size(0) == S), "positions must be [batch, seq], [batch * seq] or [seq]");
  dense(q_out, "q_out", qkv.scalar_type(), qkv);
  COB_CHECK(q_out.numel() == B * S * nq * D, "q_out must hold batch x seq x nq x head_dim elements");
  cache_ok(k_cache, v_cache, block_tables, qkv, nkv, D, B);
  COB_CHECK(wq.has_value() == wk.has_value(), "give both norm weights or neither");
  cob::RotaryParams p;
  if (wq.has_value()) {
    for (const auto* w : {&*wq, &*wk}) {
      on_device(*w, "norm weight", qkv);
      COB_CHECK(w->dim() == 1 && w->size(0) == D && w->is_contiguous(), "norm weights must be contiguous [head_dim]");
      COB_CHECK(w->scalar_type() == wq->scalar_type() &&
                    (w->scalar_type() == torch::kFloat || w->scalar_type() == qkv.scalar_type()),
                "norm weights must both be float32 or both of the operands' type");
    }
    p.w[0] = wq->data_ptr();
    p.w[1] = wk->data_ptr();
    p.w_f32 = wq->scalar_type() == torch::kFloat;
  }
  if (lens.has_value()) {
    lens_ok(*lens, "lens", B, qkv);
    p.lens = lens->data_ptr<int32_t>();
  }
  if (bias.has_value()) {
    dense(*bias, "bias", qkv.scalar_type(), qkv);
    COB_CHECK(bias->numel() == W, "bias must have (nq + 2 nkv) * head_dim elements");
    p.bias = bias->data_ptr();
  }
  apart({&q_out, &k_cache, &v_cache},
        {&qkv, &positions, &cos_t, &sin_t, &block_tables, &starts, given(wq), given(wk), given(lens), given(bias)},
        "q_out and the caches must lie in memory of their own");
  if (B * S == 0) return;
  const c10::cuda::CUDAGuard g(qkv.device());
  const int64_t e = qkv.element_size();
  const int64_t ss = three ? qkv.stride(1) : qkv.stride(0), sb = three ? qkv.stride(0) : S * qkv.stride(0);
  const char* base = static_cast<const char*>(qkv.data_ptr());
  const int64_t heads[3] = {nq, nkv, nkv}, first[3] = {0, nq, nq + nkv};
  for (int i = 0; i < 3; ++i) {
    p.in[i].p = base + first[i] * D * e;
    p.in[i].sb = sb;
    p.in[i].ss = ss;
    p.in[i].sh = D;
    p.in[i].heads = (int)heads[i];
  }
  p.out[0].p = q_out.data_ptr();
  p.out[0].sb = S * nq * D;
  p.out[0].ss = nq * D;
  p.out[0].sh = D;
  p.out[0].heads = (int)nq;
  p.pos = positions.data_ptr<int32_t>();
  p.pos_ss = 1;
  p.pos_sb = per_row ? S : 0;
  p.cos_t = cos_t.data_ptr<float>();
  p.sin_t = sin_t.data_ptr<float>();
  p.max_pos = t.max_pos;
  p.rot = t.rot;
  p.D = (int)D;
  p.batch = (int)B;
  p.seq = (int)S;
  p.eps = (float)eps;
  p.interleaved = interleaved;
  p.append = 1;
  p.block_tables = block_tables.data_ptr<int32_t>();
  p.starts = starts.data_ptr<int32_t>();
  p.k_cache = k_cache.data_ptr();
  p.v_cache = v_cache.data_ptr();
  p.max_blocks = (int)block_tables.size(1);
  p.num_blocks = (int)k_cache.size(0);
  p.dtype = code_of(qkv, "qkv");
  ok(cob::rotary_forward(p, cur()), "qk_norm_rotary_append_kv");
  for (const Tensor* t : {&q_out, &k_cache, &v_cache}) written(*t);
}

Tensor py_tree_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_tables, Tensor ctx_lens, OptTensor mask,
                         double scale, OptTensor tree_lens, OptTensor out, int64_t timeout_ns) {
  COB_CHECK(q.is_cuda() && q.dim() == 4, "q must be a CUDA tensor [batch, tree, nq, head_dim]");
  has_memory(q, "q");
  const int dtype = code_of(q, "q");
  COB_CHECK(dtype != cob::kF32, "q and the caches must be float16 or bfloat16");
  constants("tree_attention", {&q, &k_cache, &v_cache, given(out)});
  COB_CHECK(timeout_ns >= 0, "timeout_ms must not be negative");
  COB_CHECK(std::isfinite((float)scale), "scale must be finite");
  cob::TreeAttnParams p;
  const int64_t B = q.size(0), T = q.size(1), nq = q.size(2), D = q.size(3);
  COB_CHECK(D == 64 || D == 128, "head_dim must be 64 or 128, got ", D);
  COB_CHECK(T >= 1 && T <= 64, "a tree has 1 to 64 drafted tokens, got ", T);
  COB_CHECK(B <= 4096, "at most 4096 sequences, got ", B);
  COB_CHECK(k_cache.dim() == 4 && k_cache.size(1) >= 1, "caches must be [num_blocks, nkv, 16, head_dim]");
  const int64_t nkv = k_cache.size(1);
  COB_CHECK(nq >= 1 && nq % nkv == 0 && nq / nkv <= 64, "nq must be a multiple of nkv, at most 64 query heads per KV head");
  cache_ok(k_cache, v_cache, block_tables, q, nkv, D, B);
  lens_ok(ctx_lens, "ctx_lens", B, q);
  if (tree_lens.has_value()) {
    lens_ok(*tree_lens, "tree_lens", B, q);
    p.tree_lens = tree_lens->data_ptr<int32_t>();
  }
  if (mask.has_value()) {
    dense(*mask, "tree_mask", torch::kLong, q);
    const bool one = mask->dim() == 1;
    COB_CHECK(one ? mask->size(0) == T : (mask->dim() == 2 && mask->size(0) == B && mask->size(1) == T),
              "tree_mask must be int64 [tree] or [batch, tree]");
    p.mask = mask->data_ptr<int64_t>();
    p.mask_sb = one ? 0 : T;
  }
  const c10::cuda::CUDAGuard g(q.device());
  auto vec_ok = [&](const Tensor& t) {
    return t.stride(3) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && t.stride(2) % 8 == 0 &&
           reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  };
  Tensor y;
  if (out.has_value()) {
    y = *out;
    on_device(y, "out", q);
    COB_CHECK(y.sizes() == q.sizes() && y.scalar_type() == q.scalar_type(), "out must have q's shape and type");
    COB_CHECK(y.numel() == 0 || vec_ok(y), "out's heads must be contiguous and 16-byte aligned");
    writable(y, "out");
    apart({&y}, {&q, &k_cache, &v_cache, &block_tables, &ctx_lens, given(mask), given(tree_lens)}, "out must lie in memory of its own");
  } else {
    // rows past tree_lens are not written: give them a value
    y = tree_lens.has_value() ? torch::zeros(q.sizes(), q.options()) : torch::empty(q.sizes(), q.options());
  }
  if (q.numel() == 0) return y;
  // (a copy always: contiguous() would hand back a contiguous q whose start is not on a 16-byte boundary)
  const Tensor qc = vec_ok(q) ? q : q.clone(at::MemoryFormat::Contiguous);
  p.q = qc.data_ptr();
  p.q_sb = qc.stride(0), p.q_st = qc.stride(1), p.q_sh = qc.stride(2);
  p.out = y.data_ptr();
  p.o_sb = y.stride(0), p.o_st = y.stride(1), p.o_sh = y.stride(2);
  p.k_cache = k_cache.data_ptr();
  p.v_cache = v_cache.data_ptr();
  p.block_tables = block_tables.data_ptr<int32_t>();
  p.ctx_lens = ctx_lens.data_ptr<int32_t>();
  p.batch = (int)B;
  p.tree = (int)T;
  p.nq = (int)nq;
  p.nkv = (int)nkv;
  p.head_dim = (int)D;
  p.max_blocks = (int)block_tables.size(1);
  p.num_blocks = (int)k_cache.size(0);
  p.scale = (float)scale;
  p.timeout_ns = (unsigned long long)timeout_ns;
  p.dtype = dtype;
  // partials of rows cut between CTAs: memory of this call (or of the graph that captures it)
  Tensor scratch = torch::empty({(int64_t)cob::tree_attention_scratch_bytes(p)}, q.options().dtype(torch::kByte).requires_grad(false));
  ok(cob::tree_attention(p, scratch.data_ptr(), cur()), "tree_attention");
  if (out.has_value()) written(y);
  return y;
}

// the device's word, as a tensor over it
Tensor py_tree_attention_error_word(int64_t device) {
  const c10::cuda::CUDAGuard g((c10::DeviceIndex)device);
  int* word = nullptr;
  ok(cob::tree_attention_error_word(&word), "tree_attention_error_word");
  return torch::from_blob(word, {1}, torch::TensorOptions().dtype(torch::kInt).device(torch::kCUDA, (c10::DeviceIndex)device));
}

Tensor py_penalize_logits(Tensor logits, OptTensor tokens, OptTensor lens, OptTensor prompt_lens, OptTensor repetition,
                          OptTensor frequency, OptTensor presence, OptTensor bias_ids, OptTensor bias, OptTensor allowed,
                          int64_t vocab_offset, OptTensor out, OptTensor keys) {
  // the kernel looks up to 2048 entries ahead in 32-bit indexes, which must not wrap
  constexpr int64_t kMostEntries = 1ll << 30;
  COB_CHECK(logits.is_cuda() && logits.dim() == 2, "logits must be a CUDA tensor [rows, vocab]");
  has_memory(logits, "logits");
  cob::LogitsParams p;
  p.dtype = code_of(logits, "logits");
  constants("penalize_logits", {&logits, given(repetition), given(frequency), given(presence), given(bias), given(out)});
  const int64_t B = logits.size(0), V = logits.size(1);
  COB_CHECK(V >= 1 && V <= (1 << 26) && B < (1ll << 31), "logits must be [rows, vocab] with 1 to 2^26 ids");
  COB_CHECK(logits.stride(1) == 1 || V == 1, "a row's logits must be contiguous");
  COB_CHECK(vocab_offset >= 0 && vocab_offset < (1ll << 31) && vocab_offset + V < (1ll << 31), "vocab_offset must keep every id below 2^31");
  auto per_row = [&](const OptTensor& t, const char* n) -> const float* {
    if (!t.has_value()) return nullptr;
    dense(*t, n, torch::kFloat, logits);
    COB_CHECK(t->dim() == 1 && t->size(0) == B, n, " must be float32 [rows]");
    return t->data_ptr<float>();
  };
  p.repetition = per_row(repetition, "repetition");
  p.frequency = per_row(frequency, "frequency");
  p.presence = per_row(presence, "presence");
  if (tokens.has_value()) {
    on_device(*tokens, "tokens", logits);
    COB_CHECK(tokens->scalar_type() == torch::kInt && tokens->dim() == 2 && tokens->size(0) == B &&
                  (tokens->stride(1) == 1 || tokens->size(1) <= 1),
              "tokens must be int32 [rows, history], a row's ids contiguous");
    COB_CHECK(tokens->size(1) <= kMostEntries, "tokens hold at most 2^30 ids a row");
    p.tokens = tokens->data_ptr<int32_t>();
    p.ld_tokens = tokens->stride(0);
    p.history = (int)tokens->size(1);
    if (lens.has_value()) {
      lens_ok(*lens, "lens", B, logits);
      p.lens = lens->data_ptr<int32_t>();
    }
    if (prompt_lens.has_value()) {
      lens_ok(*prompt_lens, "prompt_lens", B, logits);
      p.prompt_lens = prompt_lens->data_ptr<int32_t>();
    }
  } else {
    COB_CHECK(!lens.has_value() && !prompt_lens.has_value() && !p.repetition && !p.frequency && !p.presence,
              "penalties and lengths need the rows' tokens");
  }
  COB_CHECK(bias_ids.has_value() == bias.has_value(), "give bias_ids and bias together");
  if (bias.has_value()) {
    dense(*bias_ids, "bias_ids", torch::kInt, logits);
    dense(*bias, "bias", torch::kFloat, logits);
    COB_CHECK(bias->dim() == 2 && bias->size(0) == B && bias->sizes() == bias_ids->sizes(),
              "bias_ids (int32) and bias (float32) must be [rows, entries]");
    COB_CHECK(bias->size(1) <= kMostEntries, "a row has at most 2^30 biases");
    p.bias_ids = bias_ids->data_ptr<int32_t>();
    p.bias = bias->data_ptr<float>();
    p.biases = (int)bias->size(1);
  }
  if (allowed.has_value()) {
    on_device(*allowed, "allowed", logits);
    COB_CHECK(allowed->scalar_type() == torch::kInt && allowed->dim() == 2 && allowed->size(0) == B &&
                  (allowed->stride(1) == 1 || allowed->size(1) == 1) && allowed->size(1) * 32 >= vocab_offset + V,
              "allowed must be int32 [rows, words] with a bit for every id up to vocab_offset + vocab, a row's words contiguous");
    p.allowed = reinterpret_cast<const uint32_t*>(allowed->data_ptr<int32_t>());
    p.ld_mask = allowed->stride(0);
  }
  if (keys.has_value()) {
    dense(*keys, "keys", torch::kLong, logits);
    COB_CHECK(keys->dim() == 1 && keys->size(0) == B, "keys must be int64 [rows]");
    p.keys = reinterpret_cast<unsigned long long*>(keys->data_ptr());
  }
  const c10::cuda::CUDAGuard g(logits.device());
  Tensor y;
  if (out.has_value()) {
    y = *out;
    on_device(y, "out", logits);
    COB_CHECK(y.sizes() == logits.sizes() && y.scalar_type() == logits.scalar_type() && (y.stride(1) == 1 || V == 1),
              "out must have the logits' shape and type, a row's values contiguous");
    writable(y, "out");
    COB_CHECK((y.data_ptr() == logits.data_ptr() && y.strides() == logits.strides()) || !overlap(y, logits),
              "out must be the logits themselves or lie in memory of its own");
  } else {
    y = torch::empty(logits.sizes(), logits.options());
  }
  if (out.has_value() || keys.has_value())
    apart({out.has_value() ? &y : nullptr, given(keys)},
          {given(tokens), given(lens), given(prompt_lens), given(repetition), given(frequency), given(presence), given(bias_ids),
           given(bias), given(allowed)},
          "out and keys must lie in memory of their own");
  if (keys.has_value()) COB_CHECK(!overlap(*keys, logits), "keys must lie in memory of their own");
  if (B == 0) return y;
  p.logits = logits.data_ptr();
  p.out = y.data_ptr();
  p.ld_in = logits.stride(0);
  p.ld_out = y.stride(0);
  p.rows = (int)B;
  p.vocab = (int)V;
  p.vocab_offset = (int)vocab_offset;
  ok(cob::penalize_logits(p, cur()), "penalize_logits");
  if (out.has_value()) written(y);
  if (keys.has_value()) written(*keys);
  return y;
}

}  // namespace

void register_serve(pybind11::module& m) {
  m.def("rotary", &py_rotary);
  m.def("rotary_autograd", &py_rotary_autograd);
  m.def("qk_norm_rotary", &py_qk_norm_rotary);
  m.def("qk_norm_rotary_autograd", &py_qk_norm_rotary_autograd);
  m.def("qk_norm_rotary_backward", &py_qk_norm_rotary_backward);
  m.def("qk_norm_rotary_append", &py_qk_norm_rotary_append);
  m.def("tree_attention", &py_tree_attention);
  m.def("tree_attention_error_word", &py_tree_attention_error_word);
  m.def("penalize_logits", &py_penalize_logits);
}
