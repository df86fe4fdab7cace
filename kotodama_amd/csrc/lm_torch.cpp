// The language-model operators on the native call path (attnres_torch.cpp says
// what that is): plain eager calls, recorded by C++ autograd functions with the
// ops' formulas.  A call with other strides, shapes or types than the kernels
// take is left to the Python layer (lmops.py), which copies or refuses.
//
// Why: under autograd the registered ops' Python cost 150-200 us of host time
// a call forward and backward, more than the kernels of most calls.

#include "attnres_torch_common.h"

namespace attnres_torch {
namespace {

// Strides of a (B, H, T, D) tensor, or none where the kernels would not take it
// (`align`: in 16-byte pieces).
struct Strides {
  int64_t s[3] = {0, 0, 0};
  bool ok = false;
  Strides(const Tensor& t, bool align) {
    if (!t.defined() || !dense(t) || !dtype_ok(t.scalar_type()) || t.dim() != 4) return;
    if (t.size(3) > 1 && t.stride(3) != 1) return;
    for (const int64_t n : t.sizes())
      if (n > INT32_MAX) return;
    const int64_t m = 16 / (int64_t)t.element_size();
    if (align && (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) != 0) return;
    for (int i = 0; i < 3; ++i) {
      s[i] = t.stride(i);
      if (align && t.size(i) > 1 && s[i] % m != 0) return;
    }
    ok = true;
  }
};

// An empty (B, H, T, D) tensor over (B, T, H, D) memory.
Tensor heads_inside(const Tensor& t) {
  const int64_t h = t.size(1), n = t.size(2), d = t.size(3);
  return Tensor(at::detail::empty_strided_cuda({t.size(0), h, n, d}, {n * h * d, d, h * d, 1}, t.scalar_type(),
                                               t.device()));
}

bool index_tensor(const Tensor& t, const Tensor& ref) {
  return dense(t) && (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) &&
         t.get_device() == ref.get_device();
}
int index_code(const Tensor& t) { return t.defined() && t.scalar_type() == at::kLong ? ATTNRES_INDEX_I64 : ATTNRES_INDEX_I32; }

// -------------------------------------------------------------- attention --

struct AttnCall {
  Tensor q, k, v, kv_lens, q_start;
  bool causal = true;
  double scale = 0;
  int64_t start_value = 0;

  bool fits() const {
    if (!q.defined() || q.dim() != 4 || k.dim() != 4 || v.dim() != 4) return false;
    const int64_t d = q.size(3);
    if (k.size(0) != q.size(0) || k.size(3) != d || v.sizes() != k.sizes() || k.size(1) < 1 || q.size(1) < 1 ||
        q.size(1) % k.size(1) != 0 || d % 8 != 0)
      return false;
    for (const Tensor* t : {&k, &v})
      if (t->scalar_type() != q.scalar_type() || !t->is_cuda() || t->get_device() != q.get_device()) return false;
    for (const Tensor* t : {&kv_lens, &q_start})
      if (t->defined() && (!index_tensor(*t, q) || t->dim() != 1 || t->size(0) != q.size(0) || !t->is_contiguous()))
        return false;
    return !kv_lens.defined() || !q_start.defined() || kv_lens.scalar_type() == q_start.scalar_type();
  }
  int index() const { return index_code(kv_lens.defined() ? kv_lens : q_start); }
};

bool attention_rows(const AttnCall& c, bool want_lse, Tensor* out, Tensor* lse) {
  if (!c.fits()) return false;
  const Strides sq(c.q, true), sk(c.k, true), sv(c.v, true);
  if (!sq.ok || !sk.ok || !sv.ok) return false;
  ATTNRES_RECORD("attnres_hip::attention");
  const Tensor& q = c.q;
  const int b = (int)q.size(0), h = (int)q.size(1), hk = (int)c.k.size(1), d = (int)q.size(3);
  const int64_t tq = q.size(2), tk = c.k.size(2);
  *out = heads_inside(q);
  if (want_lse) *lse = empty({b, h, tq}, at::kFloat, q.device());
  const Strides so(*out, true);
  const OnDevice on(q);
  int64_t bytes = 0;
  if (attnres_attention_workspace_size(b, h, hk, tq, tk, d, code(q.scalar_type()), 0, &bytes) != ATTNRES_OK)
    return false;
  const Tensor ws = bytes > 0 ? workspace(bytes, q.device()) : Tensor();
  return attnres_attention_fwd(ptr(q), sq.s, ptr(c.k), sk.s, ptr(c.v), sv.s, b, h, hk, tq, tk, d,
                               code(q.scalar_type()), c.causal ? 1 : 0, (float)c.scale, ptr(c.kv_lens),
                               ptr(c.q_start), c.index(), c.start_value, out->mutable_data_ptr(), so.s,
                               lse->defined() ? static_cast<float*>(lse->mutable_data_ptr()) : nullptr,
                               ws.defined() ? ws.mutable_data_ptr() : nullptr, bytes, on.stream) == ATTNRES_OK;
}

bool attention_rows_bwd(const AttnCall& c, const Tensor& out, const Tensor& lse, Tensor go, const Tensor& gl,
                        Tensor* dq, Tensor* dk, Tensor* dv) {
  if (!c.fits()) return false;
  // what was saved passes through the caller's saved-tensor hooks
  for (const Tensor* t : {static_cast<const Tensor*>(&go), &out})
    if (!t->is_cuda() || t->scalar_type() != c.q.scalar_type() || t->sizes() != c.q.sizes() ||
        t->get_device() != c.q.get_device())
      return false;
  Strides sgo(go, true);
  if (!sgo.ok) {
    if (!dense(go)) return false;
    go = go.clone(at::MemoryFormat::Contiguous);
    sgo = Strides(go, true);
  }
  const Strides sq(c.q, true), sk(c.k, true), sv(c.v, true), so(out, true);
  if (!sq.ok || !sk.ok || !sv.ok || !so.ok || !sgo.ok || !plain(lse) || lse.scalar_type() != at::kFloat ||
      lse.sizes() != c.q.sizes().slice(0, 3) || lse.get_device() != c.q.get_device())
    return false;
  if (gl.defined() && (!plain(gl) || gl.scalar_type() != at::kFloat || gl.sizes() != lse.sizes() ||
                       gl.get_device() != c.q.get_device()))
    return false;
  ATTNRES_RECORD("attnres_hip::attention_bwd");
  const Tensor& q = c.q;
  const int b = (int)q.size(0), h = (int)q.size(1), hk = (int)c.k.size(1), d = (int)q.size(3);
  const int64_t tq = q.size(2), tk = c.k.size(2);
  *dq = heads_inside(q);
  *dk = heads_inside(c.k);
  *dv = heads_inside(c.k);
  const Strides sdq(*dq, true), sdk(*dk, true), sdv(*dv, true);
  const OnDevice on(q);
  int64_t bytes = 0;
  if (attnres_attention_workspace_size(b, h, hk, tq, tk, d, code(q.scalar_type()), 1, &bytes) != ATTNRES_OK)
    return false;
  const Tensor ws = workspace(bytes, q.device());
  return attnres_attention_bwd(ptr(q), sq.s, ptr(c.k), sk.s, ptr(c.v), sv.s, ptr(out), so.s, ptr(go), sgo.s,
                               static_cast<const float*>(ptr(lse)), static_cast<const float*>(ptr(gl)), b, h, hk, tq,
                               tk, d, code(q.scalar_type()), c.causal ? 1 : 0, (float)c.scale, ptr(c.kv_lens),
                               ptr(c.q_start), c.index(), c.start_value, dq->mutable_data_ptr(), sdq.s,
                               dk->mutable_data_ptr(), sdk.s, dv->mutable_data_ptr(), sdv.s, ws.mutable_data_ptr(),
                               ws.numel() * 4, on.stream) == ATTNRES_OK;
}

struct Attention : public torch::autograd::Function<Attention> {
  static constexpr bool is_traceable = true;
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const AttnCall* c, const Tensor* out, const Tensor* lse) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, v, *out, *lse, c->kv_lens, c->q_start});
    ctx->saved_data["causal"] = c->causal;
    ctx->saved_data["scale"] = c->scale;
    ctx->saved_data["start"] = c->start_value;
    return {*out, *lse};
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list res(6);
    if (!g[0].defined() && !g[1].defined()) return res;
    const auto s = ctx->get_saved_variables();
    AttnCall c{s[0], s[1], s[2], s[5], s[6], ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(),
               ctx->saved_data["start"].toInt()};
    const Tensor go = g[0].defined() ? g[0] : at::zeros_like(s[3]);
    Tensor dq, dk, dv;
    if (at::GradMode::is_enabled() || !unwatched() || !attention_rows_bwd(c, s[3], s[4], go, g[1], &dq, &dk, &dv)) {
      const auto st = call_op("attnres_hip::attention_bwd", c.q, c.k, c.v, s[3], s[4], go, opt(g[1]), c.causal,
                              c.scale, opt(c.kv_lens), opt(c.q_start), c.start_value);
      dq = st[0].toTensor(), dk = st[1].toTensor(), dv = st[2].toTensor();
    }
    if (ctx->needs_input_grad(0)) res[0] = dq;
    if (ctx->needs_input_grad(1)) res[1] = dk;
    if (ctx->needs_input_grad(2)) res[2] = dv;
    return res;
  }
};

// ----------------------------------------------------------- qk_norm_rope --

struct RopeCall {
  Tensor q, k, wq, wk, cos, sin, positions;
  double eps = 0;
  int64_t pos_b = 0, pos_t = 0;

  bool fits() {
    if (!q.defined() || q.dim() != 4 || k.dim() != 4 || k.size(0) != q.size(0) || k.size(2) != q.size(2) ||
        k.size(3) != q.size(3))
      return false;
    const int64_t d = q.size(3), t = q.size(2), b = q.size(0);
    for (const Tensor* x : {&k, &wq, &wk})
      if (x->scalar_type() != q.scalar_type() || !x->is_cuda() || x->get_device() != q.get_device()) return false;
    for (const Tensor* w : {&wq, &wk})
      if (!plain(*w) || w->dim() != 1 || w->size(0) != d) return false;
    for (const Tensor* x : {&cos, &sin})
      if (!dense(*x) || x->get_device() != q.get_device() || x->dim() != 2 || x->size(1) != d || x->stride(1) != 1 ||
          (x->size(0) > 1 && x->stride(0) < d) || x->requires_grad())
        return false;
    if (cos.scalar_type() != sin.scalar_type() || cos.size(0) != sin.size(0) ||
        (cos.scalar_type() != q.scalar_type() && cos.scalar_type() != at::kFloat))
      return false;
    if (!positions.defined()) return cos.size(0) >= t;
    if (!index_tensor(positions, q)) return false;
    const int64_t n = positions.dim();
    if (n < 1 || n > 2 || positions.size(-1) != t) return false;
    if (n == 2 && positions.size(0) != b && positions.size(0) != 1) return false;
    pos_t = positions.stride(-1);
    pos_b = n == 2 && positions.size(0) > 1 ? positions.stride(0) : 0;
    return true;
  }
  int index() const { return index_code(positions); }
};

bool rope_rows(RopeCall& c, Tensor* yq, Tensor* yk) {
  if (!c.fits()) return false;
  const Strides sq(c.q, false), sk(c.k, false);
  if (!sq.ok || !sk.ok) return false;
  ATTNRES_RECORD("attnres_hip::qk_norm_rope");
  const Tensor& q = c.q;
  *yq = heads_inside(q);
  *yk = heads_inside(c.k);
  const Strides syq(*yq, false), syk(*yk, false);
  const OnDevice on(q);
  return attnres_qk_norm_rope_fwd(ptr(q), sq.s, ptr(c.k), sk.s, (int)q.size(0), (int)q.size(1), (int)c.k.size(1),
                                  q.size(2), (int)q.size(3), code(q.scalar_type()), ptr(c.wq), ptr(c.wk), ptr(c.cos),
                                  c.cos.stride(0), ptr(c.sin), c.sin.stride(0), c.cos.size(0),
                                  code(c.cos.scalar_type()), ptr(c.positions), c.index(), c.pos_b, c.pos_t,
                                  (float)c.eps, yq->mutable_data_ptr(), syq.s, yk->mutable_data_ptr(), syk.s,
                                  on.stream) == ATTNRES_OK;
}

bool rope_rows_bwd(RopeCall& c, const Tensor& gq, const Tensor& gk, Tensor (&d)[4]) {
  if (!c.fits()) return false;
  const Strides sq(c.q, false), sk(c.k, false), sgq(gq, false), sgk(gk, false);
  if (!sq.ok || !sk.ok || !sgq.ok || !sgk.ok) return false;
  for (const Tensor* g : {&gq, &gk})
    if (g->scalar_type() != c.q.scalar_type() || g->get_device() != c.q.get_device()) return false;
  if (gq.sizes() != c.q.sizes() || gk.sizes() != c.k.sizes()) return false;
  ATTNRES_RECORD("attnres_hip::qk_norm_rope_bwd");
  const Tensor& q = c.q;
  const int64_t dim = q.size(3);
  d[0] = heads_inside(q);
  d[1] = heads_inside(c.k);
  d[2] = empty({dim}, q.scalar_type(), q.device());
  d[3] = empty({dim}, q.scalar_type(), q.device());
  const Strides sdq(d[0], false), sdk(d[1], false);
  const OnDevice on(q);
  int64_t bytes = 0;
  if (attnres_qk_norm_rope_workspace_size((int)dim, &bytes) != ATTNRES_OK) return false;
  const Tensor ws = workspace(bytes, q.device());
  return attnres_qk_norm_rope_bwd(ptr(q), sq.s, ptr(c.k), sk.s, ptr(gq), sgq.s, ptr(gk), sgk.s, (int)q.size(0),
                                  (int)q.size(1), (int)c.k.size(1), q.size(2), (int)dim, code(q.scalar_type()),
                                  ptr(c.wq), ptr(c.wk), ptr(c.cos), c.cos.stride(0), ptr(c.sin), c.sin.stride(0),
                                  c.cos.size(0), code(c.cos.scalar_type()), ptr(c.positions), c.index(), c.pos_b,
                                  c.pos_t, (float)c.eps, d[0].mutable_data_ptr(), sdq.s, d[1].mutable_data_ptr(),
                                  sdk.s, d[2].mutable_data_ptr(), d[3].mutable_data_ptr(), ws.mutable_data_ptr(),
                                  ws.numel() * 4, on.stream) == ATTNRES_OK;
}

struct NormRope : public torch::autograd::Function<NormRope> {
  static constexpr bool is_traceable = true;
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& wq,
                               const Tensor& wk, const RopeCall* c, const Tensor* yq, const Tensor* yk) {
    ctx->save_for_backward({q, k, wq, wk, c->cos, c->sin, c->positions});
    ctx->saved_data["eps"] = c->eps;
    return {*yq, *yk};
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    RopeCall c{s[0], s[1], s[2], s[3], s[4], s[5], s[6], ctx->saved_data["eps"].toDouble()};
    Tensor d[4];
    if (at::GradMode::is_enabled() || !unwatched() || !rope_rows_bwd(c, g[0], g[1], d)) {
      const auto st = call_op("attnres_hip::qk_norm_rope_bwd", c.q, c.k, c.wq, c.wk, c.cos, c.sin, opt(c.positions),
                              c.eps, g[0], g[1]);
      for (int i = 0; i < 4; ++i) d[i] = st[i].toTensor();
    }
    variable_list res(7);
    for (int i = 0; i < 4; ++i)
      if (ctx->needs_input_grad(i)) res[i] = d[i];
    return res;
  }
};

// -------------------------------------------------------------- embedding --

bool table(const Tensor& t) {
  return dense(t) && dtype_ok(t.scalar_type()) && t.dim() == 2 && t.size(1) > 0 && t.size(1) <= INT32_MAX &&
         (t.stride(1) == 1 || t.size(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
}

bool embedding_rows(const Tensor& ids, const Tensor& w, double scale, Tensor* out) {
  if (!table(w) || !index_tensor(ids, w) || !ids.is_contiguous()) return false;
  ATTNRES_RECORD("attnres_hip::embedding");
  Dims size(ids.sizes().begin(), ids.sizes().end());
  size.push_back(w.size(1));
  *out = empty(size, w.scalar_type(), w.device());
  const OnDevice on(w);
  return attnres_embedding_fwd(ptr(ids), index_code(ids), ids.numel(), ptr(w), w.stride(0), w.size(0),
                               (int)w.size(1), code(w.scalar_type()), (float)scale, out->mutable_data_ptr(),
                               on.stream) == ATTNRES_OK;
}

bool embedding_rows_bwd(const Tensor& ids, const Tensor& go, at::ScalarType dtype, int64_t rows, double scale,
                        int64_t padding, Tensor* dw) {
  if (!plain(go) || go.scalar_type() != dtype || go.dim() < 1 || go.size(-1) < 1 || go.size(-1) > INT32_MAX ||
      !index_tensor(ids, go) || !ids.is_contiguous() || ids.sizes() != go.sizes().slice(0, go.dim() - 1))
    return false;
  ATTNRES_RECORD("attnres_hip::embedding_bwd");
  const int64_t hidden = go.size(-1);
  *dw = empty({rows, hidden}, dtype, go.device());
  const OnDevice on(go);
  int64_t bytes = 0;
  if (attnres_embedding_workspace_size(ids.numel(), rows, (int)hidden, &bytes) != ATTNRES_OK) return false;
  const Tensor ws = workspace(bytes, go.device());
  return attnres_embedding_bwd(ptr(ids), index_code(ids), ids.numel(), ptr(go), hidden, rows, (int)hidden,
                               code(dtype), (float)scale, padding, dw->mutable_data_ptr(), ws.mutable_data_ptr(),
                               ws.numel() * 4, on.stream) == ATTNRES_OK;
}

struct Embedding : public torch::autograd::Function<Embedding> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, const Tensor& w, const Tensor& ids, const Tensor* out, double scale,
                        int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = w.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    ctx->saved_data["dtype"] = (int64_t)w.scalar_type();
    return *out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const Tensor ids = ctx->get_saved_variables()[0];
    const int64_t rows = ctx->saved_data["rows"].toInt(), padding = ctx->saved_data["padding"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    const auto dtype = (at::ScalarType)ctx->saved_data["dtype"].toInt();
    Tensor dw;
    if (at::GradMode::is_enabled() || !unwatched() ||
        !embedding_rows_bwd(ids, g[0], dtype, rows, scale, padding, &dw))
      dw = call_op("attnres_hip::embedding_bwd", ids, g[0].to(dtype), rows, scale, padding)[0].toTensor();
    return {dw, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

}  // namespace

// attention(q, k, v, causal, scale, kv_lens, q_start, q_start_value, want_lse) -> out or (out, lse)
PyObject* py_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  AttnCall c;
  bool want_lse = false;
  if (n != 9 || !take(a[0], false, &c.q) || !take(a[1], false, &c.k) || !take(a[2], false, &c.v) ||
      !take(a[3], &c.causal) || !take(a[4], &c.scale) || !take(a[5], true, &c.kv_lens) ||
      !take(a[6], true, &c.q_start) || !take(a[7], &c.start_value) || !take(a[8], &want_lse) || !unwatched())
    return none();
  const bool rec = recorded({&c.q, &c.k, &c.v});
  if (!(no_tangent(c.q) && no_tangent(c.k) && no_tangent(c.v))) return none();  // refused in Python
  Tensor out, lse;
  bool ok = false;
  {
    pybind11::gil_scoped_release nogil;
    ok = attention_rows(c, want_lse || rec, &out, &lse);
  }
  if (!ok) return none();
  if (rec) {
    const variable_list o = Attention::apply(c.q, c.k, c.v, &c, &out, &lse);
    out = o[0], lse = o[1];
  }
  if (!want_lse) return wrap(out);
  return Py_BuildValue("(NN)", wrap(out), wrap(lse));
  END_HANDLE_TH_ERRORS
}

// qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps) -> (q, k)
PyObject* py_qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  RopeCall c;
  if (n != 8 || !take(a[0], false, &c.q) || !take(a[1], false, &c.k) || !take(a[2], false, &c.wq) ||
      !take(a[3], false, &c.wk) || !take(a[4], false, &c.cos) || !take(a[5], false, &c.sin) ||
      !take(a[6], true, &c.positions) || !take(a[7], &c.eps) || !unwatched())
    return none();
  const bool rec = recorded({&c.q, &c.k, &c.wq, &c.wk});
  for (const Tensor* t : {&c.q, &c.k, &c.wq, &c.wk, &c.cos, &c.sin})
    if (!no_tangent(*t)) return none();
  Tensor yq, yk;
  bool ok = false;
  {
    pybind11::gil_scoped_release nogil;
    ok = rope_rows(c, &yq, &yk);
  }
  if (!ok) return none();
  if (rec) {
    const variable_list o = NormRope::apply(c.q, c.k, c.wq, c.wk, &c, &yq, &yk);
    yq = o[0], yk = o[1];
  }
  return Py_BuildValue("(NN)", wrap(yq), wrap(yk));
  END_HANDLE_TH_ERRORS
}

// embedding(ids, weight, scale, padding_idx) -> rows
PyObject* py_embedding(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor ids, w, out;
  double scale = 0;
  int64_t padding = -1;
  if (n != 4 || !take(a[0], false, &ids) || !take(a[1], false, &w) || !take(a[2], &scale) || !take(a[3], &padding) ||
      padding < -1 || !unwatched())
    return none();
  const bool rec = recorded({&w});
  if (!no_tangent(w)) return none();
  bool ok = false;
  {
    pybind11::gil_scoped_release nogil;
    ok = w.dim() == 2 && padding < std::max<int64_t>(1, w.size(0)) && embedding_rows(ids, w, scale, &out);
  }
  if (!ok) return none();
  if (rec) out = Embedding::apply(w, ids, &out, scale, padding);
  return wrap(out);
  END_HANDLE_TH_ERRORS
}

}  // namespace attnres_torch
