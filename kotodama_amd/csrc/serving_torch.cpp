// The serving operators on the native call path (attnres_torch.cpp says what
// that is).  They are not differentiable, so a call that autograd would record is left
// to the Python layer (paged.py), as is any that the kernels do not take as it stands.

#include "attnres_torch_common.h"

namespace attnres_torch {
namespace {

// Whole numbers on the tensors' device, one contiguous dimension of n.
bool lengths(const Tensor& t, const Tensor& ref, int64_t n) {
  return dense(t) && (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) &&
         t.get_device() == ref.get_device() && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}
int index_code(const Tensor& t) {
  return t.defined() && t.scalar_type() == at::kLong ? ATTNRES_INDEX_I64 : ATTNRES_INDEX_I32;
}
// An int32 tensor on the reference's device, contiguous.
bool int32(const Tensor& t, const Tensor& ref) {
  return dense(t) && t.scalar_type() == at::kInt && t.get_device() == ref.get_device() && t.is_contiguous();
}
bool table_ok(const Tensor& t) {
  return dense(t) && t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) <= INT32_MAX && t.size(1) <= INT32_MAX &&
         (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
}

// Floating rows in 16-byte pieces: the strides of all dimensions but the last.
struct Pieces {
  int64_t s[3] = {0, 0, 0};
  bool ok = false;
  explicit Pieces(const Tensor& t) {
    if (!t.defined() || !dense(t) || !dtype_ok(t.scalar_type()) || t.dim() < 3 || t.dim() > 4) return;
    const int last = (int)t.dim() - 1;
    if (t.size(last) > 1 && t.stride(last) != 1) return;
    const int64_t m = 16 / (int64_t)t.element_size();
    if (t.numel() > 0 && (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) != 0) return;
    for (int i = 0; i <= last; ++i)
      if (t.size(i) > INT32_MAX) return;
    for (int i = 0; i < last; ++i) {
      s[i] = t.stride(i);
      if (t.size(i) > 1 && (s[i] % m != 0 || s[i] < 0)) return;
    }
    ok = true;
  }
};

bool cache_ok(const Tensor& k, const Tensor& v) {
  return k.defined() && k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && v.is_cuda() &&
         v.get_device() == k.get_device() && k.size(1) > 0;
}

Tensor ints(int64_t n, const Tensor& like) { return empty({n}, at::kInt, like.device()); }

// A tensor that a kernel wrote in place: what autograd saved of it before is out of date.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

struct SlotsCall {
  Tensor table, held, change, free_pages, free_count;
  int64_t page = 0;
  bool fits() const {
    return table.defined() && table_ok(table) && lengths(held, table, table.size(0)) &&
           lengths(change, table, table.size(0)) && int32(free_pages, table) && free_pages.dim() == 1 &&
           free_pages.size(0) <= INT32_MAX && int32(free_count, table) && free_count.numel() == 1 && page > 0 &&
           page <= INT32_MAX;
  }
};

bool take_slots(PyObject* const* a, SlotsCall* c) {
  return take(a[0], false, &c->table) && take(a[1], false, &c->held) && take(a[2], false, &c->change) &&
         take(a[3], false, &c->free_pages) && take(a[4], false, &c->free_count) && take(a[5], &c->page);
}

}  // namespace

// paged_slots(block_table, held, new, free_pages, free_count, page_size, num_tokens)
//   -> (slots, positions, q_starts, kv_lens, free_count)
PyObject* py_paged_slots(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  SlotsCall c;
  int64_t tokens = 0;
  if (n != 7 || !take_slots(a, &c) || !take(a[6], &tokens) || !unwatched() || !c.fits()) return none();
  Tensor out[5];
  bool ok = false;
  {
    pybind11::gil_scoped_release nogil;
    ATTNRES_RECORD("attnres_hip::paged_slots");
    const Tensor& t = c.table;
    const int64_t b = t.size(0), sizes[5] = {tokens, tokens, b + 1, b, 1};
    for (int i = 0; i < 5; ++i) out[i] = ints(sizes[i], t);
    const OnDevice on(t);
    ok = attnres_paged_slots(t.mutable_data_ptr(), t.stride(0), (int)b, (int)t.size(1), ptr(c.held), index_code(c.held),
                             ptr(c.change), index_code(c.change), ptr(c.free_pages), (int)c.free_pages.size(0),
                             ptr(c.free_count), (int)c.page, tokens, out_ptr<void>(out[0]), out_ptr<void>(out[1]),
                             out_ptr<void>(out[2]), out_ptr<void>(out[3]), out_ptr<void>(out[4]),
                             on.stream) == ATTNRES_OK;
    if (ok) written(t);
  }
  if (!ok) return none();
  return Py_BuildValue("(NNNNN)", wrap(out[0]), wrap(out[1]), wrap(out[2]), wrap(out[3]), wrap(out[4]));
  END_HANDLE_TH_ERRORS
}

// paged_release(block_table, held, kept, free_pages, free_count, page_size) -> free_count
PyObject* py_paged_release(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  SlotsCall c;
  if (n != 6 || !take_slots(a, &c) || !unwatched() || !c.fits()) return none();
  Tensor out;
  bool ok = false;
  {
    pybind11::gil_scoped_release nogil;
    ATTNRES_RECORD("attnres_hip::paged_release");
    const Tensor& t = c.table;
    out = ints(1, t);
    const OnDevice on(t);
    ok = attnres_paged_release(ptr(t), t.stride(0), (int)t.size(0), (int)t.size(1), ptr(c.held), index_code(c.held),
                               ptr(c.change), index_code(c.change), out_ptr<void>(c.free_pages),
                               (int)c.free_pages.size(0), ptr(c.free_count), (int)c.page, out_ptr<void>(out),
                               on.stream) == ATTNRES_OK;
    if (ok) written(c.free_pages);
  }
  return ok ? wrap(out) : none();
  END_HANDLE_TH_ERRORS
}

// paged_write(k, v, k_cache, v_cache, slots) -> True
PyObject* py_paged_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor k, v, kc, vc, slots;
  if (n != 5 || !take(a[0], false, &k) || !take(a[1], false, &v) || !take(a[2], false, &kc) ||
      !take(a[3], false, &vc) || !take(a[4], false, &slots) || !unwatched() || recorded({&k, &v, &kc, &vc}))
    return none();
  for (const Tensor* t : {&k, &v, &kc, &vc})
    if (!no_tangent(*t)) return none();
  if (!cache_ok(kc, vc) || k.dim() != 3 || v.sizes() != k.sizes() || k.size(1) != kc.size(1) || k.size(2) != kc.size(3))
    return none();
  for (const Tensor* t : {&k, &v})
    if (t->scalar_type() != kc.scalar_type() || !t->is_cuda() || t->get_device() != kc.get_device()) return none();
  const Pieces sk(k), sv(v), skc(kc), svc(vc);
  if (!sk.ok || !sv.ok || !skc.ok || !svc.ok || !lengths(slots, kc, k.size(0))) return none();
  bool ok = false;
  {
    pybind11::gil_scoped_release nogil;
    ATTNRES_RECORD("attnres_hip::paged_write");
    const OnDevice on(kc);
    ok = attnres_paged_write(ptr(k), sk.s, ptr(v), sv.s, k.size(0), (int)k.size(1), (int)k.size(2),
                             code(k.scalar_type()), out_ptr<void>(kc), skc.s, out_ptr<void>(vc), svc.s, kc.size(0),
                             (int)kc.size(2), ptr(slots), index_code(slots), on.stream) == ATTNRES_OK;
    if (ok) {
      written(kc);
      written(vc);
    }
  }
  if (!ok) return none();
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// paged_attention(q, k_cache, v_cache, block_table, kv_lens, q_starts, scale, want_lse) -> out or (out, lse)
PyObject* py_paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, kc, vc, table, kv_lens, q_starts, out, lse;
  double scale = 0;
  bool want_lse = false;
  if (n != 8 || !take(a[0], false, &q) || !take(a[1], false, &kc) || !take(a[2], false, &vc) ||
      !take(a[3], false, &table) || !take(a[4], false, &kv_lens) || !take(a[5], true, &q_starts) ||
      !take(a[6], &scale) || !take(a[7], &want_lse) || !unwatched() || recorded({&q, &kc, &vc}))
    return none();
  for (const Tensor* t : {&q, &kc, &vc})
    if (!no_tangent(*t)) return none();
  if (!cache_ok(kc, vc) || q.dim() != 3 || q.size(2) != kc.size(3) || q.size(1) < 1 || q.size(1) % kc.size(1) != 0 ||
      q.scalar_type() != kc.scalar_type() || !q.is_cuda() || q.get_device() != kc.get_device())
    return none();
  const Pieces sq(q), sk(kc), sv(vc);
  if (!sq.ok || !sk.ok || !sv.ok || !table_ok(table) || table.get_device() != kc.get_device()) return none();
  const int64_t b = table.size(0);
  if (!lengths(kv_lens, kc, b) || (q_starts.defined() ? !lengths(q_starts, kc, b + 1) : q.size(0) != b)) return none();
  bool ok = false;
  {
    pybind11::gil_scoped_release nogil;
    ATTNRES_RECORD("attnres_hip::paged_attention");
    const int64_t tokens = q.size(0);
    const int h = (int)q.size(1), hk = (int)kc.size(1), d = (int)q.size(2), dt = code(q.scalar_type());
    const int page = (int)kc.size(2), width = (int)table.size(1);
    out = empty(q.sizes(), q.scalar_type(), q.device());
    if (want_lse) lse = empty({tokens, h}, at::kFloat, q.device());
    const int64_t so[2] = {(int64_t)h * d, d};
    const OnDevice on(q);
    int64_t bytes = 0;
    if (attnres_paged_attention_workspace_size(tokens, (int)b, h, hk, d, dt, width, page, &bytes) == ATTNRES_OK) {
      const Tensor ws = bytes > 0 ? workspace(bytes, q.device()) : Tensor();
      ok = attnres_paged_attention_fwd(ptr(q), sq.s, ptr(kc), sk.s, ptr(vc), sv.s, tokens, (int)b, h, hk, d, dt,
                                       kc.size(0), page, ptr(table), table.stride(0), width, ptr(kv_lens),
                                       index_code(kv_lens), ptr(q_starts), index_code(q_starts), (float)scale,
                                       out_ptr<void>(out), so, out_ptr<float>(lse),
                                       ws.defined() ? ws.mutable_data_ptr() : nullptr, bytes, on.stream) == ATTNRES_OK;
    }
  }
  if (!ok) return none();
  if (!want_lse) return wrap(out);
  return Py_BuildValue("(NN)", wrap(out), wrap(lse));
  END_HANDLE_TH_ERRORS
}

// verify_drafts(logits, ids, q_starts, uniforms, draft_probs, temperature) -> (tokens, counts)
PyObject* py_verify_drafts(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor logits, ids, q_starts, uniforms, draft, tokens, counts;
  double temperature = 0;
  if (n != 6 || !take(a[0], false, &logits) || !take(a[1], false, &ids) || !take(a[2], false, &q_starts) ||
      !take(a[3], false, &uniforms) || !take(a[4], true, &draft) || !take(a[5], &temperature) || !unwatched() ||
      recorded({&logits, &uniforms, &draft}))
    return none();
  for (const Tensor* t : {&logits, &uniforms, &draft})
    if (!no_tangent(*t)) return none();
  if (temperature != 0 && !(temperature >= 1e-6 && temperature < 1e38)) return none();  // before it is rounded to fp32
  auto rows_ok = [](const Tensor& t) {
    return dense(t) && dtype_ok(t.scalar_type()) && t.dim() == 2 && t.size(1) > 0 && t.size(1) <= INT32_MAX &&
           (t.stride(1) == 1 || t.size(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
  };
  if (!rows_ok(logits) || !lengths(ids, logits, logits.size(0)) || q_starts.dim() != 1 || q_starts.size(0) < 1 ||
      q_starts.size(0) > INT32_MAX || !lengths(q_starts, logits, q_starts.size(0)) || !plain(uniforms) ||
      uniforms.scalar_type() != at::kFloat || uniforms.dim() != 2 || uniforms.size(0) != logits.size(0) ||
      uniforms.size(1) != 2 || uniforms.get_device() != logits.get_device())
    return none();
  if (draft.defined() &&
      (!rows_ok(draft) || draft.sizes() != logits.sizes() || draft.get_device() != logits.get_device()))
    return none();
  bool ok = false;
  {
    pybind11::gil_scoped_release nogil;
    ATTNRES_RECORD("attnres_hip::verify_drafts");
    const int64_t rows = logits.size(0), seqs = q_starts.size(0) - 1;
    int64_t bytes = 0;
    const OnDevice on(logits);
    if (attnres_verify_drafts_workspace_size(rows, (int)seqs, (int)logits.size(1), &bytes) == ATTNRES_OK) {
      tokens = empty({rows}, ids.scalar_type(), logits.device());
      counts = ints(seqs, logits);
      const Tensor ws = workspace(bytes, logits.device());
      ok = attnres_verify_drafts(ptr(logits), logits.stride(0), code(logits.scalar_type()), ptr(draft),
                                 draft.defined() ? draft.stride(0) : 0,
                                 draft.defined() ? code(draft.scalar_type()) : ATTNRES_DTYPE_F32, rows,
                                 (int)logits.size(1), ptr(ids), index_code(ids), ptr(q_starts), index_code(q_starts),
                                 (int)seqs, static_cast<const float*>(ptr(uniforms)), (float)temperature,
                                 out_ptr<void>(tokens), out_ptr<void>(counts), ws.mutable_data_ptr(), bytes,
                                 on.stream) == ATTNRES_OK;
    }
  }
  if (!ok) return none();
  return Py_BuildValue("(NN)", wrap(tokens), wrap(counts));
  END_HANDLE_TH_ERRORS
}

}  // namespace attnres_torch
