// The Python wrappers' short way into the ragged steps (spock_b200._binding).
// At decode sizes a call's time is the host's: checking nine tensors, taking
// their strides apart and converting seventeen arguments costs Python three
// times what the library's own call does. Each function here makes the checks
// of its wrapper in spock_b200/__init__.py and the C call; where a check does
// not pass (or a stream is named) it returns None and the wrapper goes on by
// itself, with its error messages. A status other than SPOCK_OK is returned as
// a number for Context.check. Tensors are torch's; the computation is the
// library's.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/spock_b200.h"

namespace {

using at::Tensor;
constexpr auto kHalf = at::kHalf, kBF16 = at::kBFloat16, kFloat = at::kFloat, kInt = at::kInt;

// An argument: a tensor, nothing (None), or neither.
struct Arg {
  const Tensor* t = nullptr;
  bool bad = false;
  explicit Arg(PyObject* o) {
    if (o == Py_None) return;
    if (THPVariable_Check(o))
      t = &THPVariable_Unpack(o);
    else
      bad = true;
  }
  bool rows(at::ScalarType type, int64_t ndim, int d) const {  // contiguous rows, any strides before
    return t && t->scalar_type() == type && t->dim() == ndim && t->is_cuda() && t->get_device() == d &&
           (t->stride(-1) == 1 || t->size(-1) <= 1);
  }
  bool whole(at::ScalarType type, int64_t ndim, int d) const {
    return t && t->scalar_type() == type && t->dim() == ndim && t->is_cuda() && t->get_device() == d &&
           t->is_contiguous();
  }
  bool none() const { return !t && !bad; }
  void* ptr() const { return t ? t->data_ptr() : nullptr; }
};
int64_t row_stride(const Tensor& t) {
  if (t.size(0) > 1) return t.stride(0);
  return t.dim() == 2 ? (t.size(1) + 7) / 8 * 8 : t.size(1) * t.size(2);
}
int64_t at_dim(const Tensor& t, int64_t dim, int64_t otherwise) { return t.size(dim) > 1 ? t.stride(dim) : otherwise; }

int device_of(const Arg& a) { return a.t && a.t->is_cuda() ? (int)a.t->get_device() : -1; }
Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
  at::AutoDispatchBelowADInplaceOrView guard;
  return at::empty(shape, like.options().dtype(type));
}
PyObject* none() { Py_RETURN_NONE; }
PyObject* code(int rc) { return PyLong_FromLong(rc); }
spock_ctx* ctx_of(PyObject* o) { return static_cast<spock_ctx*>(PyLong_AsVoidPtr(o)); }

bool paged(spock_paged_kv& kv, const Arg& k, const Arg& v, const Arg& table, const Arg& len, const Arg& start,
           at::ScalarType type, int d) {
  if ((type != kHalf && type != kBF16) || !k.rows(type, 4, d) || !v.rows(type, 4, d) || !table.rows(kInt, 2, d) ||
      !len.whole(kInt, 1, d) || !start.whole(kInt, 1, d) || k.t->sizes() != v.t->sizes() ||
      k.t->strides() != v.t->strides())
    return false;
  const int64_t batch = start.t->size(0) - 1, width = table.t->size(1);
  if (batch < 1 || table.t->size(0) != batch || len.t->size(0) != batch) return false;
  const int64_t pages = k.t->size(0), page = k.t->size(1), heads = k.t->size(2), dim = k.t->size(3);
  if (batch > INT32_MAX || pages > INT32_MAX || page > INT32_MAX || heads > INT32_MAX || width > INT32_MAX) return false;
  kv.k = k.ptr();
  kv.v = v.ptr();
  kv.page_stride = at_dim(*k.t, 0, page * heads * dim);
  kv.pos_stride = at_dim(*k.t, 1, heads * dim);
  kv.head_stride = at_dim(*k.t, 2, dim);
  kv.page_table = static_cast<const int32_t*>(table.ptr());
  kv.table_stride = batch > 1 ? table.t->stride(0) : std::max(table.t->stride(0), width);
  kv.kv_len = static_cast<const int32_t*>(len.ptr());
  kv.table_width = (int32_t)width;
  kv.num_pages = (int32_t)pages;
  kv.page_size = (int32_t)page;
  kv.kv_heads = (int32_t)heads;
  kv.head_dim = (int32_t)dim;
  kv.dtype = type == kHalf ? SPOCK_F16 : SPOCK_BF16;
  return true;
}
const int32_t* i32(const Arg& a) { return static_cast<const int32_t*>(a.ptr()); }
const float* f32(const Arg& a) { return static_cast<const float*>(a.ptr()); }

// ctx, proj, start, k_pages, v_pages, page_table, kv_len, rope, q_norm, k_norm, gated, eps, q_out
PyObject* prep(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13) return none();
  const Arg proj(a[1]), start(a[2]), k(a[3]), v(a[4]), table(a[5]), len(a[6]), rope(a[7]), qn(a[8]), kn(a[9]), qo(a[12]);
  const int d = device_of(proj), gated = PyObject_IsTrue(a[10]);
  const double eps = PyFloat_AsDouble(a[11]);
  if (PyErr_Occurred()) return PyErr_Clear(), none();
  if (d < 0 || !k.t) return none();
  const auto type = k.t->scalar_type();
  spock_paged_kv kv{};
  if (!proj.rows(type, 2, d) || !paged(kv, k, v, table, len, start, type, d) ||
      !(rope.none() || (rope.whole(kFloat, 3, d) && rope.t->size(2) == 2)) ||
      !(qn.none() || (qn.whole(type, 1, d) && qn.t->size(0) == kv.head_dim)) ||
      !(kn.none() || (kn.whole(type, 1, d) && kn.t->size(0) == kv.head_dim)))
    return none();
  const int64_t total = proj.t->size(0), width = proj.t->size(1), per = gated ? 2 : 1;
  const int64_t heads = kv.head_dim ? width / kv.head_dim - 2 * (int64_t)kv.kv_heads : 0, q_heads = heads / per;
  if (heads <= 0 || width % kv.head_dim || heads % per || q_heads > INT32_MAX) return none();
  Tensor out;
  if (qo.none()) {
    out = fresh({total, q_heads, kv.head_dim}, type, *proj.t);
  } else {
    if (!qo.whole(type, 3, d) || qo.t->size(0) != total || qo.t->size(1) != q_heads || qo.t->size(2) != kv.head_dim)
      return none();
    out = *qo.t;
  }
  void* st = c10::cuda::getCurrentCUDAStream(d).stream();
  spock_ctx* ctx = ctx_of(a[0]);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = spock_paged_attention_prep(ctx, &kv, (int32_t)(start.t->size(0) - 1), i32(start), total, proj.ptr(),
                                  row_stride(*proj.t), (int32_t)q_heads, gated, qn.ptr(), kn.ptr(), (float)eps, f32(rope),
                                  rope.t ? rope.t->size(0) : 0, rope.t ? (int32_t)(2 * rope.t->size(1)) : 0,
                                  out.data_ptr(), st);
  Py_END_ALLOW_THREADS
  return rc == SPOCK_OK ? THPVariable_Wrap(out) : code(rc);
  END_HANDLE_TH_ERRORS
}

// ctx, q, start, k_pages, v_pages, page_table, kv_len, scale, gate, out, workspace
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11) return none();
  const Arg q(a[1]), start(a[2]), k(a[3]), v(a[4]), table(a[5]), len(a[6]), gate(a[8]), given(a[9]), space(a[10]);
  const int d = device_of(q);
  const double scale = PyFloat_AsDouble(a[7]);
  if (PyErr_Occurred()) return PyErr_Clear(), none();
  if (d < 0 || !k.t) return none();
  const auto type = k.t->scalar_type();
  spock_paged_kv kv{};
  if (!q.rows(type, 3, d) || !paged(kv, k, v, table, len, start, type, d) || q.t->size(2) != kv.head_dim ||
      q.t->size(1) > INT32_MAX || !(gate.none() || (gate.rows(type, 3, d) && gate.t->sizes() == q.t->sizes())) ||
      !(given.none() || (given.whole(type, 3, d) && given.t->sizes() == q.t->sizes())) ||
      !(space.none() || space.whole(at::kByte, 1, d)))
    return none();
  const int64_t heads = q.t->size(1), dim = kv.head_dim;
  spock_ctx* ctx = ctx_of(a[0]);
  size_t bytes = 0;
  int rc = spock_paged_attention_workspace(ctx, (int32_t)heads, kv.kv_heads, kv.head_dim, &bytes);
  if (rc != SPOCK_OK) return code(rc);
  const Tensor out = given.t ? *given.t : fresh(q.t->sizes(), type, *q.t);
  const Tensor ws = space.t ? *space.t : fresh({(int64_t)bytes}, at::kByte, *q.t);
  void* st = c10::cuda::getCurrentCUDAStream(d).stream();
  Py_BEGIN_ALLOW_THREADS
  rc = spock_paged_attention(ctx, &kv, (int32_t)(start.t->size(0) - 1), i32(start), q.t->size(0), (int32_t)heads, q.ptr(),
                             row_stride(*q.t), at_dim(*q.t, 1, dim), gate.ptr(), gate.t ? row_stride(*gate.t) : 0,
                             gate.t ? at_dim(*gate.t, 1, dim) : 0, (float)scale, out.data_ptr(), ws.data_ptr(),
                             (size_t)ws.numel(), st);
  Py_END_ALLOW_THREADS
  return rc == SPOCK_OK ? THPVariable_Wrap(out) : code(rc);
  END_HANDLE_TH_ERRORS
}

// ctx, (heads, key_dim, value_dim, conv_kernel, eps), conv_weight, a_log_bias, norm_weight, qkv, conv_state, state, a,
// b, z, start, counts, state_out, conv_out, out; True: done
PyObject* span(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 20) return none();
  spock_dn_layer L{};
  L.num_heads = (int32_t)PyLong_AsLong(a[1]);
  L.key_dim = (int32_t)PyLong_AsLong(a[2]);
  L.value_dim = (int32_t)PyLong_AsLong(a[3]);
  L.conv_kernel = (int32_t)PyLong_AsLong(a[4]);
  L.eps = (float)PyFloat_AsDouble(a[5]);
  if (PyErr_Occurred()) return PyErr_Clear(), none();
  const Arg cw(a[6]), bias(a[7]), norm(a[8]), qkv(a[9]), conv(a[10]), state(a[11]), ga(a[12]), gb(a[13]), z(a[14]),
      start(a[15]), counts(a[16]), state_out(a[17]), conv_out(a[18]), out(a[19]);
  const int d = device_of(qkv);
  if (d < 0 || !cw.t || L.num_heads <= 0 || L.key_dim != 128 || L.value_dim != 128 || L.conv_kernel != 4) return none();
  const int64_t h = L.num_heads, inner = h * 128;
  auto is = [](const Arg& x, std::initializer_list<int64_t> shape) {
    return x.none() || x.t->sizes() == at::IntArrayRef(shape.begin(), shape.size());
  };
  if (!start.whole(kInt, 1, d) || !qkv.rows(kHalf, 2, d) || !ga.rows(kHalf, 2, d) || !gb.rows(kHalf, 2, d) ||
      !(z.none() || z.rows(kHalf, 2, d)) || !conv.whole(kHalf, 3, d) || !state.whole(kFloat, 4, d) ||
      !(counts.none() || counts.whole(kInt, 1, d)) || !(state_out.none() || state_out.whole(kFloat, 4, d)) ||
      !(conv_out.none() || conv_out.whole(kHalf, 3, d)) || !(out.none() || out.whole(kHalf, 2, d)) ||
      !bias.whole(kFloat, 2, d) || !norm.whole(kFloat, 1, d) || !cw.whole(cw.t->scalar_type(), cw.t->dim(), d) ||
      cw.t->element_size() != 2 || cw.t->numel() != 3 * inner * 4)
    return none();
  const int64_t batch = start.t->size(0) - 1, total = qkv.t->size(0);
  if (batch < 1 || batch > INT32_MAX || !is(qkv, {total, 3 * inner}) || !is(ga, {total, h}) || !is(gb, {total, h}) ||
      !is(z, {total, inner}) || !is(conv, {batch, 3 * inner, 4}) || !is(conv_out, {batch, 3 * inner, 4}) ||
      !is(state, {batch, h, 128, 128}) || !is(state_out, {batch, h, 128, 128}) || !is(out, {total, inner}) ||
      !is(counts, {batch}) || !is(bias, {h, 2}) || !is(norm, {128}) ||
      (total > 1 && ga.t->stride(0) != gb.t->stride(0)))
    return none();
  L.conv_weight = cw.ptr();
  L.a_log_bias = f32(bias);
  L.norm_weight = f32(norm);
  Tensor made;
  if (out.none() && state_out.none()) made = fresh({total, inner}, kHalf, *qkv.t);
  void* to = made.defined() ? made.data_ptr() : out.ptr();
  void* st = c10::cuda::getCurrentCUDAStream(d).stream();
  spock_ctx* ctx = ctx_of(a[0]);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = spock_deltanet_decode_span(ctx, &L, (int32_t)batch, i32(start), i32(counts), total, qkv.ptr(), row_stride(*qkv.t),
                                  ga.ptr(), gb.ptr(), row_stride(*ga.t), z.ptr(), z.t ? row_stride(*z.t) : 0, conv.ptr(),
                                  f32(state), conv_out.ptr(), static_cast<float*>(state_out.ptr()), to, st);
  Py_END_ALLOW_THREADS
  if (rc != SPOCK_OK) return code(rc);
  if (made.defined()) return THPVariable_Wrap(made);
  if (out.t) return Py_NewRef(a[19]);
  return PyTuple_Pack(2, a[17], a[18]);
  END_HANDLE_TH_ERRORS
}

// ctx, logits, tokens, start, u_accept, u_sample, temperature, draft_probs, emitted, out_tokens, workspace
PyObject* verify(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11) return none();
  const Arg logits(a[1]), tokens(a[2]), start(a[3]), ua(a[4]), us(a[5]), temp(a[6]), probs(a[7]), em(a[8]), ot(a[9]),
      space(a[10]);
  const int d = device_of(logits);
  if (d < 0) return none();
  const auto type = logits.t->scalar_type();
  if ((type != kFloat && type != kHalf && type != kBF16) || !logits.rows(type, 2, d) || !start.whole(kInt, 1, d)) return none();
  const int64_t total = logits.t->size(0), vocab = logits.t->size(1), batch = start.t->size(0) - 1;
  auto vec = [&](const Arg& x, at::ScalarType s, int64_t len) { return x.whole(s, 1, d) && x.t->size(0) == len; };
  if (batch < 1 || batch > INT32_MAX || !vec(tokens, kInt, total) || !vec(ua, kFloat, total) || !vec(us, kFloat, batch) ||
      !(temp.none() || vec(temp, kFloat, batch)) ||
      !(probs.none() || (probs.rows(kFloat, 2, d) && probs.t->sizes() == logits.t->sizes())) ||
      !(em.none() || vec(em, kInt, batch)) || !(ot.none() || vec(ot, kInt, total)) ||
      !(space.none() || space.whole(at::kByte, 1, d)))
    return none();
  spock_ctx* ctx = ctx_of(a[0]);
  size_t bytes = 0;
  int rc = spock_draft_verify_workspace(ctx, total, vocab, (int32_t)batch, &bytes);
  if (rc != SPOCK_OK) return code(rc);
  const Tensor emitted = em.t ? *em.t : fresh({batch}, kInt, *logits.t), out = ot.t ? *ot.t : fresh({total}, kInt, *logits.t);
  const Tensor ws = space.t ? *space.t : fresh({(int64_t)bytes}, at::kByte, *logits.t);
  void* st = c10::cuda::getCurrentCUDAStream(d).stream();
  Py_BEGIN_ALLOW_THREADS
  rc = spock_draft_verify(ctx, type == kFloat ? SPOCK_F32 : type == kHalf ? SPOCK_F16 : SPOCK_BF16, logits.ptr(),
                          total > 1 ? logits.t->stride(0) : vocab, total, vocab, (int32_t)batch,
                          i32(start), i32(tokens), f32(probs),
                          probs.t ? (total > 1 ? probs.t->stride(0) : vocab) : 0, f32(temp), f32(ua), f32(us),
                          static_cast<int32_t*>(emitted.data_ptr()), static_cast<int32_t*>(out.data_ptr()), ws.data_ptr(),
                          (size_t)ws.numel(), st);
  Py_END_ALLOW_THREADS
  if (rc != SPOCK_OK) return code(rc);
  PyObject *x = THPVariable_Wrap(emitted), *y = x ? THPVariable_Wrap(out) : nullptr;
  if (!y) return Py_XDECREF(x), nullptr;
  PyObject* both = PyTuple_Pack(2, x, y);
  Py_DECREF(x);
  Py_DECREF(y);
  return both;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"paged_attention_prep", reinterpret_cast<PyCFunction>(prep), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(attention), METH_FASTCALL, nullptr},
    {"deltanet_decode_span", reinterpret_cast<PyCFunction>(span), METH_FASTCALL, nullptr},
    {"draft_verify", reinterpret_cast<PyCFunction>(verify), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
