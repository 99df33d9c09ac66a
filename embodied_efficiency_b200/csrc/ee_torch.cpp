// ee_torch.cpp -- native host side of the prompt-layer operators: what a call
// of rotary_embed, norm_rotary_embed, prompt_attention, int8_linear,
// int8_matmul, quantize_tokens and the operators of a cache does on the host,
// without the interpreter. A call of few tokens takes the GPU 3 to 8
// us; checks, allocations and argument conversion in Python took 13 to 17 us
// around it.
//
// Every function here takes the usual call -- aligned, contiguous tensors of
// the current device, no gradients, nothing to copy -- through the C ABI and
// returns its result, or returns None for any other call, launching nothing:
// the Python function of the same name then makes the copies or raises the
// error. So nothing here reports an argument error itself.
#include <Python.h>

#include <cfloat>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/ee_b200.h"

namespace {

using at::ScalarType;
using at::Tensor;

bool aligned(const Tensor& t) { return ((uintptr_t)t.data_ptr() & 15) == 0; }
bool act_type(ScalarType s) { return s == at::kBFloat16 || s == at::kHalf; }
int act_code(ScalarType s) { return s == at::kBFloat16 ? EE_BF16 : EE_F16; }

// The operands of one call; `ok` falls with the first that is not usual.
struct Call {
  bool ok = true;
  int dev = c10::cuda::current_device();
  const bool grad = at::GradMode::is_enabled();

  const Tensor* get(PyObject* o) {  // a CUDA tensor of the current device that asks for no gradient of either mode
    if (!ok || !THPVariable_Check(o)) return fail();
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.get_device() != dev || (grad && t.requires_grad()) || t._fw_grad(0).defined()) return fail();
    return &t;
  }
  const Tensor* fail() {
    ok = false;
    return nullptr;
  }
  bool need(bool cond) { return ok = ok && cond; }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(dev).stream(); }
};

// Lets the interpreter's other threads run while a call allocates and
// launches: both may wait for the GPU (an allocation that needs a
// synchronisation, a launch queue that is full). Taken once the operands have
// been looked at; results become Python objects after its end.
class NoGil {
  PyThreadState* state_ = PyEval_SaveThread();

 public:
  NoGil() = default;
  NoGil(const NoGil&) = delete;
  ~NoGil() { PyEval_RestoreThread(state_); }
};

PyObject* none() { Py_RETURN_NONE; }
PyObject* give(int rc, const Tensor& t) { return rc == EE_OK ? THPVariable_Wrap(t) : none(); }
PyObject* give(int rc, const Tensor& t, const Tensor& u) {
  if (rc != EE_OK) return none();
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(t));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(u));
  return r;
}

bool heads_ok(const Tensor& t) {
  return t.dim() == 3 && act_type(t.scalar_type()) && t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 &&
         aligned(t);
}

// ---------------------------------------------------------------------------
// linears
// ---------------------------------------------------------------------------
struct Linear {
  int64_t n, k;
  const void *weight, *scales, *bias = nullptr, *residual = nullptr;
  int scale_dtype, epilogue = 0;
};
// weight, scales, bias, gelu, residual of a product with outputs of `type` and shape [..., n]
bool linear(Call& c, PyObject* const* a, ScalarType type, int64_t m, at::IntArrayRef lead, Linear& l) {
  const Tensor *w = c.get(a[0]), *s = c.get(a[1]);
  if (!c.need(w && s && w->dim() == 2 && w->scalar_type() == at::kChar && w->is_contiguous() && aligned(*w))) return false;
  l.n = w->size(0);
  l.k = w->size(1);
  const bool f32 = s->scalar_type() == at::kFloat;
  if (!c.need((f32 || s->scalar_type() == at::kHalf) && s->numel() == l.n && s->is_contiguous() && aligned(*s) &&
              l.k >= 16 && l.k % 16 == 0 && l.k <= 131056 && m > 0 && l.n > 0))
    return false;
  l.weight = w->data_ptr();
  l.scales = s->data_ptr();
  l.scale_dtype = f32 ? EE_F32 : EE_F16;
  if (a[2] != Py_None) {
    const Tensor* b = c.get(a[2]);
    if (!c.need(b && b->scalar_type() == type && b->numel() == l.n && b->is_contiguous() && aligned(*b))) return false;
    l.bias = b->data_ptr();
    l.epilogue |= EE_EPI_BIAS;
  }
  if (!c.need(PyBool_Check(a[3]))) return false;
  if (a[3] == Py_True) l.epilogue |= EE_EPI_GELU;
  if (a[4] != Py_None) {
    const Tensor* r = c.get(a[4]);
    if (!c.need(r && a[3] == Py_False && r->scalar_type() == type && r->is_contiguous() && aligned(*r) &&
                r->dim() == (int64_t)lead.size() + 1 && r->sizes().slice(0, lead.size()) == lead && r->size(-1) == l.n))
      return false;
    l.residual = r->data_ptr();
    l.epilogue |= EE_EPI_RESIDUAL;
  }
  return true;
}
Tensor output(const Tensor& like, at::IntArrayRef lead, int64_t n, ScalarType type) {
  c10::SmallVector<int64_t, 6> shape(lead.begin(), lead.end());
  shape.push_back(n);
  return at::empty(shape, like.options().dtype(type));
}

// int8_linear(x, weight, scales, bias, gelu, residual)
PyObject* int8_linear(PyObject*, PyObject* const* a, Py_ssize_t argc) {
  if (argc != 6) return none();
  Call c;
  const Tensor* x = c.get(a[0]);
  if (!c.need(x && x->dim() >= 1 && act_type(x->scalar_type()) && x->is_contiguous() && aligned(*x))) return none();
  const int64_t k = x->size(-1), m = k > 0 ? x->numel() / k : 0;
  const auto lead = x->sizes().slice(0, x->dim() - 1);
  Linear l;
  if (!linear(c, a + 1, x->scalar_type(), m, lead, l) || !c.need(l.k == k)) return none();
  Tensor y;
  int rc;
  {
    NoGil others;
    y = output(*x, lead, l.n, x->scalar_type());
    const size_t need = ee_int8_linear_workspace_bytes(m, k);
    const Tensor ws = at::empty({(int64_t)need}, x->options().dtype(at::kChar));
    rc = ee_int8_linear(x->data_ptr(), k, l.weight, l.scales, l.bias, l.residual, y.data_ptr(), ws.data_ptr(), need, m,
                        l.n, k, l.scale_dtype, act_code(x->scalar_type()), l.epilogue, c.stream());
  }
  return give(rc, y);
}

// int8_matmul(xq, x_scale, weight, scales, bias, gelu, residual, dtype)
PyObject* int8_matmul(PyObject*, PyObject* const* a, Py_ssize_t argc) {
  if (argc != 8 || !THPDtype_Check(a[7])) return none();
  const ScalarType type = reinterpret_cast<THPDtype*>(a[7])->scalar_type;
  Call c;
  const Tensor *x = c.get(a[0]), *sx = c.get(a[1]);
  if (!c.need(x && sx && act_type(type) && x->dim() >= 1 && x->scalar_type() == at::kChar && x->is_contiguous() &&
              aligned(*x)))
    return none();
  const int64_t k = x->size(-1), m = k > 0 ? x->numel() / k : 0;
  const auto lead = x->sizes().slice(0, x->dim() - 1);
  Linear l;
  if (!linear(c, a + 2, type, m, lead, l) ||
      !c.need(l.k == k && sx->scalar_type() == at::kFloat && sx->numel() == m && sx->is_contiguous() && aligned(*sx)))
    return none();
  Tensor y;
  int rc;
  {
    NoGil others;
    y = output(*x, lead, l.n, type);
    rc = ee_int8_gemm(static_cast<const int8_t*>(x->data_ptr()), static_cast<const float*>(sx->data_ptr()), l.weight,
                      l.scales, l.bias, l.residual, y.data_ptr(), m, l.n, k, l.scale_dtype, act_code(type), l.epilogue,
                      c.stream());
  }
  return give(rc, y);
}

// quantize_tokens(x) -> (codes, scales)
PyObject* quantize_tokens(PyObject*, PyObject* const* a, Py_ssize_t argc) {
  if (argc != 1) return none();
  Call c;
  const Tensor* x = c.get(a[0]);
  if (!c.need(x && x->dim() >= 1 && act_type(x->scalar_type()) && x->is_contiguous() && aligned(*x))) return none();
  const int64_t k = x->size(-1);
  if (!c.need(k >= 16 && k % 16 == 0 && k <= 131056 && x->numel() > 0)) return none();
  const auto lead = x->sizes().slice(0, x->dim() - 1);
  Tensor q, s;
  int rc;
  {
    NoGil others;
    q = at::empty(x->sizes(), x->options().dtype(at::kChar));
    s = output(*x, lead, 1, at::kFloat);
    rc = ee_quantize_tokens(x->data_ptr(), k, static_cast<int8_t*>(q.data_ptr()), static_cast<float*>(s.data_ptr()),
                            x->numel() / k, k, act_code(x->scalar_type()), c.stream());
  }
  return give(rc, q, s);
}

// ---------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------
// q, k, positions, sections, turns, interleaved; turns: the table of hd / 2
// frequencies on the device. w: q_weight, k_weight, eps, or nothing
PyObject* rotary(PyObject* const* a, PyObject* const* w) {
  Call c;
  const Tensor *q = c.get(a[0]), *k = c.get(a[1]), *pos = c.get(a[2]), *tab = c.get(a[4]);
  if (!c.need(q && k && pos && tab && heads_ok(*q) && heads_ok(*k) && PyTuple_Check(a[3]) && PyBool_Check(a[5])))
    return none();
  const int64_t t = q->size(0), hd = q->size(2), axes = PyTuple_GET_SIZE(a[3]);
  const bool p64 = pos->scalar_type() == at::kLong;
  int32_t sections[4] = {};
  int64_t sum = 0;
  if (!c.need(axes >= 1 && axes <= 4)) return none();
  for (int64_t i = 0; i < axes; ++i) {
    PyObject* o = PyTuple_GET_ITEM(a[3], i);
    const long v = PyLong_Check(o) ? PyLong_AsLong(o) : -1;
    if (v < 0 || v > hd) {
      PyErr_Clear();
      return none();
    }
    sections[i] = (int32_t)v;
    sum += v;
  }
  if (!c.need(sum == hd / 2 && hd % 2 == 0 && t > 0 && k->size(0) == t && k->size(2) == hd &&
              k->scalar_type() == q->scalar_type() && (p64 || pos->scalar_type() == at::kInt) && pos->is_contiguous() &&
              (pos->dim() == 2 ? pos->size(0) == axes && pos->size(1) == t : pos->dim() == 1 && axes == 1 && pos->size(0) == t) &&
              tab->scalar_type() == at::kLong && tab->numel() == hd / 2 && tab->is_contiguous()))
    return none();
  const bool interleaved = a[5] == Py_True;
  const Tensor *qw = nullptr, *kw = nullptr;
  float eps = 0.f;
  if (w) {
    qw = c.get(w[0]);
    kw = c.get(w[1]);
    eps = PyFloat_Check(w[2]) ? (float)PyFloat_AS_DOUBLE(w[2]) : 0.f;
    auto vector = [&](const Tensor* t) {
      return t->dim() == 1 && t->numel() == hd && t->is_contiguous() && aligned(*t) &&
             (t->scalar_type() == at::kFloat || t->scalar_type() == q->scalar_type());
    };
    if (!c.need(qw && kw && vector(qw) && vector(kw) && qw->scalar_type() == kw->scalar_type() && eps >= FLT_MIN &&
                eps <= FLT_MAX))
      return none();
  }
  Tensor qo, ko;
  int rc;
  {
    NoGil others;
    qo = at::empty(q->sizes(), q->options());
    ko = at::empty(k->sizes(), k->options());
    const auto *turns = static_cast<const uint64_t*>(tab->data_ptr());
    const int32_t nq = (int32_t)q->size(1), nk = (int32_t)k->size(1), act = act_code(q->scalar_type());
    if (w)
      rc = ee_norm_rotary(q->data_ptr(), q->stride(0), q->stride(1), qo.data_ptr(), qo.stride(0), qo.stride(1),
                          k->data_ptr(), k->stride(0), k->stride(1), ko.data_ptr(), ko.stride(0), ko.stride(1),
                          qw->data_ptr(), kw->data_ptr(), qw->scalar_type() == at::kFloat ? EE_F32 : act, eps,
                          pos->data_ptr(), t, p64 ? 64 : 32, turns, t, nq, nk, (int32_t)hd, sections, (int32_t)axes,
                          interleaved, act, c.stream());
    else
      rc = ee_rotary(q->data_ptr(), q->stride(0), q->stride(1), qo.data_ptr(), qo.stride(0), qo.stride(1), k->data_ptr(),
                     k->stride(0), k->stride(1), ko.data_ptr(), ko.stride(0), ko.stride(1), pos->data_ptr(), t,
                     p64 ? 64 : 32, turns, t, nq, nk, (int32_t)hd, sections, (int32_t)axes, interleaved, act, c.stream());
  }
  return give(rc, qo, ko);
}
PyObject* rotary_embed(PyObject*, PyObject* const* a, Py_ssize_t argc) { return argc == 6 ? rotary(a, nullptr) : none(); }

// norm_rotary_embed(q, k, q_weight, k_weight, positions, sections, turns, interleaved, eps)
PyObject* norm_rotary_embed(PyObject*, PyObject* const* a, Py_ssize_t argc) {
  if (argc != 9) return none();
  PyObject* const heads[6] = {a[0], a[1], a[4], a[5], a[6], a[7]};
  PyObject* const norm[3] = {a[2], a[3], a[8]};
  return rotary(heads, norm);
}

// ---------------------------------------------------------------------------
// cache
// ---------------------------------------------------------------------------
// The cache's keys, the address of its ee_cache (made and checked by KVCache,
// whose tensors the record describes), offsets, table and lengths of a call.
struct Places {
  const ee_cache* cache;
  const int32_t *cu, *table, *k_lens;
  int64_t table_row, width, n;
};
bool places(Call& c, PyObject* keys, PyObject* record, PyObject* cu_o, PyObject* table_o, PyObject* lens_o, Places& p) {
  const Tensor *k = c.get(keys), *cu = c.get(cu_o), *table = c.get(table_o), *lens = c.get(lens_o);
  if (!c.need(k && cu && table && lens && PyLong_Check(record))) return false;
  p.cache = static_cast<const ee_cache*>(PyLong_AsVoidPtr(record));
  p.n = cu->numel() - 1;
  if (!c.need(p.cache && p.cache->k_codes == k->data_ptr() && cu->dim() == 1 && cu->scalar_type() == at::kInt && cu->is_contiguous() && p.n >= 1 &&
              p.n < (1 << 30) && lens->dim() == 1 && lens->scalar_type() == at::kInt && lens->numel() == p.n &&
              lens->is_contiguous() && table->dim() == 2 && table->scalar_type() == at::kInt && table->size(0) == p.n &&
              table->size(1) >= 1 && table->stride(1) == 1 && table->size(1) <= 0x7fff0000 / p.cache->page_size))
    return false;
  p.cu = static_cast<const int32_t*>(cu->data_ptr());
  p.table = static_cast<const int32_t*>(table->data_ptr());
  p.k_lens = static_cast<const int32_t*>(lens->data_ptr());
  p.table_row = table->stride(0);
  p.width = table->size(1);
  return true;
}
bool cache_heads(const Tensor& t, const ee_cache& c) {
  return heads_ok(t) && t.size(0) > 0 && t.size(0) < (1 << 30) && t.size(1) == c.kv_heads && t.size(2) == c.head_dim;
}

// cache_write(keys, record, k, v, cu, table, k_lens) -> True
PyObject* cache_write(PyObject*, PyObject* const* a, Py_ssize_t argc) {
  if (argc != 7) return none();
  Call c;
  Places p;
  if (!places(c, a[0], a[1], a[4], a[5], a[6], p)) return none();
  const Tensor *k = c.get(a[2]), *v = c.get(a[3]);
  if (!c.need(k && v && cache_heads(*k, *p.cache) && cache_heads(*v, *p.cache) && k->size(0) == v->size(0) &&
              k->scalar_type() == v->scalar_type()))
    return none();
  int rc;
  {
    NoGil others;
    rc = ee_cache_write(p.cache, k->data_ptr(), k->stride(0), k->stride(1), v->data_ptr(), v->stride(0), v->stride(1),
                        p.cu, p.table, p.table_row, (int32_t)p.width, p.k_lens, k->size(0), (int32_t)p.n,
                        act_code(k->scalar_type()), c.stream());
  }
  if (rc != EE_OK) return none();
  Py_RETURN_TRUE;
}

// cache_read(keys, record, cu, table, k_lens, tokens, dtype) -> (k, v)
PyObject* cache_read(PyObject*, PyObject* const* a, Py_ssize_t argc) {
  if (argc != 7 || !PyLong_Check(a[5]) || !THPDtype_Check(a[6])) return none();
  const ScalarType type = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
  const int64_t tokens = PyLong_AsLongLong(a[5]);
  if (tokens < 1 || tokens >= (1 << 30) || !act_type(type)) {
    PyErr_Clear();
    return none();
  }
  Call c;
  Places p;
  if (!places(c, a[0], a[1], a[2], a[3], a[4], p)) return none();
  const Tensor& keys = THPVariable_Unpack(a[0]);
  Tensor k, v;
  int rc;
  {
    NoGil others;
    k = at::empty({tokens, p.cache->kv_heads, p.cache->head_dim}, keys.options().dtype(type));
    v = at::empty({tokens, p.cache->kv_heads, p.cache->head_dim}, keys.options().dtype(type));
    rc = ee_cache_read(p.cache, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), p.cu,
                       p.table, p.table_row, (int32_t)p.width, p.k_lens, tokens, (int32_t)p.n, act_code(type), c.stream());
  }
  return give(rc, k, v);
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
// prompt_attention(q, k, v, cu_q, cu_k, k_lens, causal, scale)
PyObject* prompt_attention(PyObject*, PyObject* const* a, Py_ssize_t argc) {
  if (argc != 8) return none();
  Call c;
  const Tensor *q = c.get(a[0]), *k = c.get(a[1]), *v = c.get(a[2]), *cq = c.get(a[3]);
  const Tensor* ck = a[4] == Py_None ? nullptr : c.get(a[4]);
  const Tensor* kl = a[5] == Py_None ? nullptr : c.get(a[5]);
  if (!c.need(q && k && v && cq && heads_ok(*q) && heads_ok(*k) && heads_ok(*v) && PyBool_Check(a[6]))) return none();
  const int64_t tq = q->size(0), tk = k->size(0), hq = q->size(1), hk = k->size(1), hd = q->size(2), n = cq->numel() - 1;
  auto table = [](const Tensor* t, int64_t len) {
    return !t || (t->dim() == 1 && t->scalar_type() == at::kInt && t->numel() == len && t->is_contiguous());
  };
  float scale = 0.f;
  if (a[7] == Py_None) {
    scale = (float)(1.0 / std::sqrt((double)hd));
  } else if (PyFloat_Check(a[7])) {
    scale = (float)PyFloat_AS_DOUBLE(a[7]);
  }
  if (!c.need(k->sizes() == v->sizes() && k->scalar_type() == q->scalar_type() && v->scalar_type() == q->scalar_type() &&
              k->size(2) == hd && tq > 0 && n >= 1 && hk >= 1 && hq % hk == 0 && table(cq, n + 1) && table(ck, n + 1) &&
              table(kl, n) && (ck || tk == tq) && tq < (1 << 30) && tk < (1 << 30) && hq < 65536 && n < (1 << 30) &&
              scale > 0.f && scale < 2.0e38f && (hd == 64 || hd == 128)))
    return none();
  const bool causal = a[6] == Py_True;
  Tensor out;
  int rc;
  {
    NoGil others;
    out = at::empty(q->sizes(), q->options());
    const size_t need = ee_prompt_attention_workspace_bytes(tq, tk, (int32_t)n, (int32_t)hq, (int32_t)hk, (int32_t)hd);
    Tensor ws;
    if (need) ws = at::empty({(int64_t)need}, q->options().dtype(at::kByte));
    rc = ee_prompt_attention(q->data_ptr(), q->stride(0), q->stride(1), k->data_ptr(), k->stride(0), k->stride(1),
                             v->data_ptr(), v->stride(0), v->stride(1), out.data_ptr(), out.stride(0), out.stride(1),
                             static_cast<const int32_t*>(cq->data_ptr()),
                             ck ? static_cast<const int32_t*>(ck->data_ptr()) : nullptr,
                             kl ? static_cast<const int32_t*>(kl->data_ptr()) : nullptr, tq, tk, (int32_t)n,
                             (int32_t)hq, (int32_t)hk, (int32_t)hd, causal, scale, act_code(q->scalar_type()),
                             need ? ws.data_ptr() : nullptr, need, c.stream());
  }
  return give(rc, out);
}

// cache_attention(keys, record, q, cu_q, table, k_lens, causal, scale, prefix)
PyObject* cache_attention(PyObject*, PyObject* const* a, Py_ssize_t argc) {
  if (argc != 9 || !PyBool_Check(a[6])) return none();
  Call c;
  Places p;
  if (!places(c, a[0], a[1], a[3], a[4], a[5], p)) return none();
  const Tensor *q = c.get(a[2]), *pk = nullptr, *pv = nullptr;
  const int64_t hk = p.cache->kv_heads, hd = p.cache->head_dim;
  if (!c.need(q && heads_ok(*q) && q->size(0) > 0 && q->size(2) == hd && q->size(1) >= 1 && q->size(1) < 65536 &&
              q->size(1) % hk == 0 && q->size(0) <= 0x7fffff00 / q->size(1)))
    return none();
  const int64_t tq = q->size(0), hq = q->size(1);
  if (a[8] != Py_None) {
    if (!c.need(PyTuple_Check(a[8]) && PyTuple_GET_SIZE(a[8]) == 2)) return none();
    pk = c.get(PyTuple_GET_ITEM(a[8], 0));
    pv = c.get(PyTuple_GET_ITEM(a[8], 1));
    if (!c.need(pk && pv && heads_ok(*pk) && heads_ok(*pv) && pk->sizes() == pv->sizes() && pk->size(0) > 0 &&
                pk->size(0) < (1 << 30) && pk->size(1) == hk && pk->size(2) == hd &&
                pk->scalar_type() == q->scalar_type() && pv->scalar_type() == q->scalar_type() && hq / hk <= 128))
      return none();
  }
  float scale = 0.f;
  if (a[7] == Py_None) {
    scale = (float)(1.0 / std::sqrt((double)hd));
  } else if (PyFloat_Check(a[7])) {
    scale = (float)PyFloat_AS_DOUBLE(a[7]);
  }
  if (!c.need(scale >= FLT_MIN && scale < 2.0e38f)) return none();
  const bool causal = a[6] == Py_True;
  const int64_t plen = pk ? pk->size(0) : 0;
  Tensor out;
  int rc;
  {
    NoGil others;
    out = at::empty(q->sizes(), q->options());
    const size_t need = ee_cache_attention_workspace_bytes(tq, (int32_t)p.n, (int32_t)hq, (int32_t)hk, (int32_t)hd,
                                                           p.cache->bits, p.width * p.cache->page_size, plen);
    Tensor ws;
    if (need) ws = at::empty({(int64_t)need}, q->options().dtype(at::kByte));
    rc = ee_cache_attention(p.cache, q->data_ptr(), q->stride(0), q->stride(1), out.data_ptr(), out.stride(0),
                            out.stride(1), p.cu, p.table, p.table_row, (int32_t)p.width, p.k_lens,
                            pk ? pk->data_ptr() : nullptr, pk ? pk->stride(0) : 0, pk ? pk->stride(1) : 0,
                            pv ? pv->data_ptr() : nullptr, pv ? pv->stride(0) : 0, pv ? pv->stride(1) : 0, plen, tq,
                            (int32_t)p.n, (int32_t)hq, causal, scale, act_code(q->scalar_type()),
                            need ? ws.data_ptr() : nullptr, need, c.stream());
  }
  return give(rc, out);
}

// C++ exceptions (out of memory in an allocation) become Python's: the Python
// function then meets the same condition and raises torch's own error.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  try {
    return F(self, a, n);
  } catch (...) {
    return none();
  }
}

#define EE_METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<name>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {EE_METHOD(int8_linear),  EE_METHOD(int8_matmul),      EE_METHOD(quantize_tokens),
                         EE_METHOD(rotary_embed), EE_METHOD(norm_rotary_embed), EE_METHOD(prompt_attention),
                         EE_METHOD(cache_write),  EE_METHOD(cache_read),        EE_METHOD(cache_attention),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ee_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_ee_torch() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", EE_TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
