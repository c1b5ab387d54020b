// li4_torch.cpp -- the paged-cache entry points on torch tensors (module li4_torch, used by llama/paged.py).
//
// A decode step calls these once or twice per layer with kernels of a few microseconds behind them, so what
// a call costs on the host decides how fast an eager step is.  Checks, output and workspace allocation and
// the launch happen here in one C call each (rope_paged_write: 42 us per eager call with the same checks in
// Python, against a 1.7 us kernel).  Argument errors raise RuntimeError; a li4_status other than LI4_OK is
// returned as an int for the caller to turn into its error.  Every C++ exception ends at the entry.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "llama_int4_b200.h"

namespace {

using at::Tensor;

struct Refused {
  std::string message;
};

template <typename... Args>
[[noreturn]] void fail(const char* what, const Args&... args) {
  throw Refused{c10::str(what, ": ", args...)};
}

Tensor tensor(const char* what, const char* name, PyObject* o) {
  if (!THPVariable_Check(o)) fail(what, name, " must be a tensor");
  const Tensor& t = THPVariable_Unpack(o);
  // These are no registered operators: a tracer would record nothing of the call, or meet a tensor without data.
  if (t.key_set().has(c10::DispatchKey::Python) || !t.has_storage() ||
      c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer))
    fail(what, name, " must be a plain tensor, outside of any tracing");
  if (c10::GradMode::is_enabled() && t.requires_grad())
    fail(what, name, " requires grad and there is no backward pass: call under torch.no_grad()");
  return t;
}

// The call's device: the first tensor's; every other tensor must be on it.
struct Device {
  const char* what;
  const char* first = nullptr;
  c10::Device dev{c10::kCPU};
  void add(const char* name, const Tensor& t) {
    if (!t.is_cuda()) fail(what, name, " is on ", t.device().str(), " (CUDA tensors only)");
    if (!first) {
      first = name;
      dev = t.device();
    } else if (t.device() != dev) {
      fail(what, name, " is on ", t.device().str(), ", ", first, " is on ", dev.str());
    }
  }
};

void ints(const char* what, const char* name, const Tensor& t, at::ScalarType type, at::IntArrayRef shape) {
  if (t.scalar_type() != type || t.sizes() != shape)
    fail(what, name, " must be ", type, " ", shape, ", got ", t.scalar_type(), " ", t.sizes());
}

int type_code(at::ScalarType t) { return t == at::kHalf ? LI4_F16 : t == at::kBFloat16 ? LI4_BF16 : -1; }

// The kernels' layout: contiguous last dimension, rows on 16-byte boundaries, no repeated rows.
bool rows_ok(const Tensor& t) {
  if (t.numel() == 0) return true;
  const int64_t d = t.dim();
  if (t.size(d - 1) != 1 && t.stride(d - 1) != 1) return false;
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) return false;
  for (int64_t i = 0; i + 1 < d; ++i)
    if (t.size(i) != 1 && (t.stride(i) <= 0 || t.stride(i) % 8 != 0)) return false;
  return true;
}

Tensor readable(const Tensor& t) { return rows_ok(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

int64_t row_stride(const Tensor& t, int64_t i) { return t.size(i) > 1 ? t.stride(i) : 0; }

void packed(const char* what, const char* name, const Tensor& t) {
  if (t.dim() != 3) fail(what, name, " must be [tokens, heads, head_dim], got ", t.sizes());
  if (type_code(t.scalar_type()) < 0) fail(what, name, " must be float16 or bfloat16, got ", t.scalar_type());
}
void same_type(const char* what, const char* name, const Tensor& t, const Tensor& q) {
  if (t.scalar_type() != q.scalar_type()) fail(what, name, " is ", t.scalar_type(), ", q is ", q.scalar_type());
}

Tensor empty(at::IntArrayRef shape, at::ScalarType type, c10::Device dev) {
  return at::detail::empty_cuda(shape, type, dev, std::nullopt);
}

Tensor output(const char* what, const char* name, PyObject* o, const Tensor& like, Device& d) {
  if (o == Py_None) return empty(like.sizes(), like.scalar_type(), d.dev);
  Tensor t = tensor(what, name, o);
  d.add(name, t);
  if (t.sizes() != like.sizes() || t.scalar_type() != like.scalar_type() || !rows_ok(t))
    fail(what, name, " must be ", like.scalar_type(), " ", like.sizes(), " with contiguous rows on 16-byte boundaries");
  return t;
}

// Whether two tensors of 16-bit values share no memory, as far as their strides show it: their ranges lie apart, or they
// are parts of one wider row (queries, keys and values of one projection): modulo some stride of theirs, what the
// dimensions of other strides span lies apart.
bool apart(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return true;
  auto span = [](const Tensor& t, int64_t modulo) {  // elements, the dimensions of strides that are multiples left out
    int64_t n = 1;
    for (int64_t i = 0; i < t.dim(); ++i)
      if (modulo == 0 || t.stride(i) % modulo != 0) n += (t.size(i) - 1) * t.stride(i);
    return n;
  };
  const int64_t pa = (int64_t)(reinterpret_cast<uintptr_t>(a.data_ptr()) / 2),
                pb = (int64_t)(reinterpret_cast<uintptr_t>(b.data_ptr()) / 2);
  if (pa + span(a, 0) <= pb || pb + span(b, 0) <= pa) return true;
  for (const Tensor* t : {&a, &b})
    for (int64_t i = 0; i < t->dim(); ++i) {
      const int64_t m = t->stride(i);
      if (t->size(i) < 2 || m < 1) continue;
      const int64_t ahead = ((pb - pa) % m + m) % m;
      if (ahead >= span(a, m) && m - ahead >= span(b, m)) return true;
    }
  return false;
}

bool same_rows(const Tensor& a, const Tensor& b) {
  if (a.data_ptr() != b.data_ptr()) return false;
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) != b.size(i) || (a.size(i) > 1 && a.stride(i) != b.stride(i))) return false;
  return true;
}

void not_over(const char* what, const char* out_name, const Tensor& out, const char* name, const Tensor& in) {
  if (!apart(out, in)) fail(what, out_name, " must not overlap ", name);
}

void cache_ok(const char* what, const char* name, const Tensor& t, const Tensor& q, int64_t kv_heads) {
  if (t.dim() != 4 || t.size(2) != kv_heads || t.size(3) != q.size(2) || t.scalar_type() != q.scalar_type())
    fail(what, name, " must be ", q.scalar_type(), " [pages, page_size, ", kv_heads, ", ", q.size(2), "], got ",
         t.scalar_type(), " ", t.sizes());
  if (!rows_ok(t)) fail(what, name, ": rows of head_dim values must be contiguous, on 16-byte boundaries");
}

int64_t integer(const char* what, const char* name, PyObject* o) {
  const long long v = PyLong_Check(o) ? PyLong_AsLongLong(o) : -1;
  if (!PyLong_Check(o) || PyErr_Occurred()) {
    PyErr_Clear();
    fail(what, name, " must be an int");
  }
  return v;
}

PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }

struct NoGil {  // the launch may wait for room in the stream's queue
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

// One attention call's common part.
PyObject* attend(const char* what, bool paged, li4_attention& a, const Tensor& q, const Tensor& cu, PyObject* scale,
                 const Tensor& out, int64_t max_queries, c10::Device dev) {
  const Tensor qr = readable(q), c = cu.contiguous();
  a.q = qr.data_ptr();
  a.out = out.data_ptr();
  a.dtype = type_code(q.scalar_type());
  a.scale = (float)(1.0 / std::sqrt((double)q.size(2)));
  if (scale != Py_None) {
    a.scale = (float)PyFloat_AsDouble(scale);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      fail(what, "scale must be a number");
    }
  }
  a.n_tokens = q.size(0);
  a.n_heads = q.size(1);
  a.head_dim = q.size(2);
  a.stride_qt = row_stride(qr, 0);
  a.stride_qh = row_stride(qr, 1);
  a.stride_ot = row_stride(out, 0);
  a.stride_oh = row_stride(out, 1);
  a.cu_seqlens = c.const_data_ptr<int32_t>();
  a.n_seqs = cu.size(0) - 1;
  a.max_queries = max_queries;
  // The workspace comes from the stream's allocator for this call alone: calls on several streams and
  // captured graphs (each with its own pool) never share one.
  const size_t need = li4_attention_workspace_bytes(&a);
  Tensor ws;
  if (need) ws = empty({(int64_t)need}, at::kByte, dev);
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  int rc;
  {
    NoGil nogil;
    rc = paged ? li4_paged_attention(&a, need ? ws.data_ptr() : nullptr, need, stream)
               : li4_prompt_attention(&a, need ? ws.data_ptr() : nullptr, need, stream);
  }
  return rc == LI4_OK ? wrap(out) : PyLong_FromLong(rc);
}

void queries_ok(const char* what, const Tensor& q, const Tensor& cu, int64_t kv_heads, int64_t max_queries) {
  packed(what, "q", q);
  if (cu.dim() != 1 || cu.size(0) < 1 || cu.scalar_type() != at::kInt)
    fail(what, "cu_seqlens must be int32 [sequences + 1], got ", cu.scalar_type(), " ", cu.sizes());
  if (kv_heads < 1 || q.size(1) < 1 || q.size(1) % kv_heads) fail(what, q.size(1), " query heads over ", kv_heads, " KV heads");
  if (max_queries < 0) fail(what, "a longest sequence of ", max_queries, " queries");
}

// (q, k, v, cu_seqlens, max_len, scale, out)
PyObject* prompt_attention(PyObject* const* v) {
  const char* what = "prompt_attention";
  const Tensor q = tensor(what, "q", v[0]), k = tensor(what, "k", v[1]), val = tensor(what, "v", v[2]),
               cu = tensor(what, "cu_seqlens", v[3]);
  Device d{what};
  d.add("q", q);
  d.add("k", k);
  d.add("v", val);
  d.add("cu_seqlens", cu);
  packed(what, "k", k);
  const int64_t max_len = integer(what, "max_len", v[4]);
  queries_ok(what, q, cu, k.size(1), max_len);
  same_type(what, "k", k, q);
  same_type(what, "v", val, q);
  if (k.size(0) != q.size(0) || k.size(2) != q.size(2) || val.sizes() != k.sizes())
    fail(what, "q ", q.sizes(), ", k ", k.sizes(), " and v ", val.sizes(), " do not match");
  const c10::cuda::CUDAGuard guard(d.dev);
  const Tensor out = output(what, "out", v[6], q, d);
  if (v[6] != Py_None) {  // (rows are read again after others are written)
    not_over(what, "out", out, "q", q);
    not_over(what, "out", out, "k", k);
    not_over(what, "out", out, "v", val);
  }
  const Tensor kr = readable(k), vr = readable(val);
  li4_attention a = {};
  a.k = kr.data_ptr();
  a.v = vr.data_ptr();
  a.n_kv_heads = k.size(1);
  a.stride_kt = row_stride(kr, 0);
  a.stride_kh = row_stride(kr, 1);
  a.stride_vt = row_stride(vr, 0);
  a.stride_vh = row_stride(vr, 1);
  return attend(what, false, a, q, cu, v[5], out, max_len, d.dev);
}

// (q, cache_k, cache_v, block_tables, kv_lens, cu_seqlens, max_new, scale, out)
PyObject* paged_attention(PyObject* const* v) {
  const char* what = "paged_attention";
  const Tensor q = tensor(what, "q", v[0]), ck = tensor(what, "cache_k", v[1]), cv = tensor(what, "cache_v", v[2]),
               bt = tensor(what, "block_tables", v[3]), lens = tensor(what, "kv_lens", v[4]),
               cu = tensor(what, "cu_seqlens", v[5]);
  Device d{what};
  d.add("q", q);
  d.add("cache_k", ck);
  d.add("cache_v", cv);
  d.add("block_tables", bt);
  d.add("kv_lens", lens);
  d.add("cu_seqlens", cu);
  if (ck.dim() != 4) fail(what, "cache_k must be [pages, page_size, kv_heads, head_dim], got ", ck.sizes());
  const int64_t max_new = integer(what, "max_new", v[6]);
  queries_ok(what, q, cu, ck.size(2), max_new);
  cache_ok(what, "cache_k", ck, q, ck.size(2));
  cache_ok(what, "cache_v", cv, q, ck.size(2));
  if (cv.sizes() != ck.sizes()) fail(what, "cache_k ", ck.sizes(), " and cache_v ", cv.sizes(), " differ");
  const int64_t B = cu.size(0) - 1;
  if (bt.dim() != 2) fail(what, "block_tables must be [requests, blocks], got ", bt.sizes());
  const int64_t width = bt.size(1);
  ints(what, "block_tables", bt, at::kInt, {B, width});
  ints(what, "kv_lens", lens, at::kInt, {B});
  const c10::cuda::CUDAGuard guard(d.dev);
  const Tensor out = output(what, "out", v[8], q, d);
  if (v[8] != Py_None) {
    not_over(what, "out", out, "q", q);
    not_over(what, "out", out, "cache_k", ck);
    not_over(what, "out", out, "cache_v", cv);
  }
  const bool table_ok = (width <= 1 || bt.stride(1) == 1) && (B <= 1 || bt.stride(0) >= width);
  const Tensor tables = table_ok ? bt : bt.contiguous(), l = lens.contiguous();
  li4_attention a = {};
  a.k = ck.data_ptr();
  a.v = cv.data_ptr();
  a.n_kv_heads = ck.size(2);
  a.stride_kp = row_stride(ck, 0);
  a.stride_kt = row_stride(ck, 1);
  a.stride_kh = row_stride(ck, 2);
  a.stride_vp = row_stride(cv, 0);
  a.stride_vt = row_stride(cv, 1);
  a.stride_vh = row_stride(cv, 2);
  a.kv_lens = l.const_data_ptr<int32_t>();
  a.block_tables = tables.const_data_ptr<int32_t>();
  a.table_stride = B > 1 ? tables.stride(0) : width;
  a.table_width = width;
  a.num_pages = ck.size(0);
  a.page_size = ck.size(1);
  return attend(what, true, a, q, cu, v[7], out, max_new, d.dev);
}

// (q, k, v, cos, sin, positions, slots, cache_k, cache_v, q_out, k_out, need_k)
PyObject* rope_paged_write(PyObject* const* v) {
  const char* what = "rope_paged_write";
  const Tensor q = tensor(what, "q", v[0]), k = tensor(what, "k", v[1]), val = tensor(what, "v", v[2]),
               positions = tensor(what, "positions", v[5]), slots = tensor(what, "slots", v[6]),
               ck = tensor(what, "cache_k", v[7]), cv = tensor(what, "cache_v", v[8]);
  Tensor cos = tensor(what, "cos", v[3]), sin = tensor(what, "sin", v[4]);
  Device d{what};
  d.add("q", q);
  d.add("k", k);
  d.add("v", val);
  d.add("cos", cos);
  d.add("sin", sin);
  d.add("positions", positions);
  d.add("slots", slots);
  d.add("cache_k", ck);
  d.add("cache_v", cv);
  packed(what, "q", q);
  packed(what, "k", k);
  same_type(what, "k", k, q);
  same_type(what, "v", val, q);
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2), Hkv = k.size(1);
  if (k.size(0) != T || k.size(2) != D || val.sizes() != k.sizes())
    fail(what, "q ", q.sizes(), ", k ", k.sizes(), " and v ", val.sizes(), " do not match");
  cache_ok(what, "cache_k", ck, q, Hkv);
  cache_ok(what, "cache_v", cv, q, Hkv);
  if (cv.sizes() != ck.sizes()) fail(what, "cache_k ", ck.sizes(), " and cache_v ", cv.sizes(), " differ");
  if (cos.dim() != 2 || cos.sizes() != sin.sizes() || cos.size(1) != D / 2 || cos.scalar_type() != at::kFloat ||
      sin.scalar_type() != at::kFloat)
    fail(what, "cos / sin must be float32 [positions, ", D / 2, "], got ", cos.scalar_type(), " ", cos.sizes(), " / ",
         sin.scalar_type(), " ", sin.sizes());
  ints(what, "positions", positions, at::kInt, {T});
  ints(what, "slots", slots, at::kLong, {T});
  const c10::cuda::CUDAGuard guard(d.dev);
  const bool want_k = v[10] != Py_None || PyObject_IsTrue(v[11]) == 1;
  const Tensor q_out = output(what, "q_out", v[9], q, d);
  Tensor k_out;
  if (want_k) k_out = output(what, "k_out", v[10], k, d);
  // an output may be its own input; nothing else may be written before it is read
  auto check = [&](const char* name, const Tensor& out, const char* own_name, const Tensor& own, const char* other_name,
                   const Tensor& other) {
    if (!same_rows(out, own)) not_over(what, name, out, own_name, own);
    not_over(what, name, out, other_name, other);
    not_over(what, name, out, "v", val);
    not_over(what, name, out, "cache_k", ck);
    not_over(what, name, out, "cache_v", cv);
  };
  if (v[9] != Py_None) check("q_out", q_out, "q", q, "k", k);
  if (v[10] != Py_None) check("k_out", k_out, "k", k, "q", q);
  if (v[9] != Py_None && v[10] != Py_None) not_over(what, "q_out", q_out, "k_out", k_out);
  auto table = [](const Tensor& t) {
    return t.is_contiguous() && !(reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) ? t : t.clone(at::MemoryFormat::Contiguous);
  };
  cos = table(cos);
  sin = table(sin);
  const Tensor qr = readable(q), kr = readable(k), vr = readable(val), p = positions.contiguous(), s = slots.contiguous();
  const int64_t st[16] = {row_stride(qr, 0), row_stride(qr, 1), row_stride(kr, 0), row_stride(kr, 1), row_stride(vr, 0), row_stride(vr, 1),
                          row_stride(q_out, 0), row_stride(q_out, 1), want_k ? row_stride(k_out, 0) : 0,
                          want_k ? row_stride(k_out, 1) : 0, row_stride(ck, 0), row_stride(ck, 1), row_stride(ck, 2), row_stride(cv, 0),
                          row_stride(cv, 1), row_stride(cv, 2)};
  void* stream = c10::cuda::getCurrentCUDAStream(d.dev.index()).stream();
  int rc;
  {
    NoGil nogil;
    rc = li4_rope_paged_write(qr.data_ptr(), kr.data_ptr(), vr.data_ptr(), type_code(q.scalar_type()), T, H, Hkv, D, st,
                              cos.const_data_ptr<float>(), sin.const_data_ptr<float>(), D / 2, cos.size(0),
                              p.const_data_ptr<int32_t>(), s.const_data_ptr<int64_t>(), q_out.data_ptr(),
                              want_k ? k_out.data_ptr() : nullptr, ck.data_ptr(), cv.data_ptr(), ck.size(0), ck.size(1),
                              stream);
  }
  if (rc != LI4_OK) return PyLong_FromLong(rc);
  PyObject* r = PyTuple_New(2);
  PyTuple_SET_ITEM(r, 0, wrap(q_out));
  if (!want_k) Py_INCREF(Py_None);
  PyTuple_SET_ITEM(r, 1, want_k ? wrap(k_out) : Py_None);
  return r;
}

// (kv_lens, new_lens, block_tables, free_pages, n_free, page_size, num_tokens, kv_lens_out, n_free_out, max_len)
PyObject* paged_append(PyObject* const* v) {
  const char* what = "paged_append";
  const Tensor kv = tensor(what, "kv_lens", v[0]), nl = tensor(what, "new_lens", v[1]),
               bt = tensor(what, "block_tables", v[2]), fp = tensor(what, "free_pages", v[3]),
               nf = tensor(what, "n_free", v[4]);
  Device d{what};
  d.add("kv_lens", kv);
  d.add("new_lens", nl);
  d.add("block_tables", bt);
  d.add("free_pages", fp);
  d.add("n_free", nf);
  if (kv.dim() != 1 || bt.dim() != 2 || fp.dim() != 1)
    fail(what, "kv_lens [requests], block_tables [requests, blocks] and free_pages [pages] expected");
  const int64_t B = kv.size(0), width = bt.size(1);
  ints(what, "kv_lens", kv, at::kInt, {B});
  ints(what, "new_lens", nl, at::kInt, {B});
  ints(what, "block_tables", bt, at::kInt, {B, width});
  ints(what, "free_pages", fp, at::kInt, {fp.size(0)});
  ints(what, "n_free", nf, at::kInt, {1});
  if ((width > 1 && bt.stride(1) != 1) || (B > 1 && bt.stride(0) < width)) fail(what, "block_tables rows must be contiguous");
  const int64_t page = integer(what, "page_size", v[5]), T = integer(what, "num_tokens", v[6]);
  if (T < 0 || T > (1 << 30)) fail(what, "num_tokens ", T);
  const int64_t max_len = v[9] == Py_None ? INT64_MAX : integer(what, "max_len", v[9]);
  const c10::cuda::CUDAGuard guard(d.dev);
  const Tensor kc = kv.contiguous(), nc = nl.contiguous(), fc = fp.contiguous();
  auto result = [&](const char* name, PyObject* o, const Tensor& like) {
    if (o == Py_None) return empty(like.sizes(), at::kInt, d.dev);
    Tensor t = tensor(what, name, o);
    d.add(name, t);
    if (t.scalar_type() != at::kInt || t.sizes() != like.sizes() || !t.is_contiguous())
      fail(what, name, " must be contiguous int32 ", like.sizes());
    return t;
  };
  const Tensor kv_out = result("kv_lens_out", v[7], kv), nf_out = result("n_free_out", v[8], nf);
  const Tensor cu = empty({B + 1}, at::kInt, d.dev), pos = empty({T}, at::kInt, d.dev),
               slots = empty({T}, at::kLong, d.dev), granted = empty({B}, at::kBool, d.dev);
  void* stream = c10::cuda::getCurrentCUDAStream(d.dev.index()).stream();
  int rc;
  {
    NoGil nogil;
    rc = li4_paged_append_within(kc.const_data_ptr<int32_t>(), nc.const_data_ptr<int32_t>(), B, bt.data_ptr<int32_t>(),
                          B > 1 ? bt.stride(0) : width, width, fc.const_data_ptr<int32_t>(), fc.size(0),
                          nf.const_data_ptr<int32_t>(), page, T, max_len, cu.data_ptr<int32_t>(), pos.data_ptr<int32_t>(),
                          slots.data_ptr<int64_t>(), kv_out.data_ptr<int32_t>(), nf_out.data_ptr<int32_t>(),
                          reinterpret_cast<uint8_t*>(granted.data_ptr()), stream);
  }
  if (rc != LI4_OK) return PyLong_FromLong(rc);
  const Tensor* all[6] = {&cu, &pos, &slots, &kv_out, &nf_out, &granted};
  PyObject* r = PyTuple_New(6);
  for (int i = 0; i < 6; ++i) PyTuple_SET_ITEM(r, i, wrap(*all[i]));
  return r;
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    if (n != N) throw Refused{c10::str("expected ", N, " arguments, got ", n)};
    return F(args);
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_RuntimeError, e.message.c_str());
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* kind = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    PyErr_Clear();
    PyErr_SetString(kind ? kind : PyExc_RuntimeError, e.what_without_backtrace());
    Py_XDECREF(kind);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "li4_torch: unknown C++ exception");
  }
  return nullptr;
}

template <PyObject* (*F)(PyObject* const*), int N>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<prompt_attention, 7>("prompt_attention"), method<paged_attention, 9>("paged_attention"),
                         method<rope_paged_write, 12>("rope_paged_write"), method<paged_append, 10>("paged_append"),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "li4_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_li4_torch(void) { return PyModule_Create(&module); }
