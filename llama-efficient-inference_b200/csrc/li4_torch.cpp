// li4_torch.cpp -- the paged-cache entry points and token_logprobs on torch tensors (module li4_torch, used by
// llama/paged.py and llama/logprobs.py).
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
#include <vector>

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

// Tensors of any types whose memory ranges may not meet.
void bytes_apart(const char* what, const char* out_name, const Tensor& out, const char* name, const Tensor& in) {
  if (out.numel() == 0 || in.numel() == 0) return;
  auto end = [](const Tensor& t) {
    int64_t n = 1;
    for (int64_t i = 0; i < t.dim(); ++i) n += (t.size(i) - 1) * t.stride(i);
    return static_cast<const char*>(t.data_ptr()) + n * t.element_size();
  };
  const char *a = static_cast<const char*>(out.data_ptr()), *b = static_cast<const char*>(in.data_ptr());
  if (a < end(in) && b < end(out)) fail(what, out_name, " must not overlap ", name);
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
                 const Tensor& out, int64_t max_queries, c10::Device dev, const li4_int4_pages* k4 = nullptr,
                 const li4_int4_pages* v4 = nullptr) {
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
  const size_t need = k4 ? li4_attention_int4_workspace_bytes(&a) : li4_attention_workspace_bytes(&a);
  Tensor ws;
  if (need) ws = empty({(int64_t)need}, at::kByte, dev);
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  int rc;
  {
    NoGil nogil;
    rc = k4 ? li4_paged_attention_int4(&a, k4, v4, need ? ws.data_ptr() : nullptr, need, stream)
         : paged ? li4_paged_attention(&a, need ? ws.data_ptr() : nullptr, need, stream)
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

void rope_tables_ok(const char* what, const Tensor& cos, const Tensor& sin, int64_t D) {
  if (cos.dim() != 2 || cos.sizes() != sin.sizes() || cos.size(1) != D / 2 || cos.scalar_type() != at::kFloat ||
      sin.scalar_type() != at::kFloat)
    fail(what, "cos / sin must be float32 [positions, ", D / 2, "], got ", cos.scalar_type(), " ", cos.sizes(), " / ",
         sin.scalar_type(), " ", sin.sizes());
}
Tensor aligned_table(const Tensor& t) {
  return t.is_contiguous() && !(reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) ? t : t.clone(at::MemoryFormat::Contiguous);
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
  rope_tables_ok(what, cos, sin, D);
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
  cos = aligned_table(cos);
  sin = aligned_table(sin);
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

// A pair (codes, params) of a cache in 4 bits.
struct Pages4 {
  Tensor codes, params;
  li4_int4_pages raw;
};
Pages4 pages4(const char* what, const char* name, PyObject* o, const Tensor& q, int64_t kv_heads, Device& d) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2) fail(what, name, " must be a pair (codes, params)");
  const std::string codes = std::string(name) + ".codes", params = std::string(name) + ".params";
  Pages4 p{tensor(what, codes.c_str(), PyTuple_GET_ITEM(o, 0)), tensor(what, params.c_str(), PyTuple_GET_ITEM(o, 1)), {}};
  d.add(codes.c_str(), p.codes);
  d.add(params.c_str(), p.params);
  const int64_t D = q.size(2), G = D / LI4_KV_GROUP;
  if (D % LI4_KV_GROUP != 0) fail(what, "head_dim ", D, ": a multiple of ", LI4_KV_GROUP, " up to 128");
  const Tensor &c = p.codes, &s = p.params;
  if (c.dim() != 4 || c.size(2) != kv_heads || c.size(3) != D / 2 || c.scalar_type() != at::kByte)
    fail(what, codes, " must be uint8 [pages, page_size, ", kv_heads, ", ", D / 2, "], got ", c.scalar_type(), " ", c.sizes());
  if (s.dim() != 5 || s.size(0) != c.size(0) || s.size(1) != c.size(1) || s.size(2) != kv_heads || s.size(3) != G ||
      s.size(4) != 2 || s.scalar_type() != q.scalar_type())
    fail(what, params, " must be ", q.scalar_type(), " [", c.size(0), ", ", c.size(1), ", ", kv_heads, ", ", G, ", 2], got ",
         s.scalar_type(), " ", s.sizes());
  if (c.numel() > 0) {
    bool ok = c.stride(3) == 1 && s.stride(4) == 1 && (G == 1 || s.stride(3) == 2) &&
              !(reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) && !(reinterpret_cast<uintptr_t>(s.data_ptr()) & 3u);
    for (int64_t i = 0; i < 3; ++i) {
      ok = ok && (c.size(i) == 1 || (c.stride(i) > 0 && c.stride(i) % 16 == 0));
      ok = ok && (s.size(i) == 1 || (s.stride(i) > 0 && s.stride(i) % 2 == 0));
    }
    if (!ok) fail(what, name, ": rows of codes must be contiguous on 16-byte boundaries, rows of params on 4-byte ones");
  }
  p.raw = {c.data_ptr(), s.data_ptr(), row_stride(c, 0), row_stride(c, 1), row_stride(c, 2),
           row_stride(s, 0) / 2, row_stride(s, 1) / 2, row_stride(s, 2) / 2};
  return p;
}

// (q, cache_k, cache_v, block_tables, kv_lens, cu_seqlens, max_new, scale, out)
PyObject* paged_attention_int4(PyObject* const* v) {
  const char* what = "paged_attention_int4";
  const Tensor q = tensor(what, "q", v[0]), bt = tensor(what, "block_tables", v[3]), lens = tensor(what, "kv_lens", v[4]),
               cu = tensor(what, "cu_seqlens", v[5]);
  Device d{what};
  d.add("q", q);
  packed(what, "q", q);
  if (!PyTuple_Check(v[1]) || PyTuple_GET_SIZE(v[1]) != 2 || !THPVariable_Check(PyTuple_GET_ITEM(v[1], 0)) ||
      THPVariable_Unpack(PyTuple_GET_ITEM(v[1], 0)).dim() != 4)
    fail(what, "cache_k must be a pair (codes [pages, page_size, kv_heads, head_dim / 2], params)");
  const int64_t kv_heads = THPVariable_Unpack(PyTuple_GET_ITEM(v[1], 0)).size(2);
  const Pages4 ck = pages4(what, "cache_k", v[1], q, kv_heads, d), cv = pages4(what, "cache_v", v[2], q, kv_heads, d);
  d.add("block_tables", bt);
  d.add("kv_lens", lens);
  d.add("cu_seqlens", cu);
  const int64_t max_new = integer(what, "max_new", v[6]);
  queries_ok(what, q, cu, kv_heads, max_new);
  if (cv.codes.sizes() != ck.codes.sizes()) fail(what, "cache_k ", ck.codes.sizes(), " and cache_v ", cv.codes.sizes(), " differ");
  const int64_t B = cu.size(0) - 1;
  if (bt.dim() != 2) fail(what, "block_tables must be [requests, blocks], got ", bt.sizes());
  const int64_t width = bt.size(1);
  ints(what, "block_tables", bt, at::kInt, {B, width});
  ints(what, "kv_lens", lens, at::kInt, {B});
  const c10::cuda::CUDAGuard guard(d.dev);
  const Tensor out = output(what, "out", v[8], q, d);
  if (v[8] != Py_None) {
    not_over(what, "out", out, "q", q);
    // (byte ranges: the cache's elements are of other sizes)
    for (const Tensor* t : {&ck.codes, &ck.params, &cv.codes, &cv.params}) bytes_apart(what, "out", out, "the cache", *t);
  }
  const bool table_ok = (width <= 1 || bt.stride(1) == 1) && (B <= 1 || bt.stride(0) >= width);
  const Tensor tables = table_ok ? bt : bt.contiguous(), l = lens.contiguous();
  li4_attention a = {};
  a.n_kv_heads = kv_heads;
  a.kv_lens = l.const_data_ptr<int32_t>();
  a.block_tables = tables.const_data_ptr<int32_t>();
  a.table_stride = B > 1 ? tables.stride(0) : width;
  a.table_width = width;
  a.num_pages = ck.codes.size(0);
  a.page_size = ck.codes.size(1);
  return attend(what, true, a, q, cu, v[7], out, max_new, d.dev, &ck.raw, &cv.raw);
}

// (q, k, v, cos, sin, positions, slots, cache_k, cache_v, q_out, k_out, v_out, need_kv)
PyObject* rope_paged_write_int4(PyObject* const* v) {
  const char* what = "rope_paged_write_int4";
  const Tensor q = tensor(what, "q", v[0]), k = tensor(what, "k", v[1]), val = tensor(what, "v", v[2]),
               positions = tensor(what, "positions", v[5]), slots = tensor(what, "slots", v[6]);
  Tensor cos = tensor(what, "cos", v[3]), sin = tensor(what, "sin", v[4]);
  Device d{what};
  d.add("q", q);
  d.add("k", k);
  d.add("v", val);
  d.add("cos", cos);
  d.add("sin", sin);
  d.add("positions", positions);
  d.add("slots", slots);
  packed(what, "q", q);
  packed(what, "k", k);
  same_type(what, "k", k, q);
  same_type(what, "v", val, q);
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2), Hkv = k.size(1);
  if (k.size(0) != T || k.size(2) != D || val.sizes() != k.sizes())
    fail(what, "q ", q.sizes(), ", k ", k.sizes(), " and v ", val.sizes(), " do not match");
  const Pages4 ck = pages4(what, "cache_k", v[7], q, Hkv, d), cv = pages4(what, "cache_v", v[8], q, Hkv, d);
  if (cv.codes.sizes() != ck.codes.sizes()) fail(what, "cache_k ", ck.codes.sizes(), " and cache_v ", cv.codes.sizes(), " differ");
  rope_tables_ok(what, cos, sin, D);
  ints(what, "positions", positions, at::kInt, {T});
  ints(what, "slots", slots, at::kLong, {T});
  const c10::cuda::CUDAGuard guard(d.dev);
  const int need = PyObject_IsTrue(v[12]);
  if (need < 0) {
    PyErr_Clear();
    fail(what, "need_kv must be a truth value");
  }
  const Tensor q_out = output(what, "q_out", v[9], q, d);
  Tensor k_out, v_out;
  if (need || v[10] != Py_None) k_out = output(what, "k_out", v[10], k, d);
  if (need || v[11] != Py_None) v_out = output(what, "v_out", v[11], val, d);
  // an output may be its own input; nothing else may be written before it is read, or twice
  struct Named {
    const char* name;
    const Tensor* t;
    bool given;
  };
  const Named outs[3] = {{"q_out", &q_out, v[9] != Py_None}, {"k_out", &k_out, v[10] != Py_None}, {"v_out", &v_out, v[11] != Py_None}};
  const Named ins[3] = {{"q", &q, true}, {"k", &k, true}, {"v", &val, true}};
  for (int i = 0; i < 3; ++i) {
    if (!outs[i].given) continue;
    for (int j = 0; j < 3; ++j)
      if (i != j || !same_rows(*outs[i].t, *ins[j].t)) not_over(what, outs[i].name, *outs[i].t, ins[j].name, *ins[j].t);
    for (int j = 0; j < i; ++j)
      if (outs[j].given) not_over(what, outs[i].name, *outs[i].t, outs[j].name, *outs[j].t);
    for (const Tensor* t : {&ck.codes, &ck.params, &cv.codes, &cv.params}) bytes_apart(what, outs[i].name, *outs[i].t, "the cache", *t);
  }
  cos = aligned_table(cos);
  sin = aligned_table(sin);
  const Tensor qr = readable(q), kr = readable(k), vr = readable(val), p = positions.contiguous(), s = slots.contiguous();
  auto strides = [](const Tensor& t, int64_t i) { return t.defined() ? row_stride(t, i) : 0; };
  const int64_t st[12] = {strides(qr, 0), strides(qr, 1), strides(kr, 0), strides(kr, 1), strides(vr, 0), strides(vr, 1),
                          strides(q_out, 0), strides(q_out, 1), strides(k_out, 0), strides(k_out, 1), strides(v_out, 0),
                          strides(v_out, 1)};
  void* stream = c10::cuda::getCurrentCUDAStream(d.dev.index()).stream();
  int rc;
  {
    NoGil nogil;
    rc = li4_rope_paged_write_int4(qr.data_ptr(), kr.data_ptr(), vr.data_ptr(), type_code(q.scalar_type()), T, H, Hkv, D, st,
                                   cos.const_data_ptr<float>(), sin.const_data_ptr<float>(), D / 2, cos.size(0),
                                   p.const_data_ptr<int32_t>(), s.const_data_ptr<int64_t>(), q_out.data_ptr(),
                                   k_out.defined() ? k_out.data_ptr() : nullptr, v_out.defined() ? v_out.data_ptr() : nullptr,
                                   &ck.raw, &cv.raw, ck.codes.size(0), ck.codes.size(1), stream);
  }
  if (rc != LI4_OK) return PyLong_FromLong(rc);
  PyObject* r = PyTuple_New(3);
  PyTuple_SET_ITEM(r, 0, wrap(q_out));
  PyTuple_SET_ITEM(r, 1, k_out.defined() ? wrap(k_out) : Py_NewRef(Py_None));
  PyTuple_SET_ITEM(r, 2, v_out.defined() ? wrap(v_out) : Py_NewRef(Py_None));
  return r;
}

// (kv_lens, block_tables, free_pages, n_free, parents, page_size, pools, kv_lens_out, n_free_out)
PyObject* paged_fork(PyObject* const* v) {
  const char* what = "paged_fork";
  const Tensor kv = tensor(what, "kv_lens", v[0]), bt = tensor(what, "block_tables", v[1]),
               fp = tensor(what, "free_pages", v[2]), nf = tensor(what, "n_free", v[3]),
               parents = tensor(what, "parents", v[4]);
  Device d{what};
  d.add("kv_lens", kv);
  d.add("block_tables", bt);
  d.add("free_pages", fp);
  d.add("n_free", nf);
  d.add("parents", parents);
  if (kv.dim() != 1 || bt.dim() != 2 || fp.dim() != 1)
    fail(what, "kv_lens [requests], block_tables [requests, blocks] and free_pages [pages] expected");
  const int64_t B = kv.size(0), width = bt.size(1), capacity = fp.size(0);
  ints(what, "kv_lens", kv, at::kInt, {B});
  ints(what, "block_tables", bt, at::kInt, {B, width});
  ints(what, "free_pages", fp, at::kInt, {capacity});
  ints(what, "n_free", nf, at::kInt, {1});
  ints(what, "parents", parents, at::kInt, {B});
  if ((width > 1 && bt.stride(1) != 1) || (B > 1 && bt.stride(0) < width)) fail(what, "block_tables rows must be contiguous");
  if (capacity > 1 && fp.stride(0) != 1) fail(what, "free_pages must be contiguous");
  const int64_t page = integer(what, "page_size", v[5]);
  PyObject* seq = PySequence_Check(v[6]) && !THPVariable_Check(v[6]) ? PySequence_Fast(v[6], "pools") : nullptr;
  if (!seq) {
    PyErr_Clear();
    fail(what, "pools must be a sequence of tensors");
  }
  struct Drop {
    PyObject* o;
    ~Drop() { Py_DECREF(o); }
  } drop{seq};
  const int64_t given = PySequence_Fast_GET_SIZE(seq);
  std::vector<void*> pools;
  std::vector<int64_t> strides, bytes;
  pools.reserve(given), strides.reserve(given), bytes.reserve(given);
  for (int64_t i = 0; i < given; ++i) {
    const char* name = "a tensor of pools";
    const Tensor t = tensor(what, name, PySequence_Fast_GET_ITEM(seq, i));
    d.add(name, t);
    if (t.dim() < 1 || t.size(0) < capacity)
      fail(what, "pools[", i, "] must have ", capacity, " pages at least, got ", t.sizes());
    if (capacity == 0) continue;  // (no page to copy, whatever the strides of an empty tensor are)
    // a page is one block of memory, in whatever order of its dimensions
    int64_t block = 1, left = 1;
    for (int64_t k = 1; k < t.dim(); ++k) left *= t.size(k);
    const int64_t values = left;
    for (bool moved = true; moved && block < values;) {
      moved = false;
      for (int64_t k = 1; k < t.dim(); ++k)
        if (t.size(k) > 1 && t.stride(k) == block) {
          block *= t.size(k);
          moved = true;
          break;
        }
    }
    const int64_t size = t.element_size();
    if (block != values || values < 1 || (t.size(0) > 1 && t.stride(0) < values))
      fail(what, "pools[", i, "]: a page must be one block of memory, apart from the others");
    pools.push_back(t.data_ptr());
    bytes.push_back(values * size);
    strides.push_back(t.size(0) > 1 ? t.stride(0) * size : values * size);
  }
  const int64_t n_pools = (int64_t)pools.size();
  const c10::cuda::CUDAGuard guard(d.dev);
  const Tensor kc = kv.contiguous(), pc = parents.contiguous();
  auto result = [&](const char* name, PyObject* o, const Tensor& like) {
    if (o == Py_None) return empty(like.sizes(), at::kInt, d.dev);
    Tensor t = tensor(what, name, o);
    d.add(name, t);
    if (t.scalar_type() != at::kInt || t.sizes() != like.sizes() || !t.is_contiguous())
      fail(what, name, " must be contiguous int32 ", like.sizes());
    return t;
  };
  const Tensor kv_out = result("kv_lens_out", v[7], kv), nf_out = result("n_free_out", v[8], nf);
  const Tensor granted = empty({B}, at::kBool, d.dev);
  const size_t need = li4_paged_fork_workspace_bytes(B, width, capacity);
  Tensor ws;
  if (need) ws = empty({(int64_t)need}, at::kByte, d.dev);
  void* stream = c10::cuda::getCurrentCUDAStream(d.dev.index()).stream();
  int rc;
  {
    NoGil nogil;
    rc = li4_paged_fork(kc.const_data_ptr<int32_t>(), pc.const_data_ptr<int32_t>(), B, bt.data_ptr<int32_t>(),
                        B > 1 ? bt.stride(0) : width, width, fp.data_ptr<int32_t>(), capacity, nf.const_data_ptr<int32_t>(),
                        page, kv_out.data_ptr<int32_t>(), nf_out.data_ptr<int32_t>(),
                        reinterpret_cast<uint8_t*>(granted.data_ptr()), pools.data(), strides.data(), bytes.data(), n_pools,
                        need ? ws.data_ptr() : nullptr, need, stream);
  }
  if (rc != LI4_OK) return PyLong_FromLong(rc);
  PyObject* r = PyTuple_New(3);
  PyTuple_SET_ITEM(r, 0, wrap(kv_out));
  PyTuple_SET_ITEM(r, 1, wrap(nf_out));
  PyTuple_SET_ITEM(r, 2, wrap(granted));
  return r;
}

// (logits, tokens, top, entropy)
PyObject* token_logprobs(PyObject* const* v) {
  const char* what = "token_logprobs";
  const Tensor logits = tensor(what, "logits", v[0]);
  Device d{what};
  d.add("logits", logits);
  if (logits.dim() != 2) fail(what, "logits must be [rows, vocabulary], got ", logits.sizes());
  const at::ScalarType type = logits.scalar_type();
  const int code = type == at::kFloat ? (int)LI4_F32 : type_code(type);
  if (code < 0) fail(what, "logits must be float32, float16 or bfloat16, got ", type);
  const int64_t T = logits.size(0), V = logits.size(1);
  Tensor tokens;
  if (v[1] != Py_None) {
    tokens = tensor(what, "tokens", v[1]);
    d.add("tokens", tokens);
    ints(what, "tokens", tokens, at::kLong, {T});
  }
  const int64_t top = integer(what, "top", v[2]);
  if (V < 1) fail(what, "an empty vocabulary");
  if (top < 0 || top > LI4_MAX_TOP || top > V) fail(what, "top ", top, " of ", V, " tokens: from 0 to ", LI4_MAX_TOP);
  const int want_entropy = PyObject_IsTrue(v[3]);
  if (want_entropy < 0) {
    PyErr_Clear();
    fail(what, "entropy must be a truth value");
  }
  const c10::cuda::CUDAGuard guard(d.dev);
  const bool rows_fine = (V == 1 || logits.stride(1) == 1) && (T <= 1 || logits.stride(0) >= V);
  const Tensor x = rows_fine ? logits : logits.contiguous();
  Tensor tc, logprobs, entropy, ids, best;
  if (tokens.defined()) {
    tc = tokens.contiguous();
    logprobs = empty({T}, at::kFloat, d.dev);
  }
  if (want_entropy) entropy = empty({T}, at::kFloat, d.dev);
  if (top > 0) {
    ids = empty({T, top}, at::kLong, d.dev);
    best = empty({T, top}, at::kFloat, d.dev);
  }
  void* stream = c10::cuda::getCurrentCUDAStream(d.dev.index()).stream();
  int rc;
  {
    NoGil nogil;
    rc = li4_token_logprobs(x.data_ptr(), code, T, V, T > 1 ? x.stride(0) : V, tc.defined() ? tc.const_data_ptr<int64_t>() : nullptr,
                            top, tc.defined() ? logprobs.data_ptr<float>() : nullptr,
                            want_entropy ? entropy.data_ptr<float>() : nullptr, top > 0 ? ids.data_ptr<int64_t>() : nullptr,
                            top > 0 ? best.data_ptr<float>() : nullptr, stream);
  }
  if (rc != LI4_OK) return PyLong_FromLong(rc);
  const Tensor* all[4] = {&logprobs, &entropy, &ids, &best};
  PyObject* r = PyTuple_New(4);
  for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(r, i, all[i]->defined() ? wrap(*all[i]) : Py_NewRef(Py_None));
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
                         method<rope_paged_write_int4, 13>("rope_paged_write_int4"),
                         method<paged_attention_int4, 9>("paged_attention_int4"),
                         method<paged_fork, 9>("paged_fork"), method<token_logprobs, 4>("token_logprobs"),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "li4_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_li4_torch(void) { return PyModule_Create(&module); }
