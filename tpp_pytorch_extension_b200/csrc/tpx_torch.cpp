// The operators of include/tpx_packed.h on torch tensors, as a Python extension module: checks of the arguments, outputs from torch's
// allocator, the call on torch's current stream. Through ctypes these cost 15 us of host time per call, several times what a decode
// step's kernels take; here 2-3 us and the launch. The CUDA library itself stays behind its C ABI: this file finds it by address.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstring>

#include "../../include/tpx_packed.h"

namespace {

PyObject* g_error = nullptr;  // the package's TpxError
struct {
  int (*head_prep)(const TpxHeadPrep*, void*);
  int (*int4_read)(const TpxInt4Cache*, const int32_t*, int64_t, uint16_t*, uint16_t*, void*);
  size_t (*scratch_bytes)(int64_t, int64_t, int64_t, int64_t, int64_t);
  int (*int4_attention)(const TpxInt4Attention*, void*);
  int (*int4_attention_behind)(const TpxInt4Attention*, void*);
  int (*packed_attention)(const TpxPackedAttention*, void*);
  int (*packed_attention_new)(const TpxPackedAttention*, const int32_t*, void*);
  const char* (*last_error)();
} g_lib;

// What is wrong with an argument; END_HANDLE_TH_ERRORS passes errors of torch itself on
struct Refused {};
[[noreturn]] void refuse(const char* fmt, ...) {
  char text[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof(text), fmt, ap);
  va_end(ap);
  PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, text);
  throw Refused();
}

#define TPX_BODY(...)                       \
  HANDLE_TH_ERRORS                          \
  try {                                     \
    __VA_ARGS__                             \
  } catch (const Refused&) {                \
    return nullptr;                         \
  }                                         \
  END_HANDLE_TH_ERRORS

struct Call {
  const char* name;
  PyObject* const* args;
  c10::DeviceIndex device = -1;  // of the tensors so far
  struct { uintptr_t from, to; } spans[12];  // memory of the arguments so far: an output may lie over none
  int spans_n = 0;

  void note(const void* from, int64_t bytes) {
    if (bytes > 0) spans[spans_n++] = {(uintptr_t)from, (uintptr_t)from + (uintptr_t)bytes};
  }
  static int64_t extent(const at::Tensor& t) {
    if (t.numel() == 0) return 0;
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); i++) last += (t.size(i) - 1) * t.stride(i);
    return (last + 1) * (int64_t)t.element_size();
  }

  void on(const at::Tensor& t, const char* what) {
    if (!t.is_cuda()) refuse("%s: %s must be on a CUDA device (this library has no CPU path)", name, what);
    if (device < 0) {
      device = t.get_device();
      const c10::DeviceIndex now = c10::cuda::current_device();
      if (device != now) refuse("%s: tensors are on cuda:%d, the current device is cuda:%d", name, (int)device, (int)now);
    }
    if (t.get_device() != device) refuse("%s: tensors are on cuda:%d and cuda:%d", name, (int)device, (int)t.get_device());
    if (t.requires_grad() && c10::GradMode::is_enabled()) refuse("%s has no backward pass: call it under torch.no_grad()", name);
  }
  bool none(int i) const { return args[i] == Py_None; }
  const at::Tensor& tensor(int i, const char* what) {
    if (!THPVariable_Check(args[i])) refuse("%s: %s must be a tensor", name, what);
    const at::Tensor& t = THPVariable_Unpack(args[i]);
    on(t, what);
    note(t.data_ptr(), extent(t));
    return t;
  }
  int64_t integer(int i, const char* what) {
    const long long v = PyLong_AsLongLong(args[i]);
    if (v == -1 && PyErr_Occurred()) throw Refused();
    if (v < 0 || v > (1ll << 31)) refuse("%s: %s is %lld", name, what, v);
    return v;
  }
  double real(int i) {
    const double v = PyFloat_AsDouble(args[i]);
    if (v == -1.0 && PyErr_Occurred()) throw Refused();
    return v;
  }
  bool truth(int i) {
    const int v = PyObject_IsTrue(args[i]);
    if (v < 0) throw Refused();
    return v != 0;
  }
  // elements between the rows of t [T, heads, dim], whose heads lie side by side
  int64_t rows(const at::Tensor& t, const char* what, int64_t heads, int64_t dim) {
    if (t.scalar_type() != at::kBFloat16 || t.dim() != 3 || t.size(1) != heads || t.size(2) != dim || (dim > 1 && t.stride(2) != 1) || (heads > 1 && t.stride(1) != dim))
      refuse("%s: %s must be bf16 [tokens, %lld, %lld] with heads side by side", name, what, (long long)heads, (long long)dim);
    if (t.size(0) < 2) return heads * dim;
    if (t.stride(0) < heads * dim) refuse("%s: rows of %s overlap", name, what);
    return t.stride(0);
  }
  // cu_seqlens of `sequences` (below 0: of any number); nullptr for None
  const int32_t* cuts(int i, int64_t sequences, int64_t T) {
    if (none(i)) {
      if (sequences >= 0 && T != sequences)
        refuse("%s: %lld tokens without cu_seqlens are not one for each of %lld sequences", name, (long long)T, (long long)sequences);
      return nullptr;
    }
    const at::Tensor& t = tensor(i, "cu_seqlens");
    if (t.scalar_type() != at::kInt || t.dim() != 1 || !t.is_contiguous() || (sequences >= 0 ? t.size(0) != sequences + 1 : t.size(0) < 2))
      refuse("%s: cu_seqlens must be contiguous int32 with one value more than there are sequences", name);
    return t.const_data_ptr<int32_t>();
  }
  at::Tensor output(int i, c10::IntArrayRef shape) {
    if (i < 0 || none(i)) return at::empty(shape, at::TensorOptions().dtype(at::kBFloat16).device(at::kCUDA, device));
    if (!THPVariable_Check(args[i])) refuse("%s: the output must be a tensor", name);
    const at::Tensor& t = THPVariable_Unpack(args[i]);
    on(t, "the output");
    if (t.scalar_type() != at::kBFloat16 || t.sizes() != shape || !t.is_contiguous()) refuse("%s: the output must be contiguous bf16 of the result's shape", name);
    const uintptr_t from = (uintptr_t)t.data_ptr(), to = from + (uintptr_t)extent(t);
    for (int k = 0; k < spans_n; k++)
      if (from < spans[k].to && spans[k].from < to) refuse("%s: the output overlaps another argument", name);
    note(t.data_ptr(), extent(t));
    return t;
  }
  void* stream() { return (void*)c10::cuda::getCurrentCUDAStream(device).stream(); }
  void done(int rc) {
    if (rc != 0) refuse("tpx error %d: %s", rc, g_lib.last_error());
  }
};

uint16_t* bf16(const at::Tensor& t) { return reinterpret_cast<uint16_t*>(t.data_ptr()); }

// A cache's layer travels as bytes: the block of the C ABI and the device
struct CacheBytes {
  TpxInt4Cache c;
  int64_t device;
};
const TpxInt4Cache* cache_of(Call& c, int i) {
  if (c.none(i)) return nullptr;
  if (!PyBytes_Check(c.args[i]) || PyBytes_GET_SIZE(c.args[i]) != sizeof(CacheBytes)) refuse("%s: not a layer of a cache", c.name);
  const CacheBytes* b = reinterpret_cast<const CacheBytes*>(PyBytes_AS_STRING(c.args[i]));
  if (c.device >= 0 && b->device != c.device) refuse("%s: tensors are on cuda:%d, the cache is on cuda:%d", c.name, (int)c.device, (int)b->device);
  if (c.device < 0) {
    const c10::DeviceIndex now = c10::cuda::current_device();
    if (b->device != now) refuse("%s: the cache is on cuda:%d, the current device is cuda:%d", c.name, (int)b->device, (int)now);
    c.device = now;
  }
  c.note(b->c.pool, b->c.pages * b->c.kv_heads * 36 * b->c.H);
  c.note(b->c.table, b->c.B * b->c.table_cols * 4);
  c.note(b->c.lengths, b->c.B * 4);
  return &b->c;
}

bool arity(const char* name, Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", name, want);
  return false;
}

PyObject* two(at::Tensor a, at::Tensor b) {
  PyObject* pa = THPVariable_Wrap(std::move(a));
  PyObject* pb = b.defined() ? THPVariable_Wrap(std::move(b)) : (Py_INCREF(Py_None), Py_None);
  PyObject* r = pa && pb ? PyTuple_Pack(2, pa, pb) : nullptr;
  Py_XDECREF(pa);
  Py_XDECREF(pb);
  return r;
}

// cache_bytes(pool, table, lengths) -> bytes
PyObject* cache_bytes(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!arity("cache_bytes", n, 3)) return nullptr;
  TPX_BODY(
    Call c{"Int4Cache", args};
    for (int i = 0; i < 3; i++)
      if (!THPVariable_Check(args[i])) refuse("Int4Cache: pool, table and lengths must be tensors");
    const at::Tensor& pool = THPVariable_Unpack(args[0]); const at::Tensor& table = THPVariable_Unpack(args[1]);
    const at::Tensor& lengths = THPVariable_Unpack(args[2]);
    const int64_t H = pool.dim() == 3 ? pool.size(2) / 36 : 0;
    if (pool.scalar_type() != at::kByte || pool.dim() != 3 || !pool.is_contiguous() || (H != 64 && H != 128) || pool.size(2) != 36 * H || pool.numel() == 0)
      refuse("Int4Cache: a pool must be contiguous uint8 [pages, kv_heads, 36 * head size], head size 64 or 128");
    if (table.scalar_type() != at::kInt || table.dim() != 2 || !table.is_contiguous() || table.numel() == 0) refuse("Int4Cache: the table must be contiguous int32 [sequences, columns]");
    if (lengths.scalar_type() != at::kInt || lengths.dim() != 1 || lengths.size(0) != table.size(0) || !lengths.is_contiguous()) refuse("Int4Cache: lengths must be int32 [sequences]");
    if (pool.device() != table.device() || pool.device() != lengths.device()) refuse("Int4Cache: pool, table and lengths must be on one device");
    CacheBytes b{};
    b.c.pool = (uint8_t*)pool.data_ptr();
    b.c.table = (const int32_t*)table.data_ptr();
    b.c.lengths = (const int32_t*)lengths.data_ptr();
    b.c.pages = pool.size(0);
    b.c.table_cols = table.size(1);
    b.c.B = table.size(0);
    b.c.kv_heads = pool.size(1);
    b.c.H = H;
    b.device = pool.is_cuda() ? pool.get_device() : -1;
    return PyBytes_FromStringAndSize((const char*)&b, sizeof(b));
  )
}

// head_prep(qkv, heads, kv_heads, head_dim, q_norm, k_norm, eps, ep, positions, cu_seqlens, cache, want_k, q_out, k_out) -> (q, k)
PyObject* head_prep(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!arity("head_prep", n, 14)) return nullptr;
  TPX_BODY(
    Call c{"qk_norm_rope", args};
    const at::Tensor& qkv = c.tensor(0, "qkv");
    TpxHeadPrep a{};
    a.Nq = c.integer(1, "heads");
    a.Nkv = c.integer(2, "kv_heads");
    a.H = c.integer(3, "head_dim");
    if (a.Nq > 4096 || a.Nkv > 1024 || a.H > 4096 || a.Nq + a.Nkv == 0) refuse("qk_norm_rope: %lld query and %lld key heads of %lld", (long long)a.Nq, (long long)a.Nkv, (long long)a.H);
    const int64_t width = (a.Nq + 2 * a.Nkv) * a.H;
    if (qkv.scalar_type() != at::kBFloat16 || qkv.dim() != 2 || qkv.size(1) != width || (width > 1 && qkv.stride(1) != 1) || (qkv.size(0) > 1 && qkv.stride(0) < width))
      refuse("qk_norm_rope: qkv must be bf16 [tokens, %lld]", (long long)width);
    a.T = qkv.size(0);
    a.ldq = a.ldk = a.ldv = a.T > 1 ? qkv.stride(0) : width;
    a.q = bf16(qkv);
    a.k = a.q + a.Nq * a.H;
    a.v = a.k + a.Nkv * a.H;
    int types = 0;
    for (int i = 4; i < 6; i++) {
      if (c.none(i)) continue;
      const at::Tensor& w = c.tensor(i, "a norm weight");
      if (w.numel() != a.H || !w.is_contiguous() || (w.scalar_type() != at::kBFloat16 && w.scalar_type() != at::kFloat)) refuse("qk_norm_rope: norm weights must be bf16 or fp32 [%lld]", (long long)a.H);
      types |= w.scalar_type() == at::kFloat ? 2 : 1;
      (i == 4 ? a.q_norm : a.k_norm) = w.data_ptr();
    }
    if (types == 3) refuse("qk_norm_rope: both norm weights must have one type");
    a.norm_is_f32 = types == 2;
    a.eps = (float)c.real(6);
    a.cache = nullptr;
    if (!c.none(7)) {
      const at::Tensor& ep = c.tensor(7, "the rotation table");
      if (ep.scalar_type() != at::kFloat || ep.dim() != 3 || ep.size(0) != 2 || !ep.is_contiguous()) refuse("qk_norm_rope: the rotation table must be contiguous fp32 [2, positions, rotated values]");
      a.ep = ep.const_data_ptr<float>();
      a.max_pos = ep.size(1);
      a.rot = a.ld_ep = ep.size(2);
      if (c.none(8) && c.none(10)) refuse("qk_norm_rope: positions are needed to rotate without a cache");
    }
    if (!c.none(8)) {
      const at::Tensor& pos = c.tensor(8, "positions");
      if (pos.scalar_type() != at::kLong || !pos.is_contiguous() || pos.numel() != a.T) refuse("qk_norm_rope: positions must be contiguous int64, one per token");
      a.pos = pos.const_data_ptr<int64_t>();
    }
    a.cache = cache_of(c, 10);
    if (a.cache) a.cu_seqlens = c.cuts(9, a.cache->B, a.T);
    else if (!c.none(9)) refuse("qk_norm_rope: cu_seqlens cuts the tokens of a cache");
    at::Tensor q = c.output(12, {a.T, a.Nq, a.H});
    at::Tensor k;
    if (c.truth(11) || !c.none(13)) k = c.output(13, {a.T, a.Nkv, a.H});
    a.q_out = bf16(q);
    a.k_out = k.defined() ? bf16(k) : nullptr;
    c.done(g_lib.head_prep(&a, c.stream()));
    return two(std::move(q), std::move(k));
  )
}

// append(k, v, cache, cu_seqlens)
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!arity("append", n, 4)) return nullptr;
  TPX_BODY(
    Call c{"append_int4", args};
    const at::Tensor& k = c.tensor(0, "k"); const at::Tensor& v = c.tensor(1, "v");
    const TpxInt4Cache* cache = cache_of(c, 2);
    if (!cache) refuse("append_int4: a cache is needed");
    TpxHeadPrep a{};
    a.Nkv = cache->kv_heads;
    a.H = cache->H;
    a.T = k.dim() ? k.size(0) : 0;
    a.ldk = c.rows(k, "k", a.Nkv, a.H);
    a.ldv = c.rows(v, "v", a.Nkv, a.H);
    if (v.size(0) != a.T) refuse("append_int4: k and v differ in their tokens");
    a.k = bf16(k);
    a.v = bf16(v);
    a.cache = cache;
    a.cu_seqlens = c.cuts(3, cache->B, a.T);
    c.done(g_lib.head_prep(&a, c.stream()));
    Py_RETURN_NONE;
  )
}

// read(cache, tokens, cu_seqlens, lengths) -> (k, v)
PyObject* read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!arity("read", n, 4)) return nullptr;
  TPX_BODY(
    Call c{"read_int4", args};
    const TpxInt4Cache* cache = cache_of(c, 0);
    if (!cache) refuse("read_int4: a cache is needed");
    TpxInt4Cache own = *cache;
    const int64_t T = c.integer(1, "tokens");
    const int32_t* cu = c.cuts(2, own.B, T);
    if (!c.none(3)) {
      const at::Tensor& l = c.tensor(3, "lengths");
      if (l.scalar_type() != at::kInt || l.dim() != 1 || l.size(0) != own.B || !l.is_contiguous()) refuse("read_int4: lengths must be int32 [%lld]", (long long)own.B);
      own.lengths = l.const_data_ptr<int32_t>();
    }
    at::Tensor k = c.output(-1, {T, own.kv_heads, own.H});
    at::Tensor v = c.output(-1, {T, own.kv_heads, own.H});
    c.done(g_lib.int4_read(&own, cu, T, bf16(k), bf16(v), c.stream()));
    return two(std::move(k), std::move(v));
  )
}

// int4_attention(q, cache, cu_seqlens, causal, scale, out, behind) -> out
PyObject* int4_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!arity("int4_attention", n, 7)) return nullptr;
  TPX_BODY(
    Call c{"attention_int4", args};
    const at::Tensor& q = c.tensor(0, "q");
    TpxInt4Attention a{};
    a.cache = cache_of(c, 1);
    if (!a.cache) refuse("attention_int4: a cache is needed");
    const int64_t H = a.cache->H; const int64_t Nkv = a.cache->kv_heads;
    a.Nq = q.dim() == 3 ? q.size(1) : 0;
    if (a.Nq == 0 || a.Nq % Nkv) refuse("attention_int4: q must be bf16 [tokens, heads, %lld], heads a multiple of %lld", (long long)H, (long long)Nkv);
    a.T = q.size(0);
    a.ldq = c.rows(q, "q", a.Nq, H);
    a.cu_seqlens = c.cuts(2, a.cache->B, a.T);
    a.causal = c.truth(3);
    a.scale = c.none(4) ? (float)(1.0 / std::sqrt((double)H)) : (float)c.real(4);
    const bool behind = c.truth(6);
    at::Tensor out = c.output(5, {a.T, a.Nq, H});
    a.scratch_bytes = g_lib.scratch_bytes(a.T, a.cache->B, a.Nq, Nkv, H);
    // of this call alone: calls on two streams, and two graphs, share nothing
    at::Tensor scratch = at::empty({(int64_t)a.scratch_bytes}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, c.device));
    a.scratch = scratch.data_ptr();
    a.q = bf16(q);
    a.out = bf16(out);
    c.done(behind ? g_lib.int4_attention_behind(&a, c.stream()) : g_lib.int4_attention(&a, c.stream()));
    return THPVariable_Wrap(std::move(out));
  )
}

// packed_attention(q, k, v, cu_seqlens, causal, scale, out, lengths) -> out
PyObject* packed_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!arity("packed_attention", n, 8)) return nullptr;
  TPX_BODY(
    Call c{"attention_packed", args};
    const at::Tensor& q = c.tensor(0, "q"); const at::Tensor& k = c.tensor(1, "k"); const at::Tensor& v = c.tensor(2, "v");
    if (q.dim() != 3 || k.dim() != 3 || k.sizes() != v.sizes() || k.size(0) != q.size(0) || k.size(1) == 0 || q.size(1) == 0 || q.size(1) % k.size(1))
      refuse("attention_packed: q, k and v must be [tokens, heads, dim], [tokens, kv_heads, dim] twice, heads a multiple of kv_heads");
    TpxPackedAttention a{};
    a.T = q.size(0);
    a.Nq = q.size(1);
    a.Nkv = k.size(1);
    a.H = q.size(2);
    a.ldq = c.rows(q, "q", a.Nq, a.H);
    a.ldk = c.rows(k, "k", a.Nkv, a.H);
    a.ldv = c.rows(v, "v", a.Nkv, a.H);
    a.cu_seqlens = c.cuts(3, -1, a.T);
    if (!a.cu_seqlens) refuse("attention_packed: cu_seqlens is needed");
    a.B = THPVariable_Unpack(args[3]).size(0) - 1;
    a.causal = c.truth(4);
    a.scale = c.none(5) ? (float)(1.0 / std::sqrt((double)a.H)) : (float)c.real(5);
    const int32_t* cached = nullptr;
    if (!c.none(7)) {
      const at::Tensor& l = c.tensor(7, "lengths");
      if (l.scalar_type() != at::kInt || l.dim() != 1 || l.size(0) != a.B || !l.is_contiguous()) refuse("attention_packed: lengths must be int32 [%lld]", (long long)a.B);
      cached = l.const_data_ptr<int32_t>();
    }
    at::Tensor out = c.output(6, {a.T, a.Nq, a.H});
    a.q = bf16(q);
    a.k = bf16(k);
    a.v = bf16(v);
    a.out = bf16(out);
    c.done(cached ? g_lib.packed_attention_new(&a, cached, c.stream()) : g_lib.packed_attention(&a, c.stream()));
    return THPVariable_Wrap(std::move(out));
  )
}

// bind(error class, addresses of the library's functions in the order of g_lib)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!arity("bind", n, 9)) return nullptr;
  static_assert(sizeof(g_lib) == 8 * sizeof(void*), "addresses");
  void* at[8];
  for (int i = 0; i < 8; i++) {
    at[i] = PyLong_AsVoidPtr(args[i + 1]);
    if (PyErr_Occurred()) return nullptr;
  }
  std::memcpy(&g_lib, at, sizeof(at));
  Py_INCREF(args[0]);
  Py_XDECREF(g_error);
  g_error = args[0];
  Py_RETURN_NONE;
}

#define TPX_FN(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {TPX_FN(bind),           TPX_FN(cache_bytes),      TPX_FN(head_prep), TPX_FN(append), TPX_FN(read),
                         TPX_FN(int4_attention), TPX_FN(packed_attention), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tpx_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tpx_torch(void) { return PyModule_Create(&module); }
