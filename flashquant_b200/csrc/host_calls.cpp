// Extension module `_host`: the host side of the package's calls for arguments that need no
// conversion.
//
// A call through ctypes costs about 20 us of interpreter time (a dozen tensor look-ups, twenty
// boxed arguments, the stream object) in front of a launch of 2-4 us, more than the GPU needs for a small
// decode step.  Here the tensors are looked at in C++ and the C ABI is called directly
// (1 x 900-token decode step, append and decode: host time 42 -> 9 us).  Every function returns
// None when an argument is not exactly what the kernels take (another type, device, layout or
// a wrong shape): the caller in kernels.py then converts it or raises.  A failing native call
// returns its status as an int.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAFunctions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <tuple>
#include <vector>

#include "flashquant_b200.h"

namespace {

using at::Tensor;
using Args = PyObject* const*;

// A tensor argument as the kernels take it: on `dev`, contiguous.  Null if it is anything else.
const Tensor* raw_tensor(PyObject* o) {
  return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
}
// Device of the call: that of its first tensor, if that is the current device; else -1.
int call_device(PyObject* o) {
  const Tensor* t = raw_tensor(o);
  if (!t || !t->is_cuda()) return -1;
  const int dev = t->get_device();
  return dev == c10::cuda::current_device() ? dev : -1;
}
const Tensor* on_device(PyObject* o, int dev) {
  const Tensor* t = raw_tensor(o);
  return t && t->is_cuda() && t->get_device() == dev ? t : nullptr;
}
const Tensor* dense(PyObject* o, int dev) {
  const Tensor* t = on_device(o, dev);
  return t && t->is_contiguous() ? t : nullptr;
}
const Tensor* dense(PyObject* o, int dev, at::ScalarType st) {
  const Tensor* t = dense(o, dev);
  return t && t->scalar_type() == st ? t : nullptr;
}
const Tensor* f32(PyObject* o, int dev) { return dense(o, dev, at::kFloat); }

// -1: not a type the kernels read
int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return FQ_F32;
    case at::kHalf: return FQ_F16;
    case at::kBFloat16: return FQ_BF16;
    default: return -1;
  }
}
fq_stream_t stream_of(int dev) {
  return reinterpret_cast<fq_stream_t>(at::cuda::getCurrentCUDAStream(dev).stream());
}
PyObject* none() { Py_RETURN_NONE; }
PyObject* done(int rc, const Tensor& out) {
  return rc == FQ_OK ? THPVariable_Wrap(out) : PyLong_FromLong(rc);
}
PyObject* done(int rc) { return PyLong_FromLong(rc); }

bool as_int(PyObject* o, int64_t& v) {
  if (!PyLong_Check(o)) return false;
  v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return v >= INT32_MIN && v <= INT32_MAX;
}
// None: 1 / sqrt(head_dim)
bool as_scale(PyObject* o, int64_t head_dim, float& v) {
  if (o == Py_None) {
    v = float(1.0 / std::sqrt(double(head_dim)));
    return head_dim > 0;
  }
  if (!PyFloat_Check(o)) return false;
  v = float(PyFloat_AS_DOUBLE(o));
  return true;
}
template <typename T = float>
T* data(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }

// ------------------------------------------------------------------------------------
// Workspaces: one per (device, stream, use), zero at first use, grown on demand.  Calls on
// different streams may overlap on the GPU and must not share counters or partial rows.  None is given
// back: a call recorded in a CUDA graph keeps the address, so a workspace that was outgrown stays too
// (each is at least twice its predecessor, all of them together less than twice the last).  Those of the
// attention over 16-bit pages are as large as they have to be: 30 to 130 MB whatever the batch, by the heads, of which only
// the first 32 KiB have to be zero.
// ------------------------------------------------------------------------------------
enum { kDecode = 0, kAttention = 1, kDense = 2 };  // uses
constexpr int64_t kDenseHead = 32768;
using Kept = std::vector<Tensor>;  // the last one is in use
std::mutex g_ws_mutex;
std::map<std::tuple<int, const void*, int>, Kept>& workspaces() {
  static auto* m = new std::map<std::tuple<int, const void*, int>, Kept>();
  return *m;  // never destroyed: the CUDA context may be gone at exit
}
Tensor workspace(int dev, int use, size_t bytes) {
  const auto key = std::make_tuple(dev, static_cast<const void*>(stream_of(dev)), use);
  size_t have = size_t(1) << 19;
  {
    std::lock_guard<std::mutex> lock(g_ws_mutex);
    const Kept& kept = workspaces()[key];
    if (!kept.empty()) {
      have = size_t(kept.back().numel());
      if (have >= bytes) return kept.back();
    }
  }
  // (not under the lock: an allocation may run Python code, which may pass the interpreter on)
  const int64_t size = int64_t(use == kDense ? bytes : std::max(bytes, 2 * have));
  Tensor t = at::empty({size}, at::TensorOptions().device(at::kCUDA, dev).dtype(at::kByte));
  t.narrow(0, 0, use == kDense ? std::min(size, kDenseHead) : size).zero_();
  std::lock_guard<std::mutex> lock(g_ws_mutex);
  Kept& kept = workspaces()[key];
  if (kept.empty() || size_t(kept.back().numel()) < size_t(t.numel())) kept.push_back(t);
  return kept.back();
}
// The native call without the interpreter lock: a full launch queue makes it wait, and so do the calls of other threads that
// use the same workspace.
struct WithoutInterpreter {
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutInterpreter() { PyEval_RestoreThread(state); }
};
template <typename F>
int native(F call) {
  WithoutInterpreter released;
  return call();
}

// Bytes for one call: what a call writes and reads back within itself is not shared with another one.
Tensor call_bytes(int dev, size_t bytes, bool zero) {
  const auto options = at::TensorOptions().device(at::kCUDA, dev).dtype(at::kByte);
  return zero ? at::zeros({int64_t(bytes)}, options) : at::empty({int64_t(bytes)}, options);
}

// (device_index, use) -> the workspaces of all streams
PyObject* py_workspaces(PyObject*, Args a, Py_ssize_t n) {
  int64_t dev, use;
  if (n != 2 || !as_int(a[0], dev) || !as_int(a[1], use)) {
    PyErr_SetString(PyExc_TypeError, "workspaces(device_index, use)");
    return nullptr;
  }
  std::vector<Tensor> found;
  {
    std::lock_guard<std::mutex> lock(g_ws_mutex);
    for (const auto& [key, kept] : workspaces())
      if (std::get<0>(key) == dev && std::get<2>(key) == use)
        found.insert(found.end(), kept.begin(), kept.end());
  }
  PyObject* list = PyList_New(0);
  for (const Tensor& t : found) {
    PyObject* o = list ? THPVariable_Wrap(t) : nullptr;
    if (!o || PyList_Append(list, o)) Py_CLEAR(list);
    Py_XDECREF(o);
  }
  return list;
}

PyObject* py_workspace(PyObject*, Args a, Py_ssize_t n) {
  int64_t dev, use;
  if (n != 3 || !as_int(a[0], dev) || !as_int(a[1], use) || !PyLong_Check(a[2])) {
    PyErr_SetString(PyExc_TypeError, "workspace(device_index, use, bytes)");
    return nullptr;
  }
  try {
    return THPVariable_Wrap(workspace(int(dev), int(use), PyLong_AsSize_t(a[2])));
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// ------------------------------------------------------------------------------------
// compress-on-append
// ------------------------------------------------------------------------------------
struct Append {
  const Tensor *key, *value, *cache, *slots;
  int dt, h, d;
  int64_t n, stride, num_slots;
};
bool append_args(PyObject* k, PyObject* v, PyObject* cache, PyObject* slots, int dev, Append& p) {
  p.key = on_device(k, dev);
  p.value = on_device(v, dev);
  p.cache = dense(cache, dev, at::kByte);
  p.slots = dense(slots, dev);
  if (!p.key || !p.value || !p.cache || !p.slots) return false;
  const Tensor &key = *p.key, &val = *p.value;
  if (key.dim() != 3 || val.sizes() != key.sizes() || val.scalar_type() != key.scalar_type())
    return false;
  p.dt = dtype_code(key);
  p.n = key.size(0);
  p.h = int(key.size(1));
  p.d = int(key.size(2));
  p.stride = key.stride(0);
  if (p.dt < 0 || key.stride(2) != 1 || key.stride(1) != p.d || p.stride % 4 != 0 ||
      val.stride(2) != 1 || val.stride(1) != p.d || val.stride(0) != p.stride)
    return false;
  if (p.cache->dim() != 3 || p.cache->size(2) != int64_t(p.h) * (p.d + 8)) return false;
  const auto st = p.slots->scalar_type();
  if (st != at::kLong && st != at::kInt) return false;
  p.num_slots = p.cache->size(0) * p.cache->size(1);
  return true;
}

// (key, value, kv_cache, slot_mapping, rotation, boundaries_k, boundaries_v or None)
PyObject* compress_append(PyObject*, Args a, Py_ssize_t n) {
  const int dev = n == 7 ? call_device(a[0]) : -1;
  if (dev < 0) return none();
  Append p;
  const Tensor *rot = f32(a[4], dev), *bk = f32(a[5], dev);
  const Tensor* bv = a[6] == Py_None ? bk : f32(a[6], dev);
  if (!rot || !bk || !bv || !append_args(a[0], a[1], a[2], a[3], dev, p)) return none();
  return done(native([&] {
    return fq_tq4_compress_append(
      p.key->data_ptr(), p.value->data_ptr(), fq_dtype(p.dt), p.n, p.h, p.d, p.stride, data(*rot),
      data(*bk), int(bk->numel()), data(*bv), int(bv->numel()), data<uint8_t>(*p.cache),
      p.num_slots, p.slots->data_ptr(), p.slots->scalar_type() == at::kLong, stream_of(dev));
  }));
}

// (key, value, kv_cache, kq_cache, slot_mapping, rotation, boundaries_k, centroids_k,
//  boundaries_v, qjl_matrix)
PyObject* compress_append_qjl(PyObject*, Args a, Py_ssize_t n) {
  const int dev = n == 10 ? call_device(a[0]) : -1;
  if (dev < 0) return none();
  Append p;
  const Tensor* plane = dense(a[3], dev, at::kByte);
  const Tensor *rot = f32(a[5], dev), *bk = f32(a[6], dev), *ck = f32(a[7], dev),
               *bv = f32(a[8], dev), *s = f32(a[9], dev);
  if (!plane || !rot || !bk || !ck || !bv || !s || !append_args(a[0], a[1], a[2], a[4], dev, p))
    return none();
  if (plane->dim() != 3 || plane->size(2) != int64_t(p.h) * (p.d / 8 + 4) ||
      plane->size(0) * plane->size(1) != p.num_slots || s->dim() != 2 || s->size(0) != p.d ||
      s->size(1) != p.d || ck->numel() != bk->numel() + 1)
    return none();
  return done(native([&] {
    return fq_tq4_compress_append_qjl(
      p.key->data_ptr(), p.value->data_ptr(), fq_dtype(p.dt), p.n, p.h, p.d, p.stride, data(*rot),
      data(*bk), int(bk->numel()), data(*ck), data(*bv), int(bv->numel()), data(*s),
      data<uint8_t>(*p.cache), data<uint8_t>(*plane), p.num_slots, p.slots->data_ptr(),
      p.slots->scalar_type() == at::kLong, stream_of(dev));
  }));
}

// ------------------------------------------------------------------------------------
// paged decode
// ------------------------------------------------------------------------------------
struct Decode {
  const Tensor *q, *cache, *table, *lens, *ck, *cv, *rot;
  int dt, hq, hkv, d, bs, splits;
  float scale;
};
// q, kv_cache, block_table, seq_lens, centroids_k, centroids_v, rotation, num_kv_heads, head_dim,
// block_size, sm_scale, num_splits; `dims` dimensions of q (the last two: heads, head_dim)
bool decode_args(Args a, PyObject* scale, PyObject* splits, int dev, int dims, Decode& p) {
  p.q = dense(a[0], dev);
  p.cache = dense(a[1], dev, at::kByte);
  p.table = on_device(a[2], dev);
  p.lens = dense(a[3], dev, at::kInt);
  p.ck = f32(a[4], dev);
  p.cv = f32(a[5], dev);
  p.rot = f32(a[6], dev);
  int64_t hkv, d, bs, sp;
  if (!p.q || !p.cache || !p.table || !p.lens || !p.ck || !p.cv || !p.rot || !as_int(a[7], hkv) ||
      !as_int(a[8], d) || !as_int(a[9], bs) || !as_int(splits, sp) || !as_scale(scale, d, p.scale))
    return false;
  p.dt = dtype_code(*p.q);
  if (p.dt < 0 || p.q->dim() != dims || p.q->size(dims - 1) != d) return false;
  if (p.table->dim() != 2 || p.table->scalar_type() != at::kInt || p.table->stride(1) != 1)
    return false;
  if (p.cache->dim() != 3 || p.cache->size(1) != bs || p.cache->size(2) != hkv * (d + 8))
    return false;
  p.hq = int(p.q->size(dims - 2));
  p.hkv = int(hkv);
  p.d = int(d);
  p.bs = int(bs);
  p.splits = int(sp);
  return true;
}
// `out` argument: None makes a new tensor like q
bool decode_out(PyObject* o, const Tensor& q, int dev, Tensor& out) {
  if (o == Py_None) {
    out = at::empty(q.sizes(), q.options());
    return true;
  }
  const Tensor* t = dense(o, dev, q.scalar_type());
  if (!t || t->sizes() != q.sizes()) return false;
  out = *t;
  return true;
}

// (q, kv_cache, block_table, seq_lens, centroids_k, centroids_v, rotation, num_kv_heads, head_dim,
//  block_size, sm_scale, out, num_splits)
PyObject* paged_decode(PyObject*, Args a, Py_ssize_t n) {
  const int dev = n == 13 ? call_device(a[0]) : -1;
  if (dev < 0) return none();
  Decode p;
  Tensor out;
  if (!decode_args(a, a[10], a[12], dev, 3, p) || !decode_out(a[11], *p.q, dev, out)) return none();
  const int seqs = int(p.q->size(0));
  Tensor ws = workspace(dev, kDecode,
                        fq_paged_decode_workspace_bytes(seqs, p.hq, p.hkv, p.d, p.splits));
  return done(native([&] {
    return fq_split_k_paged_decode(
                  p.q->data_ptr(), fq_dtype(p.dt), data<uint8_t>(*p.cache), data<int32_t>(*p.table),
                  p.table->stride(0), data<int32_t>(*p.lens), data(*p.ck), int(p.ck->numel()),
                  data(*p.cv), int(p.cv->numel()), data(*p.rot), seqs, p.hq, p.hkv, p.d, p.bs,
                  p.cache->size(0), p.scale, out.data_ptr(), p.splits, ws.data_ptr(),
                  size_t(ws.numel()), stream_of(dev));
  }),
              out);
}

// (..., sm_scale, out, num_splits, kq_cache, qjl_matrix)
PyObject* paged_decode_qjl(PyObject*, Args a, Py_ssize_t n) {
  const int dev = n == 15 ? call_device(a[0]) : -1;
  if (dev < 0) return none();
  Decode p;
  Tensor out;
  const Tensor *plane = dense(a[13], dev, at::kByte), *s = f32(a[14], dev);
  if (!plane || !s || !decode_args(a, a[10], a[12], dev, 3, p) ||
      !decode_out(a[11], *p.q, dev, out))
    return none();
  if (plane->dim() != 3 || plane->size(0) != p.cache->size(0) || plane->size(1) != p.bs ||
      plane->size(2) != int64_t(p.hkv) * (p.d / 8 + 4) || s->dim() != 2 || s->size(0) != p.d ||
      s->size(1) != p.d)
    return none();
  const int seqs = int(p.q->size(0));
  Tensor ws = workspace(dev, kDecode,
                        fq_paged_decode_workspace_bytes(seqs, p.hq, p.hkv, p.d, p.splits));
  return done(native([&] {
    return fq_split_k_paged_decode_qjl(
                  p.q->data_ptr(), fq_dtype(p.dt), data<uint8_t>(*p.cache), data<uint8_t>(*plane),
                  data<int32_t>(*p.table), p.table->stride(0), data<int32_t>(*p.lens), data(*p.ck),
                  int(p.ck->numel()), data(*p.cv), int(p.cv->numel()), data(*p.rot), data(*s), seqs,
                  p.hq, p.hkv, p.d, p.bs, p.cache->size(0), p.scale, out.data_ptr(), p.splits,
                  ws.data_ptr(), size_t(ws.numel()), stream_of(dev));
  }),
              out);
}

// (q (num_seqs, n_q, H, D), ..., sm_scale, num_splits)
PyObject* paged_decode_multi(PyObject*, Args a, Py_ssize_t n) {
  const int dev = n == 12 ? call_device(a[0]) : -1;
  if (dev < 0) return none();
  Decode p;
  if (!decode_args(a, a[10], a[11], dev, 4, p)) return none();
  const int seqs = int(p.q->size(0)), n_q = int(p.q->size(1));
  if (seqs == 0 || n_q == 0) return none();
  Tensor out = at::empty(p.q->sizes(), p.q->options());
  const int max_blocks = int(p.table->size(1));
  Tensor ws = workspace(dev, kDecode,
                        std::max(fq_split_k_paged_decode_multi_workspace_bytes(
                                     seqs, n_q, p.hq, p.hkv, p.d, p.splits),
                                 fq_paged_decode_workspace_bytes(seqs * n_q, p.hq, p.hkv, p.d,
                                                                 p.splits)));
  Tensor scratch = call_bytes(
      dev, std::max<size_t>(fq_split_k_paged_decode_multi_scratch_bytes(seqs, n_q, max_blocks), 16),
      false);
  return done(native([&] {
    return fq_split_k_paged_decode_multi(
                  p.q->data_ptr(), fq_dtype(p.dt), data<uint8_t>(*p.cache), data<int32_t>(*p.table),
                  p.table->stride(0), max_blocks, data<int32_t>(*p.lens), data(*p.ck),
                  int(p.ck->numel()), data(*p.cv), int(p.cv->numel()), data(*p.rot), seqs, n_q,
                  p.hq, p.hkv, p.d, p.bs, p.cache->size(0), p.scale, out.data_ptr(), p.splits,
                  ws.data_ptr(), size_t(ws.numel()), scratch.data_ptr(), size_t(scratch.numel()),
                  stream_of(dev));
  }),
              out);
}

// (q, kv_cache, block_table, seq_lens, centroids_k, centroids_v, rotation, num_kv_heads, head_dim,
//  block_size, sm_scale, out, cu_seqlens_q, max_q_len)
PyObject* paged_prefill(PyObject*, Args a, Py_ssize_t n) {
  const int dev = n == 14 ? call_device(a[0]) : -1;
  if (dev < 0) return none();
  Decode p;
  Tensor out;
  int64_t max_q;
  static PyObject* zero = PyLong_FromLong(0);
  const Tensor* cu = dense(a[12], dev, at::kInt);
  if (!cu || !as_int(a[13], max_q) || !decode_args(a, a[10], zero, dev, 3, p) ||
      !decode_out(a[11], *p.q, dev, out) || cu->numel() != p.lens->numel() + 1)
    return none();
  const int total = int(p.q->size(0));
  Tensor ws = call_bytes(dev, fq_paged_tq4_prefill_workspace_bytes(total, p.hq, p.d), true);
  return done(native([&] {
    return fq_paged_tq4_prefill(
                  p.q->data_ptr(), fq_dtype(p.dt), data<uint8_t>(*p.cache), data<int32_t>(*p.table),
                  p.table->stride(0), data<int32_t>(*p.lens), data<int32_t>(*cu), data(*p.ck),
                  int(p.ck->numel()), data(*p.cv), int(p.cv->numel()), data(*p.rot),
                  int(p.lens->numel()), total, int(max_q), p.hq, p.hkv, p.d, p.bs,
                  p.cache->size(0), p.scale, out.data_ptr(), ws.data_ptr(), size_t(ws.numel()),
                  stream_of(dev));
  }),
              out);
}

// ------------------------------------------------------------------------------------
// contiguous form
// ------------------------------------------------------------------------------------
// (x (N, H, D), rotation_T_even, rotation_T_odd, boundaries) -> (packed, norms)
PyObject* compress(PyObject*, Args a, Py_ssize_t n) {
  const int dev = n == 4 ? call_device(a[0]) : -1;
  if (dev < 0) return none();
  const Tensor *x = dense(a[0], dev), *even = f32(a[1], dev), *odd = f32(a[2], dev),
               *bnd = f32(a[3], dev);
  if (!x || !even || !odd || !bnd || x->dim() != 3 || dtype_code(*x) < 0) return none();
  const int64_t nt = x->size(0), h = x->size(1), d = x->size(2);
  Tensor packed = at::empty({nt, h, d / 2}, x->options().dtype(at::kByte));
  Tensor norms = at::empty({nt, h, 1}, x->options().dtype(at::kFloat));
  const int rc = native([&] {
    return fq_tq4_compress(x->data_ptr(), fq_dtype(dtype_code(*x)), data(*even), data(*odd),
                                 data(*bnd), int(bnd->numel()), data<uint8_t>(packed), data(norms),
                                 nt * h, int(d), stream_of(dev));
  });
  if (rc != FQ_OK) return done(rc);
  PyObject* t = PyTuple_New(2);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(packed));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(norms));
  return t;
}

// Tokens between the (batch, head) rows of the buffers that codes and norms are [:, :, :n] views
// of (n where there is one row); 0 if they are not.  Strides of dimensions of size one say nothing.
int64_t view_capacity(const Tensor& codes, const Tensor& norms) {
  const int64_t b = codes.size(0), h = codes.size(1), n = codes.size(2), half = codes.size(3);
  if (n == 0 || half == 0 || norms.dim() != 4 || norms.size(0) != b || norms.size(1) != h ||
      norms.size(2) != n || norms.size(3) != 1)
    return 0;
  const int64_t cap = b * h == 1 ? n : codes.stride(h > 1 ? 1 : 0) / half;
  const auto laid_out = [&](const Tensor& t, int64_t unit) {
    const int64_t want[4] = {h * cap * unit, cap * unit, unit, 1};
    for (int i = 0; i < 4; ++i)
      if (t.size(i) > 1 && t.stride(i) != want[i]) return false;
    return true;
  };
  return cap >= n && laid_out(codes, half) && laid_out(norms, 1) ? cap : 0;
}

// (q, k_packed, k_norms, v_packed, v_norms, centroids_k, centroids_v, rotation_k, rotation_v,
//  sm_scale, is_causal)
PyObject* attention(PyObject*, Args a, Py_ssize_t n) {
  const int dev = n == 11 ? call_device(a[0]) : -1;
  if (dev < 0) return none();
  const Tensor* q = dense(a[0], dev);
  const Tensor* kv[4];
  for (int i = 0; i < 4; ++i) {
    kv[i] = on_device(a[1 + i], dev);
    if (!kv[i] || kv[i]->dim() != 4 || kv[i]->scalar_type() != (i & 1 ? at::kFloat : at::kByte))
      return none();
  }
  const Tensor *ck = f32(a[5], dev), *cv = f32(a[6], dev), *rk = f32(a[7], dev), *rv = f32(a[8], dev);
  float scale;
  if (!q || q->dim() != 4 || dtype_code(*q) < 0 || !ck || !cv || !rk || !rv ||
      !as_scale(a[9], q->size(3), scale) || !PyBool_Check(a[10]))
    return none();
  const int b = int(q->size(0)), hq = int(q->size(1)), nq = int(q->size(2)), d = int(q->size(3));
  const int hkv = int(kv[0]->size(1)), nkv = int(kv[0]->size(2));
  if (kv[0]->size(0) != b || kv[0]->size(3) * 2 != d || kv[2]->sizes() != kv[0]->sizes())
    return none();
  const int64_t cap = view_capacity(*kv[0], *kv[1]);
  if (cap == 0 || view_capacity(*kv[2], *kv[3]) != cap) return none();
  Tensor out = at::empty(q->sizes(), q->options());
  Tensor ws = workspace(dev, kAttention, fq_fused_tq_attention_workspace_bytes(b, hq, nq, d));
  return done(native([&] {
    return fq_fused_tq_attention_kv(
                  q->data_ptr(), fq_dtype(dtype_code(*q)), data<uint8_t>(*kv[0]), data(*kv[1]),
                  data<uint8_t>(*kv[2]), data(*kv[3]), data(*ck), int(ck->numel()), data(*cv),
                  int(cv->numel()), data(*rk), data(*rv), b, hq, hkv, nq, nkv, cap, d, scale,
                  a[10] == Py_True, out.data_ptr(), ws.data_ptr(), size_t(ws.numel()),
                  stream_of(dev));
  }),
              out);
}

// (key, value, tables_k, tables_v, k_packed, k_norms, v_packed, v_norms, position, k_out, v_out,
//  out_position, workspace)
PyObject* cache_update(PyObject*, Args a, Py_ssize_t n) {
  const int dev = n == 13 ? call_device(a[0]) : -1;
  if (dev < 0) return none();
  const Tensor *key = dense(a[0], dev), *val = dense(a[1], dev);
  if (!key || !val || key->dim() != 4 || dtype_code(*key) < 0 || val->sizes() != key->sizes() ||
      val->scalar_type() != key->scalar_type() || !PyTuple_Check(a[2]) || !PyTuple_Check(a[3]) ||
      PyTuple_GET_SIZE(a[2]) != 5 || PyTuple_GET_SIZE(a[3]) != 5)
    return none();
  const Tensor *tk[5], *tv[5];  // Pi^T even, Pi^T odd, boundaries, centroids, Pi
  for (int i = 0; i < 5; ++i) {
    tk[i] = f32(PyTuple_GET_ITEM(a[2], i), dev);
    tv[i] = f32(PyTuple_GET_ITEM(a[3], i), dev);
    if (!tk[i] || !tv[i]) return none();
  }
  const int64_t b = key->size(0), h = key->size(1), s = key->size(2), d = key->size(3);
  const Tensor* buf[4];
  for (int i = 0; i < 4; ++i) {
    buf[i] = dense(a[4 + i], dev, i & 1 ? at::kFloat : at::kByte);
    if (!buf[i] || buf[i]->dim() != 4) return none();
    const int64_t cap = buf[0]->size(2);
    if (buf[i]->size(0) != b || buf[i]->size(1) != h || buf[i]->size(2) != cap ||
        buf[i]->size(3) != (i & 1 ? 1 : d / 2))
      return none();
  }
  int64_t at, out_at;
  if (!as_int(a[8], at) || !as_int(a[11], out_at)) return none();
  const Tensor *ko = nullptr, *vo = nullptr, *ws = nullptr;
  int64_t out_cap = 0;
  size_t need = 0;
  if (a[9] != Py_None) {
    ko = dense(a[9], dev, key->scalar_type());
    vo = dense(a[10], dev, key->scalar_type());
    if (!ko || !vo || ko->dim() != 4 || ko->sizes() != vo->sizes() || ko->size(0) != b ||
        ko->size(1) != h || ko->size(3) != d)
      return none();
    out_cap = ko->size(2);
    need = fq_cache_update_workspace_bytes(b * h, s, int(d));
    if (need) {
      ws = dense(a[12], dev, at::kByte);
      if (!ws || size_t(ws->numel()) < need) return none();
    }
  } else if (a[10] != Py_None) {
    return none();
  }
  return done(native([&] {
    return fq_cache_update(
      key->data_ptr(), val->data_ptr(), fq_dtype(dtype_code(*key)), data(*tk[0]), data(*tk[1]),
      data(*tk[4]), data(*tv[0]), data(*tv[1]), data(*tv[4]), data(*tk[2]), int(tk[2]->numel()),
      data(*tk[3]), int(tk[3]->numel()), data<uint8_t>(*buf[0]), data(*buf[1]),
      data<uint8_t>(*buf[2]), data(*buf[3]), b * h, s, buf[0]->size(2), at,
      ko ? ko->data_ptr() : nullptr, vo ? vo->data_ptr() : nullptr, out_cap, out_at, int(d),
      ws ? ws->data_ptr() : nullptr, need, stream_of(dev));
  }));
}

// ------------------------------------------------------------------------------------
// around 16-bit pages
// ------------------------------------------------------------------------------------
// A contiguous tensor in the bytes of `base` from `offset` on: the results of a call that are used together come from
// one allocation (1.2 us of host time each).
Tensor carve(const Tensor& base, int64_t offset, at::IntArrayRef sizes, at::ScalarType st) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()),
                                                      c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                      c10::scalarTypeToTypeMeta(st));
  t.unsafeGetTensorImpl()->set_storage_offset(offset / int64_t(c10::elementSize(st)));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}
// (tokens, heads, head_dim) with adjacent values of a head
const Tensor* rows(PyObject* o, int dev) {
  const Tensor* t = on_device(o, dev);
  return t && t->dim() == 3 && t->stride(2) == 1 ? t : nullptr;
}
// no two rows (of the last dimension) share memory
bool own_rows(const Tensor& t) {
  int order[3], n = 0;  // the other dimensions by their strides
  for (int i = 0; i + 1 < t.dim() && n < 3; ++i)
    if (t.size(i) > 1) order[n++] = i;
  std::sort(order, order + n, [&](int i, int j) { return t.stride(i) < t.stride(j); });
  int64_t extent = t.size(-1);
  for (int k = 0; k < n; ++k) {
    if (t.stride(order[k]) < extent) return false;
    extent += t.stride(order[k]) * (t.size(order[k]) - 1);
  }
  return true;
}
// None makes a new tensor
bool out_rows(PyObject* o, const Tensor& like, int dev, Tensor& out) {
  if (o == Py_None) {
    out = at::empty(like.sizes(), like.options());
    return true;
  }
  const Tensor* t = rows(o, dev);
  if (!t || t->scalar_type() != like.scalar_type() || t->sizes() != like.sizes() || !own_rows(*t)) return false;
  out = *t;
  return true;
}
// (num_blocks, block_size, H_kv, D), the values of a row adjacent; `written`: its rows are its own
const Tensor* pages(PyObject* o, int dev, at::ScalarType st, bool written) {
  const Tensor* t = on_device(o, dev);
  if (!t || t->dim() != 4 || t->scalar_type() != st || t->stride(3) != 1) return nullptr;
  return written && !own_rows(*t) ? nullptr : t;
}
const Tensor* ints(PyObject* o, int dev, int64_t n) {
  const Tensor* t = dense(o, dev);
  return t && t->dim() == 1 && t->size(0) == n &&
                 (t->scalar_type() == at::kLong || t->scalar_type() == at::kInt)
             ? t
             : nullptr;
}
const Tensor* frequencies(PyObject* o, int dev, int64_t head_dim) {
  const Tensor* t = dense(o, dev, at::kDouble);
  return t && t->dim() == 1 && 2 * t->size(0) <= head_dim ? t : nullptr;
}
bool is_long(const Tensor& t) { return t.scalar_type() == at::kLong; }
PyObject* pair(const Tensor& a, const Tensor* b) {
  PyObject* t = PyTuple_New(2);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(a));
  if (!b) Py_INCREF(Py_None);
  PyTuple_SET_ITEM(t, 1, b ? THPVariable_Wrap(*b) : Py_None);
  return t;
}

// (q, k or None, positions, frequencies, layout, scale, inverse, out or None)
PyObject* rotary_embed(PyObject*, Args a, Py_ssize_t n) {
  const int dev = n == 8 ? call_device(a[0]) : -1;
  if (dev < 0) return none();
  const Tensor *q = rows(a[0], dev), *k = a[1] == Py_None ? nullptr : rows(a[1], dev);
  int64_t layout;
  if (!q || (!k && a[1] != Py_None) || dtype_code(*q) < 0 || !as_int(a[4], layout) || !PyFloat_Check(a[5]) ||
      !PyBool_Check(a[6]))
    return none();
  const int64_t tokens = q->size(0), d = q->size(2);
  const Tensor *pos = ints(a[2], dev, tokens), *freq = frequencies(a[3], dev, d);
  if (!pos || !freq || (k && (k->size(0) != tokens || k->size(2) != d || k->scalar_type() != q->scalar_type())))
    return none();
  PyObject *oq = Py_None, *ok = Py_None;
  if (a[7] != Py_None) {
    if (!PyTuple_Check(a[7]) || PyTuple_GET_SIZE(a[7]) != 2) return none();
    oq = PyTuple_GET_ITEM(a[7], 0);
    ok = PyTuple_GET_ITEM(a[7], 1);
  }
  Tensor q_out, k_out;
  if (k && oq == Py_None && ok == Py_None) {
    const int64_t size = int64_t(q->element_size()), first = (q->numel() * size + 255) / 256 * 256;
    const Tensor both = at::empty({first + k->numel() * size}, q->options().dtype(at::kByte));
    q_out = carve(both, 0, q->sizes(), q->scalar_type());
    k_out = carve(both, first, k->sizes(), k->scalar_type());
  } else if (!out_rows(oq, *q, dev, q_out) || (k ? !out_rows(ok, *k, dev, k_out) : ok != Py_None)) {
    return none();
  }
  const int64_t strides[8] = {q->stride(0), q->stride(1), k ? k->stride(0) : 0, k ? k->stride(1) : 0,
                              q_out.stride(0), q_out.stride(1), k ? k_out.stride(0) : 0, k ? k_out.stride(1) : 0};
  const int rc = native([&] {
    return fq_rotary_embed(q->data_ptr(), k ? k->data_ptr() : nullptr, fq_dtype(dtype_code(*q)), tokens,
                           int(q->size(1)), k ? int(k->size(1)) : 0, int(d), int(2 * freq->size(0)), strides,
                           pos->data_ptr(), is_long(*pos), data<double>(*freq), fq_rotary_layout(layout),
                           float(PyFloat_AS_DOUBLE(a[5])), a[6] == Py_True, q_out.data_ptr(),
                           k ? k_out.data_ptr() : nullptr, stream_of(dev));
  });
  return rc == FQ_OK ? pair(q_out, k ? &k_out : nullptr) : done(rc);
}

// (q or None, key, value, key_cache, value_cache, slot_mapping, positions, frequencies, layout, scale,
//  q_out or None)
PyObject* rotary_append_dense(PyObject*, Args a, Py_ssize_t n) {
  const int dev = n == 11 ? call_device(a[1]) : -1;
  // (what is not rotated, and has no result, is left to the other path)
  if (dev < 0 || a[0] == Py_None) return none();
  const Tensor *q = rows(a[0], dev), *key = rows(a[1], dev), *val = rows(a[2], dev);
  int64_t layout;
  if (!q || !key || !val || !as_int(a[8], layout) || !PyFloat_Check(a[9])) return none();
  const auto st = key->scalar_type();
  const int64_t tokens = key->size(0), h = key->size(1), d = key->size(2);
  if ((st != at::kHalf && st != at::kBFloat16) || q->scalar_type() != st || val->scalar_type() != st ||
      val->sizes() != key->sizes() || q->size(0) != tokens || q->size(2) != d)
    return none();
  const Tensor *kc = pages(a[3], dev, st, true), *vc = pages(a[4], dev, st, true);
  const Tensor *slots = ints(a[5], dev, tokens), *pos = ints(a[6], dev, tokens), *freq = frequencies(a[7], dev, d);
  if (!kc || !vc || !slots || !pos || !freq || kc->sizes() != vc->sizes() || kc->size(2) != h || kc->size(3) != d ||
      kc->size(1) < 1)
    return none();
  Tensor q_out;
  if (!out_rows(a[10], *q, dev, q_out)) return none();
  const int64_t strides[14] = {q->stride(0), q->stride(1), key->stride(0), key->stride(1), val->stride(0),
                               val->stride(1), q_out.stride(0), q_out.stride(1), kc->stride(0), kc->stride(1),
                               kc->stride(2), vc->stride(0), vc->stride(1), vc->stride(2)};
  return done(native([&] {
    return fq_rotary_append_dense(
                  q->data_ptr(), key->data_ptr(), val->data_ptr(), fq_dtype(dtype_code(*key)), tokens,
                  int(q->size(1)), int(h), int(d), int(2 * freq->size(0)), strides, pos->data_ptr(), is_long(*pos),
                  data<double>(*freq), fq_rotary_layout(layout), float(PyFloat_AS_DOUBLE(a[9])), q_out.data_ptr(),
                  kc->data_ptr(), vc->data_ptr(), int(kc->size(1)), kc->size(0) * kc->size(1), slots->data_ptr(),
                  is_long(*slots), stream_of(dev));
  }),
              q_out);
}

// (q, key_cache, value_cache, block_table, seq_lens, sm_scale, window, out or None, return_lse)
PyObject* dense_decode(PyObject*, Args a, Py_ssize_t n) {
  const int dev = n == 9 ? call_device(a[0]) : -1;
  if (dev < 0) return none();
  const Tensor *q = rows(a[0], dev), *table = on_device(a[3], dev), *lens = dense(a[4], dev, at::kInt);
  int64_t window;
  float scale;
  if (!q || !table || !lens || !as_int(a[6], window) || window < 0 || !PyBool_Check(a[8]) ||
      !as_scale(a[5], q->size(2), scale))
    return none();
  const auto st = q->scalar_type();
  const Tensor *kc = pages(a[1], dev, st, false), *vc = pages(a[2], dev, st, false);
  const int64_t seqs = q->size(0), hq = q->size(1), d = q->size(2);
  if ((st != at::kHalf && st != at::kBFloat16) || !kc || !vc || kc->sizes() != vc->sizes() || kc->size(3) != d ||
      q->stride(0) % 2 != 0 || q->stride(1) % 2 != 0 || reinterpret_cast<uintptr_t>(q->data_ptr()) % 4 != 0 ||
      table->dim() != 2 || table->size(0) != seqs || table->scalar_type() != at::kInt || table->stride(1) != 1 ||
      lens->dim() != 1 || lens->size(0) != seqs || seqs > INT32_MAX || hq > INT32_MAX)
    return none();
  Tensor out, lse;
  if (!decode_out(a[7], *q, dev, out)) return none();
  if (a[8] == Py_True) lse = at::empty({seqs, hq}, q->options().dtype(at::kFloat));
  const int hkv = int(kc->size(2));
  const size_t need = std::max<size_t>(fq_dense_paged_decode_workspace_bytes(int(seqs), int(hq), hkv, int(d)), kDenseHead);
  // A call that is being recorded has a workspace of its own: two graphs that hold the stream's would share its
  // counters when they run side by side.
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(reinterpret_cast<cudaStream_t>(stream_of(dev)), &capture) != cudaSuccess) return none();
  Tensor ws;
  if (capture == cudaStreamCaptureStatusNone) {
    ws = workspace(dev, kDense, need);
  } else {
    ws = call_bytes(dev, need, false);
    ws.narrow(0, 0, kDenseHead).zero_();
  }
  const int rc = native([&] {
    return fq_dense_paged_decode(
        q->data_ptr(), fq_dtype(dtype_code(*q)), q->stride(0), q->stride(1), kc->data_ptr(), kc->stride(0),
        kc->stride(1), kc->stride(2), vc->data_ptr(), vc->stride(0), vc->stride(1), vc->stride(2),
        data<int32_t>(*table), table->stride(0), int(table->size(1)), data<int32_t>(*lens), int(seqs), int(hq), hkv,
        int(d), int(kc->size(1)), kc->size(0), scale, int(window), out.data_ptr(),
        lse.defined() ? data(lse) : nullptr, ws.data_ptr(), size_t(ws.numel()), stream_of(dev));
  });
  if (rc != FQ_OK || !lse.defined()) return done(rc, out);
  return pair(out, &lse);
}

struct Pool {
  const Tensor *table, *free, *count;
  Tensor count_out;  // undefined where none was given
  int64_t requests, width, stride, block_size;
};
bool pool_args(PyObject* table, PyObject* free, PyObject* count, PyObject* block_size, PyObject* out, int dev, Pool& p) {
  p.table = on_device(table, dev);
  p.free = dense(free, dev, at::kInt);
  p.count = dense(count, dev, at::kInt);
  if (!p.table || !p.free || !p.count || p.table->dim() != 2 || p.table->scalar_type() != at::kInt ||
      p.table->stride(1) != 1 || p.free->dim() != 1 || p.count->numel() != 1 || !as_int(block_size, p.block_size) ||
      p.block_size < 1)
    return false;
  p.requests = p.table->size(0);
  p.width = p.table->size(1);
  p.stride = std::max(p.table->stride(0), p.width);
  if (p.requests > INT32_MAX || p.width > INT32_MAX || (p.requests > 1 && p.table->stride(0) < p.width)) return false;
  if (out == Py_None) return true;
  const Tensor* t = dense(out, dev, at::kInt);
  if (!t || t->numel() != 1) return false;
  p.count_out = *t;
  return true;
}

// (context_lens, query_lens, block_table, free_blocks, free_count, block_size, max_tokens, free_count_out or None)
PyObject* plan_paged_step(PyObject*, Args a, Py_ssize_t n) {
  const int dev = n == 8 ? call_device(a[2]) : -1;
  if (dev < 0) return none();
  Pool p;
  int64_t room;
  if (!as_int(a[6], room) || room < 0 || !pool_args(a[2], a[3], a[4], a[5], a[7], dev, p)) return none();
  const Tensor *context = dense(a[0], dev, at::kInt), *query = dense(a[1], dev, at::kInt);
  if (!context || !query || context->dim() != 1 || query->dim() != 1 || context->size(0) != p.requests ||
      query->size(0) != p.requests)
    return none();
  const auto part = [](int64_t n) { return (n + 15) / 16 * 16; };
  const int64_t r = p.requests, sizes[6] = {4 * r, 4 * (r + 1), 8 * room, 8 * room, r, 4};
  int64_t bytes = 0;
  for (int64_t n : sizes) bytes += part(n);
  const Tensor all = at::empty({bytes}, p.table->options().dtype(at::kByte));
  int64_t offset = 0;
  int made = 0;
  const auto piece = [&](int64_t n, at::ScalarType st) {
    offset += made ? part(sizes[made - 1]) : 0;
    ++made;
    return carve(all, offset, {n}, st);
  };
  Tensor out[6];
  out[0] = piece(r, at::kInt);
  out[1] = piece(r + 1, at::kInt);
  out[2] = piece(room, at::kLong);
  out[3] = piece(room, at::kLong);
  out[4] = piece(r, at::kBool);
  out[5] = p.count_out.defined() ? p.count_out : piece(1, at::kInt);
  const int rc = native([&] {
    return fq_plan_paged_step(data<int32_t>(*context), data<int32_t>(*query), int(p.requests), data<int32_t>(*p.table),
                              p.stride, int(p.width), int(p.block_size), data<int32_t>(*p.free), p.free->numel(),
                              data<int32_t>(*p.count), room, data<int32_t>(out[0]), data<int32_t>(out[1]),
                              data<int64_t>(out[2]), data<int64_t>(out[3]), data<uint8_t>(out[4]),
                              data<int32_t>(out[5]), stream_of(dev));
  });
  if (rc != FQ_OK) return done(rc);
  PyObject* t = PyTuple_New(6);
  for (int i = 0; t && i < 6; ++i) PyTuple_SET_ITEM(t, i, THPVariable_Wrap(out[i]));
  return t;
}

// (finished, context_lens, block_table, free_blocks, free_count, block_size, free_count_out or None)
PyObject* release_pages(PyObject*, Args a, Py_ssize_t n) {
  const int dev = n == 7 ? call_device(a[2]) : -1;
  if (dev < 0) return none();
  Pool p;
  if (!pool_args(a[2], a[3], a[4], a[5], a[6], dev, p)) return none();
  const Tensor *finished = dense(a[0], dev, at::kBool), *context = dense(a[1], dev, at::kInt);
  if (!finished || !context || finished->dim() != 1 || context->dim() != 1 || finished->size(0) != p.requests ||
      context->size(0) != p.requests)
    return none();
  if (!p.count_out.defined()) p.count_out = at::empty({1}, p.count->options());
  return done(native([&] {
    return fq_release_pages(data<uint8_t>(*finished), data<int32_t>(*context), int(p.requests),
                            data<int32_t>(*p.table), p.stride, int(p.width), int(p.block_size),
                            data<int32_t>(*p.free), p.free->numel(), data<int32_t>(*p.count),
                            data<int32_t>(p.count_out), stream_of(dev));
  }),
              p.count_out);
}

// C++ exceptions (an allocation that fails) become Python ones
PyObject* g_oom = nullptr;  // torch.OutOfMemoryError
template <PyObject* (*F)(PyObject*, Args, Py_ssize_t)>
PyObject* guarded(PyObject* self, Args a, Py_ssize_t n) {
  try {
    return F(self, a, n);
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(g_oom ? g_oom : PyExc_MemoryError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

#define FQ_METHOD(f) \
  { #f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<f>)), METH_FASTCALL, nullptr }
PyMethodDef kMethods[] = {
    FQ_METHOD(compress_append), FQ_METHOD(compress_append_qjl), FQ_METHOD(paged_decode),
    FQ_METHOD(paged_decode_qjl), FQ_METHOD(paged_decode_multi), FQ_METHOD(paged_prefill),
    FQ_METHOD(compress), FQ_METHOD(attention), FQ_METHOD(cache_update),
    FQ_METHOD(rotary_embed), FQ_METHOD(rotary_append_dense), FQ_METHOD(dense_decode),
    FQ_METHOD(plan_paged_step), FQ_METHOD(release_pages),
    {"workspaces", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&py_workspaces)),
     METH_FASTCALL, nullptr},
    {"workspace", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&py_workspace)),
     METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host",
                       "host side of the package's calls for arguments that need no conversion",
                       -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
  if (PyObject* torch = PyImport_ImportModule("torch")) {
    g_oom = PyObject_GetAttrString(torch, "OutOfMemoryError");
    Py_DECREF(torch);
  }
  if (PyErr_Occurred()) return nullptr;
  return PyModule_Create(&kModule);
}
