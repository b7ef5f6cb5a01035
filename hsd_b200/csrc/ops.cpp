// Python binding of the 8-bit cache and the several-axes rotary embedding:
// the checks, output tensors, workspaces and stream lookup of one call in C++
// (a call from Python through ctypes took 11 to 48 us of host time, more than
// most of these kernels run).  The work is the C ABI's (include/hsd_b200.h); no
// kernel is launched from here.  Python signatures and documentation:
// hsd_b200/rope.py and hsd_b200/kv8.py.
//
// Refusals are ValueError or TypeError; a status from the library raises
// hsd_b200._native.HSDError.  Nothing is thrown across the interpreter.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstdio>
#include <map>
#include <string>
#include <utility>

#include "hsd_b200.h"

namespace {

struct Refused {
  PyObject* type;  // borrowed
  std::string what;
};

[[noreturn]] void refuse(PyObject* type, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  throw Refused{type, buf};
}

struct PythonError {};  // an exception is already set

PyObject* hsd_error() {
  static PyObject* cls = nullptr;
  if (!cls) {
    PyObject* m = PyImport_ImportModule("hsd_b200._native");
    if (m) {
      cls = PyObject_GetAttrString(m, "HSDError");
      Py_DECREF(m);
    }
    if (!cls) throw PythonError{};
  }
  return cls;
}

void check(int rc, const char* what) {
  if (rc != HSD_OK) refuse(hsd_error(), "%s failed (%d): %s", what, rc, hsd_last_error());
}

// ---------------------------------------------------------------- arguments
struct Args {
  PyObject* const* a;
  const char* fn;
  bool none(int i) const { return a[i] == Py_None; }
  const at::Tensor& tensor(int i, const char* name) const {
    if (!THPVariable_Check(a[i])) refuse(PyExc_TypeError, "%s: %s must be a tensor", fn, name);
    return THPVariable_Unpack(a[i]);
  }
  int64_t integer(int i) const {
    const Py_ssize_t v = PyNumber_AsSsize_t(a[i], PyExc_OverflowError);
    if (v == -1 && PyErr_Occurred()) throw PythonError{};
    return v;
  }
  double real(int i) const {
    const double v = PyFloat_AsDouble(a[i]);
    if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
    return v;
  }
};

std::string shape(const at::Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

// ``[..., rows, width]`` -> rows of one stride.
struct Rows {
  char* ptr;
  int64_t rows, stride;
  at::Tensor keep;
};

Rows rows_of(const Args& a, const at::Tensor& t, const char* name, int64_t width, bool written) {
  if (t.scalar_type() != at::kBFloat16 || !t.is_cuda())
    refuse(PyExc_TypeError, "%s: %s must be a bf16 CUDA tensor", a.fn, name);
  if (t.dim() < 2 || t.size(-1) != width)
    refuse(PyExc_ValueError, "%s: %s has shape %s, expected [..., rows, %lld]", a.fn, name,
           shape(t).c_str(), static_cast<long long>(width));
  Rows r;
  r.keep = t.dim() == 2 ? t : t.reshape({-1, width});
  if (written && r.keep.data_ptr() != t.data_ptr())
    refuse(PyExc_ValueError, "%s: %s must be rows of one stride", a.fn, name);
  if (r.keep.stride(1) != 1)
    refuse(PyExc_ValueError, "%s: %s rows must be contiguous", a.fn, name);
  r.ptr = static_cast<char*>(r.keep.data_ptr());
  r.rows = r.keep.size(0);
  r.stride = r.rows > 1 ? r.keep.stride(0) : width;  // a single row's stride is never used
  return r;
}

struct Cache {
  char* ptr;
  int64_t heads, rows, head_stride, row_stride;
};

Cache cache_of(const Args& a, const at::Tensor& t, const char* name) {
  if (t.scalar_type() != at::kBFloat16 || !t.is_cuda())
    refuse(PyExc_TypeError, "%s: %s must be a bf16 CUDA tensor", a.fn, name);
  bool ok = t.dim() >= 3 && t.size(-1) == 128 && t.stride(-1) == 1;
  for (int64_t i = 0; ok && i < t.dim() - 3; ++i) ok = t.size(i) == 1;
  if (!ok)
    refuse(PyExc_ValueError, "%s: %s must be [Hkv, KV, 128] with contiguous rows", a.fn, name);
  Cache c;
  c.ptr = static_cast<char*>(t.data_ptr());
  c.heads = t.size(-3);
  c.rows = t.size(-2);
  c.row_stride = c.rows > 1 ? t.stride(-2) : 128;
  c.head_stride = c.heads > 1 ? t.stride(-3) : 128;
  // rows are written: heads or rows in one place (an expanded tensor) would be a race
  if (c.heads > 1 && c.rows > 0 && c.head_stride == 0)
    refuse(PyExc_ValueError, "%s: %s has its heads in one place (stride 0)", a.fn, name);
  return c;
}

void same_device(const Args& a, const at::Tensor& t, const c10::Device& dev, const char* name) {
  if (t.device() != dev)
    refuse(PyExc_ValueError, "%s: %s must be on %s", a.fn, name, dev.str().c_str());
}

int32_t* status_of(const Args& a, int i, const c10::Device& dev) {
  if (a.none(i)) return nullptr;
  const at::Tensor& t = a.tensor(i, "status");
  if (t.scalar_type() != at::kInt || t.numel() < 1)
    refuse(PyExc_ValueError, "%s: status must be an int32 word", a.fn);
  same_device(a, t, dev, "status");
  return t.data_ptr<int32_t>();
}

hsd_stream_t current_stream(const c10::Device& dev) {
  return reinterpret_cast<hsd_stream_t>(c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}

void arity(const char* fn, Py_ssize_t n, Py_ssize_t want) {
  if (n != want)
    refuse(PyExc_TypeError, "%s: %zd arguments, expected %zd", fn, n, want);
}

int32_t i32(const Args& a, int64_t v, const char* name) {
  if (v < INT32_MIN || v > INT32_MAX)
    refuse(PyExc_ValueError, "%s: %s=%lld is out of range", a.fn, name, static_cast<long long>(v));
  return static_cast<int32_t>(v);
}

// Whether rows [row0, row0 + n) lie within `rows` of them (row0, n >= 0: their sum may
// pass 64 bits).
bool fits(int64_t row0, int64_t n, int64_t rows) { return n <= rows && row0 <= rows - n; }

constexpr int64_t kMaxRow = int64_t(1) << 48;  // of planes known by address alone

// ---------------------------------------------------------------- rotary
// (q, k, v, positions, turns, pair_axis, axes, scaling, k_cache, v_cache,
//  dst_row0, out, num_q_heads, num_kv_heads, status)
PyObject* rope_append_axes(PyObject* const* args, Py_ssize_t n_args) {
  const Args a{args, "rope_append_axes"};
  arity(a.fn, n_args, 15);
  const Cache kc = cache_of(a, a.tensor(8, "k_cache"), "k_cache");
  const Cache vc = cache_of(a, a.tensor(9, "v_cache"), "v_cache");
  const int64_t hkv = a.none(13) ? kc.heads : a.integer(13);
  if (kc.heads != vc.heads || kc.rows != vc.rows || kc.row_stride != vc.row_stride ||
      kc.heads != hkv || hkv <= 0 || hkv > 4096)
    refuse(PyExc_ValueError, "%s: k_cache and v_cache must have one layout of %lld heads", a.fn,
           static_cast<long long>(hkv));
  const at::Tensor& kt = a.tensor(1, "k");
  const Rows k = rows_of(a, kt, "k", hkv * 128, false);
  const Rows v = rows_of(a, a.tensor(2, "v"), "v", hkv * 128, false);
  const int64_t n = k.rows;
  if (v.rows != n) refuse(PyExc_ValueError, "%s: k and v row counts differ", a.fn);
  const int64_t row0 = a.integer(10);
  if (row0 < 0 || !fits(row0, n, kc.rows))
    refuse(PyExc_ValueError, "%s: %lld rows from row %lld on pass the cache's %lld", a.fn,
           static_cast<long long>(n), static_cast<long long>(row0),
           static_cast<long long>(kc.rows));
  const int64_t axes = a.integer(6);
  at::Tensor pos = a.tensor(3, "positions");
  if (!pos.is_cuda() || (pos.scalar_type() != at::kLong && pos.scalar_type() != at::kInt))
    refuse(PyExc_TypeError, "%s: positions must be an int64 or int32 CUDA tensor", a.fn);
  int da = -2;  // the axes' dim
  bool ok = pos.dim() >= 1 && pos.size(-1) == n;
  if (pos.dim() == 1)
    ok = ok && axes == 1;
  else if (pos.dim() == 2)
    ok = ok && pos.size(0) == axes;
  else if (pos.dim() == 3 && pos.size(0) == 1)
    ok = ok && pos.size(1) == axes;
  else if (pos.dim() == 3) {
    ok = ok && pos.size(0) == axes && pos.size(1) == 1;
    da = -3;
  } else
    ok = false;
  if (!ok)
    refuse(PyExc_ValueError, "%s: positions %s, expected [%lld, %lld]", a.fn, shape(pos).c_str(),
           static_cast<long long>(axes), static_cast<long long>(n));
  if (pos.scalar_type() == at::kInt) pos = pos.to(at::kLong);
  Rows q{}, o{};
  int64_t hq = 0;
  const bool with_q = !a.none(0);
  if (with_q) {
    const at::Tensor& qt = a.tensor(0, "q");
    hq = a.none(12) ? (qt.dim() ? qt.size(-1) / 128 : 0) : a.integer(12);
    if (hq <= 0 || hq > 4096)
      refuse(PyExc_ValueError, "%s: %lld query heads", a.fn, static_cast<long long>(hq));
    q = rows_of(a, qt, "q", hq * 128, a.none(11));
    o = a.none(11) ? q : rows_of(a, a.tensor(11, "out"), "out", hq * 128, true);
    if (q.rows != n || o.rows != n)
      refuse(PyExc_ValueError, "%s: q, out and k row counts differ", a.fn);
  } else if (!a.none(11)) {
    refuse(PyExc_ValueError, "%s: out without q", a.fn);
  }
  const c10::Device dev = kt.device();
  const at::Tensor& turns = a.tensor(4, "turns");
  const at::Tensor& pair_axis = a.tensor(5, "pair_axis");
  same_device(a, v.keep, dev, "v");
  same_device(a, a.tensor(8, "k_cache"), dev, "k_cache");
  same_device(a, a.tensor(9, "v_cache"), dev, "v_cache");
  same_device(a, pos, dev, "positions");
  same_device(a, turns, dev, "the rotary tables");
  same_device(a, pair_axis, dev, "the rotary tables");
  if (with_q) {
    same_device(a, q.keep, dev, "q");
    same_device(a, o.keep, dev, "out");
  }
  if (turns.scalar_type() != at::kLong || turns.numel() != 64 || !turns.is_contiguous() ||
      pair_axis.scalar_type() != at::kInt || pair_axis.numel() != 64 || !pair_axis.is_contiguous())
    refuse(PyExc_ValueError, "%s: the rotary tables must be contiguous int64 and int32 [64]", a.fn);
  int32_t* status = status_of(a, 14, dev);
  if (n > 0) {
    const c10::cuda::CUDAGuard guard(dev);
    check(hsd_rope_append_axes(
              q.ptr, q.stride, o.ptr, o.stride, k.ptr, k.stride, v.ptr, v.stride,
              pos.data_ptr<int64_t>(), pos.dim() > 1 ? pos.stride(da) : 0, pos.stride(-1),
              i32(a, axes, "axes"), reinterpret_cast<const uint64_t*>(turns.data_ptr<int64_t>()),
              pair_axis.data_ptr<int32_t>(), static_cast<float>(a.real(7)), i32(a, n, "rows"),
              static_cast<int32_t>(hq), static_cast<int32_t>(hkv), 128, kc.ptr, kc.head_stride,
              vc.ptr, vc.head_stride, kc.row_stride, row0, status, current_stream(dev)),
          "hsd_rope_append_axes");
  }
  if (!with_q) Py_RETURN_NONE;
  return THPVariable_Wrap(
      o.keep.as_strided({1, hq, n, 128}, {hq * 128, 128, o.keep.stride(0), 1}));
}

// ---------------------------------------------------------------- 8-bit cache
struct Planes {
  const uint64_t* ptr;
  int32_t n;
  c10::Device dev;
};

Planes planes_of(const Args& a, int i, const at::Tensor& data, const at::Tensor& scale) {
  const at::Tensor& t = a.tensor(i, "planes");
  const int64_t n = data.size(0) * data.size(1) * data.size(2);
  if (t.scalar_type() != at::kLong || t.numel() != n || !t.is_contiguous())
    refuse(PyExc_ValueError, "%s: %lld plane addresses (int64) are needed", a.fn,
           static_cast<long long>(n));
  if (!data.is_cuda()) refuse(PyExc_TypeError, "%s: the cache must be on a CUDA device", a.fn);
  same_device(a, t, data.device(), "the planes' addresses");
  same_device(a, scale, data.device(), "the scales");
  return {reinterpret_cast<const uint64_t*>(t.data_ptr<int64_t>()), i32(a, n, "planes"),
          data.device()};
}

const at::Tensor& cache_data(const Args& a, int i) {
  const at::Tensor& t = a.tensor(i, "data");
  if (t.scalar_type() != at::kChar || t.dim() != 5 || !t.is_contiguous() || t.size(4) != 128)
    refuse(PyExc_ValueError, "%s: data must be contiguous int8 [L, 2, Hkv, rows, 128]", a.fn);
  return t;
}

const at::Tensor& cache_scale(const Args& a, int i, const at::Tensor& data) {
  const at::Tensor& t = a.tensor(i, "scale");
  if (t.scalar_type() != at::kFloat || t.dim() != 4 || !t.is_contiguous() ||
      t.size(0) != data.size(0) || t.size(1) != data.size(1) || t.size(2) != data.size(2) ||
      t.size(3) != data.size(3) / 64)
    refuse(PyExc_ValueError, "%s: scale must be contiguous float32 [L, 2, Hkv, rows / 64]", a.fn);
  return t;
}

// (planes, src_row0, data, scale, row0, n_rows, status)
PyObject* kv8_seal(PyObject* const* args, Py_ssize_t n_args) {
  const Args a{args, "seal"};
  arity(a.fn, n_args, 7);
  const at::Tensor& data = cache_data(a, 2);
  const at::Tensor& scale = cache_scale(a, 3, data);
  const int64_t src = a.integer(1), row0 = a.integer(4), n = a.integer(5);
  if (n < 0 || n % 64 || row0 < 0 || row0 % 64 || !fits(row0, n, data.size(3)) || src < 0 ||
      src > kMaxRow)
    refuse(PyExc_ValueError,
           "seal: %lld rows (a multiple of 64) from row %lld, after %lld of %lld sealed",
           static_cast<long long>(n), static_cast<long long>(src), static_cast<long long>(row0),
           static_cast<long long>(data.size(3)));
  const Planes p = planes_of(a, 0, data, scale);
  int32_t* status = status_of(a, 6, p.dev);
  const c10::cuda::CUDAGuard guard(p.dev);
  check(hsd_kv8_seal(p.ptr, p.n, src, data.data_ptr<int8_t>(), data.stride(2),
                     scale.data_ptr<float>(), scale.stride(2), i32(a, row0 / 64, "block"),
                     i32(a, n / 64, "blocks"), status, current_stream(p.dev)),
        "hsd_kv8_seal");
  Py_RETURN_NONE;
}

// (data, scale, sealed, planes, row0, n_rows, dst_row0)
PyObject* kv8_unseal(PyObject* const* args, Py_ssize_t n_args) {
  const Args a{args, "unseal"};
  arity(a.fn, n_args, 7);
  const at::Tensor& data = cache_data(a, 0);
  const at::Tensor& scale = cache_scale(a, 1, data);
  const int64_t sealed = a.integer(2), row0 = a.integer(4), n = a.integer(5), dst = a.integer(6);
  if (row0 < 0 || n < 0 || !fits(row0, n, sealed) || sealed > data.size(3) || dst < 0 ||
      dst > kMaxRow)
    refuse(PyExc_ValueError, "unseal: %lld rows from row %lld of %lld to %lld",
           static_cast<long long>(n), static_cast<long long>(row0),
           static_cast<long long>(sealed), static_cast<long long>(dst));
  const Planes p = planes_of(a, 3, data, scale);
  const c10::cuda::CUDAGuard guard(p.dev);
  check(hsd_kv8_unseal(data.data_ptr<int8_t>(), data.stride(2), scale.data_ptr<float>(),
                       scale.stride(2), p.n, row0, i32(a, n, "rows"), p.ptr, dst,
                       current_stream(p.dev)),
        "hsd_kv8_unseal");
  Py_RETURN_NONE;
}

// ---------------------------------------------------------------- attention
struct Heads {
  char* ptr = nullptr;
  int64_t heads = 0, rows = 0, row_stride = 0, head_stride = 0;
  at::Tensor keep;
};

// [1, H, S, 128] or [H, S, 128] bf16
Heads heads_of(const Args& a, const at::Tensor& t, const char* name) {
  const int64_t d = t.dim();
  if ((d != 3 && d != 4) || t.size(-1) != 128)
    refuse(PyExc_ValueError, "%s: expected [1, H, S, 128] or [H, S, 128], got %s", name,
           shape(t).c_str());
  if (d == 4 && t.size(0) != 1)
    refuse(PyExc_ValueError, "%s: batch must be 1 (packed verification)", name);
  if (t.scalar_type() != at::kBFloat16) refuse(PyExc_TypeError, "%s: bf16 required", name);
  Heads h;
  h.keep = t.stride(-1) == 1 ? t : t.contiguous();
  h.ptr = static_cast<char*>(h.keep.data_ptr());
  h.heads = t.size(-3);
  h.rows = t.size(-2);
  // the stride of a single row or head is never used
  h.row_stride = h.rows > 1 ? h.keep.stride(-2) : 128;
  h.head_stride = h.heads > 1 ? h.keep.stride(-3) : 128;
  return h;
}

// Scratch of a call.  Up to kKeptScratch (few rows: partial rows for one CTA per SM)
// it is kept per device and current stream.  More (many rows: a layer's expanded
// columns, 512 bytes per column and KV head) comes from the caching allocator and goes
// back to it with the call, so that it serves other tensors between calls and no stream
// holds the largest size ever seen; the next call on the stream runs after this one.  So
// does a call that is being captured into a graph, from the graph's pool: graphs that
// share no stream share no scratch either (replays of one graph never overlap).
constexpr int64_t kKeptScratch = 2 << 20;

at::Tensor workspace(int64_t need, const c10::Device& dev) {
  if (need > kKeptScratch ||
      c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None)
    return at::detail::empty_cuda({need + 256}, at::kByte, dev, std::nullopt);
  // never destroyed: tensors must not outlive the allocator at exit
  static auto* cached = new std::map<std::pair<int, void*>, at::Tensor>;
  at::Tensor& t = (*cached)[{dev.index(), c10::cuda::getCurrentCUDAStream(dev.index()).stream()}];
  if (!t.defined())
    t = at::detail::empty_cuda({kKeptScratch + 256}, at::kByte, dev, std::nullopt);
  return t;
}

// (q, (k8, v8, k_scale, v_scale) or None, sealed, k, v, plan address, plan status,
//  scale, tail_row0, out, lse, need_lse)
PyObject* verify_attention_kv8(PyObject* const* args, Py_ssize_t n_args) {
  const Args a{args, "verify_attention_kv8"};
  arity(a.fn, n_args, 12);
  const Heads q = heads_of(a, a.tensor(0, "query"), "query");
  const auto* plan = reinterpret_cast<const hsd_plan_t*>(a.integer(5));
  const at::Tensor& plan_status = a.tensor(6, "plan status");
  const c10::Device dev = q.keep.device();
  if (!plan || !dev.is_cuda() || plan_status.device() != dev)
    refuse(PyExc_ValueError, "query and plan must be on the same CUDA device");
  const int64_t q_len = q.rows, kv_len = plan->kv_len, hq = q.heads;
  if (plan->q_len != q_len)
    refuse(PyExc_ValueError, "plan is for %d rows, query has %lld", plan->q_len,
           static_cast<long long>(q_len));
  const int64_t sealed = a.integer(2), tail_row0 = a.integer(8);
  if (sealed < 0 || sealed % 64 || sealed > kv_len || tail_row0 < 0 || tail_row0 > sealed)
    refuse(PyExc_ValueError,
           "sealed=%lld must be a multiple of 64 in [0, %lld] and tail_row0=%lld in [0, sealed]",
           static_cast<long long>(sealed), static_cast<long long>(kv_len),
           static_cast<long long>(tail_row0));
  Heads k, v;
  int64_t hkv = -1;
  if (sealed < kv_len) {
    if (a.none(3) || a.none(4))
      refuse(PyExc_ValueError, "columns %lld..%lld need the bf16 tail",
             static_cast<long long>(sealed), static_cast<long long>(kv_len));
    k = heads_of(a, a.tensor(3, "key"), "key");
    v = heads_of(a, a.tensor(4, "value"), "value");
    hkv = k.heads;
    if (v.heads != hkv || std::min(k.rows, v.rows) < kv_len - tail_row0)
      refuse(PyExc_ValueError, "tail: key and value must be [Hkv, >= %lld, 128]",
             static_cast<long long>(kv_len - tail_row0));
    same_device(a, k.keep, dev, "key");
    same_device(a, v.keep, dev, "value");
  }
  const int8_t* p8[2] = {nullptr, nullptr};
  const float* ps[2] = {nullptr, nullptr};
  int64_t h8[2] = {0, 0}, hs = 0;
  if (sealed > 0) {
    if (!PyTuple_Check(args[1]) || PyTuple_GET_SIZE(args[1]) != 4)
      refuse(PyExc_ValueError, "sealed columns need the layer's tensors (Kv8Layer)");
    const Args l{&PyTuple_GET_ITEM(args[1], 0), a.fn};
    static const char* const names[4] = {"layer.k", "layer.v", "layer.k_scale", "layer.v_scale"};
    if (hkv < 0) {
      const at::Tensor& t = l.tensor(0, names[0]);
      hkv = t.dim() == 3 ? t.size(0) : 0;
    }
    for (int i = 0; i < 2; ++i) {
      const at::Tensor& t = l.tensor(i, names[i]);
      if (t.scalar_type() != at::kChar || t.dim() != 3 || t.size(0) != hkv || t.size(2) != 128 ||
          t.size(1) < sealed || t.stride(2) != 1 || (t.size(1) > 1 && t.stride(1) != 128))
        refuse(PyExc_ValueError, "%s: int8 [%lld, >= %lld, 128] with contiguous rows", names[i],
               static_cast<long long>(hkv), static_cast<long long>(sealed));
      same_device(a, t, dev, names[i]);
      p8[i] = t.data_ptr<int8_t>();
      h8[i] = hkv > 1 ? t.stride(0) : t.size(1) * 128;
      const at::Tensor& s = l.tensor(i + 2, names[i + 2]);
      if (s.scalar_type() != at::kFloat || s.dim() != 2 || s.size(0) != hkv ||
          s.size(1) < sealed / 64 || (s.size(1) > 1 && s.stride(1) != 1))
        refuse(PyExc_ValueError, "%s: float32 [%lld, >= %lld]", names[i + 2],
               static_cast<long long>(hkv), static_cast<long long>(sealed / 64));
      same_device(a, s, dev, names[i + 2]);
      ps[i] = s.data_ptr<float>();
      const int64_t stride = hkv > 1 ? s.stride(0) : sealed / 64;
      if (i == 1 && stride != hs)
        refuse(PyExc_ValueError, "layer: k_scale and v_scale must share a head stride");
      hs = stride;
    }
  }
  if (hkv <= 0 || hq <= 0 || hq % hkv)
    refuse(PyExc_ValueError, "%lld query heads over %lld KV heads", static_cast<long long>(hq),
           static_cast<long long>(hkv));
  const int need_lse = PyObject_IsTrue(args[11]);
  if (need_lse < 0) throw PythonError{};
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor out, lse;
  if (a.none(9)) {
    out = at::detail::empty_cuda({q_len, hq, 128}, at::kBFloat16, dev, std::nullopt);
  } else {
    out = a.tensor(9, "out");
    if (out.scalar_type() != at::kBFloat16 || out.dim() != 3 || out.size(0) != q_len ||
        out.size(1) != hq || out.size(2) != 128 || !out.is_contiguous() || out.device() != dev)
      refuse(PyExc_ValueError, "out must be contiguous bf16 [%lld, %lld, 128] on %s",
             static_cast<long long>(q_len), static_cast<long long>(hq), dev.str().c_str());
  }
  if (need_lse) {
    if (a.none(10)) {
      lse = at::detail::empty_cuda({hq, q_len}, at::kFloat, dev, std::nullopt);
    } else {
      lse = a.tensor(10, "lse");
      if (lse.scalar_type() != at::kFloat || lse.dim() != 2 || lse.size(0) != hq ||
          lse.size(1) != q_len || !lse.is_contiguous() || lse.device() != dev)
        refuse(PyExc_ValueError, "lse must be contiguous float32 [%lld, %lld] on %s",
               static_cast<long long>(hq), static_cast<long long>(q_len), dev.str().c_str());
    }
  }
  const double scale = a.none(7) ? 0.08838834764831845 : a.real(7);
  const int32_t ql = i32(a, q_len, "rows"), hq32 = i32(a, hq, "heads"),
                hkv32 = i32(a, hkv, "KV heads");
  const size_t need = hsd_kv8_attention_workspace_bytes(ql, plan->kv_len, hq32, hkv32);
  const at::Tensor ws = workspace(static_cast<int64_t>(need), dev);
  const uintptr_t base = (reinterpret_cast<uintptr_t>(ws.data_ptr()) + 255) & ~uintptr_t(255);
  check(hsd_verify_attention_kv8(
            q.ptr, q.row_stride, q.head_stride, p8[0], h8[0], p8[1], h8[1], ps[0], ps[1], hs,
            static_cast<int32_t>(sealed), k.ptr, k.row_stride, k.head_stride, v.ptr, v.row_stride,
            v.head_stride, static_cast<int32_t>(tail_row0), out.data_ptr(),
            need_lse ? lse.data_ptr<float>() : nullptr, ql, plan->kv_len, hq32, hkv32, 128,
            static_cast<float>(scale), plan, reinterpret_cast<void*>(base), need,
            plan_status.data_ptr<int32_t>(), current_stream(dev)),
        "hsd_verify_attention_kv8");
  PyObject* o = THPVariable_Wrap(out);
  PyObject* l = need_lse ? THPVariable_Wrap(lse) : Py_NewRef(Py_None);
  PyObject* r = o && l ? PyTuple_Pack(2, o, l) : nullptr;
  Py_XDECREF(o);
  Py_XDECREF(l);
  return r;
}

// torch.OutOfMemoryError, which programs catch to free memory and call again.
PyObject* out_of_memory() {
  static PyObject* cls = nullptr;
  if (!cls) {
    PyObject* m = PyImport_ImportModule("torch");
    if (m) {
      cls = PyObject_GetAttrString(m, "OutOfMemoryError");
      Py_DECREF(m);
    }
    if (!cls) {
      PyErr_Clear();
      return PyExc_RuntimeError;
    }
  }
  return cls;
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    return F(args, n);
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.what.c_str());
  } catch (const PythonError&) {
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(out_of_memory(), e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

#define HSD_METHOD(f)                                                                  \
  {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<f>)), METH_FASTCALL, \
   nullptr}
PyMethodDef kMethods[] = {HSD_METHOD(rope_append_axes), HSD_METHOD(kv8_seal),
                          HSD_METHOD(kv8_unseal), HSD_METHOD(verify_attention_kv8),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "hsd_b200._ops", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops(void) {
  PyObject* m = PyModule_Create(&kModule);
  if (m && PyModule_AddStringConstant(m, "built_for", HSD_BUILT_FOR)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
