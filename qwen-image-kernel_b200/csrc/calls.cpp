// calls.cpp -- the host side of the decoder operators as one native call each: argument
// checks, output and workspace allocation and the C entry point of libqik.so.
//
// A CPython module (qik._calls) over torch's C++ tensors.  Single-token steps call these
// operators in every layer on a few rows, where the GPU needs 3 to 8 us and the host is what
// takes the time: the same checks and three allocations written in Python with a ctypes call
// took 12 to 15 us a call.  libqik.so itself stays free of torch.
//
// Refusals are Python exceptions (ValueError, TypeError); a failing entry point raises
// qik._lib.QikError with qik_last_error().  No C++ exception leaves a function.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <stdarg.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <numeric>
#include <string>
#include <vector>

#include "qik.h"

namespace {

struct Refused {};  // a Python exception is set

[[noreturn]] void refuse(PyObject* type, const char* fmt, ...) {
  char msg[600];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  PyErr_SetString(type, msg);
  throw Refused();
}

std::string shape_of(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
std::string said(const at::Tensor& t) { return shape_of(t) + " " + c10::toString(t.scalar_type()) + " on " + t.device().str(); }

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "qik: %s must be a tensor, got %s", name, Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
int64_t integer(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);  // takes numpy's integers too, through __index__
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(PyExc_TypeError, "qik: %s must be an integer", name);
  }
  return v;
}
double number(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(PyExc_TypeError, "qik: %s must be a number", name);
  }
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Refused();
  return v != 0;
}

bool aligned(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }
bool is16(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}
PyObject* out(const at::Tensor& t) {
  PyObject* o = THPVariable_Wrap(t);
  if (!o) throw Refused();
  return o;
}

PyObject* qik_error = nullptr;
void check(int rc, const char* what) {
  if (rc == QIK_OK) return;
  if (!qik_error) {
    PyObject* m = PyImport_ImportModule("qik._lib");
    qik_error = m ? PyObject_GetAttrString(m, "QikError") : nullptr;
    Py_XDECREF(m);
    if (!qik_error) throw Refused();
  }
  refuse(qik_error, "%s failed (status %d): %s", what, rc, qik_last_error());
}
// The device's status word (qik._lib.status_word, which lives as long as the process).
int* status_of(int device) {
  static int* words[64];
  if (device < 0 || device >= 64) refuse(PyExc_ValueError, "qik: device %d is out of range", device);
  if (!words[device]) {
    // (a first call may come while a graph is captured; status_ptr then keeps clear of it)
    c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
    PyObject* m = PyImport_ImportModule("qik._lib");
    PyObject* p = m ? PyObject_CallMethod(m, "status_ptr", "i", device) : nullptr;
    Py_XDECREF(m);
    if (!p) throw Refused();
    words[device] = static_cast<int*>(PyLong_AsVoidPtr(p));
    Py_DECREF(p);
  }
  return words[device];
}
void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }

// ---------------------------------------------------------------- RMS norm
// t ([..., N]) with one row pitch: contiguous tensors and rows [M, N] of a pitch as they are, copied where
// the alignment is not 16 bytes and where there are more dims that are not contiguous.
at::Tensor rows_of(const at::Tensor& t, int64_t N, int64_t& pitch) {
  pitch = N;
  if (t.is_contiguous()) return aligned(t) ? t : t.clone(at::MemoryFormat::Contiguous);
  if (t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= N && t.stride(0) % 8 == 0 && aligned(t)) {
    pitch = t.stride(0);
    return t;
  }
  return t.contiguous();
}

// add_rms_norm(x, residual, weight, eps, scales): scales None: (norm, sum); "tensor" or "row":
// (codes, scale, sum)
PyObject* add_rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    if (n != 5) refuse(PyExc_TypeError, "qik: add_rms_norm takes 5 arguments");
    const at::Tensor& x = tensor(a[0], "x");
    const bool with_r = a[1] != Py_None;
    const at::Tensor& w0 = tensor(a[2], "weight");
    const float eps = static_cast<float>(number(a[3], "eps"));
    int mode = 0;  // 0: no codes, 1: one scale, 2: a scale for each row
    if (a[4] != Py_None) {
      const char* s = PyUnicode_Check(a[4]) ? PyUnicode_AsUTF8(a[4]) : nullptr;
      mode = s && !strcmp(s, "tensor") ? 1 : s && !strcmp(s, "row") ? 2 : 0;
      if (!mode) refuse(PyExc_ValueError, "qik: fused_add_rms_norm_e4m3: scales is 'tensor' or 'row'");
    }
    const char* who = mode ? "fused_add_rms_norm_e4m3" : "fused_add_rms_norm";
    if (!x.is_cuda()) refuse(PyExc_ValueError, "qik: %s: x must be a CUDA tensor (the kernels have no CPU path)", who);
    const at::ScalarType type = x.scalar_type();
    if (!is16(type)) refuse(PyExc_TypeError, "qik: %s: bf16 or fp16, got %s", who, c10::toString(type));
    if (x.dim() == 0) refuse(PyExc_ValueError, "qik: %s: x needs at least one dimension", who);
    const int64_t N = x.size(-1);
    if (N == 0 || N % 8 || N > 32768)
      refuse(PyExc_ValueError, "qik: %s: %lld columns (a multiple of 8, at most 32768)", who, (long long)N);
    if (w0.dim() != 1 || w0.size(0) != N || w0.device() != x.device())
      refuse(PyExc_ValueError, "qik: %s: weight is %s, expected (%lld,) on %s", who, said(w0).c_str(), (long long)N,
             x.device().str().c_str());
    const bool w_f32 = w0.scalar_type() == at::kFloat;
    if (!w_f32 && w0.scalar_type() != type)
      refuse(PyExc_TypeError, "qik: %s: weight must be %s or fp32, got %s", who, c10::toString(type), c10::toString(w0.scalar_type()));
    if (!(eps >= 0.0f)) refuse(PyExc_ValueError, "qik: %s: eps must not be negative", who);
    c10::cuda::OptionalCUDAGuard guard(x.device());
    const at::Tensor w = w0.is_contiguous() && aligned(w0) ? w0 : w0.clone(at::MemoryFormat::Contiguous);
    int64_t ldx = N, ldr = N;
    const at::Tensor xr = rows_of(x, N, ldx);
    at::Tensor r;
    if (with_r) {
      const at::Tensor& r0 = tensor(a[1], "residual");
      if (r0.sizes() != x.sizes() || r0.scalar_type() != type || r0.device() != x.device())
        refuse(PyExc_ValueError, "qik: %s: residual is %s, x %s", who, said(r0).c_str(), said(x).c_str());
      r = rows_of(r0, N, ldr);
    }
    const int64_t M = x.numel() / N;
    const int device = x.device().index();
    at::Tensor y = empty(x.sizes(), mode ? at::kFloat8_e4m3fn : type, x);
    at::Tensor h = with_r ? empty(x.sizes(), type, x) : x;
    const void* rp = with_r ? r.data_ptr() : nullptr;
    void* hp = with_r ? h.data_ptr() : nullptr;
    const int f16 = type == at::kHalf;
    at::Tensor s;
    if (mode == 0) {
      if (M)
        check(qik_add_rms_norm(xr.data_ptr(), ldx, rp, ldr, w.data_ptr(), w_f32, M, N, eps, f16, hp, y.data_ptr(),
                               stream_of(device)),
              "qik_add_rms_norm");
    } else {
      s = mode == 2 ? empty(x.sizes().slice(0, x.dim() - 1), at::kFloat, x) : empty({1}, at::kFloat, x);
      const size_t ws_bytes = mode == 2 || !M ? 0 : qik_add_rms_norm_workspace_bytes(M, N);
      at::Tensor ws;
      if (ws_bytes) ws = empty({static_cast<int64_t>(ws_bytes)}, at::kByte, x);
      if (M)
        check(qik_add_rms_norm_e4m3(xr.data_ptr(), ldx, rp, ldr, w.data_ptr(), w_f32, M, N, eps, f16, hp, y.data_ptr(),
                                    s.data_ptr<float>(), mode == 2, ws_bytes ? ws.data_ptr() : nullptr, stream_of(device)),
              "qik_add_rms_norm_e4m3");
      else
        s.fill_(1e-12f);
    }
    PyObject* t = PyTuple_New(mode ? 3 : 2);
    if (!t) throw Refused();
    PyTuple_SET_ITEM(t, 0, out(y));
    if (mode) PyTuple_SET_ITEM(t, 1, out(s));
    PyObject* sum = with_r ? out(h) : (Py_INCREF(a[0]), a[0]);
    PyTuple_SET_ITEM(t, mode ? 2 : 1, sum);
    return t;
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- pages
struct Pages {
  int64_t pages, heads, page, ks[3], vs[3];  // strides: page, head, token
};
Pages pages_of(const at::Tensor& k, const at::Tensor& v, int64_t D, const at::Tensor& like) {
  if (k.dim() != 4 || k.sizes() != v.sizes() || k.size(3) != D || k.scalar_type() != like.scalar_type() ||
      v.scalar_type() != like.scalar_type() || k.device() != like.device() || v.device() != like.device())
    refuse(PyExc_ValueError, "qik: pages are %s and %s: expected two [pages, heads, page, %lld] %s on %s", said(k).c_str(),
           said(v).c_str(), (long long)D, c10::toString(like.scalar_type()), like.device().str().c_str());
  Pages p = {k.size(0), k.size(1), k.size(2), {k.stride(0), k.stride(1), k.stride(2)}, {v.stride(0), v.stride(1), v.stride(2)}};
  if (p.pages == 0 || p.heads == 0 || p.page < 16 || p.page > 4096 || (p.page & (p.page - 1)))
    refuse(PyExc_ValueError, "qik: pages are %s: a page is a power of two of 16 to 4096 tokens", shape_of(k).c_str());
  if (k.stride(3) != 1 || v.stride(3) != 1 || ((p.ks[0] | p.ks[1] | p.ks[2] | p.vs[0] | p.vs[1] | p.vs[2]) & 7) || !aligned(k) ||
      !aligned(v))
    refuse(PyExc_ValueError, "qik: pages need a unit column stride, strides of 16 bytes and 16-byte alignment");
  return p;
}

// copy_pages(k_pages, v_pages, moves): moves a list or tuple of (from, to, tokens)
PyObject* copy_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    if (n != 3) refuse(PyExc_TypeError, "qik: copy_pages takes 3 arguments");
    const at::Tensor &k = tensor(a[0], "k_pages"), &v = tensor(a[1], "v_pages");
    if (!k.is_cuda()) refuse(PyExc_ValueError, "qik: k_pages must be a CUDA tensor (the kernels have no CPU path)");
    if (k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type() || k.device() != v.device() || (k.dim() != 4 && k.dim() != 5))
      refuse(PyExc_ValueError, "qik: pages are %s and %s: expected two [layers, pages, heads, page, D] of one type on one device",
             said(k).c_str(), said(v).c_str());
    if (!PyList_Check(a[2]) && !PyTuple_Check(a[2])) refuse(PyExc_TypeError, "qik: moves is a sequence of (from, to, tokens)");
    const Py_ssize_t count = PySequence_Fast_GET_SIZE(a[2]);
    PyObject** items = PySequence_Fast_ITEMS(a[2]);
    std::vector<int32_t> moves(3 * count);
    for (Py_ssize_t i = 0; i < count; ++i) {
      PyObject* m = items[i];
      if ((!PyTuple_Check(m) && !PyList_Check(m)) || PySequence_Fast_GET_SIZE(m) != 3)
        refuse(PyExc_ValueError, "qik: moves is a sequence of (from, to, tokens)");
      for (int j = 0; j < 3; ++j) {
        const int64_t x = integer(PySequence_Fast_GET_ITEM(m, j), "a move's page or token count");
        if (x < 0 || x > 0x7FFFFFFF) refuse(PyExc_ValueError, "qik: copy_pages: move %lld is outside the pool", (long long)i);
        moves[3 * i + j] = static_cast<int32_t>(x);
      }
    }
    const int64_t at = k.dim() - 4, size = k.element_size();  // where `pages` is
    qik_page_pools p;
    p.k = k.data_ptr(), p.v = v.data_ptr();
    p.layers = at ? k.size(0) : 1;
    p.pages = k.size(at), p.heads = k.size(at + 1), p.page = k.size(at + 2), p.token_bytes = k.size(at + 3) * size;
    const int64_t D = k.size(at + 3), H = p.heads;
    auto tokens_together = [&](const at::Tensor& t) { return t.stride(at + 3) == 1 && t.stride(at + 2) == D; };
    // [pages, page, heads, D] seen with its heads first: the first tokens of a page are one run of all heads
    auto heads_together = [&](const at::Tensor& t) { return t.stride(at + 3) == 1 && t.stride(at + 1) == D && t.stride(at + 2) == H * D; };
    const bool whole = !tokens_together(k) && heads_together(k) && heads_together(v);
    if (!whole && !(tokens_together(k) && tokens_together(v)))
      refuse(PyExc_ValueError, "qik: copy_pages: in a page the tokens of a head, or the heads of a token, must be contiguous, the same in both pools");
    if (whole) p.heads = 1, p.token_bytes *= H;
    p.k_layer_bytes = at ? k.stride(0) * size : 0, p.v_layer_bytes = at ? v.stride(0) * size : 0;
    p.k_page_bytes = k.stride(at) * size, p.v_page_bytes = v.stride(at) * size;
    p.k_head_bytes = k.stride(at + 1) * size, p.v_head_bytes = v.stride(at + 1) * size;
    c10::cuda::OptionalCUDAGuard guard(k.device());
    const int rc = qik_copy_pages(&p, moves.data(), count, stream_of(k.device().index()));
    if (rc == QIK_ERR_INVALID) refuse(PyExc_ValueError, "qik: %s", qik_last_error());
    check(rc, "qik_copy_pages");
    Py_RETURN_NONE;
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- rotary
// t as [T, H, D] with a unit column stride and 16-byte rows and heads (copied otherwise).
at::Tensor heads_of(const at::Tensor& t, const char* name, int64_t T, int64_t D, const at::Tensor& like) {
  if (t.dim() != 3 || t.size(0) != T || t.size(2) != D || t.scalar_type() != like.scalar_type() || t.device() != like.device())
    refuse(PyExc_ValueError, "qik: %s is %s: expected [%lld, heads, %lld] %s on %s", name, said(t).c_str(), (long long)T,
           (long long)D, c10::toString(like.scalar_type()), like.device().str().c_str());
  if (t.stride(2) != 1 || ((t.stride(0) | t.stride(1)) & 7) || !aligned(t)) return t.clone(at::MemoryFormat::Contiguous);
  return t;
}
at::Tensor index_of(const at::Tensor& t, const char* name, int64_t T, const at::Tensor& like) {
  if (t.dim() != 1 || t.size(0) != T || (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) || t.device() != like.device())
    refuse(PyExc_ValueError, "qik: %s is %s: expected [%lld] int32 or int64 on %s", name, said(t).c_str(), (long long)T,
           like.device().str().c_str());
  return t.contiguous();
}

// rotary(q, k, v, positions, cos, sin, slots, k_pages, v_pages, interleaved): (q, k) turned, or
// with slots q alone, k and v stored
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    if (n != 10) refuse(PyExc_TypeError, "qik: rotary takes 10 arguments");
    const at::Tensor& q0 = tensor(a[0], "q");
    if (!q0.is_cuda()) refuse(PyExc_ValueError, "qik: q must be a CUDA tensor (the kernels have no CPU path)");
    if (!is16(q0.scalar_type())) refuse(PyExc_TypeError, "qik: rotary: bf16 or fp16, got %s", c10::toString(q0.scalar_type()));
    if (q0.dim() != 3 || (q0.size(2) != 64 && q0.size(2) != 128 && q0.size(2) != 256))
      refuse(PyExc_ValueError, "qik: q is %s: expected [tokens, heads, 64, 128 or 256]", shape_of(q0).c_str());
    const int64_t T = q0.size(0), D = q0.size(2);
    const at::Tensor &cos = tensor(a[4], "cos"), &sin = tensor(a[5], "sin");
    if (cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat || cos.dim() != 2 || cos.sizes() != sin.sizes() ||
        cos.size(0) == 0 || !cos.is_contiguous() || !sin.is_contiguous() || cos.device() != q0.device() || sin.device() != q0.device() ||
        !aligned(cos) || !aligned(sin))
      refuse(PyExc_ValueError, "qik: table is (cos, sin), contiguous fp32 [positions, rotary_dim / 2] on q's device");
    const int64_t pairs = cos.size(1);
    if (pairs == 0 || pairs % 8 || 2 * pairs > D)
      refuse(PyExc_ValueError, "qik: a table for %lld columns does not fit heads of %lld (a multiple of 16)", (long long)(2 * pairs),
             (long long)D);
    c10::cuda::OptionalCUDAGuard guard(q0.device());
    const at::Tensor q = heads_of(q0, "q", T, D, q0), k = heads_of(tensor(a[1], "k"), "k", T, D, q0);
    const at::Tensor pos = index_of(tensor(a[3], "positions"), "positions", T, q0);
    const bool paged = a[6] != Py_None;
    qik_rotary_args r = {};
    at::Tensor v, slots, k_out;
    r.flags = (truth(a[9]) ? QIK_ROTARY_INTERLEAVED : 0) | (q.scalar_type() == at::kHalf ? QIK_ROTARY_F16 : 0) |
              (pos.scalar_type() == at::kLong ? QIK_ROTARY_POS64 : 0);
    if (paged) {
      v = heads_of(tensor(a[2], "v"), "v", T, D, q0);
      if (v.size(1) != k.size(1))
        refuse(PyExc_ValueError, "qik: v has %lld heads, k %lld", (long long)v.size(1), (long long)k.size(1));
      slots = index_of(tensor(a[6], "slots"), "slots", T, q0);
      const at::Tensor &kp = tensor(a[7], "k_pages"), &vp = tensor(a[8], "v_pages");
      const Pages p = pages_of(kp, vp, D, q0);
      if (p.heads != k.size(1))
        refuse(PyExc_ValueError, "qik: pages hold %lld heads, k has %lld", (long long)p.heads, (long long)k.size(1));
      r.v = v.data_ptr(), r.v_st = v.stride(0), r.v_sh = v.stride(1), r.slots = slots.data_ptr();
      r.k_out = kp.data_ptr(), r.v_out = vp.data_ptr(), r.page = p.page, r.pages = p.pages;
      r.kp_s0 = p.ks[0], r.kp_sh = p.ks[1], r.kp_ss = p.ks[2], r.vp_s0 = p.vs[0], r.vp_sh = p.vs[1], r.vp_ss = p.vs[2];
      r.flags |= QIK_ROTARY_PAGED | (slots.scalar_type() == at::kLong ? QIK_ROTARY_SLOT64 : 0);
    } else {
      k_out = empty(k.sizes(), k.scalar_type(), k);
      r.k_out = k_out.data_ptr();
    }
    at::Tensor q_out = empty(q.sizes(), q.scalar_type(), q);
    r.q = q.data_ptr(), r.k = k.data_ptr(), r.q_out = q_out.data_ptr(), r.positions = pos.data_ptr();
    r.cos = cos.data_ptr<float>(), r.sin = sin.data_ptr<float>();
    r.T = T, r.HQ = q.size(1), r.HK = k.size(1), r.D = D, r.rot = 2 * pairs, r.P = cos.size(0);
    r.q_st = q.stride(0), r.q_sh = q.stride(1), r.k_st = k.stride(0), r.k_sh = k.stride(1);
    const int device = q.device().index();
    if (T) check(qik_rotary(&r, status_of(device), stream_of(device)), "qik_rotary");
    if (paged) return out(q_out);
    PyObject* t = PyTuple_New(2);
    if (!t) throw Refused();
    PyTuple_SET_ITEM(t, 0, out(q_out));
    PyTuple_SET_ITEM(t, 1, out(k_out));
    return t;
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- attention
// Where a tensor's rows are, in bytes: its address, what it spans, a row's columns, the greatest common
// divisor of the other dims' strides (of those with more than one entry; 0: a single row), the largest
// of them and what one entry of its dim spans.
struct Rows {
  int64_t at, bytes, cols, step, outer, inner;
};
Rows rows_in_memory(const at::Tensor& t) {
  const int64_t e = t.element_size();
  const bool unit = t.stride(-1) == 1;
  Rows r = {reinterpret_cast<int64_t>(t.data_ptr()), 0, unit ? t.size(-1) * e : e, 0, 0, 0};
  if (t.numel() == 0) return r;
  r.bytes = r.cols;
  int64_t n = 0;
  for (int64_t i = 0; i < t.dim() - (unit ? 1 : 0); ++i) {
    if (t.size(i) < 2) continue;
    const int64_t s = t.stride(i) * e;
    r.bytes += (t.size(i) - 1) * s;
    r.step = std::gcd(r.step, s);
    if (s > r.outer) r.outer = s, n = t.size(i);
  }
  r.inner = r.bytes - (n ? (n - 1) * r.outer : 0);
  return r;
}
// Whether a and b share memory, unless it can be shown that they do not: their spans are apart, or
// all their rows lie at two places of one period that are apart (columns or heads next to each other
// in one allocation), or what they hold of each entry of a common outer stride is apart.
bool overlap(const Rows& a, const Rows& b) {
  if (a.bytes == 0 || b.bytes == 0 || a.at + a.bytes <= b.at || b.at + b.bytes <= a.at) return false;
  auto apart = [&](int64_t period, int64_t size_a, int64_t size_b) {
    if (period == 0) return false;
    const int64_t d = ((b.at - a.at) % period + period) % period;
    return d >= size_a && d + size_b <= period;
  };
  return !apart(std::gcd(a.step, b.step), a.cols, b.cols) && !(a.outer == b.outer && apart(a.outer, a.inner, b.inner));
}
// Whether two entries of t [T, H, D] may share memory.
bool overlaps_itself(const at::Tensor& t) {
  const int64_t T = t.size(0), H = t.size(1);
  int64_t n[2] = {T, H}, s[2] = {T > 1 ? t.stride(0) : 0, H > 1 ? t.stride(1) : 0};
  if (t.numel() == 0) return false;
  if (s[0] < s[1]) std::swap(n[0], n[1]), std::swap(s[0], s[1]);
  const int64_t span = t.size(2) + (n[1] - 1) * s[1];
  return (n[1] > 1 && s[1] < t.size(2)) || (n[0] > 1 && s[0] < span);
}

// paged_attention(q, k_pages, v_pages, page_table, seq_lens, query_starts, max_new, max_kv, sm_scale,
// causal, window, sinks, out)
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    if (n != 13) refuse(PyExc_TypeError, "qik: paged_attention takes 13 arguments");
    const at::Tensor& q0 = tensor(a[0], "q");
    if (!q0.is_cuda()) refuse(PyExc_ValueError, "qik: q must be a CUDA tensor (the kernels have no CPU path)");
    if (!is16(q0.scalar_type()))
      refuse(PyExc_TypeError, "qik: paged_attention: bf16 or fp16, got %s", c10::toString(q0.scalar_type()));
    if (q0.dim() != 3 || (q0.size(2) != 64 && q0.size(2) != 128))
      refuse(PyExc_ValueError, "qik: q is %s: expected [tokens, heads, 64 or 128]", shape_of(q0).c_str());
    const int64_t T = q0.size(0), HQ = q0.size(1), D = q0.size(2);
    const at::Tensor &kp = tensor(a[1], "k_pages"), &vp = tensor(a[2], "v_pages");
    const Pages p = pages_of(kp, vp, D, q0);
    if (HQ == 0 || HQ % p.heads)
      refuse(PyExc_ValueError, "qik: %lld query heads do not share %lld key heads evenly", (long long)HQ, (long long)p.heads);
    const at::Tensor &table0 = tensor(a[3], "page_table"), &lens0 = tensor(a[4], "seq_lens"), &starts0 = tensor(a[5], "query_starts");
    for (const at::Tensor* t : {&table0, &lens0, &starts0})
      if (t->scalar_type() != at::kInt || t->device() != q0.device())
        refuse(PyExc_ValueError, "qik: page_table, seq_lens and query_starts must be int32 on %s", q0.device().str().c_str());
    if (table0.dim() != 2 || lens0.dim() != 1 || starts0.dim() != 1 || table0.size(0) != lens0.size(0) ||
        starts0.size(0) != lens0.size(0) + 1)
      refuse(PyExc_ValueError, "qik: page_table %s, seq_lens %s and query_starts %s: expected [B, W], [B] and [B + 1]",
             shape_of(table0).c_str(), shape_of(lens0).c_str(), shape_of(starts0).c_str());
    qik_paged_attn_args r = {};
    r.B = lens0.size(0), r.T = T, r.HQ = HQ, r.HK = p.heads, r.D = D, r.W = table0.size(1), r.pages = p.pages, r.page = p.page;
    r.max_new = integer(a[6], "max_new");
    if (r.max_new < 0 || r.max_new > T)
      refuse(PyExc_ValueError, "qik: max_new is %lld, q has %lld tokens", (long long)r.max_new, (long long)T);
    r.max_kv = a[7] == Py_None ? r.W * r.page : integer(a[7], "max_kv");
    const bool causal = truth(a[9]);
    const int64_t window = integer(a[10], "window"), sinks = integer(a[11], "sinks");
    if (window < 0 || sinks < 0 || r.max_kv < 0 || (window && !causal))
      refuse(PyExc_ValueError, "qik: window %lld, sinks %lld, max_kv %lld, causal %d (a window needs causal)", (long long)window,
             (long long)sinks, (long long)r.max_kv, causal);
    // nothing is behind the 2^30 keys that a page table can hold
    constexpr int64_t kMost = (1ll << 30) - 1;
    r.window = static_cast<int>(window < kMost ? window : kMost), r.sinks = static_cast<int>(sinks < kMost ? sinks : kMost);
    const double scale = a[8] == Py_None ? 1.0 / std::sqrt(static_cast<double>(D)) : number(a[8], "sm_scale");
    if (!(scale > 0.0 && scale < 1e30)) refuse(PyExc_ValueError, "qik: sm_scale must be positive and finite, got %g", scale);
    r.sm_scale = static_cast<float>(scale);
    r.flags = (causal ? QIK_PAGED_CAUSAL : 0) | (q0.scalar_type() == at::kHalf ? QIK_PAGED_F16 : 0);
    c10::cuda::OptionalCUDAGuard guard(q0.device());
    const at::Tensor q = q0.stride(2) != 1 || q0.stride(0) <= 0 || q0.stride(1) <= 0 || ((q0.stride(0) | q0.stride(1)) & 7) || !aligned(q0) ? q0.clone(at::MemoryFormat::Contiguous) : q0;
    const bool given = a[12] != Py_None;
    const at::Tensor o = given ? tensor(a[12], "out") : empty(q.sizes(), q.scalar_type(), q);
    if (given) {
      if (o.sizes() != q.sizes() || o.scalar_type() != q.scalar_type() || o.device() != q.device())
        refuse(PyExc_ValueError, "qik: out is %s: expected %s", said(o).c_str(), said(q).c_str());
      if (o.stride(2) != 1 || ((o.stride(0) | o.stride(1)) & 7) || !aligned(o))
        refuse(PyExc_ValueError, "qik: out needs a unit column stride, strides of 16 bytes and 16-byte alignment");
      // a row's place is written while other CTAs still read rows
      const Rows mem = rows_in_memory(o);
      if (overlaps_itself(o) || overlap(mem, rows_in_memory(q0)) || overlap(mem, rows_in_memory(kp)) || overlap(mem, rows_in_memory(vp)))
        refuse(PyExc_ValueError, "qik: out overlaps itself, q or the pages");
    }
    const at::Tensor table = table0.stride(1) == 1 || r.W <= 1 ? table0 : table0.contiguous();
    const at::Tensor lens = lens0.contiguous(), starts = starts0.contiguous();
    r.q = q.data_ptr(), r.out = o.data_ptr(), r.k_pages = kp.data_ptr(), r.v_pages = vp.data_ptr();
    r.page_table = table.data_ptr<int>(), r.seq_lens = lens.data_ptr<int>(), r.query_starts = starts.data_ptr<int>();
    r.q_st = q.stride(0), r.q_sh = q.stride(1), r.o_st = o.stride(0), r.o_sh = o.stride(1), r.table_st = table.stride(0);
    r.kp_s0 = p.ks[0], r.kp_sh = p.ks[1], r.kp_ss = p.ks[2], r.vp_s0 = p.vs[0], r.vp_sh = p.vs[1], r.vp_ss = p.vs[2];
    const int device = q.device().index();
    // a workspace of this call alone: torch hands its memory on only to later work of the stream
    const size_t bytes = qik_paged_attention_workspace_bytes(&r);
    at::Tensor ws;
    if (bytes) ws = empty({static_cast<int64_t>(bytes)}, at::kByte, q);
    check(qik_paged_attention(&r, bytes ? ws.data_ptr() : nullptr, bytes, status_of(device), stream_of(device)),
          "qik_paged_attention");
    if (given) {
      Py_INCREF(a[12]);
      return a[12];
    }
    return out(o);
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}
PyMethodDef methods[] = {
    {"add_rms_norm", fast<add_rms_norm>(), METH_FASTCALL, nullptr},
    {"copy_pages", fast<copy_pages>(), METH_FASTCALL, nullptr},
    {"rotary", fast<rotary>(), METH_FASTCALL, nullptr},
    {"paged_attention", fast<paged_attention>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "Native calls of the decoder operators.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&module); }
