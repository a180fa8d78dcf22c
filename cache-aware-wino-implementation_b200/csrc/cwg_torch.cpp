// cwg_torch.cpp -- torch tensors as arguments of libcwg's sequence layers and 8-bit
// product: the Python side's argument checks, compiled.
//
// A decoding step's kernel takes a few microseconds; reading type, device, sizes,
// strides and address of its eight tensors from Python took ten (measured: 9.7 us for
// the convolution's step, 15.4 us for the scan's).  Here they are read from the
// tensors directly.  The module calls the C ABI through the addresses that cwg.py
// gives it, so that there is one libcwg in the process, and returns its status; a
// tensor that does not fit raises ValueError, which names the argument.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdexcept>
#include <string>

#include "../../include/cwg.h"

namespace {

struct Entries {
  decltype(&cwg_conv1d_causal) conv1d_causal;
  decltype(&cwg_conv1d_causal_step) conv1d_causal_step;
  decltype(&cwg_ssm_scan) ssm_scan;
  decltype(&cwg_ssm_step) ssm_step;
  decltype(&cwg_fp8_quantize) fp8_quantize;
  decltype(&cwg_fp8_matmul) fp8_matmul;
} g;

[[noreturn]] void refuse(const char *name, const std::string &why) {
  throw std::invalid_argument(std::string(name) + " " + why);
}

std::string text(at::IntArrayRef v) {
  std::string s = "(";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + ")";
}

const at::Tensor &tensor(PyObject *o, const char *name) {
  if (o == Py_None) refuse(name, "is missing");
  if (!THPVariable_Check(o)) refuse(name, "is not a tensor");
  return THPVariable_Unpack(o);
}

// What all of a call's tensors have to agree on, taken from its first one.
struct Call {
  int device;
  void *stream = nullptr;
  at::ScalarType io;
  unsigned flags;

  Call(PyObject *first, const char *name, PyObject *flags_, PyObject *stream_) {
    const unsigned long f = PyLong_AsUnsignedLong(flags_);
    if (f == (unsigned long)-1 && PyErr_Occurred()) throw std::domain_error("");
    flags = (unsigned)f;
    io = flags & CWG_BF16 ? at::kBFloat16 : at::kFloat;
    if (first == Py_None || !THPVariable_Check(first) || THPVariable_Unpack(first).dim() != 2)
      refuse(name, "is not a matrix of [rows][columns]");
    const at::Tensor &t = THPVariable_Unpack(first);
    if (!t.is_cuda()) refuse(name, "is not on a CUDA device");
    device = t.get_device();
    if (device != c10::cuda::current_device())
      refuse(name, "is on cuda:" + std::to_string(device) + ", not on the current device");
    if (stream_ == Py_None) {  // the stream that torch's own operators would use
      stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    } else if (PyLong_Check(stream_)) {
      stream = PyLong_AsVoidPtr(stream_);
    } else {
      PyObject *h = PyObject_GetAttrString(stream_, "cuda_stream");
      PyObject *d = h ? PyObject_GetAttrString(stream_, "device_index") : nullptr;
      if (!d) {
        Py_XDECREF(h);
        throw std::domain_error("");
      }
      stream = PyLong_AsVoidPtr(h);
      const long at = PyLong_AsLong(d);
      Py_DECREF(h);
      Py_DECREF(d);
      if (at != device) refuse("the stream", "belongs to another device");
    }
    if (PyErr_Occurred()) throw std::domain_error("");
  }

  void common(const at::Tensor &t, const char *name, at::ScalarType type) const {
    if (t.scalar_type() != type)
      refuse(name, std::string("is ") + c10::toString(t.scalar_type()) + ", not " +
                       c10::toString(type));
    if (!t.is_cuda() || t.get_device() != device)
      refuse(name, "is not on the call's device cuda:" + std::to_string(device));
  }

  // A contiguous tensor of the given type and shape (-1: any size).
  void *dense(PyObject *o, const char *name, at::ScalarType type,
              std::initializer_list<int64_t> shape, bool optional = false) const {
    if (optional && o == Py_None) return nullptr;
    const at::Tensor &t = tensor(o, name);
    common(t, name, type);
    bool same = t.dim() == (int64_t)shape.size();
    size_t i = 0;
    for (const int64_t want : shape) {
      if (same && want >= 0 && t.size((int64_t)i) != want) same = false;
      ++i;
    }
    if (!same)
      refuse(name, "has shape " + text(t.sizes()) + ", not " +
                       text(at::IntArrayRef(shape.begin(), shape.size())));
    if (!t.is_contiguous()) refuse(name, "is not contiguous");
    return t.data_ptr();
  }

  // A [rows][cols] matrix whose rows are contiguous, and the distance between them.
  struct Rows {
    void *p;
    long long ld;
  };
  Rows rows(PyObject *o, const char *name, at::ScalarType type, int64_t rows,
            int64_t cols) const {
    const at::Tensor &t = tensor(o, name);
    common(t, name, type);
    if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols)
      refuse(name, "has shape " + text(t.sizes()) + ", not (" + std::to_string(rows) + ", " +
                       std::to_string(cols) + ")");
    if ((t.stride(1) != 1 && cols > 1) || (t.stride(0) < cols && rows > 1))
      refuse(name, "has strides " + text(t.strides()) + ": rows of " + std::to_string(cols) +
                       " neighbouring elements are needed");
    return {t.data_ptr(), rows > 1 ? (long long)t.stride(0) : (long long)cols};
  }
};

int count(int64_t v, const char *name) {
  if (v > 0x7fffffff) refuse(name, "is too large");
  return (int)v;
}

template <typename F>
PyObject *guarded(F &&f) {
  try {
    return PyLong_FromLong(f());
  } catch (const std::domain_error &) {  // the Python error is set
    return nullptr;
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_ValueError, e.what());
    return nullptr;
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    return nullptr;
  }
}

// The launch without the interpreter's lock: it may wait for room in the stream's queue.
template <typename F>
int unlocked(F &&f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS rc = f();
  Py_END_ALLOW_THREADS return rc;
}

#define NEED(N)                                                              \
  if (nargs != (N)) {                                                        \
    PyErr_Format(PyExc_TypeError, "%d arguments, not %zd", (N), nargs);      \
    return nullptr;                                                          \
  }

// (x, w, bias, y, state, starts, slots, resume, flags, stream)
PyObject *conv1d_causal(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
  NEED(10)
  return guarded([&] {
    const Call c(a[0], "x", a[8], a[9]);
    const at::Tensor &x = tensor(a[0], "x"), &w = tensor(a[1], "w"), &st = tensor(a[5], "starts");
    const int64_t tokens = x.size(0), ch = x.size(1);
    if (w.dim() != 2) refuse("w", "is not (channels, width)");
    if (st.dim() != 1 || st.size(0) < 1) refuse("starts", "is not (sequences + 1,)");
    const int64_t width = w.size(1), n = st.size(0) - 1;
    const auto xr = c.rows(a[0], "x", c.io, tokens, ch), yr = c.rows(a[3], "y", c.io, tokens, ch);
    const auto *wp = (const float *)c.dense(a[1], "w", at::kFloat, {ch, width});
    const auto *bp = (const float *)c.dense(a[2], "bias", at::kFloat, {ch}, true);
    void *sp = c.dense(a[4], "state", c.io, {-1, width - 1, ch}, true);
    const auto *starts = (const int *)c.dense(a[5], "starts", at::kInt, {n + 1});
    const auto *slots = (const int *)c.dense(a[6], "slots", at::kInt, {n}, true);
    const auto *resume = (const unsigned char *)c.dense(a[7], "resume", at::kByte, {n}, true);
    const int lines = a[4] == Py_None ? 0 : count(tensor(a[4], "state").size(0), "state");
    const int t = count(tokens, "x"), cc = count(ch, "x"), k = count(width, "w"),
              ns = count(n, "starts");
    return unlocked([&] {
      return g.conv1d_causal(xr.p, xr.ld, wp, bp, yr.p, yr.ld, sp, starts, slots, resume, t, ns,
                             lines, cc, k, c.flags, c.stream);
    });
  });
}

// (x, w, bias, y, state, slots, flags, stream)
PyObject *conv1d_causal_step(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
  NEED(8)
  return guarded([&] {
    const Call c(a[0], "x", a[6], a[7]);
    const at::Tensor &x = tensor(a[0], "x"), &w = tensor(a[1], "w");
    const int64_t n = x.size(0), ch = x.size(1);
    if (w.dim() != 2) refuse("w", "is not (channels, width)");
    const int64_t width = w.size(1);
    const auto xr = c.rows(a[0], "x", c.io, n, ch), yr = c.rows(a[3], "y", c.io, n, ch);
    const auto *wp = (const float *)c.dense(a[1], "w", at::kFloat, {ch, width});
    const auto *bp = (const float *)c.dense(a[2], "bias", at::kFloat, {ch}, true);
    void *sp = c.dense(a[4], "state", c.io, {-1, width - 1, ch});
    const auto *slots = (const int *)c.dense(a[5], "slots", at::kInt, {n}, true);
    const int lines = count(tensor(a[4], "state").size(0), "state");
    const int rows = count(n, "x"), cc = count(ch, "x"), k = count(width, "w");
    return unlocked([&] {
      return g.conv1d_causal_step(xr.p, xr.ld, wp, bp, yr.p, yr.ld, sp, slots, rows, lines, cc, k,
                                  c.flags, c.stream);
    });
  });
}

// a: u, dt, A, B, C, D, dt_bias, z, y, state; the rest differs between the two calls
void fill_ssm(const Call &c, PyObject *const *a, PyObject *slots, int64_t n, cwg_ssm &op) {
  const at::Tensor &u = tensor(a[0], "u"), &A = tensor(a[2], "A"), &B = tensor(a[3], "B");
  const int64_t rows = u.size(0), ch = u.size(1);
  if (A.dim() != 2 || A.size(1) < 1) refuse("A", "is not (channels, states)");
  const int64_t states = A.size(1);
  if (B.dim() != 2 || B.size(1) < states || B.size(1) % states)
    refuse("B", "is not (tokens, groups * states)");
  const int64_t cols = B.size(1);
  auto put = [&](int i, const char *name, int64_t width, auto &p, long long &ld) {
    const auto r = c.rows(a[i], name, c.io, rows, width);
    p = r.p;
    ld = r.ld;
  };
  put(0, "u", ch, op.u, op.ldu);
  put(1, "dt", ch, op.dt, op.lddt);
  op.A = (const float *)c.dense(a[2], "A", at::kFloat, {ch, states});
  put(3, "B", cols, op.B, op.ldb);
  put(4, "C", cols, op.C, op.ldc);
  op.D = (const float *)c.dense(a[5], "D", at::kFloat, {ch}, true);
  op.dt_bias = (const float *)c.dense(a[6], "dt_bias", at::kFloat, {ch}, true);
  if (a[7] != Py_None) put(7, "z", ch, op.z, op.ldz);
  put(8, "y", ch, op.y, op.ldy);
  op.state = (float *)c.dense(a[9], "state", at::kFloat, {-1, ch, states}, true);
  op.n_slots = a[9] == Py_None ? 0 : count(tensor(a[9], "state").size(0), "state");
  op.slots = (const int *)c.dense(slots, "slots", at::kInt, {n}, true);
  op.tokens = count(rows, "u");
  op.n_seq = count(n, "starts");
  op.channels = count(ch, "u");
  op.groups = count(cols / states, "B");
  op.states = count(states, "A");
  op.flags = c.flags;
}

// (u, dt, A, B, C, D, dt_bias, z, y, state, starts, slots, resume, workspace, flags, stream)
PyObject *ssm_scan(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
  NEED(16)
  return guarded([&] {
    const Call c(a[0], "u", a[14], a[15]);
    const at::Tensor &st = tensor(a[10], "starts");
    if (st.dim() != 1 || st.size(0) < 1) refuse("starts", "is not (sequences + 1,)");
    const int64_t n = st.size(0) - 1;
    cwg_ssm op = {};
    fill_ssm(c, a, a[11], n, op);
    op.starts = (const int *)c.dense(a[10], "starts", at::kInt, {n + 1});
    op.resume = (const unsigned char *)c.dense(a[12], "resume", at::kByte, {n}, true);
    void *ws = c.dense(a[13], "workspace", at::kByte, {-1}, true);
    const size_t size = a[13] == Py_None ? 0 : (size_t)tensor(a[13], "workspace").size(0);
    return unlocked([&] { return g.ssm_scan(&op, ws, size, c.stream); });
  });
}

// (u, dt, A, B, C, D, dt_bias, z, y, state, slots, flags, stream)
PyObject *ssm_step(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
  NEED(13)
  return guarded([&] {
    const Call c(a[0], "u", a[11], a[12]);
    tensor(a[9], "state");
    cwg_ssm op = {};
    fill_ssm(c, a, a[10], tensor(a[0], "u").size(0), op);
    return unlocked([&] { return g.ssm_step(&op, c.stream); });
  });
}

// (x, q, scale, block_rows, flags, stream)
PyObject *fp8_quantize(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
  NEED(6)
  return guarded([&] {
    const Call c(a[0], "x", a[4], a[5]);
    const at::Tensor &x = tensor(a[0], "x");
    const int64_t rows = x.size(0), cols = x.size(1);
    const long block = PyLong_AsLong(a[3]);
    if (PyErr_Occurred()) throw std::domain_error("");
    if (block != 1 && block != 128) refuse("block_rows", "is 1 or 128");
    const auto xr = c.rows(a[0], "x", c.io, rows, cols);
    const auto qr = c.rows(a[1], "q", at::kFloat8_e4m3fn, rows, cols);
    const auto sr =
        c.rows(a[2], "scale", at::kFloat, (rows + block - 1) / block, (cols + 127) / 128);
    const int r = count(rows, "x"), k = count(cols, "x");
    return unlocked([&] {
      return g.fp8_quantize(xr.p, xr.ld, qr.p, qr.ld, (float *)sr.p, sr.ld, r, k, (int)block,
                            c.flags, c.stream);
    });
  });
}

// (a, a_scale, w, w_scale, bias, y, flags, stream)
PyObject *fp8_matmul(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
  NEED(8)
  return guarded([&] {
    const Call c(a[0], "a", a[6], a[7]);
    const at::Tensor &x = tensor(a[0], "a"), &w = tensor(a[2], "w");
    if (w.dim() != 2) refuse("w", "is not (n, k)");
    const int64_t m = x.size(0), k = x.size(1), n = w.size(0), kb = (k + 127) / 128;
    const auto ar = c.rows(a[0], "a", at::kFloat8_e4m3fn, m, k);
    const auto as = c.rows(a[1], "a_scale", at::kFloat, m, kb);
    const auto wr = c.rows(a[2], "w", at::kFloat8_e4m3fn, n, k);
    const auto ws = c.rows(a[3], "w_scale", at::kFloat, (n + 127) / 128, kb);
    const auto *bias = (const float *)c.dense(a[4], "bias", at::kFloat, {n}, true);
    const auto yr = c.rows(a[5], "y", c.io, m, n);
    const int mm = count(m, "a"), nn = count(n, "w"), kk = count(k, "a");
    return unlocked([&] {
      return g.fp8_matmul(ar.p, ar.ld, (const float *)as.p, as.ld, wr.p, wr.ld,
                          (const float *)ws.p, ws.ld, bias, yr.p, yr.ld, mm, nn, kk, c.flags,
                          c.stream);
    });
  });
}

// (addresses of the six entries, in the order of Entries)
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
  NEED(6)
  void *p[6];
  for (int i = 0; i < 6; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  g.conv1d_causal = (decltype(g.conv1d_causal))p[0];
  g.conv1d_causal_step = (decltype(g.conv1d_causal_step))p[1];
  g.ssm_scan = (decltype(g.ssm_scan))p[2];
  g.ssm_step = (decltype(g.ssm_step))p[3];
  g.fp8_quantize = (decltype(g.fp8_quantize))p[4];
  g.fp8_matmul = (decltype(g.fp8_matmul))p[5];
  Py_RETURN_NONE;
}

#define FAST(NAME) {#NAME, (PyCFunction)(void (*)(void))NAME, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(conv1d_causal), FAST(conv1d_causal_step), FAST(ssm_scan),
                         FAST(ssm_step),      FAST(fp8_quantize),       FAST(fp8_matmul),
                         FAST(bind),          {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "cwg_torch", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_cwg_torch() { return PyModule_Create(&module); }
