// Native front of the calls that a projection makes, quantize(), gemm() and the Q/K and Q/K/V
// projections, and of the attention step behind them (attention_ops.py): the argument checks, the output
// allocation and the launches of a plain call, without the interpreter.
//
// Each function takes a call only if it can see that the Python front (hip.py, attention_ops.py) would accept it
// and launch at once: plain CUDA tensors, contiguous (heads and caches: rows that the kernels read in place), of the
// right dtypes and shapes, no forced schedule.
// Anything else returns None, and the Python front handles the call and raises what it raises: no error
// is decided here.  The launches are the same C ABI calls, with the interpreter lock released.
//
// Measured on a [1, 256] activation: quantize 7.3 -> 4.6 us of host time, gemm 9.4 -> 4.4 us, of which
// the HIP launch takes about 3 each.  The projections' staged form, two launches, takes
// 18 to 20 us through Python and 8 to 10 us here; the fused one 10 to 13 and 5 to 6 us.  Calls of the
// attention step back to back, each with its kernel: rope of one token 9.5 and 4.7 us, paged_append of 64
// tokens 18 and 5.6, attention of 128 tokens 14.4 and 6.6, which is its kernel.
#include <Python.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <cfloat>
#include <cmath>
#include <mutex>
#include <unordered_map>

#include "m5k.h"

namespace {

PyObject* g_stream_of = nullptr;  // torch's raw stream handle of a device index
PyObject* g_splits = nullptr;     // hip._native_splits(mode, m, n, k, device index) -> K ranges, 0: not here
PyObject* g_staged = nullptr;     // hip._native_staged(mode, m, n, k, device index, aligned, grouped) -> 0 or 1

enum Mode { INT8, FP8, B16, H16 };

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return M5K_F32;
    case at::kHalf: return M5K_F16;
    case at::kBFloat16: return M5K_BF16;
    default: return -1;
  }
}

// A tensor whose storage a kernel may read as it is: exactly torch.Tensor (or Parameter), strided (plain():
// contiguous) on a GPU, and not a wrapper of a transform (vmap, forward or reverse mode of torch.func).
const at::Tensor* plain_strided(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  const c10::DispatchKeySet keys = t.key_set();
  if (!t.is_cuda() || t.layout() != at::kStrided ||
      keys.has_any(c10::DispatchKeySet({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                        c10::DispatchKey::Functionalize, c10::DispatchKey::Python,
                                        c10::DispatchKey::Conjugate, c10::DispatchKey::Negative})) ||
      !t.has_storage())
    return nullptr;
  return &t;
}

const at::Tensor* plain(PyObject* o) {
  const at::Tensor* t = plain_strided(o);
  return t && t->is_contiguous() ? t : nullptr;
}

bool vector_of(const at::Tensor* t, int64_t n, at::ScalarType st, c10::Device d) {
  return t && t->dim() == 1 && t->size(0) == n && t->scalar_type() == st && t->device() == d;
}

bool stream_of(c10::Device d, void** out) {
  PyObject* index = PyLong_FromLong(d.index());
  if (!index) return false;
  PyObject* r = PyObject_CallOneArg(g_stream_of, index);
  Py_DECREF(index);
  if (!r) return false;
  *out = reinterpret_cast<void*>(PyLong_AsUnsignedLongLong(r));
  Py_DECREF(r);
  return !PyErr_Occurred();
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType st, c10::Device d) {
  return at::empty(shape, at::TensorOptions().dtype(st).device(d));
}

PyObject* failed(const char* name, int rc) {
  PyErr_Format(PyExc_RuntimeError, "%s failed (%d): %s", name, rc, m5k_last_error());
  return nullptr;
}

// quantize(x, mode): codes and scales of mode "int8" or "fp8".
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 2 || !PyUnicode_Check(args[1])) Py_RETURN_NONE;
  const bool i8 = PyUnicode_CompareWithASCIIString(args[1], "int8") == 0;
  if (!i8 && PyUnicode_CompareWithASCIIString(args[1], "fp8") != 0) Py_RETURN_NONE;
  const at::Tensor* x = plain(args[0]);
  if (!x || x->dim() != 2 || x->size(0) == 0 || x->size(1) == 0) Py_RETURN_NONE;
  const int code = dtype_code(x->scalar_type());
  if (code < 0) Py_RETURN_NONE;
  void* stream = nullptr;
  if (!stream_of(x->device(), &stream)) return nullptr;
  const int64_t rows = x->size(0), k = x->size(1);
  at::Tensor q = empty({rows, k}, i8 ? at::kChar : at::kByte, x->device());
  at::Tensor s = empty({rows}, at::kFloat, x->device());
  const void* xp = x->data_ptr();
  void* qp = q.data_ptr();
  float* sp = static_cast<float*>(s.data_ptr());
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = m5k_quantize_rows(xp, code, rows, k, i8 ? M5K_QUANT_INT8 : M5K_QUANT_FP8, qp, sp, stream);
  Py_END_ALLOW_THREADS
  if (rc) return failed("m5k_quantize_rows", rc);
  PyObject* qo = THPVariable_Wrap(std::move(q));
  PyObject* so = THPVariable_Wrap(std::move(s));
  PyObject* r = qo && so ? PyTuple_Pack(2, qo, so) : nullptr;
  Py_XDECREF(qo);
  Py_XDECREF(so);
  return r;
  END_HANDLE_TH_ERRORS
}

// What hip.py's planner says of a shape, kept per shape and settings of the environment (bounded:
// emptied when full).  `what`: the mode, and for a projection's route bits 4 (a route), 5 (aligned
// operands) and 6 (grouped layout).
struct Key {
  int what, device, state;
  int64_t m, n, k;
  bool operator==(const Key& o) const {
    return what == o.what && device == o.device && state == o.state && m == o.m && n == o.n && k == o.k;
  }
};
struct Hash {
  size_t operator()(const Key& x) const {
    uint64_t h = 1469598103934665603ull;
    for (uint64_t v : {uint64_t(x.what), uint64_t(x.device), uint64_t(x.state), uint64_t(x.m), uint64_t(x.n), uint64_t(x.k)})
      h = (h ^ v) * 1099511628211ull, h ^= h >> 29;
    return h;
  }
};
std::mutex g_mutex;
std::unordered_map<Key, int, Hash> g_plans;

template <class Ask>
int planned(const Key& key, Ask ask) {  // -1: a Python error is set
  {
    std::lock_guard<std::mutex> lock(g_mutex);
    const auto it = g_plans.find(key);
    if (it != g_plans.end()) return it->second;
  }
  PyObject* r = ask();
  if (!r) return -1;
  const long v = PyLong_AsLong(r);
  Py_DECREF(r);
  if (PyErr_Occurred()) return -1;
  std::lock_guard<std::mutex> lock(g_mutex);
  if (g_plans.size() >= 4096) g_plans.clear();
  g_plans[key] = static_cast<int>(v);
  return static_cast<int>(v);
}

// K ranges of an aligned INT8 or FP8 product.
int planned_splits(const Key& key, PyObject* mode) {
  return planned(key, [&] {
    return PyObject_CallFunction(g_splits, "OLLLi", mode, (long long)key.m, (long long)key.n, (long long)key.k, key.device);
  });
}

// Whether a projection runs as the GEMM and a postprocess.
int planned_staged(const Key& key, PyObject* mode, bool aligned, bool grouped) {
  return planned(key, [&] {
    return PyObject_CallFunction(g_staged, "OLLLiii", mode, (long long)key.m, (long long)key.n, (long long)key.k,
                                 key.device, int(aligned), int(grouped));
  });
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// gemm(a, b, mode, a_scales, b_scales, output_dtype, bias, bias_row_map, residual, gate, gate_row_map).
PyObject* gemm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 11 || !PyUnicode_Check(args[2])) Py_RETURN_NONE;
  PyObject* mo = args[2];
  const int mode = PyUnicode_CompareWithASCIIString(mo, "int8") == 0   ? INT8
                   : PyUnicode_CompareWithASCIIString(mo, "bf16") == 0 ? B16
                   : PyUnicode_CompareWithASCIIString(mo, "fp8") == 0  ? FP8
                   : PyUnicode_CompareWithASCIIString(mo, "fp16") == 0 ? H16
                                                                       : -1;
  if (mode < 0) Py_RETURN_NONE;
  const bool quant = mode == INT8 || mode == FP8;
  static const at::ScalarType operand[] = {at::kChar, at::kByte, at::kBFloat16, at::kHalf};
  const at::Tensor *a = plain(args[0]), *b = plain(args[1]);
  if (!a || !b || a->dim() != 2 || b->dim() != 2 || a->scalar_type() != operand[mode] ||
      b->scalar_type() != operand[mode] || a->device() != b->device())
    Py_RETURN_NONE;
  const c10::Device dev = a->device();
  const int64_t m = a->size(0), k = a->size(1), n = b->size(0);
  if (b->size(1) != k || m == 0 || n == 0 || k == 0 || (mode == FP8 && k % 128) || (mode == INT8 && k > 133144))
    Py_RETURN_NONE;
  const float *sa = nullptr, *sb = nullptr;
  if (quant) {
    const at::Tensor *ta = plain(args[3]), *tb = plain(args[4]);
    if (!vector_of(ta, m, at::kFloat, dev) || !vector_of(tb, n, at::kFloat, dev)) Py_RETURN_NONE;
    sa = static_cast<const float*>(ta->data_ptr());
    sb = static_cast<const float*>(tb->data_ptr());
  } else if (args[3] != Py_None || args[4] != Py_None) {
    Py_RETURN_NONE;
  }
  at::ScalarType out = at::kFloat;
  if (args[5] != Py_None) {
    if (!THPDtype_Check(args[5])) Py_RETURN_NONE;
    out = reinterpret_cast<THPDtype*>(args[5])->scalar_type;
  }
  const int out_code = dtype_code(out);
  if (out_code < 0) Py_RETURN_NONE;
  // A table (bias or gate): [n], or [P, n] with an int32 map of the m rows.
  auto table = [&](PyObject* to, PyObject* ro, at::ScalarType st, const void** tp, const int32_t** rp) {
    const at::Tensor* t = plain(to);
    if (!t || t->scalar_type() != st || t->device() != dev) return false;
    if (ro == Py_None) {
      if (t->dim() != 1 || t->size(0) != n) return false;
    } else {
      const at::Tensor* r = plain(ro);
      if (t->dim() != 2 || t->size(0) == 0 || t->size(1) != n || !vector_of(r, m, at::kInt, dev)) return false;
      *rp = static_cast<const int32_t*>(r->data_ptr());
    }
    *tp = t->data_ptr();
    return true;
  };
  const void *bias = nullptr, *residual = nullptr, *gate = nullptr;
  const int32_t *bias_map = nullptr, *gate_map = nullptr;
  if (args[6] != Py_None || args[7] != Py_None) {
    if (mode != INT8 || args[6] == Py_None || args[8] != Py_None || args[9] != Py_None || args[10] != Py_None ||
        !table(args[6], args[7], at::kFloat, &bias, &bias_map))
      Py_RETURN_NONE;
  } else if (args[8] != Py_None || args[9] != Py_None || args[10] != Py_None) {
    const at::Tensor* r = plain(args[8]);
    if ((mode != INT8 && mode != B16) || args[5] == Py_None || out != at::kBFloat16 || !r || r->dim() != 2 ||
        r->size(0) != m || r->size(1) != n || r->scalar_type() != at::kBFloat16 || r->device() != dev ||
        !table(args[9], args[10], at::kBFloat16, &gate, &gate_map))
      Py_RETURN_NONE;
    residual = r->data_ptr();
  }
  const int state = m5k_gemm_schedule_state();
  if (state & 0xF) Py_RETURN_NONE;  // a schedule is forced
  const void *ap = a->data_ptr(), *bp = b->data_ptr();
  int splits = 1;
  if (quant && k % 16 == 0 && aligned16(ap) && aligned16(bp)) {
    splits = planned_splits(Key{mode, dev.index(), state, m, n, k}, mo);
    if (splits < 0) return nullptr;
    if (splits == 0) Py_RETURN_NONE;
  }
  void* stream = nullptr;
  if (!stream_of(dev, &stream)) return nullptr;
  at::Tensor c = empty({m, n}, out, dev), workspace;
  if (splits > 1) workspace = empty({splits, m, n}, mode == INT8 ? at::kInt : at::kFloat, dev);
  void* cp = c.data_ptr();
  void* wp = splits > 1 ? workspace.data_ptr() : nullptr;
  const int64_t elems = splits * m * n;
  const char* name = nullptr;
  int rc = 0;
  auto* ai = static_cast<const int8_t*>(ap);
  auto* bi = static_cast<const int8_t*>(bp);
  auto* au = static_cast<const uint8_t*>(ap);
  auto* bu = static_cast<const uint8_t*>(bp);
  auto* fbias = static_cast<const float*>(bias);
  Py_BEGIN_ALLOW_THREADS
  if (mode == INT8 && splits > 1) {
    name = "m5k_gemm_i8_splitk";
    rc = m5k_gemm_i8_splitk(ai, bi, m, n, k, sa, sb, cp, out_code, fbias, bias_map, residual, gate, gate_map, splits,
                            static_cast<int32_t*>(wp), elems, stream);
  } else if (mode == INT8) {
    name = "m5k_gemm_i8";
    rc = m5k_gemm_i8(ai, bi, m, n, k, sa, sb, cp, out_code, fbias, bias_map, residual, gate, gate_map, stream);
  } else if (mode == FP8 && splits > 1) {
    name = "m5k_gemm_f8_splitk";
    rc = m5k_gemm_f8_splitk(au, bu, m, n, k, sa, sb, cp, out_code, splits, static_cast<float*>(wp), elems, stream);
  } else if (mode == FP8) {
    name = "m5k_gemm_f8";
    rc = m5k_gemm_f8(au, bu, m, n, k, sa, sb, cp, out_code, stream);
  } else {
    name = "m5k_gemm_float";
    rc = m5k_gemm_float(ap, bp, mode == B16 ? M5K_BF16 : M5K_F16, m, n, k, cp, out_code, residual, gate, gate_map, stream);
  }
  Py_END_ALLOW_THREADS
  if (rc) return failed(name, rc);
  return THPVariable_Wrap(std::move(c));
  END_HANDLE_TH_ERRORS
}

// The Q/K projection (args: a, b, gamma, cos, sin, mode, a_scales, b_scales, epsilon) and the grouped
// Q/K/V one (a, w, q_gamma, k_gamma, cos, sin, mode, a_scales, w_scales, epsilon), by the route that
// hip.projection_staged names.
constexpr int64_t HEAD = 128;

PyObject* project(PyObject* const* args, bool grouped) {
  const int at = grouped ? 4 : 3;  // index of cos
  PyObject* mo = args[at + 2];
  if (!PyUnicode_Check(mo)) Py_RETURN_NONE;
  const bool i8 = PyUnicode_CompareWithASCIIString(mo, "int8") == 0;
  if (!i8 && PyUnicode_CompareWithASCIIString(mo, "bf16") != 0) Py_RETURN_NONE;
  const at::Tensor *a = plain(args[0]), *b = plain(args[1]);
  const at::ScalarType operand = i8 ? at::kChar : at::kBFloat16;
  if (!a || !b || a->dim() != 2 || b->dim() != 2 || a->scalar_type() != operand || b->scalar_type() != operand ||
      a->device() != b->device())
    Py_RETURN_NONE;
  const c10::Device dev = a->device();
  const int64_t m = a->size(0), k = a->size(1), n = b->size(0), block = grouped ? 3 * HEAD : HEAD;
  if (b->size(1) != k || m == 0 || n == 0 || k == 0 || n % block || (i8 && k > 131071)) Py_RETURN_NONE;
  const float *sa = nullptr, *sb = nullptr;
  if (i8) {
    const at::Tensor *ta = plain(args[at + 3]), *tb = plain(args[at + 4]);
    if (!vector_of(ta, m, at::kFloat, dev) || !vector_of(tb, n, at::kFloat, dev)) Py_RETURN_NONE;
    sa = static_cast<const float*>(ta->data_ptr());
    sb = static_cast<const float*>(tb->data_ptr());
  } else if (args[at + 3] != Py_None || args[at + 4] != Py_None) {
    Py_RETURN_NONE;
  }
  const at::Tensor *g = plain(args[2]), *gk = grouped ? plain(args[3]) : g;
  const at::Tensor *cos = plain(args[at]), *sin = plain(args[at + 1]);
  if (!vector_of(g, HEAD, at::kBFloat16, dev) || !vector_of(gk, HEAD, at::kBFloat16, dev) || !aligned16(g->data_ptr()) ||
      !aligned16(gk->data_ptr()))
    Py_RETURN_NONE;
  for (const at::Tensor* t : {cos, sin})
    if (!t || t->dim() != 2 || t->size(0) != m || t->scalar_type() != at::kBFloat16 || t->device() != dev) Py_RETURN_NONE;
  const int64_t half = cos->size(1);
  if (half < 1 || half > HEAD / 2 || sin->size(1) != half) Py_RETURN_NONE;
  if (!PyFloat_CheckExact(args[at + 5])) Py_RETURN_NONE;
  const float eps = static_cast<float>(PyFloat_AS_DOUBLE(args[at + 5]));
  if (!(eps > 0.0f) || !std::isfinite(eps)) Py_RETURN_NONE;
  const int state = m5k_gemm_schedule_state();
  if (state & 0xF) Py_RETURN_NONE;  // a schedule is forced
  const void *ap = a->data_ptr(), *bp = b->data_ptr();
  const int64_t row = k * (i8 ? 1 : 2);
  const bool whole = row % 16 == 0 && aligned16(ap) && aligned16(bp), aligned = whole && row <= int64_t(1) << 23;
  const int mode = i8 ? INT8 : B16;
  const int staged = planned_staged(Key{mode | 16 | (aligned ? 32 : 0) | (grouped ? 64 : 0), dev.index(), state, m, n, k},
                                    mo, aligned, grouped);
  if (staged < 0) return nullptr;
  int splits = 1;
  if (staged && i8 && whole) {
    splits = planned_splits(Key{mode, dev.index(), state, m, n, k}, mo);
    if (splits < 0) return nullptr;
    if (splits == 0) Py_RETURN_NONE;
  }
  void* stream = nullptr;
  if (!stream_of(dev, &stream)) return nullptr;
  const int64_t heads = n / block;
  at::Tensor y[3], projected, workspace;
  for (int i = 0; i < (grouped ? 3 : 1); ++i) y[i] = empty({heads, m, HEAD}, at::kBFloat16, dev);
  if (staged) projected = empty({m, n}, at::kBFloat16, dev);
  if (splits > 1) workspace = empty({splits, m, n}, at::kInt, dev);
  void* yp[3] = {y[0].data_ptr(), grouped ? y[1].data_ptr() : nullptr, grouped ? y[2].data_ptr() : nullptr};
  void* pp = staged ? projected.data_ptr() : nullptr;
  auto* wp = splits > 1 ? static_cast<int32_t*>(workspace.data_ptr()) : nullptr;
  const void *gp = g->data_ptr(), *gkp = gk->data_ptr(), *cp = cos->data_ptr(), *sp = sin->data_ptr();
  auto* ai = static_cast<const int8_t*>(ap);
  auto* bi = static_cast<const int8_t*>(bp);
  const int r = static_cast<int>(half), dtype = i8 ? M5K_I8 : M5K_BF16;
  const char* name = nullptr;
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  if (staged) {
    if (splits > 1) {
      name = "m5k_gemm_i8_splitk";
      rc = m5k_gemm_i8_splitk(ai, bi, m, n, k, sa, sb, pp, M5K_BF16, nullptr, nullptr, nullptr, nullptr, nullptr, splits,
                              wp, splits * m * n, stream);
    } else if (i8) {
      name = "m5k_gemm_i8";
      rc = m5k_gemm_i8(ai, bi, m, n, k, sa, sb, pp, M5K_BF16, nullptr, nullptr, nullptr, nullptr, nullptr, stream);
    } else {
      name = "m5k_gemm_float";
      rc = m5k_gemm_float(ap, bp, M5K_BF16, m, n, k, pp, M5K_BF16, nullptr, nullptr, nullptr, stream);
    }
    if (rc == 0 && grouped) {
      name = "m5k_qkv_norm_rope";
      rc = m5k_qkv_norm_rope(pp, m, heads, gp, gkp, cp, sp, r, eps, yp[0], yp[1], yp[2], stream);
    } else if (rc == 0) {
      name = "m5k_qk_norm_rope";
      rc = m5k_qk_norm_rope(pp, m, n, gp, cp, sp, r, eps, yp[0], stream);
    }
  } else if (grouped) {
    name = "m5k_projection_qkv_rope";
    rc = m5k_projection_qkv_rope(ap, bp, dtype, m, heads, k, sa, sb, gp, gkp, cp, sp, r, eps, yp[0], yp[1], yp[2], stream);
  } else {
    name = "m5k_projection_qk_rope";
    rc = m5k_projection_qk_rope(ap, bp, dtype, m, n, k, sa, sb, gp, cp, sp, r, eps, yp[0], stream);
  }
  Py_END_ALLOW_THREADS
  if (rc) return failed(name, rc);
  if (!grouped) return THPVariable_Wrap(std::move(y[0]));
  PyObject* out = PyTuple_New(3);
  for (int i = 0; out && i < 3; ++i) {
    PyObject* o = THPVariable_Wrap(std::move(y[i]));
    if (!o) {
      Py_CLEAR(out);
      break;
    }
    PyTuple_SET_ITEM(out, i, o);
  }
  return out;
}

PyObject* qk(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 9) Py_RETURN_NONE;
  return project(args, false);
  END_HANDLE_TH_ERRORS
}

PyObject* qkv(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 10) Py_RETURN_NONE;
  return project(args, true);
  END_HANDLE_TH_ERRORS
}

// ---- the attention step ---------------------------------------------------------------------------

// Stride in elements, 0 along an axis of one entry.
int64_t stride(const at::Tensor& t, int d) { return t.size(d) == 1 ? 0 : t.stride(d); }

// Whether the rows (last axis) of a tensor begin at multiples of 16 bytes and are contiguous.
bool rows16(const at::Tensor& t) {
  const int last = static_cast<int>(t.dim()) - 1;
  if (t.size(last) > 1 && t.stride(last) != 1) return false;
  const int64_t unit = 16 / static_cast<int64_t>(t.element_size());
  for (int d = 0; d < last; ++d)
    if (stride(t, d) % unit) return false;
  return aligned16(t.data_ptr());
}

// The launches go to the current device.
bool current(c10::Device d) { return c10::impl::VirtualGuardImpl(d.type()).getDevice().index() == d.index(); }

// A positive finite float as attention_ops.py takes it, `absent` for None; false: let Python look at it.
bool positive(PyObject* o, float absent, float& out) {
  if (o == Py_None) {
    out = absent;
    return true;
  }
  if (!PyFloat_CheckExact(o)) return false;
  const double v = PyFloat_AS_DOUBLE(o);
  out = static_cast<float>(v);
  return v > 0.0 && v < 1e30 && out > 0.0f;
}

// A positive int below 2^30, 0 for None.
bool window_of(PyObject* o, int64_t& out) {
  out = 0;
  if (o == Py_None) return true;
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  out = PyLong_AsLongLongAndOverflow(o, &overflow);
  return !overflow && out > 0 && out < (int64_t{1} << 30);
}

// An int32 (or other) vector of n entries, null for None; false: let Python look at it.
template <class T>
bool optional_vector(PyObject* o, int64_t n, at::ScalarType st, c10::Device d, const T** out) {
  *out = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = plain(o);
  if (!vector_of(t, n, st, d)) return false;
  *out = static_cast<const T*>(t->data_ptr());
  return true;
}

// layout "half" 0, "interleaved" 1, anything else -1.
int layout_of(PyObject* o) {
  if (!PyUnicode_Check(o)) return -1;
  if (PyUnicode_CompareWithASCIIString(o, "half") == 0) return 0;
  return PyUnicode_CompareWithASCIIString(o, "interleaved") == 0 ? 1 : -1;
}

const at::Tensor* frequencies_of(PyObject* o, int64_t width, c10::Device d) {
  const at::Tensor* f = plain(o);
  return f && f->dim() == 1 && f->scalar_type() == at::kDouble && f->device() == d && f->size(0) >= 1 &&
                 2 * f->size(0) <= width
             ? f
             : nullptr;
}

// [heads, tokens, width] of a float type with contiguous channels.
const at::Tensor* heads_of(PyObject* o) {
  const at::Tensor* t = plain_strided(o);
  return t && t->dim() == 3 && t->size(0) > 0 && t->size(1) > 0 && t->size(2) > 0 &&
                 dtype_code(t->scalar_type()) >= 0 && (t->size(2) == 1 || t->stride(2) == 1)
             ? t
             : nullptr;
}

bool half_type(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

// rope(x, positions, frequencies, layout, magnitude).
PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor* x = nargs == 5 ? heads_of(args[0]) : nullptr;
  const int layout = nargs == 5 ? layout_of(args[3]) : -1;
  float magnitude;
  if (!x || layout < 0 || !current(x->device()) || args[4] == Py_None || !positive(args[4], 1.0f, magnitude))
    Py_RETURN_NONE;
  const c10::Device dev = x->device();
  const int64_t heads = x->size(0), tokens = x->size(1), width = x->size(2);
  const at::Tensor *p = plain(args[1]), *f = frequencies_of(args[2], width, dev);
  if (!f || !vector_of(p, tokens, at::kInt, dev)) Py_RETURN_NONE;
  void* stream = nullptr;
  if (!stream_of(dev, &stream)) return nullptr;
  at::Tensor y = empty({heads, tokens, width}, x->scalar_type(), dev);
  const void* xp = x->data_ptr();
  const auto* pp = static_cast<const int32_t*>(p->data_ptr());
  const auto* fp = static_cast<const double*>(f->data_ptr());
  void* yp = y.data_ptr();
  const int64_t sh = stride(*x, 0), st = stride(*x, 1), pairs = f->size(0);
  const int code = dtype_code(x->scalar_type());
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = m5k_rope(xp, code, tokens, heads, width, sh, st, pp, fp, pairs, layout, magnitude, yp, stream);
  Py_END_ALLOW_THREADS
  if (rc) return failed("m5k_rope", rc);
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// A paged cache and the vectors that describe its sequences.
struct Paged {
  const at::Tensor *k, *v;
  const int32_t *table, *starts, *context;
  int64_t sequences, width, pages, kv_heads, page_size, dim;
};

// Takes args k_cache, v_cache, page_table, query_starts, context_lengths.
bool paged_of(PyObject* const* args, Paged& out) {
  const at::Tensor *k = plain_strided(args[0]), *v = plain_strided(args[1]), *t = plain(args[2]);
  if (!k || !v || !t || k->dim() != 4 || v->sizes() != k->sizes() || v->scalar_type() != k->scalar_type() ||
      v->device() != k->device() || k->numel() == 0 || k->stride(3) != 1 || v->stride(3) != 1)
    return false;
  const c10::Device dev = k->device();
  if (t->dim() != 2 || t->scalar_type() != at::kInt || t->device() != dev || t->numel() == 0) return false;
  out = Paged{k, v, static_cast<const int32_t*>(t->data_ptr()), nullptr, nullptr, t->size(0), t->size(1),
              k->size(0), k->size(1), k->size(2), k->size(3)};
  return out.page_size <= (1 << 20) && out.width * out.page_size <= (1 << 30) && args[3] != Py_None &&
         args[4] != Py_None && optional_vector(args[3], out.sequences + 1, at::kInt, dev, &out.starts) &&
         optional_vector(args[4], out.sequences, at::kInt, dev, &out.context);
}

bool expanded(const at::Tensor& t) {
  for (int d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1 && t.stride(d) == 0) return true;
  return false;
}

// paged_append(k, v, k_cache, v_cache, page_table, query_starts, context_lengths, q, frequencies, layout, magnitude):
// the turned q, or True without one.
PyObject* paged_append(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 11) Py_RETURN_NONE;
  const at::Tensor *k = heads_of(args[0]), *v = heads_of(args[1]);
  Paged c;
  const int layout = layout_of(args[9]);
  float magnitude;
  if (!k || !v || layout < 0 || !paged_of(args + 2, c) || !current(k->device()) || args[10] == Py_None ||
      !positive(args[10], 1.0f, magnitude))
    Py_RETURN_NONE;
  const c10::Device dev = k->device();
  const int64_t tokens = k->size(1);
  if (v->sizes() != k->sizes() || v->scalar_type() != k->scalar_type() || v->device() != dev ||
      c.k->device() != dev || c.k->scalar_type() != k->scalar_type() || c.kv_heads != k->size(0) ||
      c.dim != k->size(2) || expanded(*c.k) || expanded(*c.v))
    Py_RETURN_NONE;
  const at::Tensor *f = nullptr, *q = nullptr;
  if (args[8] != Py_None && !(f = frequencies_of(args[8], c.dim, dev))) Py_RETURN_NONE;
  if (args[7] != Py_None) {
    q = heads_of(args[7]);
    if (!q || !f || q->size(1) != tokens || q->size(2) != c.dim || q->scalar_type() != k->scalar_type() ||
        q->device() != dev)
      Py_RETURN_NONE;
  }
  void* stream = nullptr;
  if (!stream_of(dev, &stream)) return nullptr;
  const int64_t heads = q ? q->size(0) : 0;
  at::Tensor y;
  if (q) y = empty({heads, tokens, c.dim}, k->scalar_type(), dev);
  const void *kp = k->data_ptr(), *vp = v->data_ptr(), *qp = q ? q->data_ptr() : nullptr;
  void *kc = c.k->data_ptr(), *vc = c.v->data_ptr(), *yp = q ? y.data_ptr() : nullptr;
  const auto* fp = f ? static_cast<const double*>(f->data_ptr()) : nullptr;
  const int64_t pairs = f ? f->size(0) : 0;
  const int code = dtype_code(k->scalar_type());
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = m5k_paged_append(kp, stride(*k, 0), stride(*k, 1), vp, stride(*v, 0), stride(*v, 1), code, tokens, c.kv_heads,
                        c.dim, kc, stride(*c.k, 0), stride(*c.k, 1), stride(*c.k, 2), vc, stride(*c.v, 0),
                        stride(*c.v, 1), stride(*c.v, 2), c.pages, c.page_size, c.table, c.width, c.sequences, c.starts,
                        c.context, qp, heads, q ? stride(*q, 0) : 0, q ? stride(*q, 1) : 0, yp, fp, pairs, layout,
                        magnitude, stream);
  Py_END_ALLOW_THREADS
  if (rc) return failed("m5k_paged_append", rc);
  if (!q) Py_RETURN_TRUE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// What both attention entries share.
struct Scores {
  float scale, softcap;
  int64_t window;
  const float* slopes;
  int splits;
  at::Tensor out, workspace;
  float* wp;
  int64_t elems;
};

// Checks q against the keys' heads and width, and the score options; allocates.  false: let Python look at it.
bool scores_of(const at::Tensor* q, int64_t kv_heads, int64_t dim, at::ScalarType st, c10::Device dev, PyObject* scale,
               PyObject* softcap, PyObject* window, PyObject* slopes, bool paged, int64_t sequences, int64_t keys,
               Scores& s) {
  if (!q || q->scalar_type() != st || !half_type(*q) || q->device() != dev || !current(dev) || q->size(2) != dim ||
      q->size(0) % kv_heads || (dim != 64 && dim != 128) || !rows16(*q))
    return false;
  const int64_t heads = q->size(0), tokens = q->size(1);
  if (tokens > (1 << 24) || heads > (1 << 16) || tokens * heads >= (int64_t{1} << 30)) return false;
  if (!positive(scale, static_cast<float>(1.0 / std::sqrt(static_cast<double>(dim))), s.scale) ||
      !positive(softcap, 0.0f, s.softcap) || !window_of(window, s.window) ||
      !optional_vector(slopes, heads, at::kFloat, dev, &s.slopes))
    return false;
  if (s.scale < FLT_MIN || (s.softcap != 0.0f && (s.softcap < FLT_MIN || s.scale / s.softcap > 1e37f))) return false;
  if (m5k_attention_plan(paged, tokens, heads, kv_heads, sequences, keys, 0, &s.splits, nullptr)) return false;
  s.out = empty({tokens, heads * dim}, st, dev);
  s.elems = 0;
  s.wp = nullptr;
  if (s.splits > 1) {
    s.elems = s.splits * tokens * heads * (dim + 2);
    s.workspace = empty({s.elems}, at::kFloat, dev);
    s.wp = static_cast<float*>(s.workspace.data_ptr());
  }
  return true;
}

// paged_attention(q, k_cache, v_cache, page_table, query_starts, context_lengths, scale, window, softcap, slopes,
// prefix_lengths).
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Paged c;
  Scores s;
  const int32_t* prefix;
  if (nargs != 11 || !paged_of(args + 1, c)) Py_RETURN_NONE;
  const at::Tensor* q = heads_of(args[0]);
  const c10::Device dev = c.k->device();
  if (!optional_vector(args[10], c.sequences, at::kInt, dev, &prefix) || (prefix && args[7] != Py_None) ||
      !rows16(*c.k) || !rows16(*c.v) ||
      !scores_of(q, c.kv_heads, c.dim, c.k->scalar_type(), dev, args[6], args[8], args[7], args[9], true, c.sequences,
                 c.width * c.page_size, s))
    Py_RETURN_NONE;
  void* stream = nullptr;
  if (!stream_of(dev, &stream)) return nullptr;
  const void *qp = q->data_ptr(), *kp = c.k->data_ptr(), *vp = c.v->data_ptr();
  void* op = s.out.data_ptr();
  const int code = dtype_code(q->scalar_type());
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = m5k_paged_attention(qp, code, q->size(1), q->size(0), static_cast<int>(c.dim), stride(*q, 0), stride(*q, 1), kp,
                           stride(*c.k, 0), stride(*c.k, 1), stride(*c.k, 2), vp, stride(*c.v, 0), stride(*c.v, 1),
                           stride(*c.v, 2), c.pages, c.page_size, c.kv_heads, c.table, c.width, c.sequences, c.starts,
                           c.context, s.scale, s.window, s.softcap, s.slopes, prefix, op, s.splits, s.wp, s.elems,
                           stream);
  Py_END_ALLOW_THREADS
  if (rc) return failed("m5k_paged_attention", rc);
  return THPVariable_Wrap(std::move(s.out));
  END_HANDLE_TH_ERRORS
}

// attention(q, k, v, causal, window, document_starts, prefix_lengths, softcap, slopes, scale).
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 10 || !PyBool_Check(args[3])) Py_RETURN_NONE;
  const at::Tensor *q = heads_of(args[0]), *k = heads_of(args[1]), *v = heads_of(args[2]);
  if (!q || !k || !v || v->sizes() != k->sizes() || v->scalar_type() != k->scalar_type() ||
      v->device() != k->device() || !rows16(*k) || !rows16(*v))
    Py_RETURN_NONE;
  const c10::Device dev = k->device();
  const int64_t kv_heads = k->size(0), keys = k->size(1), dim = k->size(2), tokens = q->size(1);
  for (const at::Tensor* t : {k, v})
    if (keys > 1 && (t->stride(1) < dim || t->stride(1) > (1 << 23))) Py_RETURN_NONE;
  const bool causal = args[3] == Py_True;
  const int32_t *starts = nullptr, *prefix;
  int64_t documents = 0;
  if (args[5] != Py_None) {
    const at::Tensor* d = plain(args[5]);
    if (!d || d->dim() != 1 || d->size(0) < 2 || d->scalar_type() != at::kInt || d->device() != dev || tokens != keys)
      Py_RETURN_NONE;
    starts = static_cast<const int32_t*>(d->data_ptr());
    documents = d->size(0) - 1;
  }
  Scores s;
  if (keys > (1 << 24) || !optional_vector(args[6], documents ? documents : 1, at::kInt, dev, &prefix) ||
      (prefix && (!causal || args[4] != Py_None)) ||
      !scores_of(q, kv_heads, dim, k->scalar_type(), dev, args[9], args[7], args[4], args[8], false, documents, keys,
                 s))
    Py_RETURN_NONE;
  void* stream = nullptr;
  if (!stream_of(dev, &stream)) return nullptr;
  const void *qp = q->data_ptr(), *kp = k->data_ptr(), *vp = v->data_ptr();
  void* op = s.out.data_ptr();
  const int code = dtype_code(q->scalar_type());
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = m5k_attention(qp, code, tokens, q->size(0), static_cast<int>(dim), stride(*q, 0), stride(*q, 1), kp,
                     stride(*k, 0), stride(*k, 1), vp, stride(*v, 0), stride(*v, 1), keys, kv_heads, s.scale, causal,
                     s.window, s.softcap, s.slopes, starts, documents, prefix, op, s.splits, s.wp, s.elems, stream);
  Py_END_ALLOW_THREADS
  if (rc) return failed("m5k_attention", rc);
  return THPVariable_Wrap(std::move(s.out));
  END_HANDLE_TH_ERRORS
}

// bind(stream_of, splits, staged): the Python callables above.
PyObject* bind(PyObject*, PyObject* args) {
  PyObject *s, *p, *q;
  if (!PyArg_ParseTuple(args, "OOO", &s, &p, &q)) return nullptr;
  PyObject** slots[] = {&g_stream_of, &g_splits, &g_staged};
  PyObject* given[] = {s, p, q};
  for (int i = 0; i < 3; ++i) {
    Py_INCREF(given[i]);
    Py_XDECREF(*slots[i]);
    *slots[i] = given[i];
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"quantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(quantize)), METH_FASTCALL, nullptr},
    {"gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gemm)), METH_FASTCALL, nullptr},
    {"qk", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(qk)), METH_FASTCALL, nullptr},
    {"qkv", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(qkv)), METH_FASTCALL, nullptr},
    {"rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rope)), METH_FASTCALL, nullptr},
    {"paged_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_append)), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_attention)), METH_FASTCALL,
     nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention)), METH_FASTCALL, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "m5k_fast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// abi_version and torch_version: what this file was compiled for, compared before the first call
// (_lib.load_fast).
PyMODINIT_FUNC PyInit_m5k_fast() {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && (PyModule_AddIntConstant(m, "abi_version", M5K_ABI_VERSION) != 0 ||
                       PyModule_AddStringConstant(m, "torch_version", M5K_TORCH_VERSION) != 0)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
