// Host side of the per-layer calls (the CPython module logssms_amd._host):
//   * a typed entry for each hot C-ABI function, so that a call converts its
//     arguments in a loop over their C types (ctypes took 2.5 us for the 46
//     arguments of a decode step);
//   * conv_recurrent, the checks and the call of one decode or verify step
//     with tensors in hand;
//   * rms_norm, quantize_fp8, rms_norm_gated_fp8 and fp8_linear, the same for
//     the 8-bit projections.
// A decode step of one sequence is an 8 us kernel behind what the host does
// to launch it: 15.8 us in Python and ctypes, 5.8 us through this module.
#include <Python.h>
#include <dlfcn.h>

#include <utility>

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/gdn_mi355x.h"

namespace {

// ---------------------------------------------------------------- the library
// This module links no libgdn_mi355x.so: bind(handle) takes the functions from
// the one instance that the package has opened (whichever file that is), so
// that typed entries, ctypes calls and gdn_last_error share its state.
#define GDN_TYPED(X)                      \
  X(gdn_prefill_frontend)                 \
  X(gdn_prefill_qk)                       \
  X(gdn_prefill_fused)                    \
  X(gdn_prefill_split)                    \
  X(gdn_prefill_workspace_bytes)          \
  X(gdn_chunk_workspace_bytes)            \
  X(gdn_chunk_gated_delta_rule_ws)        \
  X(gdn_chunk_gated_delta_rule_logged_ws) \
  X(gdn_store_chunk_log)                  \
  X(gdn_conv_snapshots)                   \
  X(gdn_conv_windows_logstate)            \
  X(gdn_conv_decode)                      \
  X(gdn_conv_decode_logstate)             \
  X(gdn_recurrent_logstate)               \
  X(gdn_fused_recurrent)                  \
  X(gdn_fused_conv_recurrent)             \
  X(gdn_logstate_restore)                 \
  X(gdn_rms_norm_gated)                   \
  X(gdn_rms_norm)                         \
  X(gdn_quantize_fp8)                     \
  X(gdn_rms_norm_gated_fp8)               \
  X(gdn_fp8_linear)
namespace lib {
#define GDN_POINTER(name) decltype(&::name) name = nullptr;
GDN_TYPED(GDN_POINTER)
GDN_POINTER(gdn_last_error)
}  // namespace lib

PyObject* bind(PyObject*, PyObject* handle) {
  void* opened = PyLong_AsVoidPtr(handle);
  if (!opened) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "the handle of an opened library expected");
    return nullptr;
  }
  auto find = [&](auto& pointer, const char* name) {
    pointer = reinterpret_cast<std::decay_t<decltype(pointer)>>(dlsym(opened, name));
    if (!pointer) PyErr_Format(PyExc_RuntimeError, "%s is not in the library", name);
    return pointer != nullptr;
  };
#define GDN_FIND(name) && find(lib::name, #name)
  if (!(true GDN_TYPED(GDN_FIND) GDN_FIND(gdn_last_error))) return nullptr;
  Py_RETURN_NONE;
}

// ---------------------------------------------------------------- typed entries
// One Python argument as its C parameter; sets a Python error and returns
// false where it does not fit.
bool convert(PyObject* o, int64_t& v) {
  v = PyLong_AsLongLong(o);
  return v != -1 || !PyErr_Occurred();
}
bool convert(PyObject* o, int& v) {
  int64_t x;
  if (!convert(o, x)) return false;
  v = static_cast<int>(x);
  if (v == x) return true;
  PyErr_SetString(PyExc_OverflowError, "argument exceeds a C int");
  return false;
}
bool convert(PyObject* o, float& v) {
  const double x = PyFloat_AsDouble(o);
  v = static_cast<float>(x);
  return x != -1.0 || !PyErr_Occurred();
}
template <class T>
bool convert(PyObject* o, T*& v) {  // a device address, or None
  void* p = o == Py_None ? nullptr : PyLong_AsVoidPtr(o);
  if (!p && PyErr_Occurred()) return false;
  v = static_cast<T*>(p);
  return true;
}

// f(args...) without the interpreter lock, as ctypes calls: a launch that waits
// for a place in a full queue does not stop the process's other Python threads.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};
template <class R, class... P, class... A>
R unlocked(R (*f)(P...), A... args) {
  const Unlocked scope;
  return f(args...);
}

bool bound(bool found) {
  if (!found) PyErr_SetString(PyExc_RuntimeError, "no library bound (logssms_amd._lib.host())");
  return found;
}

template <auto F> struct Entry;  // F: where bind() keeps the function
template <class R, class... A, R (**F)(A...)>
struct Entry<F> {
  template <size_t... I>
  static PyObject* invoke(PyObject* const* args, std::index_sequence<I...>) {
    std::tuple<A...> v{};
    if (!(convert(args[I], std::get<I>(v)) && ...)) return nullptr;
    return PyLong_FromLongLong(unlocked(*F, std::get<I>(v)...));
  }
  static PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != static_cast<Py_ssize_t>(sizeof...(A))) {
      PyErr_Format(PyExc_TypeError, "%zu arguments expected, %zd given", sizeof...(A), n);
      return nullptr;
    }
    if (!bound(*F != nullptr)) return nullptr;
    return invoke(args, std::index_sequence_for<A...>{});
  }
};

// ---------------------------------------------------------------- decode and verify
struct Failed {};  // a Python error is set

void require(bool ok, const char* what) {
  if (ok) return;
  PyErr_SetString(PyExc_AssertionError, what);
  throw Failed();
}

const at::Tensor& tensor(PyObject* o) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "a tensor expected, got %s", Py_TYPE(o)->tp_name);
    throw Failed();
  }
  return THPVariable_Unpack(o);
}
int64_t integer(PyObject* o) {
  int64_t v;
  if (!convert(o, v)) throw Failed();
  return v;
}
int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return GDN_F32;
    case at::kBFloat16: return GDN_BF16;
    case at::kHalf: return GDN_F16;
    default:
      PyErr_Format(PyExc_TypeError, "unsupported dtype %s", c10::toString(t.scalar_type()));
      throw Failed();
  }
}
int index_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kLong) return GDN_I64;
  if (t.scalar_type() == at::kInt) return GDN_I32;
  PyErr_Format(PyExc_TypeError, "index tensors must be int32 or int64, got %s", c10::toString(t.scalar_type()));
  throw Failed();
}

// conv_recurrent(mixed, row_index or None, gate, beta, conv_weight, A_log,
//   dt_bias, conv_state, recurrent_state, read_slots, write_slots, out or None,
//   num_k_heads, num_v_heads, head_k_dim, head_v_dim, conv_dim, state_len, layer)
// One decode step (write_slots [B]) or the T steps of a verify group
// (write_slots [B, T]); returns out ([rows, HV, dv], allocated when None).
PyObject* conv_recurrent(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    require(n == 19, "conv_recurrent: 19 arguments expected");
    const at::Tensor &mixed = tensor(args[0]), &gate = tensor(args[2]), &beta = tensor(args[3]);
    const at::Tensor weight = tensor(args[4]).contiguous(), A_log = tensor(args[5]).contiguous(),
                     dt_bias = tensor(args[6]).contiguous();
    const at::Tensor &conv = tensor(args[7]), &state = tensor(args[8]), &reads = tensor(args[9]),
                     &writes = tensor(args[10]);
    const int64_t H = integer(args[12]), HV = integer(args[13]), dk = integer(args[14]), dv = integer(args[15]),
                  conv_dim = integer(args[16]), state_len = integer(args[17]), layer = integer(args[18]);
    const bool verify = writes.dim() == 2;
    require(mixed.dim() == 2 && mixed.size(1) == conv_dim, "mixed_qkv must be [rows, conv_dim]");
    require(verify || writes.dim() == 1, "write slots must be [B] or [B, T]");
    const int64_t B = writes.size(0), T = verify ? writes.size(1) : 1;
    require(reads.dim() == 1 && reads.size(0) == B && (verify || mixed.size(0) == B), "one read slot per sequence");
    require(T >= 1, "at least one step");
    require(conv.dim() == 4 && conv.size(2) == conv_dim && conv.size(3) == state_len && conv.stride(3) == 1 &&
                conv.stride(2) == state_len,
            "conv_state must be [slots, layers, conv_dim, state_len] with contiguous windows");
    require(state.dim() == 5 && state.size(2) == HV && state.size(3) == dk && state.size(4) == dv &&
                state.stride(4) == 1 && state.stride(3) == dv,
            "recurrent_state must be [slots, layers, HV, dk, dv] with contiguous rows");
    const at::Tensor* rows = nullptr;
    if (args[1] != Py_None) {
      rows = &tensor(args[1]);
      require(rows->dim() == 1 && rows->size(0) == B * T, "one row index per step");
    }
    at::Tensor out = args[11] == Py_None ? at::empty({B * T, HV, dv}, mixed.options()) : tensor(args[11]);
    require(out.is_contiguous() && out.dim() == 3 && out.size(1) == HV && out.size(2) == dv &&
                (verify || out.size(0) == B),
            "out must be a contiguous [rows, HV, dv]");
    if (B > 0) {
      if (!mixed.is_cuda()) {
        PyErr_SetString(PyExc_RuntimeError, "libgdn_mi355x kernels need tensors on a ROCm device");
        throw Failed();
      }
      if (!bound(lib::gdn_fused_conv_recurrent != nullptr)) throw Failed();
      const int rc = unlocked(
          lib::gdn_fused_conv_recurrent, mixed.data_ptr(), mixed.stride(0), mixed.stride(1), dtype_code(mixed),
          rows ? rows->data_ptr() : nullptr, rows ? index_code(*rows) : 0, weight.data_ptr(), nullptr,
          static_cast<int>(state_len + 1), gate.data_ptr(),
          gate.stride(0), gate.stride(1), dtype_code(gate), beta.data_ptr(), beta.stride(0), beta.stride(1),
          dtype_code(beta), A_log.data_ptr(), dtype_code(A_log), dt_bias.data_ptr(), dtype_code(dt_bias), B, T, H, HV,
          dk, dv, conv.data_ptr(), conv.stride(0), conv.stride(1), state.data_ptr(), dtype_code(state),
          state.stride(0), state.stride(1), state.stride(2), layer, reads.data_ptr(), reads.stride(0),
          index_code(reads), writes.data_ptr(), writes.stride(0), verify ? writes.stride(1) : 0, index_code(writes),
          out.data_ptr(), static_cast<float>(1.0 / std::sqrt(static_cast<double>(dk))),
          c10::hip::getCurrentHIPStream(mixed.device().index()).stream());
      if (rc != GDN_OK) {
        PyErr_Format(rc == GDN_ERR_UNSUPPORTED ? PyExc_NotImplementedError : PyExc_RuntimeError,
                     "gdn_fused_conv_recurrent failed (%d): %s", rc, lib::gdn_last_error());
        throw Failed();
      }
    }
    return THPVariable_Wrap(out);
  } catch (const Failed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- 8-bit projections
constexpr int64_t kFp8Block = 128;
int64_t blocks_of(int64_t n) { return (n + kFp8Block - 1) / kFp8Block; }
int64_t padded16(int64_t n) { return (n + 15) / 16 * 16; }
// The stride of rows of 8-bit values that this package makes: whole cache lines
// from 513 values on, where that adds at most a quarter (2900 x 1111 x 1000: 11.8
// us with rows of 1008 bytes, 10.7 with rows of 1024).  kernel/fp8.py lays out
// weights by the same rule.
int64_t fp8_stride(int64_t cols) { return cols > 512 ? (cols + 127) / 128 * 128 : padded16(cols); }

void require_device(const at::Tensor& t) {
  if (t.is_cuda()) return;
  PyErr_SetString(PyExc_RuntimeError, "libgdn_mi355x kernels need tensors on a ROCm device");
  throw Failed();
}

// f(args..., the current stream of t's device) on that device.
template <class R, class... P, class... A>
void launch(const char* name, R (*f)(P...), const at::Tensor& t, A... args) {
  if (!bound(f != nullptr)) throw Failed();
  const c10::DeviceGuard guard(t.device());
  const int rc =
      unlocked(f, args..., static_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream()));
  if (rc == GDN_OK) return;
  PyErr_Format(rc == GDN_ERR_UNSUPPORTED ? PyExc_NotImplementedError : PyExc_RuntimeError, "%s failed (%d): %s", name, rc,
               lib::gdn_last_error());
  throw Failed();
}

// An uninitialised tensor beside `like`, on a GPU without the dispatcher's turns
// (add_rms_norm_fp8 makes three: a call takes the host 5.5 us, 6.4 through at::empty).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  if (!like.is_cuda()) return at::empty(sizes, like.options().dtype(type));
  return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

// t as [rows, cols] with unit column stride; a copy where it has no such view.
at::Tensor rows_of(const at::Tensor& t) {
  const int64_t cols = t.size(-1);
  const at::Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / cols, cols});
  return cols == 1 || r.stride(1) == 1 ? r : r.contiguous();
}

// Uninitialised quantised rows: values at a stride that is a multiple of 16
// bytes, scales block by block (strides 1, rows), as the product reads them.
struct Fp8Out {
  at::Tensor values, scales;
};
Fp8Out fp8_out(int64_t rows, int64_t cols, const at::Tensor& like) {
  const int64_t shape[] = {rows, blocks_of(cols)}, strides[] = {1, std::max<int64_t>(rows, 1)};
  Fp8Out out{fresh({rows, fp8_stride(cols)}, at::kFloat8_e4m3fn, like),
             like.is_cuda() ? at::Tensor(at::detail::empty_strided_cuda(shape, strides, at::kFloat, like.device()))
                            : at::empty_strided(shape, strides, like.options().dtype(at::kFloat))};
  if (out.values.size(1) != cols) out.values = out.values.narrow(1, 0, cols);
  return out;
}

PyObject* wrap(const at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}
template <class... T>
PyObject* tuple_of(const T&... tensors) {
  PyObject* made[] = {wrap(tensors)...};
  PyObject* result = PyTuple_New(sizeof...(T));
  for (size_t i = 0; i < sizeof...(T); ++i) {
    if (!result || !made[i]) {
      for (size_t j = i; j < sizeof...(T); ++j) Py_XDECREF(made[j]);
      Py_XDECREF(result);
      return nullptr;
    }
    PyTuple_SET_ITEM(result, i, made[i]);
  }
  return result;
}

float real(PyObject* o) {
  float v;
  if (!convert(o, v)) throw Failed();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Failed();
  return v;
}

// rms_norm(x, residual or None, weight, eps, weight_offset, residual_out or None,
//   quantize, keep) -> (values, scales, y, residual_out), None for what is not wanted
PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    require(n == 8, "rms_norm: 8 arguments expected");
    const at::Tensor& x = tensor(args[0]);
    const at::Tensor weight = tensor(args[2]).contiguous();
    const float eps = real(args[3]), offset = real(args[4]);
    const bool quantize = truth(args[6]), keep = truth(args[7]);
    require(x.dim() >= 1 && x.size(-1) > 0, "rows of at least one value");
    const int64_t cols = x.size(-1);
    require(weight.dim() == 1 && weight.size(0) == cols, "weight must be [x.shape[-1]]");
    require(weight.device() == x.device(), "all operands on one device");
    const at::Tensor x2 = rows_of(x);
    const int64_t rows = x2.size(0);
    at::Tensor res2, sum, sum2;
    const bool add = args[1] != Py_None;
    if (add) {
      const at::Tensor& residual = tensor(args[1]);
      auto like_x = [&](const at::Tensor& t) {
        return t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type() && t.device() == x.device();
      };
      require(like_x(residual), "the residual must be like x");
      res2 = rows_of(residual);
      if (args[5] != Py_None) {
        sum = tensor(args[5]);
        require(like_x(sum), "residual_out must be like x");
        sum2 = sum.dim() == 2 ? sum : sum.view({rows, cols});
        require((cols == 1 || sum2.stride(1) == 1) && (rows <= 1 || sum2.stride(0) >= cols),
                "residual_out needs rows of unit stride");
      }
    } else {
      require(args[5] == Py_None, "residual_out without a residual");
    }
    require_device(x);
    const int code = dtype_code(x), weight_code = dtype_code(weight);
    if (add && !sum.defined()) {
      sum = fresh(x.sizes(), x.scalar_type(), x);
      sum2 = sum;
    }
    Fp8Out q;
    at::Tensor y;
    if (quantize) q = fp8_out(rows, cols, x);
    if (keep) y = fresh(x.sizes(), x.scalar_type(), x);
    auto at_of = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    const int64_t sum_stride = !sum2.defined() ? 0 : sum2.is_contiguous() ? cols : sum2.stride(0);
    launch("gdn_rms_norm", lib::gdn_rms_norm, x, x2.data_ptr(), code, rows, cols, x2.stride(0), at_of(res2),
           add ? res2.stride(0) : 0, weight.data_ptr(), weight_code, offset, eps, at_of(sum2), sum_stride, at_of(y), cols,
           at_of(q.values), quantize ? q.values.stride(0) : 0, static_cast<float*>(at_of(q.scales)),
           quantize ? q.scales.stride(0) : 0, quantize ? q.scales.stride(1) : 0);
    return tuple_of(q.values, q.scales, y, sum);
  } catch (const Failed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// quantize_fp8(x) -> (values, scales)
PyObject* quantize_fp8(PyObject*, PyObject* arg) {
  HANDLE_TH_ERRORS
  try {
    const at::Tensor& x = tensor(arg);
    require(x.dim() >= 1 && x.size(-1) > 0, "rows of at least one value");
    const int code = dtype_code(x);
    require_device(x);
    const at::Tensor x2 = rows_of(x);
    const int64_t rows = x2.size(0), cols = x2.size(1);
    const Fp8Out q = fp8_out(rows, cols, x);
    launch("gdn_quantize_fp8", lib::gdn_quantize_fp8, x, x2.data_ptr(), code, rows, cols, x2.stride(0),
           q.values.data_ptr(), q.values.stride(0), q.scales.data_ptr<float>(), q.scales.stride(0), q.scales.stride(1));
    return tuple_of(q.values, q.scales);
  } catch (const Failed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// rms_norm_gated_fp8(hidden, gate, weight, eps) -> (values, scales)
PyObject* rms_norm_gated_fp8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    require(n == 4, "rms_norm_gated_fp8: 4 arguments expected");
    const at::Tensor &given = tensor(args[0]), &given_gate = tensor(args[1]);
    const at::Tensor weight = tensor(args[2]).contiguous();
    const float eps = real(args[3]);
    require(given.dim() == 3 && given.sizes() == given_gate.sizes(), "[tokens, heads, dim] expected");
    require(given.scalar_type() == given_gate.scalar_type(), "hidden states and gate of one dtype");
    require(given.device() == given_gate.device() && given.device() == weight.device(), "all operands on one device");
    const int64_t tokens = given.size(0), heads = given.size(1), dim = given.size(2);
    require(heads > 0 && dim > 0 && weight.dim() == 1 && weight.size(0) == dim, "weight must be [dim]");
    const int code = dtype_code(given), weight_code = dtype_code(weight);
    require_device(given);
    auto unit = [&](const at::Tensor& t) { return dim == 1 || t.stride(2) == 1 ? t : t.contiguous(); };
    const at::Tensor x = unit(given), gate = unit(given_gate);
    const Fp8Out q = fp8_out(tokens, heads * dim, x);
    launch("gdn_rms_norm_gated_fp8", lib::gdn_rms_norm_gated_fp8, x, x.data_ptr(), code, tokens, heads, dim, x.stride(0),
           x.stride(1), gate.data_ptr(), gate.stride(0), gate.stride(1), weight.data_ptr(), weight_code, eps,
           q.values.data_ptr(), q.values.stride(0), q.scales.data_ptr<float>(), q.scales.stride(0), q.scales.stride(1));
    return tuple_of(q.values, q.scales);
  } catch (const Failed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// 8-bit rows as the product takes them: 16-byte aligned, apart, and readable
// up to the next multiple of 16 bytes.
void check_fp8_rows(const at::Tensor& t, bool weight) {
  require(t.dim() == 2 && t.scalar_type() == at::kFloat8_e4m3fn,
          weight ? "weight values must be a 2-D float8_e4m3fn tensor" : "x values must be a 2-D float8_e4m3fn tensor");
  const int64_t rows = t.size(0), cols = t.size(1);
  require(cols > 0 && (cols == 1 || t.stride(1) == 1), "8-bit values need unit column stride");
  if (rows == 0) return;
  require(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
              (rows == 1 || (t.stride(0) % 16 == 0 && t.stride(0) >= cols)),
          "8-bit rows must start at multiples of 16 bytes and not overlap");
  require(cols % 16 == 0 || t.storage_offset() + (rows - 1) * t.stride(0) + padded16(cols) <=
                                static_cast<int64_t>(t.storage().nbytes()),
          "the last 8-bit row must be readable up to a multiple of 16 bytes");
}

// fp8_linear(x values, x scales, weight values, weight scales, out_dtype, out or None)
PyObject* fp8_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    require(n == 6, "fp8_linear: 6 arguments expected");
    const at::Tensor &x = tensor(args[0]), &xs = tensor(args[1]), &w = tensor(args[2]), &ws = tensor(args[3]);
    check_fp8_rows(x, false);
    check_fp8_rows(w, true);
    const int64_t M = x.size(0), K = x.size(1), N = w.size(0), blocks = blocks_of(K);
    require(N > 0 && w.size(1) == K, "x [M, K] and weight [N, K] must share K");
    require(xs.scalar_type() == at::kFloat && xs.dim() == 2 && xs.size(0) == M && xs.size(1) == blocks,
            "x scales must be fp32 [M, ceil(K / 128)]");
    require(ws.scalar_type() == at::kFloat && ws.dim() == 2 && ws.size(0) == blocks_of(N) && ws.size(1) == blocks,
            "weight scales must be fp32 [ceil(N / 128), ceil(K / 128)]");
    require(THPDtype_Check(args[4]), "out_dtype must be a dtype");
    const at::ScalarType type = reinterpret_cast<THPDtype*>(args[4])->scalar_type;
    require(type == at::kBFloat16 || type == at::kHalf, "out_dtype must be bfloat16 or float16");
    at::Tensor out;
    if (args[5] != Py_None) {
      out = tensor(args[5]);
      require(out.dim() == 2 && out.size(0) == M && out.size(1) == N && out.scalar_type() == type,
              "out must be [M, N] of out_dtype");
      require((N == 1 || out.stride(1) == 1) && (M <= 1 || out.stride(0) >= N), "out needs rows of unit stride");
      require(out.device() == x.device(), "all operands on one device");
    }
    require(xs.device() == x.device() && w.device() == x.device() && ws.device() == x.device(),
            "all operands on one device");
    if (!out.defined()) out = fresh({M, N}, type, x);
    if (M > 0) {
      require_device(x);
      launch("gdn_fp8_linear", lib::gdn_fp8_linear, x, x.data_ptr(), x.stride(0), xs.data_ptr<float>(), xs.stride(0),
             xs.stride(1), w.data_ptr(), w.stride(0), ws.data_ptr<float>(), ws.stride(0), ws.stride(1), M, N, K,
             out.data_ptr(), dtype_code(out), out.stride(0));
    }
    return THPVariable_Wrap(out);
  } catch (const Failed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

#define GDN_METHOD(name) {#name, reinterpret_cast<PyCFunction>(&Entry<&lib::name>::call), METH_FASTCALL, nullptr},
PyMethodDef kMethods[] = {
    {"bind", &bind, METH_O, nullptr},
    {"conv_recurrent", reinterpret_cast<PyCFunction>(&conv_recurrent), METH_FASTCALL, nullptr},
    {"rms_norm", reinterpret_cast<PyCFunction>(&rms_norm), METH_FASTCALL, nullptr},
    {"quantize_fp8", &quantize_fp8, METH_O, nullptr},
    {"rms_norm_gated_fp8", reinterpret_cast<PyCFunction>(&rms_norm_gated_fp8), METH_FASTCALL, nullptr},
    {"fp8_linear", reinterpret_cast<PyCFunction>(&fp8_linear), METH_FASTCALL, nullptr},
    GDN_TYPED(GDN_METHOD)
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&kModule); }
