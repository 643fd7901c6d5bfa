// Host side of the per-layer calls (the CPython module logssms_amd._host):
//   * a typed entry for each hot C-ABI function, so that a call converts its
//     arguments in a loop over their C types (ctypes took 2.5 us for the 46
//     arguments of a decode step);
//   * conv_recurrent, the checks and the call of one decode or verify step
//     with tensors in hand;
//   * rms_norm, quantize_fp8, rms_norm_gated_fp8 and fp8_linear, the same for
//     the 8-bit projections;
//   * apply_rotary, append_paged_kv and paged_attention, the same for the
//     full-attention layers.
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
  X(gdn_fp8_linear)                       \
  X(gdn_apply_rotary)                     \
  X(gdn_append_paged_kv)                  \
  X(gdn_paged_attention_workspace_bytes)  \
  X(gdn_paged_attention)
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

// ---------------------------------------------------------------- full attention
// The axes of a view that its rows (the last axis) are walked along, the widest step first.
struct Axes {
  int64_t stride[3], size[3];
  int n = 0;
  explicit Axes(const at::Tensor& t) {
    for (int64_t d = 0; d + 1 < t.dim(); ++d) {
      if (t.size(d) <= 1) continue;
      int at = n++;
      for (; at > 0 && stride[at - 1] < t.stride(d); --at) stride[at] = stride[at - 1], size[at] = size[at - 1];
      stride[at] = t.stride(d), size[at] = t.size(d);
    }
  }
  // Elements from the first to the last of what lies inside axis `from`, in rows of `dim`.
  int64_t span(int from, int64_t dim) const {
    for (int i = from; i < n; ++i) dim += stride[i] * (size[i] - 1);
    return dim;
  }
};
// Rows [.., dim] (up to four axes) of unit channel stride, none on top of another: every
// axis steps over what lies inside it.
bool apart(const at::Tensor& t) {
  if (t.numel() == 0) return true;
  const int64_t dim = t.size(t.dim() - 1);
  if (dim > 1 && t.stride(t.dim() - 1) != 1) return false;
  const Axes axes(t);
  for (int i = 0; i < axes.n; ++i)
    if (axes.stride[i] < axes.span(i + 1, dim)) return false;
  return true;
}
// Whether rows of a (its axes from i on) from 0 on and rows of b (from j on) from `at` on
// keep clear of each other, as far as their axes tell; each of them is apart() by itself.
bool clear_of(const Axes& a, int i, const Axes& b, int j, int64_t at, int64_t dim) {
  if (at >= a.span(i, dim) || -at >= b.span(j, dim)) return true;
  if (i == a.n || j == b.n || a.stride[i] != b.stride[j]) return false;
  // What lies inside an axis is no longer than its step: an entry of a meets the entries of
  // b that are `steps` and `steps + 1` before it, where there are such.
  const int64_t step = a.stride[i], behind = (at % step + step) % step, steps = (at - behind) / step;
  auto clear = [&](int64_t before, int64_t off) {
    return before <= -b.size[j] || before >= a.size[i] || clear_of(a, i + 1, b, j + 1, off, dim);
  };
  return clear(steps, behind) && clear(steps + 1, behind - step);
}
bool clear_of(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return true;
  const int64_t bytes = static_cast<const char*>(b.data_ptr()) - static_cast<const char*>(a.data_ptr());
  return clear_of(Axes(a), 0, Axes(b), 0, bytes / a.element_size(), a.size(a.dim() - 1));
}
// A stride that is walked: 0 along an axis of one, whatever the view says.
int64_t step(const at::Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }
at::Tensor unit_channels(const at::Tensor& t) { return t.size(2) == 1 || t.stride(2) == 1 ? t : t.contiguous(); }
// One index for each of n, side by side.
at::Tensor indices(const at::Tensor& t, int64_t n, const at::Tensor& like, const char* what) {
  require(t.dim() == 1 && t.size(0) == n, what);
  require(t.device() == like.device(), "all operands on one device");
  index_code(t);
  return t.is_contiguous() ? t : t.contiguous();
}

struct Turns {
  at::Tensor positions, turns;
  int64_t rotated = 0;
  const void* positions_at() const { return positions.defined() ? positions.data_ptr() : nullptr; }
  const double* turns_at() const { return turns.defined() ? turns.data_ptr<double>() : nullptr; }
  int code() const { return positions.defined() ? index_code(positions) : GDN_I32; }
};
Turns turns_of(PyObject* positions, PyObject* turns, const at::Tensor& x) {
  Turns t;
  const at::Tensor& given = tensor(turns);
  require(given.dim() == 1 && given.scalar_type() == at::kDouble, "frequencies must be float64 [rotated / 2]");
  require(given.device() == x.device(), "all operands on one device");
  t.turns = given.contiguous();
  t.rotated = 2 * given.size(0);
  require(t.rotated <= x.size(2), "more rotated channels than the head has");
  t.positions = indices(tensor(positions), x.size(0), x, "positions must be [tokens]");
  return t;
}

// The result of rotating x: given (like x, its rows apart) or fresh.
at::Tensor rotated_out(PyObject* given, const at::Tensor& x) {
  if (given == Py_None) return fresh(x.sizes(), x.scalar_type(), x);
  const at::Tensor& out = tensor(given);
  require(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type() && out.device() == x.device(),
          "an output must be like its input");
  require(apart(out), "an output needs rows of unit stride that do not overlap");
  return out;
}

// apply_rotary(q, k or None, positions, turns, interleaved, scale, q_out or None, k_out or None) -> (q_out, k_out)
PyObject* apply_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    require(n == 8, "apply_rotary: 8 arguments expected");
    const at::Tensor& given = tensor(args[0]);
    require(given.dim() == 3 && given.size(2) > 0, "q must be [tokens, heads, dim]");
    const int code = dtype_code(given);
    at::Tensor k, k_out;
    if (args[1] != Py_None) {
      const at::Tensor& given_k = tensor(args[1]);
      require(given_k.dim() == 3 && given_k.size(0) == given.size(0) && given_k.size(2) == given.size(2) &&
                  given_k.scalar_type() == given.scalar_type() && given_k.device() == given.device(),
              "k must be [tokens, heads, dim] like q");
      k = unit_channels(given_k);
    } else {
      require(args[7] == Py_None, "k_out without k");
    }
    const at::Tensor q = unit_channels(given);
    const Turns t = turns_of(args[2], args[3], q);
    const bool interleaved = truth(args[4]);
    const float scale = real(args[5]);
    const at::Tensor q_out = rotated_out(args[6], q);
    if (k.defined()) k_out = rotated_out(args[7], k);
    require_device(q);
    const bool both = k.defined();
    launch("gdn_apply_rotary", lib::gdn_apply_rotary, q, q.data_ptr(), step(q, 0), step(q, 1), q.size(1),
           both ? k.data_ptr() : nullptr, both ? step(k, 0) : 0, both ? step(k, 1) : 0, both ? k.size(1) : 0, code,
           q.size(0), q.size(2), t.positions_at(), t.code(), t.turns_at(), t.rotated, interleaved ? 1 : 0, scale,
           q_out.data_ptr(), step(q_out, 0), step(q_out, 1), both ? k_out.data_ptr() : nullptr,
           both ? step(k_out, 0) : 0, both ? step(k_out, 1) : 0);
    return tuple_of(q_out, k_out);
  } catch (const Failed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

void check_cache(const at::Tensor& cache, const at::Tensor& like, int64_t heads, int64_t dim) {
  require(cache.dim() == 4 && cache.size(2) == heads && cache.size(3) == dim && cache.size(1) > 0,
          "a cache must be [pages, page size, kv heads, dim]");
  require(cache.scalar_type() == like.scalar_type() && cache.device() == like.device(),
          "caches must have the dtype and the device of what goes with them");
  require(dim == 1 || cache.stride(3) == 1, "a cache needs unit channel stride");
}

// append_paged_kv(k, v, k_cache, v_cache, slots, positions or None, turns or None, interleaved, scale, q or None,
//   q_out or None) -> q_out or None
PyObject* append_paged_kv(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    require(n == 11, "append_paged_kv: 11 arguments expected");
    const at::Tensor &given_k = tensor(args[0]), &given_v = tensor(args[1]), &k_cache = tensor(args[2]),
                     &v_cache = tensor(args[3]);
    require(given_k.dim() == 3 && given_k.size(1) > 0 && given_k.size(2) > 0, "k must be [tokens, kv heads, dim]");
    require(given_v.sizes() == given_k.sizes() && given_v.scalar_type() == given_k.scalar_type() &&
                given_v.device() == given_k.device(),
            "v must be like k");
    const int code = dtype_code(given_k);
    const at::Tensor k = unit_channels(given_k), v = unit_channels(given_v);
    const int64_t tokens = k.size(0), heads = k.size(1), dim = k.size(2);
    check_cache(k_cache, k, heads, dim);
    check_cache(v_cache, k, heads, dim);
    require(v_cache.size(0) == k_cache.size(0) && v_cache.size(1) == k_cache.size(1), "caches of one size");
    require(apart(k_cache) && apart(v_cache), "a cache's rows must not overlap");
    const at::Tensor slots = indices(tensor(args[4]), tokens, k, "slots must be [tokens]");
    Turns t;
    require((args[5] == Py_None) == (args[6] == Py_None), "positions go with a rotation");
    if (args[6] != Py_None) t = turns_of(args[5], args[6], k);
    const bool interleaved = truth(args[7]);
    const float scale = real(args[8]);
    at::Tensor q, q_out;
    if (args[9] != Py_None) {
      const at::Tensor& given_q = tensor(args[9]);
      require(given_q.dim() == 3 && given_q.size(0) == tokens && given_q.size(2) == dim &&
                  given_q.scalar_type() == k.scalar_type() && given_q.device() == k.device(),
              "q must be [tokens, heads, dim] like k");
      q = unit_channels(given_q);
      q_out = rotated_out(args[10], q);
    } else {
      require(args[10] == Py_None, "q_out without q");
    }
    require_device(k);
    require(clear_of(k_cache, v_cache), "the caches must not overlap");
    const bool with_q = q.defined();
    launch("gdn_append_paged_kv", lib::gdn_append_paged_kv, k, k.data_ptr(), step(k, 0), step(k, 1), v.data_ptr(),
           step(v, 0), step(v, 1), heads, code, tokens, dim, slots.data_ptr(), index_code(slots), k_cache.data_ptr(),
           step(k_cache, 0), step(k_cache, 1), step(k_cache, 2), v_cache.data_ptr(), step(v_cache, 0),
           step(v_cache, 1), step(v_cache, 2), k_cache.size(0), k_cache.size(1), t.positions_at(), t.code(),
           t.turns_at(), t.rotated, interleaved ? 1 : 0, scale, with_q ? q.data_ptr() : nullptr,
           with_q ? step(q, 0) : 0, with_q ? step(q, 1) : 0, with_q ? q.size(1) : 0,
           with_q ? q_out.data_ptr() : nullptr, with_q ? step(q_out, 0) : 0, with_q ? step(q_out, 1) : 0);
    return wrap(q_out);
  } catch (const Failed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// paged_attention(q, k_cache, v_cache, page_table, seq_lens, shared_lens or None, group_offsets or None,
//   cu_seqlens or None, scale, out or None, lse) -> (out, lse or None)
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    require(n == 11, "paged_attention: 11 arguments expected");
    const at::Tensor &given = tensor(args[0]), &k_cache = tensor(args[1]), &v_cache = tensor(args[2]),
                     &given_table = tensor(args[3]);
    require(given.dim() == 3 && given.size(1) > 0 && given.size(2) > 0, "q must be [tokens, heads, dim]");
    const int code = dtype_code(given);
    const int64_t tokens = given.size(0), heads = given.size(1), dim = given.size(2);
    require(code != GDN_F32, "q must be bfloat16 or float16");
    require(k_cache.dim() == 4 && k_cache.size(2) > 0 && heads % k_cache.size(2) == 0,
            "the query heads must be a multiple of the key heads");
    check_cache(k_cache, given, k_cache.size(2), dim);
    check_cache(v_cache, given, k_cache.size(2), dim);
    require(v_cache.size(0) == k_cache.size(0) && v_cache.size(1) == k_cache.size(1), "caches of one size");
    // rows at multiples of 16 bytes; a copy where they are not
    const bool wide = given.stride(2) == 1 && step(given, 0) % 8 == 0 && step(given, 1) % 8 == 0 &&
                      reinterpret_cast<uintptr_t>(given.data_ptr()) % 16 == 0;
    const at::Tensor q = wide ? given : given.is_contiguous() ? given.clone() : given.contiguous();
    require(given_table.dim() == 2, "page_table must be [requests, pages]");
    require(given_table.device() == q.device(), "all operands on one device");
    const int table_code = index_code(given_table);
    const at::Tensor table = given_table.size(1) <= 1 || given_table.stride(1) == 1 ? given_table : given_table.contiguous();
    const int64_t requests = table.size(0);
    const at::Tensor lens = indices(tensor(args[4]), requests, q, "seq_lens must be [requests]");
    at::Tensor shared, offsets, cu;
    if (args[5] != Py_None) {
      const at::Tensor& t = tensor(args[5]);
      require(t.dim() == 1 && t.size(0) > 0, "shared_lens must be [groups]");
      shared = indices(t, t.size(0), q, "shared_lens must be [groups]");
    }
    const int64_t groups = shared.defined() ? shared.size(0) : 0;
    if (args[6] != Py_None) {
      require(shared.defined(), "group_offsets without shared_lens");
      offsets = indices(tensor(args[6]), groups + 1, q, "group_offsets must be [groups + 1]");
    }
    require(groups <= 1 || offsets.defined(), "several groups need their offsets");
    if (args[7] != Py_None)
      cu = indices(tensor(args[7]), requests + 1, q, "cu_seqlens must be [requests + 1]");
    else
      require(tokens == requests, "one token for each request without cu_seqlens");
    const float scale = real(args[8]);
    at::Tensor out = args[9] == Py_None ? fresh(q.sizes(), q.scalar_type(), q) : tensor(args[9]), lse;
    require(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.device() == q.device(),
            "out must be like q");
    require(apart(out), "out needs rows of unit stride that do not overlap");
    require_device(q);
    if (truth(args[10])) lse = fresh({tokens, heads}, at::kFloat, q);
    if (!bound(lib::gdn_paged_attention_workspace_bytes != nullptr)) throw Failed();
    const int64_t bytes = lib::gdn_paged_attention_workspace_bytes(tokens, requests, groups, heads, k_cache.size(2), dim,
                                                                   cu.defined() ? 1 : 0);
    const at::Tensor workspace = fresh({bytes}, at::kByte, q);
    auto at_of = [](const at::Tensor& t) -> void* { return t.defined() ? t.data_ptr() : nullptr; };
    auto code_of = [](const at::Tensor& t) { return t.defined() ? index_code(t) : GDN_I32; };
    launch("gdn_paged_attention", lib::gdn_paged_attention, q, q.data_ptr(), step(q, 0), step(q, 1), code, tokens,
           heads, dim, k_cache.data_ptr(), step(k_cache, 0), step(k_cache, 1), step(k_cache, 2), v_cache.data_ptr(),
           step(v_cache, 0), step(v_cache, 1), step(v_cache, 2), k_cache.size(2), k_cache.size(0), k_cache.size(1),
           table.data_ptr(), table_code, table.stride(0), table.size(1), lens.data_ptr(), index_code(lens), requests,
           at_of(shared), code_of(shared), at_of(offsets), code_of(offsets), groups, at_of(cu), code_of(cu), scale,
           out.data_ptr(), step(out, 0), step(out, 1), static_cast<float*>(at_of(lse)), workspace.data_ptr(), bytes);
    return tuple_of(out, lse);
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
    {"apply_rotary", reinterpret_cast<PyCFunction>(&apply_rotary), METH_FASTCALL, nullptr},
    {"append_paged_kv", reinterpret_cast<PyCFunction>(&append_paged_kv), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(&paged_attention), METH_FASTCALL, nullptr},
    GDN_TYPED(GDN_METHOD)
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&kModule); }
