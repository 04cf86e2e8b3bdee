// fast_ops.cpp -- the host path of the operators in ops.py for the calls that
// need none of their conversions, as a CPython extension.
//
// What bounds it: nothing on the GPU.  A decode step is a chain of kernels of
// 3..13 us each, and the Python body of one operator call (argument rules,
// shape arithmetic, two allocations, twenty ctypes conversions) took 13..16 us,
// so the GPU waited for the host between any two of them: the projections of
// four layers with 4096 x 14336 MLPs at 4 bits took 420 us where their kernels
// take 161.  Each function here takes the operator's arguments, looks at the
// tensors through libtorch, allocates the output (and the workspace, which
// torch's caching allocator hands out per stream) and calls the C ABI.
//
// A function returns None -- and ops.py goes on with its own body -- for
// everything that is not the plain case: another device than the current one,
// operands to be converted, expanded or made contiguous, a gradient to be
// recorded (but for attention and what decoder_ops.h has), a shape or an option that ops.py refuses, and any status other than
// MLXROCM_OK (ops.py then makes the same call and turns it into an exception).
// So the rules and messages stay in one place; here are only the conditions
// under which nothing of them applies.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <cstring>
#include <optional>
#include <stdexcept>
#include <vector>

#include "mlx_rocm_qmm.h"

namespace {

// Entry points of the library that ops.py has loaded (bind()): the extension
// does not link it, so that both always use the same one.
struct Abi {
  decltype(&mlxrocm_qmm_workspace_size) qmm_workspace_size;
  decltype(&mlxrocm_qmm_prepacked) qmm_prepacked;
  decltype(&mlxrocm_qmm_sb_image_size) qmm_sb_image_size;
  decltype(&mlxrocm_qmm_rows_supported) rows_supported;
  decltype(&mlxrocm_qmm_rows_workspace_size) rows_workspace_size;
  decltype(&mlxrocm_qmm_rows_prepacked) rows_prepacked;
  decltype(&mlxrocm_fp_qmm_workspace_size) fp_qmm_workspace_size;
  decltype(&mlxrocm_fp_qmm) fp_qmm;
  decltype(&mlxrocm_fp_qmm_rows_supported) fp_rows_supported;
  decltype(&mlxrocm_fp_qmm_rows_workspace_size) fp_rows_workspace_size;
  decltype(&mlxrocm_fp_qmm_rows) fp_rows;
  decltype(&mlxrocm_qmm_swiglu_workspace_size) swiglu_workspace_size;
  decltype(&mlxrocm_qmm_swiglu) swiglu;
  decltype(&mlxrocm_fp_qqmm_workspace_size) fp_qqmm_workspace_size;
  decltype(&mlxrocm_fp_qqmm) fp_qqmm;
  decltype(&mlxrocm_switch_glu_workspace_size) switch_glu_workspace_size;
  decltype(&mlxrocm_switch_glu) switch_glu;
  decltype(&mlxrocm_affine_quantize) affine_quantize;
  decltype(&mlxrocm_affine_dequantize) affine_dequantize;
  decltype(&mlxrocm_fp_quantize) fp_quantize;
  decltype(&mlxrocm_fp_dequantize) fp_dequantize;
  decltype(&mlxrocm_window_attention_workspace_size) window_workspace_size;
  decltype(&mlxrocm_window_attention_lse_size) window_lse_size;
  decltype(&mlxrocm_window_attention) window_attention;
  decltype(&mlxrocm_window_attention_vjp_workspace_size) vjp_workspace_size;
  decltype(&mlxrocm_window_attention_vjp) window_vjp;
  decltype(&mlxrocm_copy_strided) copy_strided;
  decltype(&mlxrocm_last_error) last_error;
  decltype(&mlxrocm_paged_attention_workspace_size) paged_workspace_size;
  decltype(&mlxrocm_paged_attention) paged_attention;
  decltype(&mlxrocm_paged_cache_update) paged_cache_update;
  decltype(&mlxrocm_verify_draft_workspace_size) verify_workspace_size;
  decltype(&mlxrocm_verify_draft) verify_draft;
  decltype(&mlxrocm_rope) rope;
  decltype(&mlxrocm_rope_cache_update) rope_cache_update;
  decltype(&mlxrocm_route_experts) route_experts;
  decltype(&mlxrocm_route_experts_vjp) route_experts_vjp;
  decltype(&mlxrocm_adapter_matmul_workspace_size) adapter_workspace_size;
  decltype(&mlxrocm_adapter_matmul_h_size) adapter_h_size;
  decltype(&mlxrocm_adapter_matmul) adapter_matmul;
  decltype(&mlxrocm_adapter_matmul_vjp_workspace_size) adapter_vjp_workspace_size;
  decltype(&mlxrocm_adapter_matmul_vjp) adapter_vjp;
};
Abi abi{};
bool bound = false;

constexpr int kAffine = -1;
constexpr int kNoMode = -2;

// "affine" -> kAffine, a floating-point mode -> its mlxrocm_fp_mode
int mode_of(PyObject* o) {
  if (!PyUnicode_CheckExact(o)) {
    return kNoMode;
  }
  Py_ssize_t n = 0;
  const char* s = PyUnicode_AsUTF8AndSize(o, &n);
  if (s == nullptr) {
    PyErr_Clear();
    return kNoMode;
  }
  const auto is = [&](const char* name) {
    return static_cast<size_t>(n) == std::strlen(name) && std::memcmp(s, name, n) == 0;
  };
  return is("affine") ? kAffine
      : is("mxfp4")   ? static_cast<int>(MLXROCM_MXFP4)
      : is("mxfp8")   ? static_cast<int>(MLXROCM_MXFP8)
      : is("nvfp4")   ? static_cast<int>(MLXROCM_NVFP4)
                      : kNoMode;
}

// group_size or bits: an exact int, or None for the mode's default; -1 otherwise
int int_or(PyObject* o, int fallback) {
  if (o == Py_None) {
    return fallback;
  }
  if (!PyLong_CheckExact(o)) {
    return -1;
  }
  int overflow = 0;
  const long v = PyLong_AsLongAndOverflow(o, &overflow);
  return overflow == 0 && v > 0 && v < 1024 ? static_cast<int>(v) : -1;
}

// The parameters of a call; false where ops.py would complain.
bool params_of(int mode, PyObject* group, PyObject* bits_obj, int* gs, int* bits) {
  if (mode == kAffine) {
    *gs = int_or(group, 64);
    *bits = int_or(bits_obj, 4);
    return (*gs == 32 || *gs == 64 || *gs == 128) && *bits >= 2 && *bits <= 8 && *bits != 7;
  }
  const int want_gs = mode == MLXROCM_NVFP4 ? 16 : 32;
  const int want_bits = mode == MLXROCM_MXFP8 ? 8 : 4;
  *gs = int_or(group, want_gs);
  *bits = int_or(bits_obj, want_bits);
  return *gs == want_gs && *bits == want_bits;
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat:
      return MLXROCM_FLOAT32;
    case at::kHalf:
      return MLXROCM_FLOAT16;
    case at::kBFloat16:
      return MLXROCM_BFLOAT16;
    default:
      return -1;
  }
}

// The device of the first operand; -1 unless that is the current GPU.
c10::DeviceIndex device_of(PyObject* o) {
  if (!THPVariable_CheckExact(o)) {
    return -1;
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda()) {
    return -1;
  }
  const c10::DeviceIndex device = t.device().index();
  return device == c10::hip::current_device() ? device : -1;
}

// A plain contiguous tensor on `device` with something in it.
const at::Tensor* tensor_of(PyObject* o, c10::DeviceIndex device) {
  if (!THPVariable_CheckExact(o)) {
    return nullptr;
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && t.device().index() == device && t.is_contiguous() &&
          t.numel() > 0 && !t.is_conj() && !t.is_neg()
      ? &t
      : nullptr;
}

// The same of two dimensions and the given type.
const at::Tensor* matrix_of(PyObject* o, c10::DeviceIndex device, at::ScalarType type) {
  const at::Tensor* t = tensor_of(o, device);
  return t != nullptr && t->dim() == 2 && t->scalar_type() == type ? t : nullptr;
}

bool fits_int(int64_t v) {
  return v > 0 && v < (int64_t{1} << 31);
}

at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type, c10::DeviceIndex device) {
  return at::Tensor(at::detail::empty_cuda(
      sizes, type, c10::Device(c10::DeviceType::CUDA, device), std::nullopt));
}

void* stream_of(c10::DeviceIndex device) {
  return c10::hip::getCurrentHIPStream(device).stream();
}

// A workspace: gone to the allocator again when the call returns, which hands
// it to later work of the same stream only.
struct Workspace {
  at::Tensor t;
  size_t bytes = 0;
  Workspace(size_t n, c10::DeviceIndex device) : bytes(n) {
    if (n != 0) {
      t = new_tensor({static_cast<int64_t>(n)}, at::kByte, device);
    }
  }
  void* ptr() const {
    return bytes != 0 ? t.data_ptr() : nullptr;
  }
};

// shape of x with its last dimension replaced
c10::SmallVector<int64_t, 6> with_last(const at::Tensor& x, int64_t last) {
  c10::SmallVector<int64_t, 6> s(x.sizes().begin(), x.sizes().end());
  s.back() = last;
  return s;
}

bool records_grad(const at::Tensor& t) {
  return t.requires_grad() && at::GradMode::is_enabled();
}

PyObject* wrap(at::Tensor&& t) {
  return THPVariable_Wrap(std::move(t));
}

#define NOT_PLAIN Py_RETURN_NONE
#define FAST_TRY try {
#define FAST_CATCH                                      \
  }                                                     \
  catch (const c10::OutOfMemoryError&) {                \
    Py_RETURN_NONE; /* ops.py allocates and raises */   \
  }                                                     \
  catch (const std::exception& e) {                     \
    PyErr_SetString(PyExc_RuntimeError, e.what());      \
    return nullptr;                                     \
  }

// quantized_matmul(x, w, scales, biases, transpose, group_size, bits, mode, sb_image)
PyObject* quantized_matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!bound || n != 9) {
    NOT_PLAIN;
  }
  FAST_TRY
  const c10::DeviceIndex device = device_of(args[0]);
  if (device < 0) {
    NOT_PLAIN;
  }
  const at::Tensor* x = tensor_of(args[0], device);
  const at::Tensor* w = matrix_of(args[1], device, at::kUInt32);
  const int mode = mode_of(args[7]);
  int gs = 0;
  int bits = 0;
  if (x == nullptr || w == nullptr || x->dim() < 1 || mode == kNoMode ||
      !params_of(mode, args[5], args[6], &gs, &bits)) {
    NOT_PLAIN;
  }
  const int code = dtype_code(x->scalar_type());
  if (code < 0 || records_grad(*x)) {
    NOT_PLAIN;
  }
  const at::Tensor* scales =
      matrix_of(args[2], device, mode == kAffine ? x->scalar_type() : at::kByte);
  const at::Tensor* biases = nullptr;
  if (scales == nullptr || records_grad(*scales)) {
    NOT_PLAIN;
  }
  if (mode == kAffine) {
    biases = matrix_of(args[3], device, x->scalar_type());
    if (biases == nullptr || records_grad(*biases) || biases->sizes() != scales->sizes()) {
      NOT_PLAIN;
    }
  } else if (args[3] != Py_None || args[8] != Py_None) {
    NOT_PLAIN;
  }
  const int transpose = PyObject_IsTrue(args[4]);
  if (transpose < 0) {
    return nullptr;
  }
  const int64_t rows_w = w->size(0);
  const int64_t codes_w = w->size(1) * 32 / bits;
  const int64_t K = transpose ? codes_w : rows_w;
  const int64_t N = transpose ? rows_w : codes_w;
  if (x->size(-1) != K || scales->size(0) != rows_w || scales->size(1) * gs != codes_w ||
      w->size(1) * 32 != codes_w * bits) {
    NOT_PLAIN;
  }
  const int64_t M = x->numel() / K;
  if (!fits_int(M) || !fits_int(N) || !fits_int(K)) {
    NOT_PLAIN;
  }
  const void* image = nullptr;
  if (args[8] != Py_None) {
    const at::Tensor* t = tensor_of(args[8], device);
    if (t == nullptr || !transpose || t->scalar_type() != x->scalar_type() ||
        t->nbytes() != abi.qmm_sb_image_size(N, K, 1, gs, code)) {
      NOT_PLAIN;
    }
    image = t->data_ptr();
  }
  at::Tensor out = new_tensor(with_last(*x, N), x->scalar_type(), device);
  void* stream = stream_of(device);
  int rc = 0;
  if (mode == kAffine) {
    const bool rows = transpose && abi.rows_supported(M, N, K, 1, gs, bits, code);
    const Workspace ws(
        rows ? abi.rows_workspace_size(M, N, K, 1, gs, bits, code)
             : abi.qmm_workspace_size(M, N, K, 1, 0, gs, bits, code, transpose),
        device);
    Py_BEGIN_ALLOW_THREADS;
    if (rows) {
      rc = abi.rows_prepacked(
          x->data_ptr(), static_cast<const uint32_t*>(w->data_ptr()), scales->data_ptr(),
          biases->data_ptr(), image, out.data_ptr(), M, N, K, 1, M * K, 0, 0, gs, bits, code,
          ws.ptr(), ws.bytes, stream);
    } else {
      rc = abi.qmm_prepacked(
          x->data_ptr(), static_cast<const uint32_t*>(w->data_ptr()), scales->data_ptr(),
          biases->data_ptr(), image, out.data_ptr(), M, N, K, 1, M * K, 0, 0, gs, bits, code,
          transpose, ws.ptr(), ws.bytes, stream);
    }
    Py_END_ALLOW_THREADS;
  } else if (transpose && abi.fp_rows_supported(M, N, K, 1, mode, code)) {
    const Workspace ws(abi.fp_rows_workspace_size(M, N, K, 1, mode, code), device);
    Py_BEGIN_ALLOW_THREADS;
    rc = abi.fp_rows(
        x->data_ptr(), static_cast<const uint32_t*>(w->data_ptr()),
        static_cast<const uint8_t*>(scales->data_ptr()), out.data_ptr(), M, N, K, 1, M * K, 0, 0,
        mode, code, ws.ptr(), ws.bytes, stream);
    Py_END_ALLOW_THREADS;
  } else {
    const Workspace ws(abi.fp_qmm_workspace_size(M, N, K, 1, 0, mode, code, transpose), device);
    Py_BEGIN_ALLOW_THREADS;
    rc = abi.fp_qmm(
        x->data_ptr(), static_cast<const uint32_t*>(w->data_ptr()),
        static_cast<const uint8_t*>(scales->data_ptr()), out.data_ptr(), M, N, K, 1, M * K, 0, 0,
        mode, code, transpose, ws.ptr(), ws.bytes, stream);
    Py_END_ALLOW_THREADS;
  }
  if (rc != MLXROCM_OK) {
    NOT_PLAIN;
  }
  return wrap(std::move(out));
  FAST_CATCH
}

// quantized_swiglu(x, gate, up, group_size, bits); gate and up are triplets
PyObject* quantized_swiglu(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!bound || n != 5) {
    NOT_PLAIN;
  }
  FAST_TRY
  const c10::DeviceIndex device = device_of(args[0]);
  if (device < 0) {
    NOT_PLAIN;
  }
  const at::Tensor* x = tensor_of(args[0], device);
  int gs = 0;
  int bits = 0;
  if (x == nullptr || x->dim() < 1 || !params_of(kAffine, args[3], args[4], &gs, &bits) ||
      !PyTuple_CheckExact(args[1]) || PyTuple_GET_SIZE(args[1]) != 3 ||
      !PyTuple_CheckExact(args[2]) || PyTuple_GET_SIZE(args[2]) != 3) {
    NOT_PLAIN;
  }
  const int code = dtype_code(x->scalar_type());
  const at::Tensor* t[2][3];
  for (int i = 0; i < 2; ++i) {
    for (int j = 0; j < 3; ++j) {
      t[i][j] = matrix_of(
          PyTuple_GET_ITEM(args[1 + i], j), device, j == 0 ? at::kUInt32 : x->scalar_type());
      if (t[i][j] == nullptr || t[i][j]->sizes() != t[0][j]->sizes()) {
        NOT_PLAIN;
      }
    }
  }
  const int64_t N = t[0][0]->size(0);
  const int64_t K = t[0][0]->size(1) * 32 / bits;
  const at::Tensor& scales = *t[0][1];
  if (code < 0 || x->size(-1) != K || t[0][2]->sizes() != scales.sizes() || scales.size(0) != N ||
      scales.size(1) * gs != K || t[0][0]->size(1) * 32 != K * bits) {
    NOT_PLAIN;
  }
  const int64_t M = x->numel() / K;
  if (M > 8 || !fits_int(N) || !fits_int(K)) {
    NOT_PLAIN;
  }
  at::Tensor out = new_tensor(with_last(*x, N), x->scalar_type(), device);
  const size_t need = abi.swiglu_workspace_size(M, N, code);
  const Workspace ws(need < 16 ? 16 : need, device);
  void* stream = stream_of(device);
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS;
  rc = abi.swiglu(
      x->data_ptr(), static_cast<const uint32_t*>(t[0][0]->data_ptr()), t[0][1]->data_ptr(),
      t[0][2]->data_ptr(), static_cast<const uint32_t*>(t[1][0]->data_ptr()),
      t[1][1]->data_ptr(), t[1][2]->data_ptr(), out.data_ptr(), ws.ptr(), M, N, K, gs, bits, code,
      stream);
  Py_END_ALLOW_THREADS;
  if (rc != MLXROCM_OK) {
    NOT_PLAIN;
  }
  return wrap(std::move(out));
  FAST_CATCH
}

// switch_glu(x, indices, gate, up, down, group_size, bits): the expert-routed gated
// MLP of nn.SwitchGLU over three (weight, scales, biases) stacks
PyObject* switch_glu(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!bound || n != 7) {
    NOT_PLAIN;
  }
  FAST_TRY
  const c10::DeviceIndex device = device_of(args[0]);
  if (device < 0) {
    NOT_PLAIN;
  }
  const at::Tensor* x = tensor_of(args[0], device);
  const at::Tensor* indices = tensor_of(args[1], device);
  int gs = 0;
  int bits = 0;
  if (x == nullptr || indices == nullptr || x->dim() < 1 || indices->dim() != x->dim() ||
      !params_of(kAffine, args[5], args[6], &gs, &bits)) {
    NOT_PLAIN;
  }
  const at::ScalarType it = indices->scalar_type();
  const int index_bytes = it == at::kLong ? 8 : it == at::kInt || it == at::kUInt32 ? 4 : 0;
  const int code = dtype_code(x->scalar_type());
  const auto lead = [](const at::Tensor& t) { return t.sizes().slice(0, t.dim() - 1); };
  if (index_bytes == 0 || code < 0 || code == MLXROCM_FLOAT32 || lead(*x) != lead(*indices)) {
    NOT_PLAIN;
  }
  const int64_t D = x->size(-1);
  const at::Tensor* t[3][3];
  for (int i = 0; i < 3; ++i) {
    PyObject* triplet = args[2 + i];
    if (!PyTuple_CheckExact(triplet) || PyTuple_GET_SIZE(triplet) != 3) {
      NOT_PLAIN;
    }
    for (int j = 0; j < 3; ++j) {
      t[i][j] = tensor_of(PyTuple_GET_ITEM(triplet, j), device);
      if (t[i][j] == nullptr || t[i][j]->dim() != 3 ||
          t[i][j]->scalar_type() != (j == 0 ? at::kUInt32 : x->scalar_type())) {
        NOT_PLAIN;
      }
    }
  }
  const int64_t E = t[0][0]->size(0);
  const int64_t F = t[0][0]->size(1);
  for (int i = 0; i < 3; ++i) {
    const int64_t rows = i < 2 ? F : D;
    const int64_t inner = i < 2 ? D : F;
    const at::Tensor& w = *t[i][0];
    if (w.size(0) != E || w.size(1) != rows || w.size(2) * 32 != inner * bits) {
      NOT_PLAIN;
    }
    for (int j = 1; j < 3; ++j) {
      const at::Tensor& s = *t[i][j];
      if (s.size(0) != E || s.size(1) != rows || s.size(2) * gs != inner) {
        NOT_PLAIN;
      }
    }
  }
  const int64_t top = indices->size(-1);
  const int64_t tokens = indices->numel() / top;
  if (!fits_int(tokens * top) || !fits_int(D) || !fits_int(F) || !fits_int(E)) {
    NOT_PLAIN;
  }
  const size_t need = abi.switch_glu_workspace_size(tokens, top, D, F, E, gs, bits, code);
  if (need == 0) {
    NOT_PLAIN;
  }
  c10::SmallVector<int64_t, 6> shape(indices->sizes().begin(), indices->sizes().end());
  shape.push_back(D);
  at::Tensor out = new_tensor(shape, x->scalar_type(), device);
  const Workspace ws(need, device);
  void* stream = stream_of(device);
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS;
  rc = abi.switch_glu(
      x->data_ptr(), indices->data_ptr(), index_bytes,
      static_cast<const uint32_t*>(t[0][0]->data_ptr()), t[0][1]->data_ptr(), t[0][2]->data_ptr(),
      static_cast<const uint32_t*>(t[1][0]->data_ptr()), t[1][1]->data_ptr(), t[1][2]->data_ptr(),
      static_cast<const uint32_t*>(t[2][0]->data_ptr()), t[2][1]->data_ptr(), t[2][2]->data_ptr(),
      out.data_ptr(), tokens, top, D, F, E, gs, bits, code, ws.ptr(), ws.bytes, stream);
  Py_END_ALLOW_THREADS;
  if (rc != MLXROCM_OK) {
    NOT_PLAIN;
  }
  return wrap(std::move(out));
  FAST_CATCH
}

// qqmm(x, w, scales, group_size, bits, mode) with a quantized w
PyObject* qqmm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!bound || n != 6) {
    NOT_PLAIN;
  }
  FAST_TRY
  const c10::DeviceIndex device = device_of(args[0]);
  if (device < 0) {
    NOT_PLAIN;
  }
  const at::Tensor* x = tensor_of(args[0], device);
  const at::Tensor* w = matrix_of(args[1], device, at::kUInt32);
  const at::Tensor* scales = matrix_of(args[2], device, at::kByte);
  const int mode = mode_of(args[5]);
  int gs = 0;
  int bits = 0;
  if (x == nullptr || w == nullptr || scales == nullptr || x->dim() < 1 || mode < 0 ||
      !params_of(mode, args[3], args[4], &gs, &bits)) {
    NOT_PLAIN;
  }
  const int code = dtype_code(x->scalar_type());
  const int64_t N = w->size(0);
  const int64_t K = w->size(1) * 32 / bits;
  if (code < 0 || x->size(-1) != K || scales->size(0) != N || scales->size(1) * gs != K) {
    NOT_PLAIN;
  }
  const int64_t M = x->numel() / K;
  if (!fits_int(M) || !fits_int(N) || !fits_int(K)) {
    NOT_PLAIN;
  }
  at::Tensor out = new_tensor(with_last(*x, N), x->scalar_type(), device);
  const size_t need = abi.fp_qqmm_workspace_size(M, N, K, mode, code);
  const Workspace ws(need < 256 ? 256 : need, device);
  void* stream = stream_of(device);
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS;
  rc = abi.fp_qqmm(
      x->data_ptr(), static_cast<const uint32_t*>(w->data_ptr()),
      static_cast<const uint8_t*>(scales->data_ptr()), out.data_ptr(), M, N, K, mode, code,
      ws.ptr(), need, stream);
  Py_END_ALLOW_THREADS;
  if (rc != MLXROCM_OK) {
    NOT_PLAIN;
  }
  return wrap(std::move(out));
  FAST_CATCH
}

// quantize(w, group_size, bits, mode)
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!bound || n != 4) {
    NOT_PLAIN;
  }
  FAST_TRY
  const c10::DeviceIndex device = device_of(args[0]);
  if (device < 0) {
    NOT_PLAIN;
  }
  const at::Tensor* w = tensor_of(args[0], device);
  const int mode = mode_of(args[3]);
  int gs = 0;
  int bits = 0;
  if (w == nullptr || w->dim() < 2 || mode == kNoMode ||
      !params_of(mode, args[1], args[2], &gs, &bits)) {
    NOT_PLAIN;
  }
  const int code = dtype_code(w->scalar_type());
  const int64_t K = w->size(-1);
  if (code < 0 || K % gs != 0) {
    NOT_PLAIN;
  }
  at::Tensor wq = new_tensor(with_last(*w, K * bits / 32), at::kUInt32, device);
  at::Tensor scales = new_tensor(
      with_last(*w, K / gs), mode == kAffine ? w->scalar_type() : at::kByte, device);
  at::Tensor biases;
  if (mode == kAffine) {
    biases = new_tensor(scales.sizes(), w->scalar_type(), device);
  }
  void* stream = stream_of(device);
  const size_t elements = static_cast<size_t>(w->numel());
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS;
  if (mode == kAffine) {
    rc = abi.affine_quantize(
        w->data_ptr(), static_cast<uint32_t*>(wq.data_ptr()), scales.data_ptr(),
        biases.data_ptr(), elements, gs, bits, code, stream);
  } else {
    rc = abi.fp_quantize(
        w->data_ptr(), static_cast<uint32_t*>(wq.data_ptr()),
        static_cast<uint8_t*>(scales.data_ptr()), elements, mode, code, stream);
  }
  Py_END_ALLOW_THREADS;
  if (rc != MLXROCM_OK) {
    NOT_PLAIN;
  }
  PyObject* out = PyTuple_New(mode == kAffine ? 3 : 2);
  if (out == nullptr) {
    return nullptr;
  }
  PyTuple_SET_ITEM(out, 0, wrap(std::move(wq)));
  PyTuple_SET_ITEM(out, 1, wrap(std::move(scales)));
  if (mode == kAffine) {
    PyTuple_SET_ITEM(out, 2, wrap(std::move(biases)));
  }
  return out;
  FAST_CATCH
}

// dequantize(w, scales, biases, group_size, bits, mode, dtype); dtype None or the
// type the result has anyway (bfloat16 where None in a floating-point mode)
PyObject* dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!bound || n != 7) {
    NOT_PLAIN;
  }
  FAST_TRY
  const c10::DeviceIndex device = device_of(args[0]);
  if (device < 0) {
    NOT_PLAIN;
  }
  const at::Tensor* w = tensor_of(args[0], device);
  const at::Tensor* scales = tensor_of(args[1], device);
  const int mode = mode_of(args[5]);
  int gs = 0;
  int bits = 0;
  if (w == nullptr || scales == nullptr || w->dim() < 2 || w->dim() != scales->dim() ||
      w->scalar_type() != at::kUInt32 || mode == kNoMode ||
      !params_of(mode, args[3], args[4], &gs, &bits)) {
    NOT_PLAIN;
  }
  at::ScalarType type = mode == kAffine ? scales->scalar_type() : at::kBFloat16;
  if (args[6] != Py_None) {
    if (!THPDtype_Check(args[6])) {
      NOT_PLAIN;
    }
    const at::ScalarType asked = reinterpret_cast<THPDtype*>(args[6])->scalar_type;
    if (mode == kAffine && asked != type) {
      NOT_PLAIN;
    }
    type = asked;
  }
  const int code = dtype_code(type);
  const int64_t K = w->size(-1) * 32 / bits;
  const auto lead = [](const at::Tensor& t) { return t.sizes().slice(0, t.dim() - 1); };
  if (code < 0 || scales->size(-1) * gs != K || w->size(-1) * 32 != K * bits ||
      lead(*w) != lead(*scales)) {
    NOT_PLAIN;
  }
  const at::Tensor* biases = nullptr;
  if (mode == kAffine) {
    biases = tensor_of(args[2], device);
    if (biases == nullptr || biases->scalar_type() != scales->scalar_type() ||
        biases->sizes() != scales->sizes()) {
      NOT_PLAIN;
    }
  } else if (args[2] != Py_None || scales->scalar_type() != at::kByte) {
    NOT_PLAIN;
  }
  at::Tensor out = new_tensor(with_last(*w, K), type, device);
  void* stream = stream_of(device);
  const size_t elements = static_cast<size_t>(out.numel());
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS;
  if (mode == kAffine) {
    rc = abi.affine_dequantize(
        static_cast<const uint32_t*>(w->data_ptr()), scales->data_ptr(), biases->data_ptr(),
        out.data_ptr(), elements, gs, bits, code, stream);
  } else {
    rc = abi.fp_dequantize(
        static_cast<const uint32_t*>(w->data_ptr()),
        static_cast<const uint8_t*>(scales->data_ptr()), out.data_ptr(), elements, mode, code,
        stream);
  }
  Py_END_ALLOW_THREADS;
  if (rc != MLXROCM_OK) {
    NOT_PLAIN;
  }
  return wrap(std::move(out));
  FAST_CATCH
}

// ---- attention (attention.py) ------------------------------------------------------

// Whether kernels take a tensor of four dimensions as it is: rows along the last one dense and
// aligned to 16 bytes
bool dense_rows(const at::Tensor& t) {
  const int64_t unit = 16 / static_cast<int64_t>(t.element_size());
  for (int i = 0; i < 3; ++i) {
    if (t.size(i) != 1 && t.stride(i) % unit != 0) {
      return false;
    }
  }
  return t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// Such a tensor on `device`, with no gradient to be recorded (or `recorded`) and no tangent.
const at::Tensor* heads_of(PyObject* o, c10::DeviceIndex device, bool recorded = false) {
  if (!THPVariable_CheckExact(o)) {
    return nullptr;
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && t.device().index() == device && t.dim() == 4 &&
          t.numel() != 0 && !t.is_conj() && !t.is_neg() && (recorded || !records_grad(t)) &&
          !t._fw_grad(0).defined() && dtype_code(t.scalar_type()) >= 0 && dense_rows(t)
      ? &t
      : nullptr;
}

// int32, dense rows
const at::Tensor* indices_of(PyObject* o, c10::DeviceIndex device, int64_t dims, int64_t rows) {
  if (!THPVariable_CheckExact(o)) {
    return nullptr;
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && t.device().index() == device && t.dim() == dims &&
          t.scalar_type() == at::kInt && t.numel() > 0 && t.size(0) == rows &&
          (dims == 1 ? t.is_contiguous() : t.stride(1) == 1)
      ? &t
      : nullptr;
}

// What a query sees: scale, a float, window, a positive int or None, keep, an int
struct Sight {
  double scale;
  int window, keep;
};
bool sight_of(PyObject* scale, PyObject* window, PyObject* keep, Sight* s) {
  constexpr int kMost = 1 << 30;
  const auto whole = [](PyObject* o, int least, int* v) {
    if (!PyLong_CheckExact(o)) {
      return false;
    }
    int overflow = 0;
    const long x = PyLong_AsLongAndOverflow(o, &overflow);
    if (overflow != 0 || x < least) {
      return false;
    }
    *v = x < kMost ? static_cast<int>(x) : kMost;
    return true;
  };
  if (!PyFloat_CheckExact(scale)) {
    return false;
  }
  s->scale = PyFloat_AS_DOUBLE(scale);
  s->window = kMost;
  return std::isfinite(static_cast<float>(s->scale)) &&
      (window == Py_None || whole(window, 1, &s->window)) && whole(keep, 0, &s->keep);
}

// Of the first three dimensions, in elements; 0 where there is one element
void strides_of(const at::Tensor& t, int64_t* to) {
  for (int i = 0; i < 3; ++i) {
    to[i] = t.size(i) == 1 ? 0 : t.stride(i);
  }
}

// A new tensor with q's sizes and memory order, if q is dense
bool like(const at::Tensor& q, c10::DeviceIndex device, at::Tensor* out) {
  if (!q.is_non_overlapping_and_dense()) {
    return false;
  }
  *out = at::Tensor(at::detail::empty_strided_cuda(
      q.sizes(), q.strides(), q.scalar_type(), c10::Device(c10::DeviceType::CUDA, device)));
  return true;
}

bool attends(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
  const int64_t D = q.size(3);
  return k.sizes() == v.sizes() && k.scalar_type() == q.scalar_type() &&
      v.scalar_type() == q.scalar_type() && k.size(3) == D && D % 8 == 0 && D <= 256 &&
      q.size(1) % k.size(1) == 0;
}

// The arguments of window_attention
struct WindowCall {
  const at::Tensor *q, *k, *v, *lengths; // lengths: may be null
  Sight sight;
  int size[6]; // B, Hq, Hkv, Lq, Lk, D
  int code;

  // (of tensors that are known to fit)
  WindowCall(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_,
             const at::Tensor* lengths_, const Sight& sight_)
      : q(&q_), k(&k_), v(&v_), lengths(lengths_), sight(sight_) {
    set_sizes();
  }

  // window_attention(q, k, v, scale, window, keep, lengths), lengths a tensor or None
  bool plain = false;
  WindowCall(PyObject* const* args, Py_ssize_t n, bool recorded) {
    const c10::DeviceIndex device = bound && n == 7 ? device_of(args[0]) : -1;
    if (device < 0 || !sight_of(args[3], args[4], args[5], &sight)) {
      return;
    }
    q = heads_of(args[0], device, recorded);
    k = heads_of(args[1], device, recorded);
    v = heads_of(args[2], device, recorded);
    if (q == nullptr || k == nullptr || v == nullptr || !attends(*q, *k, *v) ||
        k->size(0) != q->size(0)) {
      return;
    }
    lengths = nullptr;
    if (args[6] != Py_None) {
      lengths = indices_of(args[6], device, 1, q->size(0));
      if (lengths == nullptr) {
        return;
      }
    }
    for (int i = 0; i < 4; ++i) {
      if (!fits_int(q->size(i)) || !fits_int(k->size(i))) {
        return;
      }
    }
    set_sizes();
    plain = true;
  }

  void set_sizes() {
    const int64_t sizes[] = {q->size(0), q->size(1), k->size(1), q->size(2), k->size(2),
                             q->size(3)};
    for (int i = 0; i < 6; ++i) {
      size[i] = static_cast<int>(sizes[i]);
    }
    code = dtype_code(q->scalar_type());
  }
  c10::DeviceIndex device() const { return q->device().index(); }
  const int32_t* lengths_ptr() const {
    return lengths == nullptr ? nullptr : static_cast<const int32_t*>(lengths->data_ptr());
  }

  // The result, and what its gradients need if `lse` is given; undefined if it cannot be
  at::Tensor run(at::Tensor* lse) const {
    at::Tensor out;
    if (!like(*q, device(), &out)) { // (a slice of something wider: dense, in its order)
      const at::AutoGradMode off(false);
      out = at::empty_like(*q);
    }
    if (lse != nullptr) {
      *lse = new_tensor(
          {static_cast<int64_t>(abi.window_lse_size(
              size[0], size[1], size[2], size[3], size[4], size[5], sight.window, sight.keep,
              code))},
          at::kByte, device());
    }
    int64_t strides[12];
    strides_of(*q, strides);
    strides_of(*k, strides + 3);
    strides_of(*v, strides + 6);
    strides_of(out, strides + 9);
    const Workspace ws(
        abi.window_workspace_size(
            size[0], size[1], size[2], size[3], size[4], size[5], sight.window, sight.keep, code),
        device());
    const int rc = abi.window_attention(
        q->data_ptr(), k->data_ptr(), v->data_ptr(), out.data_ptr(),
        lse == nullptr ? nullptr : static_cast<float*>(lse->data_ptr()), lengths_ptr(), size[0],
        size[1], size[2], size[3], size[4], size[5], strides, static_cast<float>(sight.scale),
        sight.window, sight.keep, code, ws.ptr(), ws.bytes, stream_of(device()));
    return rc == MLXROCM_OK ? out : at::Tensor();
  }
};

struct WithoutGil { // (also where an exception leaves the block)
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};

PyObject* window_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  FAST_TRY
  const WindowCall call(args, n, false);
  if (!call.plain) {
    NOT_PLAIN;
  }
  at::Tensor out;
  {
    const WithoutGil free;
    out = call.run(nullptr);
  }
  if (!out.defined()) {
    NOT_PLAIN;
  }
  return wrap(std::move(out));
  FAST_CATCH
}

// The same where gradients are to be recorded: a node of torch's graph.  A small call, forward and
// backward, 36 us; by a node in Python 81.
struct WindowVjp : torch::autograd::Function<WindowVjp> {
  struct NotPlain {};

  static at::Tensor forward(
      torch::autograd::AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k,
      const at::Tensor& v, const at::Tensor* lengths, double scale, int64_t window, int64_t keep) {
    const Sight sight = {scale, static_cast<int>(window), static_cast<int>(keep)};
    at::Tensor lse;
    at::Tensor out = WindowCall(q, k, v, lengths, sight).run(&lse);
    if (!out.defined()) {
      throw NotPlain();
    }
    ctx->save_for_backward({q, k, v, out, lse, lengths == nullptr ? at::Tensor() : *lengths});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["window"] = window;
    ctx->saved_data["keep"] = keep;
    return out;
  }

  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3];
    const Sight sight = {
        ctx->saved_data["scale"].toDouble(), static_cast<int>(ctx->saved_data["window"].toInt()),
        static_cast<int>(ctx->saved_data["keep"].toInt())};
    const WindowCall call(q, k, v, saved[5].defined() ? &saved[5] : nullptr, sight);
    void* stream = stream_of(call.device());
    at::Tensor dout = grads[0];
    TORCH_CHECK(dtype_code(dout.scalar_type()) == call.code, "[window_attention] gradient of type ",
                dout.scalar_type(), " for a result of type ", q.scalar_type());
    if (!dense_rows(dout)) {
      at::Tensor copy = new_tensor(dout.sizes(), dout.scalar_type(), call.device());
      check(abi.copy_strided(
          dout.data_ptr(), call.code, dout.strides().data(), copy.data_ptr(), call.code, nullptr,
          4, dout.sizes().data(), stream));
      dout = copy;
    }
    torch::autograd::variable_list to;
    {
      const at::AutoGradMode off(false);
      to = {at::empty_like(q), at::empty_like(k), at::empty_like(v)};
    }
    int64_t strides[24];
    const at::Tensor* operands[] = {&q, &k, &v, &out, &dout, &to[0], &to[1], &to[2]};
    for (int i = 0; i < 8; ++i) {
      strides_of(*operands[i], strides + 3 * i);
    }
    const int* n = call.size;
    const Workspace ws(
        abi.vjp_workspace_size(
            n[0], n[1], n[2], n[3], n[4], n[5], sight.window, sight.keep, call.code),
        call.device());
    check(abi.window_vjp(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
        static_cast<const float*>(saved[4].data_ptr()), dout.data_ptr(), to[0].data_ptr(),
        to[1].data_ptr(), to[2].data_ptr(), call.lengths_ptr(), n[0], n[1], n[2], n[3], n[4], n[5],
        strides, static_cast<float>(sight.scale), sight.window, sight.keep, call.code, ws.ptr(),
        ws.bytes, stream));
    if (at::GradMode::is_enabled()) { // once differentiable
      for (at::Tensor& t : to) {
        t.set_requires_grad(true);
      }
      torch::autograd::DelayedError error(
          "trying to differentiate twice a function that was marked with @once_differentiable", 3);
      to = error.apply(std::move(to));
    }
    to.resize(7); // (nothing for what is no tensor with a gradient)
    return to;
  }

  static void check(int rc) {
    TORCH_CHECK(rc == MLXROCM_OK, abi.last_error());
  }
};

PyObject* window_attention_recorded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  FAST_TRY
  const WindowCall call(args, n, true);
  if (!call.plain || !(records_grad(*call.q) || records_grad(*call.k) || records_grad(*call.v))) {
    NOT_PLAIN;
  }
  return wrap(WindowVjp::apply(
      *call.q, *call.k, *call.v, call.lengths, call.sight.scale,
      static_cast<int64_t>(call.sight.window), static_cast<int64_t>(call.sight.keep)));
  } catch (const WindowVjp::NotPlain&) {
    Py_RETURN_NONE;
  FAST_CATCH
}

// The pages of a cache and where a batch's sequences lie in them
struct Cache {
  const at::Tensor *k, *v, *table, *lengths;
};
bool cache_of(
    PyObject* const* args, c10::DeviceIndex device, int64_t batch, at::ScalarType type, Cache* c) {
  c->k = heads_of(args[0], device);
  c->v = heads_of(args[1], device);
  c->table = indices_of(args[2], device, 2, batch);
  c->lengths = indices_of(args[3], device, 1, batch);
  return c->k != nullptr && c->v != nullptr && c->table != nullptr && c->lengths != nullptr &&
      c->k->sizes() == c->v->sizes() && c->k->scalar_type() == type &&
      c->v->scalar_type() == type && c->k->size(2) % 16 == 0 && fits_int(c->k->size(0)) &&
      fits_int(c->k->size(2)) && fits_int(c->table->size(1)) &&
      fits_int(c->table->size(1) * c->k->size(2));
}

// paged_attention(q, k_pages, v_pages, block_table, lengths, scale, window, keep)
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!bound || n != 8) {
    NOT_PLAIN;
  }
  FAST_TRY
  const c10::DeviceIndex device = device_of(args[0]);
  Sight sight;
  if (device < 0 || !sight_of(args[5], args[6], args[7], &sight)) {
    NOT_PLAIN;
  }
  const at::Tensor* q = heads_of(args[0], device);
  Cache c;
  if (q == nullptr || !cache_of(args + 1, device, q->size(0), q->scalar_type(), &c) ||
      !attends(*q, *c.k, *c.v)) {
    NOT_PLAIN;
  }
  const int64_t B = q->size(0), Hq = q->size(1), Hkv = c.k->size(1), Lq = q->size(2);
  const int64_t D = q->size(3), page = c.k->size(2), width = c.table->size(1);
  if (!fits_int(B) || !fits_int(Hq) || !fits_int(Lq)) {
    NOT_PLAIN;
  }
  at::Tensor out;
  if (!like(*q, device, &out)) {
    NOT_PLAIN;
  }
  const int code = dtype_code(q->scalar_type());
  int64_t strides[13];
  strides_of(*q, strides);
  strides_of(*c.k, strides + 3);
  strides_of(*c.v, strides + 6);
  strides_of(out, strides + 9);
  strides[12] = c.table->stride(0);
  const Workspace ws(
      abi.paged_workspace_size(
          B, Hq, Hkv, Lq, D, width * page, sight.window, sight.keep, code),
      device);
  void* stream = stream_of(device);
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS;
  rc = abi.paged_attention(
      q->data_ptr(), c.k->data_ptr(), c.v->data_ptr(),
      static_cast<const int32_t*>(c.table->data_ptr()),
      static_cast<const int32_t*>(c.lengths->data_ptr()), out.data_ptr(), B, Hq, Hkv, Lq, D,
      c.k->size(0), page, width, strides, static_cast<float>(sight.scale), sight.window,
      sight.keep, code, ws.ptr(), ws.bytes, stream);
  Py_END_ALLOW_THREADS;
  if (rc != MLXROCM_OK) {
    NOT_PLAIN;
  }
  return wrap(std::move(out));
  FAST_CATCH
}

// paged_cache_update(k, v, k_pages, v_pages, block_table, lengths): True where it was done
PyObject* paged_cache_update(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!bound || n != 6) {
    NOT_PLAIN;
  }
  FAST_TRY
  const c10::DeviceIndex device = device_of(args[0]);
  if (device < 0) {
    NOT_PLAIN;
  }
  const at::Tensor* k = heads_of(args[0], device);
  const at::Tensor* v = heads_of(args[1], device);
  Cache c;
  if (k == nullptr || v == nullptr || k->sizes() != v->sizes() ||
      k->scalar_type() != v->scalar_type() ||
      !cache_of(args + 2, device, k->size(0), k->scalar_type(), &c) ||
      k->size(1) != c.k->size(1) || k->size(3) != c.k->size(3) || !fits_int(k->size(0)) ||
      !fits_int(k->size(2)) || !fits_int(k->size(3))) {
    NOT_PLAIN;
  }
  for (int i = 0; i < 3; ++i) { // (what shares memory is refused there)
    if (c.k->size(i) > 1 && (c.k->stride(i) == 0 || c.v->stride(i) == 0)) {
      NOT_PLAIN;
    }
  }
  int64_t strides[13];
  strides_of(*k, strides);
  strides_of(*v, strides + 3);
  strides_of(*c.k, strides + 6);
  strides_of(*c.v, strides + 9);
  strides[12] = c.table->stride(0);
  void* stream = stream_of(device);
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS;
  rc = abi.paged_cache_update(
      k->data_ptr(), v->data_ptr(), c.k->data_ptr(), c.v->data_ptr(),
      static_cast<const int32_t*>(c.table->data_ptr()),
      static_cast<const int32_t*>(c.lengths->data_ptr()), k->size(0), k->size(1), k->size(2),
      k->size(3), c.k->size(0), c.k->size(2), c.table->size(1), strides,
      dtype_code(k->scalar_type()), stream);
  Py_END_ALLOW_THREADS;
  if (rc != MLXROCM_OK) {
    NOT_PLAIN;
  }
  for (const at::Tensor* pages : {c.k, c.v}) { // written to: a graph that saved them is to know
    if (!pages->is_inference()) {
      pages->unsafeGetTensorImpl()->bump_version();
    }
  }
  Py_RETURN_TRUE;
  FAST_CATCH
}

// verify_draft(draft, target_probs, draft_probs, accept, sample, lengths); draft_probs and lengths
// may be None
PyObject* verify_draft(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!bound || n != 6) {
    NOT_PLAIN;
  }
  FAST_TRY
  const c10::DeviceIndex device = device_of(args[0]);
  if (device < 0) {
    NOT_PLAIN;
  }
  const at::Tensor* draft = matrix_of(args[0], device, at::kInt);
  const at::Tensor* target = tensor_of(args[1], device);
  const at::Tensor* accept = matrix_of(args[3], device, at::kFloat);
  const at::Tensor* sample = tensor_of(args[4], device);
  if (draft == nullptr || target == nullptr || accept == nullptr || sample == nullptr ||
      target->dim() != 3 || accept->sizes() != draft->sizes() || sample->dim() != 1 ||
      sample->scalar_type() != at::kFloat) {
    NOT_PLAIN;
  }
  const int64_t B = draft->size(0), K = draft->size(1), V = target->size(2);
  const int code = dtype_code(target->scalar_type());
  const at::Tensor* probs = nullptr;
  const at::Tensor* lengths = nullptr;
  if (args[2] != Py_None) {
    probs = tensor_of(args[2], device);
    if (probs == nullptr || probs->dim() != 3 || probs->scalar_type() != target->scalar_type() ||
        probs->size(0) != B || probs->size(1) != K || probs->size(2) != V) {
      NOT_PLAIN;
    }
  }
  if (args[5] != Py_None) {
    lengths = indices_of(args[5], device, 1, B);
    if (lengths == nullptr) {
      NOT_PLAIN;
    }
  }
  if (code < 0 || target->size(0) != B || target->size(1) != K + 1 || sample->size(0) != B ||
      !fits_int(B) || !fits_int(K + 1) || !fits_int(V)) {
    NOT_PLAIN;
  }
  at::Tensor tokens = new_tensor({B, K + 1}, at::kInt, device);
  at::Tensor accepted = new_tensor({B}, at::kInt, device);
  const int64_t strides[4] = {(K + 1) * V, V, K * V, V};
  const Workspace ws(abi.verify_workspace_size(B, V), device);
  void* stream = stream_of(device);
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS;
  rc = abi.verify_draft(
      static_cast<const int32_t*>(draft->data_ptr()), target->data_ptr(),
      probs == nullptr ? nullptr : probs->data_ptr(),
      static_cast<const float*>(accept->data_ptr()),
      static_cast<const float*>(sample->data_ptr()),
      lengths == nullptr ? nullptr : static_cast<const int32_t*>(lengths->data_ptr()),
      static_cast<int32_t*>(tokens.data_ptr()), static_cast<int32_t*>(accepted.data_ptr()), B, K,
      V, strides, code, ws.ptr(), ws.bytes, stream);
  Py_END_ALLOW_THREADS;
  if (rc != MLXROCM_OK) {
    NOT_PLAIN;
  }
  PyObject* out = PyTuple_New(2);
  if (out == nullptr) {
    return nullptr;
  }
  PyTuple_SET_ITEM(out, 0, wrap(std::move(tokens)));
  PyTuple_SET_ITEM(out, 1, wrap(std::move(accepted)));
  return out;
  FAST_CATCH
}

#include "decoder_ops.h"

// bind({entry point: address}): the library whose entry points are to be called
PyObject* bind(PyObject*, PyObject* table) {
  if (!PyDict_Check(table)) {
    PyErr_SetString(PyExc_TypeError, "bind() takes a dict of addresses");
    return nullptr;
  }
  const auto take = [&](const char* name, auto& slot) {
    PyObject* v = PyDict_GetItemString(table, name); // borrowed
    if (v == nullptr) {
      PyErr_Format(PyExc_KeyError, "no address for %s", name);
      return false;
    }
    void* p = PyLong_AsVoidPtr(v);
    if (p == nullptr) {
      if (!PyErr_Occurred()) {
        PyErr_Format(PyExc_ValueError, "null address for %s", name);
      }
      return false;
    }
    slot = reinterpret_cast<std::remove_reference_t<decltype(slot)>>(p);
    return true;
  };
  bound = take("mlxrocm_qmm_workspace_size", abi.qmm_workspace_size) &&
      take("mlxrocm_qmm_prepacked", abi.qmm_prepacked) &&
      take("mlxrocm_qmm_sb_image_size", abi.qmm_sb_image_size) &&
      take("mlxrocm_qmm_rows_supported", abi.rows_supported) &&
      take("mlxrocm_qmm_rows_workspace_size", abi.rows_workspace_size) &&
      take("mlxrocm_qmm_rows_prepacked", abi.rows_prepacked) &&
      take("mlxrocm_fp_qmm_workspace_size", abi.fp_qmm_workspace_size) &&
      take("mlxrocm_fp_qmm", abi.fp_qmm) &&
      take("mlxrocm_fp_qmm_rows_supported", abi.fp_rows_supported) &&
      take("mlxrocm_fp_qmm_rows_workspace_size", abi.fp_rows_workspace_size) &&
      take("mlxrocm_fp_qmm_rows", abi.fp_rows) &&
      take("mlxrocm_qmm_swiglu_workspace_size", abi.swiglu_workspace_size) &&
      take("mlxrocm_qmm_swiglu", abi.swiglu) &&
      take("mlxrocm_fp_qqmm_workspace_size", abi.fp_qqmm_workspace_size) &&
      take("mlxrocm_fp_qqmm", abi.fp_qqmm) &&
      take("mlxrocm_switch_glu_workspace_size", abi.switch_glu_workspace_size) &&
      take("mlxrocm_switch_glu", abi.switch_glu) &&
      take("mlxrocm_affine_quantize", abi.affine_quantize) &&
      take("mlxrocm_affine_dequantize", abi.affine_dequantize) &&
      take("mlxrocm_fp_quantize", abi.fp_quantize) &&
      take("mlxrocm_fp_dequantize", abi.fp_dequantize) &&
      take("mlxrocm_window_attention_workspace_size", abi.window_workspace_size) &&
      take("mlxrocm_window_attention_lse_size", abi.window_lse_size) &&
      take("mlxrocm_window_attention", abi.window_attention) &&
      take("mlxrocm_window_attention_vjp_workspace_size", abi.vjp_workspace_size) &&
      take("mlxrocm_window_attention_vjp", abi.window_vjp) &&
      take("mlxrocm_copy_strided", abi.copy_strided) &&
      take("mlxrocm_last_error", abi.last_error) &&
      take("mlxrocm_paged_attention_workspace_size", abi.paged_workspace_size) &&
      take("mlxrocm_paged_attention", abi.paged_attention) &&
      take("mlxrocm_paged_cache_update", abi.paged_cache_update) &&
      take("mlxrocm_verify_draft_workspace_size", abi.verify_workspace_size) &&
      take("mlxrocm_verify_draft", abi.verify_draft) &&
      take("mlxrocm_rope", abi.rope) &&
      take("mlxrocm_rope_cache_update", abi.rope_cache_update) &&
      take("mlxrocm_route_experts", abi.route_experts) &&
      take("mlxrocm_route_experts_vjp", abi.route_experts_vjp) &&
      take("mlxrocm_adapter_matmul_workspace_size", abi.adapter_workspace_size) &&
      take("mlxrocm_adapter_matmul_h_size", abi.adapter_h_size) &&
      take("mlxrocm_adapter_matmul", abi.adapter_matmul) &&
      take("mlxrocm_adapter_matmul_vjp_workspace_size", abi.adapter_vjp_workspace_size) &&
      take("mlxrocm_adapter_matmul_vjp", abi.adapter_vjp);
  if (!bound) {
    return nullptr;
  }
  Py_RETURN_NONE;
}

#define FASTCALL(f) \
  {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    FASTCALL(quantized_matmul),
    FASTCALL(quantized_swiglu),
    FASTCALL(switch_glu),
    FASTCALL(qqmm),
    FASTCALL(quantize),
    FASTCALL(dequantize),
    FASTCALL(window_attention),
    FASTCALL(window_attention_recorded),
    FASTCALL(paged_attention),
    FASTCALL(paged_cache_update),
    FASTCALL(verify_draft),
    FASTCALL(rope),
    FASTCALL(rope_cache_update),
    FASTCALL(route_experts),
    FASTCALL(adapter_matmul),
    {"bind", bind, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {
    PyModuleDef_HEAD_INIT, "fast_ops", "The operators' host path for plain calls.", -1, methods,
    nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit_fast_ops(void) {
  return PyModule_Create(&module);
}
