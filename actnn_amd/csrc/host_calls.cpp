// The host side of the calls a training step makes most often: allocation of the results, the generator's
// (seed, offset), the current stream and the call into the kernels' C library, in one native function each
// instead of a dozen calls out of Python.  A module of its own beside the C library (which knows no tensors): what it
// allocates, draws and launches is what the Python functions of cpp_extension document, and those still check the
// arguments that users hand in.
//
// What it is for: calls of a few microseconds, where Python was slower than the GPU.  compress + restore of bf16
// [32, 64, 56, 56] took 47.7 us, of them 26 us of kernels and the rest host time behind them (eight torch.empty, two calls of 11
// and 22 converted arguments, checks); 34.8 now, QDropout's two passes over bf16 [128, 4096] 86.6 and 62.9.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/Context.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/actnn_hip.h"

namespace {

using at::Tensor;

// ---------------------------------------------------------------------------- arguments
struct Args {
  PyObject* const* at;
  Py_ssize_t n, i = 0;
  Args(PyObject* const* a, Py_ssize_t count, Py_ssize_t want) : at(a), n(count) {
    TORCH_CHECK(count == want, "expected ", want, " arguments, got ", count);
  }
  PyObject* tensor_object() {
    PyObject* o = at[i++];
    TORCH_CHECK_TYPE(THPVariable_Check(o), "argument ", i, " must be a tensor");
    return o;
  }
  const Tensor& tensor() { return THPVariable_Unpack(tensor_object()); }
  // whether the next `count` arguments are tensors
  bool tensors(int count) const {
    for (int k = 0; k < count; ++k)
      if (!THPVariable_Check(at[i + k])) return false;
    return true;
  }
  // (an undefined tensor for None)
  Tensor optional() { return at[i] == Py_None ? (++i, Tensor()) : tensor(); }
  int64_t integer() {
    const int64_t v = PyLong_AsLongLong(at[i++]);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
  }
  double number() {
    const double v = PyFloat_AsDouble(at[i++]);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
  }
  bool flag() {
    const int v = PyObject_IsTrue(at[i++]);
    if (v < 0) throw python_error();
    return v != 0;
  }
};

PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
template <typename... Ts> PyObject* tuple_of(const Ts&... ts) {
  PyObject* out = PyTuple_New(sizeof...(ts));
  if (!out) throw python_error();
  Py_ssize_t i = 0;
  auto put = [&](const Tensor& t) {
    PyObject* o = wrap(t);
    if (!o) {
      Py_DECREF(out);
      throw python_error();
    }
    PyTuple_SET_ITEM(out, i++, o);
  };
  (put(ts), ...);
  return out;
}

// ---------------------------------------------------------------------------- plumbing
int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return ACTNN_F32;
    case at::kHalf: return ACTNN_F16;
    case at::kBFloat16: return ACTNN_BF16;
    default: TORCH_CHECK(false, "unsupported dtype ", t);
  }
}
at::ScalarType type_of(int64_t code) {
  TORCH_CHECK(code >= ACTNN_F32 && code <= ACTNN_BF16, "unknown dtype code ", code);
  return code == ACTNN_F32 ? at::kFloat : code == ACTNN_F16 ? at::kHalf : at::kBFloat16;
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* f32(const Tensor& t) { return static_cast<float*>(ptr(t)); }
int32_t* i32(const Tensor& t) { return static_cast<int32_t*>(ptr(t)); }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
// Runs a call into the C library without the interpreter's lock (a launch may wait for room in its queue).
template <typename F> void launch(const char* what, F f) {
  int rc;
  {
    struct Unlocked {
      PyThreadState* state = PyEval_SaveThread();
      ~Unlocked() { PyEval_RestoreThread(state); }
    } unlocked;
    rc = f();
  }
  TORCH_CHECK(rc == ACTNN_OK, what, " failed: ", actnn_strerror(rc), " (code ", rc, ")");
}
Tensor empty(at::IntArrayRef size, const Tensor& like, at::ScalarType dtype) {
  return at::empty(size, at::TensorOptions().dtype(dtype).device(like.device()));
}

// A tensor argument with the Python object it came as.  What makes a new tensor of it goes through Python where its class may
// have a say, and the object goes along with the tensor: the next step works on the same one the kernel reads or writes.
class Given {
 public:
  explicit Given(PyObject* o) : object_(o), tensor_(THPVariable_Unpack(o)) { Py_INCREF(object_); }
  Given(const Given&) = delete;
  Given& operator=(const Given&) = delete;
  ~Given() { Py_DECREF(object_); }
  const Tensor& tensor() const { return tensor_; }
  void make_contiguous() {
    if (plain()) tensor_ = tensor_.contiguous();
    else replace(PyObject_CallMethod(object_, "contiguous", nullptr));
  }
  // (the kernels use 16-byte accesses; only views with a storage offset are not aligned)
  void make_aligned() {
    if (reinterpret_cast<uintptr_t>(tensor_.data_ptr()) % 16 == 0) return;
    if (plain()) tensor_ = tensor_.clone();
    else replace(PyObject_CallMethod(object_, "clone", nullptr));
  }
  Tensor empty_like() const {
    if (plain()) return at::empty_like(tensor_);
    PyObject* torch = PyImport_ImportModule("torch");
    if (!torch) throw python_error();
    PyObject* made = PyObject_CallMethod(torch, "empty_like", "O", object_);
    Py_DECREF(torch);
    const Tensor out = unpacked(made);
    Py_DECREF(made);
    return out;
  }

 private:
  // (a plain object_ stays when its tensor is replaced: only its class counts)
  bool plain() const { return THPVariable_CheckExact(object_); }
  static Tensor unpacked(PyObject* made) {
    if (!made) throw python_error();
    if (!THPVariable_Check(made)) {
      Py_DECREF(made);
      TORCH_CHECK_TYPE(false, "a tensor's class made something that is no tensor");
    }
    return THPVariable_Unpack(made);
  }
  void replace(PyObject* made) {
    tensor_ = unpacked(made);
    Py_DECREF(object_);
    object_ = made;
  }
  PyObject* object_;
  Tensor tensor_;
};

// (seed, offset) of the device's default generator, advancing the offset by 4 under its lock
struct Draw {
  uint64_t seed, offset;
  explicit Draw(const Tensor& t) {
    at::Generator gen = at::globalContext().defaultGenerator(t.device());
    std::lock_guard<std::mutex> lock(gen.mutex());
    seed = gen.current_seed();
    offset = gen.get_offset();
    gen.set_offset(offset + 4);
  }
};

// the sensitivity's multiplier: nothing, one device scalar or one fp32 value per sample on the same device
struct Mult {
  Tensor held;
  int per_sample = 0;
  Mult(Tensor mult, int64_t N, const Tensor& like) {
    if (!mult.defined()) return;
    TORCH_CHECK(mult.scalar_type() == at::kFloat && mult.device() == like.device() && (mult.numel() == 1 || mult.numel() == N),
                "the sensitivity's multiplier must be fp32 on the same device with 1 or N values");
    held = mult.contiguous();
    per_sample = mult.numel() == N && N != 1;
  }
};

constexpr int64_t kMaskBlock = 512;
int64_t mask_words(int64_t n) { return (n + kMaskBlock - 1) / kMaskBlock * 16; }
int64_t single_packed_bytes(int64_t N, int64_t G, int64_t bits) {
  const int64_t per = 8 / bits, rounded = (N + per - 1) / per * per;
  return (bits * rounded * G * 256 + 8) / 8;
}

// ---------------------------------------------------------------------------- compress / restore
// rows, N, mn | None, mx | None, factor, mult | None, initial, target, total, sens | None, stored dtype
//   -> packed, bits, scale, stored minimum, prefix
PyObject* quantize_rows(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 11);
  const Tensor rows = args.tensor();
  const int64_t N = args.integer();
  Tensor mn = args.optional(), mx = args.optional();
  const double factor = args.number();
  const Mult mult(args.optional(), N, rows);
  const int64_t initial = args.integer(), target = args.integer(), total = args.integer();
  Tensor sens = args.optional();
  const auto dtype = rows.scalar_type();
  const auto store = type_of(args.integer());
  TORCH_CHECK(N > 0 && total >= 0, "quantize_rows: no samples");
  const int64_t F = rows.numel() / N, G = (F + 255) / 256;
  const bool known = mn.defined();
  const c10::DeviceGuard guard(rows.device());
  if (!known) {
    mn = empty({N * G}, rows, dtype);
    mx = empty({N * G}, rows, dtype);
  }
  const Tensor stored = store == dtype ? mn : empty({N * G}, rows, store);
  if (!sens.defined()) sens = empty({N}, rows, at::kFloat);
  const Tensor bits = empty({N}, rows, at::kInt), prefix = empty({N + 1}, rows, at::kInt);
  const Tensor packed = empty({total * G * 8}, rows, at::kInt), scale = empty({N, G, 1}, rows, store);
  const Draw draw(rows);
  launch("quantize_activation", [&] {
      return actnn_quantize_rows(ptr(rows), ptr(mn), ptr(mx), known, (float)factor, f32(mult.held), mult.per_sample, f32(sens),
                           i32(bits), i32(prefix), (int)initial, target, ptr(scale), ptr(stored), i32(packed), draw.seed,
                           draw.offset, N, F, code_of(dtype), code_of(store), stream_of(rows));
  });
  return tuple_of(packed, bits, scale, stored, prefix);
}

// rows [N, F], width, mn | None, mx | None (of whole groups), stored dtype -> packed, scale, minimum
PyObject* quantize_rows_fixed(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 5);
  const Tensor rows = args.tensor();
  const int64_t bits = args.integer();
  const Tensor known_mn = args.optional(), known_mx = args.optional();
  const auto dtype = rows.scalar_type();
  const auto store = type_of(args.integer());
  TORCH_CHECK(rows.dim() == 2, "quantize_rows_fixed: rows must have two dimensions, got ", rows.dim());
  TORCH_CHECK(bits >= 1 && bits <= 8 && 8 % bits == 0, "quantize_rows_fixed: 8 % bits must be 0, got ", bits);
  const int64_t N = rows.size(0), F = rows.size(1), G = (F + 255) / 256;
  const c10::DeviceGuard guard(rows.device());
  const Tensor packed = empty({single_packed_bytes(N, G, bits)}, rows, at::kChar), scale = empty({N, G, 1}, rows, store);
  const bool keeps = known_mn.defined() && store == known_mn.scalar_type();       // the given minimum is what is stored
  const Tensor mn = keeps ? known_mn.view({N, G, 1}) : empty({N, G, 1}, rows, store);
  const Draw draw(rows);
  launch("quantize_fixed", [&] {
      return actnn_quantize_fixed(ptr(rows), ptr(known_mn), ptr(known_mx), (int)bits, ptr(scale), keeps ? nullptr : ptr(mn),
                            static_cast<int8_t*>(ptr(packed)), draw.seed, draw.offset, N, F, code_of(dtype), code_of(store),
                            stream_of(rows));
  });
  return tuple_of(packed, scale, mn);
}

bool holds(const Tensor& t, at::ScalarType dtype, int64_t dim) {
  return t.is_cuda() && t.is_contiguous() && t.dim() == dim && t.scalar_type() == dtype;
}
bool holds_float(const Tensor& t, int64_t dim) {
  return t.is_cuda() && t.is_contiguous() && t.dim() == dim &&
         (t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16);
}

// packed, bits, prefix, sum of the widths, scale, mn, N, F, dtype -> [N, F], or None for arguments that do not fit
// together (the caller's own checks then say which)
PyObject* unpack_rows_mixed(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 9);
  if (!args.tensors(3) || !THPVariable_Check(a[4]) || !THPVariable_Check(a[5])) Py_RETURN_NONE;
  const Tensor packed = args.tensor(), bits = args.tensor(), prefix = args.tensor();
  const int64_t total = args.integer();
  const Tensor scale = args.tensor(), mn = args.tensor();
  const int64_t N = args.integer(), F = args.integer(), G = (F + 255) / 256;
  const auto dtype = type_of(args.integer());
  if (!(holds(packed, at::kInt, 1) && holds(bits, at::kInt, 1) && holds_float(scale, 3) && holds_float(mn, 3) &&
        mn.scalar_type() == scale.scalar_type() && scale.numel() == N * G && mn.numel() == N * G && bits.numel() == N &&
        packed.numel() >= total * G * 8))
    Py_RETURN_NONE;
  const c10::DeviceGuard guard(packed.device());
  const Tensor out = empty({N, F}, packed, dtype);
  launch("unpack_mixed_precision", [&] {
      return actnn_unpack_mixed_rows(i32(packed), i32(bits), i32(prefix), ptr(scale), ptr(mn), ptr(out), N, F, code_of(dtype),
                               code_of(scale.scalar_type()), stream_of(packed));
  });
  return wrap(out);
}

// packed, width, scale, mn, N, F, dtype -> [N, F], or None as above
PyObject* unpack_rows_fixed(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 7);
  if (!args.tensors(1) || !THPVariable_Check(a[2]) || !THPVariable_Check(a[3])) Py_RETURN_NONE;
  const Tensor packed = args.tensor();
  const int64_t bits = args.integer();
  const Tensor scale = args.tensor(), mn = args.tensor();
  const int64_t N = args.integer(), F = args.integer(), G = (F + 255) / 256;
  const auto dtype = type_of(args.integer());
  if (!(bits >= 1 && bits <= 8 && 8 % bits == 0 && holds(packed, at::kChar, 1) && holds_float(scale, 3) && holds_float(mn, 3) &&
        mn.scalar_type() == scale.scalar_type() && scale.numel() == N * G && mn.numel() == N * G &&
        packed.numel() >= single_packed_bytes(N, G, bits) - 1))
    Py_RETURN_NONE;
  const c10::DeviceGuard guard(packed.device());
  const Tensor out = empty({N, F}, packed, dtype);
  launch("unpack_single_precision", [&] {
      return actnn_unpack_single_rows(static_cast<int8_t*>(ptr(packed)), (int)bits, ptr(scale), ptr(mn), ptr(out), N, F, code_of(dtype),
                                code_of(scale.scalar_type()), stream_of(packed));
  });
  return wrap(out);
}

// ---------------------------------------------------------------------------- masks
// x -> relu(x), mask;  x, p -> dropout(x), mask
PyObject* mask_forward(Args& args, bool dropout) {
  Given given(args.tensor_object());
  given.make_aligned();
  const Tensor& x = given.tensor();
  TORCH_CHECK(x.is_cuda(), "input must be a CUDA tensor!");
  const double p = dropout ? args.number() : 0.0;
  const int64_t count = x.numel();
  const c10::DeviceGuard guard(x.device());
  const Tensor y = given.empty_like(), mask = empty({mask_words(count)}, x, at::kInt);
  const int code = code_of(x.scalar_type());
  if (dropout) {
    const Draw draw(x);
    launch("dropout_forward", [&] {
      return actnn_dropout_forward(ptr(x), ptr(y), i32(mask), count, (float)p, draw.seed, draw.offset, code, stream_of(x));
  });
  } else {
    launch("relu_forward", [&] {
      return actnn_relu_forward(ptr(x), ptr(y), i32(mask), count, code, stream_of(x));
  });
  }
  return tuple_of(y, mask);
}
PyObject* relu_forward(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 1);
  return mask_forward(args, false);
}
PyObject* dropout_forward(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 2);
  return mask_forward(args, true);
}

// grad, mask[, p] -> gradient of the input
PyObject* mask_backward(Args& args, bool dropout) {
  Given given(args.tensor_object());
  given.make_contiguous();                             // (the order the kernel reads and writes in: before the result is made)
  given.make_aligned();
  const Tensor& grad = given.tensor();
  const Tensor mask = args.tensor();
  TORCH_CHECK(grad.is_cuda() && mask.is_cuda(), "grad_output must be a CUDA tensor!");
  const double p = dropout ? args.number() : 0.0;
  const c10::DeviceGuard guard(grad.device());
  const Tensor out = given.empty_like();
  const int code = code_of(grad.scalar_type());
  if (dropout)
    launch("dropout_backward", [&] {
      return actnn_dropout_backward(ptr(grad), i32(mask), ptr(out), out.numel(), (float)p, code, stream_of(grad));
  });
  else
    launch("relu_backward", [&] {
      return actnn_relu_backward(ptr(grad), i32(mask), ptr(out), out.numel(), code, stream_of(grad));
  });
  return wrap(out);
}
PyObject* relu_backward(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 2);
  return mask_backward(args, false);
}
PyObject* dropout_backward(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 3);
  return mask_backward(args, true);
}

// ---------------------------------------------------------------------------- batch norm
// x[, parameters] -> (N, C, HW, channels last) of a dense tensor the batch-norm kernels take, or None.  With parameters (None
// or tensors): None as well unless x is 16-byte aligned and each of them dense fp32 on a GPU.
PyObject* batch_norm_geometry(PyObject* const* a, Py_ssize_t n) {
  TORCH_CHECK(n >= 1, "expected a tensor");
  if (!THPVariable_Check(a[0])) Py_RETURN_NONE;
  const Tensor& x = THPVariable_Unpack(a[0]);
  const auto dtype = x.scalar_type();
  if (!x.is_cuda() || x.dim() < 2 || (dtype != at::kFloat && dtype != at::kHalf && dtype != at::kBFloat16)) Py_RETURN_NONE;
  const bool dense = x.is_contiguous();
  const bool cl = !dense && ((x.dim() == 4 && x.is_contiguous(at::MemoryFormat::ChannelsLast)) ||
                             (x.dim() == 5 && x.is_contiguous(at::MemoryFormat::ChannelsLast3d)));
  if (!dense && !cl) Py_RETURN_NONE;
  const int64_t N = x.size(0), C = x.size(1);
  int64_t HW = 1;
  for (int64_t d = 2; d < x.dim(); ++d) HW *= x.size(d);
  if (N * C * HW == 0 || actnn_batch_norm_workspace_bytes(N, C, HW, code_of(dtype), cl) < 0) Py_RETURN_NONE;
  if (n > 1 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0) Py_RETURN_NONE;
  for (Py_ssize_t i = 1; i < n; ++i) {
    if (a[i] == Py_None) continue;
    if (!THPVariable_Check(a[i])) Py_RETURN_NONE;
    const Tensor& t = THPVariable_Unpack(a[i]);
    if (t.scalar_type() != at::kFloat || !t.is_cuda() || !t.is_contiguous()) Py_RETURN_NONE;
  }
  return Py_BuildValue("(LLLO)", (long long)N, (long long)C, (long long)HW, cl ? Py_True : Py_False);
}

struct BnGeometry {
  int64_t N, C, HW;
  int code, channels_last;
  BnGeometry(Args& args, const Tensor& x) {
    N = args.integer();
    C = args.integer();
    HW = args.integer();
    channels_last = args.flag();
    code = code_of(x.scalar_type());
  }
  int64_t workspace() const { return actnn_batch_norm_workspace_bytes(N, C, HW, code, channels_last); }
  int64_t sumsq_entries() const { return actnn_batch_norm_backward_sumsq_entries(N, C, HW, code, channels_last); }
};

// x, N, C, HW, channels last, weight, bias, running mean, running variance (None or fp32), momentum, eps, factor,
// mult | None, initial, target, total, sens | None, relu, residual | None
//   -> y, mean, invstd, mn, mx, bits, packed, scale, prefix, mask, mn of y, mx of y (the last three None without relu)
PyObject* batch_norm_forward_quantize(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 19);
  const Tensor x = args.tensor();
  const BnGeometry g(args, x);
  const Tensor weight = args.optional(), bias = args.optional(), running_mean = args.optional(), running_var = args.optional();
  const double momentum = args.number(), eps = args.number(), factor = args.number();
  const Mult mult(args.optional(), g.N, x);
  const int64_t initial = args.integer(), target = args.integer(), total = args.integer();
  Tensor sens = args.optional();
  const bool relu = args.flag();
  const Tensor residual = args.optional();
  const auto dtype = x.scalar_type();
  const int64_t G = g.C * g.HW / 256, ws_bytes = g.workspace();
  const c10::DeviceGuard guard(x.device());
  const Tensor ws = empty({ws_bytes / 4}, x, at::kFloat), mean = empty({g.C}, x, at::kFloat), invstd = empty({g.C}, x, at::kFloat);
  const Tensor mn = empty({g.N * G}, x, dtype), mx = empty({g.N * G}, x, dtype), y = Given(a[0]).empty_like();
  if (!sens.defined()) sens = empty({g.N}, x, at::kFloat);
  const Tensor bits = empty({g.N}, x, at::kInt), prefix = empty({g.N + 1}, x, at::kInt);
  const Tensor packed = empty({total * G * 8}, x, at::kInt), scale = empty({g.N, G, 1}, x, dtype);
  Tensor mask, ymn, ymx;
  if (relu) {
    mask = empty({mask_words(g.N * g.C * g.HW)}, x, at::kInt);
    ymn = empty({g.N * G}, x, dtype);
    ymx = empty({g.N * G}, x, dtype);
  }
  const Draw draw(x);
  launch("batch_norm_forward_quantize", [&] {
      return actnn_batch_norm_forward_quantize(
           ptr(x), f32(weight), f32(bias), f32(running_mean), f32(running_var), ptr(y), f32(mean), f32(invstd), ptr(mn), ptr(mx),
           ptr(ws), ws_bytes, (float)factor, f32(mult.held), mult.per_sample, f32(sens), i32(bits), i32(prefix), (int)initial,
           target, ptr(scale), i32(packed), draw.seed, draw.offset, i32(mask), ptr(ymn), ptr(ymx), ptr(residual), g.N, g.C, g.HW,
           momentum, eps, g.code, g.channels_last, stream_of(x));
  });
  return tuple_of(y, mean, invstd, mn, mx, bits, packed, scale, prefix, mask, ymn, ymx);
}

// x, N, C, HW, channels last, weight, bias, running mean, running variance, momentum, eps, group ranges too
//   -> y, mean, invstd, mn, mx (None without)
PyObject* batch_norm_forward(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 12);
  const Tensor x = args.tensor();
  const BnGeometry g(args, x);
  const Tensor weight = args.optional(), bias = args.optional(), running_mean = args.optional(), running_var = args.optional();
  const double momentum = args.number(), eps = args.number();
  const bool ranges = args.flag();
  const int64_t ws_bytes = g.workspace();
  const c10::DeviceGuard guard(x.device());
  const Tensor ws = empty({ws_bytes / 4}, x, at::kFloat), y = Given(a[0]).empty_like();
  const Tensor mean = empty({g.C}, x, at::kFloat), invstd = empty({g.C}, x, at::kFloat);
  Tensor mn, mx;
  if (ranges) {
    const int64_t groups = g.N * (g.C * g.HW / 256);
    mn = empty({groups}, x, x.scalar_type());
    mx = empty({groups}, x, x.scalar_type());
  }
  launch("batch_norm_forward", [&] {
      return actnn_batch_norm_forward(ptr(x), f32(weight), f32(bias), f32(running_mean), f32(running_var), ptr(y), f32(mean), f32(invstd),
                                ptr(mn), ptr(mx), ptr(ws), ws_bytes, g.N, g.C, g.HW, momentum, eps, g.code, g.channels_last,
                                stream_of(x));
  });
  return tuple_of(y, mean, invstd, mn, mx);
}

// x, dy, N, C, HW, channels last, weight | None, mean, invstd, sumsq -> dx, dweight, dbias, squares of dx (None without)
PyObject* batch_norm_backward(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 10);
  const Tensor x = args.tensor(), dy = args.tensor();
  const BnGeometry g(args, x);
  const Tensor weight = args.optional(), mean = args.tensor(), invstd = args.tensor();
  const int64_t entries = args.flag() ? g.sumsq_entries() : 0, ws_bytes = g.workspace();
  const c10::DeviceGuard guard(x.device());
  const Tensor ws = empty({ws_bytes / 4 + entries}, x, at::kFloat), dx = Given(a[0]).empty_like();
  const Tensor dweight = empty({g.C}, x, at::kFloat), dbias = empty({g.C}, x, at::kFloat);
  launch("batch_norm_backward", [&] {
      return actnn_batch_norm_backward(ptr(x), ptr(dy), f32(weight), f32(mean), f32(invstd), ptr(dx), f32(dweight), f32(dbias), ptr(ws),
                                 ws_bytes, entries ? f32(ws) + ws_bytes / 4 : nullptr, entries, g.N, g.C, g.HW, g.code,
                                 g.channels_last, stream_of(x));
  });
  return tuple_of(dx, dweight, dbias, entries ? ws.narrow(0, ws_bytes / 4, entries) : Tensor());
}

// packed, bits, prefix, scale, mn, dy, N, C, HW, channels last, weight | None, mean, invstd, sumsq, mask | None,
// masked | None -> dx, dweight, dbias, squares of dx (None without)
PyObject* batch_norm_backward_packed(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 16);
  const Tensor packed = args.tensor(), bits = args.tensor(), prefix = args.tensor(), scale = args.tensor(), mn = args.tensor();
  const Tensor dy = args.tensor();
  const BnGeometry g(args, dy);
  const Tensor weight = args.optional(), mean = args.tensor(), invstd = args.tensor();
  const int64_t entries = args.flag() ? g.sumsq_entries() : 0, ws_bytes = g.workspace();
  const Tensor mask = args.optional(), masked = args.optional();
  const c10::DeviceGuard guard(dy.device());
  const Tensor ws = empty({ws_bytes / 4 + entries}, dy, at::kFloat), dx = Given(a[5]).empty_like();
  const Tensor dweight = empty({g.C}, dy, at::kFloat), dbias = empty({g.C}, dy, at::kFloat);
  float* squares = entries ? f32(ws) + ws_bytes / 4 : nullptr;
  if (mask.defined())
    launch("batch_norm_backward_packed_relu", [&] {
      return actnn_batch_norm_backward_packed_add_relu(
             i32(packed), i32(bits), i32(prefix), ptr(scale), ptr(mn), ptr(dy), i32(mask), ptr(masked), f32(weight), f32(mean),
             f32(invstd), ptr(dx), f32(dweight), f32(dbias), ptr(ws), ws_bytes, squares, entries, g.N, g.C, g.HW, g.code,
             g.channels_last, stream_of(dy));
  });
  else
    launch("batch_norm_backward_packed", [&] {
      return actnn_batch_norm_backward_packed(
             i32(packed), i32(bits), i32(prefix), ptr(scale), ptr(mn), ptr(dy), f32(weight), f32(mean), f32(invstd), ptr(dx),
             f32(dweight), f32(dbias), ptr(ws), ws_bytes, squares, entries, g.N, g.C, g.HW, g.code, g.channels_last,
             stream_of(dy));
  });
  return tuple_of(dx, dweight, dbias, entries ? ws.narrow(0, ws_bytes / 4, entries) : Tensor());
}

// ---------------------------------------------------------------------------- max-pool
// x (dense in its format), channels last, window, stride, padding, dilation (two each), two indices a byte -> y, indices
PyObject* max_pool2d_forward(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 11);
  const Tensor x = args.tensor();
  const bool cl = args.flag();
  int64_t v[8];
  for (int64_t& q : v) q = args.integer();
  const bool nibble = args.flag();
  TORCH_CHECK(x.is_cuda() && x.dim() == 4, "The dimension of input is not correct!");
  const int64_t N = x.size(0), C = x.size(1), H = x.size(2), W = x.size(3);
  // (rounded down, as Python's division does, also for windows larger than the padded image)
  auto out = [](int64_t size, int64_t k, int64_t s, int64_t p, int64_t d) {
    const int64_t room = size + 2 * p - d * (k - 1) - 1;
    TORCH_CHECK(s != 0, "stride must not be zero");
    return room / s - (room % s != 0 && (room < 0) != (s < 0)) + 1;
  };
  const int64_t Ho = out(H, v[0], v[2], v[4], v[6]), Wo = out(W, v[1], v[3], v[5], v[7]);
  const auto format = cl ? at::MemoryFormat::ChannelsLast : at::MemoryFormat::Contiguous;
  const c10::DeviceGuard guard(x.device());
  const auto options = at::TensorOptions().device(x.device()).memory_format(format);
  const Tensor y = at::empty({N, C, Ho, Wo}, options.dtype(x.scalar_type()));
  const Tensor idx = nibble ? empty({(N * C * Ho * Wo + 1) / 2}, x, at::kByte) : at::empty({N, C, Ho, Wo}, options.dtype(at::kChar));
  const int code = code_of(x.scalar_type());
  launch("max_pool2d_forward", [&] {
    auto to = [&](auto f, auto* index) {
      return f(ptr(x), ptr(y), index, N, C, H, W, Ho, Wo, (int)v[0], (int)v[1], (int)v[2], (int)v[3], (int)v[4], (int)v[5], code,
               stream_of(x));
    };
    if (nibble)
      return to(cl ? actnn_max_pool2d_forward_cl_nibble : actnn_max_pool2d_forward_nibble, static_cast<uint8_t*>(ptr(idx)));
    return to(cl ? actnn_max_pool2d_forward_cl : actnn_max_pool2d_forward, static_cast<int8_t*>(ptr(idx)));
  });
  return tuple_of(y, idx);
}

// grad (dense in its format), indices, channels last, two indices a byte, N, C, H, W, window, stride, padding -> gradient
PyObject* max_pool2d_backward(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 14);
  const Tensor grad = args.tensor(), idx = args.tensor();
  const bool cl = args.flag(), nibble = args.flag();
  int64_t size[4], v[6];
  for (int64_t& q : size) q = args.integer();
  for (int64_t& q : v) q = args.integer();
  TORCH_CHECK(grad.is_cuda() && grad.dim() == 4, "The dimension of grad_output is not correct!");
  const c10::DeviceGuard guard(grad.device());
  const Tensor out = at::empty({size[0], size[1], size[2], size[3]},
                               at::TensorOptions().device(grad.device()).dtype(grad.scalar_type()).memory_format(
                                   cl ? at::MemoryFormat::ChannelsLast : at::MemoryFormat::Contiguous));
  const int code = code_of(grad.scalar_type());
  launch("max_pool2d_backward", [&] {
    auto to = [&](auto f, auto* index) {
      return f(ptr(grad), index, ptr(out), size[0], size[1], size[2], size[3], grad.size(2), grad.size(3), (int)v[0], (int)v[1],
               (int)v[2], (int)v[3], (int)v[4], (int)v[5], code, stream_of(grad));
    };
    if (nibble)
      return to(cl ? actnn_max_pool2d_backward_cl_nibble : actnn_max_pool2d_backward_nibble, static_cast<uint8_t*>(ptr(idx)));
    return to(cl ? actnn_max_pool2d_backward_cl : actnn_max_pool2d_backward, static_cast<int8_t*>(ptr(idx)));
  });
  return wrap(out);
}

// ---------------------------------------------------------------------------- derivatives
// The calls below have none in forward mode, and a result without a tangent would count as a constant.  (While an autograd Function
// runs its forward pass the mode is off, and what the Function has decides.)
void no_tangents(const char* what, std::initializer_list<const Tensor*> given) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : given)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative");
}
// Nor is a backward pass recorded here (ops.py has the Functions that do): a result made of what wants a gradient is one whose
// backward pass says so, as with torch's own operators that have none.
void no_gradients(const char* what, std::initializer_list<const Tensor*> given, std::initializer_list<const Tensor*> made) {
  if (!at::GradMode::is_enabled()) return;
  torch::autograd::edge_list edges;
  for (const Tensor* t : given)
    if (t->defined() && t->requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(*t));
  if (edges.empty()) return;
  const std::shared_ptr<torch::autograd::Node> node(new torch::autograd::NotImplemented(what, std::move(edges)),
                                                    torch::autograd::deleteNode);
  for (const Tensor* t : made)
    if (t->defined()) torch::autograd::set_history(*t, node);
}

// ---------------------------------------------------------------------------- 8-bit tokens
bool is_float(const Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16;
}
// (a tensor that stands for a batch of others, or for one without values, has no memory, and may have an address all the same)
void check_on_gpu(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor!");
  TORCH_CHECK(t.has_storage() && t.storage().device().is_cuda(), name, " has no memory to read");
}
void check_float(const Tensor& t, const char* name) {
  check_on_gpu(t, name);
  TORCH_CHECK(is_float(t), "The type of ", name, " is not correct!");
}
int64_t whole16(int64_t n) { return (n + 15) / 16 * 16; }

// Rows of a tensor [..., K], an element apart from each other in a row and `ld` elements from row to row.
struct Rows {
  Tensor held;
  int64_t M, K, ld;
  Rows(const Tensor& t, const char* name) {
    check_float(t, name);
    TORCH_CHECK(t.dim() >= 1 && t.size(-1) >= 1, name, " must have rows of at least one element");
    K = t.size(-1);
    M = t.numel() / K;
    held = t.dim() == 2 ? t : t.reshape({M, K});
    if (K > 1 && held.stride(1) != 1) held = held.contiguous();
    ld = M > 1 ? held.stride(0) : K;
  }
};
// Codes [..., K] as the kernels take them: rows at multiples of 16 bytes, the last one's 16 bytes whole in memory.  What
// quantize_tokens returns is laid out like that, anything else is copied.
struct CodeRows {
  Tensor held;
  int64_t M, K, ld;
  CodeRows(const Tensor& t, const char* name) {
    check_on_gpu(t, name);
    TORCH_CHECK(t.scalar_type() == at::kChar, "The type of ", name, " is not correct!");
    TORCH_CHECK(t.dim() >= 1 && t.size(-1) >= 1, name, " must have rows of at least one code");
    K = t.size(-1);
    M = t.numel() / K;
    held = t.dim() == 2 ? t : t.reshape({M, K});
    ld = M > 1 ? held.stride(0) : whole16(K);
    const bool fits = ld < (1 << 23) && (K == 1 || held.stride(1) == 1) && ld >= K && ld % 16 == 0 &&
                      reinterpret_cast<uintptr_t>(held.data_ptr()) % 16 == 0 &&
                      held.storage_offset() + (M - 1) * ld + whole16(K) <= static_cast<int64_t>(held.storage().nbytes());
    if (!fits && M > 0) {
      const Tensor laid = at::empty({M, whole16(K)}, held.options());
      laid.narrow(1, 0, K).copy_(held);
      held = laid.narrow(1, 0, K);
      ld = whole16(K);
    }
  }
  int8_t* data() const { return static_cast<int8_t*>(held.data_ptr()); }
};
Tensor row_scales(const Tensor& t, int64_t rows, const Tensor& like, const char* name) {
  TORCH_CHECK(t.device() == like.device(), name, " must be on the same device");
  check_on_gpu(t, name);
  TORCH_CHECK(t.scalar_type() == at::kFloat, "The type of ", name, " is not correct!");
  TORCH_CHECK(t.numel() == rows, name, " must have one value for each row, ", rows, ", and has ", t.numel());
  return t.contiguous();
}
// new codes and scales for rows of the shape of `like`
struct NewCodes {
  Tensor codes, scale;
  explicit NewCodes(const Tensor& like) {
    std::vector<int64_t> size(like.sizes().begin(), like.sizes().end());
    const int64_t K = size.back();
    size.back() = whole16(K);
    codes = empty(size, like, at::kChar);
    if (K % 16) {                                        // (the first K of each row; a view would cost a short call a tenth)
      std::vector<int64_t> strides(codes.strides().begin(), codes.strides().end());
      size.back() = K;
      codes.unsafeGetTensorImpl()->set_sizes_and_strides(size, strides);
    }
    size.pop_back();
    scale = empty(size, like, at::kFloat);
  }
};

// data -> codes, scale
PyObject* quantize_tokens(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 1);
  const Tensor data = args.tensor();
  no_tangents("quantize_tokens", {&data});
  const Rows rows(data, "data");
  const c10::DeviceGuard guard(data.device());
  const NewCodes out(data);
  launch("quantize_tokens", [&] {
    return actnn_tokens_quantize(ptr(rows.held), rows.ld, static_cast<int8_t*>(ptr(out.codes)), whole16(rows.K), f32(out.scale),
                                 rows.M, rows.K, code_of(data.scalar_type()), stream_of(data));
  });
  no_gradients("quantize_tokens", {&data}, {&out.scale});
  return tuple_of(out.codes, out.scale);
}
// codes, scale, dtype -> values
PyObject* dequantize_tokens(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 3);
  const Tensor codes = args.tensor(), given = args.tensor();
  const auto dtype = type_of(args.integer());
  no_tangents("dequantize_tokens", {&given});
  const CodeRows rows(codes, "codes");
  const Tensor scale = row_scales(given, rows.M, codes, "scale");
  const c10::DeviceGuard guard(codes.device());
  const Tensor out = empty(codes.sizes(), codes, dtype);
  launch("dequantize_tokens", [&] {
    return actnn_tokens_dequantize(rows.data(), rows.ld, f32(scale), ptr(out), rows.M, rows.K, code_of(dtype), stream_of(codes));
  });
  no_gradients("dequantize_tokens", {&given}, {&out});
  return wrap(out);
}

// A weight kept as tokens, one scale for each output channel, and the bias: what linear_tokens and matmul_tokens share.
struct Weight {
  CodeRows rows;
  Tensor scale, bias;
  Weight(const Tensor& codes, const Tensor& scales, const Tensor& given_bias, const Tensor& like, int64_t K)
      : rows(codes, "weight_codes") {
    TORCH_CHECK(codes.dim() == 2, "The dimension of weight_codes is not correct!");
    TORCH_CHECK(codes.device() == like.device(), "weight_codes must be on the same device");
    TORCH_CHECK(rows.K == K, "weight_codes have ", rows.K, " features, the tokens ", K);
    TORCH_CHECK(K <= 131071, "the integer sum takes 131071 features at most, got ", K);
    scale = row_scales(scales, rows.M, codes, "weight_scale");
    if (given_bias.defined()) {
      check_float(given_bias, "bias");
      TORCH_CHECK(given_bias.device() == like.device(), "bias must be on the same device");
      TORCH_CHECK(given_bias.numel() == rows.M, "bias must have one value for each output, ", rows.M, ", and has ", given_bias.numel());
      bias = given_bias.detach().to(at::kFloat).contiguous();
    }
  }
};
Tensor product_of(const CodeRows& x, const Tensor& scale, const Weight& w, at::IntArrayRef lead, at::ScalarType dtype) {
  std::vector<int64_t> size(lead.begin(), lead.end());
  size.back() = w.rows.M;
  const Tensor out = empty(size, x.held, dtype);
  const int64_t bytes = actnn_tokens_matmul_workspace_bytes(x.M, x.K, w.rows.M);
  const Tensor workspace = bytes > 0 ? empty({bytes}, x.held, at::kByte) : Tensor();
  launch("matmul_tokens", [&] {
    return actnn_tokens_matmul(x.data(), x.ld, f32(scale), w.rows.data(), w.rows.ld, f32(w.scale), f32(w.bias), ptr(out), x.M,
                               x.K, w.rows.M, code_of(dtype), ptr(workspace), bytes, stream_of(x.held));
  });
  return out;
}
// codes, scale, weight codes, weight scale, bias | None, dtype -> product
PyObject* matmul_tokens(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 6);
  const Tensor codes = args.tensor(), given = args.tensor(), wcodes = args.tensor(), wscale = args.tensor(), bias = args.optional();
  const auto dtype = type_of(args.integer());
  no_tangents("matmul_tokens", {&given, &wscale, &bias});
  const CodeRows x(codes, "codes");
  const c10::DeviceGuard guard(codes.device());
  const Tensor scale = row_scales(given, x.M, codes, "scale");
  const Weight w(wcodes, wscale, bias, codes, x.K);
  const Tensor out = product_of(x, scale, w, codes.sizes(), dtype);
  no_gradients("matmul_tokens", {&given, &wscale, &bias}, {&out});
  return wrap(out);
}
// data, weight codes, weight scale, bias | None, whether the tokens are kept -> product, codes | None, scale | None
PyObject* linear_tokens(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 5);
  const Tensor data = args.tensor(), wcodes = args.tensor(), wscale = args.tensor(), bias = args.optional();
  const bool keep = args.flag();
  no_tangents("linear_tokens", {&data, &wscale, &bias});
  const Rows rows(data, "data");
  const c10::DeviceGuard guard(data.device());
  const Weight w(wcodes, wscale, bias, data, rows.K);
  const int64_t vector = 16 / data.element_size();
  if (!keep && rows.M >= 1 && rows.M <= 4 && rows.K <= 16384 && rows.K % vector == 0 && rows.ld % vector == 0 &&
      reinterpret_cast<uintptr_t>(rows.held.data_ptr()) % 16 == 0) {
    std::vector<int64_t> size(data.sizes().begin(), data.sizes().end());
    size.back() = w.rows.M;
    const Tensor out = empty(size, data, data.scalar_type());
    launch("linear_tokens", [&] {
      return actnn_tokens_linear_few(ptr(rows.held), rows.ld, w.rows.data(), w.rows.ld, f32(w.scale), f32(w.bias), ptr(out), rows.M,
                                     rows.K, w.rows.M, code_of(data.scalar_type()), stream_of(data));
    });
    no_gradients("linear_tokens", {&data, &wscale, &bias}, {&out});
    return tuple_of(out, Tensor(), Tensor());
  }
  const NewCodes kept(data);
  const CodeRows x(kept.codes, "codes");
  launch("linear_tokens", [&] {
    return actnn_tokens_quantize(ptr(rows.held), rows.ld, x.data(), x.ld, f32(kept.scale), rows.M, rows.K,
                                 code_of(data.scalar_type()), stream_of(data));
  });
  const Tensor out = product_of(x, kept.scale, w, data.sizes(), data.scalar_type());
  no_gradients("linear_tokens", {&data, &wscale, &bias}, {&out, &kept.scale});
  return keep ? tuple_of(out, kept.codes, kept.scale) : tuple_of(out, Tensor(), Tensor());
}
// grad_output, codes, scale, dtype -> gradient of the weight
PyObject* linear_tokens_grad_weight(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 4);
  const Tensor grad = args.tensor(), codes = args.tensor(), given = args.tensor();
  no_tangents("linear_tokens_grad_weight", {&grad, &given});
  check_on_gpu(grad, "grad_output");
  const auto type = grad.scalar_type();
  TORCH_CHECK(type == at::kHalf || type == at::kBFloat16, "The type of grad_output is not correct!");
  const auto dtype = args.at[args.i] == Py_None ? type : type_of(args.integer());
  TORCH_CHECK(dtype == type || dtype == at::kFloat, "the weight's gradient comes in the type of grad_output or in float32");
  const CodeRows x(codes, "codes");
  TORCH_CHECK(codes.device() == grad.device(), "codes must be on the same device");
  TORCH_CHECK(grad.dim() == codes.dim() && grad.dim() >= 1 && grad.sizes().slice(0, grad.dim() - 1) == codes.sizes().slice(0, codes.dim() - 1),
              "grad_output ", grad.sizes(), " and codes ", codes.sizes(), " are not of the same tokens");
  const c10::DeviceGuard guard(grad.device());
  const Tensor scale = row_scales(given, x.M, codes, "scale");
  const int64_t outputs = grad.size(-1);
  int64_t O = outputs;
  if (O == 0 || x.M == 0) {
    const Tensor out = empty({O, x.K}, grad, dtype).zero_();
    no_gradients("linear_tokens_grad_weight", {&grad, &given}, {&out});
    return wrap(out);
  }
  Tensor rows = grad.detach().reshape({x.M, O});
  if (O > 1 && rows.stride(1) != 1) rows = rows.contiguous();
  int64_t ld = x.M > 1 ? rows.stride(0) : O;
  auto pad = [&](int64_t width) {                        // rows of `width`, zeros behind the outputs
    const Tensor room = empty({x.M, width}, grad, type);
    room.narrow(1, 0, outputs).copy_(rows);
    if (width > outputs) room.narrow(1, outputs, width - outputs).zero_();
    rows = room;
    ld = width;
  };
  const bool chunks = O % 8 == 0 && ld % 8 == 0 && reinterpret_cast<uintptr_t>(rows.data_ptr()) % 16 == 0;
  if (!chunks && actnn_tokens_grad_weight_wants_chunks(x.M, O, x.K)) {
    pad((O + 7) / 8 * 8);                                // (the outputs added are cut off below)
    O = ld;
  } else if ((x.M - 1) * ld + O < 8) {                   // the kernel reads 16 bytes at least
    pad(8);
  }
  const Tensor out = empty({O, x.K}, grad, dtype);
  const int64_t bytes = actnn_tokens_grad_weight_workspace_bytes(x.M, O, x.K);
  const Tensor workspace = bytes > 0 ? empty({bytes}, grad, at::kByte) : Tensor();
  launch("linear_tokens_grad_weight", [&] {
    return actnn_tokens_grad_weight(ptr(rows), ld, x.data(), x.ld, f32(scale), ptr(out), x.M, O, x.K, code_of(type),
                                    code_of(dtype), ptr(workspace), bytes, stream_of(grad));
  });
  const Tensor made = O == outputs ? out : out.narrow(0, 0, outputs);
  no_gradients("linear_tokens_grad_weight", {&grad, &given}, {&made});
  return wrap(made);
}

// ---------------------------------------------------------------------------- group norm
// [N, C, ...] channels last, [N, ..., C] in memory; `dense`: the tensor lies like that.  (No view is made of one that does: each
// would take half a microsecond of a short call.)
struct Pixels {
  Tensor given;
  bool dense = true;
  int64_t N, C, count = 1;
  Pixels(const Tensor& t, const char* name) : given(t) {
    check_float(t, name);
    set(name);
  }
  Pixels(const Tensor& t, const char* name, at::ScalarType dtype) : given(t) {
    check_on_gpu(t, name);
    TORCH_CHECK(t.scalar_type() == dtype, "The type of ", name, " is not correct!");
    set(name);
  }
  // a new tensor of the same shape, channels last
  Tensor empty_like(at::ScalarType dtype) const {
    return at::empty_strided(given.sizes(), strides, at::TensorOptions().dtype(dtype).device(given.device()));
  }
  // the tensor, or a copy that is channels last
  Tensor laid_out() const {
    if (dense) return given;
    const Tensor copy = empty_like(given.scalar_type());
    return copy.copy_(given.detach());
  }

 private:
  std::vector<int64_t> strides;
  void set(const char* name) {
    TORCH_CHECK(given.dim() >= 2, "The dimension of ", name, " is not correct!");
    const auto size = given.sizes(), stride = given.strides();
    N = size[0];
    C = size[1];
    strides.resize(size.size());
    int64_t next = 1;
    auto place = [&](int64_t d) {
      strides[d] = next;
      if (size[d] != 1 && stride[d] != next) dense = false;
      next *= size[d] > 1 ? size[d] : 1;
    };
    place(1);
    for (int64_t d = given.dim() - 1; d >= 2; --d) {
      count *= size[d];
      place(d);
    }
    place(0);
    if (given.numel() == 0) dense = true;
  }
};
struct GroupNorm {
  int64_t groups;
  Tensor weight, bias;
  int activation;
  GroupNorm(int64_t g, const Tensor& w, const Tensor& b, int64_t act, const Pixels& x) : groups(g), activation((int)act) {
    TORCH_CHECK(groups >= 1 && x.C >= 1 && x.C % groups == 0, "the channels, ", x.C, ", must be a multiple of the groups, ", groups);
    weight = parameter(w, x, "weight");
    bias = parameter(b, x, "bias");
  }
  static Tensor parameter(const Tensor& t, const Pixels& x, const char* name) {
    if (!t.defined()) return t;
    check_float(t, name);
    TORCH_CHECK(t.device() == x.given.device(), name, " must be on the same device");
    TORCH_CHECK(t.numel() == x.C, name, " must have one value for each channel, ", x.C, ", and has ", t.numel());
    if (t.scalar_type() == at::kFloat && t.is_contiguous()) return t;
    return t.detach().to(at::kFloat).contiguous();
  }
};
// (the kernels read 16 bytes: what torch allocates has room for them, a view at the end of a smaller tensor may not)
Tensor with_room(const Tensor& t) { return t.nbytes() < 16 ? t.detach().clone() : t; }

// input, groups, weight | None, bias | None, eps, activation, whether the input is kept
//   -> output, mean, rstd, codes | None, scale | None
PyObject* group_norm_forward(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 7);
  const Tensor input = args.tensor();
  const int64_t groups = args.integer();
  const Tensor given_weight = args.optional(), given_bias = args.optional();
  const double eps = args.number();
  const int64_t activation = args.integer();
  const bool keep = args.flag();
  no_tangents("group_norm_forward", {&input, &given_weight, &given_bias});
  const Pixels x(input, "input");
  TORCH_CHECK(x.dense, "input must be channels last: [N, C, ...] with the channels of a pixel side by side in memory");
  const c10::DeviceGuard guard(input.device());
  const GroupNorm norm(groups, given_weight, given_bias, activation, x);
  const auto dtype = input.scalar_type();
  const int code = code_of(dtype);
  const Tensor from = with_room(input), y = x.empty_like(dtype);
  const Tensor mean = empty({x.N, groups}, input, at::kFloat), rstd = empty({x.N, groups}, input, at::kFloat);
  const Tensor codes = keep ? x.empty_like(at::kChar) : Tensor(), scale = keep ? empty({x.N, groups}, input, at::kFloat) : Tensor();
  const int64_t bytes = actnn_group_norm_workspace_bytes(x.N, x.C, x.count, groups, code, 0);
  const Tensor workspace = empty({bytes > 0 ? bytes : 0}, input, at::kByte);
  if (x.count == 0) {
    mean.zero_();
    rstd.zero_();
    if (keep) scale.zero_();
  }
  launch("group_norm_forward", [&] {
    return actnn_group_norm_forward(ptr(from), f32(norm.weight), f32(norm.bias), ptr(y), f32(mean), f32(rstd),
                                    static_cast<int8_t*>(ptr(codes)), f32(scale), x.N, x.C, x.count, groups, eps,
                                    norm.activation, code, ptr(workspace), bytes, stream_of(input));
  });
  no_gradients("group_norm_forward", {&input, &given_weight, &given_bias}, {&y, &mean, &rstd, &scale});
  return tuple_of(y, mean, rstd, codes, scale);
}

// grad_output, codes | None, scale | None, input | None, groups, weight | None, bias | None, mean, rstd, activation
//   -> gradients of the input, the weight and the bias (None where there is none)
PyObject* group_norm_backward(PyObject* const* a, Py_ssize_t n) {
  Args args(a, n, 10);
  const Tensor grad_output = args.tensor();
  const Tensor codes = args.optional(), given_scale = args.optional(), input = args.optional();
  const int64_t groups = args.integer();
  const Tensor given_weight = args.optional(), given_bias = args.optional(), given_mean = args.tensor(), given_rstd = args.tensor();
  const int64_t activation = args.integer();
  no_tangents("group_norm_backward",
              {&grad_output, &given_scale, &input, &given_weight, &given_bias, &given_mean, &given_rstd});
  TORCH_CHECK(codes.defined() != input.defined() && codes.defined() == given_scale.defined(),
              "group_norm_backward: either codes and scale or the input");
  const Pixels dy(grad_output, "grad_output");
  const c10::DeviceGuard guard(grad_output.device());
  const auto dtype = grad_output.scalar_type();
  const Tensor& saved = codes.defined() ? codes : input;
  const Pixels x(saved, codes.defined() ? "codes" : "input", codes.defined() ? at::kChar : dtype);
  TORCH_CHECK(saved.sizes() == grad_output.sizes(), "grad_output ", grad_output.sizes(), " and the saved input ", saved.sizes(),
              " are not of the same shape");
  TORCH_CHECK(saved.device() == grad_output.device(), "the saved input must be on the same device");
  const GroupNorm norm(groups, given_weight, given_bias, activation, dy);
  const Tensor mean = row_scales(given_mean, dy.N * groups, grad_output, "mean");
  const Tensor rstd = row_scales(given_rstd, dy.N * groups, grad_output, "rstd");
  const Tensor scale = codes.defined() ? row_scales(given_scale, dy.N * groups, grad_output, "scale") : Tensor();
  const Tensor grad = with_room(dy.laid_out()), kept = codes.defined() ? x.laid_out() : with_room(x.laid_out());
  const Tensor dx = dy.empty_like(dtype);
  const Tensor dweight = norm.weight.defined() ? empty({dy.C}, grad, at::kFloat) : Tensor();
  const Tensor dbias = norm.bias.defined() ? empty({dy.C}, grad, at::kFloat) : Tensor();
  if (dx.numel() == 0) {
    if (dweight.defined()) dweight.zero_();
    if (dbias.defined()) dbias.zero_();
  } else {
    const int code = code_of(dtype);
    const int64_t bytes = actnn_group_norm_workspace_bytes(dy.N, dy.C, dy.count, groups, code, 1);
    const Tensor workspace = empty({bytes > 0 ? bytes : 0}, grad, at::kByte);
    launch("group_norm_backward", [&] {
      return actnn_group_norm_backward(ptr(grad), codes.defined() ? static_cast<int8_t*>(ptr(kept)) : nullptr, f32(scale),
                                       codes.defined() ? nullptr : ptr(kept), f32(norm.weight), f32(norm.bias), f32(mean), f32(rstd),
                                       ptr(dx), f32(dweight), f32(dbias), dy.N, dy.C, dy.count, groups, norm.activation, code,
                                       ptr(workspace), bytes, stream_of(grad));
    });
  }
  no_gradients("group_norm_backward", {&grad_output, &given_scale, &input, &given_weight, &given_bias, &given_mean, &given_rstd},
               {&dx, &dweight, &dbias});
  return tuple_of(dx, dweight, dbias);
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  return F(args, n);
  END_HANDLE_TH_ERRORS
}
#define ACTNN_CALL(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<name>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    ACTNN_CALL(quantize_rows), ACTNN_CALL(quantize_rows_fixed), ACTNN_CALL(unpack_rows_mixed), ACTNN_CALL(unpack_rows_fixed),
    ACTNN_CALL(relu_forward), ACTNN_CALL(relu_backward), ACTNN_CALL(dropout_forward), ACTNN_CALL(dropout_backward),
    ACTNN_CALL(batch_norm_geometry), ACTNN_CALL(batch_norm_forward_quantize), ACTNN_CALL(batch_norm_forward), ACTNN_CALL(batch_norm_backward),
    ACTNN_CALL(batch_norm_backward_packed), ACTNN_CALL(max_pool2d_forward), ACTNN_CALL(max_pool2d_backward),
    ACTNN_CALL(quantize_tokens), ACTNN_CALL(dequantize_tokens), ACTNN_CALL(matmul_tokens), ACTNN_CALL(linear_tokens),
    ACTNN_CALL(linear_tokens_grad_weight), ACTNN_CALL(group_norm_forward), ACTNN_CALL(group_norm_backward), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
