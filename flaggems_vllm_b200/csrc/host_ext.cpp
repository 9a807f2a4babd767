// Native host path of the operators: argument checks, allocations and launches of the common cases in one C++ call
// each.  A decode-sized layer spends a few microseconds per kernel on the device; checked and launched from Python
// it cost the host 85 us, most of it interpreter time.
//
// Every function here serves the usual types, layouts and options and returns None for anything else (and, but for the
// operators with gradients below, for every error): the Python operator then goes its own way, which serves the rest
// and raises the errors.  Nothing is kept between calls.
#define PY_SSIZE_T_CLEAN
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <Python.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <atomic>
#include <cstdlib>
#include <cstring>
#include <optional>
#include <stdexcept>

#include "../../include/moe_sm100.h"

namespace {

std::atomic<int32_t*> g_status[64];        // status word of every device, registered by _lib.status_word

#define MOE_NONE Py_RETURN_NONE

bool is_tensor(PyObject* o) { return THPVariable_Check(o); }
const at::Tensor& tensor(PyObject* o) { return THPVariable_Unpack(o); }
bool truth(PyObject* o) { return o == Py_True; }
bool plain_bool(PyObject* o) { return o == Py_True || o == Py_False; }
bool as_int(PyObject* o, long long* v) {
  if (!PyLong_CheckExact(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) { PyErr_Clear(); return false; }
  return true;
}
bool as_double(PyObject* o, double* v) {
  if (PyFloat_CheckExact(o)) { *v = PyFloat_AS_DOUBLE(o); return true; }
  long long i;
  if (!as_int(o, &i)) return false;
  *v = (double)i;
  return true;
}
// float32 -> MOE_F32 ..., -1 otherwise
int float_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MOE_F32;
    case at::kHalf: return MOE_F16;
    case at::kBFloat16: return MOE_BF16;
    default: return -1;
  }
}
bool cuda_dense(const at::Tensor& t, int dev) { return t.is_cuda() && t.get_device() == dev && t.is_contiguous(); }
bool set_on(const char* name) { return std::getenv(name) != nullptr; }
at::Tensor bytes_on(int64_t n, const at::Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

// a switch that pins one of the other kernels, or asks for a status check after the call
bool switched() {
  static const char* const names[] = {"FLAGGEMS_B200_GENERIC_GEMM", "FLAGGEMS_B200_TC_WIDE", "FLAGGEMS_B200_TC_PAIR",
                                      "FLAGGEMS_B200_TC_PAIR_WIDE", "FLAGGEMS_B200_PRESORT", "FLAGGEMS_B200_TMA_OUT",
                                      "FLAGGEMS_B200_SMALL_M", "FLAGGEMS_B200_W8_WIDEN", "FLAGGEMS_B200_CHECK_STATUS"};
  for (const char* n : names)
    if (set_on(n)) return true;
  return false;
}

PyObject* set_status(PyObject*, PyObject* const* a, Py_ssize_t n) {
  long long dev, ptr;
  if (n != 2 || !as_int(a[0], &dev) || !as_int(a[1], &ptr) || dev < 0 || dev >= 64) {
    PyErr_SetString(PyExc_ValueError, "set_status(device, pointer)");
    return nullptr;
  }
  g_status[dev].store(reinterpret_cast<int32_t*>(ptr));
  MOE_NONE;
}

// The interpreter lock is given back for as long as a function allocates and launches: cudaMalloc may wait for the
// device, and a launch waits when the stream's queue is full, while the work it waits for may need another thread
// of the process (another stream's, another rank's).  Nothing between the braces of its scope touches a Python object.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

int32_t* status_of(int dev) { return dev >= 0 && dev < 64 ? g_status[dev].load(std::memory_order_relaxed) : nullptr; }

// fused_experts(hidden, w1, w2, topk_weights, topk_ids, inplace, activation, apply_router_weight_on_input, use_fp8_w8a8,
//   use_int8_w8a8, use_int8_w8a16, use_int4_w4a16, per_channel_quant, global_num_experts, expert_map, w1_scale, w2_scale,
//   a1_scale, a2_scale, block_shape)
PyObject* fused_experts(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 20) MOE_NONE;
  for (int i = 0; i < 5; ++i)
    if (!is_tensor(a[i])) MOE_NONE;
  for (int i : {5, 7, 8, 9, 10, 11, 12})
    if (!plain_bool(a[i])) MOE_NONE;
  const at::Tensor &x = tensor(a[0]), &w1 = tensor(a[1]), &w2 = tensor(a[2]), &tw = tensor(a[3]), &ti = tensor(a[4]);
  const char* act = PyUnicode_Check(a[6]) ? PyUnicode_AsUTF8(a[6]) : nullptr;
  if (!act || std::strcmp(act, "silu") != 0 || a[17] != Py_None || a[18] != Py_None) MOE_NONE;
  long long ng;
  if (!as_int(a[13], &ng)) MOE_NONE;
  if (!x.is_cuda() || x.dim() != 2 || w1.dim() != 3 || w2.dim() != 3 || ti.dim() != 2 || switched()) MOE_NONE;
  const int dev = x.get_device();
  const int code = float_code(x);
  if ((code != MOE_F16 && code != MOE_BF16) || !cuda_dense(x, dev) || !cuda_dense(w1, dev) || !cuda_dense(w2, dev) ||
      !cuda_dense(tw, dev) || !cuda_dense(ti, dev))
    MOE_NONE;
  const int64_t M = x.size(0), H = x.size(1), E = w1.size(0), N = w1.size(1), k = ti.size(1), I = N / 2;
  if (M <= 0 || M > 32768 || w1.size(2) != H || N % 2 != 0 || w2.size(0) != E || w2.size(1) != H || w2.size(2) != I ||
      ti.size(0) != M || !tw.sizes().equals(ti.sizes()) || tw.scalar_type() != at::kFloat)
    MOE_NONE;
  const bool ids64 = ti.scalar_type() == at::kLong;
  if (!ids64 && ti.scalar_type() != at::kInt) MOE_NONE;
  const bool fp8 = truth(a[8]), i8 = truth(a[9]), weight_only = truth(a[10]) || truth(a[11]), per_channel = truth(a[12]);
  const at::Tensor *s1 = nullptr, *s2 = nullptr;
  int mode = MOE_MODE_HALF, kind = 0;
  if (fp8 || i8 || weight_only) {
    if (!is_tensor(a[15]) || !is_tensor(a[16])) MOE_NONE;
    s1 = &tensor(a[15]);
    s2 = &tensor(a[16]);
    if (!cuda_dense(*s1, dev) || !cuda_dense(*s2, dev) || s1->scalar_type() != at::kFloat || s2->scalar_type() != at::kFloat) MOE_NONE;
    const at::ScalarType wt = fp8 ? at::kFloat8_e4m3fn : at::kChar;
    if (w1.scalar_type() != wt || w2.scalar_type() != wt) MOE_NONE;
    if (fp8 && a[19] != Py_None) {
      long long b0, b1;
      if (i8 || per_channel || !PyList_CheckExact(a[19]) || PyList_GET_SIZE(a[19]) != 2 || !as_int(PyList_GET_ITEM(a[19], 0), &b0) ||
          !as_int(PyList_GET_ITEM(a[19], 1), &b1) || b0 != 128 || b1 != 128 || H % 128 != 0 || I % 128 != 0)
        MOE_NONE;
      if (!s1->sizes().equals({E, N / 128, H / 128}) || !s2->sizes().equals({E, H / 128, I / 128})) MOE_NONE;
      mode = MOE_MODE_FP8_BLOCK;
    } else {
      if (a[19] != Py_None || s1->numel() != E * N || s2->numel() != E * H) MOE_NONE;
      if (fp8 || i8) {
        if (fp8 == i8 || !per_channel) MOE_NONE;  // per-tensor scales: the Python path
        mode = fp8 ? MOE_MODE_FP8_ROW : MOE_MODE_INT8_ROW;
        kind = fp8 ? 1 : 0;
      } else {
        mode = MOE_MODE_W8A16;
      }
    }
  } else if (w1.scalar_type() != x.scalar_type() || w2.scalar_type() != x.scalar_type()) {
    MOE_NONE;
  }
  const int32_t* emap = nullptr;
  const int64_t experts = ng == -1 ? E : ng;
  if (a[14] != Py_None) {
    if (!is_tensor(a[14])) MOE_NONE;
    const at::Tensor& m = tensor(a[14]);
    if (!cuda_dense(m, dev) || m.scalar_type() != at::kInt || m.numel() < experts) MOE_NONE;
    emap = m.const_data_ptr<int32_t>();
  }
  int32_t* status = status_of(dev);
  int64_t bytes[4];
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);  // what is served depends on the device
  if (status == nullptr || experts <= 0 || experts > (1 << 20) ||
      moe_layer_workspace(mode, code, M, (int)k, (int)experts, (int)E, (int)H, (int)I, MOE_ACT_SILU, bytes) != 0)
    MOE_NONE;
  const bool inplace = truth(a[5]), weight_on_input = truth(a[7]);
  at::Tensor out;
  int rc;
  {
    Unlocked unlocked;
    out = inplace ? x : at::empty_like(x);
    at::Tensor ws[4];
    for (int i = 0; i < 4; ++i) ws[i] = bytes_on(bytes[i], x);
    rc = moe_layer(mode, code, x.const_data_ptr(), M, (int)k, ti.const_data_ptr(), ids64, tw.const_data_ptr<float>(),
                   w1.const_data_ptr(), s1 ? s1->const_data_ptr<float>() : nullptr, w2.const_data_ptr(),
                   s2 ? s2->const_data_ptr<float>() : nullptr, out.mutable_data_ptr(), (int)experts, emap, (int)E, (int)H,
                   (int)I, weight_on_input, MOE_ACT_SILU, 0.0f, 0.0f, 0.0f, kind, nullptr, kind, nullptr, ws[0].mutable_data_ptr(),
                   ws[1].mutable_data_ptr(), ws[2].mutable_data_ptr(), ws[3].mutable_data_ptr(), 63, status,
                   c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream());
  }
  if (rc != 0) MOE_NONE;
  if (inplace) {
    Py_INCREF(a[0]);
    return a[0];
  }
  return THPVariable_Wrap(out);
}

// grouped_topk(scores, n_group, topk_group, topk, renormalize, scaling, bias, scoring_func) -> (weights, ids)
PyObject* grouped_topk(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8 || !is_tensor(a[0]) || !is_tensor(a[6]) || !plain_bool(a[4])) MOE_NONE;
  const at::Tensor &s = tensor(a[0]), &b = tensor(a[6]);
  long long groups, keep, k, func;
  double scale;
  if (!as_int(a[1], &groups) || !as_int(a[2], &keep) || !as_int(a[3], &k) || !as_int(a[7], &func) || !as_double(a[5], &scale)) MOE_NONE;
  if (!s.is_cuda() || s.dim() != 2 || b.dim() != 1) MOE_NONE;
  const int dev = s.get_device();
  const int64_t M = s.size(0), E = s.size(1);
  const int sc = float_code(s), bc = float_code(b);
  if (sc < 0 || bc < 0 || !cuda_dense(b, dev) || b.numel() != E || M <= 0 || groups <= 0 || groups > 32 || E % groups != 0 || k <= 0 ||
      k > 32 || (func != 0 && func != 1))
    MOE_NONE;
  const bool renormalize = truth(a[4]);
  at::Tensor w, ids;
  int rc;
  {
    Unlocked unlocked;
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    w = at::empty({M, k}, s.options().dtype(at::kFloat));
    ids = at::empty({M, k}, s.options().dtype(at::kInt));
    rc = moe_grouped_topk(s.const_data_ptr(), sc, s.stride(0), s.stride(1), b.const_data_ptr(), bc, nullptr, M, (int)E, (int)groups,
                          (int)keep, (int)k, renormalize, (float)scale, (int)func, w.mutable_data_ptr<float>(),
                          ids.mutable_data_ptr<int32_t>(), c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream());
  }
  if (rc != 0) MOE_NONE;
  PyObject* r = PyTuple_New(2);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(w));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(ids));
  return r;
}

// topk_route(weights, ids, rows, gating, renormalize, bias, sigmoid, scale) -> True when done
PyObject* topk_route(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8 || !plain_bool(a[4]) || !plain_bool(a[6])) MOE_NONE;
  for (int i = 0; i < 4; ++i)
    if (!is_tensor(a[i])) MOE_NONE;
  const at::Tensor &w = tensor(a[0]), &ids = tensor(a[1]), &rows = tensor(a[2]), &g = tensor(a[3]);
  double scale;
  if (!as_double(a[7], &scale) || !g.is_cuda() || g.dim() != 2 || w.dim() != 2) MOE_NONE;
  const int dev = g.get_device();
  const int64_t M = g.size(0), E = g.size(1), k = w.size(1);
  const int gc = float_code(g);
  const int kind = ids.scalar_type() == at::kInt ? 0 : (ids.scalar_type() == at::kLong ? 1 : -1);
  if (gc < 0 || kind < 0 || !cuda_dense(g, dev) || !cuda_dense(w, dev) || !cuda_dense(ids, dev) || !cuda_dense(rows, dev) ||
      w.scalar_type() != at::kFloat || rows.scalar_type() != at::kInt || w.size(0) != M || !ids.sizes().equals(w.sizes()) ||
      !rows.sizes().equals(w.sizes()) || M <= 0 || k <= 0 || k > 32 || k > E || E > 1024)
    MOE_NONE;
  const float* bias = nullptr;
  if (a[5] != Py_None) {
    if (!is_tensor(a[5])) MOE_NONE;
    const at::Tensor& b = tensor(a[5]);
    if (!cuda_dense(b, dev) || b.scalar_type() != at::kFloat || b.dim() != 1 || b.numel() != E) MOE_NONE;
    bias = b.const_data_ptr<float>();
  }
  const bool sigmoid = truth(a[6]), renormalize = truth(a[4]);
  int rc;
  {
    Unlocked unlocked;
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    rc = moe_topk_route(g.const_data_ptr(), gc, bias, nullptr, M, (int)E, (int)k, sigmoid, renormalize, (float)scale,
                        w.mutable_data_ptr<float>(), ids.mutable_data_ptr(), kind, rows.mutable_data_ptr<int32_t>(),
                        c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream());
  }
  if (rc != 0) MOE_NONE;
  Py_RETURN_TRUE;
}

// router_gemm(x, weight) -> fp32 logits
PyObject* router_gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2 || !is_tensor(a[0]) || !is_tensor(a[1])) MOE_NONE;
  const at::Tensor &x = tensor(a[0]), &w = tensor(a[1]);
  if (!x.is_cuda() || x.dim() != 2 || w.dim() != 2) MOE_NONE;
  const int dev = x.get_device(), xc = float_code(x), wc = float_code(w);
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  int32_t* status = status_of(dev);
  if (xc < 0 || wc < 0 || !status || !cuda_dense(w, dev) || w.size(1) != K || M <= 0 || K % 8 != 0 || x.stride(1) != 1 ||
      x.stride(0) % 8 != 0 || ((uintptr_t)x.const_data_ptr() & 15) || N > (1 << 30) || K > (1 << 30))
    MOE_NONE;
  at::Tensor out;
  int rc;
  {
    Unlocked unlocked;
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    out = at::empty({M, N}, x.options().dtype(at::kFloat));
    rc = moe_router_gemm_ex(x.const_data_ptr(), xc, x.stride(0), w.const_data_ptr(), wc, M, (int)N, (int)K,
                            out.mutable_data_ptr<float>(), status, c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream());
  }
  if (rc != 0) MOE_NONE;
  return THPVariable_Wrap(out);
}

// align(topk_ids, num_experts, block_size, capacity) -> (sorted_ids, expert_ids, num_tokens_post_pad)
PyObject* align(PyObject*, PyObject* const* a, Py_ssize_t n) {
  long long E, bs, cap;
  if (n != 4 || !is_tensor(a[0]) || !as_int(a[1], &E) || !as_int(a[2], &bs) || !as_int(a[3], &cap)) MOE_NONE;
  const at::Tensor& ids = tensor(a[0]);
  if (!ids.is_cuda() || !ids.is_contiguous() || E <= 0 || E > 4096 || bs <= 0 || bs > (1 << 20) || cap < 0) MOE_NONE;
  const int dev = ids.get_device();
  const bool ids64 = ids.scalar_type() == at::kLong;
  int32_t* status = status_of(dev);
  if ((!ids64 && ids.scalar_type() != at::kInt) || !status) MOE_NONE;
  const int64_t blocks = (cap + bs - 1) / bs;
  at::Tensor sorted, experts, npp;
  int rc;
  {
    Unlocked unlocked;
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    const auto opt = ids.options().dtype(at::kInt);
    sorted = at::empty({cap}, opt);
    experts = at::empty({blocks}, opt);
    npp = at::empty({1}, opt);
    rc = moe_align_block_size(ids.const_data_ptr(), ids64, ids.numel(), (int)E, (int)bs, sorted.mutable_data_ptr<int32_t>(), cap,
                              experts.mutable_data_ptr<int32_t>(), blocks, npp.mutable_data_ptr<int32_t>(), status,
                              c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream());
  }
  if (rc != 0) MOE_NONE;
  PyObject* r = PyTuple_New(3);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(sorted));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(experts));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(npp));
  return r;
}

// ---------------------------------------------------------------------------------------------
// Operators with gradients: norm of the residual stream, balance loss.  One implementation for every caller: what is not
// served here (None) the Python operator brings into one of these layouts, or refuses, and calls again.  Errors are raised.

PyObject* g_error = nullptr;  // _lib.MoeKernelError
struct KernelError : std::runtime_error { using std::runtime_error::runtime_error; };
void must(int rc) {
  if (rc != 0) throw KernelError(std::string(moe_last_error()) + " (code " + std::to_string(rc) + ")");
}

PyObject* set_error(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 1) MOE_NONE;
  Py_INCREF(a[0]);
  g_error = a[0];  // lives as long as the module
  MOE_NONE;
}

// word_beside_capture(device) -> int32 [1] of zero, complete on return, no part of the graph that the current stream captures:
// allocated and cleared on another stream, in the mode that lets this thread do so meanwhile.
PyObject* word_beside_capture(PyObject*, PyObject* const* a, Py_ssize_t n) {
  long long dev;
  if (n != 1 || !as_int(a[0], &dev)) MOE_NONE;
  at::Tensor word;
  {
    Unlocked unlocked;
    c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
    const c10::cuda::CUDAStream side = c10::cuda::getStreamFromPool(false, (c10::DeviceIndex)dev);
    c10::cuda::CUDAStreamGuard guard(side);
    word = at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, (c10::DeviceIndex)dev));
    side.synchronize();
  }
  return THPVariable_Wrap(word);
}

// Memory without the dispatcher's way to it, half of an allocation's 1.3 us: an operator of a decode step takes up to four.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, int dev) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, at::Device(at::kCUDA, (c10::DeviceIndex)dev), std::nullopt));
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Rows of the last dimension, whatever is in front of it, and how far apart they are; false where that is no single distance.
bool rows_of(const at::Tensor& t, int64_t* rows, int64_t* ld) {
  if (t.dim() < 1) return false;
  const int64_t H = t.size(-1);
  *rows = H == 0 ? 0 : t.numel() / H;
  *ld = H;
  if (t.is_contiguous()) return true;
  if (H > 1 && t.stride(-1) != 1) return false;
  int64_t inner = 0;  // rows of the dimensions behind
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (inner == 0) {
      *ld = t.stride(d);
      inner = t.size(d);
    } else if (t.stride(d) == *ld * inner) {
      inner *= t.size(d);
    } else {
      return false;
    }
  }
  return *ld >= 0;
}

bool wants_grad(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t && t->defined() && t->requires_grad()) return true;
  return false;
}

// A tangent of forward mode would be dropped (a dual tensor wants no gradient by itself) or, in place, be left on other values.
void no_tangent(std::initializer_list<const at::Tensor*> ts, const char* who) {
  for (const at::Tensor* t : ts)
    if (t && t->defined() && t->_fw_grad(0).defined()) throw std::runtime_error(std::string(who) + " has no derivative in forward mode");
}

// Gradients that a second differentiation would go through end in an error there, not in silence.
variable_list once(variable_list grads, const char* who) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list with;
  for (at::Tensor& g : grads)
    if (g.defined()) with.push_back(g.detach().requires_grad_(true));
  const auto error = std::make_shared<torch::autograd::DelayedError>(std::string(who) + " is differentiable once", (int64_t)with.size());
  with = (*error)(std::move(with));
  size_t i = 0;
  for (at::Tensor& g : grads)
    if (g.defined()) g = with[i++];
  return grads;
}

// A hook on saved tensors may hand back anything: another layout is served, another device, type or size refused.
constexpr char kChanged[] = ": what was saved for the backward pass came back with another device, type or size";

cudaStream_t stream_on(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }

struct NormArgs {
  int code, weight_code, dev;
  int64_t rows, cols, x_ld, residual_ld;
};
bool norm_args(const at::Tensor& x, const at::Tensor& w, const at::Tensor* residual, NormArgs* p) {
  if (!x.is_cuda() || x.dim() < 1 || w.dim() != 1) return false;
  p->dev = x.get_device();
  p->code = float_code(x);
  p->weight_code = float_code(w);
  p->cols = x.size(-1);
  p->residual_ld = 0;
  if (p->code < 0 || (p->weight_code != p->code && p->weight_code != MOE_F32) || !cuda_dense(w, p->dev) || w.size(0) != p->cols ||
      p->cols <= 0 || p->cols > (1 << 24) || !rows_of(x, &p->rows, &p->x_ld) || p->rows > 0x7FFFFFFF)
    return false;
  int64_t rows;
  return !residual || (residual->is_cuda() && residual->get_device() == p->dev && residual->scalar_type() == x.scalar_type() &&
                       residual->sizes().equals(x.sizes()) && rows_of(*residual, &rows, &p->residual_ld));
}

// y, and h where there is a residual
std::pair<at::Tensor, at::Tensor> norm_forward(const at::Tensor& x, const at::Tensor& w, const at::Tensor* residual, double eps,
                                               const NormArgs& p) {
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)p.dev);
  at::Tensor y = fresh(x.sizes(), x.scalar_type(), p.dev), h;
  if (residual) h = fresh(x.sizes(), x.scalar_type(), p.dev);
  must(moe_rms_norm(x.const_data_ptr(), p.x_ld, residual ? residual->const_data_ptr() : nullptr, p.residual_ld, w.const_data_ptr(), p.code,
                    p.weight_code, p.rows, p.cols, (float)eps, y.mutable_data_ptr(), p.cols, residual ? h.mutable_data_ptr() : nullptr,
                    p.cols, stream_on(p.dev)));
  return {y, h};
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& residual,
                               double eps) {
    NormArgs p;
    const at::Tensor* r = residual ? &*residual : nullptr;
    if (!norm_args(x, w, r, &p)) throw KernelError("rms_norm: unsupported operands");
    auto [y, h] = norm_forward(x, w, r, eps, p);
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["residual"] = r != nullptr;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({r ? h : x, w});
    if (r) return {y, h};
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const bool has_residual = ctx->saved_data["residual"].toBool();
    const double eps = ctx->saved_data["eps"].toDouble();
    at::Tensor h = saved[0], w = saved[1];
    const at::Tensor dy = grads[0].defined() ? grads[0].contiguous() : at::Tensor();
    const at::Tensor dh = has_residual && grads[1].defined() ? grads[1].contiguous() : at::Tensor();
    const bool want_w = ctx->needs_input_grad(1);
    const bool want_x = ctx->needs_input_grad(0) || (has_residual && ctx->needs_input_grad(2));
    variable_list out(4);
    if (!dy.defined()) {  // only the stream was used: its gradient passes through
      if (want_x && dh.defined()) out[0] = dh;
      if (has_residual) out[2] = out[0];
      if (want_w) out[1] = at::zeros_like(w);
      return once(out, "rms_norm");
    }
    NormArgs p;
    if (!norm_args(h, w, nullptr, &p)) {  // a hook may have handed back another layout
      h = h.contiguous();
      w = w.contiguous();
      if (!norm_args(h, w, nullptr, &p)) throw KernelError(std::string("rms_norm") + kChanged);
    }
    for (const at::Tensor* t : {&dy, &dh})  // the engine holds them against the outputs, nobody holds those against what was saved
      if (t->defined() && (!t->is_cuda() || t->get_device() != p.dev || t->scalar_type() != h.scalar_type() || !t->sizes().equals(h.sizes())))
        throw KernelError(std::string("rms_norm") + kChanged);
    {
      at::AutoDispatchBelowADInplaceOrView below;  // the buffers are no part of a graph
      c10::cuda::CUDAGuard guard((c10::DeviceIndex)p.dev);
      at::Tensor dx, dw, ws;
      int64_t bytes = 0;
      if (want_x) dx = fresh(h.sizes(), h.scalar_type(), p.dev);
      if (want_w) {
        dw = fresh(w.sizes(), w.scalar_type(), p.dev);
        must(moe_rms_norm_grad_workspace(p.rows, p.cols, &bytes));
        ws = fresh({bytes}, at::kByte, p.dev);
      }
      if (want_x || want_w)
        must(moe_rms_norm_grad(dy.const_data_ptr(), dh.defined() ? dh.const_data_ptr() : nullptr, h.const_data_ptr(), p.x_ld,
                               w.const_data_ptr(), p.code, p.weight_code, p.rows, p.cols, (float)eps,
                               want_x ? dx.mutable_data_ptr() : nullptr, want_w ? dw.mutable_data_ptr() : nullptr,
                               want_w ? ws.mutable_data_ptr() : nullptr, bytes, stream_on(p.dev)));
      out[0] = dx;
      out[1] = dw;
      if (has_residual) out[2] = dx;  // d h / d x = d h / d residual = 1
    }
    return once(out, "rms_norm");
  }
};

// rms_norm(x, weight, eps, residual) -> y, or (y, h) with a residual
PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  double eps;
  if (n != 4 || !is_tensor(a[0]) || !is_tensor(a[1]) || !as_double(a[2], &eps) || (a[3] != Py_None && !is_tensor(a[3]))) MOE_NONE;
  const at::Tensor &x = tensor(a[0]), &w = tensor(a[1]);
  const at::Tensor* residual = a[3] == Py_None ? nullptr : &tensor(a[3]);
  no_tangent({&x, &w, residual}, "rms_norm");
  NormArgs p;
  if (!(eps >= 0.0 && eps < 3e38) || !norm_args(x, w, residual, &p)) MOE_NONE;
  at::Tensor y, h;
  {
    Unlocked unlocked;
    if (wants_grad({&x, &w, residual})) {
      const variable_list out = RmsNorm::apply(x, w, residual ? std::optional<at::Tensor>(*residual) : std::nullopt, eps);
      y = out[0];
      if (residual) h = out[1];
    } else {
      std::tie(y, h) = norm_forward(x, w, residual, eps, p);
    }
  }
  if (!residual) return THPVariable_Wrap(y);
  PyObject* r = PyTuple_New(2);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(y));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(h));
  return r;
}

// Whether rows of `cols` elements of two tensors share memory.  Two windows of one buffer's columns do not.
bool rows_meet(const at::Tensor& a, int64_t a_rows, int64_t a_ld, const at::Tensor& b, int64_t b_rows, int64_t b_ld, int64_t cols) {
  const uintptr_t a0 = (uintptr_t)a.const_data_ptr(), b0 = (uintptr_t)b.const_data_ptr();
  const uintptr_t a_size = a.element_size(), b_size = b.element_size();
  if (a0 >= b0 + ((b_rows - 1) * b_ld + cols) * b_size || b0 >= a0 + ((a_rows - 1) * a_ld + cols) * a_size) return false;
  if (a_rows == 1) a_ld = b_ld;  // a single row has any distance
  if (b_rows == 1) b_ld = a_ld;
  if (a_ld != b_ld || a_size != b_size || (a0 - b0) % a_size != 0) return true;
  const int64_t apart = (int64_t)((a0 > b0 ? a0 - b0 : b0 - a0) / a_size) % a_ld;
  return apart < cols || a_ld - apart < cols;
}

// fused_add_rms_norm(x, residual, weight, eps) -> True when done, in place
PyObject* fused_add_rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  double eps;
  if (n != 4 || !is_tensor(a[0]) || !is_tensor(a[1]) || !is_tensor(a[2]) || !as_double(a[3], &eps)) MOE_NONE;
  const at::Tensor &x = tensor(a[0]), &residual = tensor(a[1]), &w = tensor(a[2]);
  no_tangent({&x, &residual, &w}, "fused_add_rms_norm");
  NormArgs p;
  if (!(eps >= 0.0 && eps < 3e38) || !norm_args(x, w, &residual, &p) || wants_grad({&x, &residual, &w})) MOE_NONE;
  if (p.rows > 1 && (p.x_ld < p.cols || p.residual_ld < p.cols)) MOE_NONE;
  if (p.rows > 0 && (rows_meet(x, p.rows, p.x_ld, residual, p.rows, p.residual_ld, p.cols) ||
                     rows_meet(x, p.rows, p.x_ld, w, 1, p.cols, p.cols) || rows_meet(residual, p.rows, p.residual_ld, w, 1, p.cols, p.cols)))
    MOE_NONE;
  {
    Unlocked unlocked;
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)p.dev);
    must(moe_rms_norm(x.const_data_ptr(), p.x_ld, residual.const_data_ptr(), p.residual_ld, w.const_data_ptr(), p.code, p.weight_code, p.rows,
                      p.cols, (float)eps, x.mutable_data_ptr(), p.x_ld, residual.mutable_data_ptr(), p.residual_ld, stream_on(p.dev)));
    if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
    if (!residual.is_inference()) residual.unsafeGetTensorImpl()->bump_version();
  }
  Py_RETURN_TRUE;
}

// rms_norm_quant(x, weight, eps, residual, group, format, quant_eps, scale_flags, return_norm) -> (q, scales, h?, y?)
PyObject* rms_norm_quant(PyObject*, PyObject* const* a, Py_ssize_t n) {
  double eps, quant_eps;
  long long group, format, flags;
  if (n != 9 || !is_tensor(a[0]) || !is_tensor(a[1]) || !as_double(a[2], &eps) || (a[3] != Py_None && !is_tensor(a[3])) ||
      !as_int(a[4], &group) || !as_int(a[5], &format) || !as_double(a[6], &quant_eps) || !as_int(a[7], &flags) || !plain_bool(a[8]))
    MOE_NONE;
  const at::Tensor &x = tensor(a[0]), &w = tensor(a[1]);
  const at::Tensor* residual = a[3] == Py_None ? nullptr : &tensor(a[3]);
  no_tangent({&x, &w, residual}, "rms_norm_quant");
  NormArgs p;
  if (!(eps >= 0.0 && eps < 3e38) || !(quant_eps >= 0.0 && quant_eps < 3e38) || !norm_args(x, w, residual, &p) ||
      wants_grad({&x, &w, residual}))
    MOE_NONE;
  if (group == 0) group = p.cols;
  if (group < 0 || p.cols % group != 0 || format < 0 || format > 2 || flags < 0 || flags > 3 || ((flags & 2) && format == 2) ||
      ((flags & 1) && x.dim() != 2))
    MOE_NONE;
  const int64_t groups = p.cols / group;
  at::Tensor q, s, y, h;
  {
    Unlocked unlocked;
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)p.dev);
    q = fresh(x.sizes(), format == 0 ? at::kFloat8_e4m3fn : format == 1 ? at::kFloat8_e5m2 : at::kChar, p.dev);
    if (flags & 1) {
      s = fresh({groups, p.rows}, at::kFloat, p.dev);
    } else {
      at::DimVector shape(x.sizes().begin(), x.sizes().end());
      shape.back() = groups;
      s = fresh(shape, at::kFloat, p.dev);
    }
    if (residual) h = fresh(x.sizes(), x.scalar_type(), p.dev);
    if (truth(a[8])) y = fresh(x.sizes(), x.scalar_type(), p.dev);
    must(moe_rms_norm_quant(x.const_data_ptr(), p.x_ld, residual ? residual->const_data_ptr() : nullptr, p.residual_ld, w.const_data_ptr(),
                            p.code, p.weight_code, p.rows, p.cols, (float)eps, (int)format, (int)group, (float)quant_eps, (int)flags,
                            q.mutable_data_ptr(), s.mutable_data_ptr<float>(), p.rows, y.defined() ? y.mutable_data_ptr() : nullptr,
                            residual ? h.mutable_data_ptr() : nullptr, stream_on(p.dev)));
    if (flags & 1) s = s.t();
  }
  PyObject* r = PyTuple_New(2 + (residual != nullptr) + y.defined());
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(q));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(s));
  if (residual) PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(h));
  if (y.defined()) PyTuple_SET_ITEM(r, 2 + (residual != nullptr), THPVariable_Wrap(y));
  return r;
}

struct BalanceArgs {
  int code, dev, sequences;
  int64_t tokens, experts, topk, ld;
  bool ids64;
  int32_t* status;
};
bool balance_args(const at::Tensor& l, const at::Tensor& ids, const at::Tensor* cu, const at::Tensor* pad, BalanceArgs* p) {
  if (!l.is_cuda() || l.dim() != 2 || ids.dim() != 2) return false;
  p->dev = l.get_device();
  p->code = float_code(l);
  p->experts = l.size(1);
  p->topk = ids.size(1);
  p->ids64 = ids.scalar_type() == at::kLong;
  p->status = status_of(p->dev);
  p->sequences = 1;
  if (p->code < 0 || !p->status || p->experts <= 0 || p->experts > 1024 || p->topk <= 0 || p->topk > 32 || !cuda_dense(ids, p->dev) ||
      (!p->ids64 && ids.scalar_type() != at::kInt) || !rows_of(l, &p->tokens, &p->ld) || ids.size(0) != p->tokens ||
      p->tokens * p->topk > 0x7FFF0000)
    return false;
  if (cu) {
    if (!cuda_dense(*cu, p->dev) || cu->scalar_type() != at::kInt || cu->dim() != 1 || cu->numel() < 2 || cu->numel() > 65536) return false;
    p->sequences = (int)cu->numel() - 1;
  }
  return !pad || (cuda_dense(*pad, p->dev) && pad->scalar_type() == at::kBool && pad->dim() == 1 && pad->numel() == p->tokens);
}

const int32_t* cu_pointer(const at::Tensor* cu) { return cu ? cu->const_data_ptr<int32_t>() : nullptr; }
const uint8_t* pad_pointer(const at::Tensor* pad) { return pad ? (const uint8_t*)pad->const_data_ptr() : nullptr; }

// loss, counts, and what the gradient needs (where `keep`; else it lies in the workspace: an allocation less)
std::array<at::Tensor, 3> balance_forward(const at::Tensor& l, const at::Tensor& ids, const at::Tensor* cu, const at::Tensor* pad,
                                          bool sigmoid, const BalanceArgs& p, bool keep) {
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)p.dev);
  int64_t bytes[2];
  must(moe_balance_loss_workspace(p.tokens, (int)p.experts, (int)p.topk, p.sequences, bytes));
  at::Tensor loss = fresh({}, at::kFloat, p.dev);
  at::Tensor counts = cu ? fresh({p.sequences, p.experts}, at::kInt, p.dev) : fresh({p.experts}, at::kInt, p.dev);
  at::Tensor saved, ws = fresh({bytes[0] + (keep ? 0 : bytes[1])}, at::kByte, p.dev);  // bytes[0] is a multiple of 16
  if (keep) saved = fresh({bytes[1]}, at::kByte, p.dev);
  must(moe_balance_loss(l.const_data_ptr(), p.ld, p.code, p.tokens, (int)p.experts, ids.const_data_ptr(), p.ids64, (int)p.topk, sigmoid,
                        cu_pointer(cu), p.sequences, pad_pointer(pad), loss.mutable_data_ptr<float>(), counts.mutable_data_ptr<int32_t>(),
                        keep ? saved.mutable_data_ptr() : (char*)ws.mutable_data_ptr() + bytes[0], ws.mutable_data_ptr(), bytes[0], p.status,
                        stream_on(p.dev)));
  return {loss, counts, saved};
}

struct BalanceLoss : torch::autograd::Function<BalanceLoss> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& l, const at::Tensor& ids, const std::optional<at::Tensor>& cu,
                               const std::optional<at::Tensor>& pad, bool sigmoid) {
    BalanceArgs p;
    const at::Tensor *c = cu ? &*cu : nullptr, *m = pad ? &*pad : nullptr;
    if (!balance_args(l, ids, c, m, &p)) throw KernelError("moe_balance_loss: unsupported operands");
    auto out = balance_forward(l, ids, c, m, sigmoid, p, true);
    ctx->save_for_backward({l, out[2], c ? *c : at::Tensor(), m ? *m : at::Tensor()});
    ctx->saved_data["sigmoid"] = sigmoid;
    ctx->saved_data["topk"] = p.topk;
    ctx->saved_data["sequences"] = (int64_t)p.sequences;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({out[1]});
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(5);
    if (!grads[0].defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    at::Tensor l = saved[0], counts = saved[1], cu = saved[2], pad = saved[3];
    const int64_t sequences = ctx->saved_data["sequences"].toInt();
    if (!l.is_cuda() || l.dim() != 2 || float_code(l) < 0) throw KernelError(std::string("moe_balance_loss") + kChanged);
    int64_t tokens, ld;
    if (!rows_of(l, &tokens, &ld)) {
      l = l.contiguous();
      rows_of(l, &tokens, &ld);
    }
    auto dense = [&](at::Tensor& t, at::ScalarType type, int64_t numel) {
      if (t.defined()) t = t.contiguous();
      return !t.defined() || (cuda_dense(t, l.get_device()) && t.scalar_type() == type && t.numel() == numel);
    };
    if (!counts.defined() || !dense(counts, at::kByte, 4 * (sequences * (l.size(1) + 1) + 1)) || !dense(cu, at::kInt, sequences + 1) ||
        !dense(pad, at::kBool, tokens))
      throw KernelError(std::string("moe_balance_loss") + kChanged);
    const at::Tensor dloss = grads[0].to(at::kFloat).contiguous();
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const int dev = l.get_device();
      c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
      out[0] = fresh(l.sizes(), l.scalar_type(), dev);
      must(moe_balance_loss_grad(l.const_data_ptr(), ld, float_code(l), tokens, (int)l.size(1), (int)ctx->saved_data["topk"].toInt(),
                                 ctx->saved_data["sigmoid"].toBool(), cu_pointer(cu.defined() ? &cu : nullptr), (int)sequences,
                                 pad_pointer(pad.defined() ? &pad : nullptr), counts.const_data_ptr(), dloss.const_data_ptr<float>(), out[0].mutable_data_ptr(),
                                 stream_on(dev)));
    }
    return once(out, "moe_balance_loss");
  }
};

// balance_loss(logits, topk_ids, sigmoid, cu_seqlens, is_padding) -> (loss, counts)
PyObject* balance_loss(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5 || !is_tensor(a[0]) || !is_tensor(a[1]) || !plain_bool(a[2]) || (a[3] != Py_None && !is_tensor(a[3])) ||
      (a[4] != Py_None && !is_tensor(a[4])))
    MOE_NONE;
  const at::Tensor &l = tensor(a[0]), &ids = tensor(a[1]);
  const at::Tensor *cu = a[3] == Py_None ? nullptr : &tensor(a[3]), *pad = a[4] == Py_None ? nullptr : &tensor(a[4]);
  no_tangent({&l}, "moe_balance_loss");
  BalanceArgs p;
  if (!balance_args(l, ids, cu, pad, &p)) MOE_NONE;
  const bool sigmoid = truth(a[2]);
  at::Tensor loss, counts;
  {
    Unlocked unlocked;
    if (wants_grad({&l})) {
      const variable_list out = BalanceLoss::apply(l, ids, cu ? std::optional<at::Tensor>(*cu) : std::nullopt,
                                                   pad ? std::optional<at::Tensor>(*pad) : std::nullopt, sigmoid);
      loss = out[0];
      counts = out[1];
    } else {
      auto out = balance_forward(l, ids, cu, pad, sigmoid, p, false);
      loss = out[0];
      counts = out[1];
    }
  }
  PyObject* r = PyTuple_New(2);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(loss));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(counts));
  return r;
}

// Exceptions of the operators above become Python's: a failed launch MoeKernelError, torch's own as torch raises them.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* raising(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    return F(self, a, n);
  } catch (const KernelError& e) {
    PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// No C++ exception crosses into the interpreter (an allocation can throw): it becomes the Python path's problem.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  try {
    return F(self, a, n);
  } catch (const std::exception&) {
    MOE_NONE;
  }
}

#define MOE_FN(name) {#name, (PyCFunction)(void (*)(void))guarded<name>, METH_FASTCALL, nullptr}
#define MOE_OP(name) {#name, (PyCFunction)(void (*)(void))raising<name>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {MOE_FN(set_status), MOE_FN(fused_experts), MOE_FN(grouped_topk), MOE_FN(topk_route),
                         MOE_FN(router_gemm), MOE_FN(align), MOE_FN(set_error), MOE_OP(word_beside_capture), MOE_OP(rms_norm), MOE_OP(fused_add_rms_norm),
                         MOE_OP(rms_norm_quant), MOE_OP(balance_loss), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host_ext", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host_ext(void) { return PyModule_Create(&module); }
