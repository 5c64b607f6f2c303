// The host side of the smallest calls in C++: checks, allocations and launches of an everyday inference projection, the packed
// FFN, the differentiable linear layer and the GRPO loss, on top of the C entry points of librlk_gfx950.so.
//
// Small calls are bound by their host time. In Python / here, us a call: a projection 13.9 / 5.2 (5 were the dispatch of the
// torch.library operator around it), the packed FFN 28.7 / 11.0, a linear layer with both gradients 40.6 / 27.0, the FFN with all
// its gradients 116 / 58, the GRPO loss with its gradient 59.7 / 33.5, beside kernels of 2 to 12 each; 87 / 50, 197 / 99 and 114 / 59
// in the stretches in which autograd's device thread has to be woken for every backward; in those, the SwiGLU of eight-bit copies with
// its gradients 132 / 59 and scores of hidden states with theirs 189 / 97.
//
// Every function takes everyday arguments only and answers None to anything else - other types, layouts and devices, subclasses,
// batched and functorch tensors, tangents, dispatch and function modes (torch.set_default_device() is one), tracing, profilers -, for
// which the caller goes the way it went before. The autograd functions hand what is not everyday in a backward (an operand that wants
// no gradient, gradients or saved tensors that are more than their values) to the Python functions that bind() was given. Under
// create_graph the loss does so too, whose gradient is differentiable; those of the linear layer and the FFN have no graph either way.
// Nothing is kept from one call for the next.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/record_function.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <climits>
#include <unordered_set>

#include "../../include/rlk.h"

namespace {

using at::Tensor;
using c10::DispatchKey;
using c10::DispatchKeySet;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The library's entry points, from the library that Python has loaded, and the Python functions of the general ways.
decltype(&rlk_det_gemm_bf16) gemm_entry = nullptr;
decltype(&rlk_linear_bwd_bf16) linear_bwd_entry = nullptr;
decltype(&rlk_det_gemm_swiglu_workspace_bytes) swiglu_workspace_entry = nullptr;
decltype(&rlk_det_gemm_swiglu_bf16) swiglu_entry = nullptr;
decltype(&rlk_det_gemm_swiglu_training_bf16) swiglu_training_entry = nullptr;
decltype(&rlk_swiglu_bwd) swiglu_bwd_entry = nullptr;
decltype(&rlk_grpo_workspace_bytes) grpo_workspace_entry = nullptr;
decltype(&rlk_grpo_ratio_kl_loss) grpo_entry = nullptr;
decltype(&rlk_grpo_ratio_kl_loss_bwd) grpo_bwd_entry = nullptr;
decltype(&rlk_logits_scores_workspace_bytes) scores_workspace_entry = nullptr;
decltype(&rlk_logits_scores) scores_entry = nullptr;
decltype(&rlk_logits_scores_backward) scores_bwd_entry = nullptr;
decltype(&rlk_linear_scores_workspace_bytes) linear_scores_workspace_entry = nullptr;
decltype(&rlk_linear_scores_fwd) linear_scores_entry = nullptr;
decltype(&rlk_linear_dlogits_row_stride) dlogits_stride_entry = nullptr;
decltype(&rlk_linear_dlogits_bwd) dlogits_bwd_entry = nullptr;
decltype(&rlk_block_norm_forward) norm_entry = nullptr;
decltype(&rlk_block_norm_workspace_bytes) norm_workspace_entry = nullptr;
decltype(&rlk_block_norm_backward) norm_bwd_entry = nullptr;
decltype(&rlk_mx8_encode) mx8_encode_entry = nullptr;
decltype(&rlk_mx8_swiglu_forward) mx8_swiglu_entry = nullptr;
decltype(&rlk_mx8_swiglu_backward) mx8_swiglu_bwd_entry = nullptr;
decltype(&rlk_last_error) last_error_entry = nullptr;
PyObject* general_linear_gradients = nullptr;  // (a, weight, grad, need_a, need_weight) -> (da, dw)
PyObject* general_ffn_gradients = nullptr;     // (x, gate, up, activated, three weights, grad, need of x and the weights) -> four
PyObject* general_scores_gradient = nullptr;   // (logits, target, temperature, lse, entropy, top ids, real, four gradients) -> grad
PyObject* general_linear_scores = nullptr;     // (hidden, weight, target, temperature, lse, entropy, top ids, logits, real, four gradients, two needs) -> two
PyObject* general_norm_gradients = nullptr;    // (block, residual, gate, two weights, rstd, kind, eps, scale, two gradients, five needs) -> five
PyObject* general_swiglu_gradients = nullptr;  // (dy, codes and scales of gate and up) -> (d_gate, d_up)
PyObject* general_grpo_gradient = nullptr;     // (cur, old, ref, adv, mask, g_loss, g_policy, g_kl, clip_eps, beta) -> grad

// What _lib.check() raises.
void check_status(int status, const char* what) {
  if (status == RLK_OK) return;
  const char* message = last_error_entry();
  if (message == nullptr || message[0] == 0) message = what;
  TORCH_CHECK_VALUE(status != RLK_ERR_INVALID_ARGUMENT, message);
  throw std::runtime_error(message);
}

// Nothing on this thread takes over operations: no dispatch, function or tracing mode, no functorch level.
bool everyday_thread() {
  static const uint64_t usual = (DispatchKeySet(DispatchKey::BackendSelect) | DispatchKeySet(DispatchKey::ADInplaceOrView)).raw_repr();
  return (c10::impl::tls_local_dispatch_key_set().included_.raw_repr() & ~usual) == 0 && !at::impl::torch_function_mode_enabled();
}
// ... and nothing looks at them: under a profiler the calls show as the operators that they are.
bool everyday_caller() { return everyday_thread() && !at::hasCallbacks(); }

// A tensor of values in GPU memory and nothing else.
bool everyday(const Tensor& t, at::ScalarType dtype) {
  static const uint64_t usual = (DispatchKeySet(DispatchKey::CUDA) | DispatchKeySet(DispatchKey::AutogradCUDA) |
                                 DispatchKeySet(DispatchKey::ADInplaceOrView) | DispatchKeySet(DispatchKey::AutocastCUDA)).raw_repr();
  return t.defined() && t.is_cuda() && (t.key_set().raw_repr() & ~usual) == 0 && t.scalar_type() == dtype && t.has_storage() &&
         !t._fw_grad(0).defined();
}
bool everyday(const Tensor& t, at::ScalarType dtype, const Tensor& beside) {
  return everyday(t, dtype) && t.get_device() == beside.get_device();
}

// A Python argument that is a Tensor or a Parameter, no subclass.
const Tensor* exact_tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

void* stream_of(const Tensor& t) {
  return reinterpret_cast<void*>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream());
}
Tensor empty(at::IntArrayRef shape, at::ScalarType dtype, const Tensor& like) {
  return at::empty(shape, like.options().dtype(dtype).requires_grad(false));
}

// A new reference, or the Python error that is set.
struct PyRef {
  explicit PyRef(PyObject* o) : object(o) {
    if (object == nullptr) throw python_error();
  }
  ~PyRef() { Py_DECREF(object); }
  PyRef(const PyRef&) = delete;
  PyRef& operator=(const PyRef&) = delete;
  PyObject* get() const { return object; }
  PyObject* const object;
};
Tensor tensor_or_none(PyObject* o) {
  if (o == nullptr) throw python_error();
  return o == Py_None ? Tensor() : THPVariable_Unpack(o);
}

constexpr auto kBf16 = at::kBFloat16;
bool everyday_matrix(const Tensor& t) { return t.dim() == 2 && t.is_contiguous() && t.numel() > 0; }

// a[M,K] @ weight[N,K].T
Tensor project(const Tensor& a, const Tensor& weight) {
  const int64_t m = a.size(0), k = a.size(1), n = weight.size(0);
  Tensor out = empty({m, n}, kBf16, a);
  check_status(gemm_entry(a.data_ptr(), k, 1, weight.data_ptr(), 1, k, out.data_ptr(), n, (int)m, (int)n, (int)k, 0, 0, stream_of(a)),
               "rlk_det_gemm_bf16 failed");
  return out;
}
bool projects(const Tensor& a, const Tensor& weight) {
  return everyday(a, kBf16) && everyday(weight, kBf16, a) && everyday_matrix(a) && everyday_matrix(weight) &&
         a.size(1) == weight.size(1) && a.size(0) <= INT_MAX && a.size(1) <= INT_MAX && weight.size(0) <= INT_MAX;
}

// ---------------------------------------------------------------------------
// Linear layer under autograd
// ---------------------------------------------------------------------------

// A row-major operand that the K-major loader takes as it is (_C._rows_of_chunks).
bool rows_of_chunks(const Tensor& t) {
  return t.size(1) % 8 == 0 && t.stride(1) == 1 && t.stride(0) % 8 == 0 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}

// Both gradients of a @ weight.T in one library call.
bool takes_both_gradients(const Tensor& a, const Tensor& weight, const Tensor& grad) {
  return everyday(grad, kBf16) && everyday_matrix(grad) && projects(a, weight) && everyday(a, kBf16, grad) &&
         grad.size(0) == a.size(0) && grad.size(1) == weight.size(0) && rows_of_chunks(a) && rows_of_chunks(weight) &&
         rows_of_chunks(grad);
}
variable_list both_gradients(const Tensor& a, const Tensor& weight, const Tensor& grad, int config) {
  const int64_t m = a.size(0), k = a.size(1), n = weight.size(0);
  Tensor da = empty({m, k}, kBf16, grad), dw = empty({n, k}, kBf16, grad);
  check_status(linear_bwd_entry(grad.data_ptr(), n, a.data_ptr(), k, weight.data_ptr(), k, da.data_ptr(), k, dw.data_ptr(), k, (int)m,
                                (int)k, (int)n, config, stream_of(grad)),
               "rlk_linear_bwd_bf16 failed");
  return {da, dw};
}

struct LinearFn : torch::autograd::Function<LinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& a, const Tensor& weight) {
    ctx->save_for_backward({a, weight});
    return project(a, weight);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &a = saved[0], &weight = saved[1], &grad = grads[0];
    const bool need_a = ctx->needs_input_grad(0), need_weight = ctx->needs_input_grad(1);
    if (need_a && need_weight && everyday_thread() && takes_both_gradients(a, weight, grad)) {
      const c10::OptionalDeviceGuard guard(grad.device());
      return both_gradients(a, weight, grad, RLK_LINEAR_BWD_CFG_AUTO);
    }
    const pybind11::gil_scoped_acquire gil;
    const PyRef py_a(THPVariable_Wrap(a)), py_weight(THPVariable_Wrap(weight)), py_grad(THPVariable_Wrap(grad));
    const PyRef result(PyObject_CallFunctionObjArgs(general_linear_gradients, py_a.get(), py_weight.get(), py_grad.get(),
                                                    need_a ? Py_True : Py_False, need_weight ? Py_True : Py_False, nullptr));
    return {tensor_or_none(PyTuple_GetItem(result.get(), 0)), tensor_or_none(PyTuple_GetItem(result.get(), 1))};
  }
};


// ---------------------------------------------------------------------------
// Packed gated FFN (inference)
// ---------------------------------------------------------------------------

bool takes_ffn(const Tensor& x, const Tensor& gate_up, const Tensor& down) {
  return everyday(x, kBf16) && everyday(gate_up, kBf16, x) && everyday_matrix(gate_up) && x.dim() >= 1 && x.is_contiguous() &&
         x.numel() > 0 && everyday(down, kBf16, x) && everyday_matrix(down) && gate_up.size(0) % 2 == 0 &&
         gate_up.size(1) == x.size(-1) && down.size(1) == gate_up.size(0) / 2 && x.numel() / x.size(-1) <= INT_MAX &&
         x.size(-1) <= INT_MAX && gate_up.size(0) <= INT_MAX && down.size(0) <= INT_MAX;
}

Tensor packed_ffn(const Tensor& x, const Tensor& gate_up, const Tensor& down) {
  const int64_t k = x.size(-1), m = x.numel() / k, inter = gate_up.size(0) / 2, n = down.size(0);
  Tensor activated = empty({m, inter}, kBf16, x);
  const size_t bytes = swiglu_workspace_entry(x.data_ptr(), k, gate_up.data_ptr(), k, (int)m, (int)inter, (int)k);
  Tensor workspace;
  if (bytes > 0) workspace = empty({(int64_t)(bytes / 2)}, kBf16, x);
  void* const stream = stream_of(x);
  check_status(swiglu_entry(x.data_ptr(), k, gate_up.data_ptr(), k, activated.data_ptr(), inter,
                            bytes > 0 ? workspace.data_ptr() : nullptr, bytes, (int)m, (int)inter, (int)k, stream),
               "rlk_det_gemm_swiglu_bf16 failed");
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = n;
  Tensor out = empty(shape, kBf16, x);
  check_status(gemm_entry(activated.data_ptr(), inter, 1, down.data_ptr(), 1, inter, out.data_ptr(), n, (int)m, (int)n, (int)inter, 0,
                          0, stream),
               "rlk_det_gemm_bf16 failed");
  return out;
}

// ---------------------------------------------------------------------------
// Gated FFN under autograd (_DeterministicFFNFunction in backends/rocm/ffn/ffn.py, three weights)
// ---------------------------------------------------------------------------

bool takes_ffn_training(const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down) {
  return everyday(x, kBf16) && x.dim() >= 1 && x.is_contiguous() && x.numel() > 0 && x.numel() / x.size(-1) <= INT_MAX &&
         x.size(-1) <= INT_MAX && everyday(gate, kBf16, x) && everyday_matrix(gate) && gate.size(1) == x.size(-1) &&
         everyday(up, kBf16, x) && up.is_contiguous() && up.sizes() == gate.sizes() && everyday(down, kBf16, x) &&
         everyday_matrix(down) && down.size(0) == gate.size(1) && down.size(1) == gate.size(0) && gate.size(0) <= INT_MAX;
}

struct FfnFn : torch::autograd::Function<FfnFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& input, const Tensor& gate_weight, const Tensor& up_weight,
                        const Tensor& down_weight) {
    const Tensor x = input.dim() == 2 ? input : input.view({-1, input.size(-1)});
    const int64_t m = x.size(0), k = x.size(1), inter = gate_weight.size(0);
    const Tensor gate = empty({m, inter}, kBf16, x), up = empty({m, inter}, kBf16, x), activated = empty({m, inter}, kBf16, x);
    check_status(swiglu_training_entry(x.data_ptr(), k, gate_weight.data_ptr(), up_weight.data_ptr(), k, gate.data_ptr(), up.data_ptr(),
                                       activated.data_ptr(), inter, (int)m, (int)inter, (int)k, stream_of(x)),
                 "rlk_det_gemm_swiglu_training_bf16 failed");
    ctx->save_for_backward({x, gate, up, activated, gate_weight, up_weight, down_weight});
    ctx->saved_data["shape"] = input.sizes().vec();
    const Tensor out = project(activated, down_weight);
    return input.dim() == 2 ? out : out.view(input.sizes());
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();  // x, gate, up, activated, weights of gate, up and down
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    bool need[4], all = true;
    for (int i = 0; i < 4; ++i) all &= need[i] = ctx->needs_input_grad(i);
    if (all && everyday_thread() && everyday(grads[0], kBf16) && grads[0].is_contiguous() && grads[0].sizes() == at::IntArrayRef(shape)) {
      const Tensor grad = shape.size() == 2 ? grads[0] : grads[0].view({-1, shape.back()});
      if (takes_both_gradients(s[3], s[6], grad) && everyday(s[1], kBf16, grad) && everyday_matrix(s[1]) && rows_of_chunks(s[1]) &&
          s[1].sizes() == s[3].sizes() && everyday(s[2], kBf16, grad) && everyday_matrix(s[2]) && s[2].sizes() == s[3].sizes() &&
          takes_both_gradients(s[0], s[4], s[1]) && takes_both_gradients(s[0], s[5], s[2])) {
        const c10::OptionalDeviceGuard guard(grad.device());
        // three weights that are together more than the memory-side cache holds (_MANY_WEIGHTS_BYTES)
        const int config = 3 * (int64_t)s[6].nbytes() >= ((int64_t)128 << 20) ? RLK_LINEAR_BWD_CFG_MANY_WEIGHTS : RLK_LINEAR_BWD_CFG_AUTO;
        const variable_list of_down = both_gradients(s[3], s[6], grad, config);
        const int64_t m = grad.size(0), inter = s[1].size(1);
        const Tensor d_gate = empty({m, inter}, kBf16, grad), d_up = empty({m, inter}, kBf16, grad);
        check_status(swiglu_bwd_entry(of_down[0].data_ptr(), inter, s[1].data_ptr(), inter, s[2].data_ptr(), inter, d_gate.data_ptr(),
                                      inter, d_up.data_ptr(), inter, (int)m, (int)inter, RLK_DTYPE_BF16, stream_of(grad)),
                     "rlk_swiglu_bwd failed");
        const variable_list of_gate = both_gradients(s[0], s[4], d_gate, config), of_up = both_gradients(s[0], s[5], d_up, config);
        Tensor dx = of_gate[0];
        dx.add_(of_up[0]);
        return {shape.size() == 2 ? dx : dx.view(shape), of_gate[1], of_up[1], of_down[1]};
      }
    }
    const pybind11::gil_scoped_acquire gil;
    const PyRef args(PyTuple_New(12));
    for (int i = 0; i < 7; ++i) PyTuple_SET_ITEM(args.get(), i, THPVariable_Wrap(s[i]));
    PyTuple_SET_ITEM(args.get(), 7, THPVariable_Wrap(grads[0]));
    for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(args.get(), 8 + i, PyBool_FromLong(need[i]));
    const PyRef result(PyObject_CallObject(general_ffn_gradients, args.get()));
    variable_list out;
    for (int i = 0; i < 4; ++i) out.push_back(tensor_or_none(PyTuple_GetItem(result.get(), i)));
    if (out[0].defined()) out[0] = out[0].reshape(shape);
    return out;
  }
};

// ---------------------------------------------------------------------------
// GRPO loss
// ---------------------------------------------------------------------------

// Log-probs [rollouts, tokens], one advantage per rollout, a mask of bools or none.
struct GrpoInputs {
  Tensor cur, old, ref, adv, mask;
  double clip_eps, beta;

  bool usual() const {
    constexpr auto kF32 = at::kFloat;
    return everyday(cur, kF32) && cur.dim() == 2 && cur.is_contiguous() && cur.numel() > 0 && cur.size(0) <= INT_MAX &&
           cur.size(1) <= INT_MAX && everyday(old, kF32, cur) && old.sizes() == cur.sizes() && old.is_contiguous() &&
           everyday(ref, kF32, cur) && ref.sizes() == cur.sizes() && ref.is_contiguous() && everyday(adv, kF32, cur) &&
           adv.numel() == cur.size(0) && adv.is_contiguous() &&
           (!mask.defined() || (everyday(mask, at::kBool, cur) && mask.sizes() == cur.sizes() && mask.is_contiguous()));
  }
  const uint8_t* mask_bytes() const { return mask.defined() ? static_cast<const uint8_t*>(mask.data_ptr()) : nullptr; }
};
struct GrpoOutputs {
  Tensor out3, ratio, k3, workspace;
};
const float* floats(const Tensor& t) { return t.defined() ? static_cast<const float*>(t.data_ptr()) : nullptr; }

GrpoOutputs grpo(const GrpoInputs& in) {
  const int64_t rollouts = in.cur.size(0), tokens = in.cur.size(1);
  const size_t bytes = grpo_workspace_entry((int)rollouts);
  GrpoOutputs out{empty({3}, at::kFloat, in.cur), empty({rollouts, tokens}, at::kFloat, in.cur),
                  empty({rollouts, tokens}, at::kFloat, in.cur), empty({(int64_t)(bytes / 4)}, at::kFloat, in.cur)};
  check_status(grpo_entry(floats(in.cur), floats(in.old), floats(in.ref), floats(in.adv), in.mask_bytes(), (int)rollouts, (int)tokens,
                          (float)in.clip_eps, (float)in.beta, static_cast<float*>(out.ratio.data_ptr()),
                          static_cast<float*>(out.k3.data_ptr()), static_cast<float*>(out.out3.data_ptr()), out.workspace.data_ptr(),
                          bytes, stream_of(in.cur)),
               "rlk_grpo_ratio_kl_loss failed");
  return out;
}

// The three scalars with respect to the current log-probs (_GrpoLossAutograd in backends/rocm/loss/grpo.py, with the same
// conditions for the kernel in the backward). The workspace holds the kernel's own numbers: it is not for saved-tensor hooks.
struct GrpoFn : torch::autograd::Function<GrpoFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& cur, const GrpoInputs* in, GrpoOutputs* out) {
    *out = grpo(*in);
    variable_list saved = {cur, in->old, in->ref, in->adv};
    if (in->mask.defined()) saved.push_back(in->mask);
    ctx->save_for_backward(std::move(saved));
    ctx->saved_data["workspace"] = out->workspace;
    ctx->saved_data["clip_eps"] = in->clip_eps;
    ctx->saved_data["beta"] = in->beta;
    ctx->set_materialize_grads(false);  // an unused output costs no zero tensor
    return out->out3.unbind(0);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined() && !grads[1].defined() && !grads[2].defined()) return {Tensor(), Tensor(), Tensor()};
    const variable_list saved = ctx->get_saved_variables();
    GrpoInputs in{saved[0], saved[1], saved[2], saved[3], saved.size() > 4 ? saved[4] : Tensor(),
                  ctx->saved_data["clip_eps"].toDouble(), ctx->saved_data["beta"].toDouble()};
    const Tensor workspace = ctx->saved_data["workspace"].toTensor();
    bool values = !at::GradMode::is_enabled() && everyday_thread() && in.usual() && in.cur.get_device() == workspace.get_device();
    for (const Tensor& g : grads) values = values && (!g.defined() || (everyday(g, at::kFloat, in.cur) && g.numel() == 1));
    if (values) {
      const c10::OptionalDeviceGuard guard(in.cur.device());
      Tensor grad = empty(in.cur.sizes(), at::kFloat, in.cur);
      check_status(grpo_bwd_entry(floats(in.cur), floats(in.old), floats(in.ref), floats(in.adv), in.mask_bytes(), workspace.data_ptr(),
                                  workspace.nbytes(), floats(grads[0]), floats(grads[1]), floats(grads[2]), (int)in.cur.size(0),
                                  (int)in.cur.size(1), (float)(1.0 - in.clip_eps), (float)(1.0 + in.clip_eps), (float)in.beta,
                                  static_cast<float*>(grad.data_ptr()), stream_of(in.cur)),
                   "rlk_grpo_ratio_kl_loss_bwd failed");
      return {grad, Tensor(), Tensor()};
    }
    const pybind11::gil_scoped_acquire gil;  // THPVariable_Wrap makes None of an undefined tensor
    const PyRef cur(THPVariable_Wrap(in.cur)), old(THPVariable_Wrap(in.old)), ref(THPVariable_Wrap(in.ref)), adv(THPVariable_Wrap(in.adv)),
        mask(THPVariable_Wrap(in.mask)), g_loss(THPVariable_Wrap(grads[0])), g_policy(THPVariable_Wrap(grads[1])),
        g_kl(THPVariable_Wrap(grads[2])), clip(PyFloat_FromDouble(in.clip_eps)), beta(PyFloat_FromDouble(in.beta));
    const PyRef grad(PyObject_CallFunctionObjArgs(general_grpo_gradient, cur.get(), old.get(), ref.get(), adv.get(), mask.get(),
                                                  g_loss.get(), g_policy.get(), g_kl.get(), clip.get(), beta.get(), nullptr));
    return {tensor_or_none(grad.get()), Tensor(), Tensor()};
  }
};

// ---------------------------------------------------------------------------
// Token scores, norms between blocks, eight-bit copies: the everyday calls of backends/rocm/logprob/token_scores.py,
// backends/rocm/norm/block_norm.py and of checkpointed_swiglu in backends/rocm/ffn/ffn.py
// ---------------------------------------------------------------------------

// rlk_dtype of an element type, or -1.
int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return RLK_DTYPE_BF16;
    case at::kHalf: return RLK_DTYPE_FP16;
    case at::kFloat: return RLK_DTYPE_FP32;
    default: return -1;
  }
}
bool everyday_floats(const Tensor& t) { return t.defined() && dtype_code(t) >= 0 && everyday(t, t.scalar_type()); }
bool everyday_floats(const Tensor& t, const Tensor& beside) { return everyday_floats(t) && t.get_device() == beside.get_device(); }
void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* writable(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }
PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }  // (None for an undefined tensor)

// Tensors of which some may be missing, saved for a backward, and back at their places.
void save_some(AutogradContext* ctx, const variable_list& tensors) {
  variable_list saved;
  int64_t which = 0;
  for (size_t i = 0; i < tensors.size(); ++i) {
    if (!tensors[i].defined()) continue;
    which |= (int64_t)1 << i;
    saved.push_back(tensors[i]);
  }
  ctx->save_for_backward(std::move(saved));
  ctx->saved_data["which"] = which;
}
variable_list saved_some(AutogradContext* ctx, size_t count) {
  const variable_list saved = ctx->get_saved_variables();
  const int64_t which = ctx->saved_data["which"].toInt();
  variable_list tensors(count);
  size_t next = 0;
  for (size_t i = 0; i < count; ++i)
    if (which >> i & 1) tensors[i] = saved[next++];
  return tensors;
}
// The tensors of a tuple of `count`, None as undefined ones.
variable_list tensors_of(const PyRef& tuple, int count) {
  variable_list out;
  for (int i = 0; i < count; ++i) out.push_back(tensor_or_none(PyTuple_GetItem(tuple.get(), i)));
  return out;
}

// Whether a gradient of the backward that runs, on a stream of its own, reaches from this node on one that was made on the default
// stream. The engine lets that stream wait for the gradient. Under graph capture another stream thereby joins the capture, which the
// default stream cannot, so such a backward goes to the general functions, which refuse it there.
bool reaches_default_stream() {
  const std::shared_ptr<torch::autograd::Node> start = torch::autograd::get_current_node();
  if (start == nullptr) return false;
  const auto* const wanted = torch::autograd::get_current_graph_task_exec_info();  // null or empty: all nodes
  std::vector<torch::autograd::Node*> open = {start.get()};
  std::unordered_set<torch::autograd::Node*> seen = {start.get()};
  while (!open.empty()) {
    torch::autograd::Node* const node = open.back();
    open.pop_back();
    for (const torch::autograd::Edge& edge : node->next_edges()) {
      torch::autograd::Node* const next = edge.function.get();
      if (next == nullptr || !seen.insert(next).second) continue;
      if (wanted != nullptr && !wanted->empty()) {
        const auto at = wanted->find(next);
        if (at == wanted->end() || !at->second.should_execute()) continue;
      }
      const std::optional<c10::Stream> stream = next->stream();
      if (stream.has_value()) {
        const c10::impl::VirtualGuardImpl impl(stream->device_type());
        if (*stream == impl.getDefaultStream(stream->device()) && *stream != impl.getStream(stream->device())) return true;
      }
      open.push_back(next);
    }
  }
  return false;
}
bool leaves_capture() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None && reaches_default_stream(); }

struct ScoreInputs {
  Tensor logits, target, temp;
  int64_t real;
  int top_k;

  bool usual() const {
    return everyday_floats(logits) && everyday_matrix(logits) && logits.size(0) <= INT_MAX && logits.size(1) <= RLK_SCORES_MAX_VOCAB &&
           everyday(target, at::kLong, logits) && target.dim() == 1 && target.size(0) == logits.size(0) && target.is_contiguous() &&
           (!temp.defined() || (everyday(temp, at::kFloat, logits) && temp.dim() == 1 && temp.size(0) == logits.size(0) && temp.is_contiguous())) &&
           real > 0 && real <= logits.size(1) && top_k >= 0 && top_k <= RLK_SCORES_MAX_TOP_K && top_k <= real;
  }
};

// logp, lse, entropy and, for alternatives, their log-probabilities and ids.
variable_list scores(const ScoreInputs& in) {
  const int64_t rows = in.logits.size(0), vocab = in.logits.size(1);
  variable_list out = {empty({rows}, at::kFloat, in.logits), empty({rows}, at::kFloat, in.logits), empty({rows}, at::kFloat, in.logits)};
  if (in.top_k > 0) {
    out.push_back(empty({rows, in.top_k}, at::kFloat, in.logits));
    out.push_back(empty({rows, in.top_k}, at::kLong, in.logits));
  }
  const size_t bytes = scores_workspace_entry((int)rows, in.top_k);
  const Tensor workspace = empty({(int64_t)bytes}, at::kByte, in.logits);
  check_status(scores_entry(in.logits.data_ptr(), dtype_code(in.logits), vocab, static_cast<const int64_t*>(in.target.data_ptr()),
                            floats(in.temp), (int)rows, vocab, in.real, in.top_k, writable(out[0]), writable(out[1]),
                            writable(out[2]), in.top_k > 0 ? writable(out[3]) : nullptr,
                            in.top_k > 0 ? static_cast<int64_t*>(out[4].data_ptr()) : nullptr, workspace.data_ptr(), bytes,
                            stream_of(in.logits)),
               "rlk_logits_scores failed");
  return out;
}

struct ScoresFn : torch::autograd::Function<ScoresFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const ScoreInputs* in) {
    variable_list out = scores(*in);
    save_some(ctx, {logits, in->target, in->temp, out[1], out[2], out.size() > 4 ? out[4] : Tensor()});
    ctx->saved_data["real"] = in->real;
    ctx->set_materialize_grads(false);
    if (out.size() > 4) ctx->mark_non_differentiable({out[4]});
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    grads.resize(4);  // of logp, lse, entropy and the alternatives' log-probabilities
    if (!grads[0].defined() && !grads[1].defined() && !grads[2].defined() && !grads[3].defined()) return {Tensor(), Tensor()};
    const variable_list s = saved_some(ctx, 6);
    const Tensor &lse = s[3], &entropy = s[4], &ids = s[5];
    const int64_t real = ctx->saved_data["real"].toInt();
    const int top_k = ids.defined() ? (int)ids.size(1) : 0;
    const ScoreInputs in{s[0], s[1], s[2], real, top_k};
    bool values = !at::GradMode::is_enabled() && everyday_thread() && !leaves_capture() && in.usual() && everyday(lse, at::kFloat, in.logits) &&
                  everyday(entropy, at::kFloat, in.logits) && (!ids.defined() || everyday(ids, at::kLong, in.logits));
    const int64_t rows = values ? in.logits.size(0) : 0;
    for (int i = 0; values && i < 4; ++i)
      values = !grads[i].defined() || (everyday(grads[i], at::kFloat, in.logits) && grads[i].is_contiguous() &&
                                       grads[i].numel() == rows * (i == 3 ? top_k : 1));
    if (values) {
      const c10::OptionalDeviceGuard guard(in.logits.device());
      const int64_t vocab = in.logits.size(1);
      const Tensor grad = empty({rows, vocab}, in.logits.scalar_type(), in.logits);
      check_status(scores_bwd_entry(in.logits.data_ptr(), dtype_code(in.logits), vocab, static_cast<const int64_t*>(in.target.data_ptr()),
                                    floats(in.temp), floats(lse), floats(entropy), floats(grads[0]), floats(grads[1]), floats(grads[2]),
                                    static_cast<const int64_t*>(address(ids)), floats(grads[3]), top_k, grad.data_ptr(),
                                    dtype_code(in.logits), vocab, vocab, (int)rows, vocab, real, stream_of(in.logits)),
                   "rlk_logits_scores_backward failed");
      return {grad, Tensor()};
    }
    const pybind11::gil_scoped_acquire gil;
    const PyRef args(PyTuple_New(11));
    for (int i = 0; i < 6; ++i) PyTuple_SET_ITEM(args.get(), i, wrap(s[i]));
    PyTuple_SET_ITEM(args.get(), 6, PyLong_FromLongLong(real));
    for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(args.get(), 7 + i, wrap(grads[i]));
    const PyRef grad(PyObject_CallObject(general_scores_gradient, args.get()));
    return {tensor_or_none(grad.get()), Tensor()};
  }
};

struct LinearScoreInputs {
  Tensor hidden, weight, target, temp, logits;  // logits: where they go and stay
  int64_t real;
  int top_k;

  bool usual() const {
    return projects(hidden, weight) && weight.size(0) <= RLK_SCORES_MAX_VOCAB && everyday(target, at::kLong, hidden) && target.dim() == 1 &&
           target.size(0) == hidden.size(0) && target.is_contiguous() &&
           (!temp.defined() || (everyday(temp, at::kFloat, hidden) && temp.dim() == 1 && temp.size(0) == hidden.size(0) && temp.is_contiguous())) &&
           everyday(logits, at::kFloat, hidden) && logits.dim() == 2 && logits.is_contiguous() && logits.size(0) == hidden.size(0) &&
           logits.size(1) == (weight.size(0) + 63) / 64 * 64 && real > 0 && real <= weight.size(0) && top_k >= 0 &&
           top_k <= RLK_SCORES_MAX_TOP_K && top_k <= real;
  }
};

variable_list linear_scores(const LinearScoreInputs& in) {
  const int64_t tokens = in.hidden.size(0), d = in.hidden.size(1), vocab = in.weight.size(0);
  variable_list out = {empty({tokens}, at::kFloat, in.hidden), empty({tokens}, at::kFloat, in.hidden), empty({tokens}, at::kFloat, in.hidden)};
  if (in.top_k > 0) {
    out.push_back(empty({tokens, in.top_k}, at::kFloat, in.hidden));
    out.push_back(empty({tokens, in.top_k}, at::kLong, in.hidden));
  }
  const size_t bytes = linear_scores_workspace_entry((int)tokens, (int)vocab, in.top_k);
  const Tensor workspace = empty({(int64_t)bytes}, at::kByte, in.hidden);
  check_status(linear_scores_entry(in.hidden.data_ptr(), d, in.weight.data_ptr(), d, static_cast<const int64_t*>(in.target.data_ptr()), nullptr,
                                   floats(in.temp), writable(out[0]), writable(out[1]), writable(out[2]),
                                   in.top_k > 0 ? writable(out[3]) : nullptr,
                                   in.top_k > 0 ? static_cast<int64_t*>(out[4].data_ptr()) : nullptr, writable(in.logits), in.logits.size(1),
                                   workspace.data_ptr(), bytes, (int)tokens, (int)d, (int)vocab, (int)in.real, in.top_k, stream_of(in.hidden)),
               "rlk_linear_scores_fwd failed");
  return out;
}

// The scores of a fused linear-LogP whose logits are kept (_LinearScores in backends/rocm/logprob/token_scores.py).
struct LinearScoresFn : torch::autograd::Function<LinearScoresFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const LinearScoreInputs* in) {
    variable_list out = linear_scores(*in);
    save_some(ctx, {hidden, weight, in->target, in->temp, out[1], out[2], out.size() > 4 ? out[4] : Tensor(), in->logits});
    ctx->saved_data["real"] = in->real;
    ctx->set_materialize_grads(false);
    if (out.size() > 4) ctx->mark_non_differentiable({out[4]});
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    grads.resize(4);
    if (!grads[0].defined() && !grads[1].defined() && !grads[2].defined() && !grads[3].defined()) return {Tensor(), Tensor(), Tensor()};
    const variable_list s = saved_some(ctx, 8);
    const Tensor &lse = s[4], &entropy = s[5], &ids = s[6];
    const int64_t real = ctx->saved_data["real"].toInt();
    const int top_k = ids.defined() ? (int)ids.size(1) : 0;
    const LinearScoreInputs in{s[0], s[1], s[2], s[3], s[7], real, top_k};
    const bool need_hidden = ctx->needs_input_grad(0), need_weight = ctx->needs_input_grad(1);
    bool values = !at::GradMode::is_enabled() && everyday_thread() && !leaves_capture() && in.usual() && everyday(lse, at::kFloat, in.hidden) &&
                  everyday(entropy, at::kFloat, in.hidden) && (!ids.defined() || everyday(ids, at::kLong, in.hidden));
    const int64_t tokens = values ? in.hidden.size(0) : 0;
    for (int i = 0; values && i < 4; ++i)
      values = !grads[i].defined() || (everyday(grads[i], at::kFloat, in.hidden) && grads[i].is_contiguous() &&
                                       grads[i].numel() == tokens * (i == 3 ? top_k : 1));
    if (values) {
      const c10::OptionalDeviceGuard guard(in.hidden.device());
      const int64_t d = in.hidden.size(1), vocab = in.weight.size(0), stride = dlogits_stride_entry((int)vocab);
      const Tensor dz = empty({tokens, stride}, kBf16, in.hidden);
      check_status(scores_bwd_entry(in.logits.data_ptr(), RLK_DTYPE_FP32, in.logits.size(1), static_cast<const int64_t*>(in.target.data_ptr()),
                                    floats(in.temp), floats(lse), floats(entropy), floats(grads[0]), floats(grads[1]), floats(grads[2]),
                                    static_cast<const int64_t*>(address(ids)), floats(grads[3]), top_k, dz.data_ptr(), RLK_DTYPE_BF16, stride,
                                    stride, (int)tokens, vocab, real, stream_of(in.hidden)),
                   "rlk_logits_scores_backward failed");
      const Tensor d_hidden = need_hidden ? empty({tokens, d}, kBf16, in.hidden) : Tensor();
      const Tensor d_weight = need_weight ? empty({vocab, d}, kBf16, in.hidden) : Tensor();
      check_status(dlogits_bwd_entry(dz.data_ptr(), in.hidden.data_ptr(), d, in.weight.data_ptr(), d, address(d_hidden), d, address(d_weight),
                                     d, (int)tokens, (int)d, (int)vocab, stream_of(in.hidden)),
                   "rlk_linear_dlogits_bwd failed");
      return {d_hidden, d_weight, Tensor()};
    }
    const pybind11::gil_scoped_acquire gil;
    const PyRef args(PyTuple_New(15));
    for (int i = 0; i < 8; ++i) PyTuple_SET_ITEM(args.get(), i, wrap(s[i]));
    PyTuple_SET_ITEM(args.get(), 8, PyLong_FromLongLong(real));
    for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(args.get(), 9 + i, wrap(grads[i]));
    PyTuple_SET_ITEM(args.get(), 13, PyBool_FromLong(need_hidden));
    PyTuple_SET_ITEM(args.get(), 14, PyBool_FromLong(need_weight));
    const PyRef two(PyObject_CallObject(general_linear_scores, args.get()));
    const variable_list out = tensors_of(two, 2);
    return {out[0], out[1], Tensor()};
  }
};

struct NormInputs {
  Tensor block, residual, gate, post, pre;  // rows [tokens, width]; all but the residual may be missing
  int kind;                                 // rlk_gate
  double eps, scale;

  // The type of block and normed: without a block that of the weight (an fp32 weight: of the residual).
  at::ScalarType type() const { return block.defined() ? block.scalar_type() : residual.scalar_type(); }
  bool of_type(const Tensor& t) const {
    return everyday_floats(t, residual) && t.is_contiguous() && (t.scalar_type() == type() || t.scalar_type() == at::kFloat);
  }
  bool usual() const {
    if (!(eps >= 0.0) || !everyday_floats(residual) || !everyday_matrix(residual) || residual.size(1) > RLK_NORM_MAX_WIDTH || residual.size(0) > INT_MAX) return false;
    const int64_t width = residual.size(1);
    if (block.defined() && !(everyday_floats(block, residual) && block.sizes() == residual.sizes() && block.is_contiguous())) return false;
    if (!of_type(residual)) return false;
    for (const Tensor* w : {&post, &pre})
      if (w->defined() && !(of_type(*w) && w->dim() == 1 && w->size(0) == width)) return false;
    if (kind == RLK_GATE_NONE) return !gate.defined();
    const int64_t cells = kind == RLK_GATE_CHANNEL ? width : kind == RLK_GATE_TOKEN ? residual.size(0) : residual.numel();
    return of_type(gate) && gate.numel() == cells;
  }
  rlk_block_norm describe(const Tensor& rstd) const {
    const int64_t width = residual.size(1);
    rlk_block_norm n{};
    n.block = address(block);
    n.residual = residual.data_ptr();
    n.gate = address(gate);
    n.post_weight = address(post);
    n.pre_weight = address(pre);
    n.rstd = writable(rstd);
    n.block_row_stride = n.residual_row_stride = width;
    n.gate_row_stride = kind == RLK_GATE_TOKEN ? 1 : width;
    n.tokens = residual.size(0);
    n.width = (int)width;
    n.dtype = block.defined() ? dtype_code(block) : dtype_code(residual);
    n.residual_dtype = dtype_code(residual);
    n.gate_kind = kind;
    n.gate_dtype = gate.defined() ? dtype_code(gate) : n.dtype;
    n.post_dtype = post.defined() ? dtype_code(post) : n.dtype;
    n.pre_dtype = pre.defined() ? dtype_code(pre) : n.dtype;
    n.eps = (float)eps;
    n.residual_scale = (float)scale;
    return n;
  }
};

// total (with a block) and normed (with a weight for it), in the residual's shape `shape`
variable_list norm_forward(const NormInputs& in, const Tensor& rstd, at::IntArrayRef shape) {
  const rlk_block_norm n = in.describe(rstd);
  const Tensor total = in.block.defined() ? empty(shape, in.residual.scalar_type(), in.residual) : Tensor();
  const Tensor normed = in.pre.defined() ? empty(shape, in.type(), in.residual) : Tensor();
  check_status(norm_entry(&n, address(total), address(normed), stream_of(in.residual)), "rlk_block_norm_forward failed");
  return {total, normed};
}

struct NormFn : torch::autograd::Function<NormFn> {
  using Maybe = std::optional<Tensor>;

  // (the inputs once more as arguments of their own: those are what autograd sees)
  static variable_list forward(AutogradContext* ctx, const Maybe& block, const Tensor& residual, const Maybe& gate, const Maybe& post,
                               const Maybe& pre, const NormInputs* in, at::IntArrayRef shape) {
    const Tensor rstd = empty({2, in->residual.size(0)}, at::kFloat, in->residual);
    const variable_list out = norm_forward(*in, rstd, shape);
    auto known = [](const Maybe& t) { return t.has_value() ? *t : Tensor(); };
    save_some(ctx, {known(block), residual, known(gate), known(post), known(pre), rstd});
    ctx->saved_data["kind"] = (int64_t)in->kind;
    ctx->saved_data["eps"] = in->eps;
    ctx->saved_data["scale"] = in->scale;
    ctx->saved_data["total"] = out[0].defined();
    ctx->set_materialize_grads(false);
    variable_list made;
    for (const Tensor& t : out)
      if (t.defined()) made.push_back(t);
    return made;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(7);
    const bool with_total = ctx->saved_data["total"].toBool();
    const Tensor g_total = with_total ? grads[0] : Tensor();
    const Tensor g_normed = with_total ? (grads.size() > 1 ? grads[1] : Tensor()) : grads[0];
    if (!g_total.defined() && !g_normed.defined()) return result;
    const variable_list s = saved_some(ctx, 6);
    auto rows = [](const Tensor& t) { return t.defined() && t.dim() != 2 && t.numel() > 0 ? t.reshape({-1, t.size(-1)}) : t; };
    NormInputs in{rows(s[0]), rows(s[1]), s[2], s[3], s[4], (int)ctx->saved_data["kind"].toInt(), ctx->saved_data["eps"].toDouble(),
                  ctx->saved_data["scale"].toDouble()};
    const Tensor& rstd = s[5];
    bool values = !at::GradMode::is_enabled() && everyday_thread() && !leaves_capture() && in.usual() && everyday(rstd, at::kFloat, in.residual);
    if (values && g_total.defined())
      values = everyday(g_total, in.residual.scalar_type(), in.residual) && g_total.is_contiguous() && g_total.numel() == in.residual.numel();
    if (values && g_normed.defined())
      values = everyday(g_normed, in.type(), in.residual) && g_normed.is_contiguous() && g_normed.numel() == in.residual.numel();
    if (values) {
      const c10::OptionalDeviceGuard guard(in.residual.device());
      // needs_input_grad() counts the tensors that were defined
      int place = 0;
      for (int i = 0; i < 5; ++i) {
        if (!s[i].defined()) continue;
        if (ctx->needs_input_grad(place++)) result[i] = empty(s[i].sizes(), s[i].scalar_type(), in.residual);
      }
      const rlk_block_norm n = in.describe(rstd);
      const size_t bytes = norm_workspace_entry(n.tokens, n.width);
      const Tensor workspace = empty({(int64_t)bytes}, at::kByte, in.residual);
      check_status(norm_bwd_entry(&n, address(g_total), address(g_normed), address(result[0]), address(result[1]), address(result[2]),
                                  address(result[3]), address(result[4]), workspace.data_ptr(), bytes, stream_of(in.residual)),
                   "rlk_block_norm_backward failed");
      return result;
    }
    const pybind11::gil_scoped_acquire gil;
    const PyRef args(PyTuple_New(16));
    for (int i = 0; i < 6; ++i) PyTuple_SET_ITEM(args.get(), i, wrap(s[i]));
    PyTuple_SET_ITEM(args.get(), 6, PyLong_FromLong(in.kind));
    PyTuple_SET_ITEM(args.get(), 7, PyFloat_FromDouble(in.eps));
    PyTuple_SET_ITEM(args.get(), 8, PyFloat_FromDouble(in.scale));
    PyTuple_SET_ITEM(args.get(), 9, wrap(g_total));
    PyTuple_SET_ITEM(args.get(), 10, wrap(g_normed));
    int place = 0;
    for (int i = 0; i < 5; ++i) {
      const bool need = s[i].defined() && ctx->needs_input_grad(place);
      if (s[i].defined()) ++place;
      PyTuple_SET_ITEM(args.get(), 11 + i, PyBool_FromLong(need));
    }
    const PyRef five(PyObject_CallObject(general_norm_gradients, args.get()));
    const variable_list out = tensors_of(five, 5);
    for (int i = 0; i < 5; ++i) result[i] = out[i];
    return result;
  }
};

bool takes_swiglu(const Tensor& gate, const Tensor& up) {
  return everyday_floats(gate) && gate.dim() >= 1 && gate.is_contiguous() && gate.numel() > 0 && gate.size(-1) <= (1 << 28) &&
         everyday(up, gate.scalar_type(), gate) && up.is_contiguous() && up.sizes() == gate.sizes();
}

struct Mx8SwigluFn : torch::autograd::Function<Mx8SwigluFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& gate, const Tensor& up) {
    const int64_t cols = gate.size(-1), rows = gate.numel() / cols, runs = (cols + 31) / 32;
    const Tensor y = empty(gate.sizes(), gate.scalar_type(), gate);
    Tensor codes[2], scales[2];
    for (int i = 0; i < 2; ++i) {
      codes[i] = empty({rows, cols}, at::kChar, gate);
      scales[i] = empty({rows, runs}, at::kByte, gate);
    }
    check_status(mx8_swiglu_entry(gate.data_ptr(), cols, up.data_ptr(), cols, dtype_code(gate), y.data_ptr(),
                                  static_cast<int8_t*>(codes[0].data_ptr()), static_cast<uint8_t*>(scales[0].data_ptr()),
                                  static_cast<int8_t*>(codes[1].data_ptr()), static_cast<uint8_t*>(scales[1].data_ptr()), rows, (int)cols,
                                  stream_of(gate)),
                 "rlk_mx8_swiglu_forward failed");
    ctx->save_for_backward({codes[0], scales[0], codes[1], scales[1]});
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor& dy = grads[0];
    const int64_t cols = s[0].size(1), rows = s[0].size(0);
    bool values = !at::GradMode::is_enabled() && everyday_thread() && !leaves_capture() && everyday_floats(dy) && dy.is_contiguous() && dy.numel() == rows * cols;
    for (int i = 0; values && i < 4; ++i) values = everyday(s[i], i % 2 ? at::kByte : at::kChar, dy) && s[i].is_contiguous();
    if (values) {
      const c10::OptionalDeviceGuard guard(dy.device());
      const Tensor d_gate = empty(dy.sizes(), dy.scalar_type(), dy), d_up = empty(dy.sizes(), dy.scalar_type(), dy);
      check_status(mx8_swiglu_bwd_entry(dy.data_ptr(), cols, dtype_code(dy), static_cast<const int8_t*>(s[0].data_ptr()),
                                        static_cast<const uint8_t*>(s[1].data_ptr()), static_cast<const int8_t*>(s[2].data_ptr()),
                                        static_cast<const uint8_t*>(s[3].data_ptr()), d_gate.data_ptr(), d_up.data_ptr(), nullptr, rows,
                                        (int)cols, stream_of(dy)),
                   "rlk_mx8_swiglu_backward failed");
      return {ctx->needs_input_grad(0) ? d_gate : Tensor(), ctx->needs_input_grad(1) ? d_up : Tensor()};
    }
    const pybind11::gil_scoped_acquire gil;
    const PyRef args(PyTuple_New(5));
    PyTuple_SET_ITEM(args.get(), 0, wrap(dy));
    for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(args.get(), 1 + i, wrap(s[i]));
    const PyRef two(PyObject_CallObject(general_swiglu_gradients, args.get()));
    return tensors_of(two, 2);
  }
};

// ---------------------------------------------------------------------------
// The Python module
// ---------------------------------------------------------------------------

PyObject* none() { Py_RETURN_NONE; }

// linear(a, weight) -> a @ weight.T, differentiable where an operand asks for it, or None
PyObject* py_linear(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 2 || gemm_entry == nullptr) return none();
  const Tensor *a = exact_tensor(args[0]), *weight = exact_tensor(args[1]);
  if (a == nullptr || weight == nullptr || !everyday_caller() || !projects(*a, *weight)) return none();
  const bool differentiable = at::GradMode::is_enabled() && (a->requires_grad() || weight->requires_grad());
  Tensor out;
  {
    const pybind11::gil_scoped_release no_gil;
    const c10::OptionalDeviceGuard guard(a->device());
    out = differentiable ? LinearFn::apply(*a, *weight) : project(*a, *weight);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// packed_ffn(x, gate_up, down) -> down @ swiglu(gate_up @ x), or None
PyObject* py_packed_ffn(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 3 || gemm_entry == nullptr) return none();
  const Tensor *x = exact_tensor(args[0]), *gate_up = exact_tensor(args[1]), *down = exact_tensor(args[2]);
  if (x == nullptr || gate_up == nullptr || down == nullptr || !everyday_caller() || !takes_ffn(*x, *gate_up, *down)) return none();
  if (at::GradMode::is_enabled() && (x->requires_grad() || gate_up->requires_grad() || down->requires_grad())) return none();
  Tensor out;
  {
    const pybind11::gil_scoped_release no_gil;
    const c10::OptionalDeviceGuard guard(x->device());
    out = packed_ffn(*x, *gate_up, *down);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// ffn(x, gate, up, down) -> down @ (silu(gate @ x) * (up @ x)) with the gradients of all four, or None
PyObject* py_ffn(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 4 || gemm_entry == nullptr) return none();
  const Tensor* t[4];
  for (int i = 0; i < 4; ++i) {
    t[i] = exact_tensor(args[i]);
    if (t[i] == nullptr) return none();
  }
  if (!everyday_caller() || !takes_ffn_training(*t[0], *t[1], *t[2], *t[3])) return none();
  Tensor out;
  {
    const pybind11::gil_scoped_release no_gil;
    const c10::OptionalDeviceGuard guard(t[0]->device());
    out = FfnFn::apply(*t[0], *t[1], *t[2], *t[3]);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// grpo(cur, old, ref, adv, mask or None, clip_eps, beta) -> (loss, policy, kl, ratio, k3), or None
PyObject* py_grpo(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 7 || gemm_entry == nullptr) return none();
  const Tensor* t[5] = {};
  for (int i = 0; i < 5; ++i) {
    if (i == 4 && args[i] == Py_None) break;
    t[i] = exact_tensor(args[i]);
    if (t[i] == nullptr) return none();
  }
  for (int i = 5; i < 7; ++i)
    if (!PyFloat_CheckExact(args[i]) && !PyLong_CheckExact(args[i])) return none();
  GrpoInputs in{*t[0], *t[1], *t[2], *t[3], t[4] != nullptr ? *t[4] : Tensor(), PyFloat_AsDouble(args[5]), PyFloat_AsDouble(args[6])};
  if (PyErr_Occurred()) throw python_error();
  if (!everyday_caller() || !in.usual()) return none();
  variable_list three;
  GrpoOutputs out;
  {
    const pybind11::gil_scoped_release no_gil;
    const c10::OptionalDeviceGuard guard(in.cur.device());
    if (at::GradMode::is_enabled() && in.cur.requires_grad()) {
      for (Tensor* s : {&in.old, &in.ref, &in.adv})
        if (s->requires_grad()) *s = s->detach();
      three = GrpoFn::apply(in.cur, &in, &out);
    } else {
      out = grpo(in);
      three = out.out3.unbind(0);
    }
  }
  const PyRef loss(THPVariable_Wrap(three[0])), policy(THPVariable_Wrap(three[1])), kl(THPVariable_Wrap(three[2])),
      ratio(THPVariable_Wrap(out.ratio)), k3(THPVariable_Wrap(out.k3));
  return PyTuple_Pack(5, loss.get(), policy.get(), kl.get(), ratio.get(), k3.get());
  END_HANDLE_TH_ERRORS
}

// A Python argument that is a Tensor, a Parameter or None; false for anything else.
bool tensor_or_nothing(PyObject* o, Tensor* t) {
  if (o == Py_None) return true;
  const Tensor* const exact = exact_tensor(o);
  if (exact == nullptr) return false;
  *t = *exact;
  return true;
}

// scores(logits, target, temperature or None, real vocabulary, top_k) -> (logp, lse, entropy, top_logp or None, top_ids or None), or None
PyObject* py_scores(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 5 || scores_entry == nullptr) return none();
  ScoreInputs in;
  if (!tensor_or_nothing(args[0], &in.logits) || !tensor_or_nothing(args[1], &in.target) || !tensor_or_nothing(args[2], &in.temp) ||
      !PyLong_CheckExact(args[3]) || !PyLong_CheckExact(args[4]))
    return none();
  int overflow[2];
  in.real = PyLong_AsLongLongAndOverflow(args[3], &overflow[0]);
  const long top_k = PyLong_AsLongAndOverflow(args[4], &overflow[1]);
  if (overflow[0] != 0 || overflow[1] != 0 || top_k < 0 || top_k > RLK_SCORES_MAX_TOP_K) return none();
  in.top_k = (int)top_k;
  if (!everyday_caller() || !in.usual()) return none();
  variable_list out;
  {
    const pybind11::gil_scoped_release no_gil;
    const c10::OptionalDeviceGuard guard(in.logits.device());
    out = at::GradMode::is_enabled() && in.logits.requires_grad() ? ScoresFn::apply(in.logits, &in) : scores(in);
  }
  out.resize(5);
  const PyRef logp(wrap(out[0])), lse(wrap(out[1])), entropy(wrap(out[2])), top_logp(wrap(out[3])), top_ids(wrap(out[4]));
  return PyTuple_Pack(5, logp.get(), lse.get(), entropy.get(), top_logp.get(), top_ids.get());
  END_HANDLE_TH_ERRORS
}

// reaches_default_stream() -> whether a gradient of the backward that runs, on another stream, reaches a node made on the default one
PyObject* py_reaches_default_stream(PyObject*, PyObject*) {
  HANDLE_TH_ERRORS
  return PyBool_FromLong(reaches_default_stream());
  END_HANDLE_TH_ERRORS
}

// linear_scores(hidden, weight, target, temperature or None, real vocabulary, top_k, logits to be kept) -> as scores(), or None
PyObject* py_linear_scores(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 7 || linear_scores_entry == nullptr) return none();
  LinearScoreInputs in;
  if (!tensor_or_nothing(args[0], &in.hidden) || !tensor_or_nothing(args[1], &in.weight) || !tensor_or_nothing(args[2], &in.target) ||
      !tensor_or_nothing(args[3], &in.temp) || !tensor_or_nothing(args[6], &in.logits) || !PyLong_CheckExact(args[4]) ||
      !PyLong_CheckExact(args[5]))
    return none();
  int overflow[2];
  in.real = PyLong_AsLongLongAndOverflow(args[4], &overflow[0]);
  const long top_k = PyLong_AsLongAndOverflow(args[5], &overflow[1]);
  if (overflow[0] != 0 || overflow[1] != 0 || top_k < 0 || top_k > RLK_SCORES_MAX_TOP_K) return none();
  in.top_k = (int)top_k;
  if (!everyday_caller() || !in.usual()) return none();
  variable_list out;
  {
    const pybind11::gil_scoped_release no_gil;
    const c10::OptionalDeviceGuard guard(in.hidden.device());
    const bool differentiable = at::GradMode::is_enabled() && (in.hidden.requires_grad() || in.weight.requires_grad());
    out = differentiable ? LinearScoresFn::apply(in.hidden, in.weight, &in) : linear_scores(in);
  }
  out.resize(5);
  const PyRef logp(wrap(out[0])), lse(wrap(out[1])), entropy(wrap(out[2])), top_logp(wrap(out[3])), top_ids(wrap(out[4]));
  return PyTuple_Pack(5, logp.get(), lse.get(), entropy.get(), top_logp.get(), top_ids.get());
  END_HANDLE_TH_ERRORS
}

// norm(block or None, residual, gate or None, post weight or None, weight or None, eps, scale) -> (total or None, normed or None), or None
PyObject* py_norm(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 7 || norm_entry == nullptr) return none();
  Tensor t[5];  // block, residual, gate, post, pre
  for (int i = 0; i < 5; ++i)
    if (!tensor_or_nothing(args[i], &t[i])) return none();
  for (int i = 5; i < 7; ++i)
    if (!PyFloat_CheckExact(args[i]) && !PyLong_CheckExact(args[i])) return none();
  const double eps = PyFloat_AsDouble(args[5]), scale = PyFloat_AsDouble(args[6]);
  if (PyErr_Occurred()) throw python_error();
  if (!everyday_caller() || !everyday_floats(t[1]) || t[1].dim() < 1 || !t[1].is_contiguous() || t[1].numel() == 0) return none();
  if (t[0].defined() && !(everyday_floats(t[0], t[1]) && t[0].is_contiguous() && t[0].sizes() == t[1].sizes())) return none();
  if (!t[0].defined() && (!t[4].defined() || t[2].defined() || t[3].defined())) return none();
  const at::IntArrayRef shape = t[1].sizes();
  int kind = RLK_GATE_NONE;
  if (t[2].defined()) {
    if (!everyday_floats(t[2], t[1])) return none();
    if (t[2].dim() == 1 && t[2].size(0) == shape.back()) kind = RLK_GATE_CHANNEL;
    else if (t[2].sizes() == shape) kind = RLK_GATE_FULL;
    else if (t[2].dim() == t[1].dim() && t[2].size(-1) == 1 && t[2].sizes().slice(0, shape.size() - 1) == shape.slice(0, shape.size() - 1)) kind = RLK_GATE_TOKEN;
    else return none();
  }
  // (views of rows are made where autograd does not look)
  NormInputs in;
  bool differentiable = false;
  {
    const at::NoGradGuard no_grad;
    auto rows = [](const Tensor& x) { return !x.defined() || x.dim() == 2 ? x : x.view({-1, x.size(-1)}); };
    in = NormInputs{rows(t[0]), rows(t[1]), t[2], t[3], t[4], kind, eps, scale};
  }
  if (!in.usual()) return none();
  for (const Tensor& x : t) differentiable |= x.defined() && x.requires_grad();
  variable_list out;
  {
    const pybind11::gil_scoped_release no_gil;
    const c10::OptionalDeviceGuard guard(t[1].device());
    if (differentiable && at::GradMode::is_enabled()) {
      auto maybe = [](const Tensor& x) { return x.defined() ? NormFn::Maybe(x) : NormFn::Maybe(); };
      out = NormFn::apply(maybe(t[0]), t[1], maybe(t[2]), maybe(t[3]), maybe(t[4]), &in, shape);
      if (!t[0].defined()) out.insert(out.begin(), Tensor());
      out.resize(2);
    } else {
      out = norm_forward(in, Tensor(), shape);
    }
  }
  const PyRef total(wrap(out[0])), normed(wrap(out[1]));
  return PyTuple_Pack(2, total.get(), normed.get());
  END_HANDLE_TH_ERRORS
}

// mx8_swiglu(gate, up) -> silu(gate) * up, differentiable through eight-bit copies, or None
PyObject* py_mx8_swiglu(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 2 || mx8_swiglu_entry == nullptr) return none();
  const Tensor *gate = exact_tensor(args[0]), *up = exact_tensor(args[1]);
  if (gate == nullptr || up == nullptr || !everyday_caller() || !takes_swiglu(*gate, *up)) return none();
  if (!at::GradMode::is_enabled() || !(gate->requires_grad() || up->requires_grad())) return none();
  Tensor y;
  {
    const pybind11::gil_scoped_release no_gil;
    const c10::OptionalDeviceGuard guard(gate->device());
    y = Mx8SwigluFn::apply(*gate, *up);
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

// mx8_encode(x [rows, columns]) -> (codes, scales), or None
PyObject* py_mx8_encode(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 1 || mx8_encode_entry == nullptr) return none();
  const Tensor* const x = exact_tensor(args[0]);
  if (x == nullptr || !everyday_caller() || !everyday_floats(*x) || !everyday_matrix(*x) || x->size(1) > (1 << 28)) return none();
  const int64_t rows = x->size(0), cols = x->size(1);
  Tensor codes, scales;
  {
    const pybind11::gil_scoped_release no_gil;
    const c10::OptionalDeviceGuard guard(x->device());
    codes = empty({rows, cols}, at::kChar, *x);
    scales = empty({rows, (cols + 31) / 32}, at::kByte, *x);
    check_status(mx8_encode_entry(x->data_ptr(), cols, dtype_code(*x), static_cast<int8_t*>(codes.data_ptr()),
                                  static_cast<uint8_t*>(scales.data_ptr()), rows, (int)cols, stream_of(*x)),
                 "rlk_mx8_encode failed");
  }
  const PyRef py_codes(wrap(codes)), py_scales(wrap(scales));
  return PyTuple_Pack(2, py_codes.get(), py_scales.get());
  END_HANDLE_TH_ERRORS
}

// bind(addresses of the entry points by name, the general gradients of the linear layer, the FFN, the GRPO loss, the token scores, the
// norm between blocks, the SwiGLU of eight-bit copies and the token scores of hidden states)
PyObject* py_bind(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *addresses, *linear, *ffn, *loss, *of_scores = Py_None, *of_norm = Py_None, *of_swiglu = Py_None, *of_linear_scores = Py_None;
  if (!PyArg_ParseTuple(args, "O!OOO|OOOO", &PyDict_Type, &addresses, &linear, &ffn, &loss, &of_scores, &of_norm, &of_swiglu, &of_linear_scores)) return nullptr;
  auto entry = [&](const char* name, auto& to) {
    PyObject* const at = PyDict_GetItemString(addresses, name);
    void* const address = at != nullptr ? PyLong_AsVoidPtr(at) : nullptr;
    if (PyErr_Occurred()) throw python_error();
    TORCH_CHECK(address != nullptr, "no address for ", name);
    to = reinterpret_cast<std::remove_reference_t<decltype(to)>>(address);
  };
  entry("rlk_last_error", last_error_entry);
  entry("rlk_linear_bwd_bf16", linear_bwd_entry);
  entry("rlk_det_gemm_swiglu_workspace_bytes", swiglu_workspace_entry);
  entry("rlk_det_gemm_swiglu_bf16", swiglu_entry);
  entry("rlk_det_gemm_swiglu_training_bf16", swiglu_training_entry);
  entry("rlk_swiglu_bwd", swiglu_bwd_entry);
  entry("rlk_grpo_workspace_bytes", grpo_workspace_entry);
  entry("rlk_grpo_ratio_kl_loss", grpo_entry);
  entry("rlk_grpo_ratio_kl_loss_bwd", grpo_bwd_entry);
  entry("rlk_logits_scores_workspace_bytes", scores_workspace_entry);
  entry("rlk_logits_scores_backward", scores_bwd_entry);
  entry("rlk_block_norm_workspace_bytes", norm_workspace_entry);
  entry("rlk_block_norm_backward", norm_bwd_entry);
  entry("rlk_mx8_swiglu_backward", mx8_swiglu_bwd_entry);
  entry("rlk_mx8_encode", mx8_encode_entry);
  for (const auto& [from, to] : {std::pair<PyObject*, PyObject**>{of_scores, &general_scores_gradient},
                                 {of_norm, &general_norm_gradients},
                                 {of_swiglu, &general_swiglu_gradients},
                                 {of_linear_scores, &general_linear_scores}}) {
    Py_INCREF(from);
    Py_XSETREF(*to, from);
  }
  entry("rlk_linear_scores_workspace_bytes", linear_scores_workspace_entry);
  entry("rlk_linear_dlogits_row_stride", dlogits_stride_entry);
  entry("rlk_linear_dlogits_bwd", dlogits_bwd_entry);
  entry("rlk_logits_scores", scores_entry);
  entry("rlk_linear_scores_fwd", linear_scores_entry);
  entry("rlk_block_norm_forward", norm_entry);
  entry("rlk_mx8_swiglu_forward", mx8_swiglu_entry);
  Py_INCREF(linear);
  Py_XSETREF(general_linear_gradients, linear);
  Py_INCREF(ffn);
  Py_XSETREF(general_ffn_gradients, ffn);
  Py_INCREF(loss);
  Py_XSETREF(general_grpo_gradient, loss);
  entry("rlk_det_gemm_bf16", gemm_entry);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_linear)), METH_FASTCALL, nullptr},
    {"packed_ffn", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_packed_ffn)), METH_FASTCALL, nullptr},
    {"ffn", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_ffn)), METH_FASTCALL, nullptr},
    {"grpo", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_grpo)), METH_FASTCALL, nullptr},
    {"scores", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_scores)), METH_FASTCALL, nullptr},
    {"reaches_default_stream", py_reaches_default_stream, METH_NOARGS, nullptr},
    {"linear_scores", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_linear_scores)), METH_FASTCALL, nullptr},
    {"norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_norm)), METH_FASTCALL, nullptr},
    {"mx8_swiglu", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_mx8_swiglu)), METH_FASTCALL, nullptr},
    {"mx8_encode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_mx8_encode)), METH_FASTCALL, nullptr},
    {"bind", py_bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_host() { return PyModule_Create(&module); }
