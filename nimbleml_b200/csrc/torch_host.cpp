// torch_host.cpp — the host side of the operators whose calls are short against
// Python's: layer norm and token log probabilities (over logits, and from the tied
// matrix on one rank) as autograd nodes, and the
// many-tensor AdamW step with its checks. Everything on the GPU goes through the
// C ABI (include/nimbleml_tied_ce.h); this file only checks arguments, allocates
// outputs and workspaces on torch's current stream, and keeps what the backward
// needs. Errors are Python's: ValueError for arguments, RuntimeError with the
// library's message for a failing call.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <optional>
#include <string>
#include <vector>

#include "nimbleml_tied_ce.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

void check_rc(int rc, const char* name) {
  TORCH_CHECK(rc == 0, name, " failed (", rc, "): ", nimble_tied_ce_last_error());
}

int dtype_or(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return NIMBLE_DTYPE_F32;
    case at::kHalf: return NIMBLE_DTYPE_F16;
    case at::kBFloat16: return NIMBLE_DTYPE_BF16;
    default: return -1;
  }
}
int dtype_of(const Tensor& t) {
  const int d = dtype_or(t);
  TORCH_CHECK_VALUE(d >= 0, "unsupported compute dtype torch.", at::toString(t.scalar_type()),
                    "; use float32, float16 or bfloat16");
  return d;
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

Tensor empty(at::IntArrayRef shape, const Tensor& like, at::ScalarType type) {
  return at::empty(shape, like.options().dtype(type).memory_format(c10::nullopt).requires_grad(false));
}

// These operators write through raw pointers, which neither a trace nor a tangent
// follows: a trace would keep the allocation of the results and none of the kernels,
// and a dual tensor (which does not require grad) would come out without its tangent.
void refuse_recording(const char* name) {
  TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                  !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY),
              name, " cannot be traced: the trace would not hold its kernels");
}
void refuse_tangent(const char* name, const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode(), name,
                              " has no forward-mode derivative, and an input has a tangent");
}
void refuse_transforms(const char* name, const Tensor& t) {
  refuse_recording(name);
  refuse_tangent(name, t);
}

// t in a type, contiguous; t itself, without a call to torch, where it is both.
Tensor as_type(const Tensor& t, at::ScalarType type) {
  if (t.scalar_type() == type && t.is_contiguous()) return t;
  return t.to(type).contiguous();
}

// (n, d) rows of x: a view where its rows are contiguous and do not overlap, else a
// copy; and their pitch.
Tensor rows_of(const Tensor& x, int64_t& n, int64_t& d, int64_t& pitch) {
  d = x.size(-1);
  Tensor r = x.dim() == 2 ? x : x.reshape({-1, d});
  n = r.size(0);
  if (r.stride(1) != 1 || (n > 1 && r.stride(0) < d)) r = r.contiguous();
  pitch = std::max(r.stride(0), d);
  return r;
}

// ------------------------------------------------------------------ layer norm
constexpr int64_t kMaxNorm = 8192;

struct NormArgs {
  Tensor x, gamma, beta;  // rows; parameters in the rows' type or fp32
  int64_t n, d, pitch;
};

NormArgs norm_args(const Tensor& x, const Tensor& gamma, const std::optional<Tensor>& beta) {
  NormArgs a;
  a.x = rows_of(x, a.n, a.d, a.pitch);
  const auto own = x.scalar_type();
  const bool same = gamma.scalar_type() == own && (!beta || beta->scalar_type() == own);
  const auto type = same ? own : at::kFloat;
  a.gamma = as_type(gamma, type);
  if (beta) a.beta = as_type(*beta, type);
  return a;
}

Tensor norm_forward(const NormArgs& a, const Tensor& x, double eps, Tensor* stats) {
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = empty(x.sizes(), x, x.scalar_type());
  float* mean = nullptr;
  if (stats) {
    *stats = empty({2, a.n}, x, at::kFloat);
    mean = stats->mutable_data_ptr<float>();
  }
  check_rc(nimble_layernorm_forward(a.x.const_data_ptr(), a.pitch, a.gamma.const_data_ptr(),
                                    a.beta.defined() ? a.beta.const_data_ptr() : nullptr, a.n, a.d,
                                    static_cast<float>(eps), dtype_of(a.x), dtype_of(a.gamma), y.mutable_data_ptr(),
                                    mean, stats ? mean + a.n : nullptr, stream_of(x)),
           "nimble_layernorm_forward");
  return y;
}

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& gamma, const std::optional<Tensor>& beta,
                        double eps) {
    const NormArgs a = norm_args(x, gamma, beta);
    Tensor stats;
    Tensor y = norm_forward(a, x, eps, &stats);
    ctx->save_for_backward({a.x, a.gamma, stats});
    ctx->saved_data["gamma"] = static_cast<int64_t>(gamma.scalar_type());
    ctx->saved_data["beta"] = beta ? static_cast<int64_t>(beta->scalar_type()) : int64_t(-1);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "layer_norm's backward is not differentiable itself");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &gamma = saved[1], &stats = saved[2];
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t n = x.size(0), d = x.size(1);
    const int64_t beta_type = ctx->saved_data["beta"].toInt();
    const Tensor gy = as_type(grads[0], x.scalar_type());
    Tensor gx = empty(gy.sizes(), x, x.scalar_type());
    Tensor gg = empty({d}, x, at::kFloat), gb;
    if (beta_type >= 0) gb = empty({d}, x, at::kFloat);
    size_t bytes = 0;
    check_rc(nimble_layernorm_backward_workspace_size(n, d, &bytes), "nimble_layernorm_backward_workspace_size");
    const Tensor ws = empty({static_cast<int64_t>(std::max<size_t>(bytes, 1))}, x, at::kByte);
    const float* mean = stats.const_data_ptr<float>();
    check_rc(nimble_layernorm_backward(gy.const_data_ptr(), x.const_data_ptr(), std::max(x.stride(0), d),
                                       gamma.const_data_ptr(), mean, mean + n, n, d, dtype_of(x), dtype_of(gamma),
                                       gx.mutable_data_ptr(), gg.mutable_data_ptr<float>(),
                                       gb.defined() ? gb.mutable_data_ptr<float>() : nullptr, ws.mutable_data_ptr(),
                                       bytes, stream_of(x)),
             "nimble_layernorm_backward");
    gg = as_type(gg, static_cast<at::ScalarType>(ctx->saved_data["gamma"].toInt()));
    if (gb.defined()) gb = as_type(gb, static_cast<at::ScalarType>(beta_type));
    return {gx, gg, gb, Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const Tensor& gamma, const std::optional<Tensor>& beta, double eps) {
  refuse_transforms("layer_norm", x);
  refuse_tangent("layer_norm", gamma);
  if (beta) refuse_tangent("layer_norm", *beta);
  TORCH_CHECK(x.is_cuda(), "layer_norm on B200 needs CUDA tensors; there is no CPU path");
  dtype_of(x);
  const int64_t d = x.dim() ? x.size(-1) : 0;
  auto check = [&](const Tensor& p, const char* name) {
    TORCH_CHECK_VALUE(p.dim() == 1 && p.size(0) == d, "Expected ", name, " of shape (", d, ",), got ", p.sizes());
    TORCH_CHECK_VALUE(p.device() == x.device(), name, " is on ", p.device(), ", x on ", x.device());
    dtype_of(p);
  };
  check(gamma, "gamma");
  if (beta) check(*beta, "beta");
  TORCH_CHECK_VALUE(d > 0 && d <= kMaxNorm, "layer_norm takes rows of 1 to ", kMaxNorm, " elements, got ", d);
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || gamma.requires_grad() || (beta && beta->requires_grad())))
    return LayerNormNode::apply(x, gamma, beta, eps);
  return norm_forward(norm_args(x, gamma, beta), x, eps, nullptr);
}

// -------------------------------------------------------- token log probabilities
struct RowsOut {
  Tensor x, logprob, entropy, stats, top_logprob, top_id;  // x: the rows as read; stats: max, ln sum
};

RowsOut rows_forward(const Tensor& logits, const Tensor& tokens, int64_t ignore_index, int64_t top_k, int64_t status) {
  const c10::cuda::CUDAGuard guard(logits.device());
  RowsOut o;
  int64_t n, v, pitch;
  o.x = rows_of(logits, n, v, pitch);
  const auto shape = logits.sizes().slice(0, logits.dim() - 1);
  o.logprob = empty(shape, logits, at::kFloat);
  o.entropy = empty(shape, logits, at::kFloat);
  o.stats = empty({2, n}, logits, at::kFloat);
  if (top_k) {
    std::vector<int64_t> wide(shape.begin(), shape.end());
    wide.push_back(top_k);
    o.top_logprob = empty(wide, logits, at::kFloat);
    o.top_id = empty(wide, logits, at::kLong);
  }
  float* stats = o.stats.mutable_data_ptr<float>();
  check_rc(nimble_token_logprobs_forward(
               o.x.const_data_ptr(), pitch, tokens.const_data_ptr<int64_t>(), n, v, dtype_of(logits), ignore_index,
               static_cast<int>(top_k), o.logprob.mutable_data_ptr<float>(), o.entropy.mutable_data_ptr<float>(),
               stats, stats + n, top_k ? o.top_logprob.mutable_data_ptr<float>() : nullptr,
               top_k ? o.top_id.mutable_data_ptr<int64_t>() : nullptr, reinterpret_cast<int*>(status),
               stream_of(logits)),
           "nimble_token_logprobs_forward");
  return o;
}

Tensor grad_rows(const Tensor& g) { return g.defined() ? as_type(g, at::kFloat) : g; }
const float* ptr_or_null(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }

struct TokenLogProbsNode : torch::autograd::Function<TokenLogProbsNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, int64_t ignore_index,
                               int64_t top_k, int64_t status) {
    RowsOut o = rows_forward(logits, tokens, ignore_index, top_k, status);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({o.x, tokens, o.stats, o.entropy});
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["shape"] = logits.sizes().vec();
    variable_list out{o.logprob, o.entropy};
    if (top_k) {
      ctx->mark_non_differentiable({o.top_logprob, o.top_id});
      out.push_back(o.top_logprob);
      out.push_back(o.top_id);
    }
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "the log probabilities' backward is not differentiable itself");
    if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &tokens = saved[1], &stats = saved[2], &entropy = saved[3];
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t n = x.size(0), v = x.size(1), pitch = std::max(x.stride(0), v);
    // Rows of whole 16 bytes where the logits have them, so that both sides use vectors.
    const int64_t per16 = 16 / static_cast<int64_t>(x.element_size());
    const int64_t grad_pitch = pitch % per16 == 0 ? (v + per16 - 1) / per16 * per16 : v;
    Tensor g = empty({n, grad_pitch}, x, x.scalar_type());
    const Tensor a = grad_rows(grads[0]), b = grad_rows(grads[1]);
    const float* s = stats.const_data_ptr<float>();
    check_rc(nimble_token_logprobs_backward(ptr_or_null(a), ptr_or_null(b), x.const_data_ptr(), pitch,
                                            tokens.const_data_ptr<int64_t>(), s, s + n,
                                            entropy.const_data_ptr<float>(), n, v, dtype_of(x),
                                            ctx->saved_data["ignore_index"].toInt(), g.mutable_data_ptr(), grad_pitch,
                                            stream_of(x)),
             "nimble_token_logprobs_backward");
    if (grad_pitch != v) g = g.narrow(1, 0, v);
    const auto shape = ctx->saved_data["shape"].toIntVector();
    if (shape.size() != 2) g = g.reshape(shape);
    return {g, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

py::tuple token_logprobs(const Tensor& logits, const Tensor& tokens, int64_t ignore_index, int64_t top_k,
                         int64_t status) {
  variable_list out;
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    out = TokenLogProbsNode::apply(logits, tokens, ignore_index, top_k, status);
  } else {
    RowsOut o = rows_forward(logits, tokens, ignore_index, top_k, status);
    out = {o.logprob, o.entropy};
    if (top_k) {
      out.push_back(o.top_logprob);
      out.push_back(o.top_id);
    }
  }
  if (top_k) return py::make_tuple(out[0], out[1], out[2], out[3]);
  return py::make_tuple(out[0], out[1], py::none(), py::none());
}

// ------------------------------------------------------- tied log probabilities
// The package's hooks around a tied call: `poll` raises what an earlier call reported,
// `check` waits for this one. No call queues a copy of the status word: a forward's last
// kernel raises the host's flag for all that the word holds by then, a backward's errors
// among them (a copy and its event took 7 of 38 us of a call with few tokens). A
// captured launch must not be joined by either hook.
py::object* status_hooks[2] = {nullptr, nullptr};
enum Hook { kPoll = 0, kCheck = 1 };
void set_status_hooks(py::object poll, py::object check) {
  for (py::object*& h : status_hooks) delete h;
  status_hooks[kPoll] = new py::object(std::move(poll));
  status_hooks[kCheck] = new py::object(std::move(check));
}
void status_hook(Hook which, const Tensor& t) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return;
  TORCH_CHECK(status_hooks[which], "set_status_hooks comes first");
  py::gil_scoped_acquire gil;
  try {
    (*status_hooks[which])(static_cast<int>(t.get_device()));
  } catch (py::error_already_set& e) {
    // As torch's own errors, which cross the autograd engine's threads.
    const std::string what = py::str(e.value());
    if (e.matches(PyExc_ValueError)) TORCH_CHECK_VALUE(false, what);
    TORCH_CHECK(false, what);
  }
}

// Where a forward on one shard writes: its statistics (4, N), or the results of a shard
// that is the whole vocabulary.
struct TiedOut {
  float *stats, *logprob, *entropy, *lse;
};
void tied_forward(const Tensor& h, const Tensor& w, const Tensor& tokens, int64_t v_offset, int64_t ignore_index,
                  const TiedOut& o, int64_t status, int64_t host_flag) {
  const int64_t n = h.size(0), d = h.size(1), v = w.size(0);
  size_t bytes = 0;
  check_rc(nimble_tied_logprobs_forward_workspace_size(n, d, v, dtype_of(h), &bytes),
           "nimble_tied_logprobs_forward_workspace_size");
  const Tensor ws = empty({static_cast<int64_t>(std::max<size_t>(bytes, 1))}, h, at::kByte);
  check_rc(nimble_tied_logprobs_forward(h.const_data_ptr(), w.const_data_ptr(), tokens.const_data_ptr<int64_t>(), n, d,
                                        v, v_offset, dtype_of(h), ignore_index, o.stats, o.logprob, o.entropy, o.lse,
                                        ws.mutable_data_ptr(), bytes, reinterpret_cast<int*>(status),
                                        reinterpret_cast<int*>(host_flag), stream_of(h)),
           "nimble_tied_logprobs_forward");
}

Tensor tied_shard_stats(const Tensor& h, const Tensor& w, const Tensor& tokens, int64_t v_offset, int64_t ignore_index,
                        int64_t status) {
  const c10::cuda::CUDAGuard guard(h.device());
  Tensor out = empty({4, h.size(0)}, h, at::kFloat);
  tied_forward(h, w, tokens, v_offset, ignore_index, {out.mutable_data_ptr<float>(), nullptr, nullptr, nullptr},
               status, 0);
  return out;
}

// Fills grad_hidden and fills or adds to grad_weights, those that are given.
void tied_backward(const std::optional<Tensor>& g_logprob, const std::optional<Tensor>& g_entropy, const Tensor& h,
                   const Tensor& w, const Tensor& tokens, const Tensor& lse, const Tensor& entropy, int64_t v_offset,
                   int64_t vocab_size, int64_t ignore_index, const std::optional<Tensor>& grad_hidden,
                   const std::optional<Tensor>& grad_weights, bool accumulate, int64_t slab_bytes, int64_t status) {
  const c10::cuda::CUDAGuard guard(h.device());
  const int64_t n = h.size(0), d = h.size(1), v = w.size(0);
  const int dt = dtype_of(h);
  const Tensor a = g_logprob ? grad_rows(*g_logprob) : Tensor(), b = g_entropy ? grad_rows(*g_entropy) : Tensor();
  size_t bytes = 0;
  check_rc(nimble_tied_logprobs_backward_workspace_size(n, d, v, dt, static_cast<size_t>(slab_bytes), &bytes),
           "nimble_tied_logprobs_backward_workspace_size");
  const Tensor ws = empty({static_cast<int64_t>(std::max<size_t>(bytes, 1))}, h, at::kByte);
  check_rc(nimble_tied_logprobs_backward(
               ptr_or_null(a), ptr_or_null(b), h.const_data_ptr(), w.const_data_ptr(),
               tokens.const_data_ptr<int64_t>(), lse.const_data_ptr<float>(), entropy.const_data_ptr<float>(), n, d, v,
               v_offset, vocab_size, ignore_index, dt, grad_hidden ? grad_hidden->data_ptr() : nullptr,
               grad_hidden ? dtype_of(*grad_hidden) : dt, grad_weights ? grad_weights->data_ptr() : nullptr,
               grad_weights ? dtype_of(*grad_weights) : dt, accumulate ? 1 : 0, static_cast<size_t>(slab_bytes),
               ws.mutable_data_ptr(), bytes, reinterpret_cast<int*>(status), stream_of(h)),
           "nimble_tied_logprobs_backward");
}

// Contiguous and on a 16-byte boundary, as the TMA loads need it.
Tensor for_tma(const Tensor& t) {
  const Tensor c = t.is_contiguous() ? t : t.contiguous();
  return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 == 0 ? c : c.clone();
}

struct TiedRows {
  Tensor h, w, logprob, entropy, lse;  // h, w: 16-bit, as the kernels read them
};
TiedRows tied_rows(const Tensor& hidden, const Tensor& weights, const Tensor& tokens, int64_t ignore_index,
                   int64_t status, int64_t host_flag) {
  const c10::cuda::CUDAGuard guard(hidden.device());
  TiedRows r;
  r.w = for_tma(as_type(weights, hidden.scalar_type()));
  r.h = for_tma(hidden.dim() == 2 ? hidden : hidden.reshape({-1, hidden.size(-1)}));
  status_hook(kPoll, r.h);
  const auto shape = hidden.sizes().slice(0, hidden.dim() - 1);
  r.logprob = empty(shape, hidden, at::kFloat);
  r.entropy = empty(shape, hidden, at::kFloat);
  r.lse = empty({r.h.size(0)}, hidden, at::kFloat);
  tied_forward(r.h, r.w, tokens, 0, ignore_index,
               {nullptr, r.logprob.mutable_data_ptr<float>(), r.entropy.mutable_data_ptr<float>(),
                r.lse.mutable_data_ptr<float>()},
               status, host_flag);
  return r;
}

// On one rank with the whole vocabulary (the sharded form is the package's).
struct TiedLogProbsNode : torch::autograd::Function<TiedLogProbsNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weights, const Tensor& tokens,
                               int64_t ignore_index, const std::optional<Tensor>& buffer, int64_t slab_bytes,
                               int64_t status, int64_t host_flag, bool check) {
    TiedRows r = tied_rows(hidden, weights, tokens, ignore_index, status, host_flag);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({r.h, r.w, tokens, r.lse, r.entropy});
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["slab_bytes"] = slab_bytes;
    ctx->saved_data["status"] = status;
    ctx->saved_data["host_flag"] = host_flag;
    ctx->saved_data["check"] = check;
    ctx->saved_data["weights"] = static_cast<int64_t>(weights.scalar_type());
    ctx->saved_data["shape"] = hidden.sizes().vec();
    if (buffer) ctx->saved_data["buffer"] = *buffer;
    return {r.logprob, r.entropy};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "the log probabilities' backward is not differentiable itself");
    variable_list out(9);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &h = saved[0], &w = saved[1];
    const c10::cuda::CUDAGuard guard(h.device());
    std::optional<Tensor> gh, gw;
    const auto buffer = ctx->saved_data.find("buffer");
    const bool accumulate = buffer != ctx->saved_data.end();
    if (ctx->needs_input_grad(0)) gh = empty(ctx->saved_data["shape"].toIntVector(), h, h.scalar_type());
    if (accumulate) gw = buffer->second.toTensor();
    else if (ctx->needs_input_grad(1))
      gw = empty(w.sizes(), w, static_cast<at::ScalarType>(ctx->saved_data["weights"].toInt()));
    if (*reinterpret_cast<volatile int*>(ctx->saved_data["host_flag"].toInt())) status_hook(kPoll, h);
    tied_backward(grads[0].defined() ? std::optional<Tensor>(grads[0]) : std::nullopt,
                  grads[1].defined() ? std::optional<Tensor>(grads[1]) : std::nullopt, h, w, saved[2], saved[3],
                  saved[4], 0, w.size(0), ctx->saved_data["ignore_index"].toInt(), gh, gw, accumulate,
                  ctx->saved_data["slab_bytes"].toInt(), ctx->saved_data["status"].toInt());
    if (ctx->saved_data["check"].toBool()) status_hook(kCheck, h);
    if (gh) out[0] = *gh;
    if (gw && !accumulate) out[1] = *gw;
    return out;
  }
};

py::tuple tied_token_logprobs(const Tensor& hidden, const Tensor& weights, const Tensor& tokens, int64_t ignore_index,
                              const std::optional<Tensor>& buffer, int64_t slab_bytes, int64_t status,
                              int64_t host_flag, bool check) {
  if (at::GradMode::is_enabled() && (hidden.requires_grad() || weights.requires_grad())) {
    const variable_list out =
        TiedLogProbsNode::apply(hidden, weights, tokens, ignore_index, buffer, slab_bytes, status, host_flag, check);
    if (check) status_hook(kCheck, hidden);
    return py::make_tuple(out[0], out[1]);
  }
  const TiedRows r = tied_rows(hidden, weights, tokens, ignore_index, status, host_flag);
  if (check) status_hook(kCheck, hidden);
  return py::make_tuple(r.logprob, r.entropy);
}

// ------------------------------------------------------------------------- AdamW
const Tensor& tensor_in(PyObject* o, const char* what) {
  TORCH_CHECK_VALUE(THPVariable_Check(o), what, " must be a tensor");
  return THPVariable_Unpack(o);
}

// Items of a list or tuple, borrowed.
struct Items {
  py::object seq;
  PyObject** at;
  Py_ssize_t n;
  explicit Items(const py::object& o) {
    seq = py::reinterpret_steal<py::object>(PySequence_Fast(o.ptr(), "expected a sequence of tensors"));
    if (!seq) throw py::error_already_set();
    at = PySequence_Fast_ITEMS(seq.ptr());
    n = PySequence_Fast_GET_SIZE(seq.ptr());
  }
};

constexpr int64_t kQuantBlock = 128;
void check_quantized(const Tensor& codes, const Tensor& scales) {
  TORCH_CHECK_VALUE(codes.scalar_type() == at::kFloat8_e4m3fn && codes.is_contiguous(),
                    "8-bit moments are contiguous float8_e4m3fn codes");
  TORCH_CHECK_VALUE(scales.scalar_type() == at::kFloat && scales.is_contiguous() &&
                        scales.numel() == (codes.numel() + kQuantBlock - 1) / kQuantBlock,
                    "8-bit moments need one contiguous float32 scale per ", kQuantBlock, " elements");
  TORCH_CHECK_VALUE(codes.is_cuda() && scales.device() == codes.device(), "8-bit moments live on one CUDA device");
}

// A set of at most n pointers, none of them null, in one allocation.
class PointerSet {
 public:
  explicit PointerSet(size_t n) {
    size_t size = 2;
    while (size < 2 * n) size *= 2;
    slots_.assign(size, nullptr);
  }
  bool has(const void* p) const { return slots_[find(p)] != nullptr; }
  bool insert(const void* p) {  // false where it was there
    const size_t at = find(p);
    if (slots_[at]) return false;
    slots_[at] = p;
    return true;
  }
  void clear() { std::fill(slots_.begin(), slots_.end(), nullptr); }

 private:
  size_t find(const void* p) const {  // its place, or the free one that it would take
    const uint64_t h = (reinterpret_cast<uintptr_t>(p) >> 2) * 0x9E3779B97F4A7C15ull;
    size_t at = (h >> 32) & (slots_.size() - 1);
    while (slots_[at] && slots_[at] != p) at = (at + 1) & (slots_.size() - 1);
    return at;
  }
  std::vector<const void*> slots_;
};

void adamw_step_many(const py::object& params_, const py::object& grads_, const py::object& m_, const py::object& v_,
                     const py::object& copies_, int64_t step, double lr, double beta1, double beta2, double eps,
                     double wd, bool own_steps) {
  refuse_recording("adamw_step_many");
  const Items params(params_), grads(grads_), ms(m_), vs(v_);
  std::optional<Items> copies;
  if (!copies_.is_none()) copies.emplace(copies_);
  TORCH_CHECK_VALUE(grads.n == params.n && ms.n == params.n && vs.n == params.n && (!copies || copies->n == params.n),
                    "params, grads, exp_avgs, exp_avg_sqs and copies must have one entry per tensor");
  TORCH_CHECK_VALUE(step >= 1, "step counts from 1, got ", step);
  std::vector<nimble_adamw_tensor> all;
  all.reserve(params.n);
  std::vector<Tensor> keep;  // contiguous copies of gradients, until the launches are queued
  std::vector<c10::TensorImpl*> written;
  written.reserve(6 * params.n);
  auto writes = [&](const Tensor& t) { written.push_back(t.unsafeGetTensorImpl()); };
  std::optional<at::Device> dev;
  bool eight = false;
  const bool duals = torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;  // none outside a level
  // Every tensor is checked before the first launch: a refused step leaves all of them as they were.
  for (Py_ssize_t i = 0; i < params.n; ++i) {
    if (grads.at[i] == Py_None) continue;
    const Tensor& p = tensor_in(params.at[i], "a parameter");
    const Tensor* g = &tensor_in(grads.at[i], "a gradient");
    if (duals) {
      refuse_tangent("adamw_step_many", p);
      refuse_tangent("adamw_step_many", *g);
    }
    if (!dev) {
      dev = p.device();
      TORCH_CHECK_VALUE(p.is_cuda(), "adamw_step_many needs CUDA tensors; there is no CPU path");
      eight = !THPVariable_Check(ms.at[i]);
    }
    const int64_t n = p.numel();
    TORCH_CHECK_VALUE(p.scalar_type() == at::kFloat && p.is_contiguous(),
                      "AdamW master weights must be contiguous float32 tensors");
    const int gdt = dtype_or(*g);
    TORCH_CHECK_VALUE(gdt >= 0 && g->numel() == n, "a gradient of ", g->numel(), " elements in ", g->scalar_type(),
                      " for ", n, " weights");
    TORCH_CHECK_VALUE(p.device() == *dev && g->device() == *dev, "all tensors of a step must be on one device");
    if (!g->is_contiguous()) {
      const c10::cuda::CUDAGuard guard(*dev);
      keep.push_back(g->contiguous());
      g = &keep.back();
    }
    nimble_adamw_tensor r{};
    auto moment = [&](PyObject* o, void*& values, float*& scales) {
      if (eight) {
        TORCH_CHECK_VALUE(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 2,
                          "moments are all fp32 tensors or all (codes, scales) pairs");
        const Tensor& codes = tensor_in(PyTuple_GET_ITEM(o, 0), "codes");
        const Tensor& s = tensor_in(PyTuple_GET_ITEM(o, 1), "scales");
        check_quantized(codes, s);
        TORCH_CHECK_VALUE(codes.numel() == n && codes.device() == *dev,
                          "moments must have the sizes and the device of their weights");
        values = codes.data_ptr();
        scales = static_cast<float*>(s.data_ptr());
        writes(codes);
        writes(s);
      } else {
        TORCH_CHECK_VALUE(THPVariable_Check(o), "moments are all fp32 tensors or all (codes, scales) pairs");
        const Tensor& t = THPVariable_Unpack(o);
        TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.is_contiguous(),
                          "fp32 moments must be contiguous float32 tensors");
        TORCH_CHECK_VALUE(t.numel() == n && t.device() == *dev,
                          "moments must have the sizes and the device of their weights");
        values = t.data_ptr();
        writes(t);
      }
    };
    moment(ms.at[i], r.exp_avg, r.exp_avg_scale);
    moment(vs.at[i], r.exp_avg_sq, r.exp_avg_sq_scale);
    if (copies && copies->at[i] != Py_None) {
      const Tensor& c = tensor_in(copies->at[i], "a copy");
      r.weights_copy_dtype = dtype_or(c);
      TORCH_CHECK_VALUE(r.weights_copy_dtype >= 0 && c.numel() == n && c.is_contiguous() && c.device() == *dev,
                        "a copy must be contiguous, on the device and of the size of its weights");
      r.weights_copy = c.data_ptr();
      writes(c);
    }
    if (n == 0) continue;
    writes(p);
    r.weights = static_cast<float*>(p.data_ptr());
    r.grad = g->data_ptr();
    r.n = n;
    r.grad_dtype = gdt;
    all.push_back(r);
  }
  if (all.empty()) return;
  const c10::cuda::CUDAGuard guard(*dev);
  void* stream = c10::cuda::getCurrentCUDAStream(dev->index()).stream();
  const double bc1 = 1.0 - std::pow(beta1, static_cast<double>(step));
  const double bc2 = 1.0 - std::pow(beta2, static_cast<double>(step));
  size_t start = 0, end = 0;  // of the next list: all[start, end), moved up over those that step alone
  PointerSet seen(all.size());
  auto launch = [&] {
    if (end > start)
      check_rc(nimble_adamw_step_many(all.data() + start, static_cast<int>(end - start), eight ? 8 : 32, lr, beta1,
                                      beta2, bc1, bc2, eps, wd, stream),
               "nimble_adamw_step_many");
    start = end;
    seen.clear();
  };
  auto whole = [](const nimble_adamw_tensor& t) {  // what the single step's vector kernel takes
    uintptr_t bits = 0;
    for (const void* p : {static_cast<const void*>(t.weights), t.grad, static_cast<const void*>(t.exp_avg),
                          static_cast<const void*>(t.exp_avg_sq), static_cast<const void*>(t.weights_copy)})
      bits |= reinterpret_cast<uintptr_t>(p);
    return t.n % 8 == 0 && (bits & 15) == 0;
  };
  for (size_t i = 0; i < all.size(); ++i) {
    const nimble_adamw_tensor t = all[i];
    // Weights that are listed twice: the second update follows the first.
    if (own_steps && !eight && !whole(t)) {
      if (seen.has(t.weights)) launch();
      check_rc(nimble_adamw_step(t.weights, t.grad, t.grad_dtype, static_cast<float*>(t.exp_avg),
                                 static_cast<float*>(t.exp_avg_sq), t.n, static_cast<float>(lr),
                                 static_cast<float>(beta1), static_cast<float>(beta2), static_cast<float>(bc1),
                                 static_cast<float>(bc2), static_cast<float>(eps), static_cast<float>(wd),
                                 t.weights_copy, t.weights_copy_dtype, stream),
               "nimble_adamw_step");
      continue;
    }
    if (!seen.insert(t.weights)) {
      launch();
      seen.insert(t.weights);
    }
    all[end++] = t;
  }
  launch();
  // As torch's own in-place updates: a backward pass that still needs an old value raises.
  for (c10::TensorImpl* t : written)
    if (!t->is_inference()) t->bump_version();
}

}  // namespace

PYBIND11_MODULE(nimbleml_b200_host, m) {
  m.doc() = "Host side of layer_norm, the token log probabilities and adamw_step_many over the C ABI";
  // What the package's functions begin with where their own checks come before the host's.
  m.def("begin_token_logprobs", [](const Tensor& x) { refuse_transforms("token_logprobs", x); });
  m.def("begin_tied_token_logprobs", [](const Tensor& h, const Tensor& w) {
    refuse_transforms("tied_token_logprobs", h);
    refuse_tangent("tied_token_logprobs", w);
  });
  m.def("begin_quantize", [](const Tensor& x) { refuse_transforms("quantize_moment", x); });
  m.def("begin_dequantize", [](const Tensor& codes, const Tensor& scales) {
    refuse_transforms("dequantize_moment", codes);
    refuse_tangent("dequantize_moment", scales);
  });
  m.def("layer_norm", &layer_norm);
  m.def("token_logprobs", &token_logprobs);
  m.def("set_status_hooks", &set_status_hooks);
  m.def("tied_token_logprobs", &tied_token_logprobs);
  m.def("tied_shard_stats", &tied_shard_stats);
  m.def("tied_backward", &tied_backward);
  m.def("adamw_step_many", &adamw_step_many);
}
