// Thin PyTorch-ROCm C++ extension over the C ABI (include/evodiff_hip.h): registers the hot-path entry points as
// torch operators (namespace evodiff_amd, CUDA = ROCm dispatch key) that take torch tensors, launch on PyTorch's current
// HIP stream and raise RuntimeError with ed_last_error() on failure.  It holds no kernels and no state: `handle` is the
// ed_model* (as an integer) that evodiff_amd.model.ByteNetLMTime.hip_handle() created.  Built with g++ against libtorch
// and linked to libevodiff_hip.so (__graft_entry__.build()); the ctypes binding in evodiff_amd/_lib.py is the other,
// torch-free way in.
#include "../../include/evodiff_hip.h"

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <tuple>

namespace {

ed_model* as_model(int64_t handle) {
  TORCH_CHECK(handle != 0, "evodiff_amd: null model handle");
  return reinterpret_cast<ed_model*>(static_cast<intptr_t>(handle));
}

void* current_stream(const at::Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check(int rc) { TORCH_CHECK(rc == 0, "libevodiff_hip error ", rc, ": ", ed_last_error()); }

void want(const at::Tensor& t, at::ScalarType dtype, const char* name) {
  TORCH_CHECK(t.is_cuda(), "evodiff_amd: ", name, " must live on the GPU (there is no CPU path)");
  TORCH_CHECK(t.scalar_type() == dtype && t.is_contiguous(), "evodiff_amd: ", name, " must be contiguous ", dtype);
}

ed_config config_of(int64_t handle) {
  ed_config c;
  check(ed_model_get_config(as_model(handle), &c));
  return c;
}

// (B, L) of a token tensor; every other tensor of a call is checked against them and against the model's own
// hyper-parameters, so that a caller's mistake is a RuntimeError here and never an out-of-bounds access on the device
void batch_shape(const at::Tensor& tokens, int64_t* B, int64_t* L) {
  TORCH_CHECK(tokens.dim() == 2 && tokens.size(0) > 0 && tokens.size(1) > 0, "evodiff_amd: tokens must be (batch, length)");
  *B = tokens.size(0);
  *L = tokens.size(1);
}

void want_timesteps(const ed_config& c, const at::Tensor& timesteps, int64_t B) {
  want(timesteps, at::kLong, "timesteps");
  TORCH_CHECK(c.timesteps == 0 || timesteps.numel() == B, "evodiff_amd: timesteps must hold one entry per sequence (", B,
              "), got ", timesteps.numel());
}

// ByteNetLMTime.forward(x, y) (evodiff/model.py:170-173): (B, L) int64 tokens, (B,) int64 timesteps -> (B, L, n_tokens) fp32
at::Tensor forward(int64_t handle, const at::Tensor& tokens, const at::Tensor& timesteps, int64_t n_tokens,
                   int64_t precision) {
  want(tokens, at::kLong, "tokens");
  int64_t B, L;
  batch_shape(tokens, &B, &L);
  const ed_config c = config_of(handle);
  want_timesteps(c, timesteps, B);
  TORCH_CHECK(n_tokens == c.n_tokens, "evodiff_amd: n_tokens = ", n_tokens, " but the model has ", c.n_tokens, " (it sizes the logits)");
  at::Tensor logits = at::empty({B, L, n_tokens}, tokens.options().dtype(at::kFloat));
  check(ed_forward(as_model(handle), tokens.data_ptr<int64_t>(), timesteps.data_ptr<int64_t>(), (int)B, (int)L,
                   logits.data_ptr<float>(), (int)precision, current_stream(tokens)));
  return logits;
}

// the loop of generate_oaardm (evodiff/generate.py:193-211); tokens (B, L) updated in place
at::Tensor oadm_sample_(int64_t handle, at::Tensor tokens, const at::Tensor& order, const at::Tensor& uniforms,
                        int64_t n_draw, int64_t precision, bool use_graph) {
  want(tokens, at::kLong, "tokens");
  want(order, at::kInt, "order");
  want(uniforms, at::kFloat, "uniforms");
  int64_t B, L;
  batch_shape(tokens, &B, &L);
  const int64_t n_steps = order.numel();
  TORCH_CHECK(uniforms.numel() == n_steps * B, "evodiff_amd: uniforms must be (n_steps, B)");
  check(ed_oadm_sample(as_model(handle), tokens.data_ptr<int64_t>(), order.data_ptr<int32_t>(), uniforms.data_ptr<float>(),
                       (int)B, (int)L, (int)n_steps, (int)n_draw, nullptr, (int)precision, use_graph ? 1 : 0,
                       current_stream(tokens)));
  return tokens;
}

// the loop of generate_d3pm (evodiff/generate.py:274-298); tokens (B, L) = x_t on entry, updated in place
at::Tensor d3pm_sample_(int64_t handle, at::Tensor tokens, const at::Tensor& Q, const at::Tensor& Qbar,
                        const at::Tensor& uniforms, int64_t K, int64_t t_start, int64_t n_steps, int64_t precision,
                        bool use_graph) {
  want(tokens, at::kLong, "tokens");
  want(Q, at::kDouble, "Q");
  want(Qbar, at::kDouble, "Qbar");
  want(uniforms, at::kFloat, "uniforms");
  TORCH_CHECK(Q.dim() == 3 && Q.size(1) == K && Q.size(2) == K && Qbar.sizes() == Q.sizes(), "evodiff_amd: Q / Qbar must be (timesteps, K, K)");
  int64_t B, L;
  batch_shape(tokens, &B, &L);
  TORCH_CHECK(Q.size(0) == config_of(handle).timesteps, "evodiff_amd: Q / Qbar must hold one matrix per timestep of the model");
  TORCH_CHECK(uniforms.numel() == Q.size(0) * B * L, "evodiff_amd: uniforms must be (timesteps, B, L)");
  check(ed_d3pm_sample(as_model(handle), tokens.data_ptr<int64_t>(), Q.data_ptr<double>(), Qbar.data_ptr<double>(),
                       uniforms.data_ptr<float>(), (int)B, (int)L, (int)K, (int)t_start, (int)n_steps, nullptr,
                       (int)precision, use_graph ? 1 : 0, current_stream(tokens)));
  return tokens;
}

// forward + cross entropy at the targets (analysis/sequence_perp.py:125-154): (B, L) fp32, zero where select == 0
at::Tensor score_nll(int64_t handle, const at::Tensor& tokens, const at::Tensor& timesteps, const at::Tensor& targets,
                     const c10::optional<at::Tensor>& select, int64_t n_classes, int64_t precision) {
  want(tokens, at::kLong, "tokens");
  want(targets, at::kLong, "targets");
  int64_t B, L;
  batch_shape(tokens, &B, &L);
  want_timesteps(config_of(handle), timesteps, B);
  TORCH_CHECK(targets.sizes() == tokens.sizes(), "evodiff_amd: targets must have the shape of tokens");
  if (select.has_value()) {
    want(*select, at::kByte, "select");
    TORCH_CHECK(select->numel() == B * L, "evodiff_amd: select must hold one byte per position (", B * L, ")");
  }
  at::Tensor nll = at::empty({B, L}, tokens.options().dtype(at::kFloat));
  check(ed_score_nll(as_model(handle), tokens.data_ptr<int64_t>(), timesteps.data_ptr<int64_t>(), targets.data_ptr<int64_t>(),
                     select.has_value() ? select->data_ptr<uint8_t>() : nullptr, (int)B, (int)L, (int)n_classes,
                     nll.data_ptr<float>(), (int)precision, current_stream(tokens)));
  return nll;
}

// ---- model-free operators (evodiff_amd/ops.py documents them) ----
int dtype_of(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "evodiff_amd: ", name, " must live on the GPU (there is no CPU path)");
  if (t.scalar_type() == at::kFloat) return ED_DT_FP32;
  if (t.scalar_type() == at::kBFloat16) return ED_DT_BF16;
  TORCH_CHECK(t.scalar_type() == at::kHalf, "evodiff_amd: ", name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  return ED_DT_FP16;
}

void same_device(const at::Tensor& a, const at::Tensor& b, const char* name) {
  TORCH_CHECK(a.device() == b.device(), "evodiff_amd: ", name, " must be on the device of the first operand");
}

template <typename T>
T* ptr_or_null(const c10::optional<at::Tensor>& t) { return t.has_value() ? (T*)t->data_ptr() : nullptr; }

int64_t blocks_of(int64_t k) { return (k + 127) / 128; }

// (rows, K) with one row stride and contiguous columns; other layouts are copied
at::Tensor as_rows(const at::Tensor& x, const char* name) {
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, "evodiff_amd: ", name, " must have a non-empty last dimension");
  at::Tensor r = x.dim() == 2 ? x : x.reshape({x.numel() / x.size(-1), x.size(-1)});
  return r.size(1) == 1 || r.stride(1) == 1 ? r : r.contiguous();
}

std::tuple<at::Tensor, at::Tensor> quantize(const at::Tensor& x, bool square) {
  const int dt = dtype_of(x, square ? "w" : "x");
  TORCH_CHECK(!square || x.dim() == 2, "evodiff_amd: a weight must be (N, K)");
  const c10::DeviceGuard guard(x.device());
  const at::Tensor r = as_rows(x, square ? "w" : "x");
  const int64_t rows = r.size(0), k = r.size(1), kb = blocks_of(k);
  at::Tensor q = at::empty({rows, kb * 128}, x.options().dtype(at::kFloat8_e4m3fn));
  at::Tensor scale = at::empty({square ? blocks_of(rows) : rows, kb}, x.options().dtype(at::kFloat8_e8m0fnu));
  check((square ? ed_fp8_quantize_weight : ed_fp8_quantize_rows)(r.data_ptr(), dt, r.stride(0), rows, k, (uint8_t*)q.data_ptr(),
                                                                 (uint8_t*)scale.data_ptr(), current_stream(x)));
  return {q, scale};
}

std::tuple<at::Tensor, at::Tensor> quantize_fp8(const at::Tensor& x) { return quantize(x, false); }
std::tuple<at::Tensor, at::Tensor> quantize_fp8_weight(const at::Tensor& w) { return quantize(w, true); }

at::Tensor linear_fp8(const at::Tensor& x, const c10::optional<at::Tensor>& x_scale, const at::Tensor& weight,
                      const at::Tensor& weight_scale, const c10::optional<at::Tensor>& bias,
                      c10::optional<at::ScalarType> out_dtype, bool fast_sums) {
  want(weight, at::kFloat8_e4m3fn, "weight.q");
  want(weight_scale, at::kFloat8_e8m0fnu, "weight.scale");
  same_device(weight, x, "x");
  same_device(weight, weight_scale, "weight.scale");
  TORCH_CHECK(weight.dim() == 2 && weight.size(0) > 0 && weight.size(1) > 0 && weight.size(1) % 128 == 0, "evodiff_amd: weight.q must be (N, Kb * 128)");
  const int64_t N = weight.size(0), kb = weight.size(1) / 128;
  TORCH_CHECK(weight_scale.dim() == 2 && weight_scale.size(0) == blocks_of(N) && weight_scale.size(1) == kb,
              "evodiff_amd: weight.scale must be (", blocks_of(N), ", ", kb, "), got ", weight_scale.sizes());
  int dt = ED_DT_E4M3;
  if (x_scale.has_value()) {
    want(x, at::kFloat8_e4m3fn, "x.q");
    want(*x_scale, at::kFloat8_e8m0fnu, "x.scale");
    same_device(weight, *x_scale, "x.scale");
    TORCH_CHECK(x.dim() == 2 && x_scale->dim() == 2 && x_scale->size(0) == x.size(0) && x_scale->size(1) * 128 == x.size(1),
                "evodiff_amd: x.q must be (rows, Kb * 128) and x.scale (rows, Kb)");
  } else {
    dt = dtype_of(x, "x");
  }
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0 && blocks_of(x.size(-1)) == kb, "evodiff_amd: x has ", x.dim() ? x.size(-1) : 0,
              " channels, the weight is laid out for ", kb * 128 - 127, " to ", kb * 128);
  if (bias.has_value()) {
    want(*bias, at::kFloat, "bias");
    same_device(weight, *bias, "bias");
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == N, "evodiff_amd: bias must be (", N, ")");
  }
  const at::ScalarType ot = out_dtype.has_value() ? *out_dtype : x_scale.has_value() ? at::kBFloat16 : x.scalar_type();
  TORCH_CHECK(ot == at::kFloat || ot == at::kBFloat16 || ot == at::kHalf, "evodiff_amd: out_dtype must be float32, bfloat16 or float16, got ", ot);
  TORCH_CHECK(!fast_sums || ot != at::kFloat, "evodiff_amd: fast_sums is for bfloat16 and float16 outputs: a float32 output has float32 sums");
  const c10::DeviceGuard guard(x.device());
  const at::Tensor r = as_rows(x, "x");
  const int64_t M = r.size(0), K = r.size(1);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = N;
  at::Tensor out = at::empty(shape, x.options().dtype(ot));
  const int out_code = dtype_of(out, "out") | (fast_sums ? ED_FAST_SUMS : 0);
  const int64_t need = ed_fp8_linear_workspace(M, N, K, dt, out_code);
  at::Tensor ws;
  if (need > 0) ws = at::empty({need}, x.options().dtype(at::kByte));
  check(ed_fp8_linear(r.data_ptr(), dt, r.stride(0), ptr_or_null<uint8_t>(x_scale), (const uint8_t*)weight.data_ptr(),
                      (const uint8_t*)weight_scale.data_ptr(), ptr_or_null<float>(bias), out.data_ptr(), out_code, M, N, K,
                      need > 0 ? ws.data_ptr() : nullptr, need, current_stream(x)));
  return out;
}

// Logits (..., V) as rows of one or two strides; others are copied.
struct LogitRows {
  at::Tensor t;
  int64_t rows, row_stride, inner, outer_stride;
};
LogitRows logit_rows(const at::Tensor& logits) {
  const int64_t V = logits.size(-1);
  LogitRows r{logits, V > 0 ? logits.numel() / V : 0, V, 1, 0};
  if (r.rows == 0) return r;
  for (int attempt = 0; attempt < 2; ++attempt) {
    r.t = attempt == 0 ? logits : logits.contiguous();
    if (V > 1 && r.t.stride(-1) != 1) continue;
    std::vector<std::pair<int64_t, int64_t>> lead;  // (size, stride), innermost first, neighbours joined where they are one run
    for (int64_t d = r.t.dim() - 2; d >= 0; --d) {
      const int64_t n = r.t.size(d), st = r.t.stride(d);
      if (n == 1) continue;
      if (!lead.empty() && st == lead.back().first * lead.back().second) lead.back().first *= n;
      else lead.push_back({n, st});
    }
    if (lead.size() > 2) continue;
    r.inner = lead.empty() ? 1 : lead[0].first;
    r.row_stride = lead.empty() ? V : lead[0].second;
    r.outer_stride = lead.size() > 1 ? lead[1].second : 0;
    return r;
  }
  return r;  // (a contiguous tensor always returns above)
}

void check_row_tensor(const c10::optional<at::Tensor>& t, const at::Tensor& logits, const char* name) {
  if (!t.has_value()) return;
  TORCH_CHECK(t->is_cuda(), "evodiff_amd: ", name, " must live on the GPU (there is no CPU path)");
  same_device(logits, *t, name);
  TORCH_CHECK(t->sizes() == logits.sizes().slice(0, logits.dim() - 1), "evodiff_amd: ", name, " must be shaped like the logits without classes, got ", t->sizes());
}

struct RowInputs {  // targets and select as the library reads them
  c10::optional<at::Tensor> targets, select;
};
RowInputs row_inputs(const at::Tensor& logits, const c10::optional<at::Tensor>& targets, const c10::optional<at::Tensor>& select) {
  RowInputs r;
  check_row_tensor(targets, logits, "targets");
  check_row_tensor(select, logits, "select");
  if (targets.has_value()) {
    TORCH_CHECK(targets->scalar_type() == at::kLong || targets->scalar_type() == at::kInt, "evodiff_amd: targets must be int64 or int32, got ", targets->scalar_type());
    r.targets = targets->to(at::kLong).contiguous();
  }
  if (select.has_value()) {
    TORCH_CHECK(select->scalar_type() == at::kBool || select->scalar_type() == at::kByte, "evodiff_amd: select must be bool or uint8, got ", select->scalar_type());
    r.select = select->contiguous();
  }
  return r;
}

using Maybe = c10::optional<at::Tensor>;
using Scores = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>;  // logprob, entropy, top_logprob, top_token

// stats: where the gradient's row statistics go, or nullptr
Scores scores_of(const at::Tensor& logits, const RowInputs& in, int64_t top_k, int64_t n_classes, at::Tensor* stats) {
  const int dt = dtype_of(logits, "logits");
  const LogitRows r = logit_rows(logits);
  std::vector<int64_t> shape = logits.sizes().vec();
  shape.pop_back();
  const auto f32 = logits.options().dtype(at::kFloat);
  at::Tensor logprob = in.targets.has_value() ? at::empty(shape, f32) : at::empty({0}, f32);
  at::Tensor entropy = at::empty(shape, f32);
  if (stats) *stats = at::empty({r.rows, 2}, f32);
  shape.push_back(top_k);
  at::Tensor top = at::empty(shape, f32), token = at::empty(shape, f32.dtype(at::kLong));
  const int64_t need = ed_token_logprobs_workspace(r.rows, n_classes, (int)top_k);
  at::Tensor ws;
  if (need > 0) ws = at::empty({need}, f32.dtype(at::kByte));
  check(ed_token_logprobs(r.t.data_ptr(), dt, r.row_stride, r.inner, r.outer_stride, r.rows, n_classes, ptr_or_null<int64_t>(in.targets),
                          ptr_or_null<uint8_t>(in.select), (int)top_k, in.targets.has_value() ? logprob.data_ptr<float>() : nullptr,
                          entropy.data_ptr<float>(), stats ? stats->data_ptr<float>() : nullptr, top.data_ptr<float>(),
                          token.data_ptr<int64_t>(), need > 0 ? ws.data_ptr() : nullptr, need, current_stream(logits)));
  return {logprob, entropy, top, token};
}

RowInputs checked_inputs(const at::Tensor& logits, const Maybe& targets, const Maybe& select, int64_t top_k, int64_t n_classes) {
  dtype_of(logits, "logits");
  TORCH_CHECK(logits.dim() >= 1 && n_classes >= 1 && n_classes <= logits.size(-1), "evodiff_amd: n_classes must be in [1, ", logits.dim() ? logits.size(-1) : 0, "], got ", n_classes);
  TORCH_CHECK(top_k >= 0 && top_k <= n_classes && top_k <= ED_TOP_K_MAX, "evodiff_amd: top_k must be in [0, min(n_classes, ", ED_TOP_K_MAX, ")], got ", top_k);
  return row_inputs(logits, targets, select);
}

Scores token_logprobs(const at::Tensor& logits, const Maybe& targets, const Maybe& select, int64_t top_k, int64_t n_classes) {
  const c10::DeviceGuard guard(logits.device());
  return scores_of(logits, checked_inputs(logits, targets, select, top_k, n_classes), top_k, n_classes, nullptr);
}

at::Tensor grad_of(const at::Tensor& logits, const RowInputs& in, int64_t top_k, int64_t n_classes, const at::Tensor& stats,
                   const at::Tensor& entropy, const at::Tensor& top_token, const at::Tensor (&grads)[3]) {
  const LogitRows r = logit_rows(logits);
  at::Tensor g[3];
  const float* p[3] = {nullptr, nullptr, nullptr};
  for (int i = 0; i < 3; ++i) {
    if (!grads[i].defined() || (i == 0 && !in.targets.has_value()) || (i == 2 && top_k == 0)) continue;
    TORCH_CHECK(grads[i].is_cuda() && grads[i].numel() == r.rows * (i == 2 ? top_k : 1), "evodiff_amd: gradients must have the outputs' shapes");
    same_device(logits, grads[i], "a gradient");
    g[i] = grads[i].to(at::kFloat).contiguous();
    p[i] = g[i].data_ptr<float>();
  }
  at::Tensor grad = at::empty(logits.sizes(), logits.options());
  check(ed_token_logprobs_backward(r.t.data_ptr(), dtype_of(logits, "logits"), r.row_stride, r.inner, r.outer_stride, r.rows, n_classes,
                                   logits.size(-1), ptr_or_null<int64_t>(in.targets), ptr_or_null<uint8_t>(in.select), (int)top_k,
                                   stats.data_ptr<float>(), entropy.data_ptr<float>(), top_token.data_ptr<int64_t>(), p[0], p[1], p[2],
                                   grad.data_ptr(), current_stream(logits)));
  return grad;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const Maybe& targets,
                                                const Maybe& select, int64_t top_k, int64_t n_classes) {
    const at::AutoDispatchBelowAutograd below;
    const c10::DeviceGuard guard(logits.device());
    const RowInputs in = checked_inputs(logits, targets, select, top_k, n_classes);
    at::Tensor stats;
    const Scores out = scores_of(logits, in, top_k, n_classes, &stats);
    ctx->save_for_backward({logits, in.targets.value_or(at::Tensor()), in.select.value_or(at::Tensor()), stats, std::get<1>(out), std::get<3>(out)});
    ctx->saved_data["top_k"] = top_k;
    ctx->saved_data["n_classes"] = n_classes;
    ctx->mark_non_differentiable({std::get<3>(out)});
    ctx->set_materialize_grads(false);
    return {std::get<0>(out), std::get<1>(out), std::get<2>(out), std::get<3>(out)};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const torch::autograd::variable_list saved = ctx->get_saved_variables();
    const at::Tensor& logits = saved[0];
    at::Tensor grad;
    {
      const at::AutoDispatchBelowAutograd below;
      const c10::DeviceGuard guard(logits.device());
      RowInputs in;
      if (saved[1].defined()) in.targets = saved[1];
      if (saved[2].defined()) in.select = saved[2];
      const at::Tensor given[3] = {grads[0], grads[1], grads[2]};
      grad = grad_of(logits, in, ctx->saved_data["top_k"].toInt(), ctx->saved_data["n_classes"].toInt(), saved[3], saved[4], saved[5], given);
    }
    if (at::GradMode::is_enabled()) {  // create_graph: the gradient itself has none, and says so where one is asked for
      const auto once = std::make_shared<torch::autograd::DelayedError>("token_logprobs can be differentiated once only", 1);
      grad = (*once)({grad.detach().requires_grad_()})[0];
    }
    return {grad, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// A leaf's accumulation node belongs to the stream of the graph that made it and lives as long as that graph.  A backward pass
// that is captured on another stream would make that stream wait inside the capture, which the engine's thread does not survive.
// The logits are the leaf, or a view of it.
void refuse_foreign_leaf(const at::Tensor& logits) {
  const at::TensorBase& leaf = logits.is_view() ? logits._base() : logits;
  if (!leaf.is_leaf()) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(leaf);
  if (!node) return;
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  TORCH_CHECK(hipStreamIsCapturing((hipStream_t)current_stream(logits), &status) == hipSuccess, "evodiff_amd: hipStreamIsCapturing failed");
  const auto made = node->stream();  // (its device's type is not that of a HIP stream: by number)
  TORCH_CHECK(status == hipStreamCaptureStatusNone || !made.has_value() || made->id() == c10::hip::getCurrentHIPStream(logits.device().index()).id(),
              "evodiff_amd: an eager graph of these logits is alive: let go of its results before a pass with gradients is captured");
}

// The operators have no forward-mode derivative; a dual tensor does not ask for a gradient, and below autograd its tangent is lost.
void refuse_tangent(const at::Tensor& t, const char* name) {
  TORCH_CHECK(!t._fw_grad(0).defined(), "evodiff_amd: ", name, " has no forward-mode derivative: give it the primal of a dual tensor");
}

// What has no derivative at all says so where one is asked for.
void refuse_derivatives(const at::Tensor& t, const char* name) {
  refuse_tangent(t, name);
  TORCH_CHECK(!at::GradMode::is_enabled() || !t.requires_grad(), "evodiff_amd: ", name, " has no gradient: call it under torch.no_grad() or on detached tensors");
}

// The operator again, below autograd: through the dispatcher, so that dispatch modes and tensors without data (fake ones) are met
// there and not in the kernel's own code.
template <typename Signature>
auto operator_of(const char* name) { return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>(); }

std::tuple<at::Tensor, at::Tensor> quantize_fp8_autograd(const at::Tensor& x) {
  refuse_derivatives(x, "quantize_fp8");
  static const auto op = operator_of<decltype(quantize_fp8)>("evodiff_amd::quantize_fp8");
  const at::AutoDispatchBelowAutograd below;
  return op.call(x);
}

std::tuple<at::Tensor, at::Tensor> quantize_fp8_weight_autograd(const at::Tensor& w) {
  refuse_derivatives(w, "quantize_fp8_weight");
  static const auto op = operator_of<decltype(quantize_fp8_weight)>("evodiff_amd::quantize_fp8_weight");
  const at::AutoDispatchBelowAutograd below;
  return op.call(w);
}

at::Tensor linear_fp8_autograd(const at::Tensor& x, const Maybe& x_scale, const at::Tensor& weight, const at::Tensor& weight_scale,
                               const Maybe& bias, c10::optional<at::ScalarType> out_dtype, bool fast_sums) {
  refuse_derivatives(x, "linear_fp8");
  if (bias.has_value()) refuse_derivatives(*bias, "linear_fp8");
  static const auto op = operator_of<decltype(linear_fp8)>("evodiff_amd::linear_fp8");
  const at::AutoDispatchBelowAutograd below;
  return op.call(x, x_scale, weight, weight_scale, bias, out_dtype, fast_sums);
}

Scores token_logprobs_autograd(const at::Tensor& logits, const Maybe& targets, const Maybe& select, int64_t top_k, int64_t n_classes) {
  refuse_tangent(logits, "token_logprobs");
  if (!at::GradMode::is_enabled() || !logits.requires_grad()) {
    static const auto op = operator_of<decltype(token_logprobs)>("evodiff_amd::token_logprobs");
    const at::AutoDispatchBelowAutograd below;
    return op.call(logits, targets, select, top_k, n_classes);
  }
  refuse_foreign_leaf(logits);
  const auto out = TokenLogprobs::apply(logits, targets, select, top_k, n_classes);
  return {out[0], out[1], out[2], out[3]};
}

}  // namespace

TORCH_LIBRARY(evodiff_amd, m) {
  m.def("forward(int handle, Tensor tokens, Tensor timesteps, int n_tokens, int precision) -> Tensor");
  m.def("oadm_sample_(int handle, Tensor(a!) tokens, Tensor order, Tensor uniforms, int n_draw, int precision, bool use_graph) -> Tensor(a!)");
  m.def("d3pm_sample_(int handle, Tensor(a!) tokens, Tensor Q, Tensor Qbar, Tensor uniforms, int K, int t_start, int n_steps, int precision, bool use_graph) -> Tensor(a!)");
  m.def("score_nll(int handle, Tensor tokens, Tensor timesteps, Tensor targets, Tensor? select, int n_classes, int precision) -> Tensor");
  m.def("quantize_fp8(Tensor x) -> (Tensor, Tensor)");
  m.def("quantize_fp8_weight(Tensor w) -> (Tensor, Tensor)");
  m.def("linear_fp8(Tensor x, Tensor? x_scale, Tensor weight, Tensor weight_scale, Tensor? bias, ScalarType? out_dtype, bool fast_sums=False) -> Tensor");
  m.def("token_logprobs(Tensor logits, Tensor? targets, Tensor? select, int top_k, int n_classes) -> (Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(evodiff_amd, CUDA, m) {
  m.impl("forward", &forward);
  m.impl("oadm_sample_", &oadm_sample_);
  m.impl("d3pm_sample_", &d3pm_sample_);
  m.impl("score_nll", &score_nll);
  m.impl("quantize_fp8", &quantize_fp8);
  m.impl("quantize_fp8_weight", &quantize_fp8_weight);
  m.impl("linear_fp8", &linear_fp8);
  m.impl("token_logprobs", &token_logprobs);
}

TORCH_LIBRARY_IMPL(evodiff_amd, AutogradCUDA, m) {
  m.impl("quantize_fp8", &quantize_fp8_autograd);
  m.impl("quantize_fp8_weight", &quantize_fp8_weight_autograd);
  m.impl("linear_fp8", &linear_fp8_autograd);
  m.impl("token_logprobs", &token_logprobs_autograd);
}
