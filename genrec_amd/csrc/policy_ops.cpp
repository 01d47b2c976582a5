// Autograd side of the policy-training operators: argument checks, output and scratch tensors, and the nodes whose
// backward passes call libgenrec_hip.so.  In C++ because autograd runs the backward of GPU tensors on a thread of its
// own: without Python in it a launcher-sized loss with its gradient takes a third of the time on the host.  The
// library's entry points are handed over by address (bind), so this module calls the copy that genrec_amd._lib loaded.
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <ATen/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cfloat>
#include <cmath>
#include <optional>
#include <string>

#include "genrec_hip.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

namespace {

struct Api {
    decltype(&grx_last_error) last_error;
    decltype(&grx_token_logps_scratch_bytes) token_logps_scratch_bytes;
    decltype(&grx_token_logps) token_logps;
    decltype(&grx_token_logps_backward) token_logps_backward;
    decltype(&grx_lm_token_logps_scratch_bytes) lm_token_logps_scratch_bytes;
    decltype(&grx_lm_token_logps_backward_scratch_bytes) lm_token_logps_backward_scratch_bytes;
    decltype(&grx_lm_token_logps_kept_bytes) lm_token_logps_kept_bytes;
    decltype(&grx_lm_token_logps) lm_token_logps;
    decltype(&grx_lm_token_logps_backward) lm_token_logps_backward;
    decltype(&grx_policy_loss_scratch_bytes) policy_loss_scratch_bytes;
    decltype(&grx_policy_loss) policy_loss;
    decltype(&grx_policy_loss_backward) policy_loss_backward;
} api;
PyObject* error_type = nullptr;  // genrec_amd._lib.GenrecHipError

void check(int status) {
    if (status == GRX_OK) return;
    const char* message = api.last_error();
    TORCH_CHECK(false, "libgenrec_hip status ", status, ": ", message ? message : "?");
}

void require_cuda(const Tensor& t, const char* what) {  // called from Python
    if (t.is_cuda()) return;
    PyErr_Format(error_type, "%s must live on the GPU (got device %s); genrec_amd runs on MI355X only and has no CPU path", what,
                 t.device().str().c_str());
    throw py::error_already_set();
}

void same_device(const Tensor& t, const at::Device& device, const char* what) {
    TORCH_CHECK_VALUE(t.device() == device, what, " is on ", t.device().str(), ", expected ", device.str());
}

void* stream_on(const at::Device& d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }

Tensor scratch(size_t bytes, const at::Device& d) {
    return bytes ? at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(d)) : Tensor();
}

Tensor f32_like(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kFloat)); }

template <typename T>
T* ptr(const Tensor& t) { return t.defined() ? reinterpret_cast<T*>(t.data_ptr()) : nullptr; }

double temperature_of(double t) {
    // its inverse has to be finite in fp32 too
    TORCH_CHECK_VALUE((float)t >= FLT_MIN && std::isfinite((float)t), "temperature must be at least 2^-126 and finite, got ", t);
    return t;
}

// [N] as [N, 1], [B, T] as it is, elements of a row next to each other.
Tensor rows_2d(const Tensor& t) {
    if (t.dim() == 1) return t.unsqueeze(1);
    return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous();
}

Tensor token_ids_of(const Tensor& ids, const at::Device& device) {
    TORCH_CHECK_TYPE(at::isIntegralType(ids.scalar_type(), false), "token_ids must be integers, got ", ids.scalar_type());
    same_device(ids, device, "token_ids");
    TORCH_CHECK_VALUE(ids.numel() <= GRX_MAX_TOKEN_ROWS, "at most ", GRX_MAX_TOKEN_ROWS, " rows per call, got ", ids.numel());
    return rows_2d(ids.scalar_type() == at::kLong ? ids : ids.to(at::kLong));
}

Tensor grad_rows(const Tensor& g) {
    if (!g.defined()) return g;
    return (g.scalar_type() == at::kFloat ? g : g.to(at::kFloat)).contiguous();
}

bool recording(hipStream_t s) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (s == nullptr) return false;  // the default stream cannot be recorded
    C10_HIP_CHECK(hipStreamIsCapturing(s, &status));
    return status != hipStreamCaptureStatusNone;
}

// Called by a backward pass.  Recorded into a HIP graph, its gradients cannot go to a node that was made outside of the
// recording (a leaf that a living eager graph holds too): autograd would let the recording wait for that node's stream,
// which ends the process.
void refuse_nodes_outside(const at::Device& device) {
    const auto stream = c10::hip::getCurrentHIPStream(device.index());
    if (!recording(stream.stream())) return;
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    for (size_t i = 0; i < node->num_outputs(); ++i) {
        const auto& next = node->next_edge(i);
        if (!next.is_valid() || !node->task_should_compute_output(i)) continue;
        const auto theirs = next.function->stream();
        if (!theirs || theirs->device_type() == at::kCPU || theirs->id() == stream.id()) continue;
        const c10::Device on(stream.device_type(), theirs->device_index());  // whichever name the type goes by
        const c10::hip::HIPStream other(c10::hip::HIPStream::UNCHECKED, c10::Stream(c10::Stream::UNSAFE, on, theirs->id()));
        TORCH_CHECK(recording(other.stream()),
                    "a backward pass recorded into a HIP graph needs leaves of its own: detach().requires_grad_() inside the "
                    "recording, or drop the graphs made outside of it first");
    }
}

// The kernels have no gradient of their own: under create_graph the results carry a node that says so when it is reached.
// It stands where the derivative's node would, in front of all that the results depend on -- the inputs of the node that runs
// and what came in -- whether or not the incoming gradients are constants, so that no second-order term is left out unsaid.
variable_list once(const variable_list& incoming, variable_list out) {
    if (!at::GradMode::is_enabled()) return out;
    torch::autograd::edge_list next;
    if (const auto node = torch::autograd::get_current_node())
        for (const auto& edge : node->next_edges())
            if (edge.is_valid()) next.push_back(edge);
    for (const Tensor& g : incoming)
        if (g.defined() && g.requires_grad()) next.push_back(torch::autograd::impl::gradient_edge(g));
    const auto error = std::make_shared<torch::autograd::Error>(
        "trying to differentiate twice a function of genrec_amd.policy, which is differentiable once", std::move(next));
    for (Tensor& t : out) {
        if (!t.defined()) continue;
        t = t.detach();
        torch::autograd::set_history(t, error);
    }
    return out;
}

// No gradient is asked of t, in either direction: a call may go without a node.  (A forward-mode tangent has to reach the
// node, which refuses it.)
bool constant(const Tensor& t) { return !(at::GradMode::is_enabled() && t.requires_grad()) && !t._fw_grad(0).defined(); }

int dtype_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return GRX_F32;
        case at::kBFloat16: return GRX_BF16;
        case at::kHalf: return GRX_F16;
        default: TORCH_CHECK_TYPE(false, "unsupported logits dtype ", t.scalar_type(), "; expected float32, bfloat16 or float16");
    }
    return -1;
}

// ---- log-probabilities from logits ------------------------------------------------------------------------
grx_token_logps_args token_args(const Tensor& logits, const Tensor& ids, double temperature) {
    grx_token_logps_args a = {};
    a.logits = logits.data_ptr();
    a.row_stride = logits.stride(0);
    a.pos_stride = logits.dim() == 3 ? logits.stride(1) : 0;
    a.token_ids = ptr<int64_t>(ids);
    a.ids_stride = ids.stride(0);
    a.B = (int32_t)ids.size(0);
    a.T = (int32_t)ids.size(1);
    a.V = (int32_t)logits.size(-1);
    a.dtype = dtype_code(logits);
    a.temperature = (float)temperature;
    return a;
}

// stats: where a backward pass wants them; null: in the scratch tensor.
variable_list token_forward(const Tensor& logits, const Tensor& ids, double temperature, bool entropy, float* stats) {
    const at::OptionalDeviceGuard guard(logits.device());
    const int64_t B = ids.size(0), T = ids.size(1);
    variable_list out = {f32_like({B, T}, logits)};
    if (entropy) out.push_back(f32_like({B, T}, logits));
    grx_token_logps_args a = token_args(logits, ids, temperature);
    const size_t n = api.token_logps_scratch_bytes(B * T, a.V, a.dtype);  // a multiple of 16
    const Tensor s = scratch(n + (stats ? 0 : B * T * 2 * sizeof(float)), logits.device());
    a.logps = ptr<float>(out[0]);
    a.row_stats = stats ? stats : reinterpret_cast<float*>(ptr<char>(s) + n);
    a.entropy = entropy ? ptr<float>(out[1]) : nullptr;
    check(api.token_logps(&a, ptr<void>(s), n, stream_on(logits.device())));
    return out;
}

struct TokenLogps : Function<TokenLogps> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& ids, double temperature, bool entropy) {
        const Tensor stats = f32_like({ids.size(0), ids.size(1), 2}, logits);
        const variable_list out = token_forward(logits, ids, temperature, entropy, ptr<float>(stats));
        ctx->save_for_backward({logits, ids, stats, entropy ? out[1] : Tensor()});
        ctx->saved_data["temperature"] = temperature;
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list incoming) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &ids = saved[1], &stats = saved[2], &ent = saved[3];
        const at::OptionalDeviceGuard guard(logits.device());
        refuse_nodes_outside(logits.device());
        const Tensor g = grad_rows(incoming[0]), h = incoming.size() > 1 ? grad_rows(incoming[1]) : Tensor();
        const Tensor grad = at::empty(logits.sizes(), logits.options());
        grx_token_logps_args a = token_args(logits, ids, ctx->saved_data["temperature"].toDouble());
        a.row_stats = ptr<float>(stats);
        a.entropy = ptr<float>(ent);
        a.grad_logps = ptr<float>(g);
        a.grad_entropy = ptr<float>(h);
        a.grad_logits = grad.data_ptr();
        check(api.token_logps_backward(&a, stream_on(logits.device())));
        return once(incoming, {grad, Tensor(), Tensor(), Tensor()});
    }
};

py::object outputs(const variable_list& out, at::IntArrayRef shape) {
    if (out.size() == 1) return py::cast(out[0].sizes() == shape ? out[0] : out[0].reshape(shape));
    return py::make_tuple(out[0].sizes() == shape ? out[0] : out[0].reshape(shape),
                          out[1].sizes() == shape ? out[1] : out[1].reshape(shape));
}

py::object token_logps(const Tensor& logits_, const Tensor& token_ids, double temperature, bool entropy) {
    temperature = temperature_of(temperature);
    dtype_code(logits_);
    TORCH_CHECK_VALUE((logits_.dim() == 2 || logits_.dim() == 3) && token_ids.sizes() == logits_.sizes().slice(0, logits_.dim() - 1),
                      "logits must be [..., V] with one row per token id: got ", logits_.sizes(), " for ids ", token_ids.sizes());
    TORCH_CHECK_VALUE(logits_.size(-1) >= 1, "the vocabulary is empty");
    TORCH_CHECK_VALUE(logits_.size(-1) <= 1 << 24, "the vocabulary may hold at most 2^24 tokens, got ", logits_.size(-1));
    const Tensor ids = token_ids_of(token_ids, logits_.device());
    require_cuda(logits_, "logits");
    const Tensor logits = logits_.size(-1) > 1 && logits_.stride(-1) != 1 ? logits_.contiguous() : logits_;
    if (constant(logits))
        return outputs(token_forward(logits, ids, temperature, entropy, nullptr), token_ids.sizes());
    return outputs(TokenLogps::apply(logits, ids, temperature, entropy), token_ids.sizes());
}

// ---- log-probabilities from hidden states -----------------------------------------------------------------
// [N, H] with rows of consecutive elements that start on 16 bytes and are less than 2^22 elements apart.
Tensor aligned_rows(const Tensor& t) {
    const auto aligned = [](const Tensor& x) { return reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0; };
    if (t.stride(1) == 1 && aligned(t) &&
        (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) && t.stride(0) <= 1 << 22)))
        return t;
    const Tensor c = t.contiguous();
    return aligned(c) ? c : c.clone();
}

grx_lm_token_logps_args lm_args(const Tensor& hidden, const Tensor& weight, const Tensor& ids, double temperature) {
    grx_lm_token_logps_args a = {};
    a.N = (int32_t)hidden.size(0);
    a.H = (int32_t)hidden.size(1);
    a.V = (int32_t)weight.size(0);
    a.hidden = hidden.data_ptr();
    a.hidden_stride = a.N > 1 ? hidden.stride(0) : a.H;
    a.weight = weight.data_ptr();
    a.weight_stride = a.V > 1 ? weight.stride(0) : a.H;
    a.token_ids = ptr<int64_t>(ids);
    a.temperature = (float)temperature;
    return a;
}

variable_list lm_forward(const Tensor& hidden, const Tensor& weight, const Tensor& ids, double temperature, bool entropy,
                         const Tensor& stats, const Tensor& kept) {
    const at::OptionalDeviceGuard guard(hidden.device());
    const int64_t N = hidden.size(0);
    variable_list out = {f32_like({N}, hidden)};
    if (entropy) out.push_back(f32_like({N}, hidden));
    grx_lm_token_logps_args a = lm_args(hidden, weight, ids, temperature);
    a.logps = ptr<float>(out[0]);
    a.row_stats = ptr<float>(stats);
    a.entropy = entropy ? ptr<float>(out[1]) : nullptr;
    a.kept = ptr<float>(kept);
    const size_t n = api.lm_token_logps_scratch_bytes(a.N, a.H, a.V, entropy);
    const Tensor s = scratch(n, hidden.device());
    check(api.lm_token_logps(&a, ptr<void>(s), n, stream_on(hidden.device())));
    return out;
}

// Room for the products, if that many bytes may be kept and are there: without them the backward pass forms them again.
Tensor room_to_keep(size_t bytes, int64_t keep_bytes, const at::Device& d) {
    if ((int64_t)bytes > keep_bytes) return Tensor();
    try {
        return scratch(bytes, d);
    } catch (const c10::OutOfMemoryError&) {
        return Tensor();
    }
}

struct LmTokenLogps : Function<LmTokenLogps> {
    static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& ids,
                                 double temperature, bool entropy, int64_t keep_bytes) {
        const Tensor stats = f32_like({hidden.size(0), 2}, hidden);
        const size_t n = api.lm_token_logps_kept_bytes((int32_t)hidden.size(0), (int32_t)weight.size(0));
        const Tensor kept = room_to_keep(n, keep_bytes, hidden.device());
        const variable_list out = lm_forward(hidden, weight, ids, temperature, entropy, stats, kept);
        ctx->save_for_backward({hidden, weight, ids, stats, entropy ? out[1] : Tensor(), kept});
        ctx->saved_data["temperature"] = temperature;
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list incoming) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &hidden = saved[0], &weight = saved[1], &ids = saved[2], &stats = saved[3], &ent = saved[4];
        const at::OptionalDeviceGuard guard(hidden.device());
        refuse_nodes_outside(hidden.device());
        const bool want_h = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
        const Tensor g = grad_rows(incoming[0]), h = incoming.size() > 1 ? grad_rows(incoming[1]) : Tensor();
        const Tensor grad_h = want_h ? at::empty(hidden.sizes(), hidden.options()) : Tensor();
        const Tensor grad_w = want_w ? at::empty(weight.sizes(), weight.options()) : Tensor();
        grx_lm_token_logps_args a = lm_args(hidden, weight, ids, ctx->saved_data["temperature"].toDouble());
        if (a.N == 0 && want_w) grad_w.zero_();
        a.row_stats = ptr<float>(stats);
        a.entropy = ptr<float>(ent);
        a.grad_logps = ptr<float>(g);
        a.grad_entropy = ptr<float>(h);
        a.kept = ptr<float>(saved[5]);
        a.grad_hidden = ptr<void>(grad_h);
        a.grad_weight = ptr<void>(grad_w);
        const size_t n = api.lm_token_logps_backward_scratch_bytes(a.N, a.H, a.V, want_h, want_w);
        const Tensor s = scratch(n, hidden.device());
        check(api.lm_token_logps_backward(&a, ptr<void>(s), n, stream_on(hidden.device())));
        return once(incoming, {grad_h, grad_w, Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

py::object lm_head_token_logps(const Tensor& hidden, const Tensor& weight, const Tensor& token_ids, double temperature, bool entropy,
                               int64_t keep_bytes) {
    temperature = temperature_of(temperature);
    TORCH_CHECK_VALUE(keep_bytes >= 0, "keep_bytes must not be negative, got ", keep_bytes);
    TORCH_CHECK_TYPE(hidden.scalar_type() == at::kBFloat16 && weight.scalar_type() == at::kBFloat16,
                     "hidden states and weight must be bfloat16, got ", hidden.scalar_type(), " and ", weight.scalar_type());
    TORCH_CHECK_VALUE((hidden.dim() == 2 || hidden.dim() == 3) && token_ids.sizes() == hidden.sizes().slice(0, hidden.dim() - 1),
                      "hidden must be [..., H] with one row per token id: got ", hidden.sizes(), " for ids ", token_ids.sizes());
    const int64_t H = hidden.size(-1);
    TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) == H && weight.size(0) >= 1, "weight must be [V, ", H, "], got ",
                      weight.sizes());
    TORCH_CHECK_VALUE(H >= 64 && H % 64 == 0 && H <= 1 << 16 && weight.size(0) <= 1 << 24,
                      "the hidden size must be a multiple of 64 up to 2^16 and the vocabulary at most 2^24, got ", H, ", ",
                      weight.size(0));
    const Tensor ids = token_ids_of(token_ids, hidden.device()).reshape({-1}).contiguous();
    same_device(weight, hidden.device(), "weight");
    require_cuda(hidden, "hidden");
    const Tensor rows = aligned_rows(hidden.dim() == 2 ? hidden : hidden.reshape({ids.numel(), H})), w = aligned_rows(weight);
    if (constant(rows) && constant(w))
        return outputs(lm_forward(rows, w, ids, temperature, entropy, f32_like({rows.size(0), 2}, rows), Tensor()), token_ids.sizes());
    return outputs(LmTokenLogps::apply(rows, w, ids, temperature, entropy, keep_bytes), token_ids.sizes());
}

// ---- the loss ------------------------------------------------------------------------------------------------
struct PolicyLoss : Function<PolicyLoss> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logps, const Tensor& stats, grx_policy_loss_args* a, bool want_grad) {
        const at::OptionalDeviceGuard guard(logps.device());
        const Tensor loss = f32_like({}, logps);
        const Tensor unit = want_grad ? f32_like(logps.sizes(), logps) : Tensor();
        a->loss = ptr<float>(loss);
        a->stats = ptr<float>(stats);
        a->unit_grad = ptr<float>(unit);
        const size_t n = api.policy_loss_scratch_bytes(a->R, a->T);
        const Tensor s = scratch(n, logps.device());
        check(api.policy_loss(a, ptr<void>(s), n, stream_on(logps.device())));
        if (unit.defined()) ctx->save_for_backward({unit, stats});
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list incoming) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &unit = saved[0], &stats = saved[1];
        const at::OptionalDeviceGuard guard(unit.device());
        refuse_nodes_outside(unit.device());
        const Tensor g = grad_rows(incoming[0]);
        const Tensor grad = at::empty_like(unit);
        check(api.policy_loss_backward(ptr<float>(unit), ptr<float>(stats), ptr<float>(g), unit.numel(), ptr<float>(grad),
                                       stream_on(unit.device())));
        return once(incoming, {grad, Tensor(), Tensor(), Tensor()});
    }
};

Tensor f32_rows(const Tensor& t) { return rows_2d(t.scalar_type() == at::kFloat ? t : t.detach().to(at::kFloat)); }

py::tuple policy_loss(const Tensor& logps_, const Tensor& advantages, const Tensor& mask_, const std::optional<Tensor>& old_logps,
                      const std::optional<Tensor>& ref_logps, double epsilon_low, std::optional<double> epsilon_high_,
                      std::optional<double> delta, double beta, const std::string& loss_type, const std::string& level,
                      std::optional<double> max_completion_length, std::optional<double> num_items) {
    const at::Device device = logps_.device();
    TORCH_CHECK_VALUE(logps_.dim() == 2, "logps must be [rows, positions], got ", logps_.sizes());
    const int64_t R = logps_.size(0), T = logps_.size(1);
    TORCH_CHECK_VALUE(R < 1ll << 31 && T <= 1ll << 30, "at most 2^31 - 1 rows and 2^30 positions, got ", logps_.sizes());
    const auto shaped = [&](const Tensor& t, const char* name) {
        TORCH_CHECK_VALUE(t.sizes() == logps_.sizes(), name, " must have the shape of logps ", logps_.sizes(), ", got ", t.sizes());
    };
    shaped(mask_, "mask");
    if (old_logps) shaped(*old_logps, "old_logps");
    if (ref_logps) shaped(*ref_logps, "ref_logps");
    TORCH_CHECK_VALUE(advantages.sizes() == logps_.sizes() || (advantages.dim() == 1 && advantages.size(0) == R),
                      "advantages must be [", R, "] or [", R, ", ", T, "], got ", advantages.sizes());
    const auto floating = [&](const Tensor& t, const char* name) {
        same_device(t, device, name);
        TORCH_CHECK_TYPE(t.is_floating_point(), name, " must be floating point, got ", t.scalar_type());
    };
    same_device(mask_, device, "mask");
    floating(logps_, "logps");
    if (old_logps) floating(*old_logps, "old_logps");
    if (ref_logps) floating(*ref_logps, "ref_logps");
    floating(advantages, "advantages");
    const bool grpo = loss_type == "grpo", fixed = loss_type == "dr_grpo", dapo = loss_type == "dapo";
    TORCH_CHECK_VALUE(grpo || fixed || dapo || loss_type == "bnpo", "loss_type must be 'grpo', 'bnpo', 'dr_grpo' or 'dapo', got '",
                      loss_type, "'");
    TORCH_CHECK_VALUE(level == "token" || level == "sequence", "importance_sampling_level must be 'token' or 'sequence', got '",
                      level, "'");
    const double epsilon_high = epsilon_high_.value_or(epsilon_low);
    TORCH_CHECK_VALUE(epsilon_low >= 0.0 && epsilon_low < 1.0 && epsilon_high >= 0.0 && std::isfinite(epsilon_high),
                      "epsilon_low must lie in [0, 1) and epsilon_high must not be negative, got ", epsilon_low, ", ", epsilon_high);
    TORCH_CHECK_VALUE(!delta || (*delta > 1.0 + epsilon_high && std::isfinite(*delta)),
                      "delta must lie above 1 + epsilon_high, got ", delta.value_or(0.0));
    TORCH_CHECK_VALUE(std::isfinite(beta) && std::isfinite((float)beta), "beta must be finite, got ", beta);
    TORCH_CHECK_VALUE(beta == 0.0 || ref_logps, "a KL term (beta) needs ref_logps");
    double normalizer = 0.0;
    if (fixed || dapo) {
        const std::optional<double> given = fixed ? max_completion_length : num_items;
        TORCH_CHECK_VALUE(given && *given > 0.0 && std::isfinite(*given), "loss_type '", loss_type, "' needs a positive ",
                          fixed ? "max_completion_length" : "num_items");
        normalizer = *given * (fixed ? (double)std::max<int64_t>(R, 1) : 1.0);
    }
    require_cuda(logps_, "logps");

    const Tensor logps = rows_2d(logps_.scalar_type() == at::kFloat ? logps_ : logps_.to(at::kFloat));
    const Tensor old = old_logps ? f32_rows(*old_logps) : Tensor(), ref = ref_logps ? f32_rows(*ref_logps) : Tensor();
    const Tensor adv = advantages.scalar_type() == at::kFloat ? advantages : advantages.detach().to(at::kFloat);
    const auto mask_code = [](const Tensor& m) {
        switch (m.scalar_type()) {
            case at::kBool: case at::kByte: return GRX_MASK_U8;
            case at::kInt: return GRX_MASK_I32;
            case at::kLong: return GRX_MASK_I64;
            case at::kFloat: return GRX_MASK_F32;
            default: return -1;
        }
    };
    const Tensor mask = rows_2d(mask_code(mask_) >= 0 ? mask_ : mask_.gt(0));
    const Tensor stats = f32_like({4}, logps);
    grx_policy_loss_args a = {};
    a.logps = ptr<float>(logps);
    a.logps_stride = logps.stride(0);
    if (old.defined()) {
        a.old_logps = ptr<float>(old);
        a.old_stride = old.stride(0);
    }
    if (ref.defined()) {
        a.ref_logps = ptr<float>(ref);
        a.ref_stride = ref.stride(0);
    }
    a.advantages = ptr<float>(adv);
    a.adv_row_stride = adv.stride(0);
    a.adv_pos_stride = adv.dim() == 2 ? adv.stride(1) : 0;
    a.mask = mask.data_ptr();
    a.mask_stride = mask.stride(0);
    a.mask_type = mask_code(mask);
    a.R = (int32_t)R;
    a.T = (int32_t)T;
    a.sequence_level = level == "sequence";
    a.row_mean = grpo;
    a.beta = (float)beta;
    a.epsilon_low = epsilon_low;
    a.epsilon_high = epsilon_high;
    a.delta = delta.value_or(0.0);
    a.normalizer = normalizer;
    const Tensor loss = PolicyLoss::apply(logps, stats, &a, at::GradMode::is_enabled() && logps.requires_grad());
    // with a version counter of their own: the backward pass reads the fourth number, and the caller may write over the others
    const std::vector<Tensor> s = stats.variable_data().unbind(0);
    return py::make_tuple(loss, s[0], s[1], s[2]);
}

void bind(py::object error, py::dict addresses) {
    error_type = error.release().ptr();
    const auto at = [&](const char* name) { return (void*)addresses[name].cast<uintptr_t>(); };
#define GRX_BIND(name) api.name = reinterpret_cast<decltype(api.name)>(at("grx_" #name))
    GRX_BIND(last_error);
    GRX_BIND(token_logps_scratch_bytes);
    GRX_BIND(token_logps);
    GRX_BIND(token_logps_backward);
    GRX_BIND(lm_token_logps_scratch_bytes);
    GRX_BIND(lm_token_logps_backward_scratch_bytes);
    GRX_BIND(lm_token_logps_kept_bytes);
    GRX_BIND(lm_token_logps);
    GRX_BIND(lm_token_logps_backward);
    GRX_BIND(policy_loss_scratch_bytes);
    GRX_BIND(policy_loss);
    GRX_BIND(policy_loss_backward);
}

}  // namespace

PYBIND11_MODULE(_policy_ops, m) {
    m.attr("abi_version") = GRX_ABI_VERSION;
    m.attr("struct_bytes") = py::make_tuple(sizeof(grx_token_logps_args), sizeof(grx_lm_token_logps_args), sizeof(grx_policy_loss_args));
    m.def("bind", &bind);
    m.def("token_logps", &token_logps);
    m.def("lm_head_token_logps", &lm_head_token_logps);
    m.def("policy_loss", &policy_loss);
}
