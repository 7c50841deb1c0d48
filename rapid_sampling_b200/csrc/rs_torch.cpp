// PyTorch binding: the three functions of the reference's module (sampling.cpp:5-9) with the same
// names, argument order and tensor semantics, forwarding to the C ABI of this library.
// Argument names follow the reference's README so keyword calls work as well as positional ones.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/graph_task.h>

#include <map>
#include <mutex>
#include <stdexcept>
#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/rapid_sampling_b200.h"

namespace {

[[noreturn]] void fail(int rc, const std::string& detail) {
    std::string msg = std::string(rs_status_string(rc)) + detail + " !\n";
    if (rc == RS_ERR_CUDA) throw std::runtime_error(msg + rs_last_cuda_error());
    throw std::invalid_argument(msg);  // pybind11 maps this to ValueError, as in the reference
}

// One zero-initialised workspace per (device, stream); grows, never shrinks, and is kept for the life of the
// process (release_workspaces() drops them).  Returned by value: the reference count is taken under the lock, so a
// concurrent call that grows the same entry cannot free the buffer under a caller that still uses it.  Growing
// allocates: the first call with a given shape must come before any stream capture.
std::mutex g_ws_mu;
std::map<std::pair<int, cudaStream_t>, at::Tensor> g_ws_cache;
at::Tensor workspace_for(int device, cudaStream_t stream, size_t bytes) {
    std::lock_guard<std::mutex> lk(g_ws_mu);
    at::Tensor& w = g_ws_cache[{device, stream}];
    if (!w.defined() || (size_t)w.numel() < bytes)
        w = at::zeros({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device));
    return w;
}
at::Tensor workspace_if_any(int device, cudaStream_t stream) {
    std::lock_guard<std::mutex> lk(g_ws_mu);
    const auto it = g_ws_cache.find({device, stream});
    return it == g_ws_cache.end() ? at::Tensor() : it->second;
}

// Host mirror of the device status word, one pinned int per device: the kernels store a non-zero status there as
// well, so a failure (a bounded wait that gave up, a per-row temperature out of range) is noticed by the NEXT call
// on that device from host memory alone -- no copy, no synchronisation on the hot path.
// The word is made by the first call, also where that call is being captured: a graph keeps the word's address that its
// capture saw, so a word made later would never hear of its replays.  Kept for the life of the process, for the same reason.
std::mutex g_mirror_mu;
std::map<int, int*> g_mirror;
volatile int* mirror_for(int device) {      // of the current device
    std::lock_guard<std::mutex> lk(g_mirror_mu);
    int*& word = g_mirror[device];
    if (!word) {
        void* at = nullptr;
        c10::cuda::CUDAStreamCaptureModeGuard relaxed{cudaStreamCaptureModeRelaxed};      // an allocation is no part of the graph
        if (cudaHostAlloc(&at, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable) != cudaSuccess)
            throw std::runtime_error("no pinned memory for the status word !\n");
        *(int*)at = 0;
        if (rs_set_status_mirror((int*)at) != RS_OK) {
            cudaFreeHost(at);
            throw std::runtime_error("rs_set_status_mirror failed !\n");
        }
        word = (int*)at;
    }
    return word;
}
[[noreturn]] void throw_status(const char* what, int device, int v) {
    std::string msg = std::string(what) + " on cuda:" + std::to_string(device) + " reported: " + rs_status_string(v) + " !\n";
    if (v == RS_ERR_TEMPERATURE || v == RS_ERR_TOKEN) throw std::invalid_argument(msg);
    throw std::runtime_error(msg);
}
// Raises what an earlier call on this device left in the mirror, once.
void raise_pending_status(int device, at::Tensor& ws, cudaStream_t stream) {
    volatile int* w = mirror_for(device);
    const int v = *w;
    if (v == 0) return;
    *w = 0;
    rs_clear_status(ws.data_ptr(), stream);
    if (at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None) rs_logprobs_status(stream);
    throw_status("an earlier sampling call", device, v);
}

struct Shapes {
    int64_t B, T, V;
    float* pen;
    int dtype;
};

// The reference's argument checks (sampling.cu:451-486, :975-1011) plus the ones it leaves out (device, contiguity,
// size of `states`).
Shapes check_arguments(at::Tensor& logits, at::Tensor* penalties, at::Tensor& states, bool any_dtype) {
    const bool lowp = any_dtype && (logits.dtype() == at::kHalf || logits.dtype() == at::kBFloat16);
    if (logits.dtype() != at::kFloat && !lowp)
        throw std::invalid_argument("Logits tensor must be of type float32 (FP32), got " +
                                    std::string(logits.dtype().name()) + " !\n");
    if (!logits.is_cuda() || !states.is_cuda()) throw std::invalid_argument("logits and states must be CUDA tensors !\n");
    if (logits.dim() < 1 || logits.dim() > 3) throw std::invalid_argument("logits must have shape (V,), (B,V) or (B,T,V) !\n");
    if (!logits.is_contiguous() || !states.is_contiguous()) throw std::invalid_argument("logits and states must be contiguous !\n");
    Shapes sh;
    sh.V = logits.size(-1);
    sh.B = (logits.dim() >= 2) ? logits.size(0) : 1;            // sampling.cu:983
    sh.T = (logits.dim() == 3) ? logits.size(1) : 1;            // sampling.cu:984
    sh.pen = nullptr;
    if (penalties) {
        sh.B = (penalties->dim() == 2) ? penalties->size(0) : 1;        // sampling.cu:459
        if (penalties->dtype() != at::kFloat || !penalties->is_cuda() || !penalties->is_contiguous() ||
            penalties->get_device() != logits.get_device())
            throw std::invalid_argument("penalties must be a contiguous float32 CUDA tensor on the logits' device !\n");
        if (penalties->numel() != sh.B * sh.V) throw std::invalid_argument("penalties must have shape (B, V) !\n");
        if (logits.numel() < sh.B * sh.T * sh.V) throw std::invalid_argument("logits hold fewer rows than penalties !\n");
        sh.pen = penalties->data_ptr<float>();
    }
    if (sh.V > 0 && sh.B > 0 && states.numel() * (int64_t)states.element_size() < sh.B * RS_STATE_BYTES)
        throw std::invalid_argument("states tensor is smaller than B rows of setup_rand output !\n");
    if (states.get_device() != logits.get_device()) throw std::invalid_argument("states must live on the logits' device !\n");
    sh.dtype = logits.dtype() == at::kHalf ? RS_DTYPE_F16 : logits.dtype() == at::kBFloat16 ? RS_DTYPE_BF16 : RS_DTYPE_F32;
    return sh;
}

at::Tensor sample_common(at::Tensor& logits, at::Tensor* penalties, at::Tensor& states, double presence,
                         double repetition, double decay, double temperature, int64_t top_k, double top_p,
                         bool any_dtype = false) {
    const Shapes sh = check_arguments(logits, penalties, states, any_dtype);
    const int64_t B = sh.B, T = sh.T, V = sh.V;
    float* pen = sh.pen;

    c10::cuda::CUDAGuard guard(logits.device());
    const int dev = logits.get_device();
    cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev).stream();
    const size_t wsb = rs_workspace_bytes(B, V);
    at::Tensor ws = workspace_for(dev, stream, wsb);
    raise_pending_status(dev, ws, stream);
    at::Tensor out = at::empty({B > 0 ? B : 0}, at::TensorOptions().dtype(at::kInt).device(logits.device()));
    const int dt = sh.dtype;
    const int rc = rs_sample_typed(logits.data_ptr(), dt, B, T, V, pen, states.data_ptr(), out.data_ptr<int32_t>(), temperature,
                                   top_k, top_p, presence, repetition, decay, ws.data_ptr(), (size_t)ws.numel(), stream,
                                   nullptr, nullptr);
    if (rc == RS_ERR_VOCAB) fail(rc, ", got " + std::to_string(V));
    if (rc == RS_ERR_BATCH) fail(rc, ", got B=" + std::to_string(B) + ", T=" + std::to_string(T));
    if (rc == RS_ERR_TEMPERATURE) fail(rc, ", got " + std::to_string(temperature));
    if (rc != RS_OK) fail(rc, "");
    return out;
}

// Per-row temperature / top_k / top_p tensors (B values each, or None for the neutral value in every row).
const void* row_tensor(const c10::optional<at::Tensor>& t, at::ScalarType want, int64_t B, const at::Tensor& logits,
                       const char* name) {
    if (!t.has_value()) return nullptr;
    if (t->scalar_type() != want || !t->is_cuda() || !t->is_contiguous() || t->numel() != B ||
        t->get_device() != logits.get_device())
        throw std::invalid_argument(std::string(name) + " must be a contiguous CUDA tensor of B values (" +
                                    (want == at::kInt ? "int32" : "float32") + ") on the logits' device !\n");
    return t->data_ptr();
}

}  // namespace

// Returns ids (B,) int32, or (ids, probability of the id, kept mass) when return_prob is set.
pybind11::object batch_sampling_rows(at::Tensor& logits, at::Tensor& states, c10::optional<at::Tensor> temperature,
                                     c10::optional<at::Tensor> top_k, c10::optional<at::Tensor> top_p,
                                     c10::optional<at::Tensor> penalties, double presence_penalty,
                                     double repetition_penalty, double penalty_decay, bool return_prob) {
    at::Tensor* pen_t = penalties.has_value() ? &penalties.value() : nullptr;
    const Shapes sh = check_arguments(logits, pen_t, states, true);
    const void* tp = row_tensor(temperature, at::kFloat, sh.B, logits, "temperature");
    const void* kp = row_tensor(top_k, at::kInt, sh.B, logits, "top_k");
    const void* pp = row_tensor(top_p, at::kFloat, sh.B, logits, "top_p");
    c10::cuda::CUDAGuard guard(logits.device());
    const int dev = logits.get_device();
    cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev).stream();
    at::Tensor ws = workspace_for(dev, stream, rs_rows_workspace_bytes(sh.B, sh.V));
    raise_pending_status(dev, ws, stream);
    const int64_t n = sh.B > 0 ? sh.B : 0;
    at::Tensor out = at::empty({n}, at::TensorOptions().dtype(at::kInt).device(logits.device()));
    at::Tensor prob, kept;
    if (return_prob) {
        prob = at::empty({n}, at::TensorOptions().dtype(at::kFloat).device(logits.device()));
        kept = at::empty({n}, at::TensorOptions().dtype(at::kFloat).device(logits.device()));
    }
    const int rc = rs_sample_rows(logits.data_ptr(), sh.dtype, sh.B, sh.T, sh.V, sh.pen, states.data_ptr(), out.data_ptr<int32_t>(),
                                  (const float*)tp, (const int32_t*)kp, (const float*)pp, presence_penalty, repetition_penalty,
                                  penalty_decay, return_prob ? prob.data_ptr<float>() : nullptr,
                                  return_prob ? kept.data_ptr<float>() : nullptr, ws.data_ptr(), (size_t)ws.numel(), stream);
    if (rc == RS_ERR_VOCAB) fail(rc, ", got " + std::to_string(sh.V));
    if (rc == RS_ERR_BATCH) fail(rc, ", got B=" + std::to_string(sh.B) + ", T=" + std::to_string(sh.T));
    if (rc != RS_OK) fail(rc, "");
    if (return_prob) return pybind11::make_tuple(out, prob, kept);
    return pybind11::cast(out);
}

at::Tensor setup_rand(int64_t seed, int64_t B) {
    if (B <= 0) throw std::invalid_argument("B must be positive, got B=" + std::to_string(B) + " !\n");
    at::Tensor state = at::empty({B * RS_STATE_BYTES}, at::TensorOptions().dtype(at::kChar).device(at::kCUDA));
    const int rc = rs_setup_rand(state.data_ptr(), (uint64_t)seed, B, 0, at::cuda::getCurrentCUDAStream().stream());
    if (rc != RS_OK) fail(rc, "");
    return state;
}

at::Tensor batch_sampling_temperature_topk_topp(at::Tensor& logits, at::Tensor& states, double temperature, int64_t top_k,
                                                double top_p) {
    return sample_common(logits, nullptr, states, 0.0, 0.0, 0.0, temperature, top_k, top_p);
}

at::Tensor batch_sampling_repetition_temperature_topk_topp(at::Tensor& logits, at::Tensor& penalties, at::Tensor& states,
                                                           double presence_penalty, double repetition_penalty,
                                                           double penalty_decay, double temperature, int64_t top_k,
                                                           double top_p) {
    return sample_common(logits, &penalties, states, presence_penalty, repetition_penalty, penalty_decay, temperature,
                         top_k, top_p);
}

// The same two calls for fp32, fp16 or bf16 logits (the reference's functions above stay fp32-only, as the reference's).
at::Tensor sample_any(at::Tensor& logits, at::Tensor& states, double temperature, int64_t top_k, double top_p) {
    return sample_common(logits, nullptr, states, 0.0, 0.0, 0.0, temperature, top_k, top_p, true);
}
at::Tensor sample_repetition_any(at::Tensor& logits, at::Tensor& penalties, at::Tensor& states, double presence_penalty,
                                 double repetition_penalty, double penalty_decay, double temperature, int64_t top_k,
                                 double top_p) {
    return sample_common(logits, &penalties, states, presence_penalty, repetition_penalty, penalty_decay, temperature,
                         top_k, top_p, true);
}

// ---- log probabilities ---------------------------------------------------------------------------------------------

// The same for the calls that have no workspace.  A call that is being captured does not raise: clearing the device's word would
// become a part of the graph.
static void raise_pending_logprobs(int device, cudaStream_t stream) {
    volatile int* w = mirror_for(device);
    const int v = *w;
    if (v == 0 || at::cuda::currentStreamCaptureStatusMayInitCtx() != at::cuda::CaptureStatus::None) return;
    *w = 0;
    rs_logprobs_status(stream);      // clears the device's word
    const at::Tensor ws = workspace_if_any(device, stream);      // it may have been a sampling call's, whose workspace has it too
    if (ws.defined()) rs_clear_status(ws.data_ptr(), stream);
    throw_status("an earlier call", device, v);
}

// Logits (V,), (B, V) or (B, T, V) with any strides but along V, one token per row, one temperature or one per row.
static rs_logprob_call logprob_call(const at::Tensor& logits, const c10::optional<at::Tensor>& tokens, double temperature,
                                    const c10::optional<at::Tensor>& row_temperature) {
    rs_logprob_call c = {};
    if (logits.scalar_type() != at::kFloat && logits.scalar_type() != at::kHalf && logits.scalar_type() != at::kBFloat16)
        throw std::invalid_argument("logits must be float32, float16 or bfloat16, got " + std::string(logits.dtype().name()) + " !\n");
    if (!logits.is_cuda()) throw std::invalid_argument("logits must be a CUDA tensor !\n");
    const int64_t d = logits.dim();
    if (d < 1 || d > 3) throw std::invalid_argument("logits must have shape (V,), (B,V) or (B,T,V) !\n");
    c.V = logits.size(-1);
    if (c.V < 1 || c.V > RS_LOGPROB_MAX_V) throw std::invalid_argument("Vocabulary size must lie in [1, 1048576], got " + std::to_string(c.V) + " !\n");
    if (c.V > 1 && logits.stride(-1) != 1) throw std::invalid_argument("logits must be contiguous along the vocabulary !\n");
    c.logits = logits.data_ptr();
    c.dtype = logits.scalar_type() == at::kHalf ? RS_DTYPE_F16 : logits.scalar_type() == at::kBFloat16 ? RS_DTYPE_BF16 : RS_DTYPE_F32;
    c.B = d >= 2 ? logits.size(0) : 1;
    c.T = d == 3 ? logits.size(1) : 1;
    c.stride_b = d >= 2 ? logits.stride(0) : 0;
    c.stride_t = d == 3 ? logits.stride(1) : 0;
    const at::IntArrayRef rows = logits.sizes().slice(0, d - 1);
    c.token_bits = 64;
    if (tokens.has_value()) {
        const at::Tensor& t = *tokens;
        if ((t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) || !t.is_cuda() || t.get_device() != logits.get_device())
            throw std::invalid_argument("tokens must be an int32 or int64 CUDA tensor on the logits' device !\n");
        if (t.sizes() != rows) throw std::invalid_argument("tokens must have the logits' shape without the vocabulary !\n");
        c.tokens = t.data_ptr();
        c.token_bits = t.scalar_type() == at::kInt ? 32 : 64;
        c.token_stride_b = d >= 2 ? t.stride(0) : 0;
        c.token_stride_t = d == 3 ? t.stride(1) : 0;
    }
    if (!(temperature >= 0.001 && temperature <= 1000)) fail(RS_ERR_TEMPERATURE, ", got " + std::to_string(temperature));
    c.temperature = temperature;
    if (row_temperature.has_value()) {
        const at::Tensor& t = *row_temperature;
        if (t.scalar_type() != at::kFloat || !t.is_cuda() || t.get_device() != logits.get_device())
            throw std::invalid_argument("temperature must be a float32 CUDA tensor on the logits' device !\n");
        if (t.numel() == 1) {      // strides 0: for every row
        } else if (t.sizes() == rows) {
            c.temperature_stride_b = d >= 2 ? t.stride(0) : 0;
            c.temperature_stride_t = d == 3 ? t.stride(1) : 0;
        } else if (d == 3 && t.dim() == 1 && t.size(0) == c.B) {
            c.temperature_stride_b = t.stride(0);
        } else {
            throw std::invalid_argument("temperature must hold one value, one per row, or one per sequence of (B,T,V) logits !\n");
        }
        c.row_temperature = t.data_ptr<float>();
    }
    c.stream = at::cuda::getCurrentCUDAStream(logits.get_device()).stream();
    return c;
}

static void check_logprobs(int rc) {
    if (rc != RS_OK) fail(rc, "");
}

struct Logprobs {
    at::Tensor logprobs, entropy, stats;      // stats: for the backward call, or undefined
};
static Logprobs token_logprobs_run(const at::Tensor& logits, const at::Tensor& tokens, double temperature,
                                   const c10::optional<at::Tensor>& row_temperature, bool keep_stats) {
    rs_logprob_call c = logprob_call(logits, tokens, temperature, row_temperature);
    c10::cuda::CUDAGuard guard(logits.device());
    raise_pending_logprobs(logits.get_device(), (cudaStream_t)c.stream);
    const auto f32 = at::TensorOptions().dtype(at::kFloat).device(logits.device());
    at::Tensor lp = at::empty(tokens.sizes(), f32), ent = at::empty(tokens.sizes(), f32), stats;
    if (keep_stats) stats = at::empty({c.B, c.T, 2}, f32);
    if (lp.numel() > 0)
        check_logprobs(rs_token_logprobs(&c, lp.data_ptr<float>(), ent.data_ptr<float>(), keep_stats ? stats.data_ptr<float>() : nullptr));
    return {lp, ent, stats};
}

static at::Tensor token_logprobs_backward(const at::Tensor& logits, const at::Tensor& tokens, double temperature,
                                          const c10::optional<at::Tensor>& row_temperature, const at::Tensor& entropy,
                                          const at::Tensor& stats, const c10::optional<at::Tensor>& g_logprob,
                                          const c10::optional<at::Tensor>& g_entropy) {
    rs_logprob_call c = logprob_call(logits, tokens, temperature, row_temperature);
    c10::cuda::CUDAGuard guard(logits.device());
    const int64_t d = logits.dim();
    const float* g[2] = {nullptr, nullptr};
    int64_t s[2][2] = {{0, 0}, {0, 0}};
    for (int i = 0; i < 2; i++) {
        const c10::optional<at::Tensor>& t = i ? g_entropy : g_logprob;
        if (!t.has_value()) continue;
        if (t->scalar_type() != at::kFloat || t->sizes() != tokens.sizes() || !t->is_cuda() || t->get_device() != logits.get_device())
            throw std::invalid_argument("incoming gradients must be float32 CUDA tensors of the tokens' shape !\n");
        g[i] = t->data_ptr<float>();
        s[i][0] = d >= 2 ? t->stride(0) : 0;
        s[i][1] = d == 3 ? t->stride(1) : 0;
    }
    for (const at::Tensor* t : {&entropy, &stats})
        if (t->scalar_type() != at::kFloat || !t->is_contiguous() || t->numel() != c.B * c.T * (t == &stats ? 2 : 1) || !t->is_cuda() ||
            t->get_device() != logits.get_device())
            throw std::invalid_argument("entropy and stats must be those of the forward call !\n");
    at::Tensor grad = at::empty(logits.sizes(), logits.options());
    if (grad.numel() > 0)
        check_logprobs(rs_token_logprobs_backward(&c, entropy.data_ptr<float>(), stats.data_ptr<float>(), g[0], s[0][0], s[0][1], g[1],
                                                  s[1][0], s[1][1], grad.data_ptr()));
    return grad;
}

// Gradients for nodes that belong to the legacy default stream cannot be captured: that stream waits for nothing in a capture, and
// the engine's attempt spoils the capture or ends the process.  Such are the nodes of an eager forward pass, and the accumulation
// of a leaf as long as an eager graph of it lives, an earlier step's for instance.  So such a backward call is refused, where the
// pass at hand hands such a node a gradient: what lies behind the tensors that torch.autograd.grad was asked for is left alone.
static void check_captured_backward(const at::Tensor& logits) {
    if (at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None) return;
    const auto* asked = torch::autograd::get_current_graph_task_exec_info();      // empty: every node that can be reached
    auto reached = [&](torch::autograd::Node* n) {
        if (!asked || asked->empty()) return true;
        const auto it = asked->find(n);
        return it != asked->end() && it->second.should_execute();
    };
    const auto start = logits.grad_fn() ? logits.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(logits);
    std::vector<torch::autograd::Node*> todo = {start.get()};
    std::unordered_set<torch::autograd::Node*> seen;
    while (!todo.empty()) {
        torch::autograd::Node* n = todo.back();
        todo.pop_back();
        if (!n || !reached(n) || !seen.insert(n).second) continue;
        const auto s = n->stream();
        if (s && s->device_type() == c10::DeviceType::CUDA && *s == at::cuda::getDefaultCUDAStream(s->device_index()).unwrap())
            throw std::runtime_error("the backward pass of batch_token_logprobs cannot be captured: it leads into an eager graph, made on the default "
                                     "stream, or to leaves of which such a graph is alive !\n");
        for (const auto& e : n->next_edges()) todo.push_back(e.function.get());
    }
}

struct RowTemperature {      // no input of the graph
    c10::optional<at::Tensor> t;
};
class TokenLogprobs : public torch::autograd::Function<TokenLogprobs> {
  public:
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& tokens,
                                                  double temperature, const RowTemperature& rows) {
        Logprobs r = token_logprobs_run(logits, tokens, temperature, rows.t, true);
        ctx->set_materialize_grads(false);
        ctx->saved_data["temperature"] = temperature;
        torch::autograd::variable_list keep = {logits, tokens, r.entropy, r.stats};
        if (rows.t.has_value()) keep.push_back(*rows.t);
        ctx->save_for_backward(std::move(keep));
        return {r.logprobs, r.entropy};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
        if (at::GradMode::is_enabled()) throw std::runtime_error("batch_token_logprobs is differentiable once: no create_graph !\n");
        const auto saved = ctx->get_saved_variables();
        check_captured_backward(saved[0]);
        at::Tensor grad;
        if (g[0].defined() || g[1].defined()) {
            auto maybe = [](const at::Tensor& t) { return t.defined() ? c10::optional<at::Tensor>(t) : c10::nullopt; };
            grad = token_logprobs_backward(saved[0], saved[1], ctx->saved_data["temperature"].toDouble(),
                                           saved.size() > 4 ? c10::optional<at::Tensor>(saved[4]) : c10::nullopt, saved[2], saved[3], maybe(g[0]),
                                           maybe(g[1]));
        }
        return {grad, at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

// (log probabilities, entropies); part of the autograd graph where the logits are
static pybind11::tuple token_logprobs(const at::Tensor& logits, const at::Tensor& tokens, double temperature,
                                      const c10::optional<at::Tensor>& row_temperature) {
    if (row_temperature.has_value() && row_temperature->requires_grad())
        throw std::invalid_argument("the temperature is not differentiated: it must not require a gradient !\n");
    // a result without a tangent would count as a constant
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() &&
        (logits._fw_grad(0).defined() || (row_temperature.has_value() && row_temperature->_fw_grad(0).defined())))
        throw std::invalid_argument("batch_token_logprobs is differentiable in reverse mode only: no forward-mode tangents !\n");
    if (logits.requires_grad() && at::GradMode::is_enabled()) {
        const auto r = TokenLogprobs::apply(logits, tokens, temperature, RowTemperature{row_temperature});
        return pybind11::make_tuple(r[0], r[1]);
    }
    const Logprobs r = token_logprobs_run(logits, tokens, temperature, row_temperature, false);
    return pybind11::make_tuple(r.logprobs, r.entropy);
}

// (log probabilities, ranks, entropies, top log probabilities, top ids); the first two None without tokens
static pybind11::tuple top_logprobs(const at::Tensor& logits, int64_t top_n, const c10::optional<at::Tensor>& tokens, double temperature,
                                    const c10::optional<at::Tensor>& row_temperature) {
    rs_logprob_call c = logprob_call(logits, tokens, temperature, row_temperature);
    if (top_n < 1 || top_n > RS_LOGPROB_MAX_TOP)
        throw std::invalid_argument("top_n must lie in [1, " + std::to_string(RS_LOGPROB_MAX_TOP) + "], got " + std::to_string(top_n) + " !\n");
    c10::cuda::CUDAGuard guard(logits.device());
    raise_pending_logprobs(logits.get_device(), (cudaStream_t)c.stream);
    const auto f32 = at::TensorOptions().dtype(at::kFloat).device(logits.device());
    std::vector<int64_t> rows(logits.sizes().begin(), logits.sizes().end() - 1), slots = rows;
    slots.push_back(top_n);
    at::Tensor ent = at::empty(rows, f32), top = at::empty(slots, f32), ids = at::empty(slots, f32.dtype(at::kInt)), lp, rank;
    if (tokens.has_value()) {
        lp = at::empty(rows, f32);
        rank = at::empty(rows, f32.dtype(at::kInt));
    }
    if (ent.numel() > 0)
        check_logprobs(rs_top_logprobs(&c, (int32_t)top_n, tokens.has_value() ? lp.data_ptr<float>() : nullptr,
                                       tokens.has_value() ? rank.data_ptr<int32_t>() : nullptr, ent.data_ptr<float>(),
                                       top.data_ptr<float>(), ids.data_ptr<int32_t>()));
    if (!tokens.has_value()) return pybind11::make_tuple(pybind11::none(), pybind11::none(), ent, top, ids);
    return pybind11::make_tuple(lp, rank, ent, top, ids);
}

// ---- lm_head -------------------------------------------------------------------------------------------------------

static int dtype_of(const at::Tensor& t, const char* name) {
    if (t.scalar_type() == at::kFloat) return RS_DTYPE_F32;
    if (t.scalar_type() == at::kHalf) return RS_DTYPE_F16;
    if (t.scalar_type() == at::kBFloat16) return RS_DTYPE_BF16;
    throw std::invalid_argument(std::string(name) + " must be float32, float16 or bfloat16, got " + std::string(t.dtype().name()) + " !\n");
}
// Elements between the rows of (..., n); every row must follow the one before at the same distance.
static int64_t row_stride(const at::Tensor& t, const char* name) {
    const int64_t d = t.dim();
    if (t.numel() == 0) return t.size(-1);      // strides of an empty tensor mean nothing
    if (t.size(-1) > 1 && t.stride(-1) != 1) throw std::invalid_argument(std::string(name) + " must be contiguous along the last dimension !\n");
    int64_t step = 0, rows = 1;      // of the dimensions so far, from the last
    for (int64_t i = d - 2; i >= 0; i--) {
        if (t.size(i) == 1) continue;
        if (rows == 1) step = t.stride(i);
        else if (t.stride(i) != step * rows) throw std::invalid_argument(std::string(name) + " must have rows at equal distances !\n");
        rows *= t.size(i);
    }
    return rows == 1 ? t.size(-1) : step;
}

static pybind11::tuple lm_head_quantize(const at::Tensor& weight) {
    const int dt = dtype_of(weight, "weight");
    if (!weight.is_cuda() || weight.dim() != 2) throw std::invalid_argument("weight must be a CUDA tensor of shape (V, K) !\n");
    const int64_t V = weight.size(0), K = weight.size(1);
    if (V < 1 || V > RS_HEAD_MAX_ROWS || K < 16 || K > RS_HEAD_MAX_K || K % 16 != 0)
        throw std::invalid_argument("K must be a multiple of 16 in [16, 65536] and V at least 1, got V=" + std::to_string(V) + ", K=" + std::to_string(K) + " !\n");
    const int64_t step = row_stride(weight, "weight");
    c10::cuda::CUDAGuard guard(weight.device());
    at::Tensor codes = at::empty({V, K}, weight.options().dtype(at::kFloat8_e4m3fn).memory_format(at::MemoryFormat::Contiguous));
    at::Tensor scales = at::empty({(V + 127) / 128, (K + 127) / 128}, codes.options().dtype(at::kFloat));
    const int rc = rs_head_quantize(weight.data_ptr(), dt, V, K, step, codes.data_ptr(), scales.data_ptr<float>(),
                                    at::cuda::getCurrentCUDAStream(weight.get_device()).stream());
    if (rc != RS_OK) fail(rc, "");
    return pybind11::make_tuple(codes, scales);
}

static at::Tensor lm_head_logits(const at::Tensor& hidden, const at::Tensor& codes, const at::Tensor& scales, at::ScalarType dtype,
                                 const c10::optional<at::Tensor>& out_) {
    const int hdt = dtype_of(hidden, "hidden");
    if (!hidden.is_cuda() || hidden.dim() < 1) throw std::invalid_argument("hidden must be a CUDA tensor of shape (..., K) !\n");
    const int dev = hidden.get_device();
    if (codes.scalar_type() != at::kFloat8_e4m3fn || codes.dim() != 2 || !codes.is_cuda() || codes.get_device() != dev || !codes.is_contiguous() ||
        ((uintptr_t)codes.data_ptr() & 15))
        throw std::invalid_argument("codes must be a contiguous, 16-byte aligned float8_e4m3fn tensor of shape (V, K) on the hidden states' device !\n");
    const int64_t V = codes.size(0), K = codes.size(1), M = hidden.numel() / std::max<int64_t>(hidden.size(-1), 1);
    if (V < 1 || V > RS_HEAD_MAX_ROWS || K < 16 || K > RS_HEAD_MAX_K || K % 16 != 0 || M > RS_HEAD_MAX_ROWS)
        throw std::invalid_argument("K must be a multiple of 16 in [16, 65536] and V at least 1, got V=" + std::to_string(V) + ", K=" + std::to_string(K) + " !\n");
    if (hidden.size(-1) != K) throw std::invalid_argument("hidden must have the codes' K columns !\n");
    if (scales.scalar_type() != at::kFloat || !scales.is_cuda() || scales.get_device() != dev || !scales.is_contiguous() || scales.dim() != 2 ||
        scales.size(0) != (V + 127) / 128 || scales.size(1) != (K + 127) / 128)
        throw std::invalid_argument("scales must be a contiguous float32 tensor with one value for each block of 128 x 128 codes !\n");
    const int64_t step = row_stride(hidden, "hidden");
    std::vector<int64_t> shape(hidden.sizes().begin(), hidden.sizes().end() - 1);
    shape.push_back(V);
    c10::cuda::CUDAGuard guard(hidden.device());
    cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev).stream();
    raise_pending_logprobs(dev, stream);
    at::Tensor out;
    if (out_.has_value()) {
        out = *out_;
        if (!out.is_cuda() || out.get_device() != dev || out.sizes() != at::IntArrayRef(shape) || out.scalar_type() != dtype)
            throw std::invalid_argument("out must have the hidden states' shape with V columns, the requested type, and their device !\n");
        if (out.requires_grad() && at::GradMode::is_enabled())
            throw std::invalid_argument("out must not require a gradient: the call is not differentiable !\n");
    } else {
        out = at::empty(shape, at::TensorOptions().dtype(dtype).device(hidden.device()));
    }
    const int odt = dtype_of(out, "dtype");
    const int64_t ostep = row_stride(out, "out");
    if (M > 1 && ostep < V) throw std::invalid_argument("out must have rows that do not overlap !\n");
    if (M == 0) return out;
    // the caching allocator hands the workspace out per stream and, while capturing, per graph: no two calls share it
    at::Tensor ws = at::empty({(int64_t)rs_head_workspace_bytes(M, K)}, at::TensorOptions().dtype(at::kByte).device(hidden.device()));
    const int rc = rs_head_logits(hidden.data_ptr(), hdt, M, K, step, codes.data_ptr(), scales.data_ptr<float>(), V, out.data_ptr(), odt,
                                  std::max(ostep, V), ws.data_ptr(), (size_t)ws.numel(), stream);
    if (rc != RS_OK) fail(rc, "");
    if (out_.has_value() && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();      // graphs that saved `out` notice
    return out;
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    namespace py = pybind11;
    m.def("setup_rand", &setup_rand, py::arg("seed"), py::arg("B"));
    m.def("batch_sampling_repetition_temperature_topk_topp", &batch_sampling_repetition_temperature_topk_topp,
          py::arg("logits"), py::arg("penalties"), py::arg("states"), py::arg("presence_penalty"),
          py::arg("repetition_penalty"), py::arg("penalty_decay"), py::arg("temperature"), py::arg("top_k"),
          py::arg("top_p"));
    m.def("batch_sampling_temperature_topk_topp", &batch_sampling_temperature_topk_topp, py::arg("logits"),
          py::arg("states"), py::arg("temperature"), py::arg("top_k"), py::arg("top_p"));
    m.def("batch_sampling_temperature_topk_topp_any", &sample_any, py::arg("logits"), py::arg("states"),
          py::arg("temperature"), py::arg("top_k"), py::arg("top_p"));
    m.def("batch_sampling_repetition_temperature_topk_topp_any", &sample_repetition_any, py::arg("logits"),
          py::arg("penalties"), py::arg("states"), py::arg("presence_penalty"), py::arg("repetition_penalty"),
          py::arg("penalty_decay"), py::arg("temperature"), py::arg("top_k"), py::arg("top_p"));
    m.def("batch_sampling_rows", &batch_sampling_rows, py::arg("logits"), py::arg("states"), py::arg("temperature") = py::none(),
          py::arg("top_k") = py::none(), py::arg("top_p") = py::none(), py::arg("penalties") = py::none(),
          py::arg("presence_penalty") = 0.0, py::arg("repetition_penalty") = 0.0, py::arg("penalty_decay") = 0.0,
          py::arg("return_prob") = false);
    m.def("token_logprobs", &token_logprobs, py::arg("logits"), py::arg("tokens"), py::arg("temperature"), py::arg("row_temperature"));
    m.def("top_logprobs", &top_logprobs, py::arg("logits"), py::arg("top_n"), py::arg("tokens"), py::arg("temperature"),
          py::arg("row_temperature"));
    m.def("lm_head_quantize", &lm_head_quantize, py::arg("weight"));
    m.def("lm_head_logits", [](const at::Tensor& hidden, const at::Tensor& codes, const at::Tensor& scales, py::object dtype,
                               c10::optional<at::Tensor> out) {
        if (!THPDtype_Check(dtype.ptr())) throw std::invalid_argument("dtype must be a torch.dtype !\n");
        return lm_head_logits(hidden, codes, scales, reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type, out);
    }, py::arg("hidden"), py::arg("codes"), py::arg("scales"), py::arg("dtype"), py::arg("out"));
    m.def("kernel_launch_count", []() { return rs_kernel_launch_count(); });
    m.def("device_status", []() {
        // Synchronises the current stream and returns the status word of its workspace (0 = ok), clearing word and mirror.
        const int dev = c10::cuda::current_device();
        cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev).stream();
        at::Tensor ws = workspace_for(dev, stream, 256);
        int v = rs_device_status(ws.data_ptr(), stream);
        if (v != 0) rs_clear_status(ws.data_ptr(), stream);
        const int lp = rs_logprobs_status(stream);      // the word of the calls without a workspace
        if (v == 0) v = lp;
        volatile int* w = mirror_for(dev);
        if (v == 0) v = *w;     // a status raised through another workspace of this device
        *w = 0;
        return v;
    });
    m.def("selftest_bounded_wait", [](int64_t polls) {
        // Failure-path instrumentation: one CTA waits on a barrier nothing completes; the next sampling call raises.
        const int dev = c10::cuda::current_device();
        cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev).stream();
        at::Tensor ws = workspace_for(dev, stream, 256);
        mirror_for(dev);
        const int rc = rs_selftest_bounded_wait(ws.data_ptr(), (uint32_t)polls, stream);
        if (rc != RS_OK) fail(rc, "");
    }, py::arg("polls") = 4);
    m.def("release_workspaces", []() {
        std::lock_guard<std::mutex> lk(g_ws_mu);
        g_ws_cache.clear();
    });
    m.def("version", []() { return std::string(rs_version()); });
}
