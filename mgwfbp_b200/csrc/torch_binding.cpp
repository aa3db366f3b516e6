// Host side of the language-model operators for CUDA tensors: outputs and workspaces, one launch call, and the nodes of the
// autograd graph.  The kernels stay in libmgwfbp_b200.so (lm_api.h); their addresses are handed over by bind(), so that this
// module works with whichever build of that library the process has loaded.  Arguments that the kernels do not take give no
// result here; the Python functions in front of this module then say what is wrong with them.
//
// Why it exists: for a model's window of a few hundred tokens the kernels take 10 to 20 us and the host decides.  Host time of
// forward and backward, nodes and launches in Python against here: embedding 83 and 47 us, log probabilities 109 and 57,
// cross entropy 92 and 51; without gradients 11 and 5 us for a lookup, 16 and 6 for log probabilities; clipping 161
// gradients 88 and 26.  About 40 us of a backward pass are the engine's own: a pass through one view costs as much.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <unordered_map>
#include <vector>

#include "lm_api.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct Library {
    const char* (*last_error)(void) = nullptr;
    decltype(&mgw_embedding_order_bytes) embedding_order_bytes = nullptr;
    decltype(&mgw_embedding_fwd) embedding_fwd = nullptr;
    decltype(&mgw_embedding_grad_bytes) embedding_grad_bytes = nullptr;
    decltype(&mgw_embedding_grad) embedding_grad = nullptr;
    decltype(&mgw_logprob_fwd) logprob_fwd = nullptr;
    decltype(&mgw_logprob_bwd) logprob_bwd = nullptr;
    decltype(&mgw_cross_entropy_fwd) cross_entropy_fwd = nullptr;
    decltype(&mgw_grad_clip_bytes) grad_clip_bytes = nullptr;
    decltype(&mgw_grad_clip) grad_clip = nullptr;
    int* status = nullptr;
} lib;

struct NativeError : std::runtime_error {
    using std::runtime_error::runtime_error;
};

constexpr int kBadArgument = 2;                                  // MGW_ERR_ARG

void check(int code, const char* what) {
    if (code != 0) throw NativeError(std::string(what) + " failed with code " + std::to_string(code) + ": " + lib.last_error());
}

// Launches made here, by the name under which the package counts them.
enum Launch { kEmbeddingFwd, kEmbeddingGrad, kLogprobFwd, kLogprobBwd, kCrossEntropyFwd, kCrossEntropyBwd, kGradNorm, kGradScale,
              kGradNormFinish, kLaunches };
const char* const kNames[kLaunches] = {"embedding_fwd", "embedding_grad", "logprob_fwd", "logprob_bwd", "cross_entropy_fwd",
                                       "cross_entropy_bwd", "grad_norm", "grad_scale", "grad_norm_finish"};
std::atomic<long long> launches[kLaunches];

void count(Launch which, long long n = 1) { launches[which].fetch_add(n, std::memory_order_relaxed); }

int type_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return MGW_F32;
        case at::kHalf: return MGW_F16;
        case at::kBFloat16: return MGW_BF16;
        default: return -1;
    }
}

bool wide(const Tensor& tokens) { return tokens.scalar_type() == at::kLong; }

bool fits(const Tensor& values, const Tensor& tokens) {
    TORCH_CHECK(lib.status != nullptr, "the kernels' library is not bound");
    return values.is_cuda() && tokens.device() == values.device() && type_code(values) >= 0 && values.dim() >= 1 && values.size(-1) >= 1 &&
           values.size(-1) <= 1LL << 30 && (tokens.scalar_type() == at::kInt || wide(tokens)) && tokens.numel() <= 0x7fffffffLL;
}
// one row of values for each token
bool fits_rows(const Tensor& values, const Tensor& tokens) {
    return fits(values, tokens) && values.dim() == tokens.dim() + 1 && values.sizes().slice(0, tokens.dim()) == tokens.sizes();
}

// The tensor's device is the current one while this lives; launches go to its current stream.
struct Place {
    c10::cuda::CUDAGuard guard;
    void* stream;
    explicit Place(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.get_device()).stream()) {}
};

// [n, width] with contiguous rows that lie ld elements apart
struct Rows {
    Tensor t;
    int64_t n, width, ld;
    explicit Rows(const Tensor& x) : t(x.dim() == 2 ? x : x.reshape({-1, x.size(-1)})), n(t.size(0)), width(t.size(1)), ld(t.stride(0)) {
        if ((width > 1 && t.stride(1) != 1) || (n > 1 && ld < width)) {
            t = t.contiguous();
            ld = width;
        }
        if (n <= 1) ld = width;
    }
};

float* floats(const Tensor& t) { return t.defined() ? t.mutable_data_ptr<float>() : nullptr; }
const float* const_floats(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }

at::DimVector with_last(at::IntArrayRef shape, int64_t last) {
    at::DimVector s(shape.begin(), shape.end());
    s.push_back(last);
    return s;
}

bool differentiable(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

template <typename N>
std::shared_ptr<N> node_for(const Tensor& input) {
    std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(input));
    return node;
}

// These gradients have no gradient of their own: where one could be asked for, asking raises an error.
Tensor once_differentiable(Tensor g, bool wanted) {
    if (!wanted) return g;
    torch::autograd::DelayedError refuse("trying to differentiate twice a function that was marked with @once_differentiable", 1);
    return refuse.apply({g.detach().set_requires_grad(true)})[0];
}

// ------------------------------------------------------------------------------------------------------- embedding
// order: where it is given and the sizes are such, it becomes the sorted list for the gradient.
Tensor embedding_forward(const Tensor& tokens, const Tensor& weight, double scale, int64_t padding, Tensor* order) {
    at::NoGradGuard no_grad;
    Place on(weight);
    const Rows w(weight);
    const Tensor ids = tokens.contiguous();
    Tensor out = at::empty(with_last(tokens.sizes(), w.width), w.t.options());
    if (ids.numel() == 0) return out;
    if (order != nullptr)
        if (const size_t bytes = lib.embedding_order_bytes(ids.numel(), w.n, (int)w.width, type_code(w.t)))
            *order = at::empty({(int64_t)bytes}, w.t.options().dtype(at::kByte));
    check(lib.embedding_fwd(ids.const_data_ptr(), wide(ids), ids.numel(), w.t.const_data_ptr(), w.ld, w.n, (int)w.width, type_code(w.t),
                            (float)scale, out.mutable_data_ptr(), order != nullptr && order->defined() ? order->mutable_data_ptr() : nullptr,
                            padding, lib.status, on.stream),
          "embedding_fwd");
    count(kEmbeddingFwd);
    return out;
}

Tensor embedding_gradient(const Tensor& dy, const Tensor& tokens, int64_t vocab, double scale, int64_t padding, const Tensor& order) {
    at::NoGradGuard no_grad;
    Place on(dy);
    const Rows g(dy);
    const Tensor ids = tokens.contiguous();
    const int code = type_code(dy);
    Tensor dw = at::empty({vocab, g.width}, dy.options()), work;
    const size_t bytes = lib.embedding_grad_bytes(g.n, vocab, (int)g.width, code);
    if (bytes) work = at::empty({(int64_t)bytes}, dy.options().dtype(at::kByte));
    check(lib.embedding_grad(g.t.const_data_ptr(), g.ld, ids.const_data_ptr(), wide(ids), g.n, vocab, (int)g.width, code, (float)scale,
                             padding, order.defined() ? order.const_data_ptr() : nullptr, dw.mutable_data_ptr(), bytes ? work.mutable_data_ptr() : nullptr, bytes, lib.status, on.stream),
          "embedding_grad");
    count(kEmbeddingGrad);
    return dw;
}

std::optional<Tensor> embedding_grad(const Tensor& dy, const Tensor& tokens, int64_t vocab, double scale, int64_t padding) {
    if (!fits_rows(dy, tokens) || vocab < 1 || vocab > 0x7ffffffeLL) return std::nullopt;
    return embedding_gradient(dy, tokens, vocab, scale, padding, Tensor());
}

struct EmbeddingBackward : Node {
    SavedVariable tokens;
    Tensor order;
    int64_t vocab = 0, padding = -1;
    double scale = 1.0;

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const Tensor& dy = grads[0];
        if (!dy.defined()) return {Tensor()};
        return {once_differentiable(embedding_gradient(dy, tokens.unpack(), vocab, scale, padding, order), differentiable(dy))};
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        tokens.reset_data();
        order.reset();
    }
    std::string name() const override { return "EmbeddingBackward"; }
};

std::optional<Tensor> embedding(const Tensor& tokens, const Tensor& weight, double scale, int64_t padding) {
    if (!fits(weight, tokens) || weight.dim() != 2 || weight.size(0) < 1 || weight.size(0) > 0x7ffffffeLL) return std::nullopt;
    const bool train = differentiable(weight);
    Tensor order, out = embedding_forward(tokens, weight, scale, padding, train ? &order : nullptr);
    if (train) {
        auto node = node_for<EmbeddingBackward>(weight);
        node->tokens = SavedVariable(tokens, false);
        node->order = order;
        node->vocab = weight.size(0);
        node->padding = padding;
        node->scale = scale;
        torch::autograd::set_history(out, node);
    }
    return out;
}

// --------------------------------------------------------------------------- log probabilities, entropy, alternatives
// Gradient matrix for `z`.  Rows keep the distance of a padded output layer (up to an eighth wider than the vocabulary), so
// that rows of logits and gradient start at the same place of a 16-byte block.
Tensor grad_like(const Rows& z) {
    if (z.width < z.ld && z.ld <= z.width + z.width / 8) return at::empty({z.n, z.ld}, z.t.options()).narrow(1, 0, z.width);
    return at::empty({z.n, z.width}, z.t.options());
}

int64_t row_distance(const Tensor& dz) { return dz.size(0) > 1 ? dz.stride(0) : dz.size(1); }

Tensor in_shape_of(const Tensor& dz, const Tensor& logits) { return logits.dim() == 2 ? dz : dz.view(logits.sizes()); }

struct TokenLogProbsBackward : Node {
    SavedVariable logits, tokens, entropy;
    Tensor stats;
    int64_t ignore = 0;

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined() && !grads[1].defined()) return {Tensor()};
        const Tensor x = logits.unpack(), chosen = tokens.unpack(), h = entropy.unpack();
        const bool twice = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        Place on(x);
        const Rows z(x);
        const Tensor ids = chosen.contiguous();
        const Tensor g1 = grads[0].defined() ? grads[0].contiguous() : Tensor(), g2 = grads[1].defined() ? grads[1].contiguous() : Tensor();
        Tensor dz = grad_like(z);
        if (z.n) {
            check(lib.logprob_bwd(z.t.const_data_ptr(), z.ld, z.n, (int)z.width, type_code(z.t), ids.const_data_ptr(), wide(ids), ignore,
                                  const_floats(stats), const_floats(h), const_floats(g1), const_floats(g2), nullptr, nullptr, 0, 0.f,
                                  dz.mutable_data_ptr(), row_distance(dz), on.stream),
                  "logprob_bwd");
            count(kLogprobBwd);
        }
        return {once_differentiable(in_shape_of(dz, x), twice)};
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        logits.reset_data();
        tokens.reset_data();
        entropy.reset_data();
        stats.reset();
    }
    std::string name() const override { return "TokenLogProbsBackward"; }
};

typedef std::tuple<Tensor, Tensor, std::optional<Tensor>, std::optional<Tensor>> LogProbs;

std::optional<LogProbs> token_log_probs(const Tensor& logits, const Tensor& tokens, int64_t ignore, int64_t top) {
    if (!fits_rows(logits, tokens) || top < 0 || top > std::min<int64_t>(32, logits.size(-1))) return std::nullopt;
    const bool train = differentiable(logits);
    Tensor logprob, h, stats;
    std::optional<Tensor> best, which;
    {
        at::NoGradGuard no_grad;
        Place on(logits);
        const Rows z(logits);
        const Tensor ids = tokens.contiguous();
        const auto f32 = z.t.options().dtype(at::kFloat);
        logprob = at::empty(tokens.sizes(), f32);
        h = at::empty(tokens.sizes(), f32);
        if (train) stats = at::empty({z.n, 2}, f32);
        if (top) {
            best = at::empty(with_last(tokens.sizes(), top), f32);
            which = at::empty(with_last(tokens.sizes(), top), f32.dtype(at::kLong));
        }
        if (z.n) {
            check(lib.logprob_fwd(z.t.const_data_ptr(), z.ld, z.n, (int)z.width, type_code(z.t), ids.const_data_ptr(), wide(ids), ignore,
                                  floats(logprob), floats(h), floats(stats), (int)top, top ? floats(*best) : nullptr,
                                  top ? reinterpret_cast<long long*>(which->mutable_data_ptr<int64_t>()) : nullptr, lib.status, on.stream),
                  "logprob_fwd");
            count(kLogprobFwd);
        }
    }
    if (train) {
        auto node = node_for<TokenLogProbsBackward>(logits);
        node->logits = SavedVariable(logits, false);
        node->tokens = SavedVariable(tokens, false);
        node->entropy = SavedVariable(h.detach(), false);        // an alias: the node must not own its own output
        node->stats = stats;
        node->ignore = ignore;
        torch::autograd::set_history({logprob, h}, node);
    }
    return LogProbs(logprob, h, best, which);
}

// --------------------------------------------------------------------------------------------------- cross entropy
// The forward launch has written the gradient of the logits for the gradient that the loss is expected to get.  The first
// backward pass hands it out (its launch looks at the actual gradient and recomputes the rows only where that differs); any
// further one computes its own.
struct CrossEntropyBackward : Node {
    SavedVariable logits, tokens;
    Tensor work, written;
    int64_t ignore = 0;
    double expected = 1.0;

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined()) return {Tensor()};
        const Tensor x = logits.unpack(), chosen = tokens.unpack();
        const bool twice = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        Place on(x);
        const Rows z(x);
        const Tensor ids = chosen.contiguous(), g = grads[0].contiguous();
        Tensor dz = std::move(written);
        written.reset();
        const bool have = dz.defined();
        if (!have) dz = grad_like(z);
        if (z.n) {
            check(lib.logprob_bwd(z.t.const_data_ptr(), z.ld, z.n, (int)z.width, type_code(z.t), ids.const_data_ptr(), wide(ids), ignore,
                                  const_floats(work) + 2, nullptr, nullptr, nullptr, const_floats(g),
                                  reinterpret_cast<const int*>(const_floats(work)), have, (float)expected, dz.mutable_data_ptr(),
                                  row_distance(dz), on.stream),
                  "cross_entropy_bwd");
            count(kCrossEntropyBwd);
        }
        return {once_differentiable(in_shape_of(dz, x), twice)};
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        logits.reset_data();
        tokens.reset_data();
        work.reset();
        written.reset();
    }
    std::string name() const override { return "CrossEntropyBackward"; }
};

std::optional<Tensor> cross_entropy(const Tensor& logits, const Tensor& tokens, int64_t ignore, bool mean, double expected) {
    if (!fits_rows(logits, tokens)) return std::nullopt;
    const bool train = differentiable(logits);
    Tensor loss, work, dz;
    {
        at::NoGradGuard no_grad;
        Place on(logits);
        const Rows z(logits);
        const Tensor ids = tokens.contiguous();
        const auto f32 = z.t.options().dtype(at::kFloat);
        loss = at::empty({}, f32);
        // two words (the number of rows in the mean, a counter), {m, log2 s} of every row, log probability of every row
        work = at::empty({2 + 3 * z.n}, f32);
        if (train) dz = grad_like(z);
        float* at = floats(work);
        check(lib.cross_entropy_fwd(z.t.const_data_ptr(), z.ld, z.n, (int)z.width, type_code(z.t), ids.const_data_ptr(), wide(ids), ignore,
                                    mean, (float)expected, at + 2 + 2 * z.n, train ? at + 2 : nullptr, floats(loss),
                                    train ? dz.mutable_data_ptr() : nullptr, train ? row_distance(dz) : z.width, reinterpret_cast<int*>(at),
                                    lib.status, on.stream),
              "cross_entropy_fwd");
        count(kCrossEntropyFwd);
    }
    if (train) {
        auto node = node_for<CrossEntropyBackward>(logits);
        node->logits = SavedVariable(logits, false);
        node->tokens = SavedVariable(tokens, false);
        node->work = work;
        node->written = dz;
        node->ignore = ignore;
        node->expected = expected;
        torch::autograd::set_history(loss, node);
    }
    return loss;
}

// ------------------------------------------------------------------------------------------------------------- clip
// Whether the kernels take these gradients: on one GPU, of their types, the elements of each one stretch of memory.
bool clip_supported(const std::vector<Tensor>& grads) {
    for (const Tensor& g : grads)
        if (!g.is_cuda() || g.layout() != at::kStrided || type_code(g) < 0 || g.device() != grads[0].device() ||
            !g.is_non_overlapping_and_dense())
            return false;
    return !grads.empty();
}

// The norm, and with `clip` the scaling in place, of the gradients `list` (or of its tensors' gradients); nothing where the
// kernels do not take them.
std::optional<Tensor> clip_grads(const std::vector<Tensor>& list, bool parameters, int norm, double scale, double max_norm, bool clip) {
    std::vector<Tensor> own;
    if (parameters) {
        own.reserve(list.size());
        for (const Tensor& p : list)
            if (const Tensor& g = p.grad(); g.defined()) own.push_back(g);
    }
    const std::vector<Tensor>& grads = parameters ? own : list;
    if (!clip_supported(grads)) return std::nullopt;
    TORCH_CHECK(lib.status != nullptr, "the kernels' library is not bound");
    at::NoGradGuard no_grad;
    const Tensor& first = grads[0];
    const int n = (int)grads.size();
    std::vector<unsigned long long> address(n);
    std::vector<long long> numel(n);
    std::vector<unsigned char> code(n);
    for (int i = 0; i < n; ++i) {
        address[i] = (unsigned long long)(uintptr_t)(clip ? grads[i].mutable_data_ptr() : const_cast<void*>(grads[i].const_data_ptr()));
        numel[i] = grads[i].numel();
        code[i] = (unsigned char)type_code(grads[i]);
    }
    Place on(first);
    Tensor out = at::empty({}, first.options().dtype(at::kFloat));
    const size_t bytes = lib.grad_clip_bytes(n);
    Tensor work = at::empty({(int64_t)bytes}, first.options().dtype(at::kByte));
    const int rc = lib.grad_clip(address.data(), numel.data(), code.data(), n, norm, scale, max_norm, clip, work.mutable_data_ptr(), bytes,
                                 floats(out), on.stream);
    if (rc == kBadArgument) throw py::value_error(std::string("grad_clip: ") + lib.last_error());
    check(rc, "grad_clip");
    if (clip)
        for (const Tensor& g : grads)
            if (!g.is_inference()) g.unsafeGetTensorImpl()->bump_version();          // changed in place
    const long long tables = (n + 1023) / 1024;
    count(kGradNorm, tables);
    count(clip ? kGradScale : kGradNormFinish, clip ? tables : 1);
    return out;
}

// ------------------------------------------------------------------------------------------------------------- module
template <typename F>
void take(F& f, const py::dict& addresses, const char* name) {
    f = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}

PyObject* error_class = PyExc_RuntimeError;                     // kept for the life of the process

void bind(const py::dict& addresses, uintptr_t status, const py::object& error) {
    take(lib.last_error, addresses, "mgw_last_error");
    take(lib.embedding_order_bytes, addresses, "mgw_embedding_order_bytes");
    take(lib.embedding_fwd, addresses, "mgw_embedding_fwd");
    take(lib.embedding_grad_bytes, addresses, "mgw_embedding_grad_bytes");
    take(lib.embedding_grad, addresses, "mgw_embedding_grad");
    take(lib.logprob_fwd, addresses, "mgw_logprob_fwd");
    take(lib.logprob_bwd, addresses, "mgw_logprob_bwd");
    take(lib.cross_entropy_fwd, addresses, "mgw_cross_entropy_fwd");
    take(lib.grad_clip_bytes, addresses, "mgw_grad_clip_bytes");
    take(lib.grad_clip, addresses, "mgw_grad_clip");
    lib.status = reinterpret_cast<int*>(status);
    error_class = py::object(error).release().ptr();
}

std::unordered_map<std::string, long long> launch_counts() {
    std::unordered_map<std::string, long long> out;
    for (int i = 0; i < kLaunches; ++i)
        if (const long long n = launches[i].load(std::memory_order_relaxed)) out[kNames[i]] = n;
    return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    using free_interpreter = py::call_guard<py::gil_scoped_release>;
    py::register_local_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const NativeError& e) {
            PyErr_SetString(error_class, e.what());
        }
    });
    m.attr("torch_version") = MGW_TORCH_VERSION;
    m.def("bind", &bind);
    m.def("launch_counts", &launch_counts);
    m.def("embedding", &embedding, free_interpreter());
    m.def("embedding_grad", &embedding_grad, free_interpreter());
    m.def("token_log_probs", &token_log_probs, free_interpreter());
    m.def("cross_entropy", &cross_entropy, free_interpreter());
    m.def("clip_supported", &clip_supported, free_interpreter());
    m.def("clip_grads", &clip_grads, free_interpreter());
}
