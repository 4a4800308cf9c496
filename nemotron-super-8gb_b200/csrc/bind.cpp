// The operators of dense_q's four-bit part and of router as functions of torch tensors, over the C entry points: argument
// checks, outputs from torch's allocator, the current stream, and automatic differentiation.
//
// Small calls are bound by the host. The same calls by ctypes, with a torch.autograd.Function, took 113 us for a loss of
// 200 tokens and its gradient (59 here, of which torch's engine is about 45), 11 us for one token's linear (6.2), 24 us for
// quantising a token and reading it back (14).
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/zeros.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/qmoe_b200.h"

#include <optional>
#include <sstream>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

struct Refused : std::runtime_error { using std::runtime_error::runtime_error; };

template <typename... A> [[noreturn]] void refuse(const A &...a) {
    std::ostringstream s;
    (s << ... << a);
    throw Refused(s.str());
}

#define REQUIRE(cond, ...) \
    do {                   \
        if (!(cond)) refuse(__VA_ARGS__); \
    } while (0)

void status(int code, const char *name) {
    REQUIRE(code == QMOE_OK, name, ": ", qmoe_status_string(code), " (status ", code, ")");
}

int dtype_code(at::ScalarType t) {
    switch (t) {
    case at::kFloat: return QMOE_DT_F32;
    case at::kBFloat16: return QMOE_DT_BF16;
    case at::kHalf: return QMOE_DT_F16;
    default: return -1;
    }
}

int activation(const Tensor &x) {
    REQUIRE(x.is_cuda(), "libqmoe_b200 works on CUDA tensors only (got a CPU tensor)");
    const int dt = dtype_code(x.scalar_type());
    REQUIRE(dt >= 0, "unsupported activation dtype ", x.scalar_type());
    return dt;
}

void *stream_of(const Tensor &x) { return c10::cuda::getCurrentCUDAStream(x.get_device()).stream(); }

// From torch's allocator, without the way through the dispatcher (0.3 us each: quantising a row, which takes three, 6.7 us instead of 7.7).
Tensor empty(at::IntArrayRef sizes, const Tensor &like, at::ScalarType t) { return at::detail::empty_cuda(sizes, t, like.device(), std::nullopt); }

// A matrix as the kernels read it: unit column stride, rows that do not overlap; its row stride.
Tensor rows_of(const Tensor &x, int64_t &ld) {
    const int64_t M = x.size(0), K = x.size(1);
    Tensor r = x.is_contiguous() || (x.stride(1) == 1 && (M <= 1 || x.stride(0) >= K)) ? x : x.contiguous();
    ld = M > 1 ? r.stride(0) : K;
    return r;
}

template <typename T = void> T *data(const OptTensor &t) { return t.has_value() && t->defined() ? static_cast<T *>(t->data_ptr()) : nullptr; }
template <typename T = void> T *data(const Tensor &t) { return static_cast<T *>(t.data_ptr()); }

// ------------------------------------------------------------------------------------------ four bits
// A forward-mode tangent, which torch carries on under no_grad too, would be lost.
void no_tangent(const Tensor &t, const char *who) { REQUIRE(!torch::autograd::isFwGradDefined(t), who, " operators have no forward-mode derivative"); }

void no_grad(const Tensor &t) {
    no_tangent(t, "the four-bit");
    REQUIRE(!(t.requires_grad() && at::GradMode::is_enabled()), "the four-bit operators have no gradient: call them under torch.no_grad()");
}

// The tensors of a quantised matrix [N, K], as the kernels read them.
void check_tensors(const Tensor &w, const Tensor &sc, const Tensor &s, bool per_row, int64_t N, int64_t K) {
    for (auto [name, t, width] : {std::make_tuple("w", &w, K / 2), std::make_tuple("sc", &sc, K / 16)})
        REQUIRE(t->scalar_type() == at::kByte && t->dim() == 2 && t->size(0) == N && t->size(1) == width && t->is_contiguous(),
                name, " must be contiguous uint8 [", N, ", ", width, "]");
    REQUIRE(s.scalar_type() == at::kFloat && s.numel() == (per_row ? N : 1) && s.is_contiguous(),
            "s must be float32, one value (nvfp4) or one per row (nvfp4_rows)");
}
void check_device(const Tensor &w, const Tensor &sc, const Tensor &s) {
    REQUIRE(w.is_cuda() && sc.device() == w.device() && s.device() == w.device(), "libqmoe_b200 works on CUDA tensors only, all of a weight on one device");
}

// The same for the inverse, which takes the bytes in any one-byte type and shape.
void check_stored(const Tensor &w, const Tensor &sc, const Tensor &s, bool per_row, int64_t N, int64_t K) {
    REQUIRE(N >= 0 && K >= 16 && K % 16 == 0, "a quantised matrix has rows of a positive multiple of 16 elements (got ", N, " x ", K, ")");
    for (auto [name, t, bytes] : {std::make_tuple("w", &w, N * (K / 2)), std::make_tuple("sc", &sc, N * (K / 16))})
        REQUIRE(t->element_size() == 1 && t->numel() == bytes && t->is_contiguous(), name, " must be ", bytes, " contiguous bytes for ", N, " rows of ", K, " elements");
    REQUIRE(s.scalar_type() == at::kFloat && s.numel() == (per_row ? N : 1) && s.is_contiguous(),
            "s must be float32, one value (nvfp4) or one per row (nvfp4_rows)");
    check_device(w, sc, s);
}

int64_t atoms_bytes(int64_t rows, int64_t K) { return (rows + 127) / 128 * ((K + 63) / 64) * 512; }

// A quantised matrix as a product's operand: its tensors, and its scale atoms where it has them.
void check_operand(const Tensor &w, const Tensor &sc, const OptTensor &atoms, const Tensor &s, bool per_row, int64_t N, int64_t K) {
    check_tensors(w, sc, s, per_row, N, K);
    REQUIRE(!atoms || (atoms->scalar_type() == at::kByte && atoms->numel() == atoms_bytes(N, K) && atoms->is_contiguous() && atoms->device() == w.device()),
            "sca must be the ", atoms_bytes(N, K), " bytes that prepare makes of this weight's scales, on its device");
}

Tensor scale_atoms(const Tensor &w, const Tensor &sc, const Tensor &s, bool per_row, int64_t N, int64_t K) {
    check_tensors(w, sc, s, per_row, N, K);
    check_device(w, sc, s);
    const c10::cuda::CUDAGuard guard(sc.device());
    const Tensor atoms = empty({atoms_bytes(N, K)}, sc, at::kByte);
    if (N) status(dq_scale_atoms(data<uint8_t>(sc), N, K, data<uint8_t>(atoms), stream_of(sc)), "dq_scale_atoms");
    return atoms;
}

py::tuple quantize(const Tensor &x0, bool per_row, bool for_gemm) {
    REQUIRE(x0.dim() == 2, "quantize takes a matrix [M, K]");
    const int64_t M = x0.size(0), K = x0.size(1);
    REQUIRE(K >= 16 && K % 16 == 0, "quantize takes rows of a positive multiple of 16 elements (got ", K, ")");
    REQUIRE(M > 0 || per_row, "a tensor without rows has no scale");
    no_grad(x0);
    const int dt = activation(x0);
    int64_t ld;
    const Tensor x = rows_of(x0, ld);
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor w = empty({M, K / 2}, x, at::kByte), sc = empty({M, K / 16}, x, at::kByte), s = empty({per_row ? M : 1}, x, at::kFloat);
    OptTensor atoms;
    if (for_gemm) atoms = empty({atoms_bytes(M, K)}, x, at::kByte);
    if (M)
        status(dq_quantize_nvfp4(data(x), dt, ld, M, K, per_row, data<uint8_t>(w), data<uint8_t>(sc), data<float>(s), data<uint8_t>(atoms),
                                 stream_of(x)), "dq_quantize_nvfp4");
    return py::make_tuple(w, sc, s, atoms);
}

Tensor dequant(const Tensor &w, const Tensor &sc, const Tensor &s, bool per_row, int64_t N, int64_t K) {
    check_stored(w, sc, s, per_row, N, K);
    const c10::cuda::CUDAGuard guard(w.device());
    const Tensor out = empty({N, K}, w, at::kBFloat16);
    if (N && per_row) status(dq_dequant_nvfp4(data<uint8_t>(w), data<uint8_t>(sc), data<float>(s), 1, N, K, 0, N, data(out), QMOE_DT_BF16, stream_of(w)), "dq_dequant_nvfp4");
    else if (N) status(dq_dequant_rows(1, data<uint8_t>(w), data<uint8_t>(sc), data<float>(s), N, K, 0, N, data(out), QMOE_DT_BF16, stream_of(w)), "dq_dequant_rows");
    return out;
}

// The epilogue's code, and the residual as the kernels read it.
int epilogue(const std::optional<std::string> &act, OptTensor &residual, int64_t M, int64_t N, at::ScalarType dtype, at::Device dev) {
    REQUIRE(!act || *act == "relu2", "gemm: act is None or 'relu2', and not together with a residual");
    if (!residual) return act ? 1 : 0;
    REQUIRE(!act, "gemm: act is None or 'relu2', and not together with a residual");
    no_grad(*residual);
    REQUIRE(residual->dim() == 2 && residual->size(0) == M && residual->size(1) == N && residual->scalar_type() == dtype && residual->device() == dev,
            "gemm: the residual is [M, N] in the output's dtype, on its device");
    residual = residual->contiguous();
    return 2;
}

void check_weight(const Tensor &w, int64_t N, int64_t Kw, int64_t K, at::Device dev) {
    REQUIRE(Kw == K, "gemm: ", K, " elements per activation row, ", Kw, " per weight row");
    REQUIRE(K > 0 && K % 32 == 0, "gemm takes rows of a positive multiple of 32 elements (got ", K, ")");
    REQUIRE(w.device() == dev, "gemm: weight on ", w.device(), ", activations on ", dev);
    REQUIRE(N <= (1 << 24), "gemm: at most 2^24 weight rows");
}

Tensor gemm(const Tensor &w, const Tensor &wsc, OptTensor watoms, const Tensor &ws, bool w_rows, int64_t N, int64_t Kw, const Tensor &x, const Tensor &xsc,
            OptTensor xatoms, const Tensor &xs, bool x_rows, int64_t M, int64_t K, at::ScalarType dtype, const std::optional<std::string> &act, OptTensor residual) {
    REQUIRE(dtype_code(dtype) >= 0, "unsupported output dtype ", dtype);
    check_weight(w, N, Kw, K, x.device());
    const int ep = epilogue(act, residual, M, N, dtype, x.device());
    check_operand(w, wsc, watoms, ws, w_rows, N, K);
    check_operand(x, xsc, xatoms, xs, x_rows, M, K);
    check_device(w, wsc, ws);
    check_device(x, xsc, xs);
    REQUIRE(M <= (1 << 24), "gemm: at most 2^24 rows");
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor y = empty({M, N}, x, dtype);
    if (M && N) {
        if (!watoms) watoms = scale_atoms(w, wsc, ws, w_rows, N, K);
        if (!xatoms) xatoms = scale_atoms(x, xsc, xs, x_rows, M, K);
        status(dq_gemm_nvfp4(data<uint8_t>(w), data<uint8_t>(watoms), data<float>(ws), w_rows, data<uint8_t>(x), data<uint8_t>(xatoms), data<float>(xs),
                             x_rows, (int)M, (int)N, (int)K, ep, data(residual), data(y), dtype_code(dtype), stream_of(x)), "dq_gemm_nvfp4");
    }
    return y;
}

Tensor linear_a4(const Tensor &w, const Tensor &sc, OptTensor atoms, const Tensor &s, bool w_rows, int64_t N, int64_t Kw, const Tensor &x0,
                 const std::optional<std::string> &act, OptTensor residual) {
    REQUIRE(x0.dim() >= 1, "a linear takes rows [..., K]");
    const int64_t K = x0.size(-1);
    no_grad(x0);
    const int dt = activation(x0);
    int64_t ld;
    const Tensor x = rows_of(x0.dim() == 2 ? x0 : x0.reshape({K ? x0.numel() / K : 0, K}), ld);
    const int64_t M = x.size(0);
    check_weight(w, N, Kw, K, x.device());
    check_operand(w, sc, atoms, s, w_rows, N, K);
    check_device(w, sc, s);
    std::vector<int64_t> shape = x0.sizes().vec();
    shape.back() = N;
    if (residual) {
        REQUIRE(residual->sizes() == shape, "gemm: the residual has the output's shape ", at::IntArrayRef(shape), " (got ", residual->sizes(), ")");
        residual = residual->reshape({M, N});
    }
    const int ep = epilogue(act, residual, M, N, x.scalar_type(), x.device());
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor y = empty(shape, x, x.scalar_type());
    if (M && N) {
        REQUIRE(M <= (1 << 24), "gemm: at most 2^24 rows");
        OptTensor ws;
        size_t n = 0;
        if (M > 4 || K > 16384) {   // few rows need neither
            if (!atoms) atoms = scale_atoms(w, sc, s, w_rows, N, K);
            n = dq_linear_a4_workspace_bytes(M, K);
            ws = empty({(int64_t)n}, x, at::kByte);
        }
        status(dq_linear_a4(data<uint8_t>(w), data<uint8_t>(sc), data<uint8_t>(atoms), data<float>(s), w_rows, data(x), dt, ld, (int)M, (int)N, (int)K, ep,
                            data(residual), data(y), data(ws), n, stream_of(x)), "dq_linear_a4");
    }
    return y;
}

// ------------------------------------------------------------------------------------------ router
int score_code(const std::string &score) {
    REQUIRE(score == "sigmoid" || score == "softmax", "score is 'sigmoid' or 'softmax' (got '", score, "')");
    return score == "softmax";
}

int check_logits(const Tensor &x) {
    REQUIRE(x.dim() == 2 && x.size(1) >= 1 && x.size(1) <= 1024, "logits must be [T, E] with 1 <= E <= 1024 (got ", x.sizes(), ")");
    return activation(x);
}

// A gradient that was asked for as part of a graph: a second differentiation through it is refused.
Tensor once(const Tensor &g) {
    if (!at::GradMode::is_enabled()) return g;
    Tensor v = g.detach();
    v.requires_grad_(true);
    auto f = std::make_shared<torch::autograd::DelayedError>("the router's operators are differentiable once", 1);
    return (*f)({v})[0];
}

struct RouteArgs { int64_t k, n_group, topk_group; bool norm; int score; double scaling; };

std::tuple<Tensor, Tensor, Tensor> run_route(const Tensor &x0, const OptTensor &bias, const RouteArgs &a) {
    const at::AutoGradMode off(false);
    int64_t ld;
    const Tensor x = rows_of(x0, ld);
    const int64_t T = x.size(0), E = x.size(1);
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor ids = empty({T, a.k}, x, at::kLong), w = empty({T, a.k}, x, at::kFloat);
    const Tensor n = T ? empty({E}, x, at::kInt) : at::zeros({E}, x.options().dtype(at::kInt).requires_grad(false));
    if (T)
        status(qmoe_route(data(x), dtype_code(x.scalar_type()), ld, data<float>(bias), T, (int)E, (int)a.k, (int)a.n_group, (int)a.topk_group, a.norm, a.score,
                          (float)a.scaling, data<int64_t>(ids), data<float>(w), data<int32_t>(n), stream_of(x)), "qmoe_route");
    return {ids, w, n};
}

// The operators' gradients as nodes of torch's graph. (torch::autograd::Function, which converts every argument, took 62 us
// for the loss of 200 tokens and its gradient; this 58.)
struct Gradient : torch::autograd::Node {
    torch::autograd::SavedVariable logits;
    int score;
    Gradient(const Tensor &x, int score) : Node(torch::autograd::collect_next_edges(x)), logits(x, false), score(score) {}
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        logits.reset_data();
    }
    // d logits of the output's gradient g
    virtual Tensor gradient(const Tensor &x, int64_t ld, const Tensor &g) = 0;
    torch::autograd::variable_list apply(torch::autograd::variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined()) return {Tensor()};
        Tensor dl;
        {
            const at::AutoGradMode off(false);
            const Tensor saved = logits.unpack();
            int64_t ld;
            const Tensor x = rows_of(saved, ld);
            const c10::cuda::CUDAGuard guard(x.device());
            dl = gradient(x, ld, grads[0].scalar_type() == at::kFloat ? grads[0] : grads[0].to(at::kFloat));
        }
        return {once(dl)};
    }
};

// `out` becomes the output whose gradient the node takes.
void attach(const Tensor &out, std::shared_ptr<torch::autograd::Node> node) { torch::autograd::set_history(out, node); }

bool differentiated(const Tensor &x) {
    no_tangent(x, "the router's");
    return at::GradMode::is_enabled() && x.requires_grad();
}

struct RouteBackward : Gradient {
    torch::autograd::SavedVariable ids;
    bool norm;
    double scaling;
    RouteBackward(const Tensor &x, const Tensor &ids, const RouteArgs &a) : Gradient(x, a.score), ids(ids, false), norm(a.norm), scaling(a.scaling) {}
    std::string name() const override { return "RouteBackward"; }
    void release_variables() override {
        Gradient::release_variables();
        std::lock_guard<std::mutex> lock(mutex_);
        ids.reset_data();
    }
    Tensor gradient(const Tensor &x, int64_t ld, const Tensor &g) override {
        const Tensor dl = empty(x.sizes(), x, x.scalar_type()), i = ids.unpack(), dw = g.contiguous();
        if (x.size(0))
            status(qmoe_route_backward(data(x), dtype_code(x.scalar_type()), ld, x.size(0), (int)x.size(1), (int)i.size(1), norm, score, (float)scaling,
                                       data<int64_t>(i), data<float>(dw), data(dl), stream_of(x)), "qmoe_route_backward");
        return dl;
    }
};

py::tuple route(const Tensor &logits, OptTensor bias, int64_t top_k, double scaling, int64_t n_group, int64_t topk_group, bool norm, const std::string &score) {
    const int sc = score_code(score);
    check_logits(logits);
    const int64_t E = logits.size(1);
    REQUIRE(top_k >= 1 && top_k <= std::min<int64_t>(32, E), "top_k must lie in 1..", std::min<int64_t>(32, E), " (got ", top_k, ")");
    REQUIRE(n_group >= 1 && n_group <= 32 && E % n_group == 0 && topk_group >= 1 && topk_group <= n_group && (n_group == 1 || E / n_group >= 2),
            E, " experts do not split into ", n_group, " groups of two or more, ", topk_group, " of them kept");
    REQUIRE(sc == 0 || top_k <= E / n_group * topk_group, "a softmax router leaves ", E / n_group * topk_group, " experts in ", topk_group, " groups, top_k is ", top_k);
    if (bias) {
        REQUIRE(sc == 0, "a softmax router takes no bias");
        REQUIRE(bias->dim() == 1 && bias->size(0) == E && bias->device() == logits.device(), "bias must be [E], on the logits' device");
        bias = bias->detach().to(at::kFloat).contiguous();
    }
    const RouteArgs args{top_k, n_group, topk_group, norm, sc, scaling};
    auto [ids, w, n] = run_route(logits, bias, args);
    if (differentiated(logits)) attach(w, std::shared_ptr<RouteBackward>(new RouteBackward(logits, ids, args), torch::autograd::deleteNode));
    return py::make_tuple(ids, w, n);
}

// Loss, counts, and a buffer that begins with coef * f / T' per expert, for the backward pass; the rest of it, 0.6 MB for
// 512 experts and 1.3 for 1024, is the call's workspace (an allocation of its own costs more than a microsecond).
std::tuple<Tensor, Tensor, Tensor> run_balance(const Tensor &x0, const Tensor &ids, const OptTensor &mask, int score, double coef) {
    const at::AutoGradMode off(false);
    int64_t ld;
    const Tensor x = rows_of(x0, ld);
    const int64_t T = x.size(0), E = x.size(1);
    const c10::cuda::CUDAGuard guard(x.device());
    if (!T) {
        const auto f = x.options().dtype(at::kFloat).requires_grad(false);
        return {at::zeros({}, f), at::zeros({E}, f.dtype(at::kInt)), at::zeros({E}, f)};
    }
    const size_t bytes = qmoe_balance_workspace_bytes(T, (int)E);
    const Tensor loss = empty({}, x, at::kFloat), n = empty({E}, x, at::kInt), c = empty({E + (int64_t)(bytes / 4)}, x, at::kFloat);
    status(qmoe_balance(data(x), dtype_code(x.scalar_type()), ld, data(ids), ids.scalar_type() == at::kLong, data<uint8_t>(mask), T, (int)E,
                        (int)ids.size(1), score, (float)coef, data<float>(loss), data<int32_t>(n), data<float>(c), data<float>(c) + E, bytes, stream_of(x)), "qmoe_balance");
    return {loss, n, c};
}

struct BalanceBackward : Gradient {
    torch::autograd::SavedVariable c, mask;
    BalanceBackward(const Tensor &x, const Tensor &c, const OptTensor &mask, int score) : Gradient(x, score), c(c, false), mask(mask ? *mask : Tensor(), false) {}
    std::string name() const override { return "BalanceBackward"; }
    void release_variables() override {
        Gradient::release_variables();
        std::lock_guard<std::mutex> lock(mutex_);
        c.reset_data();
        mask.reset_data();
    }
    Tensor gradient(const Tensor &x, int64_t ld, const Tensor &g) override {
        const Tensor dl = empty(x.sizes(), x, x.scalar_type()), m = mask.unpack();
        if (x.size(0))
            status(qmoe_balance_backward(data(x), dtype_code(x.scalar_type()), ld, m.defined() ? data<uint8_t>(m) : nullptr, x.size(0), (int)x.size(1), score,
                                         data<float>(c.unpack()), data<float>(g), data(dl), stream_of(x)), "qmoe_balance_backward");
        return dl;
    }
};

py::tuple balance_loss(const Tensor &logits, const Tensor &ids0, OptTensor mask, const std::string &score, double coef) {
    const int sc = score_code(score);
    check_logits(logits);
    const int64_t T = logits.size(0);
    REQUIRE(ids0.dim() == 2 && ids0.size(0) == T && ids0.size(1) >= 1 && (ids0.scalar_type() == at::kLong || ids0.scalar_type() == at::kInt),
            "ids must be int64 or int32 [T, k] with k >= 1");
    REQUIRE(ids0.device() == logits.device(), "ids must be on the logits' device");
    REQUIRE(T * ids0.size(1) <= INT32_MAX, "counts are int32: at most 2^31 - 1 ids (got ", T * ids0.size(1), ")");
    const Tensor ids = ids0.contiguous();
    if (mask) {
        REQUIRE(mask->dim() == 1 && mask->size(0) == T && mask->scalar_type() == at::kBool && mask->device() == logits.device(),
                "mask must be bool [T], on the logits' device");
        mask = mask->contiguous();
    }
    auto [loss, n, c] = run_balance(logits, ids, mask, sc, coef);
    if (differentiated(logits)) attach(loss, std::shared_ptr<BalanceBackward>(new BalanceBackward(logits, c, mask, sc), torch::autograd::deleteNode));
    return py::make_tuple(loss, n);
}

py::object error_class, memory_class;

} // namespace

PYBIND11_MODULE(qmoe_torch, m) {
    m.def("set_error_classes", [](py::object c, py::object m) { error_class = std::move(c), memory_class = std::move(m); });
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Refused &e) {
            PyErr_SetString(error_class ? error_class.ptr() : PyExc_RuntimeError, e.what());
        } catch (const c10::OutOfMemoryError &e) {
            PyErr_SetString(memory_class ? memory_class.ptr() : PyExc_MemoryError, e.what_without_backtrace());
        }
    });
    m.def("quantize", &quantize);
    m.def("scale_atoms", &scale_atoms);
    m.def("check_stored", &check_stored);
    m.def("dequant", &dequant);
    m.def("gemm", &gemm);
    m.def("linear_a4", &linear_a4);
    m.def("route", &route);
    m.def("balance_loss", &balance_loss);
    m.add_object("_cleanup", py::capsule([] { error_class = memory_class = py::object(); }));
}
