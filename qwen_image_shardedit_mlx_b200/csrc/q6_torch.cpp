// Torch surface of the dense linear and the layer norm (dense.py): argument
// checks, layouts, output and workspace allocation, and the autograd nodes, in
// front of the C ABI of libq6b200.so.  Native because the calls are short: a
// 1 x 3072 norm takes the GPU 2.5 us, and a training step's backward nodes run on
// autograd's own threads, where a Python node costs more than its kernels (a
// 32 x 256 norm, forward and backward: 135 us from Python).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <tuple>

#include "q6_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A non-zero q6_status; becomes _lib.Q6Error in Python.
struct StatusError : std::exception {
    int status;
    std::string where, text;
    StatusError(int s, const char* w) : status(s), where(w) {
        text = where + ": q6 status " + std::to_string(s) + " (" + q6_status_string(s) + ")";
    }
    const char* what() const noexcept override { return text.c_str(); }
};

void check(int status, const char* where) {
    if (status != Q6_OK) throw StatusError(status, where);
}

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kBFloat16: return Q6_DTYPE_BF16;
        case at::kHalf: return Q6_DTYPE_F16;
        case at::kFloat: return Q6_DTYPE_F32;
        default: return -1;
    }
}

bool is_half(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }

const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mutable_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

Tensor of(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor optional_of(Tensor t) { return t.defined() ? OptTensor(std::move(t)) : std::nullopt; }

// `t` with its values as they lie in memory: a tensor may stand for the negative of
// what it stores (the imaginary part of a conjugate).
Tensor stored(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
Tensor contiguous(const Tensor& t) { return t.defined() ? stored(t).contiguous() : t; }

// `t` as rows of `width` with contiguous columns and the stride between rows (a
// copy only where the layout does not allow that).
struct Rows {
    Tensor t;
    int64_t ld = 0;
};

Rows rows_of(const Tensor& given, int64_t width) {
    const Tensor t = stored(given);
    if (!t.defined() || t.is_contiguous()) return {t, width};
    Tensor t2 = t.reshape({-1, width});
    const int64_t rows = t2.size(0);
    if ((width > 1 && t2.stride(1) != 1) || (rows > 1 && t2.stride(0) < width)) return {t2.contiguous(), width};
    return {t2, rows > 1 ? t2.stride(0) : width};
}

// Rows of x that share one vector of shape `v`: [width] or [1, width] (all rows),
// or [S, width] / [S, 1, ..., width] with S the leading size of x.
int64_t sample_rows(const char* name, at::IntArrayRef v, const Tensor& x, int64_t width) {
    const int64_t m = x.numel() / x.size(-1);
    if (v.size() == 1 && v[0] == width) return m;
    bool ok = v.size() >= 2 && v.back() == width;
    for (size_t i = 1; ok && i + 1 < v.size(); ++i) ok = v[i] == 1;
    TORCH_CHECK_VALUE(ok, name, " must be [", width, "] or [samples, ", width, "], got ", v);
    if (v[0] == 1) return m;
    TORCH_CHECK_VALUE(x.dim() >= 2 && v[0] == x.size(0), name, " ", v, " does not match the samples of x ", x.sizes());
    return m ? m / v[0] : 0;  // without rows there may be no vectors either
}

void check_devices(const Tensor& x, std::initializer_list<const Tensor*> others) {
    TORCH_CHECK(x.is_cuda(), "dense ops run on CUDA tensors only (the library has no CPU path)");
    for (const Tensor* t : others)
        TORCH_CHECK_VALUE(!t->defined() || t->device() == x.device(), "all tensors must be on the same device");
}

int pack_bit(const Rows& r, int bit) {
    return r.t.defined() && (reinterpret_cast<uintptr_t>(r.t.const_data_ptr()) % 16 || r.ld % 8) ? bit : 0;
}

// Device scratch for one call (the caching allocator orders its reuse on the stream).
Tensor workspace(size_t bytes, const Tensor& like) {
    return bytes ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)) : Tensor();
}

q6_stream_t stream_of(const Tensor& x) {
    return reinterpret_cast<q6_stream_t>(c10::cuda::getCurrentCUDAStream(x.device().index()).stream());
}

void refuse_capture(const Tensor& x, const char* what) {
    if (!x.is_cuda()) return;
    c10::cuda::CUDAGuard guard(x.device());
    TORCH_CHECK(c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None, what,
                " cannot be captured in a CUDA graph with gradients: capture ", what, "_forward and ", what,
                "_backward, or call it under torch.no_grad()");
}

void refuse_second_order(const char* what) {
    TORCH_CHECK(!at::GradMode::is_enabled(), what, " is differentiable once: its backward pass has no gradient");
}

// A tangent (forward-mode differentiation) does not show in requires_grad, and an
// output without one reads as a derivative of zero.
void refuse_tangents(const char* what, std::initializer_list<const Tensor*> tensors) {
    for (const Tensor* t : tensors)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative");
}

at::DimVector with_last(const Tensor& x, int64_t n) {
    at::DimVector s(x.sizes().begin(), x.sizes().end());
    s.back() = n;
    return s;
}

Tensor like(const Tensor& x, at::IntArrayRef shape, at::ScalarType t, bool zero = false) {
    return zero ? at::zeros(shape, x.options().dtype(t)) : at::empty(shape, x.options().dtype(t));
}

// ------------------------------------------------------------------------ linear

int64_t check_linear(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& residual, const Tensor& gate) {
    const auto dt = x.scalar_type();
    TORCH_CHECK_VALUE(is_half(dt), "dense_linear takes bfloat16 or float16, got ", dt);
    TORCH_CHECK_VALUE(w.dim() == 2 && x.dim() >= 1, "weight must be 2-D and x at least 1-D, got ", w.sizes(), ", ",
                      x.sizes());
    const int64_t n = w.size(0), k = w.size(1);
    TORCH_CHECK_VALUE(n > 0 && k > 0, "weight must not be empty, got ", w.sizes());
    TORCH_CHECK_VALUE(x.size(-1) == k, "x in_features ", x.size(-1), " != weight in_features ", k);
    const std::pair<const char*, const Tensor*> named[] = {
        {"weight", &w}, {"bias", &bias}, {"residual", &residual}, {"gate", &gate}};
    for (const auto& [name, t] : named)
        TORCH_CHECK_VALUE(!t->defined() || t->scalar_type() == dt, name, " is ", t->scalar_type(), ", x is ", dt);
    TORCH_CHECK_VALUE(!bias.defined() || (bias.dim() == 1 && bias.size(0) == n), "bias must be (", n, "), got ",
                      bias.sizes());
    if (residual.defined()) {
        const auto want = with_last(x, n);
        TORCH_CHECK_VALUE(residual.sizes() == want, "residual must be ", at::IntArrayRef(want), ", got ",
                          residual.sizes());
    }
    refuse_tangents("dense_linear", {&x, &w, &bias, &residual, &gate});
    return gate.defined() ? sample_rows("gate", gate.sizes(), x, n) : x.numel() / k;
}

std::pair<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& w, const Tensor& bias, int activation,
                                         const Tensor& residual, const Tensor& gate, bool save_preact) {
    const int64_t rows_per_gate = check_linear(x, w, bias, residual, gate);
    check_devices(x, {&w, &bias, &residual, &gate});
    at::AutoDispatchBelowAutograd below;
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t n = w.size(0), k = w.size(1), m = x.numel() / k;
    const auto shape = with_last(x, n);
    Tensor y = like(x, shape, x.scalar_type());
    // the gate's gradient sums act(z) itself: rounded to 16 bits, z could cost it as much as its own rounding
    const auto zt = gate.defined() ? at::kFloat : at::kHalf;
    Tensor z = save_preact ? like(x, shape, zt) : Tensor();
    if (m == 0) return {y, z};
    const Rows rx = rows_of(x, k), rw = rows_of(w, k), rr = rows_of(residual, n), rg = rows_of(gate, n);
    const Tensor b = contiguous(bias);
    const size_t bytes =
        q6_dense_linear_workspace_bytes(m, n, k, pack_bit(rx, Q6_PACK_X) | pack_bit(rw, Q6_PACK_W));
    const Tensor ws = workspace(bytes, x);
    check(q6_dense_linear(ptr(rx.t), rx.ld, ptr(rw.t), rw.ld, ptr(b), ptr(rg.t), rg.ld, rows_per_gate, ptr(rr.t), rr.ld,
                          mutable_ptr(y), mutable_ptr(z), dtype_code(zt), m, n, k, dtype_code(x.scalar_type()),
                          activation, mutable_ptr(ws), bytes, stream_of(x)),
          "q6_dense_linear");
    return {y, z};
}

struct LinearGrads {
    Tensor x, weight, bias, gate;
};

LinearGrads linear_backward(const Tensor& dy, const Tensor& x, const Tensor& w, const Tensor& preact, int activation,
                            const Tensor& gate, int want) {
    const auto dt = dy.scalar_type();
    TORCH_CHECK_VALUE(is_half(dt), "dense_linear_backward takes bfloat16 or float16, got ", dt);
    TORCH_CHECK_VALUE(!((want & Q6_GRAD_W) && !x.defined()) && !((want & Q6_GRAD_X) && !w.defined()),
                      "the weight's gradient needs x, the gradient of x needs weight");
    TORCH_CHECK_VALUE(preact.defined() || !want || (activation == Q6_ACT_NONE && !(want & Q6_GRAD_GATE)),
                      "preact is needed with an activation or for the gate's gradient");
    TORCH_CHECK_VALUE(gate.defined() || !(want & Q6_GRAD_GATE), "the gate's gradient needs gate");
    const int64_t n = dy.dim() ? dy.size(-1) : 0;
    TORCH_CHECK_VALUE(n > 0 && (!w.defined() || (w.dim() == 2 && w.size(0) == n && w.size(1) > 0)), "dy ", dy.sizes(),
                      " does not match weight ", w.defined() ? w.sizes() : at::IntArrayRef());
    const int64_t k = w.defined() ? w.size(1) : x.defined() && x.dim() ? x.size(-1) : 1;
    const auto x_shape = with_last(dy, k);
    TORCH_CHECK_VALUE(!x.defined() || (x.sizes() == x_shape && k > 0), "x ", x.defined() ? x.sizes() : at::IntArrayRef(),
                      " does not match dy ", dy.sizes(), " and ", k, " in_features");
    TORCH_CHECK_VALUE(!preact.defined() || preact.sizes() == dy.sizes(), "preact must be ", dy.sizes(), ", got ",
                      preact.defined() ? preact.sizes() : at::IntArrayRef());
    const std::pair<const char*, const Tensor*> named[] = {
        {"x", &x}, {"weight", &w}, {"preact", &preact}, {"gate", &gate}};
    for (const auto& [name, t] : named)
        TORCH_CHECK_VALUE(!t->defined() || (t == &preact ? t->scalar_type() == at::kFloat || t->scalar_type() == at::kHalf
                                                         : t->scalar_type() == dt),
                          name, " is ", t->scalar_type(), ", dy is ", dt);
    refuse_tangents("dense_linear_backward", {&dy, &x, &w, &preact, &gate});
    const int64_t m = dy.numel() / n;
    const int64_t rows_per_gate = gate.defined() ? sample_rows("gate", gate.sizes(), dy, n) : m;
    check_devices(dy, {&x, &w, &preact, &gate});
    at::AutoDispatchBelowAutograd below;
    c10::cuda::CUDAGuard guard(dy.device());
    LinearGrads g;
    const bool none = m == 0;
    if (want & Q6_GRAD_X) g.x = like(dy, x_shape, dt, none);
    if (want & Q6_GRAD_W) g.weight = like(dy, {n, k}, dt, none);
    if (want & Q6_GRAD_BIAS) g.bias = like(dy, {n}, dt, none);
    if (want & Q6_GRAD_GATE) g.gate = like(dy, gate.sizes(), dt, none);
    if (none || !want) return g;
    const Rows ry = rows_of(dy, n), rg = rows_of(gate, n);
    const Rows rx = (want & Q6_GRAD_W) ? rows_of(x, k) : Rows{Tensor(), k};
    const Rows rw = (want & Q6_GRAD_X) ? rows_of(w, k) : Rows{Tensor(), k};
    const Tensor z = contiguous(preact);
    const int pack = pack_bit(rx, Q6_PACK_X) | pack_bit(rw, Q6_PACK_W) | pack_bit(ry, Q6_PACK_DY);
    const size_t bytes = q6_dense_linear_grad_workspace_bytes(m, n, k, rows_per_gate, activation, gate.defined(), want,
                                                              pack);
    const Tensor ws = workspace(bytes, dy);
    check(q6_dense_linear_grad(ptr(ry.t), ry.ld, ptr(rx.t), rx.ld, ptr(rw.t), rw.ld, ptr(z),
                               dtype_code(z.defined() ? z.scalar_type() : at::kHalf), ptr(rg.t), rg.ld, rows_per_gate,
                               mutable_ptr(g.x), mutable_ptr(g.weight), mutable_ptr(g.bias), mutable_ptr(g.gate), m, n,
                               k, dtype_code(dt), activation, mutable_ptr(ws), bytes, stream_of(dy)),
          "q6_dense_linear_grad");
    return g;
}

struct LinearNode : torch::autograd::Function<LinearNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias_,
                          const OptTensor& gate_, const OptTensor& residual_, int64_t activation) {
        const Tensor bias = of(bias_), gate = of(gate_), residual = of(residual_);
        const bool need_x = x.requires_grad(), need_w = w.requires_grad(), need_g = gate.defined() && gate.requires_grad();
        const bool need_b = bias.defined() && bias.requires_grad();
        const bool save = need_g || (activation != Q6_ACT_NONE && (need_x || need_w || need_b));
        auto [y, z] = linear_forward(x, w, bias, static_cast<int>(activation), residual, gate, save);
        ctx->save_for_backward({need_w ? x : Tensor(), need_x ? w : Tensor(), z, gate});
        ctx->saved_data["activation"] = activation;
        ctx->saved_data["present"] = int64_t(bias.defined()) | int64_t(gate.defined()) << 1 | int64_t(residual.defined()) << 2;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list dys) {
        refuse_second_order("dense_linear");
        const Tensor& dy = dys[0];
        if (!dy.defined()) return variable_list(6);
        refuse_capture(dy, "dense_linear");
        const auto saved = ctx->get_saved_variables();
        // edges are numbered over the tensors that were given
        const int64_t present = ctx->saved_data["present"].toInt();
        size_t edge = 0;
        const auto need = [&](bool given) { return given && ctx->needs_input_grad(edge++); };
        int want = need(true) ? Q6_GRAD_X : 0;
        want |= need(true) ? Q6_GRAD_W : 0;
        want |= need(present & 1) ? Q6_GRAD_BIAS : 0;
        want |= need(present & 2) ? Q6_GRAD_GATE : 0;
        const bool want_residual = need(present & 4);
        LinearGrads g = linear_backward(dy, saved[0], saved[1], saved[2],
                                        static_cast<int>(ctx->saved_data["activation"].toInt()), saved[3], want);
        return {g.x, g.weight, g.bias, g.gate, want_residual ? dy : Tensor(), Tensor()};
    }
};

bool wants_grad(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

Tensor dense_linear(const Tensor& x, const Tensor& w, const OptTensor& bias_, int64_t activation,
                    const OptTensor& residual_, const OptTensor& gate_) {
    const Tensor bias = of(bias_), residual = of(residual_), gate = of(gate_);
    if (!wants_grad({&x, &w, &bias, &gate, &residual}))
        return linear_forward(x, w, bias, static_cast<int>(activation), residual, gate, false).first;
    check_linear(x, w, bias, residual, gate);
    refuse_capture(x, "dense_linear");
    return LinearNode::apply(x, w, bias_, gate_, residual_, activation);
}

// -------------------------------------------------------------------- layer norm

int64_t check_norm(const Tensor& x, const Tensor& w, const Tensor& b, double eps) {
    const auto dt = x.scalar_type();
    TORCH_CHECK_VALUE(dtype_code(dt) >= 0, "layer_norm takes bfloat16, float16 or float32, got ", dt);
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "x must have a last axis of at least one value, got ", x.sizes());
    TORCH_CHECK_VALUE(eps >= 0.0, "eps must not be negative, got ", eps);
    TORCH_CHECK_VALUE(!w.defined() || !b.defined() || (w.scalar_type() == b.scalar_type() && w.sizes() == b.sizes()),
                      "the two vectors must agree, got ", w.scalar_type(), " ", w.sizes(), " and ", b.scalar_type(), " ",
                      b.sizes());
    refuse_tangents("layer_norm", {&x, &w, &b});
    const Tensor& v = w.defined() ? w : b;
    if (!v.defined()) return x.numel() / x.size(-1);
    TORCH_CHECK_VALUE(v.scalar_type() == dt || v.scalar_type() == at::kFloat, "the vectors must be ", dt,
                      " or float32, got ", v.scalar_type());
    return sample_rows("the vectors", v.sizes(), x, x.size(-1));
}

struct NormOut {
    Tensor y, mean, rstd;
};

NormOut norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, int flags, bool stats) {
    const int64_t rows_per_vec = check_norm(x, w, b, eps);
    check_devices(x, {&w, &b});
    at::AutoDispatchBelowAutograd below;
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t d = x.size(-1), m = x.numel() / d;
    NormOut out;
    out.y = like(x, x.sizes(), x.scalar_type());
    if (stats) {
        const Tensor both = like(x, {2, m}, at::kFloat);
        out.mean = both.select(0, 0);
        out.rstd = both.select(0, 1);
    }
    if (m == 0) return out;
    const Rows rx = rows_of(x, d);
    Rows rw = rows_of(w, d), rb = rows_of(b, d);
    if (w.defined() && b.defined() && rw.ld != rb.ld) rw = {rw.t.contiguous(), d}, rb = {rb.t.contiguous(), d};
    const Tensor& v = w.defined() ? w : b;
    const int dt = dtype_code(x.scalar_type());
    check(q6_layer_norm(ptr(rx.t), rx.ld, ptr(rw.t), ptr(rb.t), w.defined() ? rw.ld : rb.ld, rows_per_vec,
                        mutable_ptr(out.y), static_cast<float*>(mutable_ptr(out.mean)),
                        static_cast<float*>(mutable_ptr(out.rstd)), m, d, static_cast<float>(eps), dt,
                        v.defined() ? dtype_code(v.scalar_type()) : dt, flags, stream_of(x)),
          "q6_layer_norm");
    return out;
}

struct NormGrads {
    Tensor x, weight, bias;
};

NormGrads norm_backward(const Tensor& dy, const Tensor& x, const Tensor& w, const Tensor& mean, const Tensor& rstd,
                        at::IntArrayRef vec_shape, at::ScalarType vec_type, int flags, bool want_x, bool want_w,
                        bool want_b) {
    const auto dt = x.scalar_type();
    TORCH_CHECK_VALUE(dtype_code(dt) >= 0 && dy.scalar_type() == dt && dy.sizes() == x.sizes() && x.dim() >= 1 &&
                          x.size(-1) > 0,
                      "dy ", dy.scalar_type(), " ", dy.sizes(), " does not match x ", dt, " ", x.sizes());
    const int64_t d = x.size(-1), m = x.numel() / d;
    const std::pair<const char*, const Tensor*> named[] = {{"mean", &mean}, {"rstd", &rstd}};
    for (const auto& [name, t] : named)
        TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->numel() == m, name, " must hold ", m,
                          " float32 values, got ", t->scalar_type(), " ", t->sizes());
    TORCH_CHECK_VALUE(vec_type == dt || vec_type == at::kFloat, "the vectors must be ", dt, " or float32, got ", vec_type);
    refuse_tangents("layer_norm_backward", {&dy, &x, &w, &mean, &rstd});
    const int64_t rows_per_vec = sample_rows("the vectors", vec_shape, x, d);
    check_devices(dy, {&x, &w, &mean, &rstd});
    at::AutoDispatchBelowAutograd below;
    c10::cuda::CUDAGuard guard(dy.device());
    NormGrads g;
    const bool none = m == 0;
    if (want_x) g.x = like(x, x.sizes(), dt);
    if (want_w) g.weight = like(x, vec_shape, vec_type, none);
    if (want_b) g.bias = like(x, vec_shape, vec_type, none);
    if (none || !(want_x || want_w || want_b)) return g;
    const Rows rx = rows_of(x, d), ry = rows_of(dy, d), rw = rows_of(w, d);
    const Tensor mu = contiguous(mean), rs = contiguous(rstd);
    const int code = dtype_code(dt), bits = (want_w ? Q6_GRAD_W : 0) | (want_b ? Q6_GRAD_BIAS : 0);
    const size_t bytes = bits ? q6_layer_norm_grad_workspace_bytes(m, d, rows_per_vec, code, bits) : 0;
    const Tensor ws = workspace(bytes, x);
    check(q6_layer_norm_grad(ptr(ry.t), ry.ld, ptr(rx.t), rx.ld, ptr(rw.t), rw.ld, rows_per_vec,
                             static_cast<const float*>(ptr(mu)), static_cast<const float*>(ptr(rs)), mutable_ptr(g.x),
                             mutable_ptr(g.weight), mutable_ptr(g.bias), m, d, code, dtype_code(vec_type), flags,
                             mutable_ptr(ws), bytes, stream_of(x)),
          "q6_layer_norm_grad");
    return g;
}

struct NormNode : torch::autograd::Function<NormNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w_, const OptTensor& b_, double eps,
                          int64_t flags) {
        const Tensor w = of(w_), b = of(b_);
        NormOut out = norm_forward(x, w, b, eps, static_cast<int>(flags), true);
        const Tensor& v = w.defined() ? w : b;
        ctx->save_for_backward({x, w, out.mean, out.rstd});
        ctx->saved_data["flags"] = flags;
        ctx->saved_data["present"] = int64_t(w.defined()) | int64_t(b.defined()) << 1;
        ctx->saved_data["shape"] = v.defined() ? v.sizes().vec() : std::vector<int64_t>{x.size(-1)};
        ctx->saved_data["type"] = static_cast<int64_t>(v.defined() ? v.scalar_type() : x.scalar_type());
        return out.y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list dys) {
        refuse_second_order("layer_norm");
        const Tensor& dy = dys[0];
        if (!dy.defined()) return variable_list(5);
        refuse_capture(dy, (ctx->saved_data["flags"].toInt() & Q6_NORM_ONE_PLUS) ? "layer_norm_modulate" : "layer_norm");
        const auto saved = ctx->get_saved_variables();
        const auto shape = ctx->saved_data["shape"].toIntVector();
        const int64_t present = ctx->saved_data["present"].toInt();
        size_t edge = 0;
        const auto need = [&](bool given) { return given && ctx->needs_input_grad(edge++); };
        const bool want_x = need(true), want_w = need(present & 1), want_b = need(present & 2);
        NormGrads g = norm_backward(dy, saved[0], saved[1], saved[2], saved[3], shape,
                                    static_cast<at::ScalarType>(ctx->saved_data["type"].toInt()),
                                    static_cast<int>(ctx->saved_data["flags"].toInt()), want_x, want_w, want_b);
        return {g.x, g.weight, g.bias, Tensor(), Tensor()};
    }
};

Tensor layer_norm(const Tensor& x, const OptTensor& w_, const OptTensor& b_, double eps, int64_t flags) {
    const Tensor w = of(w_), b = of(b_);
    if (!wants_grad({&x, &w, &b})) return norm_forward(x, w, b, eps, static_cast<int>(flags), false).y;
    check_norm(x, w, b, eps);
    refuse_capture(x, (flags & Q6_NORM_ONE_PLUS) ? "layer_norm_modulate" : "layer_norm");
    return NormNode::apply(x, w_, b_, eps, flags);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const StatusError& e) {
            const auto type = py::module_::import("qwen_image_shardedit_mlx_b200._lib").attr("Q6Error");
            PyErr_SetObject(type.ptr(), type(e.status, e.where).ptr());
        }
    });
    m.def("dense_linear", &dense_linear);
    m.def("dense_linear_forward", [](const Tensor& x, const Tensor& w, const OptTensor& bias, int64_t activation,
                                     const OptTensor& residual, const OptTensor& gate, bool save_preact) {
        auto [y, z] = linear_forward(x, w, of(bias), static_cast<int>(activation), of(residual), of(gate), save_preact);
        return std::make_tuple(y, optional_of(z));
    });
    m.def("dense_linear_backward",
          [](const Tensor& dy, const OptTensor& x, const OptTensor& w, const OptTensor& preact, int64_t activation,
             const OptTensor& gate, int64_t want) {
              LinearGrads g = linear_backward(dy, of(x), of(w), of(preact), static_cast<int>(activation), of(gate),
                                              static_cast<int>(want));
              return std::make_tuple(optional_of(g.x), optional_of(g.weight), optional_of(g.bias), optional_of(g.gate));
          });
    m.def("layer_norm", &layer_norm);
    m.def("layer_norm_forward", [](const Tensor& x, const OptTensor& w, const OptTensor& b, double eps, int64_t flags) {
        NormOut o = norm_forward(x, of(w), of(b), eps, static_cast<int>(flags), true);
        return std::make_tuple(o.y, o.mean, o.rstd);
    });
    m.def("layer_norm_backward", [](const Tensor& dy, const Tensor& x, const OptTensor& w_, const Tensor& mean,
                                    const Tensor& rstd, int64_t flags, bool want_x, bool want_w, bool want_b) {
        const Tensor w = of(w_);
        TORCH_CHECK_VALUE(x.dim() >= 1, "x must have a last axis of at least one value, got ", x.sizes());
        const std::vector<int64_t> shape = w.defined() ? w.sizes().vec() : std::vector<int64_t>{x.size(-1)};
        NormGrads g = norm_backward(dy, x, w, mean, rstd, shape, w.defined() ? w.scalar_type() : x.scalar_type(),
                                    static_cast<int>(flags), want_x, want_w, want_b);
        return std::make_tuple(optional_of(g.x), optional_of(g.weight), optional_of(g.bias));
    });
}
