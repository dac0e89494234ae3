// Native tensor front end of the C ABI (include/o1d.h): argument checks, output and workspace allocation
// through torch's caching allocator, device guard, stream, and the call, in one crossing from Python.  The
// same steps written in Python around ctypes cost 40-60 us a call, several times the kernel at small sizes.
//
// Parameters (weights, biases, LayerNorm scales) are passed as they are stored when the kernels take bf16
// ones (O1D_FLAG_PARAMS_BF16); otherwise, or when the library has no such kernel for the request, they are
// converted to fp32 first.
#include <ATen/autocast_mode.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include "../../include/o1d.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

py::object *g_check = nullptr;               // _lib.check(status, what): raises

void check(int status, const char *what) {
    if (status == O1D_OK) return;
    py::gil_scoped_acquire gil;
    (*g_check)(status, what);
}

int dtype_code(const Tensor &t) {
    if (t.scalar_type() == at::kFloat) return O1D_F32;
    if (t.scalar_type() == at::kBFloat16) return O1D_BF16;
    throw py::type_error("oriented1d_b200 supports float32 and bfloat16 tensors, got torch." + std::string(c10::toString(t.scalar_type())));
}
void need_cuda(const Tensor &t) {
    if (!t.is_cuda()) throw std::runtime_error("tensor must be a CUDA tensor (oriented1d_b200 has no CPU path)");
}
void need_cuda(const OptTensor &t) { if (t) need_cuda(*t); }
Tensor as_f32(const Tensor &t) { return t.detach().to(at::kFloat).contiguous(); }
bool is_bf16(const Tensor &t) { return t.scalar_type() == at::kBFloat16; }
void *stream() { return at::cuda::getCurrentCUDAStream().stream(); }
const void *ptr(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }

// Parameters as the library takes them: the stored bf16 values, or fp32 copies.
struct Params {
    Tensor w, b;
    bool bf16;
    Params(const Tensor &w_, const OptTensor &b_) : bf16(is_bf16(w_) && (!b_ || is_bf16(*b_))) {
        w = w_.contiguous();
        if (b_) b = b_->contiguous();
        if (!bf16) widen();
    }
    void widen() {
        w = as_f32(w);
        if (b.defined()) b = as_f32(b);
        bf16 = false;
    }
    int flag() const { return bf16 ? O1D_FLAG_PARAMS_BF16 : 0; }
};
// f(flag) with the parameters as stored, and again with fp32 ones where the library declines those.
template <class F> void call(Params &p, const char *what, F &&f) {
    int rc = f(p.flag());
    if (rc == O1D_ERR_UNSUPPORTED && p.bf16) {
        p.widen();
        rc = f(0);
    }
    check(rc, what);
}

struct Dims { int64_t n, h, w, c; };
Dims dims(const Tensor &t, bool nhwc) {
    if (t.dim() != 4) throw py::value_error("expected a 4-D tensor");
    return nhwc ? Dims{t.size(0), t.size(1), t.size(2), t.size(3)} : Dims{t.size(0), t.size(2), t.size(3), t.size(1)};
}
void check_params(int64_t plan_c, int64_t K, int64_t C, const Tensor *w, const OptTensor *bias) {
    // the kernels index w as [C, K] and bias as [C]: a shorter buffer would be read past its end
    if (plan_c != C)
        throw py::value_error("plan was built for " + std::to_string(plan_c) + " channels, tensor has " + std::to_string(C));
    if (w && w->numel() != C * K)
        throw py::value_error("weight has " + std::to_string(w->numel()) + " elements, expected C*K = " + std::to_string(C * K));
    if (bias && *bias && (*bias)->numel() != C)
        throw py::value_error("bias has " + std::to_string((*bias)->numel()) + " elements, expected C = " + std::to_string(C));
}
// Extents of an output are divided by the stride before the library sees it.
void need_stride(int64_t stride) {
    if (stride <= 0) throw py::value_error("stride must be positive, got " + std::to_string(stride));
}
std::vector<int64_t> shape(int64_t n, int64_t h, int64_t w, int64_t c, bool nhwc) {
    return nhwc ? std::vector<int64_t>{n, h, w, c} : std::vector<int64_t>{n, c, h, w};
}

Tensor fprop(const Tensor &x_, const Tensor &w, const OptTensor &bias, int64_t plan_c, int64_t K, int64_t host, int64_t dev,
             int64_t stride, bool nhwc, bool identity, bool gelu) {
    const Dims d = dims(x_, nhwc);
    need_stride(stride);
    check_params(plan_c, K, d.c, &w, &bias);
    need_cuda(x_); need_cuda(w); need_cuda(bias);
    const c10::cuda::CUDAGuard guard(x_.device());
    const Tensor x = x_.contiguous();
    const int code = dtype_code(x);
    Params p(w, bias);
    Tensor y = at::empty(shape(d.n, (d.h + stride - 1) / stride, (d.w + stride - 1) / stride, d.c, nhwc), x.options());
    const int flags = (identity ? O1D_FLAG_IDENTITY : 0) | (gelu ? O1D_FLAG_GELU_INPUT : 0);
    void *out = y.data_ptr(), *st = stream();
    call(p, "o1d_fprop", [&](int pf) {
        return o1d_fprop(ptr(x), (const float *)ptr(p.w), (const float *)ptr(p.b), (const void *)host, (const void *)dev, out, (int)d.n,
                         (int)d.h, (int)d.w, (int)d.c, (int)K, (int)stride, nhwc, code, flags | pf | O1D_FLAG_MAY_CONVERT, st);
    });
    return y;
}

Tensor dgrad(const Tensor &dy_, const Tensor &w, int64_t plan_c, int64_t K, int64_t host, int64_t dev, int64_t H, int64_t W,
             int64_t stride, bool nhwc, bool identity, const OptTensor &pre_) {
    const Dims d = dims(dy_, nhwc);
    need_stride(stride);
    if (d.h != (H + stride - 1) / stride || d.w != (W + stride - 1) / stride)
        throw py::value_error("dy extents do not match ceil(H/stride) x ceil(W/stride)");
    check_params(plan_c, K, d.c, &w, nullptr);
    need_cuda(dy_); need_cuda(w);
    const c10::cuda::CUDAGuard guard(dy_.device());
    const Tensor dy = dy_.contiguous();
    const int code = dtype_code(dy);
    Params p(w, std::nullopt);
    Tensor dx = at::empty(shape(d.n, H, W, d.c, nhwc), dy.options()), pre;
    if (pre_) {
        if (pre_->sizes() != dx.sizes() || pre_->scalar_type() != dy.scalar_type())
            throw py::value_error("pre must have the shape and dtype of dx");
        need_cuda(*pre_);
        pre = pre_->contiguous();
    }
    void *out = dx.data_ptr(), *st = stream();
    call(p, "o1d_dgrad", [&](int pf) {
        return o1d_dgrad_act(ptr(dy), (const float *)ptr(p.w), ptr(pre), (const void *)host, (const void *)dev, out, (int)d.n, (int)H,
                             (int)W, (int)d.c, (int)K, (int)stride, nhwc, code, (identity ? O1D_FLAG_IDENTITY : 0) | pf | O1D_FLAG_MAY_CONVERT, st);
    });
    return dx;
}

// dw [C,1,1,K] and db [C] (or None), in fp32, or in bf16 when `bf16` is set.
std::tuple<Tensor, OptTensor> wgrad(const Tensor &dy_, const Tensor &x_, int64_t plan_c, int64_t K, int64_t host, int64_t dev,
                                    int64_t stride, bool nhwc, bool with_bias, bool gelu, bool bf16) {
    if (dy_.scalar_type() != x_.scalar_type()) throw py::type_error("dy and x must have the same dtype");
    const Dims d = dims(x_, nhwc);
    need_stride(stride);
    check_params(plan_c, K, d.c, nullptr, nullptr);
    const auto want = shape(d.n, (d.h + stride - 1) / stride, (d.w + stride - 1) / stride, d.c, nhwc);
    if (dy_.sizes() != at::IntArrayRef(want)) {
        std::ostringstream s;
        s << "dy has shape " << dy_.sizes() << ", expected the output shape of x (" << at::IntArrayRef(want) << ")";
        throw py::value_error(s.str());
    }
    need_cuda(dy_); need_cuda(x_);
    const c10::cuda::CUDAGuard guard(x_.device());
    const Tensor dy = dy_.contiguous(), x = x_.contiguous();
    const int code = dtype_code(x);
    auto opts = x.options().dtype(bf16 ? at::kBFloat16 : at::kFloat);
    Tensor dw = at::empty({d.c, 1, 1, K}, opts), db;
    if (with_bias) db = at::empty({d.c}, opts);
    const size_t bytes = std::max<size_t>(16, o1d_wgrad_workspace_bytes((int)d.n, (int)d.h, (int)d.w, (int)d.c, (int)K, (int)stride, nhwc, code));
    Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    void *st = stream();
    auto run = [&](int flag) {
        return o1d_wgrad_act(ptr(dy), ptr(x), (const void *)host, (const void *)dev, (float *)dw.data_ptr(),
                             with_bias ? (float *)db.data_ptr() : nullptr, ws.data_ptr(), bytes, (int)d.n, (int)d.h, (int)d.w, (int)d.c,
                             (int)K, (int)stride, nhwc, code, (gelu ? O1D_FLAG_GELU_INPUT : 0) | flag | O1D_FLAG_MAY_CONVERT, st);
    };
    int rc = run(bf16 ? O1D_FLAG_PARAMS_BF16 : 0);
    if (rc == O1D_ERR_UNSUPPORTED && bf16) {             // kernels that write fp32 gradients only
        dw = at::empty({d.c, 1, 1, K}, x.options().dtype(at::kFloat));
        if (with_bias) db = at::empty({d.c}, x.options().dtype(at::kFloat));
        rc = run(0);
        if (rc == O1D_OK) {
            dw = dw.to(at::kBFloat16);
            if (with_bias) db = db.to(at::kBFloat16);
        }
    }
    check(rc, "o1d_wgrad");
    return {dw, with_bias ? OptTensor(db) : std::nullopt};
}

Tensor transpose(const Tensor &t_, bool to_nhwc) {
    need_cuda(t_);
    if (t_.dim() != 4) throw py::value_error("expected a 4-D tensor");
    const c10::cuda::CUDAGuard guard(t_.device());
    const Tensor t = t_.contiguous();
    const int code = dtype_code(t);
    const int64_t n = t.size(0), hw = to_nhwc ? t.size(2) * t.size(3) : t.size(1) * t.size(2), c = to_nhwc ? t.size(1) : t.size(3);
    Tensor out = to_nhwc ? at::empty({n, t.size(2), t.size(3), c}, t.options()) : at::empty({n, c, t.size(1), t.size(2)}, t.options());
    check(o1d_transpose(ptr(t), out.data_ptr(), (int)n, (int)(to_nhwc ? c : hw), (int)(to_nhwc ? hw : c), code, stream()), "o1d_transpose");
    return out;
}

// The kernels read `expected` elements of a parameter: a shorter buffer would be read past its end.
void need_numel(const Tensor &t, int64_t expected, const char *what) {
    if (t.numel() != expected)
        throw py::value_error(std::string(what) + " has " + std::to_string(t.numel()) + " elements, expected " + std::to_string(expected));
}
// Length of the last axis of a tensor that is normalised or summed by rows.
int64_t row_length(const Tensor &x) {
    if (x.dim() == 0 || x.numel() == 0) throw py::value_error("expected a tensor with at least one row");
    return x.size(-1);
}

Tensor layer_norm_cl(const Tensor &x_, const Tensor &g, const Tensor &b, double eps, bool gelu) {
    need_numel(g, row_length(x_), "weight");
    need_numel(b, row_length(x_), "bias");
    need_cuda(x_); need_cuda(g); need_cuda(b);
    const c10::cuda::CUDAGuard guard(x_.device());
    const Tensor x = x_.contiguous();
    const int code = dtype_code(x);
    const int64_t C = x.size(-1);
    Params p(g, b);
    Tensor y = at::empty_like(x);
    void *st = stream();
    call(p, "o1d_layernorm_cl", [&](int pf) {
        return o1d_layernorm_cl(ptr(x), (const float *)ptr(p.w), (const float *)ptr(p.b), y.data_ptr(), x.numel() / C, (int)C, (float)eps,
                                code, (gelu ? 1 : 0) | pf, st);
    });
    return y;
}

// dx, dweight, dbias; the last two in fp32, or in the parameters' dtype when `as_params` is set.
std::tuple<Tensor, Tensor, Tensor> layer_norm_cl_bwd(const Tensor &x_, const Tensor &dy_, const Tensor &g, double eps, const OptTensor &b,
                                                     bool gelu, bool as_params) {
    if (dy_.sizes() != x_.sizes() || dy_.scalar_type() != x_.scalar_type()) {
        std::ostringstream s;
        s << "dy " << dy_.sizes() << " " << dy_.scalar_type() << " does not match x " << x_.sizes() << " " << x_.scalar_type();
        throw py::value_error(s.str());
    }
    const int64_t C = row_length(x_), rows = x_.numel() / C;
    need_numel(g, C, "weight");
    if (gelu && (!b || b->numel() != C)) throw py::value_error("gelu=True needs the forward call's bias");
    need_cuda(x_); need_cuda(dy_); need_cuda(g);
    if (gelu) need_cuda(b);
    const Tensor x = x_.contiguous(), dy = dy_.contiguous();
    const c10::cuda::CUDAGuard guard(x.device());
    const int code = dtype_code(x);
    Params p(g, gelu ? b : OptTensor());
    const bool out_bf16 = as_params && p.bf16;
    if (!out_bf16 && p.bf16) p.widen();
    Tensor dx = at::empty_like(x);
    auto opts = x.options().dtype(out_bf16 ? at::kBFloat16 : at::kFloat);
    Tensor dg = at::empty({C}, opts), db = at::empty({C}, opts);
    const size_t bytes = o1d_layernorm_cl_bwd_workspace_bytes(rows, (int)C);
    Tensor ws = at::empty({(int64_t)std::max<size_t>(bytes, 4)}, x.options().dtype(at::kByte));
    check(o1d_layernorm_cl_bwd(ptr(x), ptr(dy), (const float *)ptr(p.w), (const float *)ptr(p.b), dx.data_ptr(), (float *)dg.data_ptr(),
                               (float *)db.data_ptr(), ws.data_ptr(), bytes, rows, (int)C, (float)eps, code,
                               (gelu ? 1 : 0) | (out_bf16 ? O1D_FLAG_PARAMS_BF16 : 0), stream()),
          "o1d_layernorm_cl_bwd");
    if (as_params && !out_bf16) { dg = dg.to(g.scalar_type()); db = db.to(b ? b->scalar_type() : g.scalar_type()); }
    return {dx, dg, db};
}

Tensor colsum(const Tensor &x_, bool bf16) {
    const int64_t C = row_length(x_), rows = x_.numel() / C;
    need_cuda(x_);
    const c10::cuda::CUDAGuard guard(x_.device());
    const Tensor x = x_.contiguous();
    const int code = dtype_code(x);
    Tensor out = at::empty({C}, x.options().dtype(bf16 ? at::kBFloat16 : at::kFloat));
    const size_t bytes = o1d_colsum_workspace_bytes(rows, (int)C, code);
    Tensor ws = at::empty({(int64_t)std::max<size_t>(bytes, 4)}, x.options().dtype(at::kByte));
    check(o1d_colsum(ptr(x), (float *)out.data_ptr(), ws.data_ptr(), bytes, rows, (int)C, code | (bf16 ? O1D_FLAG_PARAMS_BF16 : 0), stream()),
          "o1d_colsum");
    return out;
}

Tensor pointwise_in(const Tensor &x_, const Tensor &w, const OptTensor &bias) {
    if (x_.dim() != 4) throw py::value_error("expected a 4-D tensor");
    if (w.dim() == 0) throw py::value_error("weight must be [Cout, Cin]");
    need_numel(w, w.size(0) * x_.size(1), "weight");
    if (bias) need_numel(*bias, w.size(0), "bias");
    need_cuda(x_); need_cuda(w); need_cuda(bias);
    const c10::cuda::CUDAGuard guard(x_.device());
    const Tensor x = x_.contiguous();
    const int code = dtype_code(x);
    Params p(w, bias);
    Tensor y = at::empty({x.size(0), x.size(2), x.size(3), w.size(0)}, x.options());
    void *st = stream();
    call(p, "o1d_pointwise_in", [&](int pf) {
        return o1d_pointwise_in(ptr(x), (const float *)ptr(p.w), (const float *)ptr(p.b), y.data_ptr(), (int)x.size(0), (int)x.size(1),
                                x.size(2) * x.size(3), (int)w.size(0), code | pf, st);
    });
    return y;
}

// The operator's autograd node (reference: models/dwoconv1d/dwoconv1d.py:18-69), free of Python on the
// backward thread.  An NCHW tensor whose NHWC form has a fast path (`via`) is converted on the way in and
// out, and its NHWC form is what backward keeps.
struct ConvFn : torch::autograd::Function<ConvFn> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &x_, const Tensor &w, const Tensor &theta,
                          const OptTensor &bias, const Tensor &host, const Tensor &dev, int64_t plan_c, int64_t K, int64_t stride, bool nhwc,
                          bool via, bool identity, bool gelu) {
        (void)theta;
        const Tensor x = via ? transpose(x_, true) : x_.contiguous();
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x, w});
        ctx->saved_data["host"] = host;
        ctx->saved_data["dev"] = dev;
        ctx->saved_data["p"] = std::vector<int64_t>{plan_c, K, stride, nhwc, via, identity, gelu, bias.has_value()};
        const Tensor y = fprop(x, w, bias, plan_c, K, (int64_t)host.const_data_ptr(), (int64_t)dev.const_data_ptr(), stride, nhwc || via,
                               identity, gelu);
        return via ? transpose(y, false) : y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        torch::autograd::variable_list out(13);
        Tensor dy = grads[0];
        if (!dy.defined()) return out;
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1];
        const auto p = ctx->saved_data["p"].toIntVector();
        const int64_t plan_c = p[0], K = p[1], stride = p[2], host = (int64_t)ctx->saved_data["host"].toTensor().const_data_ptr(),
                      dev = (int64_t)ctx->saved_data["dev"].toTensor().const_data_ptr();
        const bool nhwc = p[3] || p[4], via = p[4], identity = p[5], gelu = p[6], has_bias = p[7];
        if (dy.scalar_type() != x.scalar_type()) dy = dy.to(x.scalar_type());
        dy = via ? transpose(dy, true) : dy.contiguous();
        if (ctx->needs_input_grad(0)) {
            out[0] = dgrad(dy, w, plan_c, K, host, dev, x.size(nhwc ? 1 : 2), x.size(nhwc ? 2 : 3), stride, nhwc, identity,
                           gelu ? OptTensor(x) : std::nullopt);
            if (via) out[0] = transpose(out[0], false);
        }
        const bool need_w = ctx->needs_input_grad(1), need_b = has_bias && ctx->needs_input_grad(3);
        if (need_w || need_b) {
            auto [dw, db] = wgrad(dy, x, plan_c, K, host, dev, stride, nhwc, need_b, gelu, is_bf16(w));
            const auto dt = w.scalar_type();             // the bias shares the weight's dtype
            if (need_w) out[1] = dw.scalar_type() == dt ? dw : dw.to(dt);
            if (need_b) out[3] = db->scalar_type() == dt ? *db : db->to(dt);
        }
        return out;
    }
};

// Channels-last LayerNorm (and GELU) with this library's kernels on both passes.
struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &x_, const Tensor &g, const Tensor &b, double eps, bool gelu) {
        const Tensor x = x_.contiguous();
        ctx->save_for_backward({x, g, b});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["gelu"] = gelu;
        return layer_norm_cl(x, g, b, eps, gelu);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        auto [dx, dg, db] = layer_norm_cl_bwd(saved[0], grads[0], saved[1], ctx->saved_data["eps"].toDouble(), saved[2],
                                              ctx->saved_data["gelu"].toBool(), true);
        return {ctx->needs_input_grad(0) ? dx : Tensor(), ctx->needs_input_grad(1) ? dg : Tensor(), ctx->needs_input_grad(2) ? db : Tensor(),
                Tensor(), Tensor()};
    }
};
Tensor layer_norm_train(const Tensor &x, const Tensor &g, const Tensor &b, double eps, bool gelu) { return LayerNormFn::apply(x, g, b, eps, gelu); }

// Linear on channels-last activations whose bias gradient is this library's column sum; the two matrix
// products stay with the GEMM library.
struct LinearFn : torch::autograd::Function<LinearFn> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Tensor &w, const Tensor &b) {
        ctx->save_for_backward({x, w});
        ctx->saved_data["bias"] = (int64_t)b.scalar_type();
        return at::linear(x, w, b);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], dy = grads[0].reshape({-1, grads[0].size(-1)});
        torch::autograd::variable_list out(3);
        if (ctx->needs_input_grad(0)) out[0] = dy.matmul(w).reshape(x.sizes());
        if (ctx->needs_input_grad(1)) out[1] = dy.t().matmul(x.reshape({-1, x.size(-1)}));
        if (ctx->needs_input_grad(2)) {
            const auto dt = (at::ScalarType)ctx->saved_data["bias"].toInt();
            out[2] = colsum(dy, dt == at::kBFloat16);
            if (out[2].scalar_type() != dt) out[2] = out[2].to(dt);
        }
        return out;
    }
};
Tensor linear_train(const Tensor &x, const Tensor &w, const Tensor &b) {
    // An autocast region that converts an operand: the saved tensors would not be those of the product.  torch's own operator then,
    // whose graph has the conversions in it.
    if (at::autocast::is_autocast_enabled(at::kCUDA)) {
        const auto type = at::autocast::get_autocast_dtype(at::kCUDA);
        if (x.scalar_type() != type || w.scalar_type() != type || b.scalar_type() != type) return at::linear(x, w, b);
    }
    return LinearFn::apply(x, w, b);
}

// ---- 8-bit activation checkpoints --------------------------------------------------------------------
// Outputs and workspaces straight from the allocator, without the dispatcher (1.8 us a tensor, up to eight a call).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor &like) {
    return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}
// Device memory for the length of a call (kernels on the current stream may still use it: it is only handed out again there).
struct Scratch {
    c10::DataPtr mem;
    size_t bytes;
    explicit Scratch(size_t n) : bytes(n) { if (n) mem = c10::cuda::CUDACachingAllocator::get()->allocate(n); }
    void *get() const { return mem.get(); }
};
Tensor as_type(const Tensor &t, at::ScalarType type) { return t.scalar_type() == type ? t : t.to(type); }
Tensor as_sizes(const Tensor &t, at::IntArrayRef sizes) { return t.sizes() == sizes ? t : t.reshape(sizes); }
Tensor as_shape(const Tensor &t, const Tensor &like) { return as_sizes(t, like.sizes()); }
// Contiguous, and starting on 16 bytes, as tensor copies and vector loads want it.
Tensor as_vectors(const Tensor &t) {
    const Tensor c = t.contiguous();
    return ((uintptr_t)c.const_data_ptr() & 15) ? c.clone() : c;
}
// All tensors of a call live on one device: the library launches there, on that device's current stream.
void need_device(const Tensor &t, const Tensor &like, const char *what) {
    need_cuda(t);
    if (t.device() != like.device())
        throw py::value_error(std::string(what) + " is on " + t.device().str() + ", the first tensor on " + like.device().str());
}
// Nodes of the graph for the operators below: their own, since torch::autograd::Function keeps what a node needs in a dictionary of
// boxed values and wraps outputs for every kind of operator (6-10 us a step, of which the kernels of a small call take 6).
using torch::autograd::variable_list;
struct TrainNode : torch::autograd::Node {
    using torch::autograd::Node::Node;
    std::vector<torch::autograd::SavedVariable> saved;
    void keep(std::initializer_list<Tensor> tensors) {
        saved.reserve(tensors.size());
        for (const Tensor &t : tensors) saved.emplace_back(t, false);
    }
    Tensor kept(size_t i) const { return saved[i].unpack(); }
    bool need(size_t i) const { return task_should_compute_output(i); }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (auto &s : saved) s.reset_data();
    }
    variable_list apply(variable_list &&grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(num_outputs());
        if (!grads[0].defined()) return out;
        // these differentiate once; a graph of their backward pass would silently leave them out
        if (at::GradMode::is_enabled()) throw std::runtime_error(name() + " has no second derivative (create_graph=True)");
        // (the engine brings along the autocast state of the thread that called it: a product would round its operands to that type)
        const c10::impl::ExcludeDispatchKeyGuard as_given(c10::autocast_dispatch_keyset);
        backward(grads[0], out);
        return out;
    }
    virtual void backward(const Tensor &grad, variable_list &out) = 0;
};
// (What a node's forward pass calls is dispatched below autograd: recorded nowhere, and no view of anything to autograd.)
template <class N, class... In> std::shared_ptr<N> make_node(const In &...in) {
    return std::shared_ptr<N>(new N(torch::autograd::collect_next_edges(in...)), torch::autograd::deleteNode);
}
bool wants_grad(const Tensor &t) {
    if (t.defined() && t._fw_grad(0).defined()) throw std::runtime_error("no forward-mode derivative");
    return t.defined() && t.requires_grad();
}
bool wants_grad(const OptTensor &t) { return t && wants_grad(*t); }
template <class... In> bool trains(const In &...in) { return (static_cast<int>(wants_grad(in)) + ...) > 0 && at::GradMode::is_enabled(); }
// [rows, C] of a tensor whose last axis is a row; no rows is a valid tensor, no columns is not.
struct Rows {
    int64_t rows, C;
    explicit Rows(const Tensor &x) {
        if (x.dim() == 0 || x.size(-1) == 0) throw py::value_error("expected a tensor with at least one column");
        C = x.size(-1);
        rows = x.numel() / C;
        if (C > INT32_MAX) throw py::value_error("rows of more than 2^31 - 1 elements are not supported");
    }
};
// A vector for a gradient; zeros where no kernel will write it.
Tensor vector_of(int64_t n, at::ScalarType type, const Tensor &like, bool zero) {
    Tensor t = fresh({n}, type, like);
    return zero ? t.zero_() : t;
}
// The checkpoint of a tensor of [rows, C]; behind the ranges two floats a row where LayerNorm needs them.  (All in one allocation
// would be rounded up to the next 2 MB where it is large.)
struct Kept {
    Tensor codes_, side;
    int64_t rows = 0, C = 0;
    void make(const Rows &r, const Tensor &like, bool with_stats) {
        rows = r.rows; C = r.C;
        codes_ = fresh({rows * C}, at::kByte, like);
        side = fresh({rows * ((C + 127) / 128 + with_stats) * 2}, at::kFloat, like);
    }
    uint8_t *codes() const { return codes_.defined() ? (uint8_t *)codes_.data_ptr() : nullptr; }
    float *ranges() const { return side.defined() ? (float *)side.data_ptr() : nullptr; }
    float *stats() const { return side.defined() ? ranges() + rows * ((C + 127) / 128) * 2 : nullptr; }
    // in a node the memory is in saved variables, the rest is kept as it is
    Kept without() const { Kept k; k.rows = rows; k.C = C; return k; }
    Kept with(const Tensor &c, const Tensor &s) const { Kept k = *this; k.codes_ = c; k.side = s; return k; }
};
void need_kept(const Tensor &codes, const Tensor &ranges) {
    if (codes.scalar_type() != at::kByte || ranges.scalar_type() != at::kFloat)
        throw py::type_error("a checkpoint is uint8 codes and float32 ranges");
    const Rows r(codes);
    auto want = codes.sizes().vec();
    want.back() = (want.back() + 127) / 128;
    want.push_back(2);
    if (ranges.sizes() != at::IntArrayRef(want)) {
        std::ostringstream s;
        s << "ranges have shape " << ranges.sizes() << ", codes of shape " << codes.sizes() << " need " << at::IntArrayRef(want);
        throw py::value_error(s.str());
    }
}

std::tuple<Tensor, Tensor> keep8(const Tensor &x_) {
    const Rows r(x_);
    const int code = dtype_code(x_);
    need_cuda(x_);
    const c10::cuda::CUDAGuard guard(x_.device());
    const Tensor x = x_.contiguous();
    auto shape = x.sizes().vec();
    shape.back() = (shape.back() + 127) / 128;
    shape.push_back(2);
    const Tensor codes = fresh(x.sizes(), at::kByte, x), ranges = fresh(shape, at::kFloat, x);
    if (r.rows)
        check(o1d_keep8(ptr(x), (uint8_t *)codes.data_ptr(), (float *)ranges.data_ptr(), r.rows, (int)r.C, code, stream()), "o1d_keep8");
    return {codes, ranges};
}

Tensor restore8(const Tensor &codes_, const Tensor &ranges_, bool bf16) {
    need_kept(codes_, ranges_);
    const Rows r(codes_);
    need_cuda(codes_); need_device(ranges_, codes_, "ranges");
    const c10::cuda::CUDAGuard guard(codes_.device());
    const Tensor codes = codes_.contiguous();
    Tensor ranges = ranges_.contiguous();
    if ((uintptr_t)ptr(ranges) & 7) ranges = ranges.clone();      // (read in pairs; a view of a larger buffer may start between two)
    Tensor y = fresh(codes.sizes(), bf16 ? at::kBFloat16 : at::kFloat, codes);
    if (r.rows)
        check(o1d_restore8((const uint8_t *)ptr(codes), (const float *)ptr(ranges), y.data_ptr(), r.rows, (int)r.C, bf16 ? O1D_BF16 : O1D_F32, stream()),
              "o1d_restore8");
    return y;
}

// GELU(x + bias), and the checkpoint of x + bias when `keep` is set.
std::tuple<Tensor, Kept> gelu_forward(const Tensor &x_, const OptTensor &bias, bool keep) {
    const Rows r(x_);
    const int code = dtype_code(x_);
    if (bias) need_numel(*bias, r.C, "bias");
    need_cuda(x_);
    if (bias) need_device(*bias, x_, "bias");
    const c10::cuda::CUDAGuard guard(x_.device());
    const Tensor x = x_.contiguous();
    Tensor b;
    if (bias) b = is_bf16(*bias) || bias->scalar_type() == at::kFloat ? bias->contiguous() : as_f32(*bias);
    Tensor y = fresh(x.sizes(), x.scalar_type(), x);
    Kept k;
    if (keep) k.make(r, x, false);
    if (r.rows)
        check(o1d_gelu_keep8(ptr(x), (const float *)ptr(b), y.data_ptr(), k.codes(), k.ranges(), r.rows, (int)r.C,
                             code | (bias && is_bf16(b) ? O1D_FLAG_PARAMS_BF16 : 0), stream()),
              "o1d_gelu_keep8");
    return {y, k};
}

struct GeluGrads { Tensor dx, db, y; };
// dx; the bias gradient in `db_type` when `with_db` is set; the activation once more when `with_y` is.
GeluGrads gelu_backward(const Kept &k, const Tensor &dy_, bool with_db, at::ScalarType db_type, bool with_y) {
    const c10::cuda::CUDAGuard guard(dy_.device());
    const Tensor dy = dy_.contiguous();
    const int code = dtype_code(dy);
    GeluGrads g{fresh(dy.sizes(), dy.scalar_type(), dy), {}, {}};
    if (with_y) g.y = fresh(dy.sizes(), dy.scalar_type(), dy);
    const bool db16 = db_type == at::kBFloat16;
    const Scratch ws(with_db ? o1d_gelu_keep8_bwd_workspace_bytes(k.rows, (int)k.C) : 0);
    if (with_db) g.db = vector_of(k.C, db16 ? at::kBFloat16 : at::kFloat, dy, k.rows == 0);
    if (k.rows)
        check(o1d_gelu_keep8_bwd(k.codes(), k.ranges(), ptr(dy), g.dx.data_ptr(), with_y ? g.y.data_ptr() : nullptr,
                                 with_db ? (float *)g.db.data_ptr() : nullptr, ws.get(), ws.bytes, k.rows, (int)k.C, code | (db16 ? O1D_FLAG_PARAMS_BF16 : 0), stream()),
              "o1d_gelu_keep8_bwd");
    if (with_db) g.db = as_type(g.db, db_type);
    return g;
}

struct GeluKeep8 : TrainNode {
    using TrainNode::TrainNode;
    Kept k;
    at::ScalarType type, bias_type = at::kFloat;
    std::vector<int64_t> bias_sizes;
    std::string name() const override { return "gelu_keep8"; }
    void backward(const Tensor &grad, variable_list &out) override {
        const bool need_db = need(1);
        GeluGrads g = gelu_backward(k.with(kept(0), kept(1)), as_type(grad, type), need_db, bias_type, false);
        if (need(0)) out[0] = g.dx;
        if (need_db) out[1] = as_sizes(g.db, bias_sizes);
    }
};
Tensor gelu_keep8(const Tensor &x, const OptTensor &bias) {
    if (!trains(x, bias)) return std::get<0>(gelu_forward(x, bias, false));
    const auto node = make_node<GeluKeep8>(x, bias);
    const at::AutoDispatchBelowADInplaceOrView off;
    auto [y, k] = gelu_forward(x, bias, true);
    node->keep({k.codes_, k.side});
    node->k = k.without();
    node->type = x.scalar_type();
    if (bias) { node->bias_type = bias->scalar_type(); node->bias_sizes = bias->sizes().vec(); }
    torch::autograd::set_history(y, node);
    return y;
}

// The checkpoint and the statistics only when `keep` is set.
std::tuple<Tensor, Kept> ln_keep_forward(const Tensor &x_, const Tensor &g, const Tensor &b, double eps, bool keep) {
    const Rows r(x_);
    const int code = dtype_code(x_);
    need_numel(g, r.C, "weight");
    need_numel(b, r.C, "bias");
    need_cuda(x_); need_device(g, x_, "weight"); need_device(b, x_, "bias");
    const c10::cuda::CUDAGuard guard(x_.device());
    const Tensor x = x_.contiguous();
    Params p(g, b);
    Tensor y = fresh(x.sizes(), x.scalar_type(), x);
    Kept k;
    if (keep) k.make(r, x, true);
    if (r.rows)
        check(o1d_layernorm_keep8(ptr(x), (const float *)ptr(p.w), (const float *)ptr(p.b), y.data_ptr(), k.codes(), k.ranges(), k.stats(), r.rows,
                                  (int)r.C, (float)eps, code | p.flag(), stream()),
              "o1d_layernorm_keep8");
    return {y, k};
}

struct LnGrads { Tensor dx, dg, db, y; };
LnGrads ln_keep_backward(const Kept &k, const Tensor &dy_, const Tensor &g, const Tensor &b, bool with_y) {
    const c10::cuda::CUDAGuard guard(dy_.device());
    const Tensor dy = dy_.contiguous();
    const int code = dtype_code(dy);
    Params p(g, b);
    LnGrads out{fresh(dy.sizes(), dy.scalar_type(), dy), {}, {}, {}};
    const auto type = p.bf16 ? at::kBFloat16 : at::kFloat;
    out.dg = vector_of(k.C, type, dy, k.rows == 0);
    out.db = vector_of(k.C, type, dy, k.rows == 0);
    if (with_y) out.y = fresh(dy.sizes(), dy.scalar_type(), dy);
    const Scratch ws(o1d_layernorm_keep8_bwd_workspace_bytes(k.rows, (int)k.C));
    if (k.rows)
        check(o1d_layernorm_keep8_bwd(k.codes(), k.ranges(), k.stats(), ptr(dy), (const float *)ptr(p.w), (const float *)ptr(p.b), out.dx.data_ptr(),
                                      with_y ? out.y.data_ptr() : nullptr, (float *)out.dg.data_ptr(), (float *)out.db.data_ptr(), ws.get(), ws.bytes,
                                      k.rows, (int)k.C,
                                      code | p.flag(), stream()),
              "o1d_layernorm_keep8_bwd");
    out.dg = as_shape(as_type(out.dg, g.scalar_type()), g);
    out.db = as_shape(as_type(out.db, b.scalar_type()), b);
    return out;
}

struct LayerNormKeep8 : TrainNode {
    using TrainNode::TrainNode;
    Kept k;
    at::ScalarType type;
    std::string name() const override { return "layer_norm_keep8"; }
    void backward(const Tensor &grad, variable_list &out) override {
        LnGrads g = ln_keep_backward(k.with(kept(0), kept(1)), as_type(grad, type), kept(2), kept(3), false);
        if (need(0)) out[0] = g.dx;
        if (need(1)) out[1] = g.dg;
        if (need(2)) out[2] = g.db;
    }
};
Tensor layer_norm_keep8(const Tensor &x, const Tensor &g, const Tensor &b, double eps) {
    if (!trains(x, g, b)) return std::get<0>(ln_keep_forward(x, g, b, eps, false));
    const auto node = make_node<LayerNormKeep8>(x, g, b);
    const at::AutoDispatchBelowADInplaceOrView off;
    auto [y, k] = ln_keep_forward(x, g, b, eps, true);
    node->keep({k.codes_, k.side, g, b});
    node->k = k.without();
    node->type = x.scalar_type();
    torch::autograd::set_history(y, node);
    return y;
}

// ---- a block's LayerNorm -> Linear -> GELU -> Linear with 8-bit checkpoints -------------------------------
// Kept between the passes: the codes of x (from which LayerNorm's output, the first Linear's input, is formed again) and
// of the first Linear's output (from which the activation is); the four matrix products stay with the GEMM library.
Tensor sum_rows(const Tensor &dy, at::ScalarType dt) {
    const int64_t ve = dy.scalar_type() == at::kFloat ? 4 : 8;
    return as_type(dy.numel() && dy.size(-1) % ve == 0 ? colsum(as_vectors(dy), dt == at::kBFloat16) : dy.sum(0, false, at::kFloat), dt);
}
struct MlpKeep8 : TrainNode {
    using TrainNode::TrainNode;
    Kept kx, kh;
    at::ScalarType type, b1_type, b2_type;
    std::vector<int64_t> b1_sizes, b2_sizes;
    std::string name() const override { return "mlp_keep8"; }
    void backward(const Tensor &grad, variable_list &out) override {
        const Tensor g = kept(4), b = kept(5), w1 = kept(6), w2 = kept(7), dz = as_type(grad, type);
        const Tensor dz2 = dz.reshape({-1, dz.size(-1)});
        const c10::cuda::CUDAGuard guard(dz.device());
        if (need(6)) out[6] = as_sizes(sum_rows(dz2, b2_type), b2_sizes);
        GeluGrads h = gelu_backward(kh.with(kept(2), kept(3)), dz.matmul(w2), need(4), b1_type, need(5));
        if (need(4)) out[4] = as_sizes(h.db, b1_sizes);
        if (need(5)) out[5] = dz2.t().matmul(h.y.reshape({-1, h.y.size(-1)}));
        h.y = Tensor();
        if (!(need(0) || need(1) || need(2) || need(3))) return;
        LnGrads n = ln_keep_backward(kx.with(kept(0), kept(1)), h.dx.matmul(w1), g, b, need(3));
        if (need(0)) out[0] = n.dx;
        if (need(1)) out[1] = n.dg;
        if (need(2)) out[2] = n.db;
        if (need(3)) out[3] = h.dx.reshape({-1, h.dx.size(-1)}).t().matmul(n.y.reshape({-1, n.y.size(-1)}));
    }
};
Tensor mlp_keep8(const Tensor &x, const Tensor &g, const Tensor &b, const Tensor &w1, const Tensor &b1, const Tensor &w2, const Tensor &b2, double eps) {
    const Rows r(x);
    dtype_code(x);
    if (w1.dim() != 2 || w1.size(1) != r.C || w1.size(0) == 0) throw py::value_error("weight1 must be [hidden, " + std::to_string(r.C) + "]");
    if (w2.dim() != 2 || w2.size(1) != w1.size(0) || w2.size(0) == 0) throw py::value_error("weight2 must be [features, " + std::to_string(w1.size(0)) + "]");
    need_numel(g, r.C, "weight");
    need_numel(b, r.C, "bias");
    need_numel(b1, w1.size(0), "bias1");
    need_numel(b2, w2.size(0), "bias2");
    if (w1.scalar_type() != x.scalar_type() || w2.scalar_type() != x.scalar_type() || b2.scalar_type() != x.scalar_type())
        throw py::type_error("x and the Linear layers' parameters must have the same dtype");
    need_cuda(x);
    for (const Tensor *t : {&g, &b, &w1, &b1, &w2, &b2}) need_device(*t, x, "a parameter");
    const c10::cuda::CUDAGuard guard(x.device());
    const c10::impl::ExcludeDispatchKeyGuard as_given(c10::autocast_dispatch_keyset);      // the products' dtype is x's
    if (!trains(x, g, b, w1, b1, w2, b2))
        return at::linear(std::get<0>(gelu_forward(at::linear(std::get<0>(ln_keep_forward(x, g, b, eps, false)), w1), b1, false)), w2, b2);
    const auto node = make_node<MlpKeep8>(x, g, b, w1, b1, w2, b2);
    const at::AutoDispatchBelowADInplaceOrView off;
    auto [y, kx] = ln_keep_forward(x, g, b, eps, true);
    auto [a, kh] = gelu_forward(at::linear(y, w1), b1, true);
    node->keep({kx.codes_, kx.side, kh.codes_, kh.side, g, b, w1, w2});
    node->kx = kx.without(); node->kh = kh.without();
    node->type = x.scalar_type(); node->b1_type = b1.scalar_type(); node->b2_type = b2.scalar_type();
    node->b1_sizes = b1.sizes().vec(); node->b2_sizes = b2.sizes().vec();
    Tensor z = at::linear(a, w2, b2);
    torch::autograd::set_history(z, node);
    return z;
}

// ---- softmax cross entropy of a linear classifier ----------------------------------------------------
struct XentShape {
    int64_t N, D, V;
    XentShape(const Tensor &x, const Tensor &w, const OptTensor &bias, const Tensor &target, double smoothing) {
        if (x.dim() == 0 || x.size(-1) == 0) throw py::value_error("x must have at least one feature");
        D = x.size(-1);
        N = x.numel() / D;
        if (w.dim() != 2 || w.size(1) != D || w.size(0) == 0)
            throw py::value_error("weight must be [classes, " + std::to_string(D) + "]");
        V = w.size(0);
        if (w.scalar_type() != x.scalar_type()) throw py::type_error("x and weight must have the same dtype");
        if (bias) need_numel(*bias, V, "bias");
        if (target.scalar_type() != at::kLong) throw py::type_error("target must be int64 class indices");
        if (target.sizes() != x.sizes().slice(0, x.dim() - 1)) {
            std::ostringstream s;
            s << "target has shape " << target.sizes() << ", x of shape " << x.sizes() << " needs " << x.sizes().slice(0, x.dim() - 1);
            throw py::value_error(s.str());
        }
        if (!(smoothing >= 0. && smoothing <= 1.)) throw py::value_error("label_smoothing must be between 0 and 1");
        if (D > 0x7fff0000 || V > 0x7fff0000 || N > 0x7fff0000) throw py::value_error("more than 2^31 - 65536 rows, classes or features are not supported");
        need_cuda(x); need_device(w, x, "weight"); need_device(target, x, "target");
        if (bias) need_device(*bias, x, "bias");
    }
};
Tensor xent_bias(const OptTensor &b) { return !b ? Tensor() : is_bf16(*b) || b->scalar_type() == at::kFloat ? b->contiguous() : as_f32(*b); }
struct XentOut { Tensor loss, kept; };       // kept: three floats a row for the backward pass, and the number of rows that have a loss
XentOut xent_forward(const Tensor &x_, const Tensor &w_, const OptTensor &bias, const Tensor &target_, int64_t ignore, double smoothing,
                     int64_t reduction, bool train) {
    const int code = dtype_code(x_);
    const XentShape s(x_, w_, bias, target_, smoothing);
    const c10::cuda::CUDAGuard guard(x_.device());
    const Tensor x = as_vectors(x_), w = as_vectors(w_), target = target_.contiguous(), b = xent_bias(bias);
    const bool each = reduction == O1D_XENT_NONE;
    const int64_t rows = train ? 3 * s.N : 0;
    XentOut o{fresh(each ? target.sizes() : at::IntArrayRef{}, at::kFloat, x), fresh({rows + 1}, at::kFloat, x)};
    float *kept = (float *)o.kept.data_ptr();
    if (s.N == 0) {                                       // the sum of nothing, the mean of nothing
        if (!each) o.loss.fill_(reduction == O1D_XENT_SUM ? 0. : NAN);
        return o;
    }
    const Scratch ws(o1d_linear_xent_workspace_bytes(s.N, (int)s.D, (int)s.V, code, train ? O1D_XENT_FORWARD : O1D_XENT_EVALUATION));
    check(o1d_linear_xent(ptr(x), ptr(w), ptr(b), (const long long *)ptr(target), (float *)o.loss.data_ptr(), train ? kept : nullptr,
                          each ? nullptr : kept + rows, ws.get(), ws.bytes, s.N, (int)s.D, (int)s.V, ignore, (float)smoothing,
                          (int)reduction, code | (b.defined() && is_bf16(b) ? O1D_FLAG_PARAMS_BF16 : 0), stream()),
          "o1d_linear_xent");
    return o;
}

struct LinearXent : TrainNode {
    using TrainNode::TrainNode;
    int64_t ignore, reduction;
    double smoothing;
    std::string name() const override { return "linear_cross_entropy"; }
    void backward(const Tensor &grad, variable_list &out) override {
        const Tensor x_ = kept(0), w_ = kept(1), bias_ = kept(2), target_ = kept(3), stats = kept(4);
        const OptTensor bias = bias_.defined() ? OptTensor(bias_) : std::nullopt;
        const XentShape s(x_, w_, bias, target_, smoothing);
        const c10::cuda::CUDAGuard guard(x_.device());
        const Tensor x = as_vectors(x_), w = as_vectors(w_), target = target_.contiguous(), b = xent_bias(bias);
        const Tensor dloss = as_type(grad, at::kFloat).contiguous();
        const bool dx = need(0), dw = need(1), db = need(2), none = s.N == 0;
        if (dx) out[0] = fresh(x.sizes(), x.scalar_type(), x);
        if (dw) { out[1] = fresh(w.sizes(), w.scalar_type(), w); if (none) out[1].zero_(); }
        if (db) out[2] = vector_of(s.V, b.scalar_type(), x, none);
        if (!none) {
            const int code = dtype_code(x);
            const float *lse = (const float *)ptr(stats);
            const Scratch ws(o1d_linear_xent_workspace_bytes(s.N, (int)s.D, (int)s.V, code, O1D_XENT_BACKWARD));
            check(o1d_linear_xent_bwd(ptr(x), ptr(w), ptr(b), (const long long *)ptr(target), lse, lse + 3 * s.N, (const float *)ptr(dloss),
                                      dx ? out[0].data_ptr() : nullptr, dw ? out[1].data_ptr() : nullptr, db ? out[2].data_ptr() : nullptr, ws.get(),
                                      ws.bytes, s.N, (int)s.D, (int)s.V, ignore, (float)smoothing, (int)reduction,
                                      code | (b.defined() && is_bf16(b) ? O1D_FLAG_PARAMS_BF16 : 0), ::stream()),
                  "o1d_linear_xent_bwd");
        }
        if (db) out[2] = as_shape(as_type(out[2], bias->scalar_type()), *bias);
    }
};
Tensor linear_xent(const Tensor &x, const Tensor &w, const OptTensor &bias, const Tensor &target, int64_t ignore, double smoothing, int64_t reduction) {
    if (!trains(x, w, bias)) return xent_forward(x, w, bias, target, ignore, smoothing, reduction, false).loss;
    const auto node = make_node<LinearXent>(x, w, bias);
    const at::AutoDispatchBelowADInplaceOrView off;
    XentOut o = xent_forward(x, w, bias, target, ignore, smoothing, reduction, true);
    node->keep({x, w, bias ? *bias : Tensor(), target, o.kept});
    node->ignore = ignore; node->reduction = reduction; node->smoothing = smoothing;
    torch::autograd::set_history(o.loss, node);
    return o.loss;
}

Tensor conv(const Tensor &x, const Tensor &w, const Tensor &theta, const OptTensor &bias, const Tensor &host, const Tensor &dev,
            int64_t plan_c, int64_t K, int64_t stride, bool nhwc, bool via, bool identity, bool gelu) {
    return ConvFn::apply(x, w, theta, bias, host, dev, plan_c, K, stride, nhwc, via, identity, gelu);
}

}  // namespace

PYBIND11_MODULE(_o1d_torch, m) {
    m.def("set_check", [](py::object f) { g_check = new py::object(std::move(f)); });
    m.def("fprop", &fprop, py::call_guard<py::gil_scoped_release>());
    m.def("dgrad", &dgrad, py::call_guard<py::gil_scoped_release>());
    m.def("wgrad", &wgrad, py::call_guard<py::gil_scoped_release>());
    m.def("conv", &conv, py::call_guard<py::gil_scoped_release>());
    m.def("layer_norm_train", &layer_norm_train, py::call_guard<py::gil_scoped_release>());
    m.def("linear_train", &linear_train, py::call_guard<py::gil_scoped_release>());
    m.def("transpose", &transpose, py::call_guard<py::gil_scoped_release>());
    m.def("layer_norm_cl", &layer_norm_cl, py::call_guard<py::gil_scoped_release>());
    m.def("layer_norm_cl_bwd", &layer_norm_cl_bwd, py::call_guard<py::gil_scoped_release>());
    m.def("colsum", &colsum, py::call_guard<py::gil_scoped_release>());
    m.def("pointwise_in", &pointwise_in, py::call_guard<py::gil_scoped_release>());
    m.def("keep8", &keep8, py::call_guard<py::gil_scoped_release>());
    m.def("restore8", &restore8, py::call_guard<py::gil_scoped_release>());
    m.def("gelu_keep8", &gelu_keep8, py::call_guard<py::gil_scoped_release>());
    m.def("mlp_keep8", &mlp_keep8, py::call_guard<py::gil_scoped_release>());
    m.def("linear_xent", &linear_xent, py::call_guard<py::gil_scoped_release>());
    m.def("layer_norm_keep8", &layer_norm_keep8, py::call_guard<py::gil_scoped_release>());
}
