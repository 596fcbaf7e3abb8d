// torch bindings of the 4-bit floating point linear layer and the affine layer norm: turing_utils::*
// operators over the C ABI (include/ctu_b200.h), with their argument checks, outputs and gradients.
//
// A single token's call takes 2 to 6 us on the GPU, so what a caller waits for is the host: these ops
// are registered from C++.  torch supplies memory, streams, device guards and the autograd graph; all
// arithmetic is behind the C ABI.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <cmath>
#include <initializer_list>
#include <optional>
#include <string>
#include <tuple>

#include "../../include/ctu_b200.h"

// The torch build that this library fits, read from the file before it is loaded.
extern "C" __attribute__((visibility("default"), used)) const char ctu_built_for_torch[] =
    "ctu-built-for-torch=" CTU_BUILT_FOR_TORCH;

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using Three = std::tuple<Tensor, Tensor, Tensor>;

void check(int rc) { TORCH_CHECK(rc == CTU_OK, ctu_last_error()); }

void *stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// The C ABI wants dense, 16-byte aligned tensors; the rare other one is copied.
Tensor dense(const Tensor &t) {
    Tensor c = t.contiguous();
    if (reinterpret_cast<uintptr_t>(c.const_data_ptr()) & 15u) c = c.clone(at::MemoryFormat::Contiguous);
    return c;
}

int norm_dtype(at::ScalarType t, const char *what) {
    switch (t) {
    case at::kBFloat16: return CTU_DTYPE_BF16;
    case at::kHalf: return CTU_DTYPE_FP16;
    case at::kFloat: return CTU_DTYPE_FP32;
    default: TORCH_CHECK(false, what, " must be float16, bfloat16, or float32");
    }
}

// ---------------------------------------------------------------------------- 4-bit floating point
// The block scales' dtype names the format: float8_e4m3fn is nvfp4 (blocks of 16), float8_e8m0fnu mxfp4
// (blocks of 32).
struct Operand {
    Tensor codes, scales;
    int64_t rows, k;
    int format;
};

int64_t block_of(int format) { return format == CTU_FP4_NVFP4 ? 16 : 32; }

Operand operand(const Tensor &codes, const Tensor &scales, const char *name) {
    TORCH_CHECK(codes.is_cuda() && codes.dim() == 2 && codes.scalar_type() == at::kByte, name,
                " must be a 2D uint8 CUDA tensor of packed FP4 codes");
    const at::ScalarType type = scales.scalar_type();
    TORCH_CHECK(type == at::kFloat8_e4m3fn || type == at::kFloat8_e8m0fnu, name,
                " block scales must be float8_e4m3fn (nvfp4) or float8_e8m0fnu (mxfp4)");
    Operand o;
    o.format = type == at::kFloat8_e4m3fn ? CTU_FP4_NVFP4 : CTU_FP4_MXFP4;
    o.rows = codes.size(0);
    o.k = 2 * codes.size(1);
    TORCH_CHECK(o.k > 0 && o.k % 32 == 0, name, " width must be positive and divisible by 32");
    const int64_t mt = (o.rows + 127) / 128, kt = (o.k / block_of(o.format) + 3) / 4;
    TORCH_CHECK(scales.device() == codes.device() && scales.sizes() == at::IntArrayRef({mt, kt, 32, 16}), name,
                " block scales must be [", mt, ", ", kt, ", 32, 16] tiles on the same device");
    o.codes = dense(codes);
    o.scales = dense(scales);
    return o;
}

Tensor vector(const Tensor &t, int64_t count, const c10::Device &device, const char *name, bool scalar) {
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.device() == device && (t.numel() == count || (scalar && t.numel() == 1)),
                name, " must be float32 on the same device, ", count, " values", scalar ? " or one" : "");
    TORCH_CHECK(!t.requires_grad() || !at::GradMode::is_enabled(), name, " has no gradient here: detach it");
    return t.contiguous();
}

const uint8_t *bytes(const Tensor &t) { return static_cast<const uint8_t *>(t.const_data_ptr()); }

Three fp4_quantize(const Tensor &input, c10::string_view format, int64_t rotation) {
    TORCH_CHECK(format == "nvfp4" || format == "mxfp4", "FP4 format must be 'nvfp4' or 'mxfp4'");
    const int fmt = format == "nvfp4" ? CTU_FP4_NVFP4 : CTU_FP4_MXFP4;
    TORCH_CHECK(input.is_cuda() && input.dim() == 2, "FP4 quantizer input must be a 2D CUDA tensor");
    const at::ScalarType type = input.scalar_type();
    TORCH_CHECK(type == at::kBFloat16 || type == at::kHalf, "FP4 quantizer input must be float16 or bfloat16");
    TORCH_CHECK(rotation == 0 || rotation == 256, "FP4 quantizer rotation must be 0 or 256");
    const int64_t rows = input.size(0), k = input.size(1), step = rotation ? rotation : 32;
    TORCH_CHECK(k > 0 && k % step == 0, "FP4 quantizer width must be positive and divisible by ", step);
    const c10::cuda::CUDAGuard guard(input.device());
    const Tensor x = dense(input);
    Tensor codes = at::empty({rows, k / 2}, x.options().dtype(at::kByte));
    Tensor scales = at::empty({(rows + 127) / 128, (k / block_of(fmt) + 3) / 4, 32, 16},
                              x.options().dtype(fmt == CTU_FP4_NVFP4 ? at::kFloat8_e4m3fn : at::kFloat8_e8m0fnu));
    Tensor row = at::empty({rows, 1}, x.options().dtype(at::kFloat));
    check(ctu_fp4_quantize(x.const_data_ptr(), rows, k, norm_dtype(type, "FP4 quantizer input"), fmt,
                           static_cast<int>(rotation), codes.data_ptr<uint8_t>(), static_cast<uint8_t *>(scales.data_ptr()),
                           row.data_ptr<float>(), stream_of(x)));
    return {codes, scales, row};
}

Tensor fp4_dequantize(const Tensor &codes, const Tensor &block_scale, const Tensor &scale, at::ScalarType out_dtype) {
    const Operand o = operand(codes, block_scale, "codes");
    const int dtype = norm_dtype(out_dtype, "FP4 dequantizer output");
    const Tensor s = vector(scale, o.rows, codes.device(), "row scale", true);
    const c10::cuda::CUDAGuard guard(codes.device());
    Tensor out = at::empty({o.rows, o.k}, codes.options().dtype(out_dtype));
    check(ctu_fp4_dequantize(bytes(o.codes), bytes(o.scales), s.const_data_ptr<float>(), s.numel(), o.rows, o.k, o.format,
                             dtype, out.data_ptr(), stream_of(codes)));
    return out;
}

Tensor fp4_linear(const Tensor &activation, const Tensor &weight, const Tensor &activation_block_scale,
                  const Tensor &weight_block_scale, const Tensor &activation_scale, const Tensor &weight_scale,
                  const OptTensor &bias) {
    const Operand a = operand(activation, activation_block_scale, "activation");
    const Operand w = operand(weight, weight_block_scale, "weight");
    const c10::Device device = activation.device();
    TORCH_CHECK(weight.device() == device, "all FP4 linear tensors must use the same CUDA device");
    TORCH_CHECK(w.k == a.k && w.format == a.format, "activation and weight must have the same K and the same FP4 format");
    const Tensor a_s = vector(activation_scale, a.rows, device, "activation scale", false);
    const Tensor w_s = vector(weight_scale, w.rows, device, "weight scale", true);
    Tensor b;
    if (bias.has_value()) b = vector(*bias, w.rows, device, "bias", false);
    const c10::cuda::CUDAGuard guard(device);
    Tensor out = at::empty({a.rows, w.rows}, activation.options().dtype(at::kBFloat16));
    check(ctu_fp4_linear(bytes(a.codes), bytes(w.codes), bytes(a.scales), bytes(w.scales), a_s.const_data_ptr<float>(),
                         w_s.const_data_ptr<float>(), w_s.numel(), b.defined() ? b.const_data_ptr<float>() : nullptr,
                         out.data_ptr(), a.rows, w.rows, a.k, a.format, stream_of(activation)));
    return out;
}

Tensor fp4_linear_grad_input(const Tensor &grad_output, const Tensor &weight, const Tensor &weight_block_scale,
                             const Tensor &weight_scale, int64_t rotation) {
    const Operand w = operand(weight, weight_block_scale, "weight");
    const c10::Device device = weight.device();
    TORCH_CHECK(grad_output.device() == device && grad_output.scalar_type() == at::kBFloat16 && grad_output.dim() == 2,
                "grad_output must be a 2D bfloat16 tensor on the weight's device");
    TORCH_CHECK(grad_output.size(1) == w.rows, "grad_output must be [M, N] with the weight's N");
    TORCH_CHECK(w.rows > 0 && w.rows % 8 == 0, "FP4 linear gradient requires N divisible by 8");
    TORCH_CHECK((rotation == 0 || rotation == 256) && w.k % (rotation ? rotation : 32) == 0,
                "FP4 linear gradient rotation must be 0, or 256 with K divisible by it");
    const Tensor w_s = vector(weight_scale, w.rows, device, "weight scale", true);
    const c10::cuda::CUDAGuard guard(device);
    const Tensor g = dense(grad_output);
    const int64_t m = g.size(0);
    Tensor dx = at::empty({m, w.k}, g.options());
    if (m == 0) return dx;
    Tensor workspace = at::empty({ctu_fp4_grad_workspace_bytes(m, w.rows, w.k)}, weight.options());
    check(ctu_fp4_linear_grad_input(g.const_data_ptr(), bytes(w.codes), bytes(w.scales), w_s.const_data_ptr<float>(),
                                    w_s.numel(), static_cast<int>(rotation), workspace.data_ptr(), dx.data_ptr(), m, w.rows,
                                    w.k, w.format, stream_of(weight)));
    return dx;
}

Tensor convrot_fp4_linear(const Tensor &x, const Tensor &weight, const Tensor &weight_block_scale,
                          const Tensor &weight_scale, const OptTensor &bias, int64_t rotation) {
    const auto [codes, scales, row] =
        fp4_quantize(x, weight_block_scale.scalar_type() == at::kFloat8_e8m0fnu ? "mxfp4" : "nvfp4", rotation);
    return fp4_linear(codes, weight, scales, weight_block_scale, row, weight_scale, bias);
}

// ---------------------------------------------------------------------------- affine layer norm
Tensor norm_vector(const OptTensor &t, const Tensor &input, int64_t hidden, const char *name) {
    if (!t.has_value() || !t->defined()) return Tensor();
    TORCH_CHECK(t->device() == input.device() && t->dim() == 1 && t->size(0) == hidden &&
                    (t->scalar_type() == input.scalar_type() || t->scalar_type() == at::kFloat),
                "LayerNorm ", name, " must be [hidden] on the input's device, of its type or float32");
    return dense(*t);
}

struct Norm {
    int64_t hidden;
    Tensor weight, bias;
    int dtype;
    at::ScalarType weight_type;
};

Norm norm_of(const Tensor &input, const OptTensor &weight, const OptTensor &bias) {
    TORCH_CHECK(input.is_cuda() && input.dim() >= 1, "LayerNorm input must be a CUDA tensor");
    Norm n;
    n.dtype = norm_dtype(input.scalar_type(), "LayerNorm input");
    n.hidden = input.size(-1);
    TORCH_CHECK(n.hidden > 0, "LayerNorm dimensions must be positive");
    n.weight = norm_vector(weight, input, n.hidden, "weight");
    n.bias = norm_vector(bias, input, n.hidden, "bias");
    TORCH_CHECK(!n.weight.defined() || !n.bias.defined() || n.weight.scalar_type() == n.bias.scalar_type(),
                "LayerNorm weight and bias must have the same type");
    n.weight_type = n.weight.defined() ? n.weight.scalar_type() : n.bias.defined() ? n.bias.scalar_type() : input.scalar_type();
    return n;
}

const void *pointer(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }

Three layer_norm(const Tensor &input, const OptTensor &weight, const OptTensor &bias, double epsilon) {
    const Norm n = norm_of(input, weight, bias);
    TORCH_CHECK(std::isfinite(epsilon) && epsilon > 0.0, "LayerNorm epsilon must be finite and positive");
    const c10::cuda::CUDAGuard guard(input.device());
    const Tensor x = dense(input);
    const int64_t rows = x.numel() / n.hidden;
    Tensor out = at::empty(x.sizes(), x.options());
    Tensor mean = at::empty({rows}, x.options().dtype(at::kFloat));
    Tensor rstd = at::empty({rows}, x.options().dtype(at::kFloat));
    check(ctu_layer_norm(x.const_data_ptr(), pointer(n.weight), pointer(n.bias), out.data_ptr(), mean.data_ptr<float>(),
                         rstd.data_ptr<float>(), rows, n.hidden, static_cast<float>(epsilon), n.dtype,
                         norm_dtype(n.weight_type, "LayerNorm weight"), stream_of(x)));
    return {out, mean, rstd};
}

// `needs`: 1 for dx, 2 for dweight, 4 for dbias; what is not needed, or has no parameter, comes back empty.
Three layer_norm_backward(const Tensor &grad, const Tensor &input, const Tensor &mean, const Tensor &rstd,
                          const OptTensor &weight, const OptTensor &bias, int64_t needs) {
    const Norm n = norm_of(input, weight, bias);
    TORCH_CHECK(grad.sizes() == input.sizes() && grad.scalar_type() == input.scalar_type() && grad.device() == input.device(),
                "LayerNorm gradient must match the input's shape, type and device");
    const int64_t rows = input.numel() / n.hidden;
    for (const Tensor &t : {mean, rstd})
        TORCH_CHECK(t.scalar_type() == at::kFloat && t.device() == input.device() && t.numel() == rows && t.is_contiguous(),
                    "LayerNorm statistics must be contiguous float32 [rows] on the input's device");
    const c10::cuda::CUDAGuard guard(input.device());
    const Tensor x = dense(input), g = dense(grad);
    const auto params = x.options().dtype(n.weight_type);
    const bool want_w = (needs & 2) && n.weight.defined(), want_b = (needs & 4) && n.bias.defined();
    Tensor dx, dw, db, workspace;
    if (needs & 1) dx = at::empty(x.sizes(), x.options());
    if (want_w) dw = at::empty({n.hidden}, params);
    if (want_b) db = at::empty({n.hidden}, params);
    if (want_w || want_b)
        workspace = at::empty({ctu_layer_norm_backward_workspace_bytes(rows, n.hidden)}, x.options().dtype(at::kByte));
    auto out = [](const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; };
    check(ctu_layer_norm_backward(g.const_data_ptr(), x.const_data_ptr(), pointer(n.weight), mean.const_data_ptr<float>(),
                                  rstd.const_data_ptr<float>(), out(dx), out(dw), out(db), out(workspace), rows, n.hidden,
                                  n.dtype, norm_dtype(n.weight_type, "LayerNorm weight"), stream_of(x)));
    for (Tensor *t : {&dx, &dw, &db})
        if (!t->defined()) *t = at::empty({0}, x.options());
    return {dx, dw, db};
}

// ---------------------------------------------------------------------------- gradients
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wants_grad(const OptTensor &t) { return t.has_value() && t->defined() && t->requires_grad(); }

void no_second_derivative(const char *what) {
    TORCH_CHECK(!at::GradMode::is_enabled(), what, " has no second derivative");  // create_graph=True
}

// A tangent would be lost below the autograd keys, and read as zero by whoever asks for it.
void no_forward_mode(const char *what, std::initializer_list<OptTensor> inputs) {
    for (const OptTensor &t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t.has_value() || !t->defined() || !t->_fw_grad(/*level=*/0).defined(), what,
                                    " has no forward-mode derivative");
}

struct LayerNormGrad : torch::autograd::Function<LayerNormGrad> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const OptTensor &weight, const OptTensor &bias,
                                 double epsilon) {
        static const auto op = c10::Dispatcher::singleton()
                                   .findSchemaOrThrow("turing_utils::layer_norm", "")
                                   .typed<Three(const Tensor &, const OptTensor &, const OptTensor &, double)>();
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, mean, rstd] = op.call(x, weight, bias, epsilon);
        ctx->save_for_backward({x, mean, rstd, weight.value_or(Tensor()), bias.value_or(Tensor())});
        ctx->saved_data["needs"] = static_cast<int64_t>(x.requires_grad()) + 2 * static_cast<int64_t>(wants_grad(weight)) +
                                   4 * static_cast<int64_t>(wants_grad(bias));
        ctx->mark_non_differentiable({mean, rstd});
        ctx->set_materialize_grads(false);
        return {y, mean, rstd};
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        no_second_derivative("LayerNorm");
        no_forward_mode("the LayerNorm gradient", {grads[0]});
        static const auto op = c10::Dispatcher::singleton()
                                   .findSchemaOrThrow("turing_utils::layer_norm_backward", "")
                                   .typed<Three(const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                                const OptTensor &, const OptTensor &, int64_t)>();
        const variable_list saved = ctx->get_saved_variables();
        const int64_t needs = ctx->saved_data["needs"].toInt();
        auto maybe = [](const Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); };
        at::AutoDispatchBelowADInplaceOrView below;
        auto [dx, dw, db] = op.call(grads[0], saved[0], saved[1], saved[2], maybe(saved[3]), maybe(saved[4]), needs);
        return {needs & 1 ? dx : Tensor(), needs & 2 ? dw : Tensor(), needs & 4 ? db : Tensor(), Tensor()};
    }
};

Three layer_norm_autograd(const Tensor &x, const OptTensor &weight, const OptTensor &bias, double epsilon) {
    no_forward_mode("LayerNorm", {x, weight, bias});
    if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(weight) || wants_grad(bias))) {
        const variable_list out = LayerNormGrad::apply(x, weight, bias, epsilon);
        return {out[0], out[1], out[2]};
    }
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("turing_utils::layer_norm", "")
                               .typed<Three(const Tensor &, const OptTensor &, const OptTensor &, double)>();
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(x, weight, bias, epsilon);
}

struct LinearGrad : torch::autograd::Function<LinearGrad> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const Tensor &weight_block_scale,
                          const Tensor &weight_scale, const OptTensor &bias, int64_t rotation) {
        static const auto op = c10::Dispatcher::singleton()
                                   .findSchemaOrThrow("turing_utils::convrot_fp4_linear", "")
                                   .typed<Tensor(const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                                 const OptTensor &, int64_t)>();
        TORCH_CHECK(!weight_scale.requires_grad() && !wants_grad(bias),
                    "the FP4 linear's weight scale and bias are frozen: detach them");
        TORCH_CHECK(x.scalar_type() == at::kBFloat16 && weight.size(0) % 8 == 0,
                    "the FP4 linear's gradient takes bfloat16 input and N divisible by 8");
        ctx->save_for_backward({weight, weight_block_scale, weight_scale});
        ctx->saved_data["rotation"] = rotation;
        at::AutoDispatchBelowADInplaceOrView below;
        return op.call(x, weight, weight_block_scale, weight_scale, bias, rotation);
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        no_second_derivative("the FP4 linear");
        no_forward_mode("the FP4 linear's gradient", {grads[0]});
        static const auto op =
            c10::Dispatcher::singleton()
                .findSchemaOrThrow("turing_utils::fp4_linear_grad_input", "")
                .typed<Tensor(const Tensor &, const Tensor &, const Tensor &, const Tensor &, int64_t)>();
        const variable_list saved = ctx->get_saved_variables();
        at::AutoDispatchBelowADInplaceOrView below;
        return {op.call(grads[0], saved[0], saved[1], saved[2], ctx->saved_data["rotation"].toInt()), Tensor(), Tensor(),
                Tensor(), Tensor(), Tensor()};
    }
};

Tensor convrot_fp4_linear_autograd(const Tensor &x, const Tensor &weight, const Tensor &weight_block_scale,
                                   const Tensor &weight_scale, const OptTensor &bias, int64_t rotation) {
    no_forward_mode("the FP4 linear", {x, weight_scale, bias});
    if (at::GradMode::is_enabled() && (x.requires_grad() || weight_scale.requires_grad() || wants_grad(bias)))
        return LinearGrad::apply(x, weight, weight_block_scale, weight_scale, bias, rotation);
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("turing_utils::convrot_fp4_linear", "")
                               .typed<Tensor(const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                             const OptTensor &, int64_t)>();
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(x, weight, weight_block_scale, weight_scale, bias, rotation);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(turing_utils, m) {
    m.def("fp4_quantize(Tensor x, str format='nvfp4', int rotation=0) -> (Tensor, Tensor, Tensor)");
    m.def("fp4_dequantize(Tensor codes, Tensor block_scale, Tensor scale, ScalarType out_dtype=bfloat16) -> Tensor");
    m.def(
        "fp4_linear(Tensor activation, Tensor weight, Tensor activation_block_scale, Tensor weight_block_scale, "
        "Tensor activation_scale, Tensor weight_scale, Tensor? bias=None) -> Tensor");
    m.def(
        "fp4_linear_grad_input(Tensor grad_output, Tensor weight, Tensor weight_block_scale, Tensor weight_scale, "
        "int rotation=0) -> Tensor");
    m.def(
        "convrot_fp4_linear(Tensor x, Tensor weight, Tensor weight_block_scale, Tensor weight_scale, "
        "Tensor? bias=None, int rotation=256) -> Tensor");
    m.def("layer_norm(Tensor x, Tensor? weight=None, Tensor? bias=None, float epsilon=1e-5) -> (Tensor, Tensor, Tensor)");
    m.def(
        "layer_norm_backward(Tensor grad, Tensor x, Tensor mean, Tensor rstd, Tensor? weight=None, Tensor? bias=None, "
        "int needs=7) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(turing_utils, CompositeExplicitAutograd, m) {
    m.impl("fp4_quantize", TORCH_FN(fp4_quantize));
    m.impl("fp4_dequantize", TORCH_FN(fp4_dequantize));
    m.impl("fp4_linear", TORCH_FN(fp4_linear));
    m.impl("fp4_linear_grad_input", TORCH_FN(fp4_linear_grad_input));
    m.impl("convrot_fp4_linear", TORCH_FN(convrot_fp4_linear));
    m.impl("layer_norm", TORCH_FN(layer_norm));
    m.impl("layer_norm_backward", TORCH_FN(layer_norm_backward));
}

TORCH_LIBRARY_IMPL(turing_utils, Autograd, m) {
    m.impl("convrot_fp4_linear", TORCH_FN(convrot_fp4_linear_autograd));
    m.impl("layer_norm", TORCH_FN(layer_norm_autograd));
}
