// Dispatcher ops of the training operators (crumpet_amd.training): the bias by
// buckets, the window attention, the residual sum with its norms and the
// linear layer with an 8-bit copy of its input.
//
// Each operator is three ops: the one that users call, with its gradient
// registered for autograd; `<op>_forward`, which also returns what the
// backward pass keeps; and `<op>_backward`.  All of them have fakes
// (crumpet_amd/_native.py), so torch.compile traces through them.  Every impl
// checks shapes, types and devices, makes what the kernels need dense and
// aligned, takes the current stream of the tensors' device and calls the C ABI
// of libcrumpet_hip.so.  Workspaces come from the caching allocator within the
// call.  Optional results that nobody asked for come back with no elements.
#include <ATen/core/Tensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <initializer_list>
#include <optional>
#include <tuple>

#include "crumpet_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

void* stream_of(const Tensor& t) {
    return static_cast<void*>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream());
}

void check_status(int status) {
    TORCH_CHECK(status == CRUMPET_OK, "crumpet_ops: ", crumpet_last_error(), " (", crumpet_status_string(status), ")");
}

int32_t code_of(const Tensor& t, const char* what, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return CRUMPET_DTYPE_F32;
        case at::kHalf: return CRUMPET_DTYPE_F16;
        case at::kBFloat16: return CRUMPET_DTYPE_BF16;
        default: TORCH_CHECK(false, what, ": ", name, " must be float32, float16 or bfloat16");
    }
}

void check_device(const Tensor& t, const Tensor& like, const char* what, const char* name) {
    TORCH_CHECK(t.device() == like.device(), what, ": ", name, " must be on ", like.device(), ", got ", t.device());
}

bool has(const Maybe& t) { return t.has_value() && t->defined(); }
void* ptr(const Tensor& t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }
float* floats(const Tensor& t) { return static_cast<float*>(ptr(t)); }

// Without a call where there is nothing to do: a few of them are a microsecond.
Tensor as_type(const Tensor& t, at::ScalarType type) { return t.scalar_type() == type ? t : t.to(type); }

// Dense and 16-byte aligned.
Tensor dense(const Tensor& t) {
    Tensor c = t.is_contiguous() ? t : t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}

// A parameter in fp32, dense; undefined where it is absent.
Tensor parameter(const Maybe& p, const Tensor& like, at::IntArrayRef shape, const char* what, const char* name) {
    if (!has(p)) return Tensor();
    check_device(*p, like, what, name);
    code_of(*p, what, name);
    TORCH_CHECK(p->sizes() == shape, what, ": ", name, " must have shape ", shape, ", got ", p->sizes());
    return dense(as_type(*p, at::kFloat));
}

void no_gradient(const Maybe& t, const char* what, const char* name) {
    TORCH_CHECK(!(at::GradMode::is_enabled() && has(t) && t->requires_grad()), what, ": ", name, " has no gradient");
}
void once_differentiable(const char* what) {
    TORCH_CHECK(!at::GradMode::is_enabled(), what, ": second derivatives are not provided (create_graph=True)");
}

bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants(const Maybe& t) { return has(t) && t->requires_grad(); }
bool any_grad(std::initializer_list<bool> wanted) {
    if (!at::GradMode::is_enabled()) return false;
    for (bool w : wanted)
        if (w) return true;
    return false;
}
Tensor asked(const Tensor& t, bool want) { return want ? t : Tensor(); }
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }

template <typename F>
auto dispatcher_op(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

// ---- bias by buckets ------------------------------------------------------------

void check_ints(const Tensor& t, const Tensor& like, const char* what, const char* name) {
    check_device(t, like, what, name);
    TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous(), what, ": ", name, " must be dense int32");
}

Tensor bucket_bias(const Tensor& table, const Tensor& index, const Tensor& order, const Tensor& segments,
                   const Maybe& firsts) {
    const char* what = "relative_position_bias";
    TORCH_CHECK(table.dim() == 2, what, ": table must have shape [buckets, heads]");
    TORCH_CHECK(index.dim() == 2, what, ": index must have shape [queries, keys]");
    check_ints(index, table, what, "index");
    const int32_t dt = code_of(table, what, "table");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(table.device());
    const Tensor t = table.contiguous();
    const int64_t pairs = index.numel();
    Tensor out = at::empty({table.size(1), index.size(0), index.size(1)}, table.options());
    if (out.numel() == 0) return out;
    TORCH_CHECK(table.size(0) > 0, what, ": the table has no rows");
    check_status(crumpet_bucket_bias(out.data_ptr(), t.data_ptr(), dt, index.data_ptr<int32_t>(), t.size(0), t.size(1),
                                     pairs, stream_of(t)));
    return out;
}

Tensor bucket_bias_backward(const Tensor& grad, const Tensor& order, const Tensor& segments, const Maybe& firsts,
                            int64_t buckets) {
    const char* what = "relative_position_bias";
    TORCH_CHECK(grad.dim() == 3, what, ": the gradient must have shape [heads, queries, keys]");
    const int32_t dt = code_of(grad, what, "the gradient");
    check_ints(order, grad, what, "order");
    check_ints(segments, grad, what, "segments");
    TORCH_CHECK(segments.dim() == 2 && segments.size(1) == 2, what, ": segments must have shape [n, 2]");
    const int64_t heads = grad.size(0), pairs = grad.size(1) * grad.size(2), n = segments.size(0);
    TORCH_CHECK(order.numel() == pairs, what, ": order must hold every pair");
    if (has(firsts)) {
        check_ints(*firsts, grad, what, "firsts");
        TORCH_CHECK(firsts->numel() == buckets + 1, what, ": firsts must hold buckets + 1 numbers");
    }
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(grad.device());
    const Tensor g = grad.contiguous();
    Tensor out = at::empty({buckets, heads}, grad.options());
    if (out.numel() == 0) return out;
    Tensor partial;
    if (has(firsts)) partial = at::empty({std::max<int64_t>(1, n) * heads}, grad.options().dtype(at::kFloat));
    check_status(crumpet_bucket_bias_backward(out.data_ptr(), ptr(g), dt, buckets, heads, pairs,
                                              static_cast<const int32_t*>(ptr(order)), segments.data_ptr<int32_t>(), n,
                                              has(firsts) ? firsts->data_ptr<int32_t>() : nullptr, ptr(partial),
                                              stream_of(g)));
    return out;
}

struct BucketBias : torch::autograd::Function<BucketBias> {
    static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& index, const Tensor& order,
                          const Tensor& segments, const Maybe& firsts) {
        ctx->save_for_backward({order, segments, has(firsts) ? *firsts : Tensor()});
        ctx->saved_data["buckets"] = table.size(0);
        at::AutoDispatchBelowADInplaceOrView below;
        static const auto op = dispatcher_op<decltype(bucket_bias)>("crumpet_ops::bucket_bias");
        return op.call(table, index, order, segments, firsts);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once_differentiable("relative_position_bias");
        const auto saved = ctx->get_saved_variables();
        static const auto op = dispatcher_op<decltype(bucket_bias_backward)>("crumpet_ops::bucket_bias_backward");
        return {op.call(grads[0], saved[0], saved[1], maybe(saved[2]), ctx->saved_data["buckets"].toInt()), Tensor(),
                Tensor(), Tensor(), Tensor()};
    }
};

Tensor bucket_bias_autograd(const Tensor& table, const Tensor& index, const Tensor& order, const Tensor& segments,
                            const Maybe& firsts) {
    if (any_grad({wants(table)})) return BucketBias::apply(table, index, order, segments, firsts);
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = dispatcher_op<decltype(bucket_bias)>("crumpet_ops::bucket_bias");
    return op.call(table, index, order, segments, firsts);
}

// ---- window attention -----------------------------------------------------------

struct Attention {
    Tensor qkv, bias, mask;
    int64_t strides[2], B, N, C, D;
    int32_t dtype, mask_dtype = 0;
    int64_t mask_batch = 0, mask_stride = 0;
    const int64_t* region = nullptr;
};

Attention attention_of(const Tensor& qkv, const Tensor& bias, int64_t heads, const Maybe& mask, at::IntArrayRef region,
                       const char* what) {
    Attention a;
    TORCH_CHECK(qkv.dim() == 3, what, ": qkv must have shape [windows, tokens, 3 heads head_dim]");
    a.dtype = code_of(qkv, what, "qkv");
    TORCH_CHECK(heads > 0 && qkv.size(2) % (3 * heads) == 0, what, ": qkv's last axis must be 3 heads head_dim, got ",
                qkv.size(2), " for ", heads, " heads");
    a.B = qkv.size(0), a.N = qkv.size(1), a.C = qkv.size(2) / 3, a.D = a.C / heads;
    // window and token strides of 16 bytes and unit channel stride are read in place
    const int64_t align = 16 / qkv.element_size();
    const bool in_place = qkv.stride(2) == 1 && qkv.stride(0) % align == 0 && qkv.stride(1) % align == 0 &&
                          reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 == 0;
    a.qkv = in_place ? qkv : dense(qkv);
    a.strides[0] = a.qkv.stride(0), a.strides[1] = a.qkv.stride(1);
    check_device(bias, qkv, what, "bias");
    code_of(bias, what, "bias");
    TORCH_CHECK(bias.dim() == 3 && bias.size(0) == heads && bias.size(1) == a.N && bias.size(2) == a.N, what,
                ": bias must have shape [", heads, ", ", a.N, ", ", a.N, "], got ", bias.sizes());
    a.bias = dense(bias.to(at::kFloat));
    if (has(mask)) {
        check_device(*mask, qkv, what, "mask");
        a.mask_dtype = code_of(*mask, what, "mask");
        TORCH_CHECK(mask->dim() == 3 && mask->size(1) == a.N && mask->size(2) == a.N, what,
                    ": mask must have shape [masks, ", a.N, ", ", a.N, "], got ", mask->sizes());
        TORCH_CHECK(mask->size(0) > 0 || a.B == 0, what, ": mask holds no window");
        a.mask = mask->stride(2) == 1 && mask->stride(1) == a.N ? *mask : mask->contiguous();
        a.mask_batch = a.mask.size(0), a.mask_stride = a.mask.stride(0);
    }
    TORCH_CHECK(region.empty() || region.size() == 9, what, ": region takes nine numbers");
    if (!region.empty()) a.region = region.data();
    return a;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> attention_forward(const Tensor& qkv, const Tensor& bias, int64_t heads,
                                                             const Maybe& mask, at::IntArrayRef region, double scale,
                                                             bool keep) {
    const char* what = "window_attention";
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(qkv.device());
    const Attention a = attention_of(qkv, bias, heads, mask, region, what);
    const auto f32 = qkv.options().dtype(at::kFloat);
    const bool rest = keep && a.dtype != CRUMPET_DTYPE_F32;
    Tensor out = at::empty({a.B, a.N, a.C}, qkv.options());
    Tensor out_rest = rest ? at::empty({a.B, a.N, a.C}, qkv.options()) : at::empty({0}, qkv.options());
    const int64_t rows = keep ? a.B * heads * a.N : 0;
    Tensor row_max = at::empty({rows}, f32), row_inv = at::empty({rows}, f32);
    // with no rows the arguments are checked all the same
    check_status(crumpet_window_attention(ptr(out), ptr(out_rest), floats(row_max), floats(row_inv), ptr(a.qkv),
                                          a.strides, a.dtype, a.B, heads, a.N, a.D, floats(a.bias), ptr(a.mask),
                                          a.mask_dtype, a.mask_batch, a.mask_stride, a.region,
                                          static_cast<float>(scale), stream_of(qkv)));
    return {out, out_rest, row_max, row_inv};
}

Tensor window_attention(const Tensor& qkv, const Tensor& bias, int64_t heads, const Maybe& mask, at::IntArrayRef region,
                        double scale) {
    return std::get<0>(attention_forward(qkv, bias, heads, mask, region, scale, false));
}

std::tuple<Tensor, Tensor, Tensor, Tensor> window_attention_forward(const Tensor& qkv, const Tensor& bias,
                                                                    int64_t heads, const Maybe& mask,
                                                                    at::IntArrayRef region, double scale) {
    return attention_forward(qkv, bias, heads, mask, region, scale, true);
}

std::tuple<Tensor, Tensor> window_attention_backward(const Tensor& grad, const Tensor& qkv, const Tensor& bias,
                                                     int64_t heads, const Maybe& mask, at::IntArrayRef region,
                                                     double scale, const Tensor& out, const Tensor& out_rest,
                                                     const Tensor& row_max, const Tensor& row_inv, bool want_bias) {
    const char* what = "window_attention";
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(qkv.device());
    const Attention a = attention_of(qkv, bias, heads, mask, region, what);
    const auto f32 = qkv.options().dtype(at::kFloat);
    check_device(grad, qkv, what, "the gradient");
    const int64_t rows = a.B * heads * a.N;
    TORCH_CHECK(grad.sizes() == at::IntArrayRef({a.B, a.N, a.C}) && grad.scalar_type() == qkv.scalar_type(), what,
                ": the gradient must be like the output");
    TORCH_CHECK(out.sizes() == grad.sizes() && out.scalar_type() == qkv.scalar_type() && out.is_contiguous() &&
                    (a.dtype == CRUMPET_DTYPE_F32 ||
                     (out_rest.sizes() == grad.sizes() && out_rest.scalar_type() == qkv.scalar_type() &&
                      out_rest.is_contiguous())) &&
                    row_max.numel() == rows && row_inv.numel() == rows && row_max.scalar_type() == at::kFloat &&
                    row_inv.scalar_type() == at::kFloat && row_max.is_contiguous() && row_inv.is_contiguous(),
                what, ": the kept tensors are not those of the forward pass");
    for (const Tensor* t : {&out, &out_rest, &row_max, &row_inv}) check_device(*t, qkv, what, "a kept tensor");
    Tensor dqkv = at::empty({a.B, a.N, 3 * a.C}, qkv.options());
    Tensor dbias = want_bias ? (rows == 0 ? at::zeros({heads, a.N, a.N}, f32) : at::empty({heads, a.N, a.N}, f32))
                             : at::empty({0}, f32);
    if (rows > 0) {
        const Tensor g = dense(grad);
        const Tensor work = at::empty({crumpet_window_attention_workspace(a.B, heads, a.N)},
                                      qkv.options().dtype(at::kByte));
        check_status(crumpet_window_attention_backward(
            ptr(dqkv), want_bias ? floats(dbias) : nullptr, ptr(g), ptr(out), ptr(out_rest), floats(row_max),
            floats(row_inv), ptr(a.qkv), a.strides, a.dtype, a.B, heads, a.N, a.D, floats(a.bias), ptr(a.mask),
            a.mask_dtype, a.mask_batch, a.mask_stride, a.region, static_cast<float>(scale), ptr(work),
            stream_of(qkv)));
    }
    return {dqkv, dbias.to(bias.scalar_type())};
}

struct WindowAttention : torch::autograd::Function<WindowAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& qkv, const Tensor& bias, int64_t heads, const Maybe& mask,
                          at::IntArrayRef region, double scale) {
        at::AutoDispatchBelowADInplaceOrView below;
        static const auto op = dispatcher_op<decltype(window_attention_forward)>("crumpet_ops::window_attention_forward");
        const auto [out, rest, row_max, row_inv] = op.call(qkv, bias, heads, mask, region, scale);
        ctx->save_for_backward({qkv, bias, has(mask) ? *mask : Tensor(), out, rest, row_max, row_inv});
        ctx->saved_data["heads"] = heads;
        ctx->saved_data["region"] = region.vec();
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["bias"] = wants(bias);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once_differentiable("window_attention");
        const auto s = ctx->get_saved_variables();
        const bool want = ctx->saved_data["bias"].toBool();
        static const auto op = dispatcher_op<decltype(window_attention_backward)>("crumpet_ops::window_attention_backward");
        const auto [dqkv, dbias] =
            op.call(grads[0], s[0], s[1], ctx->saved_data["heads"].toInt(), maybe(s[2]),
                    ctx->saved_data["region"].toIntVector(), ctx->saved_data["scale"].toDouble(), s[3], s[4], s[5],
                    s[6], want);
        return {dqkv, asked(dbias, want), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor window_attention_autograd(const Tensor& qkv, const Tensor& bias, int64_t heads, const Maybe& mask,
                                 at::IntArrayRef region, double scale) {
    no_gradient(mask, "window_attention", "mask");
    if (any_grad({wants(qkv), wants(bias)})) return WindowAttention::apply(qkv, bias, heads, mask, region, scale);
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = dispatcher_op<decltype(window_attention)>("crumpet_ops::window_attention");
    return op.call(qkv, bias, heads, mask, region, scale);
}

// ---- residual sum and norms -------------------------------------------------------

struct Norm {
    Tensor x, y, post_weight, post_bias, gate, scale, weight, bias;
    int64_t samples = 1, tokens, C;
    int32_t x_dtype, dtype;
    bool per_sample = false;
};

Norm norm_of(const Tensor& x, const Tensor& y, bool post, const Maybe& post_weight, const Maybe& post_bias,
             const Maybe& gate, const Maybe& scale, const Maybe& weight, const Maybe& bias, const char* what) {
    Norm a;
    TORCH_CHECK(x.dim() >= 1, what, ": x must have a channel axis");
    check_device(y, x, what, "y");
    TORCH_CHECK(x.sizes() == y.sizes(), what, ": x and y must have one shape, got ", x.sizes(), " and ", y.sizes());
    a.x_dtype = code_of(x, what, "x"), a.dtype = code_of(y, what, "y");
    TORCH_CHECK(a.x_dtype == a.dtype || a.x_dtype == CRUMPET_DTYPE_F32, what, ": x must be float32 or of y's type");
    TORCH_CHECK(post || !(has(post_weight) || has(post_bias)), what, ": post_weight and post_bias need post=True");
    a.C = x.size(-1);
    a.per_sample = has(gate) && gate->dim() == 2;
    if (a.per_sample || has(scale)) {
        TORCH_CHECK(x.dim() >= 2, what, ": x must have shape [samples, ..., channels]");
        a.samples = x.size(0);
    }
    a.tokens = a.samples * a.C > 0 ? x.numel() / (a.samples * a.C) : 0;
    a.x = dense(x), a.y = dense(y);
    a.post_weight = parameter(post_weight, x, {a.C}, what, "post_weight");
    a.post_bias = parameter(post_bias, x, {a.C}, what, "post_bias");
    a.gate = a.per_sample ? parameter(gate, x, {a.samples, a.C}, what, "gate") : parameter(gate, x, {a.C}, what, "gate");
    a.scale = parameter(scale, x, {a.samples}, what, "scale");
    a.weight = parameter(weight, x, {a.C}, what, "weight");
    a.bias = parameter(bias, x, {a.C}, what, "bias");
    return a;
}

std::tuple<Tensor, Tensor> residual_norm(const Tensor& x, const Tensor& y, int64_t norm, bool post,
                                         const Maybe& post_weight, const Maybe& post_bias, const Maybe& gate,
                                         const Maybe& scale, const Maybe& weight, const Maybe& bias, double eps) {
    const char* what = "residual_norm";
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const Norm a = norm_of(x, y, post, post_weight, post_bias, gate, scale, weight, bias, what);
    Tensor sum = at::empty(x.sizes(), x.options()), out = at::empty(y.sizes(), y.options());
    if (x.numel() == 0) return {sum, out};
    check_status(crumpet_residual_norm(ptr(sum), ptr(out), ptr(a.x), a.x_dtype, ptr(a.y), a.dtype, a.samples, a.tokens,
                                       a.C, static_cast<int32_t>(norm), post, floats(a.post_weight), floats(a.post_bias),
                                       floats(a.gate), a.per_sample, floats(a.scale), floats(a.weight), floats(a.bias),
                                       static_cast<float>(eps), stream_of(x)));
    return {sum, out};
}

// want: bits for weight, bias, gate, post_weight, post_bias
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> residual_norm_backward(
    const Maybe& grad_sum, const Maybe& grad_out, const Tensor& x, const Tensor& y, int64_t norm, bool post,
    const Maybe& post_weight, const Maybe& post_bias, const Maybe& gate, const Maybe& scale, const Maybe& weight,
    const Maybe& bias, double eps, int64_t want) {
    const char* what = "residual_norm";
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const Norm a = norm_of(x, y, post, post_weight, post_bias, gate, scale, weight, bias, what);
    const auto f32 = x.options().dtype(at::kFloat);
    const Maybe* params[5] = {&weight, &bias, &gate, &post_weight, &post_bias};
    Tensor grads[5];
    bool any = false;
    for (int i = 0; i < 5; ++i) {
        const bool w = (want >> i & 1) != 0 && has(*params[i]);
        any = any || w;
        grads[i] = !w ? at::empty({0}, f32) : x.numel() == 0 ? at::zeros((*params[i])->sizes(), f32)
                                                             : at::empty((*params[i])->sizes(), f32);
    }
    Tensor dx = at::empty(x.sizes(), x.options()), dy = at::empty(y.sizes(), y.options());
    if (x.numel() > 0) {
        Tensor gs, go;
        if (has(grad_sum)) {
            TORCH_CHECK(grad_sum->sizes() == x.sizes() && grad_sum->scalar_type() == x.scalar_type(), what,
                        ": the sum's gradient must be like x");
            check_device(*grad_sum, x, what, "the sum's gradient");
            gs = dense(*grad_sum);
        }
        if (has(grad_out)) {
            TORCH_CHECK(grad_out->sizes() == y.sizes() && grad_out->scalar_type() == y.scalar_type(), what,
                        ": the normed gradient must be like y");
            check_device(*grad_out, x, what, "the normed gradient");
            go = dense(*grad_out);
        }
        Tensor work;
        if (any)
            work = at::empty({crumpet_residual_norm_workspace(a.samples, a.tokens, a.C)}, x.options().dtype(at::kByte));
        check_status(crumpet_residual_norm_backward(
            ptr(dx), ptr(dy), floats(grads[0]), floats(grads[1]), floats(grads[2]), floats(grads[3]), floats(grads[4]),
            ptr(gs), ptr(go), ptr(a.x), a.x_dtype, ptr(a.y), a.dtype, a.samples, a.tokens, a.C,
            static_cast<int32_t>(norm), post, floats(a.post_weight), floats(a.post_bias), floats(a.gate), a.per_sample,
            floats(a.scale), floats(a.weight), static_cast<float>(eps), ptr(work), stream_of(x)));
    }
    for (int i = 0; i < 5; ++i)
        if (has(*params[i])) grads[i] = as_type(grads[i], (*params[i])->scalar_type());
    return {dx, dy, grads[0], grads[1], grads[2], grads[3], grads[4]};
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& y, int64_t norm, bool post,
                                 const Maybe& post_weight, const Maybe& post_bias, const Maybe& gate,
                                 const Maybe& scale, const Maybe& weight, const Maybe& bias, double eps) {
        at::AutoDispatchBelowADInplaceOrView below;
        static const auto op = dispatcher_op<decltype(residual_norm)>("crumpet_ops::residual_norm");
        const auto [sum, out] = op.call(x, y, norm, post, post_weight, post_bias, gate, scale, weight, bias, eps);
        variable_list kept = {x, y};
        for (const Maybe* p : {&post_weight, &post_bias, &gate, &scale, &weight, &bias})
            kept.push_back(has(*p) ? **p : Tensor());
        ctx->save_for_backward(kept);
        ctx->set_materialize_grads(false);
        ctx->saved_data["norm"] = norm;
        ctx->saved_data["post"] = post;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["want"] = static_cast<int64_t>(wants(weight)) | static_cast<int64_t>(wants(bias)) << 1 |
                                  static_cast<int64_t>(wants(gate)) << 2 | static_cast<int64_t>(wants(post_weight)) << 3 |
                                  static_cast<int64_t>(wants(post_bias)) << 4;
        return {sum, out};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once_differentiable("residual_norm");
        const auto s = ctx->get_saved_variables();
        const int64_t want = ctx->saved_data["want"].toInt();
        static const auto op = dispatcher_op<decltype(residual_norm_backward)>("crumpet_ops::residual_norm_backward");
        const auto [dx, dy, dw, db, dgate, dpw, dpb] =
            op.call(maybe(grads[0]), maybe(grads[1]), s[0], s[1], ctx->saved_data["norm"].toInt(),
                    ctx->saved_data["post"].toBool(), maybe(s[2]), maybe(s[3]), maybe(s[4]), maybe(s[5]), maybe(s[6]),
                    maybe(s[7]), ctx->saved_data["eps"].toDouble(), want);
        return {dx,       dy,       Tensor(), Tensor(), asked(dpw, want & 8), asked(dpb, want & 16),
                asked(dgate, want & 4), Tensor(), asked(dw, want & 1), asked(db, want & 2), Tensor()};
    }
};

std::tuple<Tensor, Tensor> residual_norm_autograd(const Tensor& x, const Tensor& y, int64_t norm, bool post,
                                                  const Maybe& post_weight, const Maybe& post_bias, const Maybe& gate,
                                                  const Maybe& scale, const Maybe& weight, const Maybe& bias,
                                                  double eps) {
    no_gradient(scale, "residual_norm", "scale");
    if (any_grad({wants(x), wants(y), wants(post_weight), wants(post_bias), wants(gate), wants(weight), wants(bias)})) {
        const auto r = ResidualNorm::apply(x, y, norm, post, post_weight, post_bias, gate, scale, weight, bias, eps);
        return {r[0], r[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = dispatcher_op<decltype(residual_norm)>("crumpet_ops::residual_norm");
    return op.call(x, y, norm, post, post_weight, post_bias, gate, scale, weight, bias, eps);
}

// ---- linear with an 8-bit copy of its input -------------------------------------------

struct Linear8 {
    Tensor x, weight, bias;
    int64_t rows, K, n_out;
    int32_t dtype;
};

Linear8 linear_of(const Tensor& x, const Tensor& weight, const Maybe& bias, const char* what) {
    Linear8 a;
    TORCH_CHECK(x.dim() >= 1 && weight.dim() == 2, what, ": x must have a channel axis, weight shape [out, in]");
    a.dtype = code_of(x, what, "x");
    check_device(weight, x, what, "weight");
    a.K = x.size(-1), a.n_out = weight.size(0);
    TORCH_CHECK(weight.size(1) == a.K && weight.scalar_type() == x.scalar_type(), what,
                ": weight must have shape [out, ", a.K, "] and x's type, got ", weight.sizes(), " of ",
                weight.scalar_type());
    a.rows = a.K > 0 ? x.numel() / a.K : 0;
    a.x = dense(x), a.weight = dense(weight);
    if (has(bias)) {
        check_device(*bias, x, what, "bias");
        TORCH_CHECK(bias->dim() == 1 && bias->size(0) == a.n_out && bias->scalar_type() == x.scalar_type(), what,
                    ": bias must have shape [", a.n_out, "] and x's type");
        a.bias = dense(*bias);
    }
    return a;
}

std::tuple<Tensor, Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& weight, const Maybe& bias,
                                                  int64_t activation, bool keep) {
    const char* what = "linear_8bit";
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const Linear8 a = linear_of(x, weight, bias, what);
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = a.n_out;
    const auto bytes = x.options().dtype(at::kChar);
    Tensor y = at::empty(shape, x.options());
    Tensor codes = at::empty({keep ? a.rows : 0, a.K}, bytes);
    Tensor exps = at::empty({keep ? a.rows : 0, (a.K + 31) / 32}, bytes);
    // with no rows the arguments are checked all the same
    check_status(crumpet_linear_8bit(ptr(y), static_cast<int8_t*>(ptr(codes)), static_cast<int8_t*>(ptr(exps)),
                                     ptr(a.x), a.dtype, a.rows, a.K, ptr(a.weight), ptr(a.bias), a.n_out,
                                     static_cast<int32_t>(activation), stream_of(x)));
    return {y, codes, exps};
}

Tensor linear_8bit(const Tensor& x, const Tensor& weight, const Maybe& bias, int64_t activation) {
    return std::get<0>(linear_forward(x, weight, bias, activation, false));
}

std::tuple<Tensor, Tensor, Tensor> linear_8bit_forward(const Tensor& x, const Tensor& weight, const Maybe& bias,
                                                       int64_t activation) {
    return linear_forward(x, weight, bias, activation, true);
}

std::tuple<Tensor, Tensor, Tensor> linear_8bit_backward(const Tensor& grad, const Tensor& codes, const Tensor& exps,
                                                        const Tensor& weight, int64_t activation, bool want_x,
                                                        bool want_weight, bool want_bias) {
    const char* what = "linear_8bit";
    TORCH_CHECK(weight.dim() == 2 && grad.dim() >= 1 && codes.dim() == 2 && exps.dim() == 2, what,
                ": the kept tensors are not those of the forward pass");
    const int64_t rows = codes.size(0), K = weight.size(1), n_out = weight.size(0);
    const int32_t dt = code_of(weight, what, "weight");
    TORCH_CHECK(grad.size(-1) == n_out && grad.numel() == rows * n_out && grad.scalar_type() == weight.scalar_type(),
                what, ": the gradient must be like the output");
    TORCH_CHECK(codes.scalar_type() == at::kChar && exps.scalar_type() == at::kChar && codes.size(1) == K &&
                    exps.size(0) == rows && exps.size(1) == (K + 31) / 32 && codes.is_contiguous() &&
                    exps.is_contiguous(),
                what, ": the kept tensors are not those of the forward pass");
    for (const Tensor* t : {&codes, &exps, &weight}) check_device(*t, grad, what, "a kept tensor");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(grad.device());
    const auto opts = grad.options();
    std::vector<int64_t> shape = grad.sizes().vec();
    shape.back() = K;
    const auto made = [&](bool want, at::IntArrayRef s) {
        return !want ? at::empty({0}, opts) : rows == 0 ? at::zeros(s, opts) : at::empty(s, opts);
    };
    Tensor dx = made(want_x, shape), dw = made(want_weight, {n_out, K}), db = made(want_bias, {n_out});
    if (rows > 0 && (want_x || want_weight || want_bias)) {
        const Tensor g = dense(grad), w = dense(weight);
        const int64_t size = crumpet_linear_8bit_workspace(rows, K, n_out);
        TORCH_CHECK(size >= 0, what, ": ", crumpet_last_error());
        const Tensor work = at::empty({size}, opts.dtype(at::kByte));
        check_status(crumpet_linear_8bit_backward(
            want_x ? ptr(dx) : nullptr, want_weight ? ptr(dw) : nullptr, want_bias ? ptr(db) : nullptr, ptr(g), dt,
            static_cast<const int8_t*>(ptr(codes)), static_cast<const int8_t*>(ptr(exps)), rows, K, ptr(w), n_out,
            static_cast<int32_t>(activation), ptr(work), stream_of(grad)));
    }
    return {dx, dw, db};
}

struct Linear8bit : torch::autograd::Function<Linear8bit> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& bias,
                          int64_t activation) {
        at::AutoDispatchBelowADInplaceOrView below;
        static const auto op = dispatcher_op<decltype(linear_8bit_forward)>("crumpet_ops::linear_8bit_forward");
        const auto [y, codes, exps] = op.call(x, weight, bias, activation);
        ctx->save_for_backward({codes, exps, weight});
        ctx->saved_data["activation"] = activation;
        ctx->saved_data["x"] = wants(x);
        ctx->saved_data["weight"] = wants(weight);
        ctx->saved_data["bias"] = wants(bias);
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once_differentiable("linear_8bit");
        const auto s = ctx->get_saved_variables();
        const bool x = ctx->saved_data["x"].toBool(), w = ctx->saved_data["weight"].toBool(),
                   b = ctx->saved_data["bias"].toBool();
        static const auto op = dispatcher_op<decltype(linear_8bit_backward)>("crumpet_ops::linear_8bit_backward");
        const auto [dx, dw, db] = op.call(grads[0], s[0], s[1], s[2], ctx->saved_data["activation"].toInt(), x, w, b);
        return {asked(dx, x), asked(dw, w), asked(db, b), Tensor()};
    }
};

Tensor linear_8bit_autograd(const Tensor& x, const Tensor& weight, const Maybe& bias, int64_t activation) {
    if (any_grad({wants(x), wants(weight), wants(bias)})) return Linear8bit::apply(x, weight, bias, activation);
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = dispatcher_op<decltype(linear_8bit)>("crumpet_ops::linear_8bit");
    return op.call(x, weight, bias, activation);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(crumpet_ops, ops) {
    const std::vector<at::Tag> tags = {at::Tag::pt2_compliant_tag, at::Tag::needs_fixed_stride_order};
    ops.def("bucket_bias(Tensor table, Tensor index, Tensor order, Tensor segments, Tensor? firsts) -> Tensor", tags);
    ops.def("bucket_bias_backward(Tensor grad, Tensor order, Tensor segments, Tensor? firsts, int buckets) -> Tensor",
            tags);
    ops.def("window_attention(Tensor qkv, Tensor bias, int heads, Tensor? mask, int[] region, float scale) -> Tensor",
            tags);
    ops.def(
        "window_attention_forward(Tensor qkv, Tensor bias, int heads, Tensor? mask, int[] region, float scale) -> "
        "(Tensor, Tensor, Tensor, Tensor)",
        tags);
    ops.def(
        "window_attention_backward(Tensor grad, Tensor qkv, Tensor bias, int heads, Tensor? mask, int[] region, float "
        "scale, Tensor out, Tensor out_rest, Tensor row_max, Tensor row_inv, bool want_bias) -> (Tensor, Tensor)",
        tags);
    ops.def(
        "residual_norm(Tensor x, Tensor y, int norm, bool post, Tensor? post_weight, Tensor? post_bias, Tensor? gate, "
        "Tensor? scale, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor)",
        tags);
    ops.def(
        "residual_norm_backward(Tensor? grad_sum, Tensor? grad_out, Tensor x, Tensor y, int norm, bool post, Tensor? "
        "post_weight, Tensor? post_bias, Tensor? gate, Tensor? scale, Tensor? weight, Tensor? bias, float eps, int "
        "want) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
        tags);
    ops.def("linear_8bit(Tensor x, Tensor weight, Tensor? bias, int activation) -> Tensor", tags);
    ops.def("linear_8bit_forward(Tensor x, Tensor weight, Tensor? bias, int activation) -> (Tensor, Tensor, Tensor)",
            tags);
    ops.def(
        "linear_8bit_backward(Tensor grad, Tensor codes, Tensor exps, Tensor weight, int activation, bool want_x, bool "
        "want_weight, bool want_bias) -> (Tensor, Tensor, Tensor)",
        tags);
}

TORCH_LIBRARY_IMPL(crumpet_ops, CUDA, ops) {
    ops.impl("bucket_bias", &bucket_bias);
    ops.impl("bucket_bias_backward", &bucket_bias_backward);
    ops.impl("window_attention", &window_attention);
    ops.impl("window_attention_forward", &window_attention_forward);
    ops.impl("window_attention_backward", &window_attention_backward);
    ops.impl("residual_norm", &residual_norm);
    ops.impl("residual_norm_backward", &residual_norm_backward);
    ops.impl("linear_8bit", &linear_8bit);
    ops.impl("linear_8bit_forward", &linear_8bit_forward);
    ops.impl("linear_8bit_backward", &linear_8bit_backward);
}

TORCH_LIBRARY_IMPL(crumpet_ops, AutogradCUDA, ops) {
    ops.impl("bucket_bias", &bucket_bias_autograd);
    ops.impl("window_attention", &window_attention_autograd);
    ops.impl("residual_norm", &residual_norm_autograd);
    ops.impl("linear_8bit", &linear_8bit_autograd);
}
