// Autograd of the training operators in C++: argument checks, allocation and launch of one call cost the host some 10 us here, five times that in Python.
// The module holds no kernels: it calls the entry points of libdedf.so (include/dedf.h), whose addresses diffusion_edf_amd/_lib.py hands over.  Launches
// go to the stream that the caller names (its current one); autograd runs a backward pass on the stream of its forward pass.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/DeviceGuard.h>
#include <cmath>
#include <optional>
#include <string>
#include <vector>
#include "../../include/dedf.h"

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

namespace {

struct Api {
    decltype(&dedf_edge_attention) attention;
    decltype(&dedf_edge_attention_backward) attention_backward;
    decltype(&dedf_edge_attention_scratch_bytes) attention_scratch;
    decltype(&dedf_norm_gate_residual) norm;
    decltype(&dedf_norm_gate_residual_backward) norm_backward;
    decltype(&dedf_norm_scratch_bytes) norm_scratch;
    decltype(&dedf_channel_dropout) dropout;
} api{};

void init(const std::vector<uintptr_t>& at) {
    TORCH_CHECK(at.size() == 7, "7 entry points");
    api.attention = reinterpret_cast<decltype(api.attention)>(at[0]);
    api.attention_backward = reinterpret_cast<decltype(api.attention_backward)>(at[1]);
    api.attention_scratch = reinterpret_cast<decltype(api.attention_scratch)>(at[2]);
    api.norm = reinterpret_cast<decltype(api.norm)>(at[3]);
    api.norm_backward = reinterpret_cast<decltype(api.norm_backward)>(at[4]);
    api.norm_scratch = reinterpret_cast<decltype(api.norm_scratch)>(at[5]);
    api.dropout = reinterpret_cast<decltype(api.dropout)>(at[6]);
}

void* stream_of(int64_t s) { return reinterpret_cast<void*>(static_cast<uintptr_t>(s)); }
template <class T> T* data(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
Tensor given(const Maybe& t) { return t.has_value() ? *t : Tensor(); }
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }          // (autograd takes no undefined inputs)
Tensor whole(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
int type_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? DEDF_F32 : t.scalar_type() == at::kHalf ? DEDF_F16 : t.scalar_type() == at::kBFloat16 ? DEDF_BF16 : -1; }
bool is_float(const Tensor& t) { return t.scalar_type() == at::kFloat; }
bool has_shape(const Tensor& t, at::IntArrayRef shape) { return t.sizes() == shape; }
Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }
void check(const char* what, int rc) {
    TORCH_CHECK_VALUE(rc != DEDF_ERR_INVALID, what, " refused its arguments (", rc, ")");
    TORCH_CHECK_NOT_IMPLEMENTED(rc != DEDF_ERR_UNSUPPORTED, what, " does not support this call (", rc, ")");
    TORCH_CHECK(rc == DEDF_OK, what, " failed (", rc, ")");
}
// all on one GPU
void check_gpu(const char* what, const Tensor& first, std::initializer_list<Tensor> rest) {
    for (const Tensor& t : rest) TORCH_CHECK_VALUE(!t.defined() || t.device() == first.device(), what, ": tensors on different devices");
    TORCH_CHECK(first.is_cuda(), what, " needs GPU tensors: the product has no CPU path");
}
void check_dropout(double p, const Tensor& rng, const Tensor& x) {
    TORCH_CHECK_VALUE(p >= 0.0 && p < 1.0, "dropout probability ", p, ": in [0, 1)");
    if (p == 0.0) return;
    TORCH_CHECK_VALUE(rng.defined(), "dropout needs rng, an int64 tensor [seed, offset] (dropout_rng)");
    TORCH_CHECK_VALUE(rng.scalar_type() == at::kLong && has_shape(rng, {2}), "rng: int64 [seed, offset], got ", rng.scalar_type(), " ", rng.sizes());
    TORCH_CHECK_VALUE(rng.device() == x.device(), "rng on ", rng.device(), ", the features on ", x.device());
}
// What these calls would leave out without a word: the tangent of a forward-mode dual tensor, and themselves in a trace (they are no registered operators)
void check_mode(const char* what, std::initializer_list<Tensor> all) {
    for (const Tensor& t : all)
        TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), what, ": forward-mode derivatives are not supported");
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(), what, " cannot be traced by torch.jit");
}
bool wants_grad(std::initializer_list<Tensor> all) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor& t : all) if (t.defined() && t.requires_grad()) return true;
    return false;
}
// gradients of a backward pass that autograd itself records: using them again raises
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list there;
    for (const Tensor& g : grads) if (g.defined()) there.push_back(g);
    auto error = std::make_shared<torch::autograd::DelayedError>("the training operators are differentiable once", static_cast<int64_t>(there.size()));
    for (Tensor& g : there) g = g.detach().requires_grad_(true);
    there = (*error)(std::move(there));
    size_t i = 0;
    for (Tensor& g : grads) if (g.defined()) g = there[i++];
    return grads;
}

// ---- edge attention -------------------------------------------------------------------------------------------------------------------------

struct Attn { Tensor alpha, value, dot, logits, table, dst, rowptr, length, bounds; int64_t n_dst; double p; };

dedf_edge_attn describe(const Attn& a, const Tensor& rng) {
    dedf_edge_attn x{};
    x.n_edges = a.value.size(0); x.n_dst = static_cast<int>(a.n_dst);
    x.heads = static_cast<int>(a.value.size(1)); x.k = static_cast<int>(a.alpha.size(2)); x.d = static_cast<int>(a.value.size(2));
    x.type = type_of(a.value); x.n_buckets = a.table.defined() ? static_cast<int>(a.table.size(0)) : 0;
    x.alpha = data<void>(a.alpha); x.alpha_stride = a.alpha.stride(0); x.value = data<void>(a.value); x.value_stride = a.value.stride(0);
    x.alpha_dot = data<float>(a.dot); x.dst = data<int32_t>(a.dst); x.rowptr = data<int32_t>(a.rowptr);
    x.edge_logits = data<float>(a.logits); x.edge_length = data<float>(a.length); x.bias_boundaries = data<float>(a.bounds); x.bias_table = data<float>(a.table);
    x.dropout = a.p; x.rng = data<int64_t>(rng);
    return x;
}
// out; for training also out in 32 bits, the rows' norms and the random words' seed and offset
struct AttnOut { Tensor out, out_f, norm, used; };
AttnOut attention_forward(const Attn& a, const Tensor& rng, int64_t stream, bool train) {
    const c10::OptionalDeviceGuard guard(a.value.device());
    const dedf_edge_attn x = describe(a, rng);
    const auto f = a.value.options();
    AttnOut r;
    r.out = at::empty({a.n_dst, x.heads, x.d}, f);
    if (train) {
        if (x.type != DEDF_F32) r.out_f = at::empty({a.n_dst, x.heads, x.d}, f.dtype(at::kFloat));
        r.norm = at::empty({a.n_dst, x.heads, 2}, f.dtype(at::kDouble));
        if (a.p > 0.0) r.used = at::empty({2}, f.dtype(at::kLong));
    }
    const Tensor scratch = bytes(static_cast<int64_t>(api.attention_scratch(&x, 0)), a.value);
    check("dedf_edge_attention", api.attention(&x, data<void>(r.out), data<float>(r.out_f), data<double>(r.norm), data<int64_t>(r.used), data<void>(scratch),
                                               scratch.numel(), stream_of(stream)));
    return r;
}

struct EdgeAttention : Function<EdgeAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& alpha, const Tensor& value, const Tensor& dot, const Maybe& logits, const Maybe& table, const Tensor& dst,
                          const Tensor& rowptr, const Maybe& length, const Maybe& bounds, const Maybe& rng, int64_t n_dst, double p, int64_t stream) {
        const Attn a{alpha, value, dot, given(logits), given(table), dst, rowptr, given(length), given(bounds), n_dst, p};
        const AttnOut r = attention_forward(a, given(rng), stream, true);
        ctx->save_for_backward({alpha, value, dot, a.logits, a.table, dst, rowptr, a.length, a.bounds, r.out_f.defined() ? r.out_f : r.out, r.norm, r.used});
        ctx->saved_data["n_dst"] = n_dst; ctx->saved_data["p"] = p; ctx->saved_data["stream"] = stream;
        return r.out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Attn a{s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], ctx->saved_data["n_dst"].toInt(), ctx->saved_data["p"].toDouble()};
        variable_list d(13);
        {
            const at::NoGradGuard no_grad;
            const c10::OptionalDeviceGuard guard(a.value.device());
            const dedf_edge_attn x = describe(a, s[11]);
            const Tensor up = grads[0].contiguous();
            if (ctx->needs_input_grad(0)) d[0] = at::empty(a.alpha.sizes(), a.alpha.options());
            if (ctx->needs_input_grad(1)) d[1] = at::empty(a.value.sizes(), a.value.options());
            if (ctx->needs_input_grad(2)) d[2] = at::empty_like(a.dot);
            size_t input = 3;          // (inputs that are not there are not counted)
            if (a.logits.defined() && ctx->needs_input_grad(input++)) d[3] = at::empty_like(a.logits);
            if (a.table.defined() && ctx->needs_input_grad(input++)) d[4] = at::empty_like(a.table);
            const Tensor scratch = bytes(static_cast<int64_t>(api.attention_scratch(&x, 1)), a.value);
            check("dedf_edge_attention_backward", api.attention_backward(&x, data<double>(s[10]), data<float>(s[9]), data<void>(up), data<void>(d[0]), data<void>(d[1]),
                                                                         data<float>(d[2]), data<float>(d[3]), data<float>(d[4]), data<void>(scratch), scratch.numel(),
                                                                         stream_of(ctx->saved_data["stream"].toInt())));
        }
        return once(d);
    }
};

// the tensor itself where an edge's (heads, channels) lie together, whatever the distance of two edges, else a copy
Tensor edge_rows(const Tensor& x) {
    const bool inner = (x.size(2) == 1 || x.stride(2) == 1) && (x.size(1) == 1 || x.stride(1) == x.size(2));
    return inner && x.stride(0) >= 0 ? x : x.contiguous();
}

Tensor edge_attention(const Tensor& alpha, const Tensor& value, const Tensor& dot, const Tensor& dst, const Tensor& rowptr, int64_t n_dst, const Maybe& logits_, const Maybe& length_,
                      const Maybe& bounds_, const Maybe& table_, double p, const Maybe& rng_, int64_t stream) {
    Tensor logits = given(logits_), length = given(length_), bounds = given(bounds_), table = given(table_), rng = given(rng_);
    TORCH_CHECK_VALUE(alpha.dim() == 3 && value.dim() == 3 && alpha.size(0) == value.size(0) && alpha.size(1) == value.size(1), "alpha (E, H, K) and value (E, H, D): got ",
                      alpha.sizes(), " and ", value.sizes());
    TORCH_CHECK_TYPE(type_of(value) >= 0 && alpha.scalar_type() == value.scalar_type(), "alpha and value: both float32, float16 or bfloat16, got ", alpha.scalar_type(), " and ",
                     value.scalar_type());
    const int64_t E = alpha.size(0), H = alpha.size(1), K = alpha.size(2), D = value.size(2);
    TORCH_CHECK_VALUE(H > 0 && K > 0 && D > 0, "alpha ", alpha.sizes(), ", value ", value.sizes(), ": empty rows");
    TORCH_CHECK_VALUE(E == dst.size(0), E, " edges, the segments hold ", dst.size(0));
    TORCH_CHECK_VALUE((has_shape(dot, {H, K}) || has_shape(dot, {1, H, K})) && is_float(dot), "alpha_dot: float32 (", H, ", ", K, "), got ", dot.scalar_type(), " ", dot.sizes());
    TORCH_CHECK_VALUE(!logits.defined() || (has_shape(logits, {E}) && is_float(logits)), "edge_logits: float32 (", E, ",)");
    if (!table.defined()) {
        TORCH_CHECK_VALUE(!length.defined() && !bounds.defined(), "edge_length and bias_boundaries come with bias_table");
    } else {
        TORCH_CHECK_VALUE(table.dim() == 2 && table.size(1) == H && table.size(0) > 0 && is_float(table), "bias_table: float32 (B, ", H, "), got ", table.scalar_type(), " ", table.sizes());
        TORCH_CHECK_VALUE(length.defined() && has_shape(length, {E}) && is_float(length), "edge_length: float32 (", E, ",)");
        const int64_t B = table.size(0);
        TORCH_CHECK_VALUE(B == 1 || (bounds.defined() && has_shape(bounds, {B - 1}) && is_float(bounds)), "bias_boundaries: float32 (", B - 1, ",)");
        if (B == 1) bounds = Tensor();
    }
    TORCH_CHECK_NOT_IMPLEMENTED(H <= 16 && H * K <= 256 && H * ((D + 3) / 4) <= 256 && (!table.defined() || (table.size(0) <= 1024 && table.numel() <= 2048)),
                                "at most 16 heads, 256 attention features and 1024 value channels an edge (head widths rounded up to multiples of 4), 1024 buckets, 2048 bias entries");
    check_dropout(p, rng, value);
    check_mode("edge_attention", {alpha, value, dot, logits, table});
    check_gpu("edge_attention", value, {alpha, dot, logits, length, bounds, table});
    TORCH_CHECK_VALUE(dst.device() == value.device(), "segments on ", dst.device(), ", the features on ", value.device());
    const Attn a{edge_rows(alpha), edge_rows(value), dot.contiguous(), whole(logits), whole(table), dst, rowptr, whole(length), whole(bounds), n_dst, p};
    rng = p > 0.0 ? rng.contiguous() : Tensor();
    if (wants_grad({alpha, value, dot, logits, table}))
        return EdgeAttention::apply(a.alpha, a.value, a.dot, maybe(a.logits), maybe(a.table), a.dst, a.rowptr, maybe(a.length), maybe(a.bounds), maybe(rng), n_dst, p, stream);
    return attention_forward(a, rng, stream, false).out;
}

// ---- the norms around a block -----------------------------------------------------------------------------------------------------------------

// irreps of a feature row as drop.RowShape has them
struct Shape { std::vector<int> mul, degree; int64_t width, channels, scalars; };

struct Norm { Tensor x, y, gate, post_w, post_b, next_w, next_b; double scale, eps, p; };

dedf_norm describe(const Norm& n, const Shape& s, const Tensor& rng) {
    dedf_norm a{};
    a.type = type_of(n.x); a.n_rows = static_cast<int>(n.x.size(0)); a.n_blocks = static_cast<int>(s.mul.size());
    a.groups = n.gate.defined() ? static_cast<int>(n.gate.size(0)) : 1;
    for (size_t i = 0; i < s.mul.size(); ++i) { a.mul[i] = s.mul[i]; a.degree[i] = s.degree[i]; }
    a.x = data<void>(n.x); a.y = data<void>(n.y); a.gate = data<void>(n.gate); a.gate_f = n.gate.defined() && is_float(n.gate);
    a.scale = static_cast<float>(n.scale); a.eps = static_cast<float>(n.eps);
    a.post_weight = data<float>(n.post_w); a.post_bias = data<float>(n.post_b); a.next_weight = data<float>(n.next_w); a.next_bias = data<float>(n.next_b);
    a.dropout = n.p; a.rng = data<int64_t>(rng);
    return a;
}
struct NormOut { Tensor h, z, used; };
NormOut norm_forward(const Norm& n, const Shape& s, const Tensor& rng, int64_t stream, bool train) {
    const c10::OptionalDeviceGuard guard(n.x.device());
    const dedf_norm a = describe(n, s, rng);
    NormOut r;
    if (n.y.defined()) r.h = at::empty_like(n.x);
    if (n.next_w.defined()) r.z = at::empty_like(n.x);
    if (train && n.p > 0.0) r.used = at::empty({2}, n.x.options().dtype(at::kLong));
    check("dedf_norm_gate_residual", api.norm(&a, data<void>(r.h), data<void>(r.z), data<int64_t>(r.used), stream_of(stream)));
    return r;
}

struct NormGateResidual : Function<NormGateResidual> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& y, const Maybe& gate, const Maybe& post_w, const Maybe& post_b, const Maybe& next_w,
                                 const Maybe& next_b, const Maybe& rng, const std::vector<int64_t>& mul, const std::vector<int64_t>& degree, double scale, double eps, double p, int64_t stream) {
        const Norm n{x, given(y), given(gate), given(post_w), given(post_b), given(next_w), given(next_b), scale, eps, p};
        const Shape s{{mul.begin(), mul.end()}, {degree.begin(), degree.end()}, 0, 0, 0};
        const NormOut r = norm_forward(n, s, given(rng), stream, true);
        ctx->save_for_backward({n.x, n.y, n.gate, n.post_w, n.post_b, n.next_w, n.next_b, r.used});
        ctx->saved_data["mul"] = mul; ctx->saved_data["degree"] = degree; ctx->saved_data["scale"] = scale; ctx->saved_data["eps"] = eps; ctx->saved_data["p"] = p;
        ctx->saved_data["stream"] = stream;
        ctx->set_materialize_grads(false);
        variable_list out;
        if (r.h.defined()) out.push_back(r.h);
        if (r.z.defined()) out.push_back(r.z);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Norm n{s[0], s[1], s[2], s[3], s[4], s[5], s[6], ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["p"].toDouble()};
        const auto mul = ctx->saved_data["mul"].toIntVector(), degree = ctx->saved_data["degree"].toIntVector();
        const Shape shape{{mul.begin(), mul.end()}, {degree.begin(), degree.end()}, 0, 0, 0};
        variable_list d(14);
        size_t next_out = 0;
        const Tensor up_h = n.y.defined() ? grads[next_out++] : Tensor(), up_z = n.next_w.defined() ? grads[next_out] : Tensor();
        if (!up_h.defined() && !up_z.defined()) return d;
        {
            const at::NoGradGuard no_grad;
            const c10::OptionalDeviceGuard guard(n.x.device());
            const dedf_norm a = describe(n, shape, s[7]);
            const Tensor gh = whole(up_h), gz = whole(up_z);
            size_t input = 0;          // (inputs that are not there are not counted)
            for (size_t i = 0; i < 7; ++i) if (s[i].defined() && ctx->needs_input_grad(input++)) d[i] = at::empty_like(s[i]);
            const Tensor scratch = bytes(static_cast<int64_t>(api.norm_scratch(&a)), n.x);
            check("dedf_norm_gate_residual_backward", api.norm_backward(&a, data<void>(gh), data<void>(gz), data<void>(d[0]), data<void>(d[1]), data<void>(d[2]), data<float>(d[3]),
                                                                        data<float>(d[4]), data<float>(d[5]), data<float>(d[6]), data<void>(scratch), scratch.numel(),
                                                                        stream_of(ctx->saved_data["stream"].toInt())));
        }
        return once(d);
    }
};

void check_rows(const char* name, const Tensor& x, const Shape& s) {
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) == s.width, name, ": expected (rows, ", s.width, "), got ", x.sizes());
    TORCH_CHECK_TYPE(type_of(x) >= 0, name, ": float32, float16 or bfloat16, got ", x.scalar_type());
    TORCH_CHECK_NOT_IMPLEMENTED(x.size(0) < (int64_t{1} << 31), name, ": fewer than 2**31 rows");
}
void check_affine(const std::string& name, Tensor& weight, Tensor& bias, const Shape& s) {
    if (!weight.defined()) { TORCH_CHECK_VALUE(!bias.defined(), name, "_bias without ", name, "_weight"); return; }
    TORCH_CHECK_VALUE(is_float(weight) && has_shape(weight, {s.channels}), name, "_weight: float32 (", s.channels, ",), got ", weight.scalar_type(), " ", weight.sizes());
    if (s.scalars == 0) { TORCH_CHECK_VALUE(!bias.defined() || bias.numel() == 0, name, "_bias: no channels of degree 0"); bias = Tensor(); }
    else TORCH_CHECK_VALUE(bias.defined() && is_float(bias) && has_shape(bias, {s.scalars}), name, "_bias: float32 (", s.scalars, ",) for the channels of degree 0");
    weight = weight.contiguous();
    bias = whole(bias);
}

std::vector<Maybe> norm_gate_residual(const Tensor& x, const Maybe& y_, const Shape& shape, double scale, const Maybe& gate_, const Maybe& post_w_, const Maybe& post_b_, double p,
                                      const Maybe& rng_, const Maybe& next_w_, const Maybe& next_b_, double eps, int64_t stream) {
    Tensor y = given(y_), gate = given(gate_), post_w = given(post_w_), post_b = given(post_b_), rng = given(rng_), next_w = given(next_w_), next_b = given(next_b_);
    check_rows("x", x, shape);
    TORCH_CHECK_VALUE(!y.defined() || (y.sizes() == x.sizes() && y.scalar_type() == x.scalar_type()), "y: ", x.scalar_type(), " ", x.sizes(), " like x");
    if (gate.defined()) {
        TORCH_CHECK_VALUE(gate.dim() == 2 && gate.size(1) == shape.channels && (x.size(0) == 0 || (gate.size(0) > 0 && x.size(0) % gate.size(0) == 0)), "gate: (G, ", shape.channels,
                          ") with G a divisor of ", x.size(0), " rows, got ", gate.sizes());
        TORCH_CHECK_NOT_IMPLEMENTED(gate.size(0) < (int64_t{1} << 31), "gate: fewer than 2**31 rows");
        TORCH_CHECK_TYPE(gate.scalar_type() == x.scalar_type() || is_float(gate), "gate: ", x.scalar_type(), " or float32, got ", gate.scalar_type());
    }
    check_affine("post", post_w, post_b, shape);
    check_affine("next", next_w, next_b, shape);
    TORCH_CHECK_VALUE(y.defined() || next_w.defined(), "weight: float32 (", shape.channels, ",)");
    TORCH_CHECK_VALUE(eps >= 1e-30, "eps ", eps, ": at least 1e-30");
    check_dropout(p, rng, x);
    check_mode("norm_gate_residual", {x, y, gate, post_w, post_b, next_w, next_b});
    check_gpu("norm_gate_residual", x, {y, gate, post_w, post_b, next_w, next_b});
    const Norm n{x.contiguous(), whole(y), whole(gate), post_w, post_b, next_w, next_b, scale, eps, p};
    rng = p > 0.0 ? rng.contiguous() : Tensor();
    Tensor h, z;
    if (wants_grad({n.x, n.y, n.gate, post_w, post_b, next_w, next_b})) {
        const variable_list out = NormGateResidual::apply(n.x, maybe(n.y), maybe(n.gate), maybe(n.post_w), maybe(n.post_b), maybe(n.next_w), maybe(n.next_b), maybe(rng), std::vector<int64_t>(shape.mul.begin(), shape.mul.end()),
                                                          std::vector<int64_t>(shape.degree.begin(), shape.degree.end()), scale, eps, p, stream);
        size_t at = 0;
        if (n.y.defined()) h = out[at++];
        if (n.next_w.defined()) z = out[at];
    } else {
        const NormOut r = norm_forward(n, shape, rng, stream, false);
        h = r.h; z = r.z;
    }
    return {h.defined() ? Maybe(h) : Maybe(), z.defined() ? Maybe(z) : Maybe()};
}

// ---- channel dropout ------------------------------------------------------------------------------------------------------------------------------

Tensor dropout_launch(const Tensor& x, const Shape& s, double p, const Tensor& rng, const Tensor& used, int64_t stream) {
    const c10::OptionalDeviceGuard guard(x.device());
    const Tensor out = at::empty_like(x);
    check("dedf_channel_dropout", api.dropout(type_of(x), static_cast<int>(x.size(0)), static_cast<int>(s.mul.size()), s.mul.data(), s.degree.data(), data<void>(x), p, data<int64_t>(rng),
                                              data<void>(out), data<int64_t>(used), stream_of(stream)));
    return out;
}
struct Dropout : Function<Dropout> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& rng, const std::vector<int64_t>& mul, const std::vector<int64_t>& degree, double p, int64_t stream) {
        const Tensor used = at::empty({2}, x.options().dtype(at::kLong));
        ctx->save_for_backward({used});
        ctx->saved_data["mul"] = mul; ctx->saved_data["degree"] = degree; ctx->saved_data["p"] = p; ctx->saved_data["stream"] = stream;
        return dropout_launch(x, Shape{{mul.begin(), mul.end()}, {degree.begin(), degree.end()}, 0, 0, 0}, p, rng, used, stream);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto mul = ctx->saved_data["mul"].toIntVector(), degree = ctx->saved_data["degree"].toIntVector();
        variable_list d(6);
        {
            const at::NoGradGuard no_grad;
            d[0] = dropout_launch(grads[0].contiguous(), Shape{{mul.begin(), mul.end()}, {degree.begin(), degree.end()}, 0, 0, 0}, ctx->saved_data["p"].toDouble(),
                                  ctx->get_saved_variables()[0], Tensor(), ctx->saved_data["stream"].toInt());
        }
        return once(d);
    }
};
Tensor equivariant_dropout(const Tensor& x, const Shape& shape, double p, const Maybe& rng_, int64_t stream) {
    const Tensor rng = given(rng_);
    check_rows("x", x, shape);
    check_dropout(p, rng, x);
    if (p > 0.0) check_mode("equivariant_dropout", {x});          // (else the result is x itself)
    check_gpu("equivariant_dropout", x, {});
    if (p == 0.0) return x;
    const Tensor in = x.contiguous(), words = rng.contiguous();
    if (wants_grad({in}))
        return Dropout::apply(in, words, std::vector<int64_t>(shape.mul.begin(), shape.mul.end()), std::vector<int64_t>(shape.degree.begin(), shape.degree.end()), p, stream);
    return dropout_launch(in, shape, p, words, Tensor(), stream);
}

}  // namespace

PYBIND11_MODULE(_dedf_torch, m) {
    py::class_<Shape>(m, "Shape").def(py::init([](std::vector<int> mul, std::vector<int> degree, int64_t width, int64_t channels, int64_t scalars) {
        return Shape{std::move(mul), std::move(degree), width, channels, scalars};
    }));
    m.def("init", &init);
    m.def("edge_attention", &edge_attention, py::call_guard<py::gil_scoped_release>());
    m.def("norm_gate_residual", &norm_gate_residual, py::call_guard<py::gil_scoped_release>());
    m.def("equivariant_dropout", &equivariant_dropout, py::call_guard<py::gil_scoped_release>());
}
