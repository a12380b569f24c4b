// C++ host layer of attention and rotary positions (namespace `torchpairwise_b200`): schemas, checks, allocation, the current
// stream and the autograd nodes on top of the C ABI.  The reference has no such operators, so the namespace is this library's own.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <nvtx3/nvToolsExt.h>
#include <torch/autograd.h>
#include <torch/library.h>

#include <cmath>

#include "../../../include/tpw_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

#define TPW_CALL(expr)                                                        \
    do {                                                                      \
        int status_ = (expr);                                                 \
        TORCH_CHECK(status_ == TPW_OK, #expr " failed: ", tpw_last_error());  \
    } while (0)

struct NvtxRange {
    explicit NvtxRange(const char *name) { nvtxRangePushA(name); }
    ~NvtxRange() { nvtxRangePop(); }
    NvtxRange(const NvtxRange &) = delete;
    NvtxRange &operator=(const NvtxRange &) = delete;
};

tpw_stream_t stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

int code_of(const char *name, const Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return TPW_F32;
        case at::kDouble: return TPW_F64;
        case at::kHalf: return TPW_F16;
        case at::kBFloat16: return TPW_BF16;
        default: TORCH_CHECK(false, name, ": expected a floating point tensor, got ", t.scalar_type());
    }
}
void require_cuda(const Tensor &t) {
    TORCH_CHECK(t.is_cuda(), "torchpairwise (B200 build) runs on CUDA tensors only (no CPU path); got a tensor on ", t.device());
}
void same_kind(const char *name, const char *arg, const Tensor &t, const Tensor &first) {
    require_cuda(t);
    TORCH_CHECK(t.get_device() == first.get_device(), "Expected all tensors to be on the same device");
    TORCH_CHECK(t.scalar_type() == first.scalar_type(), name, ": ", arg, " has type ", t.scalar_type(), ", the first tensor ", first.scalar_type());
}

// at::empty without the dispatcher, 1 us less each; the callers below hold the device's guard
Tensor fresh(at::IntArrayRef sizes, const Tensor &like, at::ScalarType type) {
    return Tensor(at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt));
}
Tensor fresh(at::IntArrayRef sizes, const Tensor &like) { return fresh(sizes, like, like.scalar_type()); }

// Forward-mode derivatives have no rule here.  A tensor that carries a tangent need not require a gradient, so without this the result would have
// none and count as constant.
void no_tangents(const char *name, std::initializer_list<const Tensor *> tensors) {
    for (const Tensor *t : tensors)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), name, ": forward-mode derivatives are not provided");
}

bool wants_node(std::initializer_list<const Tensor *> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : tensors)
        if (t->requires_grad()) return true;
    return false;
}

// A view whose features lie side by side and whose strides the kernels can use as they are (views of a packed projection, transposed
// batches); anything else is copied.  Broadcast dimensions and negative or odd strides of 16-bit rows count as anything else: the
// tensor-core kernels fetch rows in pieces of 16 bytes.
Tensor laid_out(const Tensor &x) {
    if (x.is_neg() || x.numel() == 0) return x.contiguous();
    bool fits = x.size(3) == 1 || x.stride(3) == 1;
    for (int d = 0; d < 3; ++d) fits = fits && (x.size(d) == 1 || x.stride(d) > 0);
    if (fits && x.element_size() == 2 && x.size(3) % 8 == 0) {
        fits = reinterpret_cast<uintptr_t>(x.const_data_ptr()) % 16 == 0;
        for (int d = 0; d < 3; ++d) fits = fits && (x.size(d) == 1 || x.stride(d) % 8 == 0);
    }
    return fits ? x : x.contiguous();
}
void strides_of(const Tensor &x, int64_t (&s)[3]) {
    // a dimension of one token has no stride of its own: the one that a dense tensor would have
    const int64_t dense[3] = {x.size(1) * x.size(2) * x.size(3), x.size(2) * x.size(3), x.size(3)};
    for (int d = 0; d < 3; ++d) s[d] = x.size(d) == 1 ? dense[d] : x.stride(d);
}

tpw_attention describe(const Tensor &q, const Tensor &k, const Tensor &v, const OptTensor &lengths, bool causal, int64_t window, double scale) {
    tpw_attention a = {};
    a.dtype = code_of("attention", q);
    a.causal = causal;
    a.window = window;
    a.B = q.size(0); a.Nq = q.size(1); a.Hq = q.size(2); a.D = q.size(3);
    a.Nk = k.size(1); a.Hk = k.size(2);
    a.scale = scale;
    a.q = q.const_data_ptr(); a.k = k.const_data_ptr(); a.v = v.const_data_ptr();
    strides_of(q, a.q_stride);
    strides_of(k, a.k_stride);
    strides_of(v, a.v_stride);
    a.key_lengths = lengths.has_value() ? lengths->const_data_ptr<int32_t>() : nullptr;
    return a;
}

Tensor scratch_for(int64_t bytes, const Tensor &like) {
    TORCH_CHECK(bytes >= 0, "attention: ", tpw_last_error());
    return bytes > 0 ? fresh({bytes}, like, at::kByte) : Tensor();
}

// out and lse, of the caller's rank; for a backward also the rest of out where it is rounded to 16 bits
variable_list attention_forward(const Tensor &q_, const Tensor &k_, const Tensor &v_, const OptTensor &lengths, bool causal, int64_t window, double scale,
                                Tensor *rest) {
    NvtxRange range("torchpairwise_b200::attention");
    c10::cuda::CUDAGuard dg(q_.device());
    const bool unbatched = q_.dim() == 3;
    auto four = [&](const Tensor &t) { return laid_out(unbatched ? t.unsqueeze(0) : t); };
    const Tensor q = four(q_), k = four(k_), v = four(v_);
    tpw_attention a = describe(q, k, v, lengths, causal, window, scale);
    Tensor out = fresh(q.sizes(), q);
    Tensor lse = fresh({a.B, a.Hq, a.Nq}, q, a.dtype == TPW_F64 ? at::kDouble : at::kFloat);
    a.out = out.mutable_data_ptr();
    a.lse = lse.mutable_data_ptr();
    if (rest && q.element_size() == 2) {
        *rest = fresh(q.sizes(), q);
        a.out_rest = rest->mutable_data_ptr();
    }
    Tensor scratch = scratch_for(tpw_attention_scratch_bytes(&a), q);
    TPW_CALL(tpw_attention_forward(&a, scratch.defined() ? scratch.mutable_data_ptr() : nullptr, scratch.defined() ? scratch.numel() : 0, stream_of(q)));
    if (unbatched) return {out.squeeze(0), lse.squeeze(0)};
    return {out, lse};
}

struct AttentionFn : torch::autograd::Function<AttentionFn> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const OptTensor &lengths, bool causal,
                                 int64_t window, double scale) {
        at::AutoDispatchBelowADInplaceOrView guard;
        Tensor rest;
        variable_list r = attention_forward(q, k, v, lengths, causal, window, scale, &rest);
        // the caller's own tensors are saved, so that a change in place before backward is an error
        ctx->save_for_backward({q, k, v, r[0], r[1], lengths.has_value() ? *lengths : Tensor(), rest});
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["window"] = window;
        ctx->saved_data["scale"] = scale;
        ctx->set_materialize_grads(false);
        return r;
    }
    static variable_list backward(AutogradContext *ctx, variable_list go) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "attention: gradients of gradients are not provided");
        no_tangents("attention", {&go[0], &go[1]});
        NvtxRange range("torchpairwise_b200::attention_backward");
        auto s = ctx->get_saved_variables();
        const bool unbatched = s[0].dim() == 3;
        c10::cuda::CUDAGuard dg(s[0].device());
        auto four = [&](const Tensor &t) { return unbatched ? t.unsqueeze(0) : t; };
        const Tensor q = laid_out(four(s[0])), k = laid_out(four(s[1])), v = laid_out(four(s[2])), out = four(s[3]), lse = four(s[4]);
        const bool wants_q = ctx->needs_input_grad(0), wants_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
        if ((!go[0].defined() && !go[1].defined()) || (!wants_q && !wants_kv)) return variable_list(7);
        const Tensor g = go[0].defined() ? laid_out(four(go[0])) : at::zeros(q.sizes(), q.options());
        tpw_attention a = describe(q, k, v, s[5].defined() ? OptTensor(s[5]) : c10::nullopt, ctx->saved_data["causal"].toBool(),
                                   ctx->saved_data["window"].toInt(), ctx->saved_data["scale"].toDouble());
        a.out = out.data_ptr();
        a.lse = lse.data_ptr();
        a.out_rest = s[6].defined() ? s[6].data_ptr() : nullptr;
        a.grad_out = g.const_data_ptr();
        strides_of(g, a.grad_out_stride);
        Tensor gl, dq, dk, dv;
        if (go[1].defined()) {
            gl = go[1].contiguous();
            a.grad_lse = gl.const_data_ptr();
        }
        if (wants_q) {
            dq = fresh(q.sizes(), q);
            a.grad_q = dq.mutable_data_ptr();
        }
        if (wants_kv) {
            dk = fresh(k.sizes(), k);
            dv = fresh(v.sizes(), v);
            a.grad_k = dk.mutable_data_ptr();
            a.grad_v = dv.mutable_data_ptr();
        }
        Tensor scratch = scratch_for(tpw_attention_backward_scratch_bytes(&a), q);
        TPW_CALL(tpw_attention_backward(&a, scratch.defined() ? scratch.mutable_data_ptr() : nullptr, scratch.defined() ? scratch.numel() : 0, stream_of(q)));
        auto back = [&](const Tensor &t, bool wanted) { return !wanted ? Tensor() : unbatched ? t.squeeze(0) : t; };
        return {back(dq, wants_q), back(dk, ctx->needs_input_grad(1)), back(dv, ctx->needs_input_grad(2)), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> attention(const Tensor &q, const Tensor &k, const Tensor &v, bool causal, c10::optional<int64_t> window,
                                     const OptTensor &key_lengths, c10::optional<double> scale) {
    require_cuda(q);
    same_kind("attention", "k", k, q);
    same_kind("attention", "v", v, q);
    code_of("attention", q);
    TORCH_CHECK(q.dim() == 3 || q.dim() == 4, "q must be 3-D (unbatched) or 4-D (batched) tensor: [batch,] tokens, heads, features");
    TORCH_CHECK(k.dim() == q.dim() && v.dim() == q.dim(), "q, k and v must have the same number of dimensions");
    const int64_t f = q.dim() - 1;
    TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have the same shape. Got: ", k.sizes(), ", ", v.sizes());
    TORCH_CHECK(q.size(f) == k.size(f), "q and k must have same number of features. Got: q.size(", f, ")=", q.size(f), ", k.size(", f, ")=", k.size(f));
    TORCH_CHECK(q.size(f) >= 1 && q.size(f) <= 256, "attention: ", q.size(f), " features per head: 1 to 256 are supported");
    TORCH_CHECK(f == 2 || q.size(0) == k.size(0), "batch_size of q and k do not match.");
    const int64_t hq = q.size(f - 1), hk = k.size(f - 1);
    TORCH_CHECK(hq == 0 || (hk > 0 && hq % hk == 0), "attention: the ", hq, " query heads must be a multiple of the ", hk, " key heads");
    TORCH_CHECK(!window.has_value() || *window >= 1, "attention: window must be at least 1. Got ", window.value_or(0));
    TORCH_CHECK(!window.has_value() || causal, "attention: a window needs causal=True");
    const double c = scale.value_or(1.0 / std::sqrt(static_cast<double>(q.size(f))));
    TORCH_CHECK(c > 0 && std::isfinite(c), "attention: scale must be positive and finite. Got ", c);
    OptTensor lengths;
    if (key_lengths.has_value()) {
        const Tensor &n = *key_lengths;
        require_cuda(n);
        TORCH_CHECK(n.get_device() == q.get_device(), "Expected all tensors to be on the same device");
        TORCH_CHECK(n.scalar_type() == at::kInt || n.scalar_type() == at::kLong, "key_lengths must be int32 or int64, got ", n.scalar_type());
        const int64_t batch = f == 2 ? 1 : q.size(0);
        TORCH_CHECK(n.numel() == batch && n.dim() <= 1, "key_lengths must hold one length for each of the ", batch, " sequences. Got shape ", n.sizes());
        lengths = n.scalar_type() == at::kInt ? n.contiguous() : n.clamp(0, k.size(f - 2)).to(at::kInt).contiguous();
    }
    no_tangents("attention", {&q, &k, &v});
    if (!wants_node({&q, &k, &v})) {   // serving: no node, 2 us less
        at::AutoDispatchBelowADInplaceOrView guard;
        auto r = attention_forward(q, k, v, lengths, causal, window.value_or(0), c, nullptr);
        return {r[0], r[1]};
    }
    auto r = AttentionFn::apply(q, k, v, lengths, causal, window.value_or(0), c);
    return {r[0], r[1]};
}

// ---- rotary positions ---------------------------------------------------------------------------------------------
variable_list rotary_forward(const Tensor &q_, const OptTensor &k_, const Tensor &cos_, const Tensor &sin_, const OptTensor &positions, bool interleaved,
                             bool inverse) {
    NvtxRange range("torchpairwise_b200::rotary_embedding");
    c10::cuda::CUDAGuard dg(q_.device());
    const bool unbatched = q_.dim() == 3;
    auto four = [&](const Tensor &t) {
        Tensor x = unbatched ? t.unsqueeze(0) : t;
        return x.is_neg() || (x.size(3) != 1 && x.stride(3) != 1) ? x.contiguous() : x;
    };
    const Tensor cos = cos_.contiguous(), sin = sin_.contiguous();
    tpw_rotary a = {};
    const Tensor x[2] = {four(q_), k_.has_value() ? four(*k_) : Tensor()};
    variable_list out;
    for (int w = 0; w < 2 && x[w].defined(); ++w) {
        a.H[w] = x[w].size(2);
        a.x[w] = x[w].const_data_ptr();
        strides_of(x[w], a.stride[w]);
        Tensor y = fresh(x[w].sizes(), x[w]);
        a.out[w] = y.mutable_data_ptr();
        out.push_back(unbatched ? y.squeeze(0) : y);
    }
    a.dtype = code_of("rotary_embedding", q_);
    a.interleaved = interleaved;
    a.inverse = inverse;
    a.B = x[0].size(0); a.N = x[0].size(1); a.D = x[0].size(3);
    a.half = cos.size(1);
    a.length = cos.size(0);
    a.cos = cos.const_data_ptr<float>();
    a.sin = sin.const_data_ptr<float>();
    if (positions.has_value()) {
        const Tensor &p = *positions;
        a.positions = p.const_data_ptr<int64_t>();
        a.position_stride[0] = p.dim() == 2 && p.size(0) > 1 ? p.stride(0) : 0;
        a.position_stride[1] = p.dim() >= 1 && p.size(-1) > 1 ? p.stride(-1) : 0;
    }
    TPW_CALL(tpw_rotary_apply(&a, stream_of(q_)));
    return out;
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const OptTensor &k, const Tensor &cos, const Tensor &sin, const OptTensor &positions,
                                 bool interleaved, bool inverse) {
        at::AutoDispatchBelowADInplaceOrView guard;
        variable_list out = rotary_forward(q, k, cos, sin, positions, interleaved, inverse);
        ctx->save_for_backward({cos, sin, positions.has_value() ? *positions : Tensor()});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["inverse"] = inverse;
        ctx->saved_data["pair"] = k.has_value();
        ctx->set_materialize_grads(false);
        return out;
    }
    // the turn back is the same operator, so gradients of gradients come with it
    static variable_list backward(AutogradContext *ctx, variable_list go) {
        auto s = ctx->get_saved_variables();
        const bool inter = ctx->saved_data["interleaved"].toBool(), inverse = !ctx->saved_data["inverse"].toBool(), pair = ctx->saved_data["pair"].toBool();
        const OptTensor at_ = s[2].defined() ? OptTensor(s[2]) : c10::nullopt;
        variable_list g(7);
        const bool first = go[0].defined() && ctx->needs_input_grad(0), second = pair && go[1].defined() && ctx->needs_input_grad(1);
        if (first) {
            auto r = turn(go[0], second ? OptTensor(go[1]) : c10::nullopt, s[0], s[1], at_, inter, inverse);
            g[0] = r[0];
            if (second) g[1] = r[1];
        } else if (second) {
            g[1] = turn(go[1], c10::nullopt, s[0], s[1], at_, inter, inverse)[0];
        }
        return g;
    }
    static variable_list turn(const Tensor &q, const OptTensor &k, const Tensor &cos, const Tensor &sin, const OptTensor &positions, bool interleaved, bool inverse) {
        no_tangents("rotary_embedding", {&q, k.has_value() ? &*k : &q, &cos, &sin});
        if (wants_node({&q, k.has_value() ? &*k : &q})) return apply(q, k, cos, sin, positions, interleaved, inverse);
        at::AutoDispatchBelowADInplaceOrView guard;
        return rotary_forward(q, k, cos, sin, positions, interleaved, inverse);
    }
};

variable_list rotary(const Tensor &q, const OptTensor &k, const Tensor &cos, const Tensor &sin, const OptTensor &positions, bool interleaved) {
    require_cuda(q);
    code_of("rotary_embedding", q);
    TORCH_CHECK(q.dim() == 3 || q.dim() == 4, "q must be 3-D (unbatched) or 4-D (batched) tensor: [batch,] tokens, heads, features");
    const int64_t f = q.dim() - 1;
    if (k.has_value()) {
        same_kind("rotary_embedding", "k", *k, q);
        TORCH_CHECK(k->dim() == q.dim(), "q and k must have the same number of dimensions");
        for (int64_t d = 0; d <= f; ++d)
            TORCH_CHECK(d == f - 1 || k->size(d) == q.size(d), "q and k may only differ in their number of heads. Got: ", q.sizes(), ", ", k->sizes());
    }
    for (const Tensor *t : {&cos, &sin}) {
        require_cuda(*t);
        TORCH_CHECK(t->get_device() == q.get_device(), "Expected all tensors to be on the same device");
        TORCH_CHECK(t->scalar_type() == at::kFloat && t->dim() == 2, "cos and sin must be float32 tables [length, turned features / 2]");
    }
    TORCH_CHECK(!(at::GradMode::is_enabled() && (cos.requires_grad() || sin.requires_grad())), "rotary_embedding: the tables receive no gradient");
    TORCH_CHECK(cos.sizes() == sin.sizes(), "cos and sin must have the same shape. Got: ", cos.sizes(), ", ", sin.sizes());
    TORCH_CHECK(2 * cos.size(1) <= q.size(f), "rotary_embedding: the tables turn ", 2 * cos.size(1), " features, a head has ", q.size(f));
    const int64_t batch = f == 2 ? 1 : q.size(0), tokens = q.size(f - 2);
    OptTensor at_;
    if (positions.has_value()) {
        const Tensor &p = *positions;
        require_cuda(p);
        TORCH_CHECK(p.get_device() == q.get_device(), "Expected all tensors to be on the same device");
        TORCH_CHECK(p.scalar_type() == at::kInt || p.scalar_type() == at::kLong, "positions must be int32 or int64, got ", p.scalar_type());
        TORCH_CHECK((p.dim() == 1 && p.size(0) == tokens) || (p.dim() == 2 && f == 3 && (p.size(0) == batch || p.size(0) == 1) && p.size(1) == tokens),
                    "positions must be [tokens] or [batch, tokens]. Got ", p.sizes(), " for ", q.sizes());
        at_ = p.to(at::kLong);
    } else {
        TORCH_CHECK(cos.size(1) == 0 || cos.size(0) >= tokens, "rotary_embedding: ", tokens, " tokens, the tables end at ", cos.size(0));
    }
    return RotaryFn::turn(q, k, cos, sin, at_, interleaved, false);
}

Tensor rotary_one(const Tensor &q, const Tensor &cos, const Tensor &sin, const OptTensor &positions, bool interleaved) {
    return rotary(q, c10::nullopt, cos, sin, positions, interleaved)[0];
}
std::tuple<Tensor, Tensor> rotary_two(const Tensor &q, const Tensor &k, const Tensor &cos, const Tensor &sin, const OptTensor &positions, bool interleaved) {
    auto r = rotary(q, k, cos, sin, positions, interleaved);
    return {r[0], r[1]};
}

std::tuple<Tensor, Tensor> rotary_table(const Tensor &frequencies, int64_t length, double magnitude) {
    require_cuda(frequencies);
    TORCH_CHECK(frequencies.scalar_type() == at::kDouble && frequencies.dim() == 1, "rotary_table: frequencies must be a float64 vector");
    TORCH_CHECK(length >= 0, "rotary_table: negative length");
    TORCH_CHECK(!(at::GradMode::is_enabled() && frequencies.requires_grad()), "rotary_table: the frequencies receive no gradient");
    no_tangents("rotary_table", {&frequencies});
    c10::cuda::CUDAGuard dg(frequencies.device());
    const Tensor f = frequencies.contiguous();
    Tensor cos = at::empty({length, f.size(0)}, f.options().dtype(at::kFloat)), sin = at::empty_like(cos);
    TPW_CALL(tpw_rotary_table(f.const_data_ptr<double>(), magnitude, cos.mutable_data_ptr<float>(), sin.mutable_data_ptr<float>(), length, f.size(0), stream_of(f)));
    return {cos, sin};
}

TORCH_LIBRARY(torchpairwise_b200, m) {
    m.def("attention(Tensor q, Tensor k, Tensor v, bool causal=False, int? window=None, Tensor? key_lengths=None, float? scale=None) -> (Tensor, Tensor)");
    m.def("rotary_embedding(Tensor q, Tensor cos, Tensor sin, Tensor? positions=None, bool interleaved=False) -> Tensor");
    m.def("rotary_embedding.pair(Tensor q, Tensor k, Tensor cos, Tensor sin, Tensor? positions=None, bool interleaved=False) -> (Tensor, Tensor)");
    m.def("rotary_table(Tensor frequencies, int length, float magnitude=1.) -> (Tensor, Tensor)");
}
void register_ops(torch::Library &m) {
    m.impl("attention", attention);
    m.impl("rotary_embedding", rotary_one);
    m.impl("rotary_embedding.pair", rotary_two);
    m.impl("rotary_table", rotary_table);
}
TORCH_LIBRARY_IMPL(torchpairwise_b200, AutogradCUDA, m) { register_ops(m); }
TORCH_LIBRARY_IMPL(torchpairwise_b200, CUDA, m) { register_ops(m); }

} // namespace
