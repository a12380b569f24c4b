// C++ host layer of the cache of quantised keys and values (namespace `torchpairwise_b200`): schemas, checks, allocation and the current
// stream on top of the C ABI.  The reference has no such operators.  None is differentiable: what wants a gradient is refused.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <nvtx3/nvToolsExt.h>
#include <torch/library.h>

#include <cmath>

#include "../../../include/tpw_b200.h"

namespace {

using at::Tensor;

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

int code_of(const char *name, at::ScalarType type) {
    switch (type) {
        case at::kFloat: return TPW_F32;
        case at::kHalf: return TPW_F16;
        case at::kBFloat16: return TPW_BF16;
        default: TORCH_CHECK(false, name, ": expected float32, float16 or bfloat16, got ", type);
    }
}
void on_device(const Tensor &t, const Tensor &first) {
    TORCH_CHECK(t.is_cuda(), "torchpairwise (B200 build) runs on CUDA tensors only (no CPU path); got a tensor on ", t.device());
    TORCH_CHECK(t.get_device() == first.get_device(), "Expected all tensors to be on the same device");
}
void no_gradient(const char *name, const Tensor &t) {
    TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), name, ": a quantised cache passes no gradient on; call it under torch.no_grad() or detach");
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), name, ": forward-mode derivatives are not provided");
}

Tensor fresh(at::IntArrayRef sizes, const Tensor &like, at::ScalarType type) {
    return Tensor(at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt));
}

// A view whose features lie side by side, with strides that are read as they are; anything else is copied.
Tensor laid_out(const Tensor &x_) {
    const Tensor x = x_.resolve_neg();
    return x.size(3) != 1 && x.stride(3) != 1 ? x.contiguous() : x;
}
// Queries: many of them go through attention's tensor-core kernels, which fetch 16-bit rows in pieces of 16 bytes and take no broadcast dimensions
Tensor laid_out_queries(const Tensor &x_) {
    const Tensor x = x_.resolve_neg();
    bool fits = x.size(3) == 1 || x.stride(3) == 1;
    for (int d = 0; d < 3; ++d) fits = fits && (x.size(d) == 1 || x.stride(d) > 0);
    if (fits && x.element_size() == 2 && x.size(3) % 8 == 0) {
        fits = reinterpret_cast<uintptr_t>(x.const_data_ptr()) % 16 == 0;
        for (int d = 0; d < 3; ++d) fits = fits && (x.size(d) == 1 || x.stride(d) % 8 == 0);
    }
    return fits ? x : x.contiguous();
}
void strides_of(const Tensor &x, int64_t (&s)[3]) {
    // a dimension of one has no stride of its own: the one that a dense tensor would have
    const int64_t dense[3] = {x.size(1) * x.size(2) * x.size(3), x.size(2) * x.size(3), x.size(3)};
    for (int d = 0; d < 3; ++d) s[d] = x.size(d) == 1 ? dense[d] : x.stride(d);
}

// A cache as its four tensors, the lengths beside it
struct Cache {
    tpw_cache c = {};
    Tensor lengths;
    Cache(const char *name, const Tensor &k_codes, const Tensor &v_codes, const Tensor &k_scales, const Tensor &v_scales, int64_t features, int64_t bits,
          const Tensor &key_lengths) {
        TORCH_CHECK(bits == 4 || bits == 8, name, ": bits must be 4 or 8. Got ", bits);
        TORCH_CHECK(features >= 1 && features <= 128, name, ": ", features, " features per head: 1 to 128 are supported");
        const int64_t groups = (features + 31) / 32, row = tpw_cache_row_bytes((int)bits, features);
        for (const Tensor *t : {&k_codes, &v_codes}) {
            on_device(*t, k_codes);
            TORCH_CHECK(t->scalar_type() == at::kByte && t->dim() == 4 && t->size(3) == row, name, ": codes must be uint8 [batch, heads, capacity, ", row, "] for ", features,
                        " features in ", bits, " bits. Got ", t->scalar_type(), " ", t->sizes());
            TORCH_CHECK(t->sizes() == k_codes.sizes(), name, ": the codes of keys and values must have the same shape. Got: ", k_codes.sizes(), ", ", t->sizes());
            TORCH_CHECK(t->size(2) % 64 == 0, name, ": the capacity must be a multiple of 64. Got ", t->size(2));
        }
        for (const Tensor *t : {&k_scales, &v_scales}) {
            on_device(*t, k_codes);
            TORCH_CHECK(t->scalar_type() == at::kBFloat16 && t->dim() == 5 && t->size(0) == k_codes.size(0) && t->size(1) == k_codes.size(1) && t->size(2) == k_codes.size(2) &&
                            (t->size(3) == 1 || t->size(3) == groups) && t->size(4) == 2 && t->size(3) == k_scales.size(3),
                        name, ": scales must be bfloat16 [batch, heads, capacity, 1 or ", groups, ", 2], alike for keys and values. Got ", t->scalar_type(), " ", t->sizes());
            no_gradient(name, *t);
        }
        const Tensor *all[4] = {&k_codes, &v_codes, &k_scales, &v_scales};
        for (int i = 0; i < 4; ++i) {
            TORCH_CHECK(all[i]->is_contiguous() && !all[i]->is_neg(), name, ": the cache's tensors must be contiguous");
            for (int j = 0; j < i && all[i]->numel() > 0; ++j) TORCH_CHECK(all[i]->const_data_ptr() != all[j]->const_data_ptr(), name, ": the cache's tensors must be four");
        }
        on_device(key_lengths, k_codes);
        TORCH_CHECK(key_lengths.scalar_type() == at::kInt || key_lengths.scalar_type() == at::kLong, "key_lengths must be int32 or int64, got ", key_lengths.scalar_type());
        TORCH_CHECK(key_lengths.dim() == 1 && key_lengths.size(0) == k_codes.size(0), "key_lengths must hold one length for each of the ", k_codes.size(0), " sequences. Got shape ",
                    key_lengths.sizes());
        lengths = key_lengths.scalar_type() == at::kInt ? key_lengths.resolve_neg().contiguous() : key_lengths.clamp(-1, INT32_MAX).to(at::kInt).contiguous();
        c.bits = (int32_t)bits;
        c.groups = (int32_t)k_scales.size(3);
        c.B = k_codes.size(0); c.H = k_codes.size(1); c.capacity = k_codes.size(2); c.D = features;
        c.codes[0] = const_cast<void *>(k_codes.const_data_ptr());
        c.codes[1] = const_cast<void *>(v_codes.const_data_ptr());
        c.scales[0] = const_cast<void *>(k_scales.const_data_ptr());
        c.scales[1] = const_cast<void *>(v_scales.const_data_ptr());
        c.lengths = lengths.const_data_ptr<int32_t>();
    }
};

void cache_write(const Tensor &k_codes, const Tensor &v_codes, const Tensor &k_scales, const Tensor &v_scales, int64_t features, int64_t bits, const Tensor &k,
                 const Tensor &v, const Tensor &key_lengths) {
    NvtxRange range("torchpairwise_b200::cache_write");
    on_device(k_codes, k_codes);
    c10::cuda::CUDAGuard dg(k_codes.device());
    const Cache cache("cache_write", k_codes, v_codes, k_scales, v_scales, features, bits, key_lengths);
    tpw_cache_rows a = {};
    a.dtype = code_of("cache_write", k.scalar_type());
    TORCH_CHECK(v.scalar_type() == k.scalar_type(), "cache_write: k has type ", k.scalar_type(), ", v ", v.scalar_type());
    TORCH_CHECK(k.dim() == 4 && k.size(0) == cache.c.B && k.size(2) == cache.c.H && k.size(3) == features, "cache_write: k and v must be [", cache.c.B, ", tokens, ", cache.c.H, ", ",
                features, "]. Got ", k.sizes());
    TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have the same shape. Got: ", k.sizes(), ", ", v.sizes());
    const Tensor *in[2] = {&k, &v};
    Tensor x[2];
    for (int w = 0; w < 2; ++w) {
        on_device(*in[w], k_codes);
        no_gradient("cache_write", *in[w]);
        x[w] = laid_out(*in[w]);
        a.x[w] = const_cast<void *>(x[w].const_data_ptr());
        strides_of(x[w], a.stride[w]);
    }
    a.N = k.size(1);
    // refuses tensors of inference mode outside of it: before anything is written
    for (const Tensor *t : {&k_codes, &v_codes, &k_scales, &v_scales}) t->unsafeGetTensorImpl()->bump_version();
    TPW_CALL(tpw_cache_write(&cache.c, &a, stream_of(k_codes)));
}

std::tuple<Tensor, Tensor> cache_read(const Tensor &k_codes, const Tensor &v_codes, const Tensor &k_scales, const Tensor &v_scales, int64_t features, int64_t bits,
                                      const Tensor &key_lengths, c10::optional<int64_t> tokens, at::ScalarType dtype) {
    NvtxRange range("torchpairwise_b200::cache_read");
    on_device(k_codes, k_codes);
    c10::cuda::CUDAGuard dg(k_codes.device());
    const Cache cache("cache_read", k_codes, v_codes, k_scales, v_scales, features, bits, key_lengths);
    tpw_cache_rows a = {};
    a.dtype = code_of("cache_read", dtype);
    TORCH_CHECK(!tokens.has_value() || (*tokens >= 0 && *tokens < (int64_t(1) << 30)), "cache_read: tokens must be at least 0 and below 2^30. Got ", tokens.value_or(0));
    a.from_start = !tokens.has_value();
    a.N = tokens.value_or(cache.c.capacity);
    Tensor out[2];
    for (int w = 0; w < 2; ++w) {
        out[w] = fresh({cache.c.B, a.N, cache.c.H, features}, k_codes, dtype);
        a.x[w] = out[w].mutable_data_ptr();
    }
    TPW_CALL(tpw_cache_read(&cache.c, &a, stream_of(k_codes)));
    return {out[0], out[1]};
}

std::tuple<Tensor, Tensor> cache_attention(const Tensor &q_, const Tensor &k_codes, const Tensor &v_codes, const Tensor &k_scales, const Tensor &v_scales, int64_t features,
                                           int64_t bits, const Tensor &key_lengths, bool causal, c10::optional<int64_t> window, c10::optional<double> scale) {
    NvtxRange range("torchpairwise_b200::cache_attention");
    on_device(q_, q_);
    on_device(k_codes, q_);
    c10::cuda::CUDAGuard dg(q_.device());
    const Cache cache("cache_attention", k_codes, v_codes, k_scales, v_scales, features, bits, key_lengths);
    tpw_cache_attention_args a = {};
    a.dtype = code_of("cache_attention", q_.scalar_type());
    TORCH_CHECK(q_.dim() == 4 && q_.size(0) == cache.c.B && q_.size(3) == features, "cache_attention: q must be [", cache.c.B, ", queries, heads, ", features, "]. Got ", q_.sizes());
    a.Nq = q_.size(1); a.Hq = q_.size(2);
    TORCH_CHECK(a.Hq == 0 || (cache.c.H > 0 && a.Hq % cache.c.H == 0), "cache_attention: the ", a.Hq, " query heads must be a multiple of the ", cache.c.H, " key heads");
    TORCH_CHECK(!window.has_value() || *window >= 1, "cache_attention: window must be at least 1. Got ", window.value_or(0));
    TORCH_CHECK(!window.has_value() || causal, "cache_attention: a window needs causal=True");
    a.scale = scale.value_or(1.0 / std::sqrt(static_cast<double>(features)));
    TORCH_CHECK(a.scale > 0 && std::isfinite(a.scale), "cache_attention: scale must be positive and finite. Got ", a.scale);
    no_gradient("cache_attention", q_);
    const Tensor q = laid_out_queries(q_);
    a.q = q.const_data_ptr();
    strides_of(q, a.q_stride);
    a.causal = causal;
    a.window = window.value_or(0);
    Tensor out = fresh(q.sizes(), q, q.scalar_type()), lse = fresh({cache.c.B, a.Hq, a.Nq}, q, at::kFloat), scratch;
    a.out = out.mutable_data_ptr();
    a.lse = lse.mutable_data_ptr<float>();
    const int64_t bytes = tpw_cache_attention_scratch_bytes(&cache.c, &a);
    TORCH_CHECK(bytes >= 0, "cache_attention: ", tpw_last_error());
    if (bytes > 0) scratch = fresh({bytes}, q, at::kByte);
    TPW_CALL(tpw_cache_attention(&cache.c, &a, bytes > 0 ? scratch.mutable_data_ptr() : nullptr, bytes, stream_of(q)));
    return {out, lse};
}

#define TPW_CACHE_FIELDS "Tensor k_codes, Tensor v_codes, Tensor k_scales, Tensor v_scales, int features, int bits, "
TORCH_LIBRARY_FRAGMENT(torchpairwise_b200, m) {
    m.def("cache_write(Tensor(a!) k_codes, Tensor(b!) v_codes, Tensor(c!) k_scales, Tensor(d!) v_scales, int features, int bits, Tensor k, Tensor v, Tensor key_lengths) -> ()");
    m.def("cache_read(" TPW_CACHE_FIELDS "Tensor key_lengths, int? tokens=None, ScalarType dtype=bfloat16) -> (Tensor, Tensor)");
    m.def("cache_attention(Tensor q, " TPW_CACHE_FIELDS "Tensor key_lengths, bool causal=False, int? window=None, float? scale=None) -> (Tensor, Tensor)");
}
void register_ops(torch::Library &m) {
    m.impl("cache_write", cache_write);
    m.impl("cache_read", cache_read);
    m.impl("cache_attention", cache_attention);
}
TORCH_LIBRARY_IMPL(torchpairwise_b200, AutogradCUDA, m) { register_ops(m); }
TORCH_LIBRARY_IMPL(torchpairwise_b200, CUDA, m) { register_ops(m); }

} // namespace
