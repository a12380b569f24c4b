// C entry points of attention: argument checks and the choice of kernels.
#include "attention.cuh"

namespace tpw {
namespace {

int check(const tpw_attention *a, bool backward) {
    TPW_CHECK_ARG(a != nullptr, "tpw_attention: NULL arguments");
    TPW_CHECK_ARG(a->dtype == TPW_F32 || a->dtype == TPW_F64 || a->dtype == TPW_F16 || a->dtype == TPW_BF16, "tpw_attention: unsupported dtype %d", a->dtype);
    TPW_CHECK_ARG(a->B >= 0 && a->Nq >= 0 && a->Nk >= 0 && a->Hq >= 0 && a->Hk >= 0, "tpw_attention: negative size");
    TPW_CHECK_ARG(a->D >= 1 && a->D <= 256, "tpw_attention: %lld features per head: 1 to 256 are supported", (long long)a->D);
    TPW_CHECK_ARG(a->Hq == 0 || (a->Hk > 0 && a->Hq % a->Hk == 0), "tpw_attention: %lld query heads are no multiple of %lld key heads", (long long)a->Hq, (long long)a->Hk);
    TPW_CHECK_ARG(a->Nq < (1LL << 30) && a->Nk < (1LL << 30), "tpw_attention: more than 2^30 tokens");
    TPW_CHECK_ARG(a->Hq <= (1LL << 20) && a->B <= (1LL << 30), "tpw_attention: more than 2^20 heads or 2^30 sequences");
    TPW_CHECK_ARG(a->window >= 0, "tpw_attention: negative window");
    TPW_CHECK_ARG(a->window == 0 || a->causal, "tpw_attention: a window needs causal attention");
    TPW_CHECK_ARG(a->scale > 0 && isfinite(a->scale), "tpw_attention: scale must be positive and finite");
    // scores are powers of two in 32 bits but for double: a factor that is 0 or infinite there makes masked scores NaN
    const float factor = static_cast<float>(a->scale * 1.4426950408889634074);
    TPW_CHECK_ARG(a->dtype == TPW_F64 || (factor > 0.f && isfinite(factor)), "tpw_attention: scale %g is beyond the range of 32-bit scores", a->scale);
    const bool rows = a->B > 0 && a->Nq > 0 && a->Hq > 0, keys = a->B > 0 && a->Nk > 0 && a->Hk > 0;
    TPW_CHECK_ARG(!rows || (a->q && a->out), "tpw_attention: NULL pointer");
    TPW_CHECK_ARG(!keys || (a->k && a->v), "tpw_attention: NULL pointer");
    if (backward) {
        TPW_CHECK_ARG(!rows || (a->grad_out && a->lse), "tpw_attention_backward: NULL pointer");
        TPW_CHECK_ARG((a->grad_k == nullptr) == (a->grad_v == nullptr), "tpw_attention_backward: grad_k and grad_v go together");
    }
    return TPW_OK;
}

bool nothing(const tpw_attention &a) { return a.B == 0 || a.Nq == 0 || a.Hq == 0; }

AttnSplits splits_of(int dtype, const AttnParams &P) {
    return attn_few_fits(dtype, P) ? attn_few_splits(P) : attn_tc_fits(dtype, P) ? attn_tc_splits(P) : attn_f32_fits(dtype, P) ? attn_f32_splits(P) : AttnSplits();
}
long long split_bytes(const AttnParams &P, const AttnSplits &splits) {
    return splits.count > 1 ? 4 * splits.count * P.B * P.Hq * P.Nq * (P.D + 1) : 0;
}
long long forward_bytes(int dtype, const AttnParams &P) {
    return attn_parts_fits(dtype, P) ? attn_parts_bytes(P, false) : split_bytes(P, splits_of(dtype, P));
}
long long backward_bytes(int dtype, const AttnParams &P) {
    return attn_rows_bytes(dtype, P) + (attn_parts_backward_fits(dtype, P) ? attn_parts_bytes(P, true) : 0);
}

} // namespace
} // namespace tpw

extern "C" {

int64_t tpw_attention_scratch_bytes(const tpw_attention *a) {
    tpw::clear_error();
    if (tpw::check(a, false) != TPW_OK) return -1;
    if (tpw::nothing(*a)) return 0;
    const tpw::AttnParams P = tpw::attn_params(*a);
    return tpw::forward_bytes(a->dtype, P);
}

int tpw_attention_forward(const tpw_attention *a, void *scratch, int64_t scratch_bytes, tpw_stream_t stream) {
    tpw::clear_error();
    const int e = tpw::check(a, false);
    if (e != TPW_OK || tpw::nothing(*a)) return e;
    const tpw::AttnParams P = tpw::attn_params(*a);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool f32 = tpw::attn_f32_fits(a->dtype, P);
    if (f32 || tpw::attn_tc_fits(a->dtype, P)) {
        const int64_t bytes = tpw::forward_bytes(a->dtype, P);
        TPW_CHECK_ARG(bytes == 0 || (scratch && tpw::aligned16(scratch) && scratch_bytes >= bytes),
                      "tpw_attention_forward: scratch of %lld bytes, 16-byte aligned, is needed", (long long)bytes);
        if (tpw::attn_parts_fits(a->dtype, P)) return tpw::attn_parts_forward(P, scratch, s);
        tpw::AttnSplits splits = tpw::splits_of(a->dtype, P);
        splits.out = static_cast<float *>(scratch);
        splits.lse = splits.out ? splits.out + splits.count * P.B * P.Hq * P.Nq * P.D : nullptr;
        const int e = f32 ? tpw::attn_f32_forward(P, splits, s) : tpw::attn_few_fits(a->dtype, P) ? tpw::attn_few_forward(a->dtype, P, splits, s) : tpw::attn_tc_forward(a->dtype, P, splits, s);
        return e != TPW_OK || splits.count == 1 ? e : tpw::attn_join(a->dtype, P, splits, s);
    }
    return tpw::attn_simple_forward(a->dtype, P, s);
}

int64_t tpw_attention_backward_scratch_bytes(const tpw_attention *a) {
    tpw::clear_error();
    if (tpw::check(a, true) != TPW_OK) return -1;
    if (tpw::nothing(*a)) return 0;
    return tpw::backward_bytes(a->dtype, tpw::attn_params(*a));
}

int tpw_attention_backward(const tpw_attention *a, void *scratch, int64_t scratch_bytes, tpw_stream_t stream) {
    tpw::clear_error();
    int e = tpw::check(a, true);
    if (e != TPW_OK) return e;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (tpw::nothing(*a)) {
        // no query reads the keys: their gradients are zero
        const size_t bytes = (size_t)(a->B * a->Nk * a->Hk * a->D) * (a->dtype == TPW_F64 ? 8 : a->dtype == TPW_F32 ? 4 : 2);
        if (bytes && a->grad_k) {
            TPW_CUDA_OK(cudaMemsetAsync(a->grad_k, 0, bytes, s));
            TPW_CUDA_OK(cudaMemsetAsync(a->grad_v, 0, bytes, s));
        }
        return TPW_OK;
    }
    tpw::AttnParams P = tpw::attn_params(*a);
    const long long bytes = tpw::backward_bytes(a->dtype, P);
    TPW_CHECK_ARG(scratch && tpw::aligned16(scratch) && scratch_bytes >= bytes, "tpw_attention_backward: scratch of %lld bytes, 16-byte aligned, is needed", bytes);
    if (!P.dq && !P.dk) return TPW_OK;
    const bool tensor = tpw::attn_tc_backward_fits(a->dtype, P);
    e = tpw::attn_rows(a->dtype, P, scratch, tensor, s);
    if (e != TPW_OK) return e;
    if (tensor) return tpw::attn_tc_backward(a->dtype, P, s);
    if (tpw::attn_parts_backward_fits(a->dtype, P)) return tpw::attn_parts_backward(P, static_cast<unsigned char *>(scratch) + tpw::attn_rows_bytes(a->dtype, P), s);
    if (tpw::attn_f32_backward_fits(a->dtype, P)) return tpw::attn_f32_backward(P, s);
    return tpw::attn_simple_backward(a->dtype, P, s);
}

} // extern "C"
