// C entry points of the cache of quantised keys and values: argument checks.
#include "cache.cuh"

namespace tpw {
namespace {

int check(const tpw_cache *c) {
    TPW_CHECK_ARG(c != nullptr, "tpw_cache: NULL arguments");
    TPW_CHECK_ARG(c->bits == 4 || c->bits == 8, "tpw_cache: %d bits: 4 and 8 are supported", c->bits);
    TPW_CHECK_ARG(c->D >= 1 && c->D <= 128, "tpw_cache: %lld features per head: 1 to 128 are supported", (long long)c->D);
    TPW_CHECK_ARG(c->groups == 1 || c->groups == (c->D + 31) / 32, "tpw_cache: %d groups: one, or one of every 32 features", c->groups);
    TPW_CHECK_ARG(c->B >= 0 && c->H >= 0 && c->capacity >= 0, "tpw_cache: negative size");
    TPW_CHECK_ARG(c->capacity % 64 == 0 && c->capacity < (1LL << 30), "tpw_cache: capacity %lld: a multiple of 64 below 2^30 is needed", (long long)c->capacity);
    TPW_CHECK_ARG(c->H <= (1LL << 20) && c->B <= (1LL << 30), "tpw_cache: more than 2^20 heads or 2^30 sequences");
    const bool some = c->B > 0 && c->H > 0 && c->capacity > 0;
    TPW_CHECK_ARG(c->lengths || c->B == 0, "tpw_cache: NULL lengths");
    for (int w = 0; w < 2; ++w) {
        TPW_CHECK_ARG(!some || (c->codes[w] && c->scales[w]), "tpw_cache: NULL pointer");
        TPW_CHECK_ARG(aligned16(c->codes[w]) && aligned16(c->scales[w]), "tpw_cache: codes and scales must be 16-byte aligned");
    }
    return TPW_OK;
}
bool known(int dtype) { return dtype == TPW_F32 || dtype == TPW_F16 || dtype == TPW_BF16; }

int check_rows(const tpw_cache *c, const tpw_cache_rows *r) {
    const int e = check(c);
    if (e != TPW_OK) return e;
    TPW_CHECK_ARG(r != nullptr, "tpw_cache_rows: NULL arguments");
    TPW_CHECK_ARG(known(r->dtype), "tpw_cache_rows: unsupported dtype %d", r->dtype);
    TPW_CHECK_ARG(r->N >= 0 && r->N < (1LL << 30), "tpw_cache_rows: %lld tokens", (long long)r->N);
    TPW_CHECK_ARG((r->x[0] && r->x[1]) || c->B == 0 || c->H == 0 || r->N == 0, "tpw_cache_rows: NULL pointer");
    return TPW_OK;
}

int check_attention(const tpw_cache *c, const tpw_cache_attention_args *a) {
    const int e = check(c);
    if (e != TPW_OK) return e;
    TPW_CHECK_ARG(a != nullptr, "tpw_cache_attention: NULL arguments");
    TPW_CHECK_ARG(known(a->dtype), "tpw_cache_attention: unsupported dtype %d", a->dtype);
    TPW_CHECK_ARG(a->Nq >= 0 && a->Nq < (1LL << 30) && a->Hq >= 0 && a->Hq <= (1LL << 20), "tpw_cache_attention: %lld queries of %lld heads", (long long)a->Nq, (long long)a->Hq);
    TPW_CHECK_ARG(a->Hq == 0 || (c->H > 0 && a->Hq % c->H == 0), "tpw_cache_attention: %lld query heads are no multiple of %lld key heads", (long long)a->Hq, (long long)c->H);
    TPW_CHECK_ARG(a->window >= 0, "tpw_cache_attention: negative window");
    TPW_CHECK_ARG(a->window == 0 || a->causal, "tpw_cache_attention: a window needs causal attention");
    const float factor = static_cast<float>(a->scale * 1.4426950408889634074);
    TPW_CHECK_ARG(a->scale > 0 && isfinite(a->scale) && factor > 0.f && isfinite(factor), "tpw_cache_attention: scale %g: positive and finite, also in 32 bits, is needed", a->scale);
    TPW_CHECK_ARG((a->q && a->out) || c->B == 0 || a->Nq == 0 || a->Hq == 0, "tpw_cache_attention: NULL pointer");
    TPW_CHECK_ARG(aligned16(a->out), "tpw_cache_attention: out must be 16-byte aligned");
    return TPW_OK;
}

CacheAttnParams attention_params(const tpw_cache &c, const tpw_cache_attention_args &a) {
    CacheAttnParams P = {};
    P.c = cache_params(c);
    P.q = a.q;
    for (int i = 0; i < 3; ++i) P.q_s[i] = a.q_stride[i];
    P.out = a.out;
    P.lse = a.lse;
    P.Nq = a.Nq;
    P.Hq = a.Hq;
    P.group = a.Hq / c.H;
    P.window = a.window < c.capacity ? a.window : 0;   // a window over all keys is none: nothing is to be added to 2^63 - 1
    P.causal = a.causal;
    P.dtype = a.dtype;
    P.scale = a.scale;
    P.scale_log2 = (float)(a.scale * 1.4426950408889634074);
    return P;
}

} // namespace
} // namespace tpw

extern "C" {

int64_t tpw_cache_row_bytes(int bits, int64_t D) {
    if ((bits != 4 && bits != 8) || D < 1 || D > 128) return 0;
    return tpw::cache_width(D) * 4 * bits;
}

int tpw_cache_write(const tpw_cache *c, const tpw_cache_rows *rows, tpw_stream_t stream) {
    tpw::clear_error();
    const int e = tpw::check_rows(c, rows);
    if (e != TPW_OK || c->B == 0 || c->H == 0 || rows->N == 0 || c->capacity == 0) return e;
    return tpw::cache_write(tpw::cache_params(*c), *rows, static_cast<cudaStream_t>(stream));
}

int tpw_cache_read(const tpw_cache *c, const tpw_cache_rows *rows, tpw_stream_t stream) {
    tpw::clear_error();
    const int e = tpw::check_rows(c, rows);
    if (e != TPW_OK || c->B == 0 || c->H == 0 || rows->N == 0) return e;
    return tpw::cache_read(tpw::cache_params(*c), *rows, static_cast<cudaStream_t>(stream));
}

int64_t tpw_cache_attention_scratch_bytes(const tpw_cache *c, const tpw_cache_attention_args *a) {
    tpw::clear_error();
    if (tpw::check_attention(c, a) != TPW_OK) return -1;
    if (c->B == 0 || a->Nq == 0 || a->Hq == 0) return 0;
    return tpw::cache_attention_bytes(tpw::attention_params(*c, *a));
}

int tpw_cache_attention(const tpw_cache *c, const tpw_cache_attention_args *a, void *scratch, int64_t scratch_bytes, tpw_stream_t stream) {
    tpw::clear_error();
    const int e = tpw::check_attention(c, a);
    if (e != TPW_OK || c->B == 0 || a->Nq == 0 || a->Hq == 0) return e;
    tpw::CacheAttnParams P = tpw::attention_params(*c, *a);
    const int64_t bytes = tpw::cache_attention_bytes(P);
    if (bytes < 0) return TPW_ERR_INVALID;
    TPW_CHECK_ARG(bytes == 0 || (scratch && tpw::aligned16(scratch) && scratch_bytes >= bytes), "tpw_cache_attention: scratch of %lld bytes, 16-byte aligned, is needed", (long long)bytes);
    P.status = tpw::device_status_ptr();
    return tpw::cache_attention(P, scratch, scratch_bytes, static_cast<cudaStream_t>(stream));
}

} // extern "C"
