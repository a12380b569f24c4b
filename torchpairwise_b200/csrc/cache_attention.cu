// Attention over a cache of quantised keys and values: which kernels.
//
// Few query rows to a key head read the codes as they lie (cache_few.cuh).  Many make attention a matter of matrix products, and there each key tile is
// read by many tiles of queries: keys and values are turned into the queries' type once, into scratch, and go through the kernels of
// attention.  Scratch is bounded: sequences go a few at a time, 128 MB of keys and values or one sequence, so that L2 holds most of what was just written.
#include "cache.cuh"

namespace tpw {
namespace {

constexpr long long kSlice = 128LL << 20;

int few(const CacheAttnParams &P, void *scratch, long long *bytes, cudaStream_t s) {
    return P.c.bits == 4 ? cache_few_4(P, scratch, bytes, s) : cache_few_8(P, scratch, bytes, s);
}

struct Slices {
    long long row, sequence, step;   // bytes of a token and head, of a sequence's keys (or values); sequences at a time
    explicit Slices(const CacheAttnParams &P) {
        row = P.c.D * 2;
        sequence = (P.c.capacity * P.c.H * row + 15) / 16 * 16;
        step = sequence > 0 ? kSlice / (2 * sequence) : P.c.B;
        step = step < 1 ? 1 : step < P.c.B ? step : P.c.B;
    }
    long long bytes() const { return 2 * sequence * step; }
};
tpw_attention slice(const CacheAttnParams &P, const Slices &S, void *scratch, long long first, long long count) {
    const long long e = 2;   // bytes of a number
    tpw_attention a = {};
    a.dtype = P.dtype;
    a.causal = P.causal;
    a.window = P.window;
    a.B = count; a.Nq = P.Nq; a.Nk = P.c.capacity; a.Hq = P.Hq; a.Hk = P.c.H; a.D = P.c.D;
    a.scale = P.scale;
    a.q = static_cast<const unsigned char *>(P.q) + first * P.q_s[0] * e;
    a.k = scratch;
    a.v = static_cast<unsigned char *>(scratch) + S.sequence * S.step;
    for (int i = 0; i < 3; ++i) a.q_stride[i] = P.q_s[i];
    a.k_stride[0] = a.v_stride[0] = S.sequence / e;
    a.k_stride[1] = a.v_stride[1] = P.c.D;
    a.k_stride[2] = a.v_stride[2] = P.c.capacity * P.c.D;
    a.key_lengths = P.c.lengths + first;
    a.out = static_cast<unsigned char *>(P.out) + first * P.Nq * P.Hq * S.row;
    a.lse = P.lse ? P.lse + first * P.Hq * P.Nq : nullptr;
    return a;
}

// Measured (bfloat16, 4 bits, [2, 16384, 8, 128] ragged): 192 rows 103 us as few and 132 as many, 256 rows 130 and 133, 512 rows 239 and 141; [8, 4096, 8, 128] the same; [1, 1000]
// 31 and 25 at 192.  Float32 stays: [2, 8192, 8, 128] 512 rows 263 and 821 us, [2, 8192, 8, 64] 1024 rows 302 and 325.
bool is_few(const CacheAttnParams &P) {
    if (P.dtype == TPW_F32 || P.group * P.Nq <= 192) return true;
    const tpw_attention a = slice(P, Slices(P), reinterpret_cast<void *>(256), 0, 1);   // of the scratch only its alignment takes part
    const AttnParams A = attn_params(a);
    return !attn_tc_fits(a.dtype, A);   // attention's own kernels for odd widths are slower still
}

} // namespace

long long cache_attention_bytes(const CacheAttnParams &P) {
    long long bytes = -1;
    if (is_few(P)) return few(P, nullptr, &bytes, nullptr), bytes;
    const Slices S(P);
    const tpw_attention a = slice(P, S, reinterpret_cast<void *>(256), 0, S.step);
    bytes = tpw_attention_scratch_bytes(&a);
    return bytes < 0 ? bytes : S.bytes() + bytes;
}

int cache_attention(const CacheAttnParams &P, void *scratch, long long bytes, cudaStream_t s) {
    if (is_few(P)) return few(P, scratch, nullptr, s);
    const Slices S(P);
    for (long long first = 0; first < P.c.B; first += S.step) {
        const long long count = P.c.B - first < S.step ? P.c.B - first : S.step;
        const tpw_attention a = slice(P, S, scratch, first, count);
        CacheParams c = P.c;
        c.B = count;
        c.lengths += first;
        for (int w = 0; w < 2; ++w) {
            c.codes[w] += first * c.H * c.capacity * c.row_bytes;
            c.scales[w] += first * c.H * c.capacity * c.groups;
        }
        int e = TPW_OK;
        if (c.capacity > 0) e = cache_expand(c, P.dtype, {const_cast<void *>(a.k), const_cast<void *>(a.v)}, a.k_stride, P.window > 0 ? P.Nq - 1 + P.window : 0, s);
        if (e == TPW_OK) e = tpw_attention_forward(&a, static_cast<unsigned char *>(scratch) + S.bytes(), bytes - S.bytes(), s);
        if (e != TPW_OK) return e;
    }
    return TPW_OK;
}

} // namespace tpw
