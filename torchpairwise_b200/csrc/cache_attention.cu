// Attention over a cache of quantised keys and values: which kernels.
//
// Few query rows to a key head read the codes as they lie (cache_few.cuh).  Many make attention a matter of matrix products, and there each key tile is
// read by many tiles of queries: keys and values are turned into half precision once, into scratch, and go through the kernels of
// attention.  Sequences go a few at a time, 128 MB of keys and values or one sequence, so that L2 holds most of what was just written; for bfloat16 there are
// queries and results of as many beside them.  Both scratch and the grids that fill it follow the capacity, not the lengths: short sequences in a large capacity pay for it.
// Half precision also for bfloat16 queries: what codes stand for has more than bfloat16's 8 digits, and keys rounded to them made the results 2.4 times as
// far off (chunk of 256 on 16384 keys: 0.0041 against 0.0017).  Its exponents do not reach, so each head's keys and values, and the queries and results
// with them, are moved by a power of two.
#include "cache.cuh"

namespace tpw {
namespace {

constexpr long long kSlice = 128LL << 20;
// half precision: a head's keys are brought below 2^8, its values below 2^14, so that their digits are normal numbers down to 2^-22 and 2^-28 of the
// highest, and queries, multiplied by what their keys were divided by, overflow only where scores do
constexpr int kKeys = 8, kValues = 14;

int few(const CacheAttnParams &P, void *scratch, long long *bytes, cudaStream_t s) {
    TPW_CHECK_ARG(P.group * P.Nq < (1LL << 30), "tpw_cache_attention: more than 2^30 query rows to a key head");
    return P.c.bits == 4 ? cache_few_4(P, scratch, bytes, s) : cache_few_8(P, scratch, bytes, s);
}

// Scratch of the many: keys and values of a slice; for bfloat16 also its heads' ranges, queries and results in half precision; then attention's own.
struct Slices {
    long long sequence, step, ranges, queries;   // bytes of a sequence's keys (or values); sequences at a time; bytes of the others
    explicit Slices(const CacheAttnParams &P) {
        auto round = [](long long bytes) { return (bytes + 255) / 256 * 256; };
        sequence = round(P.c.capacity * P.c.H * P.c.D * 2);
        // no more queries than keys and values
        const long long asked = P.Nq * P.Hq * P.c.D * 2;
        step = P.c.B;
        if (sequence > 0 && step > kSlice / (2 * sequence)) step = kSlice / (2 * sequence);
        if (step > kSlice / asked) step = kSlice / asked;
        if (step < 1) step = 1;
        const bool wide = P.dtype == TPW_BF16;
        ranges = wide ? round(step * P.c.H * 2 * kRangeParts * 4) : 0;
        queries = wide ? round(step * asked) : 0;
    }
    long long bytes() const { return 2 * sequence * step + ranges + 2 * queries; }
    unsigned char *values(void *scratch) const { return static_cast<unsigned char *>(scratch) + sequence * step; }
    unsigned char *range(void *scratch) const { return static_cast<unsigned char *>(scratch) + 2 * sequence * step; }
    unsigned char *query(void *scratch) const { return range(scratch) + ranges; }
    unsigned char *result(void *scratch) const { return query(scratch) + queries; }
};
tpw_attention slice(const CacheAttnParams &P, const Slices &S, void *scratch, long long first, long long count) {
    tpw_attention a = {};
    a.dtype = TPW_F16;
    a.causal = P.causal;
    a.window = P.window;
    a.B = count; a.Nq = P.Nq; a.Nk = P.c.capacity; a.Hq = P.Hq; a.Hk = P.c.H; a.D = P.c.D;
    a.scale = P.scale;
    a.k = scratch;
    a.v = S.values(scratch);
    if (P.dtype == TPW_F16) {
        a.q = static_cast<const unsigned char *>(P.q) + first * P.q_s[0] * 2;
        for (int i = 0; i < 3; ++i) a.q_stride[i] = P.q_s[i];
        a.out = static_cast<unsigned char *>(P.out) + first * P.Nq * P.Hq * P.c.D * 2;
    } else {
        a.q = S.query(scratch);
        a.q_stride[0] = P.Nq * P.Hq * P.c.D;
        a.q_stride[1] = P.Hq * P.c.D;
        a.q_stride[2] = P.c.D;
        a.out = S.result(scratch);
    }
    a.k_stride[0] = a.v_stride[0] = S.sequence / 2;
    a.k_stride[1] = a.v_stride[1] = P.c.D;
    a.k_stride[2] = a.v_stride[2] = P.c.capacity * P.c.D;
    a.key_lengths = P.c.lengths + first;
    a.lse = P.lse ? P.lse + first * P.Hq * P.Nq : nullptr;
    return a;
}

// Measured (bfloat16, us, as few and as many): [2, 16384, 8, 128] ragged, 4 bits, 192 rows 124 / 117, 224 rows 139 / 117, 256 rows 156 / 118; [4, 8000, 8, 64] in 8 bits 192 rows 108 / 105, 224 rows
// 123 / 105; [1, 1000, 8, 128] 224 rows 29 / 35; [8, 12345, 8, 128] through a window of 4096, 224 rows 229 / 333 (the capacity counts), 256 rows 257 / 336.
// Float32 stays: 512 rows [2, 8192, 8, 128] 263 us, 821 through attention's float32 kernels; where the times meet, 1024 rows [2, 8192, 8, 64] 302 and 325, was the last
// measurement, so that for prompts of thousands of rows the few-row kernel, whose time grows with them, is the slower one.
bool is_few(const CacheAttnParams &P) {
    if (P.dtype == TPW_F32 || P.group * P.Nq <= 192) return true;
    const tpw_attention a = slice(P, Slices(P), reinterpret_cast<void *>(256), 0, 1);   // of the scratch only its alignment takes part
    const bool pieces = aligned16(P.q) && aligned16(P.out) && P.q_s[0] % 8 == 0 && P.q_s[1] % 8 == 0 && P.q_s[2] % 8 == 0;
    return !pieces || !attn_tc_fits(a.dtype, attn_params(a));   // attention's own kernels for odd widths are slower still
}

} // namespace

long long cache_attention_bytes(const CacheAttnParams &P) {
    long long bytes = -1;
    if (is_few(P)) return few(P, nullptr, &bytes, nullptr), bytes;
    const Slices S(P);
    // the last slice has fewer sequences, for which attention may cut the keys into more ranges
    for (const long long count : {S.step, P.c.B % S.step}) {
        if (count == 0) continue;
        const tpw_attention a = slice(P, S, reinterpret_cast<void *>(256), 0, count);
        const long long more = tpw_attention_scratch_bytes(&a);
        if (more < 0) return more;
        if (S.bytes() + more > bytes) bytes = S.bytes() + more;
    }
    return bytes;
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
        const bool wide = P.dtype == TPW_BF16;
        uint32_t *highest = wide ? reinterpret_cast<uint32_t *>(S.range(scratch)) : nullptr;
        const long long last = P.window > 0 ? P.Nq - 1 + P.window : 0;   // what the first query sees, and the others on
        int e = wide ? cache_ranges(c, last, highest, s) : TPW_OK;
        if (e == TPW_OK) e = cache_expand(c, TPW_F16, {const_cast<void *>(a.k), const_cast<void *>(a.v)}, a.k_stride, last, highest, {kKeys, kValues}, s);
        if (e == TPW_OK && wide) {
            const int64_t stride[3] = {P.q_s[0], P.q_s[1], P.q_s[2]};
            e = cache_convert(false, static_cast<const unsigned char *>(P.q) + first * P.q_s[0] * 2, const_cast<void *>(a.q), stride, highest, kKeys, count, P.Nq, P.Hq, P.c.H, P.c.D, s);
        }
        if (e == TPW_OK) e = tpw_attention_forward(&a, static_cast<unsigned char *>(scratch) + S.bytes(), bytes - S.bytes(), s);
        if (e == TPW_OK && wide)
            e = cache_convert(true, a.out, static_cast<unsigned char *>(P.out) + first * P.Nq * P.Hq * P.c.D * 2, a.q_stride, highest + count * c.H * kRangeParts, kValues, count, P.Nq, P.Hq, P.c.H,
                              P.c.D, s);
        if (e != TPW_OK) return e;
    }
    return TPW_OK;
}

} // namespace tpw
