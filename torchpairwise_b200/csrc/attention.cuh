// What the attention kernels share: the arguments as a kernel gets them, which pairs are seen, and the entry points of the files.
#pragma once
#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

namespace tpw {

struct AttnParams {
    const void *q, *k, *v, *dout;
    long long q_s[3], k_s[3], v_s[3], do_s[3];   // batch, token, head
    const int *key_lengths;
    void *out, *lse, *rest, *dq, *dk, *dv;
    const void *dlse;
    long long B, Nq, Nk, Hq, Hk, D, group;       // group = Hq / Hk
    long long window;                            // 0: none
    int causal;
    double scale;
    // backward: rows of the pitch Nqp, [B, Hq, Nqp], of what a walk over the queries needs (attention_rows_kernel)
    void *row_lse, *row_delta;
    long long Nqp;
    unsigned *row_max;                           // half precision on the tensor cores: largest |dO_i|^2, |dlse_i| and |v_j|^2 (attention_rows.cu)
    int *status;
};

inline AttnParams attn_params(const tpw_attention &a) {
    AttnParams P = {};
    P.q = a.q; P.k = a.k; P.v = a.v; P.dout = a.grad_out;
    for (int i = 0; i < 3; ++i) {
        P.q_s[i] = a.q_stride[i];
        P.k_s[i] = a.k_stride[i];
        P.v_s[i] = a.v_stride[i];
        P.do_s[i] = a.grad_out_stride[i];
    }
    P.key_lengths = a.key_lengths;
    P.out = a.out; P.lse = a.lse; P.rest = a.out_rest; P.dq = a.grad_q; P.dk = a.grad_k; P.dv = a.grad_v;
    P.dlse = a.grad_lse;
    P.B = a.B; P.Nq = a.Nq; P.Nk = a.Nk; P.Hq = a.Hq; P.Hk = a.Hk; P.D = a.D;
    P.group = a.Hk > 0 ? a.Hq / a.Hk : 1;
    P.window = a.window;
    P.causal = a.causal;
    P.scale = a.scale;
    P.Nqp = (a.Nq + 127) / 128 * 128;
    return P;
}

// attention_simple.cu: any type, head width and stride, on the CUDA cores
int attn_simple_forward(int dtype, const AttnParams &P, cudaStream_t s);
int attn_simple_backward(int dtype, const AttnParams &P, cudaStream_t s);
// attention_rows.cu: what both gradient walks need of each query row
long long attn_rows_bytes(int dtype, const AttnParams &P);
int attn_rows(int dtype, AttnParams &P, void *scratch, bool tensor, cudaStream_t s);

// abi.cu: cudaFuncSetAttribute of a kernel's dynamic shared memory, once per device; `done` is the kernel's own word
int allow_shared_memory(const void *kernel, int bytes, std::atomic<unsigned long long> &done);
template <auto *KERNEL> int allow_shared_memory(int bytes) {
    static std::atomic<unsigned long long> done{0};
    return allow_shared_memory(reinterpret_cast<const void *>(KERNEL), bytes, done);
}
// 16-bit rows of [batch, tokens, heads, features] that lie the given numbers of bytes apart, as boxes of 64 features (128-byte
// swizzle) by `box_tokens` tokens; what lies beyond the tensor reads as zero
int make_tensor_map_heads(CUtensorMap *map, const void *base, uint64_t features, uint64_t tokens, uint64_t heads, uint64_t batch,
                          uint64_t token_pitch, uint64_t head_pitch, uint64_t batch_pitch, uint32_t box_tokens);
// the keys cut into ranges whose parts are joined afterwards
struct AttnSplits {
    int count = 1, keys = 0;             // ranges and keys of each
    float *out = nullptr, *lse = nullptr; // [count, B, Hq, Nq, D] outputs and [count, B, Hq, Nq] log-sums of the ranges
};
// attention_forward.cu: 16-bit types on the tensor cores
bool attn_tc_fits(int dtype, const AttnParams &P);
AttnSplits attn_tc_splits(const AttnParams &P);
int attn_tc_forward(int dtype, const AttnParams &P, const AttnSplits &splits, cudaStream_t s);
// attention_f32.cu: float32 up to 128 features on the tensor cores in three tf32 products
bool attn_f32_fits(int dtype, const AttnParams &P);
bool attn_f32_backward_fits(int dtype, const AttnParams &P);
AttnSplits attn_f32_splits(const AttnParams &P);
int attn_f32_forward(const AttnParams &P, const AttnSplits &splits, cudaStream_t s);
int attn_f32_backward(const AttnParams &P, cudaStream_t s);
// attention_parts.cu: float32 up to 64 features on the 16-bit tensor cores, operands as sums of three bfloat16 numbers, which lie in scratch
bool attn_parts_fits(int dtype, const AttnParams &P);
bool attn_parts_backward_fits(int dtype, const AttnParams &P);
long long attn_parts_bytes(const AttnParams &P, bool backward);
int attn_parts_forward(const AttnParams &P, void *scratch, cudaStream_t s);
int attn_parts_backward(const AttnParams &P, void *scratch, cudaStream_t s);
// attention_few.cu: few query rows
bool attn_few_fits(int dtype, const AttnParams &P);
AttnSplits attn_few_splits(const AttnParams &P);
int attn_few_forward(int dtype, const AttnParams &P, const AttnSplits &splits, cudaStream_t s);
int attn_join(int dtype, const AttnParams &P, const AttnSplits &splits, cudaStream_t s);
// attention_backward.cu
bool attn_tc_backward_fits(int dtype, const AttnParams &P);
int attn_tc_backward(int dtype, const AttnParams &P, cudaStream_t s);

#ifdef __CUDACC__
namespace {

// The keys [lo, hi) that query i of a sequence sees, and the queries [qlo, qhi) that see key j; off = length - Nq.
struct Seen {
    int length, off, nq, window;   // window: 0 none
    bool causal;
    __device__ __forceinline__ Seen(const AttnParams &P, long long b) {
        const int nk = (int)P.Nk;
        int n = P.key_lengths ? P.key_lengths[b] : nk;
        length = n < 0 ? 0 : n > nk ? nk : n;
        nq = (int)P.Nq;
        off = length - nq;
        causal = P.causal != 0;
        window = (int)(P.window < nk ? P.window : 0);   // a window over all keys is none
    }
    __device__ __forceinline__ int hi(int i) const {
        const int h = causal && i + off + 1 < length ? i + off + 1 : length;
        return h > 0 ? h : 0;
    }
    __device__ __forceinline__ int lo(int i) const {
        const int l = window ? i + off + 1 - window : 0;
        return l > 0 ? l : 0;
    }
    __device__ __forceinline__ int qlo(int j) const {
        const int l = causal ? j - off : 0;
        return l > 0 ? l : 0;
    }
    __device__ __forceinline__ int qhi(int j) const {
        const int h = window && j - off + window < nq ? j - off + window : nq;
        return j < length && h > 0 ? h : 0;
    }
};

// what rounding to T took from x
template <typename T> __device__ __forceinline__ T rest_of(float x) { return (T)(x - (float)(T)x); }

template <typename T> struct AttnAcc { typedef float type; };
template <> struct AttnAcc<double> { typedef double type; };

} // namespace
#endif

} // namespace tpw
