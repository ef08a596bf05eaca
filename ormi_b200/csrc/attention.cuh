// Masked attention: the parameters that its kernels share and the rule that decides which keys a query sees.
#pragma once
#include "op_math.cuh"
#include "operators.h"

namespace ormi_b200 {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Strides4 { int64_t b, t, h; };        // batch, position, head, in elements; head_dim is contiguous

struct AttnParams {
    const void *q, *k, *v;
    void* out;
    float* lse;                               // [batch, heads, q_len], natural logarithm; may be NULL in the forward pass
    const float* slopes;
    const int32_t *q_docs, *k_docs, *prefix, *key_len, *q_start;
    Strides4 qs, ks, vs, os;
    int batch, q_len, k_len, heads, kv_heads, group, dim;
    int causal;
    float scale, cap, inv_cap;
    // backward pass
    const void* dout;
    void *dq, *dk, *dv;
    float* delta;                             // [batch, heads, q_len]: sum over head_dim of dout * out
    Strides4 dos, dqs, dks, dvs;
    // keys split over several blocks (few queries over a long cache): partial results of each part
    float *part_out, *part_max, *part_sum;    // [split][batch][heads][q_len] (x dim); maxima and sums in base 2
    int splits;
};

// What one batch row's masks come to.
struct RowMask {
    int start, keys, prefix, causal;
    const int32_t *q_docs, *k_docs;
};
__device__ __forceinline__ RowMask row_mask(const AttnParams& p, int b) {
    RowMask m;
    m.start = p.q_start ? p.q_start[b] : p.k_len - p.q_len;
    m.keys = p.key_len ? max(0, min(p.key_len[b], p.k_len)) : p.k_len;
    m.prefix = p.prefix ? p.prefix[b] : 0;
    m.causal = p.causal;
    m.q_docs = p.q_docs ? p.q_docs + (int64_t)b * p.q_len : nullptr;
    m.k_docs = p.k_docs ? p.k_docs + (int64_t)b * p.k_len : nullptr;
    return m;
}
// One past the last key that the query at position `pos` may see, documents aside.
__device__ __forceinline__ int key_end(const RowMask& m, int pos) {
    return m.causal ? min(m.keys, max(pos < 0x7fffffff ? pos + 1 : pos, m.prefix)) : m.keys;
}

void attention_simple(ormi_b200_ctx* ctx, AttnParams& p, int dtype);
void attention_backward_simple(ormi_b200_ctx* ctx, AttnParams& p, int dtype);
bool attention_few_supported(const AttnParams& p, int dtype);
void attention_few(ormi_b200_ctx* ctx, AttnParams& p);
void attention_join(ormi_b200_ctx* ctx, const AttnParams& p, int dtype);
void attention_delta(ormi_b200_ctx* ctx, const AttnParams& p, int dtype);

}  // namespace ormi_b200
