// Softmax attention with capped scores, distance bias, document and prefix masks: argument checks, the choice of the
// kernel, and the kernels that take every case (fp32 arithmetic, any head size up to 256, any stride).
//
//   z = scale q.k;  z = cap tanh(z / cap);  z -= slope |pos - j|;   o = softmax(z) v over the visible keys;  lse = log sum exp z
//   backward:  p = exp(z - lse);  dv = p^T do;  dz = p (do v^T - rowsum(do o)) (1 - (capped / cap)^2);  dq = scale dz k;  dk = scale dz^T q
//
// One pass over the keys with the running maximum and sum of the softmax.  The query heads that share a key/value head are
// packed into the rows of one tile (row = query * group + head of the group), so shared keys are read once and the
// gradients of a shared head are summed inside one block, in a fixed order.  Bound by the FMA pipe where there are blocks
// enough (24 TFLOP/s forward, 17 backward at 2048 tokens, 16 heads, head_dim 64, fp32), by latency below.
#include <algorithm>
#include <cmath>
#include <vector>

#include "attention_tc.cuh"

namespace ormi_b200 {
namespace {

constexpr int kThreads = 256;               // 16 x 16 threads over a tile

__device__ __forceinline__ int64_t at(const Strides4& s, int b, int t, int h) { return (int64_t)b * s.b + (int64_t)t * s.t + (int64_t)h * s.h; }

// Rows [first, first + R) of a [.., dim] operand into shared memory as fp32, zero behind `limit` rows and behind dim: a warp per
// row, so that finding a row is not every element's work.
template <typename T, int R, int DP, typename F>
__device__ __forceinline__ void load_rows(float (*dst)[DP + 4], int first, int limit, int dim, F&& row_ptr) {
    const int lane = threadIdx.x & 31;
#pragma unroll 4
    for (int r = threadIdx.x >> 5; r < R; r += kThreads / 32) {
        const bool in = first + r < limit;
        const T* row = in ? (const T*)row_ptr(first + r) : nullptr;
#pragma unroll
        for (int d = lane; d < DP; d += 32) dst[r][d] = in && d < dim ? to_f32(row[d]) : 0.f;
    }
}

// acc[i][j] = A[ty + 16 i] . B[tx + 16 j]
template <int RI, int RJ, int DP>
__device__ __forceinline__ void dot_tile(const float (*A)[DP + 4], const float (*B)[DP + 4], int dim, int ty, int tx, float (&acc)[RI][RJ]) {
#pragma unroll
    for (int i = 0; i < RI; ++i)
#pragma unroll
        for (int j = 0; j < RJ; ++j) acc[i][j] = 0.f;
#pragma unroll 2
    for (int d = 0; d < dim; d += 4) {
        float4 a[RI], b[RJ];
#pragma unroll
        for (int i = 0; i < RI; ++i) a[i] = *(const float4*)&A[ty + 16 * i][d];
#pragma unroll
        for (int j = 0; j < RJ; ++j) b[j] = *(const float4*)&B[tx + 16 * j][d];
#pragma unroll
        for (int i = 0; i < RI; ++i)
#pragma unroll
            for (int j = 0; j < RJ; ++j) {
                acc[i][j] = fmaf(a[i].x, b[j].x, acc[i][j]);
                acc[i][j] = fmaf(a[i].y, b[j].y, acc[i][j]);
                acc[i][j] = fmaf(a[i].z, b[j].z, acc[i][j]);
                acc[i][j] = fmaf(a[i].w, b[j].w, acc[i][j]);
            }
    }
}

// out[i][c] (rows ty + 16 i, columns 64 c + 4 tx .. + 3) += sum over k of W(row, k) * V[k][column]
template <int RI, int K, int DP, typename W>
__device__ __forceinline__ void add_tile(float4 (&out)[RI][DP / 64], const float (*V)[DP + 4], int ty, int tx, W&& weight) {
    for (int k = 0; k < K; ++k) {
        float w[RI];
#pragma unroll
        for (int i = 0; i < RI; ++i) w[i] = weight(ty + 16 * i, k);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            const float4 v = *(const float4*)&V[k][c * 64 + tx * 4];
#pragma unroll
            for (int i = 0; i < RI; ++i) {
                out[i][c].x = fmaf(w[i], v.x, out[i][c].x);
                out[i][c].y = fmaf(w[i], v.y, out[i][c].y);
                out[i][c].z = fmaf(w[i], v.z, out[i][c].z);
                out[i][c].w = fmaf(w[i], v.w, out[i][c].w);
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ void store4(T* row, int d, int dim, const float4& v, float by) {
    const float x[4] = {v.x, v.y, v.z, v.w};
    for (int k = 0; k < 4; ++k) if (d + k < dim) row[d + k] = from_f32<T>(x[k] * by);
}

// Sum / maximum over the 16 threads of a tile row.
__device__ __forceinline__ float row_sum(float v) { for (int o = 8; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o); return v; }
__device__ __forceinline__ float row_max(float v) { for (int o = 8; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o)); return v; }

struct RowOf { int t, h, pos, end, doc; float slope; };   // one packed row: query, head, position, key_end, document, slope in base 2
__device__ __forceinline__ RowOf row_of(const AttnParams& p, const RowMask& m, int kvh, int r) {
    RowOf o{0, 0, 0, 0, 0, 0.f};
    if (r >= p.q_len * p.group) return o;                  // a row of padding sees nothing
    o.t = r / p.group;
    o.h = kvh * p.group + r % p.group;
    o.pos = m.start + o.t;
    o.end = key_end(m, o.pos);
    o.doc = m.q_docs ? m.q_docs[o.t] : 0;
    o.slope = p.slopes ? p.slopes[o.h] * kLog2e : 0.f;
    return o;
}
__device__ __forceinline__ bool sees(const RowMask& m, const RowOf& o, int j) { return j < o.end && (!m.k_docs || m.k_docs[j] == o.doc); }
// Base-2 score of a pair from the raw product; dtanh = derivative of the cap.
__device__ __forceinline__ float score2(const AttnParams& p, const RowOf& o, int j, float raw, float& dcap) {
    float z = raw * p.scale;
    dcap = 1.f;
    if (p.cap > 0.f) {
        const float th = tanhf(z * p.inv_cap);
        dcap = 1.f - th * th;
        z = p.cap * th;
    }
    return z * kLog2e - o.slope * fabsf((float)(o.pos - j));
}

template <typename T, int BM, int BN, int DP>
__global__ void __launch_bounds__(kThreads) attn_forward(AttnParams p) {
    constexpr int RI = BM / 16, RJ = BN / 16;
    extern __shared__ float smem[];
    auto Q = (float (*)[DP + 4])smem;
    auto K = Q + BM;
    auto V = K + BN;
    auto P = (float (*)[BN + 4])(V + BN);
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const int b = blockIdx.y / p.kv_heads, kvh = blockIdx.y % p.kv_heads;
    const int rows = p.q_len * p.group, first = blockIdx.x * BM;
    const RowMask m = row_mask(p, b);
    load_rows<T, BM, DP>(Q, first, rows, p.dim, [&](int r) { return (const T*)p.q + at(p.qs, b, r / p.group, kvh * p.group + r % p.group); });
    RowOf o[RI];
    float top[RI], total[RI];
    float4 acc[RI][DP / 64];
#pragma unroll
    for (int i = 0; i < RI; ++i) {
        o[i] = row_of(p, m, kvh, first + ty + 16 * i);
        top[i] = -INFINITY; total[i] = 0.f;
        for (int c = 0; c < DP / 64; ++c) acc[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const int last = min(first + BM, rows) - 1;
    const int end = last >= first ? key_end(m, m.start + last / p.group) : 0;      // positions grow with the row
    const int tiles = (end + BN - 1) / BN, per = (tiles + p.splits - 1) / p.splits;
    const int lo = blockIdx.z * per, hi = min(lo + per, tiles);
    for (int n = lo; n < hi; ++n) {
        if (m.k_docs) {                              // a tile of other documents is not loaded at all
            bool any = false;
            for (int i = 0; i < RI; ++i) for (int j = 0; j < RJ; ++j) any |= sees(m, o[i], n * BN + tx + 16 * j);
            if (!__syncthreads_or(any)) continue;
        }
        __syncthreads();
        load_rows<T, BN, DP>(K, n * BN, m.keys, p.dim, [&](int j) { return (const T*)p.k + at(p.ks, b, j, kvh); });
        load_rows<T, BN, DP>(V, n * BN, m.keys, p.dim, [&](int j) { return (const T*)p.v + at(p.vs, b, j, kvh); });
        __syncthreads();
        float s[RI][RJ];
        dot_tile<RI, RJ, DP>(Q, K, p.dim, ty, tx, s);
#pragma unroll
        for (int i = 0; i < RI; ++i) {
            float big = top[i];
#pragma unroll
            for (int j = 0; j < RJ; ++j) {
                const int key = n * BN + tx + 16 * j;
                float d;
                s[i][j] = sees(m, o[i], key) ? score2(p, o[i], key, s[i][j], d) : -INFINITY;
                big = fmaxf(big, s[i][j]);
            }
            big = row_max(big);
            const float base = big == -INFINITY ? 0.f : big, keep = exp2f(top[i] - base);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < RJ; ++j) {
                s[i][j] = exp2f(s[i][j] - base);
                sum += s[i][j];
                P[ty + 16 * i][tx + 16 * j] = s[i][j];
            }
            total[i] = total[i] * keep + row_sum(sum);
            top[i] = big;
#pragma unroll
            for (int c = 0; c < DP / 64; ++c) { acc[i][c].x *= keep; acc[i][c].y *= keep; acc[i][c].z *= keep; acc[i][c].w *= keep; }
        }
        __syncthreads();
        add_tile<RI, BN, DP>(acc, V, ty, tx, [&](int r, int k) { return P[r][k]; });
    }
#pragma unroll
    for (int i = 0; i < RI; ++i) {
        const int r = first + ty + 16 * i;
        if (r >= rows) continue;
        const int64_t line = ((int64_t)b * p.heads + o[i].h) * p.q_len + o[i].t;
        if (p.splits > 1) {
            const int64_t part = (int64_t)blockIdx.z * p.batch * p.heads * p.q_len + line;
            for (int c = 0; c < DP / 64; ++c) store4(p.part_out + part * p.dim, c * 64 + tx * 4, p.dim, acc[i][c], 1.f);
            if (tx == 0) { p.part_max[part] = top[i]; p.part_sum[part] = total[i]; }
        } else {
            const float by = total[i] > 0.f ? 1.f / total[i] : total[i] == 0.f ? 0.f : total[i];
            T* out = (T*)p.out + at(p.os, b, o[i].t, o[i].h);
            for (int c = 0; c < DP / 64; ++c) store4(out, c * 64 + tx * 4, p.dim, acc[i][c], by);
            if (p.lse && tx == 0) p.lse[line] = top[i] == -INFINITY ? -INFINITY : (top[i] + log2f(total[i])) * kLn2;
        }
    }
}

// Joins the parts of a split: a block per (batch, head, query), its four warps sharing the parts, a lane four columns.
template <typename T>
__global__ void __launch_bounds__(128) attn_join(AttnParams p) {
    __shared__ float box[4][256];
    __shared__ float sums[4];
    const int64_t lines = (int64_t)p.batch * p.heads * p.q_len, line = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int t = line % p.q_len, h = line / p.q_len % p.heads, b = line / p.q_len / p.heads;
    float top = -INFINITY;
    for (int s = lane; s < p.splits; s += 32) top = fmaxf(top, p.part_max[s * lines + line]);
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.f : top;
    float total = 0.f;
    for (int c = 0; c < p.dim; c += 128) {
        float v[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll 4
        for (int s = warp; s < p.splits; s += 4) {
            const float by = exp2f(p.part_max[s * lines + line] - base);
            sum += by * p.part_sum[s * lines + line];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int d = c + lane + 32 * k;
                if (d < p.dim) v[k] = fmaf(by, p.part_out[(s * lines + line) * p.dim + d], v[k]);
            }
        }
        if (c == 0) total = sum;
#pragma unroll
        for (int k = 0; k < 4; ++k) if (c + lane + 32 * k < p.dim) box[warp][c + lane + 32 * k] = v[k];
    }
    if (lane == 0) sums[warp] = total;
    __syncthreads();
    total = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    const float by = total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;
    T* out = (T*)p.out + at(p.os, b, t, h);
    for (int d = threadIdx.x; d < p.dim; d += 128) out[d] = from_f32<T>(((box[0][d] + box[1][d]) + (box[2][d] + box[3][d])) * by);
    if (p.lse && threadIdx.x == 0) p.lse[line] = top == -INFINITY ? -INFINITY : (top + log2f(total)) * kLn2;
}

template <typename T>
__global__ void __launch_bounds__(256) attn_delta(AttnParams p) {
    const int64_t lines = (int64_t)p.batch * p.heads * p.q_len, line = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (line >= lines) return;
    const int lane = threadIdx.x & 31;
    const int h = line % p.heads, t = line / p.heads % p.q_len, b = line / p.heads / p.q_len;      // heads innermost: neighbours in memory
    const T* o = (const T*)p.out + at(p.os, b, t, h);
    const T* g = (const T*)p.dout + at(p.dos, b, t, h);
    float s = 0.f;
    for (int d = lane; d < p.dim; d += 32) s = fmaf(to_f32(o[d]), to_f32(g[d]), s);
    s = warp_sum(s);
    if (lane == 0) p.delta[((int64_t)b * p.heads + h) * p.q_len + t] = s;
}

// Rows of the partial gradients of a split loop, and a row's place among them.
template <bool QUERY> __host__ __device__ inline int64_t part_rows(const AttnParams& p) { return (int64_t)p.batch * (QUERY ? (int64_t)p.q_len * p.heads : (int64_t)p.k_len * p.kv_heads); }
template <bool QUERY> __device__ __forceinline__ int64_t part_row(const AttnParams& p, int b, int t, int h) {
    return QUERY ? ((int64_t)b * p.q_len + t) * p.heads + h : ((int64_t)b * p.k_len + t) * p.kv_heads + h;
}

// dk and dv of one tile of keys: a loop over the packed query rows.  QUERY: dq of one tile of rows, a loop over the keys.
template <typename T, int B, int DP, bool QUERY>
__global__ void __launch_bounds__(kThreads) attn_backward(AttnParams p) {
    constexpr int RI = B / 16;
    extern __shared__ float smem[];
    auto Q = (float (*)[DP + 4])smem;          // q and dout of a tile of rows, k and v of a tile of keys
    auto G = Q + B;
    auto K = G + B;
    auto V = K + B;
    auto P = (float (*)[B + 4])(V + B);        // [row][key]: probabilities, then gradients of the scores
    auto Z = P + B;
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const int b = blockIdx.y / p.kv_heads, kvh = blockIdx.y % p.kv_heads;
    const int rows = p.q_len * p.group;
    const RowMask m = row_mask(p, b);
    auto load_queries = [&](int first) {
        load_rows<T, B, DP>(Q, first, rows, p.dim, [&](int r) { return (const T*)p.q + at(p.qs, b, r / p.group, kvh * p.group + r % p.group); });
        load_rows<T, B, DP>(G, first, rows, p.dim, [&](int r) { return (const T*)p.dout + at(p.dos, b, r / p.group, kvh * p.group + r % p.group); });
    };
    auto load_keys = [&](int first) {
        load_rows<T, B, DP>(K, first, m.keys, p.dim, [&](int j) { return (const T*)p.k + at(p.ks, b, j, kvh); });
        load_rows<T, B, DP>(V, first, m.keys, p.dim, [&](int j) { return (const T*)p.v + at(p.vs, b, j, kvh); });
    };
    float4 one[RI][DP / 64], two[RI][DP / 64];      // dk and dv of the keys, or dq of the rows and nothing
#pragma unroll
    for (int i = 0; i < RI; ++i)
        for (int c = 0; c < DP / 64; ++c) one[i][c] = two[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int mine = blockIdx.x * B;
    if (QUERY) load_queries(mine); else load_keys(mine);
    int lo = 0, hi = (rows + B - 1) / B;
    if (QUERY) {
        const int last = min(mine + B, rows) - 1;
        hi = (key_end(m, m.start + last / p.group) + B - 1) / B;
    } else if (mine >= m.keys) hi = 0;
    if (p.splits > 1) {                              // a part of the loop for each block in z
        const int per = (max(hi, 0) + p.splits - 1) / p.splits;
        lo = blockIdx.z * per;
        hi = min(lo + per, hi);
    }
    for (int n = lo; n < hi; ++n) {
        const int row0 = QUERY ? mine : n * B, key0 = QUERY ? n * B : mine;
        if (!QUERY) {
            const int last = min(row0 + B, rows) - 1;                 // the furthest that any row of this tile sees
            if (key_end(m, m.start + last / p.group) <= key0) continue;
        }
        if (m.k_docs) {                              // a tile of other documents is not loaded at all
            bool any = false;
            for (int i = 0; i < RI; ++i) {
                const RowOf o = row_of(p, m, kvh, row0 + ty + 16 * i);
                for (int j = 0; j < RI; ++j) any |= sees(m, o, key0 + tx + 16 * j);
            }
            if (!__syncthreads_or(any)) continue;
        }
        __syncthreads();
        if (QUERY) load_keys(key0); else load_queries(row0);
        __syncthreads();
        float s[RI][RI], g[RI][RI];
        dot_tile<RI, RI, DP>(Q, K, p.dim, ty, tx, s);
        dot_tile<RI, RI, DP>(G, V, p.dim, ty, tx, g);
#pragma unroll
        for (int i = 0; i < RI; ++i) {
            const RowOf o = row_of(p, m, kvh, row0 + ty + 16 * i);
            const bool live = row0 + ty + 16 * i < rows;
            const int64_t line = ((int64_t)b * p.heads + o.h) * p.q_len + o.t;
            const float lse2 = live ? p.lse[line] * kLog2e : 0.f, delta = live ? p.delta[line] : 0.f;
#pragma unroll
            for (int j = 0; j < RI; ++j) {
                const int key = key0 + tx + 16 * j;
                float prob = 0.f, dz = 0.f;
                if (sees(m, o, key)) {
                    float d;
                    prob = exp2f(score2(p, o, key, s[i][j], d) - lse2);
                    dz = prob * (g[i][j] - delta) * d * p.scale;
                }
                P[ty + 16 * i][tx + 16 * j] = prob;
                Z[ty + 16 * i][tx + 16 * j] = dz;
            }
        }
        __syncthreads();
        if (QUERY) add_tile<RI, B, DP>(one, K, ty, tx, [&](int r, int k) { return Z[r][k]; });
        else {
            add_tile<RI, B, DP>(one, Q, ty, tx, [&](int r, int k) { return Z[k][r]; });
            add_tile<RI, B, DP>(two, G, ty, tx, [&](int r, int k) { return P[k][r]; });
        }
    }
#pragma unroll
    for (int i = 0; i < RI; ++i) {
        const int r = mine + ty + 16 * i;
        if (r >= (QUERY ? rows : p.k_len)) continue;
        if (p.splits > 1) {
            const int64_t at_row = part_row<QUERY>(p, b, r / (QUERY ? p.group : 1), QUERY ? kvh * p.group + r % p.group : kvh);
            for (int c = 0; c < DP / 64; ++c) {
                const int d = c * 64 + tx * 4;
                store4(p.part_out + ((int64_t)blockIdx.z * part_rows<QUERY>(p) + at_row) * p.dim, d, p.dim, one[i][c], 1.f);
                if (!QUERY) store4(p.part_out + ((int64_t)(p.splits + blockIdx.z) * part_rows<QUERY>(p) + at_row) * p.dim, d, p.dim, two[i][c], 1.f);
            }
            continue;
        }
        for (int c = 0; c < DP / 64; ++c) {
            const int d = c * 64 + tx * 4;
            if (QUERY) store4((T*)p.dq + at(p.dqs, b, r / p.group, kvh * p.group + r % p.group), d, p.dim, one[i][c], 1.f);
            else {
                store4((T*)p.dk + at(p.dks, b, r, kvh), d, p.dim, one[i][c], 1.f);
                store4((T*)p.dv + at(p.dvs, b, r, kvh), d, p.dim, two[i][c], 1.f);
            }
        }
    }
}

// The parts of a split backward loop, added in order: a warp per row.
template <typename T, bool QUERY>
__global__ void __launch_bounds__(256) attn_backward_join(AttnParams p) {
    const int64_t rows = part_rows<QUERY>(p), row = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) % rows, which = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) / rows;
    if (which >= (QUERY ? 1 : 2)) return;
    const int heads = QUERY ? p.heads : p.kv_heads, len = QUERY ? p.q_len : p.k_len;
    const int h = row % heads, t = row / heads % len, b = row / heads / len;
    T* out = QUERY ? (T*)p.dq + at(p.dqs, b, t, h) : which ? (T*)p.dv + at(p.dvs, b, t, h) : (T*)p.dk + at(p.dks, b, t, h);
    for (int d = threadIdx.x & 31; d < p.dim; d += 32) {
        float v = 0.f;
        for (int s = 0; s < p.splits; ++s) v += p.part_out[((which * p.splits + s) * rows + row) * p.dim + d];
        out[d] = from_f32<T>(v);
    }
}

template <typename K>
void allow_smem(K kernel, int bytes) { ORMI_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)); }

int tiles(int64_t n, int per) {
    const int64_t t = (n + per - 1) / per;
    if (t > 0x7fffffff) throw Error("ormi_b200_attention: too many rows");
    return (int)t;
}

template <typename T, int BM, int BN, int DP>
void run_forward(ormi_b200_ctx* ctx, AttnParams& p) {
    const int smem = ((BM + 2 * BN) * (DP + 4) + BM * (BN + 4)) * 4;
    allow_smem(attn_forward<T, BM, BN, DP>, smem);
    const int rows = tiles((int64_t)p.q_len * p.group, BM), pairs = p.batch * p.kv_heads;
    // Few rows over many keys: the keys are split until there are two blocks per SM (four of the small ones, which wait for
    // their loads most of the time), each with two tiles of keys at least. Single tokens of 15 sequences over 11652
    // keys in fp32: 107 us; with half the blocks and four tiles at least, 163.
    const int key_tiles = std::max(1, (p.k_len + BN - 1) / BN);
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({((BM < 64 ? 4ll : 2ll) * ctx->num_sms + (int64_t)rows * pairs - 1) / ((int64_t)rows * pairs), key_tiles / 2, 128}));
    const size_t lines = (size_t)p.batch * p.heads * p.q_len;
    Scratch part(ctx, p.splits > 1 ? p.splits * lines * (p.dim + 2) * 4 : 0);
    if (p.splits > 1) {
        p.part_out = (float*)part.ptr;
        p.part_max = p.part_out + p.splits * lines * p.dim;
        p.part_sum = p.part_max + p.splits * lines;
    }
    attn_forward<T, BM, BN, DP><<<dim3(rows, pairs, p.splits), kThreads, smem, ctx->stream>>>(p);
    ORMI_CUDA(cudaGetLastError());
    count_launch(ctx);
    if (p.splits > 1) attention_join(ctx, p, sizeof(T) == 4 ? ORMI_F32 : ORMI_BF16);
    part.release();
}

// Tiles of 64 rows have the best ratio of arithmetic to shared memory; where they would leave SMs idle, smaller ones spread the
// work (half the arithmetic per load, four times the blocks), and up to 16 rows would be mostly padding in them. With head_dim
// 65 to 128, 64 rows take 32 keys at a time: 77 KB and two blocks per SM, where 64 keys (119 KB) leave one (800 tokens: 127 against 134 us).
bool spread(ormi_b200_ctx* ctx, const AttnParams& p, int64_t rows) { return (rows + 63) / 64 * p.batch * p.kv_heads < ctx->num_sms; }

template <typename T>
void forward_by_size(ormi_b200_ctx* ctx, AttnParams& p) {
    const int64_t rows = (int64_t)p.q_len * p.group;
    const int tile = rows <= 16 ? 16 : spread(ctx, p, rows) ? 32 : 64;
    if (p.dim <= 64) { if (tile == 16) run_forward<T, 16, 64, 64>(ctx, p); else if (tile == 32) run_forward<T, 32, 64, 64>(ctx, p); else run_forward<T, 64, 64, 64>(ctx, p); }
    else if (p.dim <= 128) { if (tile == 16) run_forward<T, 16, 64, 128>(ctx, p); else if (tile == 32) run_forward<T, 32, 64, 128>(ctx, p); else run_forward<T, 64, 32, 128>(ctx, p); }
    else { if (tile == 16) run_forward<T, 16, 32, 256>(ctx, p); else run_forward<T, 64, 32, 256>(ctx, p); }
}

template <typename T, int B, int DP, bool QUERY>
void run_backward(ormi_b200_ctx* ctx, AttnParams& p) {
    const int smem = (4 * B * (DP + 4) + 2 * B * (B + 4)) * 4;
    auto kernel = attn_backward<T, B, DP, QUERY>;
    const int64_t rows = QUERY ? (int64_t)p.q_len * p.group : p.k_len;
    if (!rows) return;
    allow_smem(kernel, smem);
    const int blocks_x = tiles(rows, B), pairs = p.batch * p.kv_heads;
    // Too few blocks for two per SM: the loop is cut, with two turns left for each part, and the parts are added afterwards
    // (333 tokens, 4 heads over 2, head_dim 40, fp32: 179 -> 81 us for the whole backward pass).
    const int64_t turns = ((QUERY ? (int64_t)p.k_len : (int64_t)p.q_len * p.group) + B - 1) / B;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({2ll * ctx->num_sms / ((int64_t)blocks_x * pairs), turns / 2, 16}));
    Scratch part(ctx, p.splits > 1 ? (size_t)p.splits * (QUERY ? 1 : 2) * part_rows<QUERY>(p) * p.dim * 4 : 0);
    p.part_out = (float*)part.ptr;
    kernel<<<dim3(blocks_x, pairs, p.splits), kThreads, smem, ctx->stream>>>(p);
    ORMI_CUDA(cudaGetLastError());
    count_launch(ctx);
    if (p.splits > 1) {
        attn_backward_join<T, QUERY><<<tiles(part_rows<QUERY>(p) * (QUERY ? 1 : 2), 8), 256, 0, ctx->stream>>>(p);
        ORMI_CUDA(cudaGetLastError());
        count_launch(ctx);
    }
    part.release();
}

template <typename T, bool QUERY>
void backward_by_size(ormi_b200_ctx* ctx, AttnParams& p) {
    const bool small = spread(ctx, p, QUERY ? (int64_t)p.q_len * p.group : p.k_len);
    if (p.dim <= 64) { if (small) run_backward<T, 32, 64, QUERY>(ctx, p); else run_backward<T, 64, 64, QUERY>(ctx, p); }
    else if (p.dim <= 128) { if (small) run_backward<T, 32, 128, QUERY>(ctx, p); else run_backward<T, 64, 128, QUERY>(ctx, p); }
    else run_backward<T, 32, 256, QUERY>(ctx, p);
}

}  // namespace

void attention_simple(ormi_b200_ctx* ctx, AttnParams& p, int dtype) {
    if (dtype == ORMI_F32) forward_by_size<float>(ctx, p); else forward_by_size<bf16>(ctx, p);
}

void attention_backward_simple(ormi_b200_ctx* ctx, AttnParams& p, int dtype) {
    if (dtype == ORMI_F32) { backward_by_size<float, false>(ctx, p); backward_by_size<float, true>(ctx, p); }
    else { backward_by_size<bf16, false>(ctx, p); backward_by_size<bf16, true>(ctx, p); }
}

void attention_join(ormi_b200_ctx* ctx, const AttnParams& p, int dtype) {
    const int64_t lines = (int64_t)p.batch * p.heads * p.q_len;
    if (dtype == ORMI_F32) attn_join<float><<<tiles(lines, 1), 128, 0, ctx->stream>>>(p); else attn_join<bf16><<<tiles(lines, 1), 128, 0, ctx->stream>>>(p);
    ORMI_CUDA(cudaGetLastError());
    count_launch(ctx);
}

void attention_delta(ormi_b200_ctx* ctx, const AttnParams& p, int dtype) {
    const int64_t lines = (int64_t)p.batch * p.heads * p.q_len;
    if (!lines) return;
    if (dtype == ORMI_F32) attn_delta<float><<<tiles(lines, 8), 256, 0, ctx->stream>>>(p); else attn_delta<bf16><<<tiles(lines, 8), 256, 0, ctx->stream>>>(p);
    ORMI_CUDA(cudaGetLastError());
    count_launch(ctx);
}

// ------------------------------------------------------------------------------------------------ arguments
namespace {

void heads_check(const char* op, const char* name, const ormi_b200_view& v, const ormi_b200_view& like, bool same_shape, bool output) {
    view_check(op, name, v, 4, 4);
    auto n = [&] { return std::string(name); };
    OP_NEED(v.dtype == like.dtype, op, n() + " has another type than q");
    OP_NEED(v.shape[3] <= 1 || v.strides[3] == 1, op, n() + ": head_dim is not contiguous");
    if (same_shape) for (int d = 0; d < 4; ++d) OP_NEED(v.shape[d] == like.shape[d], op, n() + " has another shape");
    if (output && count_of(v)) {
        // rows of head_dim values that lie apart: sorted by stride, each dimension steps over everything inside it
        int order[3] = {0, 1, 2};
        std::sort(order, order + 3, [&](int a, int b) { return v.strides[a] < v.strides[b]; });
        int64_t inner = v.shape[3];
        for (int d : order) {
            if (v.shape[d] <= 1) continue;
            OP_NEED(v.strides[d] >= inner, op, n() + ": its rows overlap");
            inner = (v.shape[d] - 1) * v.strides[d] + inner;
        }
    }
}

void ints_check(const char* op, const char* name, const ormi_b200_view& v, int64_t rows, int64_t cols) {
    if (!v.data) return;
    view_check(op, name, v, cols < 0 ? 1 : 2, cols < 0 ? 1 : 2);
    OP_NEED(v.dtype == ORMI_I32 && contiguous(v) && v.shape[0] == rows && (cols < 0 || v.shape[1] == cols), op,
            std::string(name) + (cols < 0 ? " is not [batch] I32, contiguous" : " is not [batch, length] I32, contiguous"));
}

void forward_check(const char* op, const ormi_b200_attention_args& a, bool backward) {
    view_check(op, "q", a.q, 4, 4);
    OP_NEED(a.q.dtype == ORMI_F32 || a.q.dtype == ORMI_BF16, op, "q is F32 or BF16");
    heads_check(op, "q", a.q, a.q, true, false);
    heads_check(op, "k", a.k, a.q, false, false);
    heads_check(op, "v", a.v, a.k, true, false);
    heads_check(op, "out", a.out, a.q, true, !backward);
    const int64_t b = a.q.shape[0], nq = a.q.shape[1], h = a.q.shape[2], d = a.q.shape[3], nk = a.k.shape[1], hk = a.k.shape[2];
    OP_NEED(a.k.shape[0] == b && a.k.shape[3] == d, op, "k has another batch or head_dim than q");
    OP_NEED(d >= 1 && d <= 256, op, "head_dim is 1 to 256");
    OP_NEED(h == 0 || (hk >= 1 && h % hk == 0), op, "heads is not a multiple of kv_heads");
    OP_NEED(h > 0 || hk == 0, op, "heads is zero");
    OP_NEED(b * hk <= 65535, op, "batch * kv_heads is above 65535");
    OP_NEED(b * h * nq <= (int64_t)1 << 30 && nk <= (int64_t)1 << 30, op, "batch * heads * q_len or k_len is above 2^30");
    if (a.lse.data || backward) {
        view_check(op, "lse", a.lse, 3, 3);
        OP_NEED(a.lse.dtype == ORMI_F32 && contiguous(a.lse) && a.lse.shape[0] == b && a.lse.shape[1] == h && a.lse.shape[2] == nq, op, "lse is not [batch, heads, q_len] F32, contiguous");
    }
    if (a.slopes.data) {
        view_check(op, "slopes", a.slopes, 1, 1);
        OP_NEED(a.slopes.dtype == ORMI_F32 && contiguous(a.slopes) && a.slopes.shape[0] == h, op, "slopes is not [heads] F32, contiguous");
    }
    OP_NEED((a.q_docs.ndim == 0) == (a.k_docs.ndim == 0), op, "q_docs and k_docs go together");
    ints_check(op, "q_docs", a.q_docs, b, nq);
    ints_check(op, "k_docs", a.k_docs, b, nk);
    ints_check(op, "prefix", a.prefix, b, -1);
    ints_check(op, "key_len", a.key_len, b, -1);
    ints_check(op, "q_start", a.q_start, b, -1);
    OP_NEED(std::isfinite(a.scale), op, "scale is not finite");
    OP_NEED(a.cap >= 0.f && std::isfinite(a.cap), op, "cap is negative or not finite");
    OP_NEED(a.cap == 0.f || std::isfinite(1.f / a.cap), op, "cap is too small: 1 / cap is not finite");
}

// Whether two views whose spans overlap are slices of one buffer that never meet, such as the gradients of q, k and v side by
// side in every position: for a stride that both step by, one lies behind the other within its period.
bool side_by_side(const ormi_b200_view& a, const ormi_b200_view& b) {
    const ormi_b200_view &lo = a.data <= b.data ? a : b, &hi = a.data <= b.data ? b : a;
    if (((const char*)hi.data - (const char*)lo.data) % dtype_bytes(lo.dtype)) return false;
    const int64_t off = ((const char*)hi.data - (const char*)lo.data) / dtype_bytes(lo.dtype);
    auto inner = [](const ormi_b200_view& v, int64_t period) {       // extent of what steps by less than the period
        int64_t last = 0;
        for (int d = 0; d < v.ndim; ++d) if (v.strides[d] < period) last += (v.shape[d] - 1) * v.strides[d];
        return last + 1;
    };
    for (int d = 0; d < 3; ++d) {
        const int64_t period = lo.strides[d];
        if (period <= 0) continue;
        // everything that steps by the period or more steps by a multiple of it, in both
        bool both = true;
        for (auto* v : {&lo, &hi}) for (int e = 0; e < v->ndim; ++e) both = both && (v->shape[e] <= 1 || v->strides[e] < period || v->strides[e] % period == 0);
        if (both && off % period >= inner(lo, period) && off % period + inner(hi, period) <= period) return true;
    }
    return false;
}

struct Named { const char* name; const ormi_b200_view* v; };

void apart_check(const char* op, const std::vector<Named>& outs, const std::vector<Named>& ins) {
    for (size_t i = 0; i < outs.size(); ++i) {
        for (auto& in : ins) OP_NEED(!overlap(*outs[i].v, *in.v), op, std::string(outs[i].name) + " overlaps " + in.name);
        for (size_t j = 0; j < i; ++j)
            OP_NEED(!overlap(*outs[i].v, *outs[j].v) || side_by_side(*outs[i].v, *outs[j].v), op, std::string(outs[i].name) + " overlaps " + outs[j].name);
    }
}

std::vector<Named> inputs_of(const ormi_b200_attention_args& a) {
    return {{"q", &a.q}, {"k", &a.k}, {"v", &a.v}, {"slopes", &a.slopes}, {"q_docs", &a.q_docs}, {"k_docs", &a.k_docs}, {"prefix", &a.prefix}, {"key_len", &a.key_len}, {"q_start", &a.q_start}};
}

Strides4 strides_of(const ormi_b200_view& v) { return {v.strides[0], v.strides[1], v.strides[2]}; }

AttnParams params_of(const ormi_b200_attention_args& a) {
    AttnParams p{};
    p.q = a.q.data; p.k = a.k.data; p.v = a.v.data; p.out = a.out.data; p.lse = (float*)a.lse.data;
    p.slopes = (const float*)a.slopes.data;
    p.q_docs = (const int32_t*)a.q_docs.data; p.k_docs = (const int32_t*)a.k_docs.data;
    p.prefix = (const int32_t*)a.prefix.data; p.key_len = (const int32_t*)a.key_len.data; p.q_start = (const int32_t*)a.q_start.data;
    p.qs = strides_of(a.q); p.ks = strides_of(a.k); p.vs = strides_of(a.v); p.os = strides_of(a.out);
    p.batch = (int)a.q.shape[0]; p.q_len = (int)a.q.shape[1]; p.heads = (int)a.q.shape[2]; p.dim = (int)a.q.shape[3];
    p.k_len = (int)a.k.shape[1]; p.kv_heads = (int)a.k.shape[2]; p.group = p.kv_heads ? p.heads / p.kv_heads : 1;
    p.causal = a.causal != 0; p.scale = a.scale; p.cap = a.cap; p.inv_cap = a.cap > 0.f ? 1.f / a.cap : 0.f;
    p.splits = 1;
    return p;
}

}  // namespace

void attention_check(const ormi_b200_attention_args& a) {
    forward_check("attention", a, false);
    apart_check("attention", {{"out", &a.out}, {"lse", &a.lse}}, inputs_of(a));
}

void attention(ormi_b200_ctx* ctx, const ormi_b200_attention_args& a) {
    AttnParams p = params_of(a);
    if (!p.batch || !p.q_len || !p.heads) return;
    written(ctx, a.out);
    written(ctx, a.lse);
    // up to 64 packed rows: a tile of 128 queries of one head would be mostly padding
    if (attention_few_supported(p, a.q.dtype)) attention_few(ctx, p);
    else if (attention_tc_supported(p, a.q.dtype)) attention_tc(ctx, p);
    else attention_simple(ctx, p, a.q.dtype);
}

void attention_backward_check(const ormi_b200_attention_backward_args& a) {
    const char* op = "attention_backward";
    const ormi_b200_attention_args& f = a.forward;
    forward_check(op, f, true);
    heads_check(op, "dout", a.dout, f.q, true, false);
    heads_check(op, "dq", a.dq, f.q, true, true);
    heads_check(op, "dk", a.dk, f.k, true, true);
    heads_check(op, "dv", a.dv, f.k, true, true);
    auto ins = inputs_of(f);
    ins.push_back({"out", &f.out}); ins.push_back({"lse", &f.lse}); ins.push_back({"dout", &a.dout});
    apart_check(op, {{"dq", &a.dq}, {"dk", &a.dk}, {"dv", &a.dv}}, ins);
}

void attention_backward(ormi_b200_ctx* ctx, const ormi_b200_attention_backward_args& a) {
    AttnParams p = params_of(a.forward);
    if (!p.batch || !p.kv_heads) return;
    p.dout = a.dout.data; p.dq = a.dq.data; p.dk = a.dk.data; p.dv = a.dv.data;
    p.dos = strides_of(a.dout); p.dqs = strides_of(a.dq); p.dks = strides_of(a.dk); p.dvs = strides_of(a.dv);
    for (auto* v : {&a.dq, &a.dk, &a.dv}) written(ctx, *v);
    Scratch delta(ctx, (size_t)p.batch * p.heads * p.q_len * 4);
    p.delta = (float*)delta.ptr;
    if (attention_backward_tc_supported(p, a.forward.q.dtype)) {
        attention_backward_tc(ctx, p);
    } else {
        attention_delta(ctx, p, a.forward.q.dtype);
        attention_backward_simple(ctx, p, a.forward.q.dtype);
    }
    delta.release();
}

}  // namespace ormi_b200
