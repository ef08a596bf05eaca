// Forward attention on the tensor cores: bf16, head_dim up to 128.
//
// A block owns 256 queries of one head, as two tiles of 128 rows, and walks the tiles of 128 keys that any of them sees.
// Warp 0 loads (TMA: Q once, K and V through a ring), warp 1 issues the products (tcgen05), warp 2 blanks the rows of V
// behind key_len, and a warpgroup per tile of queries turns scores into probabilities: a thread owns a row, so the running
// maximum and sum of the softmax need no exchange.  In tensor memory a tile has its scores S (128 columns), overwritten in
// place by the probabilities as bf16, which the second product reads as its A operand, and its output O.  While one
// warpgroup works on its scores the tensor cores run the other tile's products.
//
// Bound by the chain of one warpgroup: its scores, 340 clocks for a maximum over 128 columns, 1330 for the exponentials (1024
// at the special function unit's rate), 512 for the product with V and 512 for the next scores; two tiles of queries are
// what tensor memory holds at head_dim 128.  8192 tokens, 16 heads, causal: 240 us, 1147 TFLOP/s over the visible pairs alone
// at 1965 MHz, 273 us in a loop, where the power limit leaves 1710 MHz; with distance bias 320 and 337 us.
//
// O is rescaled only when a row's maximum has grown by more than 2^8 since the last time: probabilities up to 256 lose
// nothing in fp32 sums nor, relatively, in bf16.
#include <algorithm>
#include <cmath>
#include <limits>

#include "attention_tc.cuh"

namespace ormi_b200 {
namespace {

using namespace tc;

constexpr int kThreads = 384;                    // warps 0-3: load, multiply, blank, (idle); 4-7 and 8-11: softmax of a tile each

template <int DP> struct ForwardShape {
    static constexpr int kOperand = kTile * DP * 2;            // bytes of a tile of Q, K or V
    static constexpr int kStages = DP == 128 ? 4 : 8;
    static constexpr int kSmem = 1024 + (2 + kStages) * kOperand + kMaxTiles + 8 * 512 + 256;
};

template <int DP, bool CAP, bool BIAS, bool DOCS>
__global__ void __launch_bounds__(kThreads, 1)
attn_forward_tc(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ TcParams p) {
    using Shape = ForwardShape<DP>;
    constexpr int ST = Shape::kStages, OP = Shape::kOperand;
    extern __shared__ unsigned char raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    unsigned char* mem = raw + (base - smem_u32(raw));
    const uint32_t q_at = base, ring = base + 2 * OP;
    unsigned char* cls = mem + (2 + ST) * OP;                  // two bits for each tile of queries
    int* docs = reinterpret_cast<int*>(cls + kMaxTiles);       // 128 for each softmax warp
    const uint32_t bars = smem_u32(docs + 8 * 128);
    const uint32_t q_full = bars, v_blank = bars + 8, blank_go = bars + 16;
    auto s_full = [&](int w) { return bars + 24 + 8 * w; };
    auto o_full = [&](int w) { return bars + 40 + 8 * w; };
    auto p_full = [&](int w) { return bars + 56 + 8 * w; };
    auto kv_full = [&](int s) { return bars + 72 + 8 * s; };
    auto kv_empty = [&](int s) { return bars + 72 + 8 * (ST + s); };
    __shared__ uint32_t tmem_slot;
    __shared__ Abort ab;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = blockIdx.x / p.a.heads, h = blockIdx.x % p.a.heads, kvh = h / p.a.group;
    const int q0 = (int)(gridDim.y - 1 - blockIdx.y) * 2 * kTile;         // causal: the longest rows first
    const RowMask m = row_mask(p.a, b);
    // key_end of the first and the last query of each tile
    int lo[2], hi[2];
    for (int w = 0; w < 2; ++w) {
        const int first = q0 + w * kTile, last = min(first + kTile, p.a.q_len) - 1;
        lo[w] = key_end(m, m.start + first);
        hi[w] = first < p.a.q_len ? key_end(m, m.start + last) : 0;
    }
    const int tiles = (max(max(hi[0], hi[1]), 0) + kTile - 1) / kTile;
    const int blank_tile = m.keys < p.a.k_len && m.keys % kTile ? m.keys / kTile : -1;
    if (threadIdx.x == 0) {
        ab.flag = 0; ab.err = p.err;
        mbar_init(q_full, 1); mbar_init(v_blank, 1); mbar_init(blank_go, 1);
        for (int w = 0; w < 2; ++w) { mbar_init(s_full(w), 1); mbar_init(o_full(w), 1); mbar_init(p_full(w), 4); }
        for (int s = 0; s < ST; ++s) { mbar_init(kv_full(s), 1); mbar_init(kv_empty(s), 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        // Q does not depend on the classes: it is on its way while they are being worked out
        mbar_expect_tx(q_full, 2 * OP);
        for (int w = 0; w < 2; ++w)
            for (int x = 0; x < DP / 64; ++x) tma_load_4d(q_at + w * OP + x * box_bytes(kTile), &map_q, q_full, 64 * x, q0 + w * kTile, h, b);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // classes of the tiles, and which union tile holds the last valid key in its middle
    for (int j = threadIdx.x; j < tiles; j += kThreads) {
        int c = 0;
        for (int w = 0; w < 2; ++w) c |= tile_class(p, b, q0 / kUnit + 2 * w, lo[w], hi[w], 2 * j) << (2 * w);
        cls[j] = (unsigned char)c;
    }
    fence_before();
    __syncthreads();
    fence_after();
    // all of tensor memory is this block's, so it starts at column 0 (checked: every address below is a constant)
    constexpr uint32_t tmem = 0;
    const bool whole = tmem_slot == tmem;
    if (!whole && threadIdx.x == 0) atomicCAS(p.err, 0, 20);
    auto s_at = [&](int w) { return tmem + w * 128; };
    auto o_at = [&](int w) { return tmem + 256 + w * 128; };

    if (!whole) {
    } else if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 0 && lane == 0) {
            // ---------------------------------------------------------------- loads
            int seq = 0;
            bool ok = true;
            for (int j = 0; j < tiles && ok; ++j) {
                if (!cls[j]) continue;
                for (int kv = 0; kv < 2 && ok; ++kv, ++seq) {
                    const int s = seq % ST;
                    ok = mbar_wait(kv_empty(s), (seq / ST & 1) ^ 1, ab, 21);
                    if (!ok) break;
                    mbar_expect_tx(kv_full(s), OP);
                    for (int x = 0; x < DP / 64; ++x) tma_load_4d(ring + s * OP + x * box_bytes(kTile), kv ? &map_v : &map_k, kv_full(s), 64 * x, j * kTile, kvh, b);
                }
            }
            // nothing of this block's is in flight when it leaves
            ok = ok && mbar_wait(q_full, 0, ab, 21);
            for (int i = 0; i < ST && ok; ++i, ++seq) ok = mbar_wait(kv_empty(seq % ST), (seq / ST & 1) ^ 1, ab, 21);
        } else if (warp == 1) {
            // ---------------------------------------------------------------- products
            int u = -1, prev = 0, prev_j = -1, used_p[2] = {0, 0}, last[2] = {tiles - 1, tiles - 1};
            for (int w = 0; w < 2; ++w) while (last[w] >= 0 && !(cls[last[w]] >> (2 * w) & 3)) --last[w];
            bool ok = warp_wait(q_full, 0, ab, 22);
            for (int j = 0; j <= tiles && ok; ++j) {
                const int c = j < tiles ? cls[j] : 0;
                if (!c && j < tiles) continue;
                if (c) ++u;
                const int k_seq = 2 * u, v_seq = (c ? 2 * (u - 1) : 2 * u) + 1;      // K of this tile, V of the one before
                const uint32_t k_buf = ring + (k_seq % ST) * OP, v_buf = ring + (v_seq % ST) * OP;
                bool have_k = false, have_v = false;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    if (!ok) break;
                    if (prev >> (2 * w) & 3) {
                        if (!have_v) {
                            ok = warp_wait(kv_full(v_seq % ST), v_seq / ST & 1, ab, 23);
                            if (ok && prev_j == blank_tile) {              // warp 2 may begin: these rows have landed
                                if (lane == 0) mbar_arrive(blank_go);
                                ok = warp_wait(v_blank, 0, ab, 24);
                            }
                            have_v = true;
                        }
                        ok = ok && warp_wait(p_full(w), used_p[w] & 1, ab, 25);
                        if (!ok) break;
                        fence_after();
                        if (elect()) {
                            product_tn<DP>(o_at(w), s_at(w), v_buf, used_p[w] > 0);
                            if (prev_j == last[w]) commit(o_full(w));
                        }
                        ++used_p[w];
                    }
                    if (c >> (2 * w) & 3) {
                        if (!have_k) { ok = warp_wait(kv_full(k_seq % ST), k_seq / ST & 1, ab, 26); have_k = true; }
                        if (!ok) break;
                        fence_after();
                        if (elect()) {
                            product_nt<DP, kTile>(s_at(w), q_at + w * OP, k_buf);
                            commit(s_full(w));
                        }
                    }
                }
                if (!ok) break;
                if (elect()) {
                    if (prev) commit(kv_empty(v_seq % ST));
                    if (c) commit(kv_empty(k_seq % ST));
                }
                prev = c;
                prev_j = j;
            }
        } else if (warp == 2 && blank_tile >= 0 && blank_tile < tiles && cls[blank_tile]) {
            // ---------------------------------------------------------------- rows of V behind key_len: zero, whatever they held
            // (the issuer says when V has landed: a parity wait of this warp's own on the ring could be a phase late or early)
            int u = 0;
            for (int j = 0; j < blank_tile; ++j) u += cls[j] != 0;
            const int s = (2 * u + 1) % ST;
            if (warp_wait(blank_go, 0, ab, 27)) {
                const int first = m.keys % kTile;
                for (int x = 0; x < DP / 64; ++x)
                    for (int i = first * 8 + lane; i < kTile * 8; i += 32)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(ring + s * OP + x * box_bytes(kTile) + i * 16), "r"(0) : "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(v_blank);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // -------------------------------------------------------------------- softmax: one row per thread
        const int w = warp / 4 - 1;
        const int t = q0 + w * kTile + (threadIdx.x & 127);
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;                       // this warp's 32 lanes of tensor memory
        const bool live = t < p.a.q_len;
        const int pos = m.start + t, end = live ? key_end(m, pos) : 0;
        const int my_doc = DOCS && live ? m.q_docs[t] : 0;
        const float slope = BIAS ? p.a.slopes[h] * kLog2e : 0.f;
        int* my_docs = docs + (warp - 4) * 128;
        float top = -INFINITY, total = 0.f;
        int n = 0;
        bool ok = true;
        auto class_at = [&](int j) { return cls[j] >> (2 * w) & 3; };
        auto next_tile = [&](int j) { do ++j; while (j < tiles && class_at(j) == kSkip); return j; };
        int ahead[4];                                            // documents of the tile to come, asked for a tile ahead
        auto fetch = [&](int j) {
            if (DOCS && j < tiles && class_at(j) == kDocs)
#pragma unroll
                for (int k = 0; k < 4; ++k) ahead[k] = j * kTile + k * 32 + lane < p.a.k_len ? m.k_docs[j * kTile + k * 32 + lane] : 0;
        };
        int next = next_tile(-1);
        fetch(next);
        while (next < tiles) {
            const int j = next, c = class_at(j), key0 = j * kTile;
            if (DOCS && c == kDocs) {
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 4; ++k) my_docs[k * 32 + lane] = ahead[k];
                __syncwarp();
            }
            next = next_tile(j);
            fetch(next);
            ok = warp_wait(s_full(w), n & 1, ab, 28);
            if (!ok) break;
            fence_after();
            float2 z[64];
#pragma unroll
            for (int i = 0; i < 4; ++i) ld32(s_at(w) + lanes + 32 * i, reinterpret_cast<uint32_t*>(z) + 32 * i);
            wait_ld();
            // With neither cap nor bias the raw products go through max and exponential as they are, the scale (positive)
            // riding on the subtraction of the maximum.
            constexpr bool PLAIN = !CAP && !BIAS;
            if (CAP) {
                if (cap_is_polynomial<64>(p.cap, z)) {
#pragma unroll
                    for (int i = 0; i < 64; ++i) z[i] = cap_polynomial(p.cap, z[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 64; ++i) z[i] = cap_any(p.cap, z[i]);
                }
            }
            if (BIAS) {
                const float ahead = (float)(pos - key0);
                if (__all_sync(0xffffffffu, pos - key0 >= kTile - 1)) {          // every key at or before the query: the distance is linear
                    const float first = -slope * ahead;
#pragma unroll
                    for (int i = 0; i < 64; ++i) {
                        const float2 far = fma2(both(slope), make_float2((float)(2 * i), (float)(2 * i + 1)), both(first));
                        z[i] = CAP ? add2(z[i], far) : fma2(z[i], both(p.scale_log2), far);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 64; ++i) {
                        if (!CAP) z[i] = mul2(z[i], both(p.scale_log2));
                        z[i] = make_float2(fmaf(-slope, fabsf(ahead - (float)(2 * i)), z[i].x), fmaf(-slope, fabsf(ahead - (float)(2 * i + 1)), z[i].y));
                    }
                }
            }
            if (DOCS && c == kDocs) {
#pragma unroll
                for (int i = 0; i < 64; i += 2) {
                    const int4 d = *reinterpret_cast<const int4*>(&my_docs[2 * i]);
                    if (d.x != my_doc) z[i].x = -INFINITY;
                    if (d.y != my_doc) z[i].y = -INFINITY;
                    if (d.z != my_doc) z[i + 1].x = -INFINITY;
                    if (d.w != my_doc) z[i + 1].y = -INFINITY;
                }
            }
            if (c >= kPartial) {
                const int left = end - key0;
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    if (2 * i >= left) z[i].x = -INFINITY;
                    if (2 * i + 1 >= left) z[i].y = -INFINITY;
                }
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 64; ++i) mx[i & 3] = max3(mx[i & 3], z[i].x, z[i].y);
            const float seen = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            const float big = fmaxf(top, PLAIN ? seen * p.scale_log2 : seen);
            if (__any_sync(0xffffffffu, big > top + 8.f)) {
                const float by = big == -INFINITY ? 1.f : ex2(top - big);
                top = big;
                total *= by;
                if (n) {                                       // the product before this tile's scores is complete: commits are in order
#pragma unroll 1
                    for (int x = 0; x < DP; x += 32) {
                        uint32_t o[32];
                        ld32(o_at(w) + lanes + x, o);
                        wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
                        st32(o_at(w) + lanes + x, o);
                    }
                }
            }
            const float from = top == -INFINITY ? 0.f : top;
            float2 sum[2] = {both(0.f), both(0.f)};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                uint32_t pk[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 a = PLAIN ? fma2(z[16 * x + i], both(p.scale_log2), both(-from)) : add2(z[16 * x + i], both(-from));
                    const float2 e = make_float2(ex2(a.x), ex2(a.y));
                    sum[i & 1] = add2(sum[i & 1], e);
                    pk[i] = pack_bf16x2(e.x, e.y);
                }
                st16(s_at(w) + lanes + 16 * x, pk);
            }
            total += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(w));
            ++n;
        }
        // (a warpgroup that saw no key still waits for its queries: their memory is written below)
        if (ok) ok = n ? warp_wait(o_full(w), 0, ab, 29) : warp_wait(q_full, 0, ab, 29);
        if (ok) {
            fence_after();
            const float by = total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;
            // this warpgroup's queries have been multiplied for the last time: their memory stages the rows
            const int t0 = q0 + w * kTile + (warp & 3) * 32;
            bf16* out = (bf16*)p.a.out + (int64_t)b * p.a.os.b + (int64_t)t0 * p.a.os.t + (int64_t)h * p.a.os.h;
            store_rows<DP>(o_at(w) + lanes, n > 0, q_at + (warp - 4) * (64 * DP), by, p.a.q_len - t0, p.a.dim, [&](int r) { return out + r * p.a.os.t; });
            if (live && p.a.lse) p.a.lse[((int64_t)b * p.a.heads + h) * p.a.q_len + t] = top == -INFINITY ? -INFINITY : (top + log2f(total)) * kLn2;
        }
    }
    // ------------------------------------------------------------------------ teardown
    __syncwarp();
    if (ab.flag) {                                             // let copies that are still in flight land before the block goes away
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 200000ull) { }
    }
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_slot), "r"(512) : "memory");
    }
}

// Smallest and largest document of every unit of 64 positions, of the queries and then of the keys: a warp per unit.
__global__ void __launch_bounds__(256) attn_doc_bounds(TcParams p, int2* bounds) {
    int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t q_count = (int64_t)p.a.batch * p.q_units;
    if (at >= q_count + (int64_t)p.a.batch * p.k_units) return;
    bounds += at;
    const bool keys = at >= q_count;
    if (keys) at -= q_count;
    const int units = keys ? p.k_units : p.q_units, len = keys ? p.a.k_len : p.a.q_len;
    const int32_t* docs = (keys ? p.a.k_docs : p.a.q_docs) + at / units * len;
    const int first = at % units * kUnit + (threadIdx.x & 31);
    int lo = INT32_MAX, hi = INT32_MIN;
    for (int i = first; i < min(first + kUnit, len); i += 32) { lo = min(lo, docs[i]); hi = max(hi, docs[i]); }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if ((threadIdx.x & 31) == 0) *bounds = make_int2(lo, hi);
}

template <int DP, bool CAP, bool BIAS, bool DOCS>
void launch_forward(ormi_b200_ctx* ctx, const CUtensorMap* maps, const TcParams& p) {
    auto kernel = attn_forward_tc<DP, CAP, BIAS, DOCS>;
    constexpr int smem = ForwardShape<DP>::kSmem;
    ORMI_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    kernel<<<dim3(p.a.batch * p.a.heads, (p.a.q_len + 2 * kTile - 1) / (2 * kTile)), kThreads, smem, ctx->stream>>>(maps[0], maps[1], maps[2], p);
    ORMI_CUDA(cudaGetLastError());
    count_launch(ctx);
}

template <int DP>
void launch_by_mask(ormi_b200_ctx* ctx, const CUtensorMap* maps, const TcParams& p) {
    const bool cap = p.a.cap > 0.f, bias = p.a.slopes, docs = p.a.k_docs;
    if (cap) {
        if (bias) docs ? launch_forward<DP, true, true, true>(ctx, maps, p) : launch_forward<DP, true, true, false>(ctx, maps, p);
        else docs ? launch_forward<DP, true, false, true>(ctx, maps, p) : launch_forward<DP, true, false, false>(ctx, maps, p);
    } else {
        if (bias) docs ? launch_forward<DP, false, true, true>(ctx, maps, p) : launch_forward<DP, false, true, false>(ctx, maps, p);
        else docs ? launch_forward<DP, false, false, true>(ctx, maps, p) : launch_forward<DP, false, false, false>(ctx, maps, p);
    }
}

}  // namespace

// A 4-D map (head_dim, position, head, batch) with boxes of 64 values x `rows` positions: reads behind any extent give zero.
void head_map(ormi_b200_ctx* ctx, CUtensorMap* map, const void* ptr, const Strides4& s, int batch, int len, int heads, int dim, int rows) {
    cuuint64_t dims[4] = {(cuuint64_t)dim, (cuuint64_t)len, (cuuint64_t)heads, (cuuint64_t)batch};
    // the stride of an extent of one is never used, but is checked
    cuuint64_t strides[3] = {(cuuint64_t)(len > 1 ? s.t * 2 : 16), (cuuint64_t)(heads > 1 ? s.h * 2 : 16), (cuuint64_t)(batch > 1 ? s.b * 2 : 16)};
    cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, one[4] = {1, 1, 1, 1};
    ctx->drv.check(ctx->drv.TensorMapEncodeTiled(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(ptr), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                                 CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE),
                   "cuTensorMapEncodeTiled");
}

// TMA wants 16-byte addresses and strides; a stride of zero (a broadcast operand) is left to the other kernels.
bool map_allowed(const void* ptr, const Strides4& s, int batch, int len, int heads) {
    auto good = [](int64_t stride, int extent) { return extent <= 1 || (stride > 0 && stride % 8 == 0 && stride * 2 < (int64_t)1 << 40); };
    return (uintptr_t)ptr % 16 == 0 && good(s.b, batch) && good(s.t, len) && good(s.h, heads);
}

size_t bounds_bytes(const AttnParams& p) {
    // (the forward kernel looks at two tiles of queries, of which the second may not exist)
    return p.k_docs ? (size_t)p.batch * (units_of(p.q_len + kTile) + units_of(p.k_len)) * sizeof(int2) : 0;
}

CapTerms cap_terms(const AttnParams& a) {
    CapTerms t{};
    if (!(a.cap > 0.f)) return t;
    const double k = (double)a.scale / a.cap, c = (double)a.scale * 1.4426950408889634;
    static const double terms[4] = {0.9999999028730692, -0.333313732975708, 0.1327115660233386, -0.04756107721454571};
    t.cap_log2 = a.cap * kLog2e;
    // A coefficient below fp32's normal numbers (a cap far above any score) is worth nothing, so the polynomial ends where its
    // term would matter (2^-24 of the score); one above them (a cap far below) leaves no place for the polynomial at all.
    double limit = 0.4;
    for (int i = 0; i < 4; ++i) {
        t.poly[i] = (float)(c * terms[i] * std::pow(k, 2 * i));
        if (!std::isfinite(t.poly[i])) limit = -1;
        else if (i && std::abs(t.poly[i]) < std::numeric_limits<float>::min()) limit = std::min(limit, std::pow(0x1p-24 / std::abs(terms[i]), 0.5 / i));
    }
    t.poly_limit = (float)(limit < 0 ? -1 : std::min(limit / std::abs(k), 1e18));     // (its square is an fp32 number)
    t.exp_per_raw = (float)(2 * 1.4426950408889634 * k);
    t.minus_inv_cap2 = -1.f / (t.cap_log2 * t.cap_log2);
    return t;
}

TcParams tc_params(ormi_b200_ctx* ctx, const AttnParams& a, int2* bounds) {
    TcParams p{};
    p.a = a;
    p.q_units = units_of(a.q_len + kTile);
    p.k_units = units_of(a.k_len);
    p.scale_log2 = a.scale * kLog2e;
    p.cap = cap_terms(a);
    p.err = device_error_word(ctx);
    ctx->gemm_err_pending = true;
    if (a.k_docs) {
        int2* kb = bounds + (size_t)a.batch * p.q_units;
        attn_doc_bounds<<<(int)(((int64_t)a.batch * (p.q_units + p.k_units) + 7) / 8), 256, 0, ctx->stream>>>(p, bounds);
        ORMI_CUDA(cudaGetLastError());
        count_launch(ctx);
        p.q_bounds = bounds; p.k_bounds = kb;
    }
    return p;
}

// Scales and caps whose products with log2(e), ratio and square are fp32 numbers; others go to the kernels that use tanhf.
bool cap_terms_exist(const AttnParams& p) {
    const double scale = std::abs((double)p.scale), cap = p.cap;
    return scale <= 1e30 && (cap == 0 || (cap >= 1e-15 && cap <= 1e35 && scale <= 1e30 * cap));
}

bool attention_tc_supported(const AttnParams& p, int dtype) {
    return dtype == ORMI_BF16 && cap_terms_exist(p) && p.scale > 0.f && p.dim <= 128 && p.dim % 8 == 0 && p.k_len >= 1 && p.k_len <= kMaxTiles * kTile && p.q_len <= 65535 * 2 * kTile &&
           (int64_t)p.batch * p.heads < 0x7fffffff && map_allowed(p.q, p.qs, p.batch, p.q_len, p.heads) && map_allowed(p.k, p.ks, p.batch, p.k_len, p.kv_heads) &&
           map_allowed(p.v, p.vs, p.batch, p.k_len, p.kv_heads) && map_allowed(p.out, p.os, p.batch, p.q_len, p.heads);
}

void attention_tc(ormi_b200_ctx* ctx, AttnParams& a) {
    Scratch bounds(ctx, bounds_bytes(a));
    const TcParams p = tc_params(ctx, a, (int2*)bounds.ptr);
    CUtensorMap maps[3];
    head_map(ctx, &maps[0], a.q, a.qs, a.batch, a.q_len, a.heads, a.dim);
    head_map(ctx, &maps[1], a.k, a.ks, a.batch, a.k_len, a.kv_heads, a.dim);
    head_map(ctx, &maps[2], a.v, a.vs, a.batch, a.k_len, a.kv_heads, a.dim);
    if (a.dim <= 64) launch_by_mask<64>(ctx, maps, p); else launch_by_mask<128>(ctx, maps, p);
    bounds.release();
}

}  // namespace ormi_b200
