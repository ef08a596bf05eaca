// Attention of few queries over many keys (one new token of every sequence over its cache): bf16, head_dim up to 128.
//
// Bound by memory: every key and value is read once and takes part in as many products as there are packed rows (query x
// head of the group), 16 of which fill the tile of a warp-level product (mma.sync m16n8k16; the rows of a 128-row tensor-core
// tile would be padding).  A block takes a part of the keys of one key/value head; its four warps take 16 keys at a time in
// turn, each through a ring of its own that one lane fills by TMA, so no warp waits for another until the end, where
// their maxima, sums and outputs are joined through shared memory.  The parts of a head are joined by a second launch.
// Three blocks of 64 KB are resident per SM: a warp's chain of products and exponentials is long, so warps count for more
// than the depth of a ring (32 sequences over 8192 keys, 32 heads over 8: 6370 GB/s in a loop, 5820 alone behind a fill of the
// caches; two blocks of 96 KB 4950; lengths that differ from sequence to sequence 5900).
#include <algorithm>

#include "attention_tc.cuh"

namespace ormi_b200 {
namespace {

constexpr int kWarps = 4, kKeys = 16;
template <int DP> struct FewShape {
    static constexpr int kStages = 256 / DP;
    static constexpr int kStage = 2 * kKeys * DP * 2;            // bytes: 16 keys and 16 values
    static constexpr int kBoxes = 1024 + kWarps * kStages * kStage;
    static constexpr int kSmem = kBoxes > kWarps * 16 * (DP + 2) * 4 ? kBoxes : kWarps * 16 * (DP + 2) * 4;
};

__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The two packed rows of a thread: lane / 4 and that + 8.
struct FewRow { int t, h, pos, end, doc; float slope; bool live; };

template <int DP, bool CAP>
__global__ void __launch_bounds__(kWarps * 32, 3)
attn_few(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnParams p,
         const __grid_constant__ CapTerms cap, int part_keys, int* err) {
    constexpr int kStages = FewShape<DP>::kStages, kStage = FewShape<DP>::kStage, kBox16 = kKeys * 128;
    extern __shared__ unsigned char raw[];
    const uint32_t base = (tc::smem_u32(raw) + 1023u) & ~1023u;
    __shared__ __align__(8) unsigned long long bars[kWarps][kStages];
    __shared__ tc::Abort ab;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = blockIdx.y / p.kv_heads, kvh = blockIdx.y % p.kv_heads;
    const int rows = p.q_len * p.group, row0 = blockIdx.z * 16;
    const RowMask m = row_mask(p, b);
    FewRow r[2];
    int end = 0, all_end = INT32_MAX;                            // one past the last key that any row, or every row, of this tile may see
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int at = row0 + (lane >> 2) + 8 * i;
        r[i].live = at < rows;
        const int safe = r[i].live ? at : 0;
        r[i].t = safe / p.group;
        r[i].h = kvh * p.group + safe % p.group;
        r[i].pos = m.start + r[i].t;
        r[i].end = r[i].live ? key_end(m, r[i].pos) : 0;
        r[i].doc = m.q_docs ? m.q_docs[r[i].t] : 0;
        r[i].slope = p.slopes ? p.slopes[r[i].h] * kLog2e : 0.f;
        end = max(end, r[i].end);
        if (r[i].live) all_end = min(all_end, r[i].end);
    }
    end = __reduce_max_sync(0xffffffffu, end);
    all_end = m.k_docs ? 0 : __reduce_min_sync(0xffffffffu, all_end);
    const int first = blockIdx.x * part_keys, last = min(end, first + part_keys);
    // Q as A operands: rows lane / 4 and + 8, columns 2 (lane % 4) and + 8 of every 16
    uint32_t q[DP / 16][4];
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 16 * k + 8 * (i >> 1) + 2 * (lane & 3);
            const FewRow& x = r[i & 1];
            q[k][i] = x.live && d < p.dim ? *reinterpret_cast<const uint32_t*>((const bf16*)p.q + (int64_t)b * p.qs.b + (int64_t)x.t * p.qs.t + (int64_t)x.h * p.qs.h + d) : 0u;
        }
    const uint32_t ring = base + warp * (kStages * kStage);
    // boxes of 64 columns: 16 rows of 128 bytes, their 16-byte chunks c at c ^ (row & 7) (TMA's 128-byte swizzle)
    auto slot = [&](int stage, int which, int y, int c) { return ring + stage * kStage + (which * (DP / 64) + (c >> 3)) * kBox16 + y * 128 + (((c & 7) ^ (y & 7)) << 4); };
    auto bar = [&](int stage) { return tc::smem_u32(&bars[warp][stage]); };
    auto ask = [&](int key0, int stage) {
        if (key0 >= last || lane != 0) return;
        tc::mbar_expect_tx(bar(stage), kStage);
#pragma unroll
        for (int x = 0; x < DP / 64; ++x) {
            tc::tma_load_4d(ring + stage * kStage + x * kBox16, &map_k, bar(stage), 64 * x, key0, kvh, b);
            tc::tma_load_4d(ring + stage * kStage + (DP / 64 + x) * kBox16, &map_v, bar(stage), 64 * x, key0, kvh, b);
        }
    };
    if (threadIdx.x == 0) {
        ab.flag = 0; ab.err = err;
        for (int i = 0; i < kWarps * kStages; ++i) tc::mbar_init(tc::smem_u32(&bars[0][0]) + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    float o[DP / 8][4], top[2] = {-INFINITY, -INFINITY}, total[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    const float scale2 = p.scale * kLog2e;
    int key0 = first + warp * kKeys;
    for (int k = 0; k < kStages; ++k) ask(key0 + k * kWarps * kKeys, k);
    bool ok = true;
    for (int n = 0; key0 < last; key0 += kWarps * kKeys, ++n) {
        const int stage = n % kStages;
        ok = tc::warp_wait(bar(stage), n / kStages & 1, ab, 61);
        if (!ok) break;
        if (key0 + kKeys > m.keys) {                             // what lies behind key_len is blanked, whatever it held
            for (int i = lane; i < 2 * kKeys * (DP / 8); i += 32) {
                const int y = i / (DP / 8) % kKeys;
                if (key0 + y >= m.keys) asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(slot(stage, i / (DP / 8) / kKeys, y, i % (DP / 8))), "r"(0) : "memory");
            }
            __syncwarp();
        }
        float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
            uint32_t kb[4];
            ldmatrix(kb, slot(stage, 0, (lane >> 4) * 8 + (lane & 7), 2 * k + (lane >> 3 & 1)));
            mma16(s[0], q[k], kb[0], kb[1]);
            mma16(s[1], q[k], kb[2], kb[3]);
        }
        if (CAP) {
            // the polynomial wherever it holds: beyond it the cap is off by a few 1e-7 of the cap, whatever the score
            float2 z[4] = {{s[0][0], s[0][1]}, {s[0][2], s[0][3]}, {s[1][0], s[1][1]}, {s[1][2], s[1][3]}};
            const bool small = cap_is_polynomial<4>(cap, z);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float2 c = cap_polynomial(cap, z[i]);
                if (!small) {
                    const float2 far = cap_any(cap, z[i]);
                    if (!(fabsf(z[i].x) <= cap.poly_limit)) c.x = far.x;
                    if (!(fabsf(z[i].y) <= cap.poly_limit)) c.y = far.y;
                }
                s[i >> 1][2 * (i & 1)] = c.x; s[i >> 1][2 * (i & 1) + 1] = c.y;
            }
        } else {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] *= scale2;
        }
        if (p.slopes) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] -= r[i >> 1].slope * fabsf((float)(r[i >> 1].pos - (key0 + 8 * n + 2 * (lane & 3) + (i & 1))));
        }
        if (key0 + kKeys > all_end) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + 8 * n + 2 * (lane & 3) + (i & 1);
                    if (key >= r[i >> 1].end || (m.k_docs && m.k_docs[key] != r[i >> 1].doc)) s[n][i] = -INFINITY;
                }
        }
        float big[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) big[i] = fmaxf(top[i], fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1])));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            big[i] = fmaxf(big[i], __shfl_xor_sync(0xffffffffu, big[i], 1));
            big[i] = fmaxf(big[i], __shfl_xor_sync(0xffffffffu, big[i], 2));
        }
        if (__any_sync(0xffffffffu, big[0] > top[0] || big[1] > top[1])) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float by = big[i] == -INFINITY ? 1.f : tc::ex2(top[i] - big[i]);
                top[i] = big[i];
                total[i] *= by;
#pragma unroll
                for (int x = 0; x < DP / 8; ++x) { o[x][2 * i] *= by; o[x][2 * i + 1] *= by; }
            }
        }
        const float from[2] = {top[0] == -INFINITY ? 0.f : top[0], top[1] == -INFINITY ? 0.f : top[1]};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) { s[n][i] = tc::ex2(s[n][i] - from[i >> 1]); total[i >> 1] += s[n][i]; }
        const uint32_t a[4] = {pack_bf16x2(s[0][0], s[0][1]), pack_bf16x2(s[0][2], s[0][3]), pack_bf16x2(s[1][0], s[1][1]), pack_bf16x2(s[1][2], s[1][3])};
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) {
            uint32_t vb[4];
            ldmatrix_t(vb, slot(stage, 1, (lane >> 3 & 1) * 8 + (lane & 7), 2 * x + (lane >> 4)));
            mma16(o[2 * x], a, vb[0], vb[1]);
            mma16(o[2 * x + 1], a, vb[2], vb[3]);
        }
        __syncwarp();                                            // every lane has read the slot
        ask(key0 + kStages * kWarps * kKeys, stage);
    }
    if (!ok) {                                                   // giving up: let copies that are still in flight land
        const unsigned long long t0 = tc::global_ns();
        while (tc::global_ns() - t0 < 200000ull) { }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        total[i] += __shfl_xor_sync(0xffffffffu, total[i], 1);
        total[i] += __shfl_xor_sync(0xffffffffu, total[i], 2);
    }
    __syncthreads();                                             // the rings become the box of the four warps' results
    float* box = reinterpret_cast<float*>(raw);                  // [warp][16][DP + 2]: output, maximum, sum
    auto line_of = [&](int w, int y) { return box + (w * 16 + y) * (DP + 2); };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float* to = line_of(warp, (lane >> 2) + 8 * i);
#pragma unroll
        for (int x = 0; x < DP / 8; ++x) { to[8 * x + 2 * (lane & 3)] = o[x][2 * i]; to[8 * x + 2 * (lane & 3) + 1] = o[x][2 * i + 1]; }
        if ((lane & 3) == 0) { to[DP] = top[i]; to[DP + 1] = total[i]; }
    }
    __syncthreads();
    const int64_t lines = (int64_t)p.batch * p.heads * p.q_len;
    for (int y = warp; y < 16; y += kWarps) {
        const int at = row0 + y;
        if (at >= rows) break;
        const int t = at / p.group, h = kvh * p.group + at % p.group;
        const int64_t line = ((int64_t)b * p.heads + h) * p.q_len + t;
        float big = -INFINITY, sum = 0.f, by[kWarps];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) big = fmaxf(big, line_of(w, y)[DP]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            by[w] = big == -INFINITY ? 0.f : tc::ex2(line_of(w, y)[DP] - big);
            sum += line_of(w, y)[DP + 1] * by[w];
        }
        const bool whole = p.splits == 1;
        const float over = !whole ? 1.f : sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
        for (int d = lane; d < p.dim; d += 32) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) v += line_of(w, y)[d] * by[w];
            if (whole) ((bf16*)p.out)[(int64_t)b * p.os.b + (int64_t)t * p.os.t + (int64_t)h * p.os.h + d] = from_f32<bf16>(v * over);
            else p.part_out[(blockIdx.x * lines + line) * p.dim + d] = v;
        }
        if (lane == 0) {
            if (!whole) { p.part_max[blockIdx.x * lines + line] = big; p.part_sum[blockIdx.x * lines + line] = sum; }
            else if (p.lse) p.lse[line] = big == -INFINITY ? -INFINITY : (big + log2f(sum)) * kLn2;
        }
    }
}

template <int DP, bool CAP>
void launch_few(ormi_b200_ctx* ctx, AttnParams& p) {
    constexpr int smem = FewShape<DP>::kSmem;
    auto kernel = attn_few<DP, CAP>;
    ORMI_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    CUtensorMap maps[2];
    head_map(ctx, &maps[0], p.k, p.ks, p.batch, p.k_len, p.kv_heads, p.dim, kKeys);
    head_map(ctx, &maps[1], p.v, p.vs, p.batch, p.k_len, p.kv_heads, p.dim, kKeys);
    int* err = device_error_word(ctx);
    ctx->gemm_err_pending = true;
    // Three blocks are resident per SM.  Long caches are cut into four rounds of blocks, so that sequences of different
    // lengths even out, with 512 keys each at least; short ones into one round, with 64 keys (a ring's worth of one turn).
    const int64_t pairs = (int64_t)p.batch * p.kv_heads, row_tiles = ((int64_t)p.q_len * p.group + 15) / 16, round = 3ll * ctx->num_sms;
    const int64_t long_cut = std::min<int64_t>((4 * round + pairs * row_tiles - 1) / (pairs * row_tiles), p.k_len / 512);
    const int64_t short_cut = std::min<int64_t>(round / (pairs * row_tiles), p.k_len / 64);
    const int64_t cut = std::max<int64_t>(1, std::min<int64_t>(std::max(long_cut, short_cut), 1024));
    const int part_keys = (int)(((p.k_len + cut - 1) / cut + 63) / 64 * 64);
    p.splits = (p.k_len + part_keys - 1) / part_keys;
    const size_t lines = (size_t)p.batch * p.heads * p.q_len;
    Scratch part(ctx, p.splits > 1 ? p.splits * lines * (p.dim + 2) * 4 : 0);
    if (p.splits > 1) {
        p.part_out = (float*)part.ptr;
        p.part_max = p.part_out + p.splits * lines * p.dim;
        p.part_sum = p.part_max + p.splits * lines;
    }
    kernel<<<dim3(p.splits, (unsigned)pairs, (unsigned)row_tiles), kWarps * 32, smem, ctx->stream>>>(maps[0], maps[1], p, cap_terms(p), part_keys, err);
    ORMI_CUDA(cudaGetLastError());
    count_launch(ctx);
    if (p.splits > 1) attention_join(ctx, p, ORMI_BF16);
    part.release();
}

}  // namespace

bool attention_few_supported(const AttnParams& p, int dtype) {
    return dtype == ORMI_BF16 && cap_terms_exist(p) && p.dim <= 128 && p.dim % 8 == 0 && p.k_len >= 1 && (int64_t)p.q_len * p.group <= 64 && map_allowed(p.q, p.qs, p.batch, p.q_len, p.heads) &&
           map_allowed(p.k, p.ks, p.batch, p.k_len, p.kv_heads) && map_allowed(p.v, p.vs, p.batch, p.k_len, p.kv_heads);
}

void attention_few(ormi_b200_ctx* ctx, AttnParams& p) {
    if (p.dim <= 64) { if (p.cap > 0.f) launch_few<64, true>(ctx, p); else launch_few<64, false>(ctx, p); }
    else { if (p.cap > 0.f) launch_few<128, true>(ctx, p); else launch_few<128, false>(ctx, p); }
}

}  // namespace ormi_b200
