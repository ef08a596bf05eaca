// Backward attention on the tensor cores: bf16, head_dim up to 128.
//
// Two kernels, so that no gradient is summed with atomics and results do not depend on the order of blocks:
//   attn_back_q    a block owns 128 queries of one head and walks the tiles of 128 keys: dQ += dS K.  It also writes
//                  delta = rowsum(dO O), which the second kernel reads.
//   attn_back_kv   a block owns 128 keys of one key/value head and walks the tiles of 128 queries, over all query heads that
//                  share the head.  Scores are computed transposed (rows = keys), so that probabilities and score
//                  gradients, rounded to bf16 in tensor memory, are the A operands of dV += P^T dO and dK += dS^T Q directly.
//                  Blocks of a cluster share the heads and add their dK and dV up through each other's shared memory, in a
//                  fixed order: with four heads in one block the longest block took most of the launch.
// The price is that both compute the scores (7 products instead of 5).  2 x 4096 tokens, 16 heads over 4, causal, head_dim
// 128: 430 us, 799 TFLOP/s counting the five, alone at 1965 MHz, 476 us in a loop at 1750 MHz.  Warp 0 loads, warp 1 issues the
// products, warp 2 fetches the queries' statistics (or blanks the keys behind key_len), and two warpgroups do the arithmetic, each half of the
// columns of a tile: while they work on the gradients of a tile the tensor cores multiply its probabilities and compute
// the next scores, and the other way round.  (Tiles of 64, one warpgroup each, were slower: a product of 64 columns takes
// the tensor cores as long as one of 128.)
#include <algorithm>

#include "attention_tc.cuh"

namespace ormi_b200 {
namespace {

using namespace tc;

constexpr int kThreads = 384;

struct Stat { float lse2[kTile], delta[kTile]; int end[kTile], doc[kTile]; };      // of 128 queries; the first two negated

template <int DP> struct BackShape {
    static constexpr int kOperand = kTile * DP * 2;
    static constexpr int kStages = DP == 128 ? 2 : 4;
    static constexpr int kSmem = 1024 + (2 + 2 * kStages) * kOperand + kMaxTiles * 2 + kStages * (int)sizeof(Stat) + 256;
};

// The tiles whose class is not kSkip, in order, class in the top two bits; by one warp.
template <typename F>
__device__ __forceinline__ int list_tiles(unsigned short* list, int tiles, F&& class_of) {
    const int lane = threadIdx.x & 31;
    int n = 0;
    for (int first = 0; first < tiles; first += 32) {
        const int c = first + lane < tiles ? class_of(first + lane) : kSkip;
        const unsigned hit = __ballot_sync(0xffffffffu, c != kSkip);
        if (c != kSkip) list[n + __popc(hit & ((1u << lane) - 1))] = (unsigned short)((first + lane) | c << 14);
        n += __popc(hit);
    }
    return n;
}
__device__ __forceinline__ int tile_of(unsigned short entry) { return entry & 0x3fff; }

// A operand of 128 bf16 columns that two warpgroups wrote into the first halves of their own 64 columns.
template <int DP>
__device__ __forceinline__ void product_halves(uint32_t d, uint32_t a, uint32_t b, uint32_t accumulate) {
    const uint64_t db = desc_mn<kTile>(b);
#pragma unroll
    for (int k = 0; k < 8; ++k) mma_ts(d, a + (k / 4) * 64 + (k % 4) * 8, db + ((k * 2048) >> 4), idesc(DP, true), accumulate || k > 0);
}

__device__ __forceinline__ void leave(Abort& ab, int warp, uint32_t tmem) {
    __syncwarp();
    if (ab.flag) {                                             // let copies that are still in flight land before the block goes away
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 200000ull) { }
    }
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <int DP, bool CAP, bool BIAS, bool DOCS>
__global__ void __launch_bounds__(kThreads, 1)
attn_back_kv(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
             const __grid_constant__ CUtensorMap map_do, const __grid_constant__ TcParams p) {
    using Shape = BackShape<DP>;
    constexpr int ST = Shape::kStages, OP = Shape::kOperand;
    extern __shared__ unsigned char raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    unsigned char* mem = raw + (base - smem_u32(raw));
    const uint32_t k_at = base, v_at = base + OP;
    auto q_at = [&](int s) { return base + (2 + 2 * s) * OP; };
    auto do_at = [&](int s) { return base + (3 + 2 * s) * OP; };
    Stat* stats = reinterpret_cast<Stat*>(mem + (2 + 2 * ST) * OP);
    unsigned short* list = reinterpret_cast<unsigned short*>(stats + ST);
    const uint32_t bars = smem_u32(list + kMaxTiles);
    const uint32_t kv_full = bars, s_full = bars + 8, dp_full = bars + 16, p_ready = bars + 24, ds_ready = bars + 32, done = bars + 40;
    auto q_full = [&](int s) { return bars + 48 + 8 * s; };
    auto do_full = [&](int s) { return bars + 48 + 8 * (ST + s); };
    auto empty = [&](int s) { return bars + 48 + 8 * (2 * ST + s); };
    auto stat_full = [&](int s) { return bars + 48 + 8 * (3 * ST + s); };
    auto stat_empty = [&](int s) { return bars + 48 + 8 * (4 * ST + s); };
    __shared__ uint32_t tmem_slot;
    __shared__ int list_size;
    __shared__ Abort ab;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % p.cluster, head_group = blockIdx.x / p.cluster;
    const int b = head_group / p.a.kv_heads, kvh = head_group % p.a.kv_heads;
    const int heads = p.a.group / p.cluster, first_head = kvh * p.a.group + rank * heads;      // this block's query heads
    const int key0 = blockIdx.y * kTile;                                   // causal: the first keys are seen by most queries
    const RowMask m = row_mask(p.a, b);
    if (warp == 2) {
        const int n = key0 >= m.keys ? 0 : list_tiles(list, (p.a.q_len + kTile - 1) / kTile, [&](int t) {
            const int first = t * kTile, last = min(first + kTile, p.a.q_len) - 1;
            return tile_class(p, b, 2 * t, key_end(m, m.start + first), key_end(m, m.start + last), key0 / kUnit);
        });
        if (lane == 0) list_size = n;
    }
    if (threadIdx.x == 0) {
        ab.flag = 0; ab.err = p.err;
        mbar_init(kv_full, 1); mbar_init(s_full, 1); mbar_init(dp_full, 1); mbar_init(done, 1);
        mbar_init(p_ready, 8); mbar_init(ds_ready, 8);
        for (int s = 0; s < ST; ++s) { mbar_init(q_full(s), 1); mbar_init(do_full(s), 1); mbar_init(empty(s), 1); mbar_init(stat_full(s), 1); mbar_init(stat_empty(s), 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        // the resident operands do not depend on the list: they are on their way while it is being made
        mbar_expect_tx(kv_full, 2 * OP);
        for (int x = 0; x < DP / 64; ++x) {
            tma_load_4d(k_at + x * box_bytes(kTile), &map_k, kv_full, 64 * x, key0, kvh, b);
            tma_load_4d(v_at + x * box_bytes(kTile), &map_v, kv_full, 64 * x, key0, kvh, b);
        }
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    // all of tensor memory is this block's, so it starts at column 0 (checked: every address below is a constant)
    constexpr uint32_t tmem = 0, s_at = tmem, dp_at = tmem + 128, dv_at = tmem + 256, dk_at = tmem + 384;
    const bool whole = tmem_slot == tmem;
    if (!whole && threadIdx.x == 0) atomicCAS(p.err, 0, 20);
    const int per_head = list_size, total = per_head * heads;

    if (!whole) {
    } else if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 0) {
            if (lane == 0) {
                bool ok = true;
                int i = 0;
                for (; i < total && ok; ++i) {
                    const int s = i % ST, h = first_head + i / per_head, q0 = tile_of(list[i % per_head]) * kTile;
                    ok = mbar_wait(empty(s), (i / ST & 1) ^ 1, ab, 31);
                    if (!ok) break;
                    mbar_expect_tx(q_full(s), OP);
                    for (int x = 0; x < DP / 64; ++x) tma_load_4d(q_at(s) + x * box_bytes(kTile), &map_q, q_full(s), 64 * x, q0, h, b);
                    mbar_expect_tx(do_full(s), OP);
                    for (int x = 0; x < DP / 64; ++x) tma_load_4d(do_at(s) + x * box_bytes(kTile), &map_do, do_full(s), 64 * x, q0, h, b);
                }
                ok = ok && mbar_wait(kv_full, 0, ab, 31);             // nothing of this block's is in flight when it leaves
                for (int k = 0; k < ST && ok; ++k, ++i) ok = mbar_wait(empty(i % ST), (i / ST & 1) ^ 1, ab, 31);
            }
        } else if (warp == 1) {
            if (total) {
                bool ok = warp_wait(kv_full, 0, ab, 32);
                auto scores = [&](int i) {
                    ok = ok && warp_wait(q_full(i % ST), i / ST & 1, ab, 33);
                    if (!ok) return;
                    fence_after();
                    if (elect()) {
                        product_nt<DP, kTile>(s_at, k_at, q_at(i % ST));
                        commit(s_full);
                    }
                };
                auto gaps = [&](int i) {
                    ok = ok && warp_wait(do_full(i % ST), i / ST & 1, ab, 34);
                    if (!ok) return;
                    fence_after();
                    if (elect()) {
                        product_nt<DP, kTile>(dp_at, v_at, do_at(i % ST));
                        commit(dp_full);
                    }
                };
                scores(0);
                gaps(0);
                // P sits in the scores' columns and dS in the columns of dP: the next tile's products follow their readers in order
                for (int i = 0; i < total && ok; ++i) {
                    ok = warp_wait(p_ready, i & 1, ab, 35);
                    if (!ok) break;
                    fence_after();
                    if (elect()) product_halves<DP>(dv_at, s_at, do_at(i % ST), i > 0);
                    if (i + 1 < total) scores(i + 1);
                    ok = ok && warp_wait(ds_ready, i & 1, ab, 36);
                    if (!ok) break;
                    fence_after();
                    if (elect()) {
                        product_halves<DP>(dk_at, dp_at, q_at(i % ST), i > 0);
                        commit(empty(i % ST));
                    }
                    if (i + 1 < total) gaps(i + 1);
                }
                if (elect()) commit(done);
            }
        } else if (warp == 2) {
            // the queries' statistics; a row that sees nothing, or does not exist, gets an infinite one: its probabilities vanish
            for (int i = 0; i < total; ++i) {
                const int s = i % ST, h = first_head + i / per_head, q0 = tile_of(list[i % per_head]) * kTile;
                float l[4], d[4];
                int e[4], doc[4];
    #pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int t = q0 + k * 32 + lane;
                    const bool live = t < p.a.q_len;
                    const int64_t line = ((int64_t)b * p.a.heads + h) * p.a.q_len + t;
                    l[k] = live ? p.a.lse[line] * kLog2e : INFINITY;
                    if (l[k] == -INFINITY) l[k] = INFINITY;
                    d[k] = live ? p.a.delta[line] : 0.f;
                    e[k] = live ? key_end(m, m.start + t) : 0;
                    doc[k] = DOCS && live ? m.q_docs[t] : 0;
                }
                if (!warp_wait(stat_empty(s), (i / ST & 1) ^ 1, ab, 37)) break;
    #pragma unroll
                for (int k = 0; k < 4; ++k) {
                    stats[s].lse2[k * 32 + lane] = -l[k]; stats[s].delta[k * 32 + lane] = -d[k];
                    stats[s].end[k * 32 + lane] = e[k];
                    if (DOCS) stats[s].doc[k * 32 + lane] = doc[k];
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(stat_full(s));
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int w = warp / 4 - 1, row = threadIdx.x & 127, key = key0 + row;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        const bool live = key < m.keys;
        const int my_doc = DOCS && live ? m.k_docs[key] : 0;
        bool ok = true;
        for (int i = 0; i < total; ++i) {
            const int s = i % ST, entry = list[i % per_head], q0 = tile_of(entry) * kTile;
            const int cls = entry >> 14;
            const Stat& st = stats[s];
            const float slope = BIAS ? p.a.slopes[first_head + i / per_head] * kLog2e : 0.f;
            const float ahead = (float)(m.start + q0 + 64 * w - key);
            ok = warp_wait(stat_full(s), i / ST & 1, ab, 38) && warp_wait(s_full, i & 1, ab, 38);
            if (!ok) break;
            fence_after();
            float2 z[32], g[32];                        // g: what the gradient of a raw product is a multiple of
            ld32(s_at + lanes + 64 * w, reinterpret_cast<uint32_t*>(z));
            ld32(s_at + lanes + 64 * w + 32, reinterpret_cast<uint32_t*>(z) + 32);
            wait_ld();
            // the capped score, its slope and the exponential of two columns: the polynomial runs on the FMA pipe while the
            // special function unit is busy with the exponentials before it
            auto expo = [&](int c, const float2& neg_lse2) {
                if (CAP) g[c] = cap_slope(p.cap, z[c]);
                if (BIAS) {
                    if (!CAP) z[c] = mul2(z[c], both(p.scale_log2));
                    z[c] = make_float2(fmaf(-slope, fabsf(ahead + (float)(2 * c)), z[c].x), fmaf(-slope, fabsf(ahead + (float)(2 * c + 1)), z[c].y));
                }
                z[c] = CAP || BIAS ? add2(z[c], neg_lse2) : fma2(z[c], both(p.scale_log2), neg_lse2);
                z[c] = make_float2(ex2(z[c].x), ex2(z[c].y));
            };
            if (!CAP || cap_is_polynomial<32>(p.cap, z)) {
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    const float4 l = *reinterpret_cast<const float4*>(&st.lse2[64 * w + 2 * c]);
                    if (CAP) { z[c] = cap_polynomial(p.cap, z[c]); z[c + 1] = cap_polynomial(p.cap, z[c + 1]); }
                    expo(c, make_float2(l.x, l.y));
                    expo(c + 1, make_float2(l.z, l.w));
                }
            } else {
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    const float4 l = *reinterpret_cast<const float4*>(&st.lse2[64 * w + 2 * c]);
                    z[c] = cap_any(p.cap, z[c]); z[c + 1] = cap_any(p.cap, z[c + 1]);
                    expo(c, make_float2(l.x, l.y));
                    expo(c + 1, make_float2(l.z, l.w));
                }
            }
            uint32_t pk[32];
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
                if (cls >= kPartial) {
                    const int4 e = *reinterpret_cast<const int4*>(&st.end[64 * w + 2 * c]);
                    int4 d = make_int4(my_doc, my_doc, my_doc, my_doc);
                    if (DOCS) { if (cls == kDocs) d = *reinterpret_cast<const int4*>(&st.doc[64 * w + 2 * c]); }
                    if ((key >= e.x) | (d.x != my_doc)) { z[c].x = 0.f; if (CAP) g[c].x = 0.f; }
                    if ((key >= e.y) | (d.y != my_doc)) { z[c].y = 0.f; if (CAP) g[c].y = 0.f; }
                    if ((key >= e.z) | (d.z != my_doc)) { z[c + 1].x = 0.f; if (CAP) g[c + 1].x = 0.f; }
                    if ((key >= e.w) | (d.w != my_doc)) { z[c + 1].y = 0.f; if (CAP) g[c + 1].y = 0.f; }
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    pk[c + k] = pack_bf16x2(z[c + k].x, z[c + k].y);
                    g[c + k] = CAP ? mul2(g[c + k], z[c + k]) : z[c + k];
                }
            }
            st32(s_at + lanes + 64 * w, pk);
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_ready);
            ok = warp_wait(dp_full, i & 1, ab, 39);
            if (!ok) break;
            fence_after();
            float2 gap[32];
            ld32(dp_at + lanes + 64 * w, reinterpret_cast<uint32_t*>(gap));
            ld32(dp_at + lanes + 64 * w + 32, reinterpret_cast<uint32_t*>(gap) + 32);
            wait_ld();
            if (cls >= kPartial) {                      // a masked pair's V may hold anything
#pragma unroll
                for (int c = 0; c < 32; ++c) { if (g[c].x == 0.f) gap[c].x = 0.f; if (g[c].y == 0.f) gap[c].y = 0.f; }
            }
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
                const float4 d = *reinterpret_cast<const float4*>(&st.delta[64 * w + 2 * c]);
                const float2 x = mul2(g[c], add2(gap[c], make_float2(d.x, d.y))), y = mul2(g[c + 1], add2(gap[c + 1], make_float2(d.z, d.w)));
                pk[c] = pack_bf16x2(x.x, x.y);
                pk[c + 1] = pack_bf16x2(y.x, y.y);
            }
            st32(dp_at + lanes + 64 * w, pk);
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) { mbar_arrive(ds_ready); mbar_arrive(stat_empty(s)); }
        }
        // (keys that nobody sees still wait for their K and V: that memory is written below)
        if (ok) ok = total ? warp_wait(done, 0, ab, 40) : warp_wait(kv_full, 0, ab, 40);
        if (ok) {
            // warpgroup 0 takes dV out of tensor memory, warpgroup 1 dK; keys that nobody sees get zero
            fence_after();
            const int first = key0 + (warp & 3) * 32, row = threadIdx.x & 127;
            const Strides4& os = w ? p.a.dks : p.a.dvs;
            bf16* out = (bf16*)(w ? p.a.dk : p.a.dv) + (int64_t)b * os.b + (int64_t)first * os.t + (int64_t)kvh * os.h;
            if (p.cluster == 1) {
                store_rows<DP>((w ? dk_at : dv_at) + lanes, total > 0, base + (warp - 4) * (64 * DP), w ? p.a.scale : 1.f, p.a.k_len - first, p.a.dim, [&](int r) { return out + r * os.t; });
            } else {
                // into the idle operand buffers, for the cluster: rows of fp32, their 16-byte chunks c at c ^ row
                const uint32_t to = base + w * (kTile * DP * 4) + row * (DP * 4);
#pragma unroll 1
                for (int x = 0; x < DP; x += 32) {
                    uint32_t o[32];
                    if (total) { ld32((w ? dk_at : dv_at) + lanes + x, o); wait_ld(); }
                    else for (int i = 0; i < 32; ++i) o[i] = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + (((x / 4 + i) ^ (row & (DP / 4 - 1))) << 4)), "r"(o[4 * i]), "r"(o[4 * i + 1]), "r"(o[4 * i + 2]), "r"(o[4 * i + 3]) : "memory");
                }
            }
        }
    }
    __syncwarp();
    if (p.cluster > 1) {
        auto meet = [&] {
            asm volatile("barrier.cluster.arrive.release;" ::: "memory");
            asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        };
        meet();
        if (whole && !ab.flag) {
            // rows rank, rank + cluster, ... of both: the sum over the cluster's blocks in their order.  A lane holds four columns.
            constexpr int LPR = DP / 4, RPW = 32 / LPR;
            const int mine = kTile / p.cluster, c = lane % LPR;
            const float by_k = p.a.scale;
#pragma unroll 2
            for (int i = warp * RPW + lane / LPR; i < 2 * mine; i += kThreads / 32 * RPW) {
                const int which = i >= mine, row = (i - which * mine) * p.cluster + rank, key = key0 + row;
                const uint32_t at = base + which * (kTile * DP * 4) + row * (DP * 4) + ((c ^ (row & (DP / 4 - 1))) << 4);
                float4 v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    v[r] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (r >= p.cluster) continue;
                    uint32_t peer;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at), "r"(r));
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[r].x), "=f"(v[r].y), "=f"(v[r].z), "=f"(v[r].w) : "r"(peer));
                }
                if (key >= p.a.k_len || 4 * c >= p.a.dim) continue;
                const Strides4& os = which ? p.a.dks : p.a.dvs;
                const float by = which ? by_k : 1.f;
                bf16* out = (bf16*)(which ? p.a.dk : p.a.dv) + (int64_t)b * os.b + (int64_t)key * os.t + (int64_t)kvh * os.h + 4 * c;
                *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2((((v[0].x + v[1].x) + v[2].x) + v[3].x) * by, (((v[0].y + v[1].y) + v[2].y) + v[3].y) * by),
                                                            pack_bf16x2((((v[0].z + v[1].z) + v[2].z) + v[3].z) * by, (((v[0].w + v[1].w) + v[2].w) + v[3].w) * by));
            }
        }
        meet();                                                // nobody leaves while another reads its memory
    }
    leave(ab, warp, tmem_slot);
}

template <int DP, bool CAP, bool BIAS, bool DOCS>
__global__ void __launch_bounds__(kThreads, 1)
attn_back_q(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
            const __grid_constant__ CUtensorMap map_do, const __grid_constant__ CUtensorMap map_o, const __grid_constant__ TcParams p) {
    using Shape = BackShape<DP>;
    // K is read twice, by the scores and a whole tile later by dQ; V once: three slots and one (six and two of half the size)
    constexpr int KS = Shape::kStages * 3 / 2, VS = Shape::kStages / 2, OP = Shape::kOperand;
    extern __shared__ unsigned char raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    unsigned char* mem = raw + (base - smem_u32(raw));
    const uint32_t q_at = base, do_at = base + OP;
    auto k_at = [&](int s) { return base + (2 + s) * OP; };
    auto v_at = [&](int s) { return base + (2 + KS + s) * OP; };
    const uint32_t o_at = k_at(KS - 1);                                          // O's tile, until delta has been computed
    float* deltas = reinterpret_cast<float*>(mem + (2 + KS + VS) * OP);          // of the 128 queries: two halves
    int* docs = reinterpret_cast<int*>(deltas + 2 * kTile);                      // 64 for each compute warp
    unsigned short* list = reinterpret_cast<unsigned short*>(docs + 8 * 64);
    const uint32_t bars = smem_u32(list + kMaxTiles);
    const uint32_t q_full = bars, dp_full = bars + 8, ds_ready = bars + 16, done = bars + 24, blank_go = bars + 32, blanked = bars + 40;
    auto s_full = [&](int x) { return bars + 48 + 8 * x; };
    auto s_empty = [&](int x) { return bars + 64 + 8 * x; };
    const uint32_t o_full = bars + 80, o_read = bars + 88;
    auto k_full = [&](int s) { return bars + 96 + 8 * s; };
    auto k_empty = [&](int s) { return bars + 96 + 8 * (KS + s); };
    auto v_full = [&](int s) { return bars + 96 + 8 * (2 * KS + s); };
    auto v_empty = [&](int s) { return bars + 96 + 8 * (2 * KS + VS + s); };
    __shared__ uint32_t tmem_slot;
    __shared__ int list_size;
    __shared__ Abort ab;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = blockIdx.x / p.a.heads, h = blockIdx.x % p.a.heads, kvh = h / p.a.group;
    const int q0 = (int)(gridDim.y - 1 - blockIdx.y) * kTile;
    const RowMask m = row_mask(p.a, b);
    const int blank_tile = m.keys < p.a.k_len && m.keys % kTile ? m.keys / kTile : -1;
    if (warp == 2) {
        const int lo = key_end(m, m.start + q0), hi = key_end(m, m.start + min(q0 + kTile, p.a.q_len) - 1);
        const int n = list_tiles(list, (max(hi, 0) + kTile - 1) / kTile, [&](int j) { return tile_class(p, b, q0 / kUnit, lo, hi, 2 * j); });
        if (lane == 0) list_size = n;
    }
    if (threadIdx.x == 0) {
        ab.flag = 0; ab.err = p.err;
        mbar_init(q_full, 1); mbar_init(dp_full, 1); mbar_init(ds_ready, 8); mbar_init(done, 1); mbar_init(blank_go, 1); mbar_init(blanked, 1);
        for (int x = 0; x < 2; ++x) { mbar_init(s_full(x), 1); mbar_init(s_empty(x), 8); }
        mbar_init(o_full, 1); mbar_init(o_read, 8);
        for (int s = 0; s < KS; ++s) { mbar_init(k_full(s), 1); mbar_init(k_empty(s), 1); }
        for (int s = 0; s < VS; ++s) { mbar_init(v_full(s), 1); mbar_init(v_empty(s), 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        // (O is needed even where no key is seen: delta is written for every query)
        mbar_expect_tx(o_full, OP);
        for (int x = 0; x < DP / 64; ++x) tma_load_4d(o_at + x * box_bytes(kTile), &map_o, o_full, 64 * x, q0, h, b);
        mbar_expect_tx(q_full, 2 * OP);
        for (int x = 0; x < DP / 64; ++x) {
            tma_load_4d(do_at + x * box_bytes(kTile), &map_do, q_full, 64 * x, q0, h, b);
            tma_load_4d(q_at + x * box_bytes(kTile), &map_q, q_full, 64 * x, q0, h, b);
        }
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    constexpr uint32_t tmem = 0, dp_at = tmem + 256, dq_at = tmem + 384;         // as above
    const bool whole = tmem_slot == tmem;
    if (!whole && threadIdx.x == 0) atomicCAS(p.err, 0, 20);
    auto s_at = [&](int x) { return tmem + 128 * x; };
    const int total = list_size;

    if (!whole) {
    } else if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 0) {
            if (lane == 0) {
                bool ok = true;
                auto load_k = [&](int i) {
                    const int s = i % KS;
                    ok = ok && mbar_wait(k_empty(s), (i / KS & 1) ^ 1, ab, 41) && (i != KS - 1 || mbar_wait(o_read, 0, ab, 41));
                    if (!ok) return;
                    mbar_expect_tx(k_full(s), OP);
                    for (int x = 0; x < DP / 64; ++x) tma_load_4d(k_at(s) + x * box_bytes(kTile), &map_k, k_full(s), 64 * x, tile_of(list[i]) * kTile, kvh, b);
                };
                auto load_v = [&](int i) {
                    const int s = i % VS;
                    ok = ok && mbar_wait(v_empty(s), (i / VS & 1) ^ 1, ab, 41);
                    if (!ok) return;
                    mbar_expect_tx(v_full(s), OP);
                    for (int x = 0; x < DP / 64; ++x) tma_load_4d(v_at(s) + x * box_bytes(kTile), &map_v, v_full(s), 64 * x, tile_of(list[i]) * kTile, kvh, b);
                };
                // in the order in which the slots come free: V of a tile when the one before has been multiplied, K a tile ahead of it
                if (total) { load_k(0); load_v(0); }
                if (total > 1) load_k(1);
                for (int i = 1; i < total && ok; ++i) {
                    load_v(i);
                    if (i + 1 < total) load_k(i + 1);
                }
                // nothing of this block's is in flight when it leaves
                ok = ok && mbar_wait(q_full, 0, ab, 41) && mbar_wait(o_read, 0, ab, 41);
                for (int k = 0; k < KS; ++k) ok = ok && mbar_wait(k_empty((total + k) % KS), ((total + k) / KS & 1) ^ 1, ab, 41);
                for (int k = 0; k < VS; ++k) ok = ok && mbar_wait(v_empty((total + k) % VS), ((total + k) / VS & 1) ^ 1, ab, 41);
            }
        } else if (warp == 1) {
            if (total) {
                bool ok = warp_wait(q_full, 0, ab, 42);
                auto scores = [&](int i) {
                    ok = ok && warp_wait(k_full(i % KS), i / KS & 1, ab, 43);
                    if (ok && tile_of(list[i]) == blank_tile) {            // warp 2 blanks the rows behind key_len first
                        if (lane == 0) mbar_arrive(blank_go);
                        ok = warp_wait(blanked, 0, ab, 43);
                    }
                    ok = ok && warp_wait(s_empty(i & 1), (i / 2 & 1) ^ 1, ab, 44);
                    if (!ok) return;
                    fence_after();
                    if (elect()) {
                        product_nt<DP, kTile>(s_at(i & 1), q_at, k_at(i % KS));
                        commit(s_full(i & 1));
                    }
                };
                auto gaps = [&](int i) {
                    ok = ok && warp_wait(v_full(i % VS), i / VS & 1, ab, 45);
                    if (!ok) return;
                    fence_after();
                    if (elect()) {
                        product_nt<DP, kTile>(dp_at, do_at, v_at(i % VS));
                        commit(dp_full);
                        commit(v_empty(i % VS));
                    }
                };
                scores(0);
                gaps(0);
                for (int i = 0; i < total && ok; ++i) {
                    if (i + 1 < total) scores(i + 1);                        // runs while the gradients of tile i are computed
                    ok = ok && warp_wait(ds_ready, i & 1, ab, 46);
                    if (!ok) break;
                    fence_after();
                    if (elect()) {
                        product_halves<DP>(dq_at, dp_at, k_at(i % KS), i > 0);
                        commit(k_empty(i % KS));
                    }
                    if (i + 1 < total) gaps(i + 1);
                }
                if (elect()) commit(done);
            }
        } else if (warp == 2) {
            if (total && blank_tile >= 0 && tile_of(list[total - 1]) == blank_tile) {
                const int s = (total - 1) % KS;
                if (warp_wait(blank_go, 0, ab, 47)) {
                    for (int x = 0; x < DP / 64; ++x)
                        for (int i = m.keys % kTile * 8 + lane; i < kTile * 8; i += 32)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(k_at(s) + x * box_bytes(kTile) + i * 16), "r"(0) : "memory");
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(blanked);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int64_t lines = ((int64_t)b * p.a.heads + h) * p.a.q_len;
        const int w = warp / 4 - 1, t = q0 + (threadIdx.x & 127);
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        const bool live = t < p.a.q_len;
        const int pos = m.start + t, end = live ? key_end(m, pos) : 0;
        const int my_doc = DOCS && live ? m.q_docs[t] : 0;
        const float slope = BIAS ? p.a.slopes[h] * kLog2e : 0.f;
        float lse2 = live ? p.a.lse[lines + t] * kLog2e : INFINITY;
        if (lse2 == -INFINITY) lse2 = INFINITY;
        // delta of the block's queries: a row per thread, half of the columns for each warpgroup, from the swizzled tiles
        bool ok = warp_wait(q_full, 0, ab, 47) && warp_wait(o_full, 0, ab, 47);
        float half = 0.f;
        if (ok) {
            const int row = threadIdx.x & 127;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                const int c = w * (DP / 16) + k;                  // 16-byte chunk of the row
                const uint32_t at = (c >> 3) * box_bytes(kTile) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
                uint32_t x[4], y[4];
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(o_at + at) : "memory");
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(y[0]), "=r"(y[1]), "=r"(y[2]), "=r"(y[3]) : "r"(do_at + at) : "memory");
#pragma unroll
                for (int e = 0; e < 4; ++e) half = fmaf(bf16_hi(x[e]), bf16_hi(y[e]), fmaf(bf16_lo(x[e]), bf16_lo(y[e]), half));
            }
        }
        deltas[w * kTile + (threadIdx.x & 127)] = half;
        __syncwarp();
        if (lane == 0) mbar_arrive(o_read);                      // the third slot is free for keys
        asm volatile("bar.sync 1, 256;" ::: "memory");           // the eight compute warps; all of them come here
        const float delta = deltas[threadIdx.x & 127] + deltas[kTile + (threadIdx.x & 127)];
        if (w == 0 && live) p.a.delta[lines + t] = delta;
        int* my_docs = docs + (warp - 4) * 64;
        int ahead_docs[2];                                       // documents of the tile to come, asked for a tile ahead
        auto fetch = [&](int i) {
            if (DOCS && list[i] >> 14 == kDocs) {
                const int k = tile_of(list[i]) * kTile + 64 * w + lane;
                ahead_docs[0] = k < p.a.k_len ? m.k_docs[k] : 0;
                ahead_docs[1] = k + 32 < p.a.k_len ? m.k_docs[k + 32] : 0;
            }
        };
        if (total) fetch(0);
        for (int i = 0; i < total && ok; ++i) {
            const int entry = list[i], key0 = tile_of(entry) * kTile + 64 * w;
            const int cls = entry >> 14;
            if (DOCS && cls == kDocs) {
                __syncwarp();
                my_docs[lane] = ahead_docs[0]; my_docs[lane + 32] = ahead_docs[1];
                __syncwarp();
            }
            if (i + 1 < total) fetch(i + 1);
            ok = warp_wait(s_full(i & 1), i / 2 & 1, ab, 48);
            if (!ok) break;
            fence_after();
            float2 z[32], g[32];
            ld32(s_at(i & 1) + lanes + 64 * w, reinterpret_cast<uint32_t*>(z));
            ld32(s_at(i & 1) + lanes + 64 * w + 32, reinterpret_cast<uint32_t*>(z) + 32);
            wait_ld();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_empty(i & 1));
            const float ahead = (float)(pos - key0);
            const int left = end - key0;
            auto expo = [&](int c) {                                  // as in attn_back_kv
                if (CAP) g[c] = cap_slope(p.cap, z[c]);
                if (BIAS) {
                    if (!CAP) z[c] = mul2(z[c], both(p.scale_log2));
                    z[c] = make_float2(fmaf(-slope, fabsf(ahead - (float)(2 * c)), z[c].x), fmaf(-slope, fabsf(ahead - (float)(2 * c + 1)), z[c].y));
                }
                z[c] = CAP || BIAS ? add2(z[c], both(-lse2)) : fma2(z[c], both(p.scale_log2), both(-lse2));
                z[c] = make_float2(ex2(z[c].x), ex2(z[c].y));
                g[c] = CAP ? mul2(g[c], z[c]) : z[c];
            };
            if (!CAP || cap_is_polynomial<32>(p.cap, z)) {
#pragma unroll
                for (int c = 0; c < 32; ++c) { if (CAP) z[c] = cap_polynomial(p.cap, z[c]); expo(c); }
            } else {
#pragma unroll
                for (int c = 0; c < 32; ++c) { z[c] = cap_any(p.cap, z[c]); expo(c); }
            }
            if (DOCS && cls == kDocs) {
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    const int4 d = *reinterpret_cast<const int4*>(&my_docs[2 * c]);
                    if (d.x != my_doc) g[c].x = 0.f;
                    if (d.y != my_doc) g[c].y = 0.f;
                    if (d.z != my_doc) g[c + 1].x = 0.f;
                    if (d.w != my_doc) g[c + 1].y = 0.f;
                }
            }
            if (cls >= kPartial) {
#pragma unroll
                for (int c = 0; c < 32; ++c) {
                    if (2 * c >= left) g[c].x = 0.f;
                    if (2 * c + 1 >= left) g[c].y = 0.f;
                }
            }
            ok = warp_wait(dp_full, i & 1, ab, 49);
            if (!ok) break;
            fence_after();
            float2 gap[32];
            ld32(dp_at + lanes + 64 * w, reinterpret_cast<uint32_t*>(gap));
            ld32(dp_at + lanes + 64 * w + 32, reinterpret_cast<uint32_t*>(gap) + 32);
            wait_ld();
            if (cls >= kPartial) {                      // a masked pair's V may hold anything
#pragma unroll
                for (int c = 0; c < 32; ++c) { if (g[c].x == 0.f) gap[c].x = 0.f; if (g[c].y == 0.f) gap[c].y = 0.f; }
            }
            uint32_t pk[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) {
                const float2 x = mul2(g[c], add2(gap[c], both(-delta)));
                pk[c] = pack_bf16x2(x.x, x.y);
            }
            st32(dp_at + lanes + 64 * w, pk);
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ds_ready);
        }
        if (ok && total) ok = warp_wait(done, 0, ab, 50);
        if (ok) {
            fence_after();
            const int first = q0 + (warp & 3) * 32;
            bf16* out = (bf16*)p.a.dq + (int64_t)b * p.a.dqs.b + (int64_t)first * p.a.dqs.t + (int64_t)h * p.a.dqs.h;
            const int x = w * (DP / 2);                                            // a half of the columns each
            store_rows<DP / 2>(dq_at + lanes + x, total > 0, q_at + (warp - 4) * (32 * DP), p.a.scale, p.a.q_len - first, p.a.dim - x, [&](int r) { return out + r * p.a.dqs.t + x; });
        }
    }
    leave(ab, warp, tmem_slot);
}

template <int DP, bool CAP, bool BIAS, bool DOCS>
void launch_backward(ormi_b200_ctx* ctx, const CUtensorMap* maps, const TcParams& p) {
    constexpr int smem = BackShape<DP>::kSmem;
    auto kv = attn_back_kv<DP, CAP, BIAS, DOCS>;
    auto q = attn_back_q<DP, CAP, BIAS, DOCS>;
    ORMI_CUDA(cudaFuncSetAttribute(kv, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    ORMI_CUDA(cudaFuncSetAttribute(q, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    q<<<dim3(p.a.batch * p.a.heads, (p.a.q_len + kTile - 1) / kTile), kThreads, smem, ctx->stream>>>(maps[0], maps[1], maps[2], maps[3], maps[4], p);
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(p.a.batch * p.a.kv_heads * p.cluster, (p.a.k_len + kTile - 1) / kTile);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = smem;
    config.stream = ctx->stream;
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = p.cluster; cluster.val.clusterDim.y = 1; cluster.val.clusterDim.z = 1;
    config.attrs = &cluster;
    config.numAttrs = 1;
    ORMI_CUDA(cudaLaunchKernelEx(&config, kv, maps[0], maps[1], maps[2], maps[3], p));
    ORMI_CUDA(cudaGetLastError());
    count_launch(ctx, 2);
}

template <int DP>
void launch_by_mask(ormi_b200_ctx* ctx, const CUtensorMap* maps, const TcParams& p) {
    const bool cap = p.a.cap > 0.f, bias = p.a.slopes, docs = p.a.k_docs;
    if (cap) {
        if (bias) docs ? launch_backward<DP, true, true, true>(ctx, maps, p) : launch_backward<DP, true, true, false>(ctx, maps, p);
        else docs ? launch_backward<DP, true, false, true>(ctx, maps, p) : launch_backward<DP, true, false, false>(ctx, maps, p);
    } else {
        if (bias) docs ? launch_backward<DP, false, true, true>(ctx, maps, p) : launch_backward<DP, false, true, false>(ctx, maps, p);
        else docs ? launch_backward<DP, false, false, true>(ctx, maps, p) : launch_backward<DP, false, false, false>(ctx, maps, p);
    }
}

}  // namespace

bool attention_backward_tc_supported(const AttnParams& p, int dtype) {
    return attention_tc_supported(p, dtype) && p.q_len >= 1 && p.q_len <= kMaxTiles * kTile && map_allowed(p.dout, p.dos, p.batch, p.q_len, p.heads) &&
           map_allowed(p.dq, p.dqs, p.batch, p.q_len, p.heads) && map_allowed(p.dk, p.dks, p.batch, p.k_len, p.kv_heads) && map_allowed(p.dv, p.dvs, p.batch, p.k_len, p.kv_heads);
}

void attention_backward_tc(ormi_b200_ctx* ctx, AttnParams& a) {
    Scratch bounds(ctx, bounds_bytes(a));
    TcParams p = tc_params(ctx, a, (int2*)bounds.ptr);
    // A block alone keeps its set-up (loads, tensor memory, first products: 5 us) for more tiles; a cluster spreads the work
    // of a key/value head where blocks would leave SMs idle, and evens out the uneven lists that documents make (packed
    // documents, 2 x 4096 tokens, 16 heads over 4: 279 us alone, 260 us in twos, 304 us in fours; without documents 431, 446
    // and 513 us).
    const int64_t blocks = (int64_t)a.batch * a.kv_heads * ((a.k_len + kTile - 1) / kTile);
    p.cluster = a.group % 4 == 0 && blocks * 4 <= ctx->num_sms ? 4 : a.group % 2 == 0 && (blocks * 2 <= ctx->num_sms || a.k_docs) ? 2 : 1;
    CUtensorMap maps[5];
    head_map(ctx, &maps[0], a.q, a.qs, a.batch, a.q_len, a.heads, a.dim);
    head_map(ctx, &maps[1], a.k, a.ks, a.batch, a.k_len, a.kv_heads, a.dim);
    head_map(ctx, &maps[2], a.v, a.vs, a.batch, a.k_len, a.kv_heads, a.dim);
    head_map(ctx, &maps[3], a.dout, a.dos, a.batch, a.q_len, a.heads, a.dim);
    head_map(ctx, &maps[4], a.out, a.os, a.batch, a.q_len, a.heads, a.dim);
    if (a.dim <= 64) launch_by_mask<64>(ctx, maps, p); else launch_by_mask<128>(ctx, maps, p);
    bounds.release();
}

}  // namespace ormi_b200
