// What the tensor-core attention kernels share: the tensor maps, which tiles of keys a tile of queries meets, and the
// score of a pair.
#pragma once
#include "attention.cuh"
#include "tc.cuh"

namespace ormi_b200 {

constexpr int kTile = 128, kUnit = 64;           // positions of a tile, and of half of one
constexpr int kMaxTiles = 8192;                  // tiles of keys (of queries in attn_back_kv) that a block keeps a class for: 2^20 positions
enum TileClass { kSkip = 0, kFull = 1, kPartial = 2, kDocs = 3 };   // no pair visible; every pair; look at positions; and at documents too

// Raw products to capped base-2 scores (below).  With a cap: cap * log2(e), 2 log2(e) scale / cap, -1 / cap_log2^2, the
// polynomial and the largest |raw| for it.
struct CapTerms { float cap_log2, exp_per_raw, minus_inv_cap2, poly[4], poly_limit; };

struct TcParams {
    AttnParams a;
    const int2 *q_bounds, *k_bounds;             // smallest and largest document of every unit, [batch][units]; NULL without documents
    int q_units, k_units;                        // even
    float scale_log2;                            // scale * log2(e)
    CapTerms cap;
    int cluster;                                 // backward pass: blocks that share the query heads of a key/value head
    int* err;
};

// Class of a tile of queries (the two units from q_unit on) against a tile of keys (two from k_unit on).  `lo` and `hi`: key_end of the first
// query and of the last one that exists.
__device__ __forceinline__ int tile_class(const TcParams& p, int b, int q_unit, int lo, int hi, int k_unit) {
    const int key0 = k_unit * kUnit;
    if (key0 >= hi) return kSkip;
    const int c = key0 + kTile <= lo ? kFull : kPartial;
    if (!p.k_bounds) return c;
    const int2* qb = p.q_bounds + (int64_t)b * p.q_units + q_unit;
    const int2* kb = p.k_bounds + (int64_t)b * p.k_units + k_unit;
    const int2 q = make_int2(min(qb[0].x, qb[1].x), max(qb[0].y, qb[1].y)), k = make_int2(min(kb[0].x, kb[1].x), max(kb[0].y, kb[1].y));
    if (k.y < q.x || k.x > q.y) return kSkip;
    return k.x == k.y && q.x == q.y ? c : kDocs;
}

// Raw products to base-2 scores under a cap: z = cap tanh(x), x = raw * scale / cap; the derivative 1 - tanh(x)^2 follows from
// z.  Scores are a few units wide and caps tens of units, so |x| is small: up to 0.4, tanh(x) / x is a polynomial of four
// terms in x^2 (Chebyshev fit, relative error 1e-7), its coefficients scaled on the host so that it takes raw^2 and gives
// z / raw.  A warp whose products leave that range takes tanh(x) = 1 - 2 / (e^2x + 1): two operations of the special
// function unit, off by a few 1e-7 of the cap.
template <int N>
__device__ __forceinline__ bool cap_is_polynomial(const CapTerms& p, const float2 (&z)[N]) {
    float big = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) big = tc::max3(big, fabsf(z[i].x), fabsf(z[i].y));
    return __all_sync(0xffffffffu, big <= p.poly_limit);
}
__device__ __forceinline__ float2 cap_polynomial(const CapTerms& p, const float2& raw) {
    const float2 u = tc::mul2(raw, raw);
    float2 t = tc::fma2(u, tc::both(p.poly[3]), tc::both(p.poly[2]));
    t = tc::fma2(u, t, tc::both(p.poly[1]));
    return tc::mul2(raw, tc::fma2(u, t, tc::both(p.poly[0])));
}
__device__ __forceinline__ float2 cap_any(const CapTerms& p, const float2& raw) {
    return make_float2(fmaf(-2.f * p.cap_log2, __fdividef(1.f, tc::ex2(raw.x * p.exp_per_raw) + 1.f), p.cap_log2),
                       fmaf(-2.f * p.cap_log2, __fdividef(1.f, tc::ex2(raw.y * p.exp_per_raw) + 1.f), p.cap_log2));
}
__device__ __forceinline__ float2 cap_slope(const CapTerms& p, const float2& z) { return tc::fma2(tc::mul2(z, z), tc::both(p.minus_inv_cap2), tc::both(1.f)); }

// A warp's 32 rows x COLS columns of fp32 accumulators in tensor memory (a row per lane) as bf16 to global memory, times `by`:
// through a staging buffer of the warp (32 x COLS x 2 bytes), so that neighbouring lanes write a whole row and not each lane
// 16 bytes of its own.  have: false gives zeros.  row_ptr(r): where row r goes; columns from `cols` on and rows from `rows`
// on are left out.
template <int COLS, typename F>
__device__ __forceinline__ void store_rows(uint32_t taddr, bool have, uint32_t stage, float by, int rows, int cols, F&& row_ptr) {
    constexpr int LPR = COLS / 8, MASK = LPR < 8 ? LPR - 1 : 7;
    const int lane = threadIdx.x & 31;
    uint32_t o[COLS];
    if (have) {
#pragma unroll
        for (int x = 0; x < COLS; x += 32) tc::ld32(taddr + x, o + x);
        tc::wait_ld();
    } else {
#pragma unroll
        for (int x = 0; x < COLS; ++x) o[x] = 0;
    }
#pragma unroll
    for (int i = 0; i < LPR; ++i) {
        uint32_t v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = pack_bf16x2(__uint_as_float(o[8 * i + 2 * k]) * by, __uint_as_float(o[8 * i + 2 * k + 1]) * by);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * (COLS * 2) + ((i ^ (lane & MASK)) << 4)), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < LPR; ++k) {
        const int r = k * (32 / LPR) + lane / LPR, c = lane % LPR;
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(stage + r * (COLS * 2) + ((c ^ (r & MASK)) << 4)) : "memory");
        if (r < rows && 8 * c < cols) *reinterpret_cast<uint4*>((bf16*)row_ptr(r) + 8 * c) = v;
    }
}

bool attention_tc_supported(const AttnParams& p, int dtype);
void attention_tc(ormi_b200_ctx* ctx, AttnParams& p);
bool attention_backward_tc_supported(const AttnParams& p, int dtype);
void attention_backward_tc(ormi_b200_ctx* ctx, AttnParams& p);

// host side (attention_tc.cu)
void head_map(ormi_b200_ctx* ctx, CUtensorMap* map, const void* ptr, const Strides4& s, int batch, int len, int heads, int dim, int rows = kTile);
bool map_allowed(const void* ptr, const Strides4& s, int batch, int len, int heads);
TcParams tc_params(ormi_b200_ctx* ctx, const AttnParams& p, int2* bounds);
size_t bounds_bytes(const AttnParams& p);
CapTerms cap_terms(const AttnParams& p);
bool cap_terms_exist(const AttnParams& p);
template <typename T> inline int units_of(T len) { return (int)((len + kTile - 1) / kTile) * 2; }

}  // namespace ormi_b200
