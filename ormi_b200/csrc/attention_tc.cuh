// What the tensor-core attention kernels share: the tensor maps, which tiles of keys a tile of queries meets, and the
// score of a pair.
#pragma once
#include "attention.cuh"
#include "tc.cuh"

namespace ormi_b200 {

constexpr int kTile = 128;                       // queries, and keys, of a tile
constexpr int kMaxTiles = 8192;                  // tiles of keys (or queries) that a block keeps a class for: 2^20 positions
enum TileClass { kSkip = 0, kFull = 1, kPartial = 2 };   // no pair visible; every pair; look at each

struct TcParams {
    AttnParams a;
    const int2 *q_bounds, *k_bounds;             // smallest and largest document of every tile, [batch][tiles]; NULL without documents
    int q_tiles, k_tiles;
    float scale_log2, cap_log2;                  // scale * log2(e), cap * log2(e)
    float x_per_raw, exp_per_raw, poly_limit;    // with a cap: scale / cap, 2 log2(e) scale / cap, the largest |raw| for the polynomial
    int* err;
};

// Class of (queries first .. first + 127, tile of keys j).  `lo` and `hi`: key_end of the first and the last row that exists.
__device__ __forceinline__ int tile_class(const TcParams& p, int b, int q_tile, int lo, int hi, int j) {
    const int key0 = j * kTile;
    if (key0 >= hi) return kSkip;
    int c = key0 + kTile <= lo ? kFull : kPartial;
    if (p.k_bounds) {
        const int2 q = p.q_bounds[(int64_t)b * p.q_tiles + q_tile], k = p.k_bounds[(int64_t)b * p.k_tiles + j];
        if (k.y < q.x || k.x > q.y) return kSkip;
        if (!(k.x == k.y && q.x == q.y)) c = kPartial;
    }
    return c;
}

// Raw products to base-2 scores under a cap, in place: z = cap tanh(x), x = raw * scale / cap; `dcap`, when given, receives
// 1 - tanh(x)^2.  Scores are a few units wide and caps tens of units, so |x| is small: while a warp's largest |x| is at most
// 0.5, tanh(x) = x P(x^2) with P of degree 4 (Chebyshev fit, relative error 6e-8 in fp32), all on the FMA pipe.  Above that,
// tanh(x) = 1 - 2 / (e^2x + 1), two operations of the special function unit: off by a few 1e-7 of the cap.
template <int N, bool SLOPE>
__device__ __forceinline__ void cap_scores(const TcParams& p, float2 (&z)[N], float2* dcap) {
    float big = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) big = tc::max3(big, fabsf(z[i].x), fabsf(z[i].y));
    if (__all_sync(0xffffffffu, big <= p.poly_limit)) {
        const float2 k = tc::both(p.x_per_raw), c = tc::both(p.scale_log2);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float2 x = tc::mul2(z[i], k), u = tc::mul2(x, x);
            float2 t = tc::fma2(u, tc::both(0.017141319046484527f), tc::both(-0.052989241174570344f));
            t = tc::fma2(u, t, tc::both(0.13324828997681853f));
            t = tc::fma2(u, t, tc::both(-0.3333307189419646f));
            t = tc::fma2(u, t, tc::both(0.9999999870693153f));
            if (SLOPE) dcap[i] = tc::fma2(tc::mul2(u, t), make_float2(-t.x, -t.y), tc::both(1.f));
            z[i] = tc::mul2(tc::mul2(z[i], c), t);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            // r = 1 / (e^2x + 1): tanh = 1 - 2 r, 1 - tanh^2 = 4 r (1 - r)
            const float rx = __fdividef(1.f, tc::ex2(z[i].x * p.exp_per_raw) + 1.f), ry = __fdividef(1.f, tc::ex2(z[i].y * p.exp_per_raw) + 1.f);
            if (SLOPE) dcap[i] = make_float2(4.f * rx * (1.f - rx), 4.f * ry * (1.f - ry));
            z[i] = make_float2(fmaf(-2.f * p.cap_log2, rx, p.cap_log2), fmaf(-2.f * p.cap_log2, ry, p.cap_log2));
        }
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

}  // namespace ormi_b200
