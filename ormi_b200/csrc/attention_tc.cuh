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
    float scale_log2;                            // scale * log2(e); with a cap: 2 log2(e) scale / cap
    float cap_log2;                              // cap * log2(e)
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

// Base-2 score from the raw product.  Without a cap: one multiplication.  With one: cap tanh(x) = cap (1 - 2 / (e^2x + 1)),
// 2x in base 2 being raw * scale_log2; the error of that form is a few 1e-7 of the cap, whatever x.
template <bool CAP>
__device__ __forceinline__ float score_log2(const TcParams& p, float raw) {
    if (!CAP) return raw * p.scale_log2;
    return p.cap_log2 - __fdividef(2.f * p.cap_log2, tc::ex2(raw * p.scale_log2) + 1.f);
}

bool attention_tc_supported(const AttnParams& p, int dtype);
void attention_tc(ormi_b200_ctx* ctx, AttnParams& p);
bool attention_backward_tc_supported(const AttnParams& p, int dtype);
void attention_backward_tc(ormi_b200_ctx* ctx, AttnParams& p);

// host side (attention_tc.cu)
void head_map(ormi_b200_ctx* ctx, CUtensorMap* map, const void* ptr, const Strides4& s, int batch, int len, int heads, int dim);
bool map_allowed(const void* ptr, const Strides4& s, int batch, int len, int heads);
TcParams tc_params(ormi_b200_ctx* ctx, const AttnParams& p, int2* bounds);
size_t bounds_bytes(const AttnParams& p);

}  // namespace ormi_b200
