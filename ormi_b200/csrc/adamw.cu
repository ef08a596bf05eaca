// AdamW over many tensors in one launch, with states in 32 bits or in 8.
//
//   g = grad * gs;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p -= lr wd p + lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// Bound by memory: 28 bytes per parameter with fp32 gradients and states, 16 with 8-bit states.  The tensors' descriptors
// travel as kernel parameters (no copy to the device, so a call can be captured); a block takes a chunk of one tensor and
// finds it by binary search over the running chunk counts.
//
// 8-bit states: e4m3 codes of m and of sqrt(v) (the root halves the exponent range: 2^17.8 of a block's codes span 2^35 of
// v), one fp32 scale per 128 elements.  An update moves sqrt(v) by a fraction of a per cent, far less than half a step of a
// 3-bit mantissa (6 %): rounding to nearest would freeze the state, so codes are rounded up with the probability of
// what they are above the code below (unbiased), from 16 bits each of a 32-bit hash.  A code depends on the last bits of
// m and v, so these are computed operation by operation (no contraction into FMAs): the formulas evaluated in fp32 in their
// written order give the same codes on any machine.
#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>
#include <vector>

#include "op_math.cuh"
#include "operators.h"
#include "tc.cuh"

namespace ormi_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;                 // elements per block: 32 blocks of 128 that share a scale

struct Tensor {
    float* param;
    const void* grad;
    void *m, *v;
    float *m_scales, *v_scales;
    bf16* copy16;
    int64_t n;
    float decay;
    int first_chunk;                          // running count of chunks before this tensor
    int index;                                // position in the caller's list (part of the rounding hash)
    uint8_t grad_f32, vec;                    // vec: every pointer allows 4-element accesses
};
struct Common {
    float b1, b2, c1, c2, eps, lr, inv_bc1, inv_sqrt_bc2;      // c1 = 1 - b1, c2 = 1 - b2
    double b1_d, b2_d;
    const float* device_lr;
    const float* grad_scale;
    const int64_t* device_step;
    int64_t step;
    uint32_t seed;
    int n;
};
template <int N> struct Batch { Common c; Tensor t[N]; };

// Two rounds of xor-shift and multiply (constants of C. Wellons' published search): every input bit reaches every output bit.
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x ^= x >> 16; x *= 0x7feb352du;
    x ^= x >> 15; x *= 0x846ca68bu;
    return x ^ (x >> 16);
}

// 0 <= a <= 448 to an e4m3 value, up with the probability u / 2^16 of what it is above the value below (u: 16 bits).  From 2^-6
// on the value below is a with the last 20 bits of its mantissa cut off: adding u << 4 carries with that probability, 448
// itself has nothing to carry from.  Below, values are 2^-9 apart.
__device__ __forceinline__ float to_e4m3_grid(float a, uint32_t u) {
    if (a < 0x1p-6f) return floorf(a * 512.f + (float)u * (1.f / 65536.f)) * 0x1p-9f;
    return __uint_as_float((__float_as_uint(a) + (u << 4)) & 0xfff00000u);
}

struct Rates { float lr, inv_bc1, inv_sqrt_bc2, gs; uint32_t key; };

// The step number and what follows from it: from the host, or from the device counter of a captured step.
__device__ __forceinline__ Rates rates_of(const Common& c) {
    Rates r{c.lr, c.inv_bc1, c.inv_sqrt_bc2, 1.f, 0};
    int64_t step = c.step;
    if (c.device_step) {
        step = *c.device_step + 1;
        r.inv_bc1 = 1.f / (float)(1.0 - pow(c.b1_d, (double)step));
        r.inv_sqrt_bc2 = (float)(1.0 / sqrt(1.0 - pow(c.b2_d, (double)step)));
    }
    if (c.device_lr) r.lr = *c.device_lr;
    if (c.grad_scale) r.gs = *c.grad_scale;
    r.key = mix32(c.seed ^ (uint32_t)step);
    return r;
}

// b1 m + c1 g and b2 v + (c2 g) g, each operation rounded by itself
__device__ __forceinline__ float next_m(const Common& c, float m, float g) { return __fadd_rn(__fmul_rn(c.b1, m), __fmul_rn(c.c1, g)); }
__device__ __forceinline__ float next_v(const Common& c, float v, float g) { return __fadd_rn(__fmul_rn(c.b2, v), __fmul_rn(__fmul_rn(c.c2, g), g)); }

__device__ __forceinline__ float quick_inverse(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// The quotient is an approximate one (2 ulp of the update, which is a small part of the parameter): an exact division costs
// as much as the rest of the update.
__device__ __forceinline__ float updated(float p, float m, float root, float decay, const Rates& r, float eps) {
    return p - (r.lr * decay * p + r.lr * r.inv_bc1 * m * quick_inverse(root * r.inv_sqrt_bc2 + eps));
}

// Four gradients from element i on.
__device__ __forceinline__ float4 grads4(const Tensor& t, int64_t i) {
    if (t.grad_f32) return *reinterpret_cast<const float4*>((const float*)t.grad + i);
    const uint2 u = *reinterpret_cast<const uint2*>((const bf16*)t.grad + i);
    return make_float4(bf16_lo(u.x), bf16_hi(u.x), bf16_lo(u.y), bf16_hi(u.y));
}

template <int N> __device__ __forceinline__ const Tensor& tensor_of(const Batch<N>& b, int chunk) {
    int lo = 0, hi = b.c.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (b.t[mid].first_chunk <= chunk) lo = mid; else hi = mid - 1;
    }
    return b.t[lo];
}

// States in 32 bits, any alignment.
template <int N>
__global__ void __launch_bounds__(kThreads) adamw_f32(const __grid_constant__ Batch<N> b) {
    __shared__ Rates shared_rates;
    if (threadIdx.x == 0) shared_rates = rates_of(b.c);
    __syncthreads();
    const Rates r = shared_rates;
    const Tensor t = tensor_of(b, blockIdx.x);
    const int64_t base = (int64_t)((int)blockIdx.x - t.first_chunk) * kChunk, end = min(base + kChunk, t.n);
    float* pm = (float*)t.m;
    float* pv = (float*)t.v;
    // four elements at a time; every load of the chunk is asked for first (33.6 million parameters with bf16 copies: 154 us,
    // 6560 GB/s; element by element 195 us)
    if (t.vec && end - base == kChunk) {
        float4 p[4], m[4], v[4], g[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t i = base + (k * kThreads + threadIdx.x) * 4;
            p[k] = *reinterpret_cast<const float4*>(t.param + i);
            m[k] = *reinterpret_cast<const float4*>(pm + i);
            v[k] = *reinterpret_cast<const float4*>(pv + i);
            g[k] = grads4(t, i);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t i = base + (k * kThreads + threadIdx.x) * 4;
            auto one = [&](float& p, float& m, float& v, float g) {
                m = next_m(b.c, m, g * r.gs); v = next_v(b.c, v, g * r.gs);
                p = updated(p, m, sqrtf(v), t.decay, r, b.c.eps);
            };
            one(p[k].x, m[k].x, v[k].x, g[k].x); one(p[k].y, m[k].y, v[k].y, g[k].y);
            one(p[k].z, m[k].z, v[k].z, g[k].z); one(p[k].w, m[k].w, v[k].w, g[k].w);
            *reinterpret_cast<float4*>(t.param + i) = p[k];
            *reinterpret_cast<float4*>(pm + i) = m[k];
            *reinterpret_cast<float4*>(pv + i) = v[k];
            if (t.copy16) *reinterpret_cast<uint2*>(t.copy16 + i) = make_uint2(pack_bf16x2(p[k].x, p[k].y), pack_bf16x2(p[k].z, p[k].w));
        }
        return;
    }
    for (int64_t i = base + threadIdx.x; i < end; i += kThreads) {
        const float g = (t.grad_f32 ? ((const float*)t.grad)[i] : __bfloat162float(((const bf16*)t.grad)[i])) * r.gs;
        const float m = next_m(b.c, pm[i], g), v = next_v(b.c, pv[i], g);
        const float p = updated(t.param[i], m, sqrtf(v), t.decay, r, b.c.eps);
        pm[i] = m; pv[i] = v; t.param[i] = p;
        if (t.copy16) t.copy16[i] = __float2bfloat16_rn(p);
    }
}

// The 128 elements that share a scale, 4 per lane: new parameters in p, new states as codes.  `h` are the elements' hashes.
// Two elements per instruction where there is such an instruction: this kernel is bound by instructions as much as by memory.
__device__ __forceinline__ void step_block(const Common& c, const Rates& r, float decay, const uint32_t (&h)[4], const float (&g)[4], const float (&cm)[4], const float (&cv)[4], float sm, float sv,
                                           float (&p)[4], float (&qm)[4], float (&qv)[4], float& hi_m, float& hi_v) {
    using namespace tc;
    // a packed product and a packed sum were seen to be fused into one operation; a packed product and two plain sums are not
    auto sum_of = [](const float2& a, const float2& b) { return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)); };
    float2 m[2], root[2];
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float2 grad = mul2(make_float2(g[2 * k], g[2 * k + 1]), both(r.gs)), old = mul2(make_float2(cv[2 * k], cv[2 * k + 1]), both(sv));
        m[k] = sum_of(mul2(both(c.b1), mul2(make_float2(cm[2 * k], cm[2 * k + 1]), both(sm))), mul2(both(c.c1), grad));
        const float2 v = sum_of(mul2(both(c.b2), mul2(old, old)), mul2(mul2(both(c.c2), grad), grad));
        root[k] = make_float2(sqrtf(v.x), sqrtf(v.y));
        const float2 den = fma2(root[k], both(r.inv_sqrt_bc2), both(c.eps));
        const float2 up = mul2(mul2(m[k], both(r.lr * r.inv_bc1)), make_float2(quick_inverse(den.x), quick_inverse(den.y)));
        const float2 now = make_float2(p[2 * k], p[2 * k + 1]), off = fma2(now, both(r.lr * decay), up);
        p[2 * k] = now.x - off.x;
        p[2 * k + 1] = now.y - off.y;
        top_m = max(max(top_m, mag(m[k].x)), mag(m[k].y));
        top_v = max(max(top_v, __float_as_uint(root[k].x)), __float_as_uint(root[k].y));
    }
    hi_m = __uint_as_float(__reduce_max_sync(0xffffffffu, top_m));
    hi_v = __uint_as_float(__reduce_max_sync(0xffffffffu, top_v));
    // codes per unit, 448 / top: one half of the warp divides for m, the other for sqrt(v).  Below 1.3e-36 that leaves fp32 (only
    // m gets there: the root of the smallest v is 3.7e-23), so a small m is lifted by 2^64 first, which is exact.
    float top = hi_m;
    if (hi_m < 0x1p-100f) {
        top *= 0x1p64f;
        m[0] = mul2(m[0], both(0x1p64f)); m[1] = mul2(m[1], both(0x1p64f));
    }
    const float mine = threadIdx.x & 16 ? hi_v : top, up = mine > 0.f ? __fmul_rn(1.f / mine, 448.f) : 0.f;
    const float2 up_m = both(__shfl_sync(0xffffffffu, up, 0)), up_v = both(__shfl_sync(0xffffffffu, up, 16));
    uint32_t a[4], b[4], least = 0xffffffffu;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float2 x = mul2(m[k], up_m), y = mul2(root[k], up_v);
        // magnitudes as integers, at most 448 (a product of two roundings may lie just above)
        a[2 * k] = min(mag(x.x), 0x43e00000u); a[2 * k + 1] = min(mag(x.y), 0x43e00000u);
        b[2 * k] = min(__float_as_uint(y.x), 0x43e00000u); b[2 * k + 1] = min(__float_as_uint(y.y), 0x43e00000u);
        least = min(min(least, min(a[2 * k], a[2 * k + 1])), min(b[2 * k], b[2 * k + 1]));
    }
    if (least >= 0x3c800000u) {                                 // 2^-6: everything has a full mantissa
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            a[k] = (a[k] + ((h[k] << 4) & 0xffff0u)) & 0xfff00000u;
            b[k] = (b[k] + ((h[k] >> 12) & 0xffff0u)) & 0xfff00000u;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool some = k & 1 ? root[k / 2].y > 0.f : root[k / 2].x > 0.f;
            a[k] = __float_as_uint(to_e4m3_grid(__uint_as_float(a[k]), h[k] & 0xffffu));
            b[k] = __float_as_uint(to_e4m3_grid(some ? fmaxf(__uint_as_float(b[k]), 0x1p-9f) : 0.f, h[k] >> 16));
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float sign = k & 1 ? m[k / 2].y : m[k / 2].x;
        qm[k] = __uint_as_float(a[k] | (__float_as_uint(sign) & 0x80000000u));
        qv[k] = __uint_as_float(b[k]);
    }
    // a state that is not a number stays one: the clamp above took it for a large value
    if (!(hi_m < INFINITY)) { for (int k = 0; k < 4; ++k) qm[k] = NAN; }
    if (!(hi_v < INFINITY)) { for (int k = 0; k < 4; ++k) qv[k] = NAN; }
}

__device__ __forceinline__ void codes4(uint32_t u, float (&v)[4]) {
    const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u & 0xffff), __NV_E4M3), hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u >> 16), __NV_E4M3);
    const float2 a = __half22float2(lo), b = __half22float2(hi);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
__device__ __forceinline__ uint32_t to_codes4(const float (&v)[4]) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E4M3) | (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[2], v[3]), __NV_SATFINITE, __NV_E4M3) << 16;
}

// States in 8 bits: a warp owns the 128 elements that share a scale; four in a row per lane where aligned, else 32 apart.
template <int N>
__global__ void __launch_bounds__(kThreads, 4) adamw_e4m3(const __grid_constant__ Batch<N> b) {
    __shared__ Rates shared_rates;
    if (threadIdx.x == 0) shared_rates = rates_of(b.c);
    __syncthreads();
    const Rates r = shared_rates;
    const Tensor t = tensor_of(b, blockIdx.x);
    const int64_t base = (int64_t)((int)blockIdx.x - t.first_chunk) * kChunk, end = min(base + kChunk, t.n);
    const uint32_t key = mix32(r.key + (uint32_t)t.index);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    e4m3* cm = (e4m3*)t.m;
    e4m3* cv = (e4m3*)t.v;
    if (t.vec && end - base == kChunk) {
        // A warp takes four blocks.  All their values are asked for at once, into shared memory (cp.async, every lane its own
        // pieces: nobody waits for anybody), so that 160 KB per SM are on their way without holding registers (134 million parameters:
        // 388 us, 5560 GB/s alone at 1965 MHz, 421 us in a loop, where the power limit leaves 1730 MHz; loads into registers, two
        // blocks per SM: 457 us alone).
        constexpr int TURNS = kChunk / (kThreads / 32 * 128);
        __shared__ __align__(16) struct { float4 p[kThreads], g[kThreads]; uint32_t m[kThreads], v[kThreads]; } box[TURNS];
        auto first_of = [&](int k) { return base + (k * (kThreads / 32) + warp) * 128; };
        auto copy = [](void* to, const void* from, auto bytes) {
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(tc::smem_u32(to)), "l"(from), "n"(decltype(bytes)::value) : "memory");
        };
        using B4 = std::integral_constant<int, 4>; using B8 = std::integral_constant<int, 8>; using B16 = std::integral_constant<int, 16>;
        float sm[TURNS], sv[TURNS];
#pragma unroll
        for (int k = 0; k < TURNS; ++k) {
            const int64_t first = first_of(k), i = first + lane * 4;
            copy(&box[k].p[threadIdx.x], t.param + i, B16{});
            if (t.grad_f32) copy(&box[k].g[threadIdx.x], (const float*)t.grad + i, B16{}); else copy(&box[k].g[threadIdx.x], (const bf16*)t.grad + i, B8{});
            copy(&box[k].m[threadIdx.x], cm + i, B4{});
            copy(&box[k].v[threadIdx.x], cv + i, B4{});
            asm volatile("cp.async.commit_group;" ::: "memory");
            sm[k] = t.m_scales[first >> 7]; sv[k] = t.v_scales[first >> 7];
        }
#pragma unroll
        for (int k = 0; k < TURNS; ++k) {
            if (k == 0) asm volatile("cp.async.wait_group 3;" ::: "memory");
            else if (k == 1) asm volatile("cp.async.wait_group 2;" ::: "memory");
            else if (k == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
            else asm volatile("cp.async.wait_group 0;" ::: "memory");
            const int64_t first = first_of(k), i = first + lane * 4;
            const float4 pp = box[k].p[threadIdx.x];
            float4 gg = box[k].g[threadIdx.x];
            if (!t.grad_f32) {
                const uint32_t lo = __float_as_uint(gg.x), hi = __float_as_uint(gg.y);
                gg = make_float4(bf16_lo(lo), bf16_hi(lo), bf16_lo(hi), bf16_hi(hi));
            }
            float p[4] = {pp.x, pp.y, pp.z, pp.w}, m[4], v[4], qm[4], qv[4], hi_m, hi_v;
            const float g[4] = {gg.x, gg.y, gg.z, gg.w};
            codes4(box[k].m[threadIdx.x], m);
            codes4(box[k].v[threadIdx.x], v);
            const uint32_t h[4] = {mix32((uint32_t)i ^ key), mix32((uint32_t)(i + 1) ^ key), mix32((uint32_t)(i + 2) ^ key), mix32((uint32_t)(i + 3) ^ key)};
            step_block(b.c, r, t.decay, h, g, m, v, sm[k], sv[k], p, qm, qv, hi_m, hi_v);
            *reinterpret_cast<float4*>(t.param + i) = make_float4(p[0], p[1], p[2], p[3]);
            *reinterpret_cast<uint32_t*>(cm + i) = to_codes4(qm);
            *reinterpret_cast<uint32_t*>(cv + i) = to_codes4(qv);
            if (t.copy16) *reinterpret_cast<uint2*>(t.copy16 + i) = make_uint2(pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]));
            if (lane == 0) { t.m_scales[first >> 7] = hi_m * (1.f / 448.f); t.v_scales[first >> 7] = hi_v * (1.f / 448.f); }
        }
        return;
    }
    for (int64_t first = base + warp * 128; first < end; first += kThreads / 32 * 128) {
        const float sm = t.m_scales[first >> 7], sv = t.v_scales[first >> 7];
        float p[4], g[4], m[4], v[4], qm[4], qv[4], hi_m, hi_v;
        auto at = [&](int e) { return first + e * 32 + lane; };
        // behind the end: zeros, which leave zeros
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool in = at(e) < end;
            p[e] = in ? t.param[at(e)] : 0.f;
            g[e] = !in ? 0.f : t.grad_f32 ? ((const float*)t.grad)[at(e)] : __bfloat162float(((const bf16*)t.grad)[at(e)]);
            m[e] = in ? float(cm[at(e)]) : 0.f;
            v[e] = in ? float(cv[at(e)]) : 0.f;
        }
        const uint32_t h[4] = {mix32((uint32_t)at(0) ^ key), mix32((uint32_t)at(1) ^ key), mix32((uint32_t)at(2) ^ key), mix32((uint32_t)at(3) ^ key)};
        step_block(b.c, r, t.decay, h, g, m, v, sm, sv, p, qm, qv, hi_m, hi_v);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (at(e) >= end) continue;
            t.param[at(e)] = p[e];
            if (t.copy16) t.copy16[at(e)] = __float2bfloat16_rn(p[e]);
            cm[at(e)] = from_f32<e4m3>(qm[e]);
            cv[at(e)] = from_f32<e4m3>(qv[e]);
        }
        if (lane == 0) { t.m_scales[first >> 7] = hi_m * (1.f / 448.f); t.v_scales[first >> 7] = hi_v * (1.f / 448.f); }
    }
}

__global__ void count_step(int64_t* step) { ++*step; }

template <int N>
void launch(ormi_b200_ctx* ctx, Batch<N>& b, int chunks, int state_bits) {
    if (state_bits == 32) adamw_f32<N><<<chunks, kThreads, 0, ctx->stream>>>(b);
    else adamw_e4m3<N><<<chunks, kThreads, 0, ctx->stream>>>(b);
    ORMI_CUDA(cudaGetLastError());
    count_launch(ctx);
}

// The context's bf16 copy of `param` when it is a plain copy of exactly these n values (it is rewritten along with them);
// any other copy that overlaps is stale and goes.  A captured step keeps rewriting the copy on every replay, so its graph
// holds the copy's block.
void* kept_copy(ormi_b200_ctx* ctx, const ormi_b200_adamw_tensor& t) {
    if (ctx->shadows.empty()) return nullptr;
    auto it = ctx->shadows.find(t.param);
    const bool whole = it != ctx->shadows.end() && it->second.ld == it->second.cols && (int64_t)it->second.rows * it->second.cols == t.n;
    if (!whole || t.copy16) { shadow_drop(ctx, t.param, (size_t)t.n * 4); return nullptr; }
    const Shadow16 keep = it->second;
    ctx->shadows.erase(it);
    shadow_drop(ctx, t.param, (size_t)t.n * 4);
    ctx->shadows[t.param] = keep;
    shadow_borrow(ctx, t.param, keep);
    return keep.ptr;
}

}  // namespace

void adamw_check(const ormi_b200_adamw_tensor* t, int n, const ormi_b200_adamw_config& c) {
    const char* op = "adamw";
    OP_NEED(c.state_bits == 32 || c.state_bits == 8, op, "state_bits is 32 or 8");
    OP_NEED(c.device_step || c.step >= 1, op, "step counts from 1");
    OP_NEED(c.beta1 >= 0 && c.beta1 < 1 && c.beta2 >= 0 && c.beta2 < 1, op, "beta1 and beta2 lie in [0, 1)");
    OP_NEED(c.eps >= 0 && std::isfinite(c.eps), op, "eps is negative or not finite");
    OP_NEED(c.eps == 0 || (float)c.eps >= std::numeric_limits<float>::min(), op, "eps is above zero and below 2^-126");
    OP_NEED(std::isfinite(c.lr), op, "lr is not finite");
    OP_NEED((uintptr_t)c.device_step % 8 == 0 && (uintptr_t)c.device_lr % 4 == 0 && (uintptr_t)c.grad_scale % 4 == 0, op, "a device scalar does not start on a whole element");
    struct Range { const char* lo; const char* hi; bool out; int tensor; };
    std::vector<Range> ranges;
    for (int i = 0; i < n; ++i) {
        const ormi_b200_adamw_tensor& x = t[i];
        auto who = [&] { return "tensor " + std::to_string(i) + ": "; };
        OP_NEED(x.n >= 0 && x.n < (int64_t)1 << 40, op, who() + "n is negative or above 2^40");
        if (x.n == 0) continue;
        OP_NEED(x.param && x.grad && x.m && x.v, op, who() + "param, grad, m and v are needed");
        OP_NEED(x.grad_dtype == ORMI_F32 || x.grad_dtype == ORMI_BF16, op, who() + "grad is F32 or BF16");
        OP_NEED(std::isfinite(x.weight_decay), op, who() + "weight_decay is not finite");
        OP_NEED((x.m_scales && x.v_scales) == (c.state_bits == 8) && (c.state_bits == 8 || (!x.m_scales && !x.v_scales)), op, who() + "m_scales and v_scales go with 8-bit states, and only with them");
        const uintptr_t state = c.state_bits == 32 ? 4 : 1;
        OP_NEED((uintptr_t)x.param % 4 == 0 && (uintptr_t)x.grad % dtype_bytes(x.grad_dtype) == 0 && (uintptr_t)x.m % state == 0 && (uintptr_t)x.v % state == 0 &&
                (uintptr_t)x.m_scales % 4 == 0 && (uintptr_t)x.v_scales % 4 == 0 && (uintptr_t)x.copy16 % 2 == 0, op, who() + "a buffer does not start on a whole element");
        auto add = [&](const void* p, int64_t bytes, bool out) { if (p) ranges.push_back({(const char*)p, (const char*)p + bytes, out, i}); };
        add(x.param, x.n * 4, true); add(x.grad, x.n * dtype_bytes(x.grad_dtype), false);
        add(x.m, x.n * (int64_t)state, true); add(x.v, x.n * (int64_t)state, true);
        add(x.m_scales, (x.n + 127) / 128 * 4, true); add(x.v_scales, (x.n + 127) / 128 * 4, true);
        add(x.copy16, x.n * 2, true);
    }
    auto scalar = [&](const void* p, int64_t bytes, bool out) { if (p) ranges.push_back({(const char*)p, (const char*)p + bytes, out, -1}); };
    scalar(c.device_step, 8, true); scalar(c.device_lr, 4, false); scalar(c.grad_scale, 4, false);
    // what is written lies apart from everything else (the same tensor twice would be updated by two blocks at once)
    std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
    const char* end_any = nullptr; const char* end_out = nullptr;
    for (const Range& r : ranges) {
        OP_NEED(!(r.lo < end_out || (r.out && r.lo < end_any)), op, (r.tensor < 0 ? std::string("a device scalar") : "tensor " + std::to_string(r.tensor)) + ": a buffer that is written overlaps another one");
        end_any = std::max(end_any, r.hi);
        if (r.out) end_out = std::max(end_out, r.hi);
    }
}

void adamw(ormi_b200_ctx* ctx, const ormi_b200_adamw_tensor* t, int n, const ormi_b200_adamw_config& c) {
    Common common{};
    common.b1 = (float)c.beta1; common.b2 = (float)c.beta2; common.c1 = (float)(1.0 - c.beta1); common.c2 = (float)(1.0 - c.beta2);
    common.b1_d = c.beta1; common.b2_d = c.beta2;
    common.eps = (float)c.eps; common.lr = (float)c.lr;
    if (!c.device_step) {
        common.inv_bc1 = 1.f / (float)(1.0 - std::pow(c.beta1, (double)c.step));
        common.inv_sqrt_bc2 = (float)(1.0 / std::sqrt(1.0 - std::pow(c.beta2, (double)c.step)));
    }
    common.device_lr = c.device_lr; common.grad_scale = c.grad_scale; common.device_step = c.device_step;
    common.step = c.step; common.seed = c.seed;
    // 44 descriptors fit the classic 4 KB of kernel parameters; more tensors go 300 at a time (24 KB)
    auto run = [&](auto batch) {
        constexpr int cap = sizeof(batch.t) / sizeof(Tensor);
        int i = 0;
        while (i < n) {
            batch.c = common;
            int64_t chunks = 0;
            int k = 0;
            for (; i < n && k < cap; ++i) {
                const ormi_b200_adamw_tensor& x = t[i];
                if (x.n == 0) continue;
                const int64_t mine = (x.n + kChunk - 1) / kChunk;
                if (chunks + mine > 0x7fffffff) break;
                Tensor& d = batch.t[k++];
                d.param = (float*)x.param; d.grad = x.grad; d.m = x.m; d.v = x.v;
                d.m_scales = (float*)x.m_scales; d.v_scales = (float*)x.v_scales;
                void* kept = kept_copy(ctx, x);
                d.copy16 = (bf16*)(x.copy16 ? x.copy16 : kept);
                d.n = x.n; d.decay = x.weight_decay; d.first_chunk = (int)chunks; d.index = i;
                d.grad_f32 = x.grad_dtype == ORMI_F32;
                const uintptr_t states = (uintptr_t)x.m | (uintptr_t)x.v;
                d.vec = ((uintptr_t)x.param | (c.state_bits == 32 ? states : states * 4)) % 16 == 0 && (uintptr_t)x.grad % (d.grad_f32 ? 16 : 8) == 0 && (uintptr_t)d.copy16 % 8 == 0;
                chunks += mine;
                auto note = [&](void* p, size_t bytes) { written(ctx, p, bytes); };
                if (c.state_bits == 32) { note(x.m, (size_t)x.n * 4); note(x.v, (size_t)x.n * 4); }
                if (ctx->capturing) ctx->capture_writes.push_back({x.param, (size_t)x.n * 4});
            }
            if (!k) break;
            batch.c.n = k;
            launch(ctx, batch, (int)chunks, c.state_bits);
        }
    };
    if (n <= 44) run(Batch<44>{}); else run(Batch<300>{});
    if (c.device_step) {
        count_step<<<1, 1, 0, ctx->stream>>>(c.device_step);
        ORMI_CUDA(cudaGetLastError());
        count_launch(ctx);
    }
}

}  // namespace ormi_b200
