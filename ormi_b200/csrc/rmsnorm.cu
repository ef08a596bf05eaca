// Root-mean-square norm with the residual's addition, forward and backward.
//
//   forward    s = x + r;  rstd = (mean(s^2) + eps)^-1/2;  y = s * rstd * w;   optionally y as e4m3 codes with scales
//   backward   c = mean(dy w s) * rstd^2;   dx = rstd * (dy w - s c) + ds;   dw = sum over rows of dy s rstd
//
// Both are bound by memory: every element is read and written once and takes a handful of operations.
#include <algorithm>
#include <atomic>

#include "op_math.cuh"
#include "operators.h"

namespace ormi_b200 {
namespace {

struct NormParams {
    const void *x, *residual, *weight;
    void *out, *residual_out;
    float *rstd, *scales;
    int64_t x_row, residual_row, out_row, residual_out_row;   // elements between rows
    int64_t rows;
    int cols, group, groups, weight_f32;
    float eps;
};

__device__ __forceinline__ float weight_at(const void* w, int f32, int c) {
    return !w ? 1.f : f32 ? ((const float*)w)[c] : __bfloat162float(((const bf16*)w)[c]);
}

// The factor 448 / top of a group of e4m3 codes leaves fp32 below 1.3e-36: a smaller group is lifted by 2^64 first (exact).
__device__ __forceinline__ float lift_of(float top) { return top < 0x1p-100f ? 0x1p64f : 1.f; }
__device__ __forceinline__ float codes_per_unit(float top, float lift) { return top > 0.f ? 448.f * (1.f / (top * lift)) : 0.f; }

// One block per row, any width, any alignment (rows too wide for norm_row): three passes over the row (four with one scale for the row), the second
// and later ones out of the caches.  Each element is handled by the same thread in every pass, so `out` and
// `residual_out` may be the inputs.
template <typename T, typename O>
__global__ void __launch_bounds__(256) norm_any(NormParams p) {
    __shared__ float box[33];
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = (const T*)p.x + row * p.x_row;
        const T* r = p.residual ? (const T*)p.residual + row * p.residual_row : nullptr;
        T* keep = p.residual_out ? (T*)p.residual_out + row * p.residual_out_row : nullptr;
        O* out = (O*)p.out + row * p.out_row;
        // after the first pass the sum is read back from residual_out, which may have replaced x or the residual
        auto value = [&](int c) { return keep ? to_f32(keep[c]) : r ? to_f32(from_f32<T>(to_f32(x[c]) + to_f32(r[c]))) : to_f32(x[c]); };
        float sq = 0.f;
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
            const T s = r ? from_f32<T>(to_f32(x[c]) + to_f32(r[c])) : x[c];
            if (keep) keep[c] = s;
            sq += to_f32(s) * to_f32(s);
        }
        const float rstd = 1.f / sqrtf(block_sum(sq, box) / (float)p.cols + p.eps);
        if (p.rstd && threadIdx.x == 0) p.rstd[row] = rstd;
        auto y = [&](int c) { return value(c) * rstd * weight_at(p.weight, p.weight_f32, c); };
        if (!p.scales) {
            for (int c = threadIdx.x; c < p.cols; c += blockDim.x) out[c] = from_f32<O>(y(c));
        } else if (p.group == 0) {
            uint32_t m = 0;
            for (int c = threadIdx.x; c < p.cols; c += blockDim.x) m = max(m, mag(y(c)));
            const float top = block_max_mag(m, (uint32_t*)box);
            const float lift = lift_of(top), up = codes_per_unit(top, lift);
            if (threadIdx.x == 0) p.scales[row] = top * (1.f / 448.f);
            for (int c = threadIdx.x; c < p.cols; c += blockDim.x) out[c] = from_f32<O>(y(c) * lift * up);
        } else {
            // a warp per group of 128 columns
            const int lane = threadIdx.x & 31;
            for (int g = threadIdx.x >> 5; g < p.groups; g += blockDim.x >> 5) {
                float v[4];
                uint32_t m = 0;
                for (int k = 0; k < 4; ++k) {
                    const int c = g * 128 + k * 32 + lane;
                    v[k] = c < p.cols ? y(c) : 0.f;
                    m = max(m, mag(v[k]));
                }
                const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, m));
                const float lift = lift_of(top), up = codes_per_unit(top, lift);
                if (lane == 0) p.scales[row * p.groups + g] = top * (1.f / 448.f);
                for (int k = 0; k < 4; ++k) {
                    const int c = g * 128 + k * 32 + lane;
                    if (c < p.cols) out[c] = from_f32<O>(v[k] * lift * up);
                }
            }
        }
        __syncthreads();
    }
}

// Four 32-bit registers of a row: 16 bytes of it where everything is aligned, else four single elements 32 columns apart.
template <typename T, bool AL> struct Piece {
    static constexpr int VEC = AL ? 16 / (int)sizeof(T) : 4;
    static constexpr int CHUNK = 32 * VEC;                     // columns of a warp's 32 pieces
    uint32_t w[4];
    // column of element e: first + e where aligned, first + 32 e where not
    static __device__ __forceinline__ int first(int chunk) { return chunk * CHUNK + (threadIdx.x & 31) * (AL ? VEC : 1); }
    static __device__ __forceinline__ int col(int c0, int e) { return c0 + (AL ? e : 32 * e); }
    __device__ __forceinline__ void load(const T* row, int c0, int cols) {
        if (AL) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (c0 < cols) v = *reinterpret_cast<const uint4*>(row + c0);
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = c0 + 32 * e < cols ? __float_as_uint(to_f32(row[c0 + 32 * e])) : 0u;
        }
    }
    __device__ __forceinline__ float get(int e) const {
        if (AL && sizeof(T) == 2) return e & 1 ? bf16_hi(w[e >> 1]) : bf16_lo(w[e >> 1]);
        return __uint_as_float(w[e]);
    }
};

// VEC values to a row of type O, in Piece order.
template <typename O, bool AL, int VEC>
__device__ __forceinline__ void put(O* row, int c0, int cols, const float (&v)[VEC]) {
    if (!AL) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) if (c0 + 32 * e < cols) row[c0 + 32 * e] = from_f32<O>(v[e]);
        return;
    }
    if (c0 >= cols) return;
    if (sizeof(O) == 4) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) *reinterpret_cast<float4*>((float*)row + c0 + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    } else if (sizeof(O) == 2) {
        uint32_t u[VEC / 2];
#pragma unroll
        for (int e = 0; e < VEC; e += 2) u[e / 2] = pack_bf16x2(v[e], v[e + 1]);
        if (VEC == 8) *reinterpret_cast<uint4*>(row + c0) = make_uint4(u[0], u[1], u[2 % (VEC / 2)], u[3 % (VEC / 2)]);
        else *reinterpret_cast<uint2*>(row + c0) = make_uint2(u[0], u[1]);
    } else {
        uint32_t u[VEC / 4];
#pragma unroll
        for (int e = 0; e < VEC; e += 4)
            u[e / 4] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[e], v[e + 1]), __NV_SATFINITE, __NV_E4M3) |
                       (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[e + 2], v[e + 3]), __NV_SATFINITE, __NV_E4M3) << 16;
        if (VEC == 8) *reinterpret_cast<uint2*>(row + c0) = make_uint2(u[0], u[1 % (VEC / 4)]);
        else *reinterpret_cast<uint32_t*>(row + c0) = u[0];
    }
}

template <bool AL, int VEC>
__device__ __forceinline__ void weights(const void* w, int f32, int c0, int cols, float (&v)[VEC]) {
    if (!w) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = 1.f;
    } else if (!AL) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = c0 + 32 * e < cols ? weight_at(w, f32, c0 + 32 * e) : 0.f;
    } else if (c0 >= cols) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = 0.f;
    } else if (f32) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
            const float4 x = __ldg(reinterpret_cast<const float4*>((const float*)w + c0 + e));
            v[e] = x.x; v[e + 1] = x.y; v[e + 2] = x.z; v[e + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
            const uint2 x = __ldg(reinterpret_cast<const uint2*>((const bf16*)w + c0 + e));
            v[e] = bf16_lo(x.x); v[e + 1] = bf16_hi(x.x); v[e + 2] = bf16_lo(x.y); v[e + 3] = bf16_hi(x.y);
        }
    }
}

// One row per block (of as many warps as the row needs), or per warp for narrow rows: the row is read once and stays in
// registers, four pieces per thread, so that all its loads are in flight together (16384 x 4096 bf16 with residual: 84 us,
// 6360 GB/s; three passes through the caches 406 us).
template <typename T, typename O, bool AL, bool WARP_ROW>
__global__ void __launch_bounds__(WARP_ROW ? 256 : 1024) norm_row(NormParams p) {
    using P = Piece<T, AL>;
    constexpr int NV = 4, VEC = P::VEC;
    __shared__ float box[33];
    const int warp = threadIdx.x >> 5, nw = WARP_ROW ? 1 : blockDim.x >> 5;
    const int64_t row = WARP_ROW ? (int64_t)blockIdx.x * 8 + warp : blockIdx.x;
    if (WARP_ROW && row >= p.rows) return;
    const T* x = (const T*)p.x + row * p.x_row;
    P a[NV], r[NV];
    int c0[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        c0[v] = P::first(WARP_ROW ? v : v * nw + warp);
        a[v].load(x, c0[v], p.cols);
    }
    if (p.residual) {
#pragma unroll
        for (int v = 0; v < NV; ++v) r[v].load((const T*)p.residual + row * p.residual_row, c0[v], p.cols);
    }
    float s[NV][VEC], sq = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            s[v][e] = a[v].get(e);
            if (p.residual) s[v][e] = to_f32(from_f32<T>(s[v][e] + r[v].get(e)));
            sq = fmaf(s[v][e], s[v][e], sq);
        }
    }
    if (p.residual_out) {
#pragma unroll
        for (int v = 0; v < NV; ++v) put<T, AL, VEC>((T*)p.residual_out + row * p.residual_out_row, c0[v], p.cols, s[v]);
    }
    sq = WARP_ROW ? warp_sum(sq) : block_sum(sq, box);
    const float rstd = 1.f / sqrtf(sq / (float)p.cols + p.eps);
    if (p.rstd && (WARP_ROW ? (threadIdx.x & 31) : threadIdx.x) == 0) p.rstd[row] = rstd;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        float w[VEC];
        weights<AL, VEC>(p.weight, p.weight_f32, c0[v], p.cols, w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[v][e] *= rstd * w[e];
    }
    if (sizeof(O) == 1) {
        if (p.group == 0) {
            uint32_t m = 0;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < VEC; ++e) m = max(m, mag(s[v][e]));
            const float top = WARP_ROW ? __uint_as_float(__reduce_max_sync(0xffffffffu, m)) : block_max_mag(m, (uint32_t*)box);
            const float lift = lift_of(top), up = codes_per_unit(top, lift);
            if ((WARP_ROW ? (threadIdx.x & 31) : threadIdx.x) == 0) p.scales[row] = top * (1.f / 448.f);
            if (lift != 1.f) {
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) s[v][e] *= lift;
            }
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < VEC; ++e) s[v][e] *= up;
        } else {
            // 128 columns are a warp's piece, or half of it where a piece holds 8 values
            const uint32_t half = VEC == 8 ? (threadIdx.x & 16 ? 0xffff0000u : 0x0000ffffu) : 0xffffffffu;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                uint32_t m = 0;
#pragma unroll
                for (int e = 0; e < VEC; ++e) m = max(m, mag(s[v][e]));
                const float top = __uint_as_float(__reduce_max_sync(half, m));
                const float lift = lift_of(top), up = codes_per_unit(top, lift);
                if ((threadIdx.x & (VEC == 8 ? 15 : 31)) == 0 && c0[v] < p.cols) p.scales[row * p.groups + c0[v] / 128] = top * (1.f / 448.f);
                if (lift != 1.f) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) s[v][e] *= lift;
                }
#pragma unroll
                for (int e = 0; e < VEC; ++e) s[v][e] *= up;
            }
        }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) put<O, AL, VEC>((O*)p.out + row * p.out_row, c0[v], p.cols, s[v]);
}

struct NormBackParams {
    const void *dout, *s, *weight, *dresidual;
    const float* rstd;
    void *dx, *dweight;
    float* partial;                                            // [parts][cols] partial sums of dweight
    int64_t dout_row, s_row, dresidual_row, dx_row;
    int64_t rows;
    int cols, weight_f32;
    int parts;
};

template <typename T>
__global__ void __launch_bounds__(256) norm_back_any(NormBackParams p) {
    __shared__ float box[33];
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* dy = (const T*)p.dout + row * p.dout_row;
        const T* s = (const T*)p.s + row * p.s_row;
        const T* ds = p.dresidual ? (const T*)p.dresidual + row * p.dresidual_row : nullptr;
        T* dx = (T*)p.dx + row * p.dx_row;
        const float rstd = p.rstd[row];
        float dot = 0.f;
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x) dot += to_f32(dy[c]) * weight_at(p.weight, p.weight_f32, c) * to_f32(s[c]);
        const float k = block_sum(dot, box) / (float)p.cols * rstd * rstd;
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
            float v = rstd * (to_f32(dy[c]) * weight_at(p.weight, p.weight_f32, c) - to_f32(s[c]) * k);
            if (ds) v += to_f32(ds[c]);
            dx[c] = from_f32<T>(v);
        }
    }
}

// Partial sums of dweight over a slice of the rows: 32 columns x 8 rows at a time.  Runs before norm_back_any, which may
// write dx over dout.
template <typename T>
__global__ void __launch_bounds__(256) norm_dweight_any(NormBackParams p) {
    __shared__ float box[8][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t per = (p.rows + p.parts - 1) / p.parts, lo = blockIdx.y * per, hi = min(lo + per, p.rows);
    float acc = 0.f;
    if (c < p.cols)
        for (int64_t row = lo + w; row < hi; row += 8)
            acc += to_f32(((const T*)p.dout)[row * p.dout_row + c]) * (to_f32(((const T*)p.s)[row * p.s_row + c]) * p.rstd[row]);
    box[w][lane] = acc;
    __syncthreads();
    if (w == 0 && c < p.cols) {
        for (int k = 1; k < 8; ++k) acc += box[k][lane];
        p.partial[(int64_t)blockIdx.y * p.cols + c] = acc;
    }
}

// Rows in registers, as in the forward pass.  A block takes every gridDim-th row (or its warps do), keeps its columns' part of
// dweight in registers from row to row and writes it once.  The rows to come are on their way meanwhile: aligned ones into
// shared memory, where every thread copies (cp.async) and reads back its own pieces, so nobody waits for anybody; others
// into registers, one row ahead (16384 x 4096 bf16: 90 us and 5 us for the join; registers for all of them 110 us).  With 1024 threads there are 64 registers each: the weights are read again for every row.
__device__ __forceinline__ void copy16(void* to, const void* from, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "r"(in ? 16 : 0) : "memory");
}
// bytes of shared memory in front of the copies, and of one row's copies
__host__ __device__ constexpr int back_sum_bytes(bool warp_row, int chunk) { return warp_row ? 2 * chunk * 4 : 0; }
__host__ __device__ constexpr int back_stage_bytes(int threads, int nv) { return 3 * nv * threads * 16; }

template <typename T, bool AL, int THREADS, int NV, int STAGES>   // THREADS: 0 = a row per warp, 8 warps; else the most that a row takes
__global__ void __launch_bounds__(THREADS ? THREADS : 256) norm_back_row(NormBackParams p) {
    using P = Piece<T, AL>;
    constexpr bool WARP_ROW = THREADS == 0, RING = AL, AHEAD = !RING && THREADS <= 512, HOLD = THREADS <= 512;
    constexpr int VEC = P::VEC;
    extern __shared__ __align__(16) unsigned char shared[];
    float* sum_dw = reinterpret_cast<float*>(shared);          // WARP_ROW: one row of dweight
    uint4* ring = reinterpret_cast<uint4*>(shared + back_sum_bytes(WARP_ROW, P::CHUNK));
    __shared__ float box[2][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = WARP_ROW ? 1 : blockDim.x >> 5;
    const int64_t step = WARP_ROW ? (int64_t)gridDim.x * 8 : gridDim.x;
    int64_t row = WARP_ROW ? (int64_t)blockIdx.x * 8 + warp : blockIdx.x;
    int c0[NV];
    float w[NV][VEC], dw[NV][VEC];
    P dy[NV], s[NV], ds[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        c0[v] = P::first(WARP_ROW ? v : v * nw + warp);
        if (HOLD) weights<AL, VEC>(p.weight, p.weight_f32, c0[v], p.cols, w[v]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) dw[v][e] = 0.f;
    }
    auto fetch = [&](int64_t r, P (&a)[NV], P (&b)[NV], P (&c)[NV]) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            a[v].load((const T*)p.dout + r * p.dout_row, c0[v], p.cols);
            b[v].load((const T*)p.s + r * p.s_row, c0[v], p.cols);
            if (p.dresidual) c[v].load((const T*)p.dresidual + r * p.dresidual_row, c0[v], p.cols);
        }
    };
    auto slot = [&](int stage, int which, int v) { return ring + ((stage * 3 + which) * NV + v) * blockDim.x + threadIdx.x; };
    auto ask = [&](int64_t r, int stage) {
        if (r < p.rows) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const bool in = c0[v] < p.cols;
                const int c = in ? c0[v] : 0;
                copy16(slot(stage, 0, v), (const T*)p.dout + r * p.dout_row + c, in);
                copy16(slot(stage, 1, v), (const T*)p.s + r * p.s_row + c, in);
                if (p.dresidual) copy16(slot(stage, 2, v), (const T*)p.dresidual + r * p.dresidual_row + c, in);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto take = [&](int stage, int which, P (&a)[NV]) {
#pragma unroll
        for (int v = 0; v < NV; ++v) { const uint4 u = *slot(stage, which, v); a[v].w[0] = u.x; a[v].w[1] = u.y; a[v].w[2] = u.z; a[v].w[3] = u.w; }
    };
    const float by = 1.f / (float)p.cols;
    float rstd = row < p.rows ? p.rstd[row] : 0.f;
    if (RING) {
#pragma unroll
        for (int k = 0; k < STAGES - 1; ++k) ask(row + k * step, k);
    } else if (row < p.rows) fetch(row, dy, s, ds);
    int stage = 0;
    for (int turn = 0; row < p.rows; turn ^= 1) {
        const int64_t next = row + step;
        if (RING) {
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
            take(stage, 0, dy);
            take(stage, 1, s);
            if (p.dresidual) take(stage, 2, ds);
            const int last = stage == 0 ? STAGES - 1 : stage - 1;          // what was taken a turn ago
            ask(row + (STAGES - 1) * step, last);
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
        float dot = 0.f;
        if (!HOLD) {
#pragma unroll
            for (int v = 0; v < NV; ++v) weights<AL, VEC>(p.weight, p.weight_f32, c0[v], p.cols, w[v]);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < VEC; ++e) dot = fmaf(dy[v].get(e) * w[v][e], s[v].get(e), dot);
        P dy2[NV], s2[NV], ds2[NV];
        if (AHEAD && next < p.rows) fetch(next, dy2, s2, ds2);
        const float rstd2 = next < p.rows ? p.rstd[next] : 0.f;
        dot = warp_sum(dot);
        if (!WARP_ROW) {
            // one barrier per row: the two boxes take turns
            if (lane == 0) box[turn][warp] = dot;
            __syncthreads();
            dot = 0.f;
            for (int k = 0; k < nw; ++k) dot += box[turn][k];
        }
        const float k = dot * by * rstd * rstd;
        T* dx = (T*)p.dx + row * p.dx_row;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float g = dy[v].get(e), x = s[v].get(e);
                o[e] = rstd * (g * w[v][e] - x * k);
                if (p.dresidual) o[e] += ds[v].get(e);
                dw[v][e] = fmaf(g, x * rstd, dw[v][e]);
            }
            put<T, AL, VEC>(dx, c0[v], p.cols, o);
        }
        row = next;
        rstd = rstd2;
        if (AHEAD) {
#pragma unroll
            for (int v = 0; v < NV; ++v) { dy[v] = dy2[v]; s[v] = s2[v]; ds[v] = ds2[v]; }
        } else if (!RING && row < p.rows) fetch(row, dy, s, ds);
    }
    if (!p.dweight) return;
    float* out = p.partial + (int64_t)blockIdx.x * p.cols;
    if (!WARP_ROW) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < VEC; ++e) { const int c = P::col(c0[v], e); if (c < p.cols) out[c] = dw[v][e]; }
        return;
    }
    for (int k = 0; k < 8; ++k) {                              // the warps in order
        if (warp == k) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < VEC; ++e) { const int c = P::col(c0[v], e); if (c < p.cols) sum_dw[c] = k ? sum_dw[c] + dw[v][e] : dw[v][e]; }
        }
        __syncthreads();
    }
    for (int c = threadIdx.x; c < p.cols; c += 256) out[c] = sum_dw[c];
}

// dweight[c] = sum of the partial rows in order: 32 columns per block, its 32 warps share the rows.
__global__ void __launch_bounds__(1024) norm_dweight_join(const float* __restrict__ partial, int parts, int cols, void* dweight, int f32) {
    __shared__ float box[32][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float acc = 0.f;
    if (c < cols) for (int k = w; k < parts; k += 32) acc += partial[(int64_t)k * cols + c];
    box[w][lane] = acc;
    __syncthreads();
    if (w == 0 && c < cols) {
        for (int k = 1; k < 32; ++k) acc += box[k][lane];
        if (f32) ((float*)dweight)[c] = acc; else ((bf16*)dweight)[c] = __float2bfloat16_rn(acc);
    }
}

// ------------------------------------------------------------------------------------------------ host side
// The leading dimensions of a view as one row index: rows and the stride between them.  Throws when they do not collapse.
constexpr int64_t kMaxCols = (int64_t)1 << 30;                   // a step past the last column is still an int
struct Rows { int64_t rows, stride; };
Rows rows_of(const char* op, const char* name, const ormi_b200_view& v) {
    Rows r{1, 0};
    if (count_of(v) == 0) {                                       // the strides of an empty buffer say nothing
        for (int d = 0; d < v.ndim - 1; ++d) r.rows *= v.shape[d];
        return r;
    }
    bool first = true;
    for (int d = v.ndim - 2; d >= 0; --d) {
        if (v.shape[d] == 1) continue;
        if (first) { r.stride = v.strides[d]; first = false; }
        else OP_NEED(v.strides[d] == r.rows * r.stride, op, std::string(name) + ": the leading dimensions do not collapse into one row stride");
        r.rows *= v.shape[d];
    }
    return r;
}

void matrix_check(const char* op, const char* name, const ormi_b200_view& v, const ormi_b200_view& like, bool same_type) {
    view_check(op, name, v, 1, 4);
    auto n = [&] { return std::string(name); };
    OP_NEED(v.ndim == like.ndim, op, n() + " has another shape");
    for (int d = 0; d < v.ndim; ++d) OP_NEED(v.shape[d] == like.shape[d], op, n() + " has another shape");
    OP_NEED(v.shape[v.ndim - 1] <= 1 || v.strides[v.ndim - 1] == 1 || count_of(v) == 0, op, n() + ": the last dimension is not contiguous");
    if (same_type) OP_NEED(v.dtype == like.dtype, op, n() + " has another type");
    OP_NEED(v.dtype == ORMI_F32 || v.dtype == ORMI_BF16 || (!same_type && v.dtype == ORMI_E4M3), op, n() + " has a type that is not taken here");
    rows_of(op, name, v);
}

// An output's rows must not lie on one another.
void output_check(const char* op, const char* name, const ormi_b200_view& v) {
    const Rows r = rows_of(op, name, v);
    OP_NEED(r.rows <= 1 || count_of(v) == 0 || r.stride >= v.shape[v.ndim - 1], op, std::string(name) + ": its rows overlap");
}

void weight_check(const char* op, const char* name, const ormi_b200_view& v, int64_t cols) {
    view_check(op, name, v, 1, 1);
    OP_NEED(v.dtype == ORMI_F32 || v.dtype == ORMI_BF16, op, std::string(name) + " is F32 or BF16");
    OP_NEED(v.shape[0] == cols && (cols <= 1 || v.strides[0] == 1), op, std::string(name) + " is not [cols], contiguous");
}

void rstd_check(const char* op, const ormi_b200_view& v, int64_t rows) {
    view_check(op, "rstd", v, 1, 4);
    OP_NEED(v.dtype == ORMI_F32 && contiguous(v) && count_of(v) == rows, op, "rstd is not [rows] F32, contiguous");
}

void apart(const char* op, const char* out_name, const ormi_b200_view& out, const char* in_name, const ormi_b200_view& in, bool in_place) {
    if (!overlap(out, in) || (in_place && same_place(out, in))) return;
    throw Error(std::string("ormi_b200_") + op + ": " + out_name + " overlaps " + in_name);
}

// Whether 16-byte accesses (8- and 4-byte ones for narrower outputs) work on every row of a matrix.
bool rows_aligned(const void* p, int64_t row, int elem, int vec) {
    const int bytes = std::min(16, elem * vec);
    return !p || ((uintptr_t)p % bytes == 0 && row * elem % bytes == 0);
}

template <typename T, typename O, bool AL>
void launch_norm_row(ormi_b200_ctx* ctx, const NormParams& p) {
    constexpr int chunk = Piece<T, AL>::CHUNK;
    const int chunks = (p.cols + chunk - 1) / chunk;
    if (chunks <= 4) norm_row<T, O, AL, true><<<(int)((p.rows + 7) / 8), 256, 0, ctx->stream>>>(p);
    else norm_row<T, O, AL, false><<<(int)p.rows, (chunks + 3) / 4 * 32, 0, ctx->stream>>>(p);
}

template <typename T, typename O>
void launch_norm(ormi_b200_ctx* ctx, const NormParams& p) {
    constexpr int vec = 16 / sizeof(T);
    const bool al = p.cols % vec == 0 && rows_aligned(p.x, p.x_row, sizeof(T), vec) && rows_aligned(p.residual, p.residual_row, sizeof(T), vec) &&
                    rows_aligned(p.residual_out, p.residual_out_row, sizeof(T), vec) && rows_aligned(p.out, p.out_row, sizeof(O), vec) &&
                    rows_aligned(p.weight, 0, 4, 4);
    // 32 warps of four pieces hold a row of 16384 columns, 32768 where a piece is 8 bf16 values
    const int most = 128 * (al ? Piece<T, true>::CHUNK : Piece<T, false>::CHUNK);
    if (p.cols <= most && p.rows < 0x7fffffff) {
        if (al) launch_norm_row<T, O, true>(ctx, p); else launch_norm_row<T, O, false>(ctx, p);
    } else {
        norm_any<T, O><<<(int)std::min<int64_t>(p.rows, (int64_t)ctx->num_sms * 8), 256, 0, ctx->stream>>>(p);
    }
    ORMI_CUDA(cudaGetLastError());
    count_launch(ctx);
}

template <typename T, bool AL, int THREADS, int NV, int STAGES>
int launch_norm_back_row(ormi_b200_ctx* ctx, const NormBackParams& p, int threads, bool dry) {
    auto kernel = norm_back_row<T, AL, THREADS, NV, STAGES>;
    const int smem = back_sum_bytes(!THREADS, Piece<T, AL>::CHUNK) + (AL ? STAGES * back_stage_bytes(threads, NV) : 0);
    // the limit holds for the current device only, so it is set by every call
    if (smem) ORMI_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, back_sum_bytes(!THREADS, Piece<T, AL>::CHUNK) + (AL ? STAGES * back_stage_bytes(THREADS ? THREADS : 256, NV) : 0)));
    static std::atomic<int> per_sm[33];                        // by warps: asking costs more than a small launch
    int most = per_sm[threads / 32];
    if (!most) {
        int n = 0;
        ORMI_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem));
        per_sm[threads / 32] = most = std::max(1, n);
    }
    const int grid = (int)std::min<int64_t>(THREADS ? p.rows : (p.rows + 7) / 8, (int64_t)ctx->num_sms * most);
    if (!dry) kernel<<<grid, threads, smem, ctx->stream>>>(p);
    return grid;
}

template <typename T, bool AL>
int launch_norm_back_rows(ormi_b200_ctx* ctx, const NormBackParams& p, bool dry) {
    // One piece per thread up to 512 threads, so that the registers allow two blocks of them; a piece of 8 bf16 values takes
    // twice the registers of one of 4.  Three rows of copies per block, two where that would leave one block per SM.
    const int pieces = (p.cols + Piece<T, AL>::CHUNK - 1) / Piece<T, AL>::CHUNK, warps2 = (pieces + 1) / 2;
    if (pieces <= 2) return launch_norm_back_row<T, AL, 0, 2, 3>(ctx, p, 256, dry);
    if (pieces <= 16) return launch_norm_back_row<T, AL, 512, 1, 3>(ctx, p, pieces * 32, dry);
    if (warps2 <= 16) return launch_norm_back_row<T, AL, 512, 2, sizeof(T) == 4 ? 2 : 3>(ctx, p, warps2 * 32, dry);
    return launch_norm_back_row<T, AL, 1024, 2, 2>(ctx, p, warps2 * 32, dry);
}

template <typename T>
void launch_norm_back(ormi_b200_ctx* ctx, NormBackParams& p) {
    constexpr int vec = 16 / sizeof(T);
    const bool al = p.cols % vec == 0 && rows_aligned(p.dout, p.dout_row, sizeof(T), vec) && rows_aligned(p.s, p.s_row, sizeof(T), vec) &&
                    rows_aligned(p.dresidual, p.dresidual_row, sizeof(T), vec) && rows_aligned(p.dx, p.dx_row, sizeof(T), vec) && rows_aligned(p.weight, 0, 4, 4);
    // 32 warps of two pieces
    const bool in_registers = p.rows > 0 && p.cols <= 64 * (al ? Piece<T, true>::CHUNK : Piece<T, false>::CHUNK);
    if (in_registers) p.parts = al ? launch_norm_back_rows<T, true>(ctx, p, true) : launch_norm_back_rows<T, false>(ctx, p, true);
    else p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(256, p.rows / 64));
    Scratch partial(ctx, p.dweight ? (size_t)p.parts * p.cols * 4 : 0);
    p.partial = (float*)partial.ptr;
    if (in_registers) {
        if (al) launch_norm_back_rows<T, true>(ctx, p, false); else launch_norm_back_rows<T, false>(ctx, p, false);
        count_launch(ctx);
    } else {
        if (p.dweight) { norm_dweight_any<T><<<dim3((p.cols + 31) / 32, p.parts), 256, 0, ctx->stream>>>(p); count_launch(ctx); }
        if (p.rows) { norm_back_any<T><<<(int)std::min<int64_t>(p.rows, (int64_t)ctx->num_sms * 8), 256, 0, ctx->stream>>>(p); count_launch(ctx); }
    }
    if (p.dweight) {
        norm_dweight_join<<<(p.cols + 31) / 32, 1024, 0, ctx->stream>>>(p.partial, p.parts, p.cols, p.dweight, p.weight_f32);
        count_launch(ctx);
    }
    ORMI_CUDA(cudaGetLastError());
    partial.release();
}

}  // namespace

void rmsnorm_check(const ormi_b200_rmsnorm_args& a) {
    const char* op = "rmsnorm";
    matrix_check(op, "x", a.x, a.x, true);
    const int64_t cols = a.x.shape[a.x.ndim - 1], rows = rows_of(op, "x", a.x).rows;
    OP_NEED(cols >= 1, op, "x has no columns");
    OP_NEED(cols <= kMaxCols, op, "x has more than 2^30 columns");
    OP_NEED(a.eps >= 0.f, op, "eps is negative or not a number");
    if (a.residual.data) matrix_check(op, "residual", a.residual, a.x, true);
    if (a.residual_out.data) {
        matrix_check(op, "residual_out", a.residual_out, a.x, true);
        output_check(op, "residual_out", a.residual_out);
    }
    if (a.weight.data) weight_check(op, "weight", a.weight, cols);
    matrix_check(op, "out", a.out, a.x, false);
    output_check(op, "out", a.out);
    if (a.rstd.data) rstd_check(op, a.rstd, rows);
    OP_NEED((a.out.dtype == ORMI_E4M3) == (a.scales.data != nullptr), op, "scales go with an E4M3 out, and only with it");
    if (a.scales.data) {
        OP_NEED(a.group == 0 || a.group == 128, op, "group is 0 (one scale for a row) or 128");
        view_check(op, "scales", a.scales, 1, 4);
        const int64_t groups = a.group ? (cols + a.group - 1) / a.group : 1;
        OP_NEED(a.scales.dtype == ORMI_F32 && contiguous(a.scales) && count_of(a.scales) == rows * groups, op, "scales is not [rows, groups] F32, contiguous");
    }
    const struct { const char* name; const ormi_b200_view& v; } outs[] = {{"out", a.out}, {"residual_out", a.residual_out}, {"rstd", a.rstd}, {"scales", a.scales}};
    const struct { const char* name; const ormi_b200_view& v; } ins[] = {{"x", a.x}, {"residual", a.residual}, {"weight", a.weight}};
    for (int i = 0; i < 4; ++i) {
        for (auto& in : ins) apart(op, outs[i].name, outs[i].v, in.name, in.v, i < 2 && in.v.data != a.weight.data);
        for (int j = 0; j < i; ++j) apart(op, outs[i].name, outs[i].v, outs[j].name, outs[j].v, false);
    }
}

void rmsnorm(ormi_b200_ctx* ctx, const ormi_b200_rmsnorm_args& a) {
    const int64_t cols = a.x.shape[a.x.ndim - 1];
    const Rows x = rows_of("rmsnorm", "x", a.x);
    if (x.rows == 0) return;
    NormParams p{};
    p.x = a.x.data; p.residual = a.residual.data; p.weight = a.weight.data; p.out = a.out.data; p.residual_out = a.residual_out.data;
    p.rstd = (float*)a.rstd.data; p.scales = (float*)a.scales.data;
    p.x_row = x.stride;
    if (p.residual) p.residual_row = rows_of("rmsnorm", "residual", a.residual).stride;
    if (p.residual_out) p.residual_out_row = rows_of("rmsnorm", "residual_out", a.residual_out).stride;
    p.out_row = rows_of("rmsnorm", "out", a.out).stride;
    p.rows = x.rows; p.cols = (int)cols; p.group = a.group; p.eps = a.eps;
    p.groups = a.group ? (int)((cols + a.group - 1) / a.group) : 1;
    p.weight_f32 = a.weight.dtype == ORMI_F32;
    for (auto* v : {&a.out, &a.residual_out, &a.rstd, &a.scales}) written(ctx, *v);
    auto by_out = [&](auto t) {
        using T = decltype(t);
        if (a.out.dtype == ORMI_F32) launch_norm<T, float>(ctx, p);
        else if (a.out.dtype == ORMI_BF16) launch_norm<T, bf16>(ctx, p);
        else launch_norm<T, e4m3>(ctx, p);
    };
    if (a.x.dtype == ORMI_F32) by_out(float{}); else by_out(bf16{});
}

void rmsnorm_backward_check(const ormi_b200_rmsnorm_backward_args& a) {
    const char* op = "rmsnorm_backward";
    matrix_check(op, "dout", a.dout, a.dout, true);
    const int64_t cols = a.dout.shape[a.dout.ndim - 1], rows = rows_of(op, "dout", a.dout).rows;
    OP_NEED(cols >= 1, op, "dout has no columns");
    OP_NEED(cols <= kMaxCols, op, "dout has more than 2^30 columns");
    matrix_check(op, "s", a.s, a.dout, true);
    if (a.dresidual.data) matrix_check(op, "dresidual", a.dresidual, a.dout, true);
    matrix_check(op, "dx", a.dx, a.dout, true);
    output_check(op, "dx", a.dx);
    rstd_check(op, a.rstd, rows);
    if (a.weight.data) weight_check(op, "weight", a.weight, cols);
    if (a.dweight.data) {
        weight_check(op, "dweight", a.dweight, cols);
        if (a.weight.data) OP_NEED(a.dweight.dtype == a.weight.dtype, op, "dweight has another type than weight");
    }
    const struct { const char* name; const ormi_b200_view& v; } ins[] = {{"dout", a.dout}, {"s", a.s}, {"weight", a.weight}, {"rstd", a.rstd}, {"dresidual", a.dresidual}};
    for (int i = 0; i < 5; ++i) {
        apart(op, "dx", a.dx, ins[i].name, ins[i].v, i == 0 || i == 4);
        apart(op, "dweight", a.dweight, ins[i].name, ins[i].v, false);
    }
    apart(op, "dweight", a.dweight, "dx", a.dx, false);
}

void rmsnorm_backward(ormi_b200_ctx* ctx, const ormi_b200_rmsnorm_backward_args& a) {
    const Rows dout = rows_of("rmsnorm_backward", "dout", a.dout);
    NormBackParams p{};
    p.dout = a.dout.data; p.s = a.s.data; p.weight = a.weight.data; p.dresidual = a.dresidual.data;
    p.rstd = (const float*)a.rstd.data; p.dx = a.dx.data; p.dweight = a.dweight.data;
    p.dout_row = dout.stride;
    p.s_row = rows_of("rmsnorm_backward", "s", a.s).stride;
    if (p.dresidual) p.dresidual_row = rows_of("rmsnorm_backward", "dresidual", a.dresidual).stride;
    p.dx_row = rows_of("rmsnorm_backward", "dx", a.dx).stride;
    p.rows = dout.rows; p.cols = (int)a.dout.shape[a.dout.ndim - 1];
    p.weight_f32 = (a.weight.data ? a.weight.dtype : a.dweight.dtype) == ORMI_F32;
    written(ctx, a.dx);
    written(ctx, a.dweight);
    if (a.dout.dtype == ORMI_F32) launch_norm_back<float>(ctx, p); else launch_norm_back<bf16>(ctx, p);
}

}  // namespace ormi_b200
