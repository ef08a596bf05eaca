// Root-mean-square norm with the residual's addition, forward and backward.
//
//   forward    s = x + r;  rstd = (mean(s^2) + eps)^-1/2;  y = s * rstd * w;   optionally y as e4m3 codes with scales
//   backward   c = mean(dy w s) * rstd^2;   dx = rstd * (dy w - s c) + ds;   dw = sum over rows of dy s rstd
//
// Both are bound by memory: every element is read and written once and takes a handful of operations.
#include <algorithm>

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

// One block per row, any width, any alignment: three passes over the row (four with one scale for the row), the second
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
            const float up = top > 0.f ? 448.f * (1.f / top) : 0.f;
            if (threadIdx.x == 0) p.scales[row] = top * (1.f / 448.f);
            for (int c = threadIdx.x; c < p.cols; c += blockDim.x) out[c] = from_f32<O>(y(c) * up);
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
                const float up = top > 0.f ? 448.f * (1.f / top) : 0.f;
                if (lane == 0) p.scales[row * p.groups + g] = top * (1.f / 448.f);
                for (int k = 0; k < 4; ++k) {
                    const int c = g * 128 + k * 32 + lane;
                    if (c < p.cols) out[c] = from_f32<O>(v[k] * up);
                }
            }
        }
        __syncthreads();
    }
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
        else op_need(v.strides[d] == r.rows * r.stride, op, std::string(name) + ": the leading dimensions do not collapse into one row stride");
        r.rows *= v.shape[d];
    }
    return r;
}

void matrix_check(const char* op, const char* name, const ormi_b200_view& v, const ormi_b200_view& like, bool same_type) {
    view_check(op, name, v, 1, 4);
    const std::string n(name);
    op_need(v.ndim == like.ndim, op, n + " has another shape");
    for (int d = 0; d < v.ndim; ++d) op_need(v.shape[d] == like.shape[d], op, n + " has another shape");
    op_need(v.shape[v.ndim - 1] <= 1 || v.strides[v.ndim - 1] == 1 || count_of(v) == 0, op, n + ": the last dimension is not contiguous");
    if (same_type) op_need(v.dtype == like.dtype, op, n + " has another type");
    op_need(v.dtype == ORMI_F32 || v.dtype == ORMI_BF16 || (!same_type && v.dtype == ORMI_E4M3), op, n + " has a type that is not taken here");
    rows_of(op, name, v);
}

// An output's rows must not lie on one another.
void output_check(const char* op, const char* name, const ormi_b200_view& v) {
    const Rows r = rows_of(op, name, v);
    op_need(r.rows <= 1 || count_of(v) == 0 || r.stride >= v.shape[v.ndim - 1], op, std::string(name) + ": its rows overlap");
}

void weight_check(const char* op, const char* name, const ormi_b200_view& v, int64_t cols) {
    view_check(op, name, v, 1, 1);
    op_need(v.dtype == ORMI_F32 || v.dtype == ORMI_BF16, op, std::string(name) + " is F32 or BF16");
    op_need(v.shape[0] == cols && (cols <= 1 || v.strides[0] == 1), op, std::string(name) + " is not [cols], contiguous");
}

void rstd_check(const char* op, const ormi_b200_view& v, int64_t rows) {
    view_check(op, "rstd", v, 1, 4);
    op_need(v.dtype == ORMI_F32 && contiguous(v) && count_of(v) == rows, op, "rstd is not [rows] F32, contiguous");
}

void apart(const char* op, const char* out_name, const ormi_b200_view& out, const char* in_name, const ormi_b200_view& in, bool in_place) {
    if (!overlap(out, in) || (in_place && same_place(out, in))) return;
    throw Error(std::string("ormi_b200_") + op + ": " + out_name + " overlaps " + in_name);
}

template <typename T, typename O>
void launch_norm(ormi_b200_ctx* ctx, const NormParams& p) {
    const int grid = (int)std::min<int64_t>(p.rows, (int64_t)ctx->num_sms * 8);
    norm_any<T, O><<<grid, 256, 0, ctx->stream>>>(p);
    ORMI_CUDA(cudaGetLastError());
    count_launch(ctx);
}

template <typename T>
void launch_norm_back(ormi_b200_ctx* ctx, NormBackParams& p) {
    Scratch partial(ctx, p.dweight ? (size_t)256 * p.cols * 4 : 0);
    if (p.dweight) {
        p.partial = (float*)partial.ptr;
        p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(256, p.rows / 64));
        norm_dweight_any<T><<<dim3((p.cols + 31) / 32, p.parts), 256, 0, ctx->stream>>>(p);
        norm_dweight_join<<<(p.cols + 31) / 32, 1024, 0, ctx->stream>>>(p.partial, p.parts, p.cols, p.dweight, p.weight_f32);
        count_launch(ctx, 2);
    }
    if (p.rows) {
        const int grid = (int)std::min<int64_t>(p.rows, (int64_t)ctx->num_sms * 8);
        norm_back_any<T><<<grid, 256, 0, ctx->stream>>>(p);
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
    op_need(cols >= 1, op, "x has no columns");
    op_need(a.eps >= 0.f, op, "eps is negative or not a number");
    if (a.residual.data) matrix_check(op, "residual", a.residual, a.x, true);
    if (a.residual_out.data) {
        matrix_check(op, "residual_out", a.residual_out, a.x, true);
        output_check(op, "residual_out", a.residual_out);
    }
    if (a.weight.data) weight_check(op, "weight", a.weight, cols);
    matrix_check(op, "out", a.out, a.x, false);
    output_check(op, "out", a.out);
    if (a.rstd.data) rstd_check(op, a.rstd, rows);
    op_need((a.out.dtype == ORMI_E4M3) == (a.scales.data != nullptr), op, "scales go with an E4M3 out, and only with it");
    if (a.scales.data) {
        op_need(a.group == 0 || a.group == 128, op, "group is 0 (one scale for a row) or 128");
        view_check(op, "scales", a.scales, 1, 4);
        const int64_t groups = a.group ? (cols + a.group - 1) / a.group : 1;
        op_need(a.scales.dtype == ORMI_F32 && contiguous(a.scales) && count_of(a.scales) == rows * groups, op, "scales is not [rows, groups] F32, contiguous");
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
    op_need(cols >= 1, op, "dout has no columns");
    matrix_check(op, "s", a.s, a.dout, true);
    if (a.dresidual.data) matrix_check(op, "dresidual", a.dresidual, a.dout, true);
    matrix_check(op, "dx", a.dx, a.dout, true);
    output_check(op, "dx", a.dx);
    rstd_check(op, a.rstd, rows);
    if (a.weight.data) weight_check(op, "weight", a.weight, cols);
    if (a.dweight.data) {
        weight_check(op, "dweight", a.dweight, cols);
        if (a.weight.data) op_need(a.dweight.dtype == a.weight.dtype, op, "dweight has another type than weight");
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
