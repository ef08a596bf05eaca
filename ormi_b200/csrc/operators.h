// Transformer-block operators on raw buffers: what their files share on the host side.
#pragma once
#include <cuda_runtime.h>

#include <string>

#include "context.h"
#include "ormi_b200.h"

namespace ormi_b200 {

// Argument checks (throw Error, touch no device) and launchers of the entry points in abi.cu.
void rmsnorm_check(const ormi_b200_rmsnorm_args& a);
void rmsnorm(ormi_b200_ctx* ctx, const ormi_b200_rmsnorm_args& a);
void rmsnorm_backward_check(const ormi_b200_rmsnorm_backward_args& a);
void rmsnorm_backward(ormi_b200_ctx* ctx, const ormi_b200_rmsnorm_backward_args& a);
void attention_check(const ormi_b200_attention_args& a);
void attention(ormi_b200_ctx* ctx, const ormi_b200_attention_args& a);
void attention_backward_check(const ormi_b200_attention_backward_args& a);
void attention_backward(ormi_b200_ctx* ctx, const ormi_b200_attention_backward_args& a);
void adamw_check(const ormi_b200_adamw_tensor* t, int n, const ormi_b200_adamw_config& c);
void adamw(ormi_b200_ctx* ctx, const ormi_b200_adamw_tensor* t, int n, const ormi_b200_adamw_config& c);

[[noreturn]] inline void op_fail(const char* op, const std::string& what) { throw Error(std::string("ormi_b200_") + op + ": " + what); }
// The text is only put together when the check fails: small calls are bound by the host.
#define OP_NEED(ok, op, what) do { if (!(ok)) op_fail(op, what); } while (0)

inline int dtype_bytes(int dtype) { return dtype == ORMI_F32 || dtype == ORMI_I32 ? 4 : dtype == ORMI_BF16 ? 2 : 1; }

// First and one-past-last byte that a view can touch (first == last: nothing).
struct Span { const char* lo; const char* hi; };
inline Span span_of(const ormi_b200_view& v) {
    int64_t last = 0;
    for (int d = 0; d < v.ndim; ++d) {
        if (v.shape[d] == 0) return {(const char*)v.data, (const char*)v.data};
        last += (v.shape[d] - 1) * v.strides[d];
    }
    return {(const char*)v.data, (const char*)v.data + (last + 1) * dtype_bytes(v.dtype)};
}
inline bool overlap(const ormi_b200_view& a, const ormi_b200_view& b) {
    if (!a.data || !b.data) return false;
    const Span x = span_of(a), y = span_of(b);
    return x.lo < x.hi && y.lo < y.hi && x.lo < y.hi && y.lo < x.hi;
}
inline bool same_place(const ormi_b200_view& a, const ormi_b200_view& b) {
    if (a.data != b.data || a.dtype != b.dtype || a.ndim != b.ndim) return false;
    for (int d = 0; d < a.ndim; ++d)
        if (a.shape[d] != b.shape[d] || (a.shape[d] > 1 && a.strides[d] != b.strides[d])) return false;
    return true;
}

// The checks every view goes through: rank, extents, alignment to the element, and that neither the number of elements (2^48,
// repeated ones included) nor the way to the last one (2^56 elements) comes near 63 bits.
inline void view_check(const char* op, const char* name, const ormi_b200_view& v, int lo_rank, int hi_rank) {
    auto n = [&] { return std::string(name); };
    OP_NEED(v.ndim >= 1 && v.ndim <= 4, op, v.data ? n() + " has " + std::to_string(v.ndim) + " dimensions" : n() + " is missing");
    int64_t count = 1;
    for (int d = 0; d < v.ndim; ++d) count *= v.shape[d] != 0;
    OP_NEED(v.data || !count, op, n() + " is missing");              // nothing at no address is an empty buffer
    OP_NEED(v.dtype >= ORMI_F32 && v.dtype <= ORMI_I32, op, n() + " has an unknown type");
    OP_NEED(v.ndim >= lo_rank && v.ndim <= hi_rank, op, n() + " has " + std::to_string(v.ndim) + " dimensions, " +
            (lo_rank == hi_rank ? std::to_string(lo_rank) : std::to_string(lo_rank) + " to " + std::to_string(hi_rank)) + " wanted");
    for (int d = 0; d < v.ndim; ++d) {
        OP_NEED(v.shape[d] >= 0 && v.shape[d] < (int64_t)1 << 31, op, n() + " has an extent below zero or above 2^31 - 1");
        OP_NEED(v.strides[d] >= 0 && v.strides[d] < (int64_t)1 << 40, op, n() + " has a stride below zero or above 2^40");
    }
    double elements = 1, last = 0;
    for (int d = 0; d < v.ndim; ++d) { elements *= (double)v.shape[d]; last += (double)v.shape[d] * (double)v.strides[d]; }
    OP_NEED(elements <= 0x1p48 && (elements == 0 || last <= 0x1p56), op, n() + " is too large");
    OP_NEED((uintptr_t)v.data % dtype_bytes(v.dtype) == 0, op, n() + " does not start on a whole element");
}
inline int64_t count_of(const ormi_b200_view& v) {
    int64_t n = 1;
    for (int d = 0; d < v.ndim; ++d) n *= v.shape[d];
    return n;
}
inline bool contiguous(const ormi_b200_view& v) {
    if (count_of(v) == 0) return true;                            // the strides of an empty buffer say nothing
    int64_t want = 1;
    for (int d = v.ndim - 1; d >= 0; --d) {
        if (v.shape[d] != 1 && v.strides[d] != want) return false;
        want *= v.shape[d];
    }
    return true;
}

// Scratch of one call from the context's pool, given back when the launches are queued (the pool is ordered by the
// stream).  The pool caches by exact size: sizes are rounded up to a power of two so that lengths that change from call
// to call share blocks.
struct Scratch {
    ormi_b200_ctx* ctx;
    void* ptr = nullptr;
    size_t bytes = 0;
    Scratch(ormi_b200_ctx* c, size_t want) : ctx(c) {
        if (!want) return;
        bytes = 1 << 16;
        while (bytes < want) bytes <<= 1;
        ptr = pool_alloc(ctx, bytes);
    }
    Scratch(const Scratch&) = delete;
    // the normal end: an overwritten guard zone is reported
    void release() { void* p = ptr; ptr = nullptr; if (p) pool_free(ctx, p, bytes); }
    ~Scratch() { try { release(); } catch (...) {} }
};

inline void written(ormi_b200_ctx* ctx, const ormi_b200_view& v) {
    if (!v.data) return;
    const Span s = span_of(v);
    written(ctx, s.lo, (size_t)(s.hi - s.lo));
}

inline void count_launch(ormi_b200_ctx* ctx, int n = 1) { ctx->counters["launches"] += n; }

}  // namespace ormi_b200
