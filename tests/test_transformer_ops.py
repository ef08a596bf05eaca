"""RMS norm with residual, masked attention and many-tensor AdamW through ormi_b200.ops: refusals on the CPU, numerics on the
GPU against plain 64-bit evaluations with elementwise bounds (tests/block_reference.py)."""
import ctypes
import math
import os
import types

import numpy as np
import pytest

from ormi_b200 import graph as G
from ormi_b200 import ops
from ormi_b200._lib import BackendError, lib, check

V = ops.view
NODEV = types.SimpleNamespace(index=0, handle=None)


# ------------------------------------------------------------------------------------------------ refusals (no GPU)

def refused(call, *words):
    with pytest.raises((BackendError, ValueError, TypeError)) as e:
        call()
    assert any(w in str(e.value) for w in words), str(e.value)


def accepted(call):
    """Arguments are checked before the context: a good call fails on the missing context only."""
    with pytest.raises(BackendError) as e:
        call()
    assert "ctx is NULL" in str(e.value), str(e.value)


def norm_args(**change):
    a = dict(x=V(0x1000, (4, 64), "bf16"), weight=V(0x4000, (64,)), out=V(0x8000, (4, 64), "bf16"))
    a.update(change)
    return lambda: ops.rmsnorm(NODEV, a.pop("x"), a.pop("weight"), a.pop("out"), **a)


def test_norm_accepts_what_is_documented():
    accepted(norm_args())
    accepted(norm_args(weight=None))
    accepted(norm_args(out=V(0x1000, (4, 64), "bf16")))                                       # in place
    accepted(norm_args(residual=V(0x2000, (4, 64), "bf16"), residual_out=V(0x2000, (4, 64), "bf16")))
    accepted(norm_args(x=V(0x1000, (2, 2, 64), "bf16"), out=V(0x8000, (2, 2, 64), "bf16")))
    accepted(norm_args(x=V(0x1000, (4, 64), "bf16", (0, 1))))                                 # one row for all: an input may repeat
    accepted(norm_args(out=V(0x8000, (4, 64), "e4m3"), scales=V(0x9000, (4, 1)), group=128))
    accepted(norm_args(x=V(0, (0, 64), "bf16"), out=V(0, (0, 64), "bf16")))


@pytest.mark.parametrize("words, change", [
    ("another shape", dict(out=V(0x8000, (4, 63), "bf16"))),
    ("another type", dict(residual=V(0x2000, (4, 64)))),
    ("not contiguous", dict(x=V(0x1000, (4, 64), "bf16", (128, 2)))),
    ("do not collapse", dict(x=V(0x1000, (2, 2, 64), "bf16", (64, 200, 1)), out=V(0x8000, (2, 2, 64), "bf16"))),
    ("rows overlap", dict(out=V(0x8000, (4, 64), "bf16", (32, 1)))),
    ("type that is not taken", dict(x=V(0x1000, (4, 64), "i32"), out=V(0x8000, (4, 64), "i32"))),
    ("weight", dict(weight=V(0x4000, (63,)))),
    ("scales", dict(out=V(0x8000, (4, 64), "e4m3"))),
    ("scales", dict(scales=V(0x9000, (4,)))),
    ("scales", dict(out=V(0x8000, (4, 64), "e4m3"), scales=V(0x9000, (4, 2)), group=128)),
    ("group", dict(out=V(0x8000, (4, 64), "e4m3"), scales=V(0x9000, (4, 1)), group=64)),
    ("overlaps x", dict(out=V(0x1002, (4, 64), "bf16"))),
    ("overlaps weight", dict(rstd=V(0x4000, (4,)))),
    ("overlaps out", dict(rstd=V(0x8000, (4,)))),
    ("overlaps out", dict(residual=V(0x1000, (4, 64), "bf16"), out=V(0x1000, (4, 64), "bf16"), residual_out=V(0x1000, (4, 64), "bf16"))),
    ("rstd", dict(rstd=V(0x9000, (5,)))),
    ("eps", dict(eps=-1.0)),
    ("eps", dict(eps=float("nan"))),
    ("missing", dict(out=None)),
    ("whole element", dict(x=V(0x1001, (4, 64), "bf16"))),
    ("stride below zero", dict(x=V(0x1000, (4, 64), "bf16", (-64, 1)))),
    ("no columns", dict(x=V(0x1000, (4, 0), "bf16"), out=V(0x8000, (4, 0), "bf16"))),
])
def test_norm_refuses(words, change):
    refused(norm_args(**change), words)


def norm_back(**change):
    a = dict(dout=V(0x1000, (4, 64), "bf16"), s=V(0x2000, (4, 64), "bf16"), weight=V(0x3000, (64,)), rstd=V(0x4000, (4,)), dx=V(0x5000, (4, 64), "bf16"), dweight=V(0x6000, (64,)))
    a.update(change)
    return lambda: ops.rmsnorm_backward(NODEV, a.pop("dout"), a.pop("s"), a.pop("weight"), a.pop("rstd"), a.pop("dx"), a.pop("dweight"), **a)


def test_norm_backward_arguments():
    accepted(norm_back())
    accepted(norm_back(dx=V(0x1000, (4, 64), "bf16")))
    accepted(norm_back(dweight=None))
    accepted(norm_back(weight=None, dweight=V(0x6000, (64,), "bf16")))
    refused(norm_back(dx=V(0x2000, (4, 64), "bf16")), "dx overlaps s")
    refused(norm_back(dweight=V(0x6000, (64,), "bf16")), "another type than weight")
    refused(norm_back(dresidual=V(0x7000, (4, 64))), "another type")
    refused(norm_back(rstd=None), "rstd is missing")
    refused(norm_back(dweight=V(0x5000, (64,))), "overlaps dx")


def attn_args(b=2, nq=16, nk=16, h=4, hk=2, d=32, t="bf16", **change):
    a = dict(q=V(0x100000, (b, nq, h, d), t), k=V(0x200000, (b, nk, hk, d), t), v=V(0x300000, (b, nk, hk, d), t), out=V(0x400000, (b, nq, h, d), t))
    a.update(change)
    return lambda: ops.attention(NODEV, a.pop("q"), a.pop("k"), a.pop("v"), a.pop("out"), **a)


def test_attention_accepts_what_is_documented():
    accepted(attn_args())
    accepted(attn_args(t="f32", d=256))
    accepted(attn_args(nq=0))
    accepted(attn_args(prefix=V(0x500000, (2,), "i32")))
    accepted(attn_args(nk=0, k=V(0, (2, 0, 2, 32), "bf16"), v=V(0, (2, 0, 2, 32), "bf16")))
    accepted(attn_args(k=V(0x200000, (2, 16, 2, 32), "bf16", (0, 32, 512, 1))))
    accepted(attn_args(causal=True, prefix=V(0x500000, (2,), "i32"), key_len=V(0x500100, (2,), "i32"), q_start=V(0x500200, (2,), "i32"),
                       q_docs=V(0x600000, (2, 16), "i32"), k_docs=V(0x600000, (2, 16), "i32"), slopes=V(0x700000, (4,)), cap=30.0, lse=V(0x800000, (2, 4, 16))))


@pytest.mark.parametrize("words, change", [
    ("head_dim is 1 to 256", dict(d=257)),
    ("above 2^30", dict(nk=(1 << 30) + 1)),
    ("above 2^30", dict(b=1, nq=1 << 29)),
    ("multiple of kv_heads", dict(h=3)),
    ("another type", dict(k=V(0x200000, (2, 16, 2, 32), "f32"))),
    ("another batch", dict(k=V(0x200000, (3, 16, 2, 32), "bf16"), v=V(0x300000, (3, 16, 2, 32), "bf16"))),
    ("another shape", dict(v=V(0x300000, (2, 15, 2, 32), "bf16"))),
    ("not contiguous", dict(q=V(0x100000, (2, 16, 4, 32), "bf16", (4096, 256, 64, 2)))),
    ("F32 or BF16", dict(t="e4m3")),
    ("4 wanted", dict(q=V(0x100000, (16, 4, 32), "bf16"))),
    ("rows overlap", dict(out=V(0x400000, (2, 16, 4, 32), "bf16", (0, 128, 32, 1)))),
    ("lse", dict(lse=V(0x800000, (2, 16, 4)))),
    ("slopes", dict(slopes=V(0x700000, (2,)))),
    ("go together", dict(q_docs=V(0x600000, (2, 16), "i32"))),
    ("k_docs", dict(q_docs=V(0x600000, (2, 16), "i32"), k_docs=V(0x600000, (2, 17), "i32"))),
    ("key_len", dict(key_len=V(0x500000, (2,), "f32"))),
    ("key_len", dict(key_len=V(0x500000, (4,), "i32", (2,)))),
    ("scale is not finite", dict(scale=float("inf"))),
    ("cap", dict(cap=-1.0)),
    ("out overlaps q", dict(out=V(0x100000, (2, 16, 4, 32), "bf16"))),
    ("lse overlaps key_len", dict(lse=V(0x800000, (2, 4, 16)), key_len=V(0x800000, (2,), "i32"))),
    ("missing", dict(v=None)),
])
def test_attention_refuses(words, change):
    refused(attn_args(**change), words)


def attn_back(**change):
    t = "bf16"
    a = dict(dout=V(0x10000, (2, 16, 4, 32), t), q=V(0x20000, (2, 16, 4, 32), t), k=V(0x30000, (2, 16, 2, 32), t), v=V(0x40000, (2, 16, 2, 32), t),
             out=V(0x50000, (2, 16, 4, 32), t), lse=V(0x60000, (2, 4, 16)), dq=V(0x70000, (2, 16, 4, 32), t), dk=V(0x80000, (2, 16, 2, 32), t), dv=V(0x90000, (2, 16, 2, 32), t))
    a.update(change)
    names = ("dout", "q", "k", "v", "out", "lse", "dq", "dk", "dv")
    return lambda: ops.attention_backward(NODEV, *(a.pop(n) for n in names), **a)


def test_attention_backward_arguments():
    accepted(attn_back())
    joint = lambda first, n: V(0x70000 + first * 64, (2, 16, n, 32), "bf16", (16 * 8 * 32, 8 * 32, 32, 1))      # noqa: E731
    accepted(attn_back(dq=joint(0, 4), dk=joint(4, 2), dv=joint(6, 2)))                   # slices of one gradient
    refused(attn_back(lse=None), "lse")
    refused(attn_back(dk=V(0x30000, (2, 16, 2, 32), "bf16")), "dk overlaps k")
    refused(attn_back(dv=V(0x80000, (2, 16, 2, 32), "bf16")), "dv overlaps dk")
    refused(attn_back(dq=joint(0, 4), dk=joint(3, 2), dv=joint(6, 2)), "dk overlaps dq")
    refused(attn_back(dq=joint(0, 4), dk=joint(4, 2), dv=joint(7, 2)), "dv overlaps dq")          # runs into the next position
    heads_first = lambda first, n: V(0x70000 + first * 16 * 64, (2, 16, n, 32), "bf16", (8 * 16 * 32, 32, 16 * 32, 1))      # noqa: E731
    accepted(attn_back(dq=heads_first(0, 4), dk=heads_first(4, 2), dv=heads_first(6, 2)))
    refused(attn_back(dq=heads_first(0, 4), dk=heads_first(4, 2), dv=heads_first(5, 2)), "dv overlaps dk")
    refused(attn_back(dq=V(0x70000, (2, 16, 2, 32), "bf16")), "another shape")
    refused(attn_back(dk=V(0x80000, (2, 16, 2, 32), "bf16", (1024, 64, 0, 1))), "rows overlap")


def adam(states=32, **change):
    s = "f32" if states == 32 else "e4m3"
    a = dict(params=[V(0x10000, (10, 30))], grads=[V(0x20000, (300,), "bf16")], m=[V(0x30000, (300,), s)], v=[V(0x40000, (300,), s)])
    if states == 8:
        a.update(m_scales=[V(0x50000, (3,))], v_scales=[V(0x60000, (3,))])
    step = dict(lr=1e-3)
    for k in list(change):
        if k in ("step", "lr", "device_step", "grad_scale"):
            step[k] = change.pop(k)
    a.update(change)
    return lambda: ops.AdamW(NODEV, a.pop("params"), a.pop("grads"), a.pop("m"), a.pop("v"), **a).step(**step)


def test_adamw_arguments():
    accepted(adam())
    accepted(adam(8))
    accepted(adam(device_step=0x8000))
    accepted(adam(copies=[V(0x70000, (300,), "bf16")]))
    accepted(adam(params=[], grads=[], m=[], v=[]))
    refused(adam(step=0), "counts from 1")
    refused(adam(betas=(1.0, 0.9)), "beta")
    refused(adam(eps=-1.0), "eps")
    refused(adam(lr=float("nan")), "lr")
    refused(adam(weight_decay=[1.0, 2.0]), "one buffer for each")
    refused(adam(weight_decay=float("inf")), "weight_decay")
    refused(adam(m=[V(0x30000, (299,))]), "299 elements")
    refused(adam(m=[V(0x10000, (300,))]), "overlaps")
    refused(adam(m=[V(0x30000, (300,), "bf16")]), "another type")
    refused(adam(params=[V(0x10000, (10, 30), "f32", (60, 1))]), "not contiguous")
    refused(adam(8, m_scales=[V(0x50000, (2,))]), "2 elements")
    refused(adam(8, v_scales=None), "m_scales", "elements")
    refused(adam(params=[V(0x10000, (300,))] * 2, grads=[V(0x20000, (300,))] * 2, m=[V(0x30000, (300,))] * 2, v=[V(0x40000, (300,))] * 2), "overlaps")
    refused(adam(device_step=0x8004), "whole element")


def test_device_arrays_convert_to_and_from_bf16_and_e4m3_like_torch():
    torch = pytest.importorskip("torch")
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(codes, ops._E4M3_VALUES, equal_nan=True)


# ------------------------------------------------------------------------------------------------ numerics (GPU)

torch = pytest.importorskip("torch")
from block_reference import ACC, F8, HALF, Attention, close, mix32  # noqa: E402

gpu = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float32


def randn(*shape, dtype=FP, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7919 * len(shape) + sum(shape))
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def done(dev):
    dev.sync()


# ---- RMS norm

@gpu
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 7), (5, 64), (2, 128), (33, 129), (4, 1000), (7, 1111), (3, 2048), (2, 4096), (300, 520), (1, 8200), (2, 20001), (2, 40000), (1, 70000)])
@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_forward(device, rows, cols, dtype, residual):
    x, w = randn(rows, cols, dtype=dtype), randn(cols, dtype=dtype, seed=1)
    r = randn(rows, cols, dtype=dtype, seed=2, scale=3.0) if residual else None
    out, s, rstd = torch.empty_like(x), torch.empty_like(x), torch.empty(rows, device="cuda")
    torch.cuda.synchronize()
    ops.rmsnorm(device, x, w, out, residual=r, residual_out=s, rstd=rstd, eps=1e-5)
    done(device)
    stream = (x.to(FP) + r.to(FP)).to(dtype) if residual else x
    assert torch.equal(s, stream)
    want = 1 / torch.sqrt(stream.to(F8).square().mean(1) + 1e-5)
    near = (cols + 8) * 2.0 ** -24
    close("rstd", rstd, want, near * want)
    y = stream.to(F8) * want[:, None] * w.to(F8)
    close("out", out, y, (HALF[dtype] + near + 2.0 ** -22) * 1.01 * y.abs())


@gpu
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 100), (5, 128), (2, 300), (3, 1111), (4, 4096), (2, 40000)])
@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("group", [0, 128])
def test_norm_to_eight_bits(device, rows, cols, dtype, group):
    x, w = randn(rows, cols, dtype=dtype), randn(cols, dtype=FP, seed=1)
    x[0, : cols // 2] = 0
    groups = -(-cols // 128) if group else 1
    out, scales = torch.empty(rows, cols, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(rows, groups, device="cuda")
    torch.cuda.synchronize()
    ops.rmsnorm(device, x, w, out, scales=scales, group=group, eps=1e-5)
    done(device)
    y = x.to(F8) / torch.sqrt(x.to(F8).square().mean(1, keepdim=True) + 1e-5) * w.to(F8)
    near = (cols + 16) * 2.0 ** -24 + 2.0 ** -21
    width = group or cols
    parts = torch.nn.functional.pad(y, (0, groups * width - cols)).view(rows, groups, width)
    close("scales", scales, parts.abs().amax(2) / 448, near * parts.abs().amax(2) / 448)
    step = scales.to(F8).repeat_interleave(width, 1)[:, :cols]
    # half a step of e4m3: 2^-4 of the value, or half of 2^-9 in units of the scale
    close("values", out.to(F8) * step, y, 1.01 * (2.0 ** -4 + near) * y.abs() + 1.01 * 2.0 ** -10 * step)


@gpu
def test_norm_strided_rows_in_place_and_three_dimensions(device):
    base = randn(6, 5, 96, dtype=BF)
    x = base[:, :, :64]                                              # rows 96 apart
    res = randn(6, 5, 64, dtype=BF, seed=3)
    stream = (x.to(FP) + res.to(FP)).to(BF)
    keep = base[:, :, 64:].clone()
    w = randn(64, dtype=BF, seed=4)
    out = torch.empty(6, 5, 64, device="cuda", dtype=FP)
    torch.cuda.synchronize()
    ops.rmsnorm(device, x, w, out, residual=res, residual_out=x)
    done(device)
    assert torch.equal(x, stream) and torch.equal(base[:, :, 64:], keep)
    y = stream.to(F8) / torch.sqrt(stream.to(F8).square().mean(-1, keepdim=True) + 1e-6) * w.to(F8)
    close("out", out, y, 2.0 ** -17 * y.abs())
    again = x.clone()
    torch.cuda.synchronize()
    ops.rmsnorm(device, again, None, again)
    done(device)
    y = stream.to(F8) / torch.sqrt(stream.to(F8).square().mean(-1, keepdim=True) + 1e-6)
    close("in place", again, y, 1.02 * 2.0 ** -8 * y.abs())


@gpu
def test_norm_keeps_what_is_not_finite_in_its_row(device):
    for cols in (64, 1111):
        x = randn(4, cols, dtype=BF)
        x[1, 3], x[2, 5] = float("nan"), float("inf")
        out = torch.empty_like(x)
        o8, sc = torch.empty(4, cols, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(4, 1, device="cuda")
        torch.cuda.synchronize()
        ops.rmsnorm(device, x, None, out)
        ops.rmsnorm(device, x, None, o8, scales=sc)
        done(device)
        assert bool(out[[0, 3]].isfinite().all()) and bool(out[1].isnan().all()) and bool(out[2, 5].isnan())
        assert bool(sc[[0, 3]].isfinite().all()) and bool(sc[1].isnan())


@gpu
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 7), (65, 64), (2, 129), (130, 1000), (70, 1111), (700, 2048), (3, 4096), (1000, 520), (2, 20001), (129, 33000), (0, 64)])
@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("skip", [False, True])
def test_norm_backward(device, rows, cols, dtype, skip):
    s, dy, w = randn(rows, cols, dtype=dtype, scale=2.0), randn(rows, cols, dtype=dtype, seed=1), randn(cols, dtype=dtype, seed=2)
    ds = randn(rows, cols, dtype=dtype, seed=3) if skip else None
    rstd = torch.rsqrt(s.float().square().mean(1) + 1e-5)
    dx, dw = torch.empty_like(s), torch.full_like(w, 9.0)
    torch.cuda.synchronize()
    ops.rmsnorm_backward(device, dy, s, w, rstd, dx, dw, dresidual=ds)
    done(device)
    x, g, inv = s.to(F8), dy.to(F8), rstd.to(F8)[:, None]
    gw = g * w.to(F8)
    c = (gw * x).mean(1, keepdim=True) * inv * inv if cols else 0
    want = inv * (gw - x * c) + (ds.to(F8) if skip else 0)
    size = inv * (gw.abs() + x.abs() * (gw * x).abs().mean(1, keepdim=True) * inv * inv) + (ds.to(F8).abs() if skip else 0)
    close("dx", dx, want, 1.01 * (HALF[dtype] * want.abs() + (cols + 16) * 2.0 ** -24 * size))
    want, size = (g * x * inv).sum(0), (g * x * inv).abs().sum(0)
    close("dweight", dw, want, 1.01 * (HALF[dtype] * want.abs() + (rows + 16) * 2.0 ** -24 * size))


@gpu
def test_norm_backward_agrees_with_differences(device):
    rows, cols = 3, 40
    s, dy, w = (randn(rows, cols, seed=1), randn(rows, cols, seed=2), randn(cols, seed=3))
    rstd = torch.rsqrt(s.square().mean(1) + 1e-5)
    dx, dw = torch.empty_like(s), torch.empty_like(w)
    torch.cuda.synchronize()
    ops.rmsnorm_backward(device, dy, s, w, rstd, dx, dw)
    done(device)

    def loss(x, w):
        return (x / torch.sqrt(x.square().mean(1, keepdim=True) + 1e-5) * w * dy.to(F8)).sum()
    h = 1e-5
    for i, j in ((0, 0), (1, 17), (2, 39)):
        e = torch.zeros_like(s, dtype=F8)
        e[i, j] = h
        slope = (loss(s.to(F8) + e, w.to(F8)) - loss(s.to(F8) - e, w.to(F8))) / (2 * h)
        assert abs(float(slope - dx[i, j])) < 1e-5
        slope = (loss(s.to(F8), w.to(F8) + e[i]) - loss(s.to(F8), w.to(F8) - e[i])) / (2 * h)
        assert abs(float(slope - dw[j])) < 1e-4


@gpu
def test_norm_backward_without_weight_in_place(device):
    s, dy = randn(50, 256, dtype=BF), randn(50, 256, dtype=BF, seed=1)
    rstd = torch.rsqrt(s.float().square().mean(1) + 1e-6)
    apart = torch.empty_like(s)
    dw = torch.empty(256, device="cuda")
    torch.cuda.synchronize()
    ops.rmsnorm_backward(device, dy, s, None, rstd, apart, dw)
    ops.rmsnorm_backward(device, dy, s, None, rstd, dy)
    done(device)
    assert torch.equal(apart, dy)


# ---- attention

def run_attention(device, q, k, v, back=True, layout=None, **masks):
    b, nq, h, d = q.shape
    out, lse = torch.full_like(q, 7.0, memory_format=torch.contiguous_format), torch.full((b, h, nq), 7.0, device="cuda")
    torch.cuda.synchronize()
    ops.attention(device, q, k, v, out, lse, **masks)
    done(device)
    ref = Attention(q, k, v, **masks)
    want, bound, want_lse, lse_bound = ref.forward()
    close("out", out, want, bound)
    close("lse", lse, want_lse, lse_bound)
    if back:
        dout = randn(b, nq, h, d, dtype=q.dtype, seed=11)
        dq, dk, dv = (torch.full_like(x, 5.0, memory_format=torch.contiguous_format) for x in (q, k, v))
        torch.cuda.synchronize()
        ops.attention_backward(device, dout, q, k, v, out, lse, dq, dk, dv, **masks)
        done(device)
        for (name, (want, bound)), got in zip(ref.backward(dout, out, lse).items(), (dq, dk, dv)):
            close(name, got, want, bound)
    return out, lse


def qkv(b, nq, nk, h, hk, d, dtype, scale=1.0):
    return randn(b, nq, h, d, dtype=dtype, seed=1, scale=scale), randn(b, nk, hk, d, dtype=dtype, seed=2), randn(b, nk, hk, d, dtype=dtype, seed=3)


@gpu
@pytest.mark.parametrize("d", [1, 8, 24, 64, 72, 100, 128, 136, 256])
@pytest.mark.parametrize("dtype", [FP, BF])
def test_attention_head_sizes(device, d, dtype):
    run_attention(device, *qkv(2, 150, 150, 4, 2, d, dtype), causal=True)


@gpu
@pytest.mark.parametrize("nq, nk", [(1, 1), (1, 2), (2, 1), (63, 64), (64, 63), (127, 129), (128, 128), (129, 128), (130, 300), (255, 257), (300, 40), (513, 700)])
@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_lengths(device, nq, nk, dtype, causal):
    run_attention(device, *qkv(2, nq, nk, 2, 1, 64, dtype), causal=causal)


@gpu
@pytest.mark.parametrize("h, hk", [(1, 1), (3, 3), (6, 2), (8, 1), (5, 1), (32, 4)])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_heads(device, h, hk, d):
    run_attention(device, *qkv(2, 140, 140, h, hk, d, BF), causal=True, cap=20.0)


MASKS = {
    "cap": lambda: dict(cap=5.0),
    "bias": lambda: dict(slopes=torch.tensor([0.5, 0.1, 0.0, 2.0], device="cuda")),
    "bias_causal": lambda: dict(slopes=torch.tensor([0.5, 0.1, 0.0, 2.0], device="cuda"), causal=True),
    "prefix": lambda: dict(causal=True, prefix=ints(0, 200, 77)),
    "prefix_alone": lambda: dict(prefix=ints(0, 200, 77)),
    "prefix_everything": lambda: dict(causal=True, prefix=ints(1000, -5, 1)),
    "key_len": lambda: dict(key_len=ints(0, 131, 300)),
    "key_len_causal": lambda: dict(key_len=ints(1, 64, 290), causal=True, q_start=ints(0, 0, 0)),
    "start": lambda: dict(causal=True, q_start=ints(-50, 10, 1000)),
    "docs": lambda: dict(q_docs=torch.arange(300, device="cuda").div(70, rounding_mode="floor").int().repeat(3, 1), k_docs=torch.arange(300, device="cuda").div(70, rounding_mode="floor").int().repeat(3, 1), causal=True),
    "docs_mixed": lambda: dict(q_docs=(torch.arange(900, device="cuda").view(3, 300) * 7 % 5).int(), k_docs=(torch.arange(900, device="cuda").view(3, 300) * 3 % 4).int()),
    "docs_apart": lambda: dict(q_docs=torch.full((3, 300), 1, device="cuda", dtype=torch.int32), k_docs=torch.full((3, 300), 2, device="cuda", dtype=torch.int32)),
    "all": lambda: dict(causal=True, cap=10.0, slopes=torch.tensor([0.05, 0.1, 0.0, 0.2], device="cuda"), prefix=ints(5, 130, 260), key_len=ints(300, 200, 129), q_start=ints(0, 3, -4),
                        q_docs=torch.arange(300, device="cuda").div(90, rounding_mode="floor").int().repeat(3, 1), k_docs=torch.arange(300, device="cuda").div(90, rounding_mode="floor").int().repeat(3, 1)),
}


@gpu
@pytest.mark.parametrize("name", sorted(MASKS))
@pytest.mark.parametrize("d, dtype", [(64, FP), (64, BF), (128, BF), (40, BF)])
def test_attention_masks(device, name, d, dtype):
    run_attention(device, *qkv(3, 300, 300, 4, 2, d, dtype), **MASKS[name]())


@gpu
@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("nq, nk, h, hk, d", [(1, 1, 8, 8, 64), (1, 3000, 8, 1, 128), (1, 4097, 32, 8, 128), (2, 2000, 12, 4, 80), (5, 777, 4, 4, 64), (1, 20000, 2, 2, 128), (3, 1500, 40, 1, 128), (1, 700, 6, 2, 256), (1, 900, 3, 1, 20)])
def test_attention_of_few_queries_over_a_long_cache(device, nq, nk, h, hk, d, dtype):
    """The serving form: padded cache, lengths per sequence, whatever lies behind a length is never used."""
    b = 3
    q, k, v = qkv(b, nq, nk, h, hk, d, dtype)
    k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))          # cache stored head by head
    length = ints(nk, max(nq, nk // 3), nq)
    for i in range(b):
        k[i, int(length[i]):] = float("nan")
        v[i, int(length[i]):] = float("inf")
    run_attention(device, q, k, v, back=False, causal=True, key_len=length, q_start=length - nq, cap=30.0)
    run_attention(device, q, k, v, back=False, causal=True, key_len=length, q_start=length - nq, slopes=torch.linspace(0.01, 0.5, h, device="cuda"))
    length[1] = 0
    k[1], v[1] = float("nan"), float("nan")
    out, lse = run_attention(device, q, k, v, back=False, key_len=length)
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())


@gpu
@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_padded_batch_with_junk_behind_the_lengths(device, dtype, d):
    b, n = 3, 260
    q, k, v = qkv(b, n, n, 4, 2, d, dtype)
    length = ints(260, 131, 0)
    for i in range(b):
        k[i, int(length[i]):] = float("nan")
        v[i, int(length[i]):] = float("-inf")
    run_attention(device, q, k, v, causal=True, key_len=length, q_start=ints(0, 0, 0))


@gpu
@pytest.mark.parametrize("d", [64, 80, 128])
def test_attention_strided_operands(device, d):
    """Slices of one product as operands, slices of one buffer as gradients; what lies around them stays."""
    b, n, h, hk = 2, 200, 4, 2
    joint = randn(b, n, h + 2 * hk + 1, d, dtype=BF)
    q, k, v = joint[:, :, :h], joint[:, :, h:h + hk], joint[:, :, h + hk:h + 2 * hk]
    out_base = torch.full((b, n, h + 1, d), 3.0, device="cuda", dtype=BF)
    lse = torch.empty(b, h, n, device="cuda")
    grad = torch.full_like(joint, 3.0)
    dq, dk, dv = grad[:, :, :h], grad[:, :, h:h + hk], grad[:, :, h + hk:h + 2 * hk]
    dout = randn(b, h, n, d, dtype=BF, seed=4).transpose(1, 2)
    torch.cuda.synchronize()
    ops.attention(device, q, k, v, out_base[:, :, :h], lse, causal=True)
    ops.attention_backward(device, dout, q, k, v, out_base[:, :, :h], lse, dq, dk, dv, causal=True)
    done(device)
    ref = Attention(q, k, v, causal=True)
    want, bound, _, _ = ref.forward()
    close("out", out_base[:, :, :h], want, bound)
    for (name, (want, bound)), got in zip(ref.backward(dout, out_base[:, :, :h], lse).items(), (dq, dk, dv)):
        close(name, got, want, bound)
    assert bool((out_base[:, :, h:] == 3).all()) and bool((grad[:, :, h + 2 * hk:] == 3).all())


@gpu
def test_attention_unaligned_and_broadcast_operands(device):
    b, n, h, d = 2, 100, 2, 64
    flat = randn(b * n * h * d + 1, dtype=BF)
    q = flat[1:].view(b, n, h, d)                                     # starts on an odd element
    k = randn(1, n, 1, d, dtype=BF, seed=2).expand(b, n, h, d)        # one key / value head for everything
    v = randn(1, n, 1, d, dtype=BF, seed=3).expand(b, n, h, d)
    run_attention(device, q, k, v, causal=True)


@gpu
@pytest.mark.parametrize("dtype", [FP, BF])
def test_attention_large_scores(device, dtype):
    """Scores far apart: the running maximum moves by hundreds, most probabilities vanish."""
    run_attention(device, *qkv(1, 300, 600, 2, 2, 64, dtype, scale=40.0), causal=True)
    q, k, v = qkv(1, 200, 520, 2, 2, 64, dtype)
    k = (k.float() * torch.linspace(0.1, 30, 520, device="cuda")[None, :, None, None]).to(dtype)      # growing keys: a new maximum in every tile
    run_attention(device, q, k, v)


@gpu
def test_attention_gradients_agree_with_differences(device):
    b, n, h, hk, d = 1, 9, 2, 1, 8
    q, k, v = qkv(b, n, n, h, hk, d, FP)
    masks = dict(causal=True, cap=2.0, slopes=torch.tensor([0.3, 0.0], device="cuda"), prefix=ints(3))
    out, lse = torch.empty_like(q), torch.empty(b, h, n, device="cuda")
    dout = randn(b, n, h, d, seed=5)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    torch.cuda.synchronize()
    ops.attention(device, q, k, v, out, lse, **masks)
    ops.attention_backward(device, dout, q, k, v, out, lse, dq, dk, dv, **masks)
    done(device)
    loss = lambda *x: float((Attention(*x, **masks).forward()[0] * dout.to(F8)).sum())      # noqa: E731
    h_ = 1e-5
    for which, grad in enumerate((dq, dk, dv)):
        for at in ((0, 0, 0, 0), (0, 4, 0, 3), (0, 8, grad.shape[2] - 1, 7)):
            two = []
            for sign in (1, -1):
                x = [t.to(F8).clone() for t in (q, k, v)]
                x[which][at] += sign * h_
                two.append(_loss64(x, masks, dout))
            assert abs((two[0] - two[1]) / (2 * h_) - float(grad[at])) < 2e-5


def _loss64(x, masks, dout):
    a = Attention.__new__(Attention)
    HALF[F8] = 0.0
    try:
        Attention.__init__(a, *x, **masks)
        return float((a.forward()[0] * dout.to(F8)).sum())
    finally:
        del HALF[F8]


@gpu
@pytest.mark.parametrize("dtype, d", [(FP, 64), (BF, 64), (BF, 128)])
def test_attention_is_deterministic(device, dtype, d):
    q, k, v = qkv(2, 300, 300, 8, 2, d, dtype)
    dout = randn(2, 300, 8, d, dtype=dtype, seed=8)
    first = None
    for _ in range(3):
        out, lse = torch.empty_like(q), torch.empty(2, 8, 300, device="cuda")
        g = [torch.empty_like(x) for x in (q, k, v)]
        torch.cuda.synchronize()
        ops.attention(device, q, k, v, out, lse, causal=True)
        ops.attention_backward(device, dout, q, k, v, out, lse, *g, causal=True)
        done(device)
        now = [out, lse, *g]
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


@gpu
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-4, 3.0])
@pytest.mark.parametrize("nq", [3, 200])
def test_attention_scales(device, scale, nq):
    run_attention(device, *qkv(1, nq, 260, 2, 1, 64, BF), scale=scale, causal=True)
    run_attention(device, *qkv(1, nq, 260, 2, 1, 64, BF), scale=scale, cap=4.0)


@gpu
@pytest.mark.parametrize("group", [2, 3, 4, 8])
@pytest.mark.parametrize("nk", [100, 1500])
def test_attention_gradients_of_shared_heads(device, group, nk):
    """Few blocks (clusters share the heads), many, groups that do not divide into clusters."""
    docs = (torch.arange(nk, device="cuda") // 300).int()[None].repeat(2, 1)
    run_attention(device, *qkv(2, nk, nk, 2 * group, 2, 72, BF), causal=True, q_docs=docs, k_docs=docs)
    run_attention(device, *qkv(2, nk, nk, 2 * group, 2, 128, BF))


@gpu
def test_attention_rows_that_are_not_finite_stay_alone(device):
    """A query that is not finite spoils its own row; the others, keys behind key_len and NaN included, come out as without it."""
    for nq in (4, 300):
        q, k, v = qkv(1, nq, 300, 4, 2, 64, BF)
        want = torch.empty_like(q)
        got, bad = torch.empty_like(q), q.clone()
        bad[0, nq // 2, 1] = float("nan")
        bad[0, nq // 2, 2] = float("inf")
        torch.cuda.synchronize()
        ops.attention(device, q, k, v, want, causal=True, key_len=ints(260), q_start=ints(0))
        ops.attention(device, bad, k, v, got, causal=True, key_len=ints(260), q_start=ints(0))
        done(device)
        rows = torch.ones(nq, 4, dtype=torch.bool, device="cuda")
        rows[nq // 2, 1:3] = False
        assert torch.equal(got[0][rows], want[0][rows]) and bool(got[0, nq // 2, 1].isnan().all())


@gpu
def test_attention_of_nothing(device):
    q, k, v = qkv(2, 5, 0, 2, 2, 64, BF)
    out, lse = run_attention(device, q, k, v, back=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    q, k, v = qkv(2, 0, 5, 2, 2, 64, BF)
    dk, dv = torch.full_like(k, 5.0), torch.full_like(v, 5.0)
    lse = torch.empty(2, 2, 0, device="cuda")
    torch.cuda.synchronize()
    ops.attention(device, q, k, v, torch.empty_like(q), lse)
    ops.attention_backward(device, q, q, k, v, q, lse, q, dk, dv)
    done(device)
    assert bool((dk == 0).all()) and bool((dv == 0).all())


# ---- AdamW

def adam_state(sizes, grads=FP, bits=32, seed=0):
    s = types.SimpleNamespace()
    s.p = [randn(n, seed=seed + i) for i, n in enumerate(sizes)]
    s.g = [randn(n, seed=seed + 50 + i, scale=0.1, dtype=grads) for i, n in enumerate(sizes)]
    s.ms = s.vs = None
    if bits == 32:
        s.m = [randn(n, seed=seed + 100 + i, scale=0.05) for i, n in enumerate(sizes)]
        s.v = [randn(n, seed=seed + 150 + i, scale=0.1).square() for i, n in enumerate(sizes)]
    else:
        s.m = [randn(n, seed=seed + 100 + i, scale=90.0).clamp(-448, 448).to(torch.float8_e4m3fn) for i, n in enumerate(sizes)]
        s.v = [randn(n, seed=seed + 150 + i, scale=90.0).abs().clamp(0, 448).to(torch.float8_e4m3fn) for i, n in enumerate(sizes)]
        s.ms = [randn(-(-n // 128), seed=seed + 200 + i).abs() * 1e-3 for i, n in enumerate(sizes)]
        s.vs = [randn(-(-n // 128), seed=seed + 250 + i).abs() * 1e-3 for i, n in enumerate(sizes)]
    return s


def adam_reference(p, g, m, v, lr, wd, b1, b2, eps, t, gs=1.0):
    """New p, m, v and the size of the update, in 64 bits."""
    g = g.to(F8) * gs
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    up = lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    return p.to(F8) * (1 - lr * wd) - up, m, v, up


SIZES = [1, 3, 128, 129, 4096, 4097, 10007, 2, 70000]


@gpu
@pytest.mark.parametrize("grads", [FP, BF])
@pytest.mark.parametrize("copies", [False, True])
@pytest.mark.parametrize("step", [1, 2, 5000])
def test_adamw_states_in_32_bits(device, grads, copies, step):
    s = adam_state(SIZES, grads)
    before = [[x.clone() for x in y] for y in (s.p, s.m, s.v)]
    c = [torch.empty(n, device="cuda", dtype=BF) for n in SIZES] if copies else None
    wd = [0.1 * (i % 3) for i in range(len(SIZES))]
    opt = ops.AdamW(device, s.p, s.g, s.m, s.v, copies=c, weight_decay=wd, betas=(0.9, 0.99), eps=1e-6)
    gs = torch.tensor([0.25], device="cuda")
    torch.cuda.synchronize()
    opt.step(lr=0.01, step=step, grad_scale=gs)
    done(device)
    for i in range(len(SIZES)):
        p, m, v, up = adam_reference(before[0][i], s.g[i], before[1][i].to(F8), before[2][i].to(F8), 0.01, wd[i], 0.9, 0.99, 1e-6, step, 0.25)
        g = s.g[i].to(F8).abs() * 0.25
        # m, v: constants rounded to fp32 (1 - beta2 to 2^-24 of itself) and three roundings of terms that may cancel
        close("m", s.m[i], m, 4 * 2.0 ** -24 * (0.9 * before[1][i].to(F8).abs() + 0.1 * g))
        close("v", s.v[i], v, 5 * 2.0 ** -24 * v)
        slack = 0.01 * (4 * 2.0 ** -24 * (0.9 * before[1][i].to(F8).abs() + 0.1 * g) / (1 - 0.9 ** step)) / (torch.sqrt(v / (1 - 0.99 ** step)) + 1e-6)
        close("p", s.p[i], p, 3 * 2.0 ** -24 * before[0][i].to(F8).abs() + 16 * 2.0 ** -24 * up.abs() + 2 * slack)
        if copies:
            assert torch.equal(c[i], s.p[i].to(BF))


@gpu
def test_adamw_unaligned_tensors_and_many_of_them(device):
    """Slices that start anywhere, more tensors than one launch takes; what lies between them stays."""
    n, each = 700, 37
    base = [torch.zeros(n * (each + 3) + 1, device="cuda") for _ in range(4)]
    cut = lambda x: [x[1 + i * (each + 3):][:each] for i in range(n)]      # noqa: E731
    for k, x in enumerate(base):
        for y in cut(x)[:1]:
            pass
        x.copy_(randn(x.numel(), seed=k).abs() if k == 3 else randn(x.numel(), seed=k))
    before = [x.clone() for x in base]
    opt = ops.AdamW(device, *(cut(x) for x in base), weight_decay=0.1)
    torch.cuda.synchronize()
    opt.step(lr=0.01)
    done(device)
    p, m, v, up = adam_reference(before[0], before[1], before[2].to(F8), before[3].to(F8), 0.01, 0.1, 0.9, 0.999, 1e-8, 1)
    live = torch.zeros(base[0].numel(), dtype=torch.bool, device="cuda")
    for y in cut(live):
        y.fill_(True)
    for got, want, old in ((base[0], p, before[0]), (base[2], m, before[2]), (base[3], v, before[3])):
        assert torch.equal(got[~live], old[~live])
        close("tensors", got[live], want[live], 1e-5 * (want[live].abs() + old[live].to(F8).abs() + up[live].abs() + 0.01))


@gpu
@pytest.mark.parametrize("grads", [FP, BF])
def test_adamw_states_in_8_bits(device, grads):
    s = adam_state(SIZES, grads, bits=8)
    s.ms[3].zero_(), s.vs[3].zero_()                     # a state that starts from nothing
    wide = lambda c, sc: c.to(F8) * sc.to(F8).repeat_interleave(128)[: c.numel()]      # noqa: E731
    old = [(p.clone(), wide(m, a), wide(v, b).square()) for p, m, v, a, b in zip(s.p, s.m, s.v, s.ms, s.vs)]
    opt = ops.AdamW(device, s.p, s.g, s.m, s.v, m_scales=s.ms, v_scales=s.vs, weight_decay=0.01, betas=(0.9, 0.95), seed=1234)
    torch.cuda.synchronize()
    opt.step(lr=0.01, step=7)
    done(device)
    for i, n in enumerate(SIZES):
        p, m, v, up = adam_reference(old[i][0], s.g[i], old[i][1], old[i][2], 0.01, 0.01, 0.9, 0.95, 1e-8, 7)
        slack = 2.0 ** -21 * 0.01 * (old[i][1].abs() + s.g[i].to(F8).abs()) / (1 - 0.9 ** 7) / (torch.sqrt(v / (1 - 0.95 ** 7)) + 1e-8)
        close("p", s.p[i], p, 4 * 2.0 ** -24 * old[i][0].to(F8).abs() + 2.0 ** -19 * up.abs() + slack)
        h = mix32(torch.arange(n, device="cuda") ^ int(mix32(torch.tensor((int(mix32(torch.tensor(1234 ^ 7))) + i) & 0xffffffff))))
        # fp32 errors of the new states: m is a sum of two terms, each rounded from a product (and the decoded m before it), that
        # may cancel: four half steps of the terms' size.  sqrt(v): only positive terms, a few half steps of itself.
        terms = 0.9 * old[i][1].abs() + 0.1 * s.g[i].to(F8).abs()
        for name, codes, scales, value, bits, err in (("m", s.m[i], s.ms[i], m, h & 0xffff, 4 * 2.0 ** -24 * terms),
                                                      ("sqrt(v)", s.v[i], s.vs[i], v.sqrt(), h >> 16, 8 * 2.0 ** -24 * v.sqrt())):
            blocks = torch.nn.functional.pad(value, (0, -n % 128)).view(-1, 128)
            top = blocks.abs().amax(1)
            worst = torch.nn.functional.pad(err, (0, -n % 128)).view(-1, 128).amax(1)
            close(name + " scales", scales, top / 448, (worst + 4 * 2.0 ** -24 * top) / 448)
            up = torch.where(top > 0, 448 / top, 0.0).repeat_interleave(128)[:n]
            a = (value.abs() * up).clamp(max=448.0)
            # a moves with its own error and with that of the largest value of its block
            a_err = err * up + a * ((worst / top).nan_to_num().repeat_interleave(128)[:n] + 4 * 2.0 ** -24)
            if name != "m":
                a = torch.where(value > 0, a.clamp(min=2.0 ** -9), a)
            step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
            low = torch.floor(a / step)
            share, u = a / step - low, bits.to(F8) / 65536
            want = (low + (share + u >= 1)) * step
            # only a rounding whose border lies within that error (and the border itself is 2^-16 wide) may differ
            edge = 1.01 * a_err / step + 2.0 ** -15
            unsure = ((share + u - 1).abs() <= edge) | (share <= edge) | (share >= 1 - edge)
            got = codes.to(F8)
            assert bool(((got.abs() == want.clamp(max=448.0)) | unsure).all()), name
            close(name + " codes", got.abs(), a, step + 2 * a_err)
            assert bool(((got == 0) | (torch.sign(got) == torch.sign(value)) | (value.abs() <= err)).all())


@gpu
def test_adamw_8_bit_codes_are_those_of_the_formulas_in_fp32(device):
    """m, sqrt(v), scales and codes evaluated operation by operation in fp32, in their written order, twice in a row: bit for bit."""
    n = 1 << 20
    s = adam_state([n, 1000], bits=8)
    m, r, ms, rs = ([x.clone() for x in y] for y in (s.m, s.v, s.ms, s.vs))
    gs = torch.tensor([0.5], device="cuda")
    opt = ops.AdamW(device, s.p, s.g, s.m, s.v, m_scales=s.ms, v_scales=s.vs, betas=(0.9, 0.95), seed=99)
    torch.cuda.synchronize()
    for step in (5, 6):
        opt.step(lr=0.01, step=step, grad_scale=gs)
        done(device)
        for i in range(2):
            size = s.p[i].numel()
            wide = lambda x: x.repeat_interleave(128)[:size]      # noqa: E731
            g = s.g[i] * gs
            nm = 0.9 * (m[i].float() * wide(ms[i])) + (1 - 0.9) * g
            nr = torch.sqrt(0.95 * (r[i].float() * wide(rs[i])).square() + (1 - 0.95) * g * g)
            h = mix32(torch.arange(size, device="cuda") ^ int(mix32(torch.tensor((int(mix32(torch.tensor(99 ^ step))) + i) & 0xffffffff))))
            for name, x, bits, codes, scales, old, old_scale in (("m", nm, h & 0xffff, s.m[i], s.ms[i], m, ms), ("r", nr, h >> 16, s.v[i], s.vs[i], r, rs)):
                top = torch.nn.functional.pad(x, (0, -size % 128)).view(-1, 128).abs().amax(1)
                assert torch.equal(scales, top * (1 / torch.tensor(448.0, device="cuda"))), name
                a = (x * wide((1 / top) * 448)).abs().clamp(max=448)
                if name == "r":
                    a = torch.where(x > 0, a.clamp(min=2.0 ** -9), a)
                e = torch.frexp(a)[1].clamp(min=-5) - 1
                unit = torch.ldexp(torch.ones_like(a), e - 3)
                want = torch.copysign(torch.floor(a / unit + bits.float() / 65536) * unit, x).to(torch.float8_e4m3fn)
                assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)), name
                old[i], old_scale[i] = codes.clone(), scales.clone()


@gpu
def test_adamw_8_bit_rounding_has_no_drift(device):
    """The mean of the rounded state over many seeds is the state: sqrt(v) of a constant gradient grows as it would in 32 bits."""
    n = 4096
    g = [torch.full((n,), 0.5, device="cuda")]
    g[0][::2] = 0.1
    p = [torch.zeros(n, device="cuda")]
    m, v = [torch.zeros(n, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)]
    ms, vs = torch.zeros(n // 128, device="cuda"), torch.zeros(n // 128, device="cuda")
    opt = ops.AdamW(device, p, g, [m], [v], m_scales=[ms], v_scales=[vs], betas=(0.9, 0.99))
    torch.cuda.synchronize()
    steps = 300
    for _ in range(steps):
        opt.step(lr=0.0)
    done(device)
    value = v.float().view(-1, 128) * vs[:, None]
    for k, grad in ((0, 0.1), (1, 0.5)):
        want = grad * math.sqrt(1 - 0.99 ** steps)
        # 2048 samples of a value that is off by a step (12 %) at most, each with a memory of about 100 steps
        assert abs(float(value[:, k::2].mean()) - want) < 0.03 * want


no_guard_zones = pytest.mark.skipif(os.environ.get("ORMI_B200_POOL_CANARY", "0") not in ("", "0"), reason="a capture is refused while guard zones are on")


@gpu
@no_guard_zones
def test_adamw_with_a_device_counter_captured_and_replayed(device):
    from ormi_b200.runtime import Device
    dev = Device(0)
    try:
        n = 5000
        one, two = adam_state([n]), adam_state([n])
        count, lr = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.tensor([0.02], device="cuda")
        a = ops.AdamW(dev, one.p, one.g, one.m, one.v, weight_decay=0.1)
        b = ops.AdamW(dev, two.p, two.g, two.m, two.v, weight_decay=0.1)
        torch.cuda.synchronize()
        a.step(device_step=count, device_lr=lr)
        with dev.capture() as step:
            a.step(device_step=count, device_lr=lr)
        for _ in range(4):
            step.launch()
        for _ in range(5):
            b.step(lr=0.02)
        dev.sync()
        assert int(count) == 5
        for x, y in ((one.p, two.p), (one.m, two.m), (one.v, two.v)):
            assert float((x[0] - y[0]).abs().max()) < 1e-6
        step.destroy()
    finally:
        dev.close()


# ---- offsets past 32 bits

@gpu
def test_attention_over_a_cache_whose_offsets_pass_32_bits(device):
    """Two sequences of 524 293 positions, 32 heads of 128: 4.3e9 elements each for keys and values; one new token and 130 of them."""
    b, nk, h, d = 2, (1 << 19) + 5, 32, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.empty(b, nk, h, d, device="cuda", dtype=BF).normal_(generator=g) for _ in range(2))
    assert k.numel() > 1 << 32
    for nq in (1, 130):
        q = randn(b, nq, h, d, dtype=BF, seed=nq)
        out, lse = torch.empty_like(q), torch.empty(b, h, nq, device="cuda")
        torch.cuda.synchronize()
        ops.attention(device, q, k, v, out, lse, causal=True, scale=0.3)
        done(device)
        for i, n in ((0, 0), (1, 31)):
            ref = Attention(q[i:i + 1, :, n:n + 1], k[i:i + 1, :, n:n + 1], v[i:i + 1, :, n:n + 1], causal=True, scale=0.3)
            want, bound, want_lse, lse_bound = ref.forward()
            close("out", out[i:i + 1, :, n:n + 1], want, bound)
            close("lse", lse[i:i + 1, n:n + 1], want_lse, lse_bound)
            del ref, want, bound
    del k, v
    torch.cuda.empty_cache()


@gpu
def test_norm_over_rows_whose_offsets_pass_32_bits(device):
    rows, cols = (1 << 20) + 7, 4096
    x = torch.empty(rows, cols, device="cuda", dtype=BF).normal_(generator=torch.Generator(device="cuda").manual_seed(2))
    out, rstd, w = torch.empty_like(x), torch.empty(rows, device="cuda"), randn(cols, dtype=BF, seed=3)
    torch.cuda.synchronize()
    ops.rmsnorm(device, x, w, out, rstd=rstd)
    done(device)
    pick = torch.tensor([0, 1 << 19, (1 << 20) + 1, rows - 1], device="cuda")
    y = x[pick].to(F8) / torch.sqrt(x[pick].to(F8).square().mean(1, keepdim=True) + 1e-6)
    close("out", out[pick], y * w.to(F8), 1.02 * 2.0 ** -8 * (y * w.to(F8)).abs())
    dx, s = x, out.clone()
    torch.cuda.synchronize()                                        # the copy runs on another stream
    ops.rmsnorm_backward(device, out, s, w, rstd, dx)
    done(device)
    s, inv = out[pick].to(F8), rstd[pick].to(F8)[:, None]
    gw = s * w.to(F8)
    want = inv * (gw - s * (gw * s).mean(1, keepdim=True) * inv * inv)
    size = inv * (gw.abs() + s.abs() * (gw * s).abs().mean(1, keepdim=True) * inv * inv)
    close("dx", dx[pick], want, 1.01 * (2.0 ** -8 * want.abs() + (cols + 16) * 2.0 ** -24 * size))
    del x, out, dx, y, s
    torch.cuda.empty_cache()


@gpu
def test_attention_of_many_documents_in_a_long_row(device):
    """2^18 + 3 positions in documents of 100: nearly every pair of tiles is skipped."""
    n, h, d = (1 << 18) + 3, 2, 64
    q, k, v = (randn(1, n, h, d, dtype=BF, seed=i) for i in range(3))
    dout = randn(1, n, h, d, dtype=BF, seed=7)
    docs = (torch.arange(n, device="cuda") // 100).int()[None]
    out, lse = torch.empty_like(q), torch.empty(1, h, n, device="cuda")
    g = [torch.empty_like(q) for _ in range(3)]
    torch.cuda.synchronize()
    ops.attention(device, q, k, v, out, lse, causal=True, q_docs=docs, k_docs=docs)
    ops.attention_backward(device, dout, q, k, v, out, lse, *g, causal=True, q_docs=docs, k_docs=docs)
    done(device)
    for first in (0, 100, 1300, 131000, n // 100 * 100):
        cut = slice(first, min(first + 100, n))
        ref = Attention(q[:, cut], k[:, cut], v[:, cut], causal=True)
        want, bound, want_lse, lse_bound = ref.forward()
        close("out", out[:, cut], want, bound)
        close("lse", lse[:, :, cut], want_lse, lse_bound)
        for (name, (want, bound)), got in zip(ref.backward(dout[:, cut], out[:, cut], lse[:, :, cut]).items(), g):
            close(name, got[:, cut], want, bound)


@gpu
def test_two_contexts_and_their_threads_at_once(device):
    """Two contexts' streams side by side, queued by one host thread and by a thread each: the results of calls made alone."""
    import threading
    from ormi_b200.runtime import Device
    devs = [device, Device(0), Device(0), Device(0)]
    try:
        jobs = []
        for i, (n, dt, dd) in enumerate(((700, BF, 64), (900, BF, 128), (300, FP, 64), (5, BF, 128))):
            q, k, v = qkv(2, n, 1100, 4, 2, dd, dt)
            jobs.append((q, k, v, randn(2, n, 4, dd, dtype=dt, seed=30 + i)))
        blank = lambda q, k, v, dout: [torch.empty_like(q), torch.empty(2, 4, q.shape[1], device="cuda"), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)]      # noqa: E731

        def run(dev, job, got, times):
            q, k, v, dout = job
            for _ in range(times):
                ops.attention(dev, q, k, v, got[0], got[1], causal=True)
                ops.attention_backward(dev, dout, q, k, v, got[0], got[1], got[2], got[3], got[4], causal=True)
        want, side, apart = ([blank(*job) for job in jobs] for _ in range(3))
        torch.cuda.synchronize()
        for job, got in zip(jobs, want):
            run(device, job, got, 1)
            done(device)
        for i, (job, got) in enumerate(zip(jobs, side)):
            run(devs[i % 2], job, got, 20)
        threads = [threading.Thread(target=run, args=(devs[i], jobs[i], apart[i], 20)) for i in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for d in devs:
            d.sync()
        for other in (side, apart):
            assert all(torch.equal(x, y) for one, two in zip(want, other) for x, y in zip(one, two))
    finally:
        for d in devs[1:]:
            d.close()


# ---- together, and inside the training loop

@gpu
@pytest.mark.parametrize("matmul", ["fp32", "bf16"])
def test_a_block_of_operators_trains_as_its_formulas_say(matmul):
    """Norm, projection, attention, projection, norm, their gradients and an AdamW step, the products through the lazy graph."""
    from ormi_b200.runtime import Device
    dev = Device(0)
    dev.set_option("matmul", matmul)
    try:
        B, N, W, H, HK, D = 2, 40, 128, 4, 2, 32
        T, E = B * N, (H + 2 * HK) * D
        rng = np.random.default_rng(5)
        host = {k: rng.standard_normal(s).astype(np.float32) * c for k, s, c in (
            ("x", (T, W), 1.0), ("r", (T, W), 1.0), ("g1", (W,), 1.0), ("wqkv", (W, E), W ** -0.5), ("wo", (H * D, W), (H * D) ** -0.5), ("g2", (W,), 1.0), ("c", (T, W), 1.0))}
        docs = np.repeat(np.arange(2), N // 2)[None].repeat(B, 0).astype(np.int32)
        masks = dict(causal=True, cap=8.0)

        leaf = lambda b: G.Node(G.OpEnum.LEAF, data=b, requires_grad=True)      # noqa: E731
        x, r, c = (dev.upload(host[k]) for k in ("x", "r", "c"))
        g1, g2 = dev.upload(host["g1"]), dev.upload(host["g2"])
        wqkv, wo = dev.leaf(host["wqkv"], True), dev.leaf(host["wo"], True)
        d = ops.upload(dev, docs, "i32")
        s1, h1, s2, h2, a = (dev.buffer([T, n]) for n in (W, W, W, W, H * D))
        rstd1, rstd2, lse = dev.buffer([T]), dev.buffer([T]), dev.buffer([B, H, N])
        heads = lambda b, first, n, width: ops.view(b.dev_ptr + first * D * 4, (B, N, n, D), "f32", (N * width, width, D, 1))      # noqa: E731
        parts = lambda b: (heads(b, 0, H, E), heads(b, H, HK, E), heads(b, H + HK, HK, E))      # noqa: E731

        ops.rmsnorm(dev, x, g1, h1, residual=r, residual_out=s1, rstd=rstd1)
        h1n = leaf(h1)
        qkv = G.matmul(h1n, wqkv)
        dev.realize([qkv])
        ops.attention(dev, *parts(qkv.data), heads(a, 0, H, H * D), lse, q_docs=d, k_docs=d, **masks)
        an = leaf(a)
        o = G.matmul(an, wo)
        dev.realize([o])
        ops.rmsnorm(dev, o, g2, h2, residual=s1, residual_out=s2, rstd=rstd2)

        ds2, ds1, dg1, dg2, dqkv = dev.buffer([T, W]), dev.buffer([T, W]), dev.buffer([W]), dev.buffer([W]), dev.buffer([T, E])
        ops.rmsnorm_backward(dev, c, s2, g2, rstd2, ds2, dg2)
        o.grad = leaf(ds2)
        G.compute_gradients(o)
        dev.realize([an.grad, wo.grad])
        ops.attention_backward(dev, heads(an.grad.data, 0, H, H * D), *parts(qkv.data), heads(a, 0, H, H * D), lse, *parts(dqkv), q_docs=d, k_docs=d, **masks)
        qkv.grad = leaf(dqkv)
        G.compute_gradients(qkv)
        dev.realize([h1n.grad, wqkv.grad])
        ops.rmsnorm_backward(dev, h1n.grad, s1, g1, rstd1, ds1, dg1, dresidual=ds2)

        t = {k: torch.tensor(v, dtype=F8, requires_grad=True) for k, v in host.items()}
        norm = lambda v, g: v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-6) * g      # noqa: E731
        z1 = t["x"] + t["r"]
        q, k, v = (norm(z1, t["g1"]) @ t["wqkv"]).view(B, N, H + 2 * HK, D).split([H, HK, HK], 2)
        k, v = (y.repeat_interleave(H // HK, 2) for y in (k, v))
        z = 8.0 * torch.tanh(torch.einsum("bqhd,bkhd->bhqk", q, k) * D ** -0.5 / 8.0)
        td = torch.tensor(docs)
        seen = torch.tril(torch.ones(N, N, dtype=torch.bool))[None] & (td[:, :, None] == td[:, None, :])
        att = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(z.masked_fill(~seen[:, None], -math.inf), -1), v).reshape(T, H * D)
        z2 = att @ t["wo"] + z1
        out = norm(z2, t["g2"])
        (out * t["c"]).sum().backward()
        # fp32: a few hundred roundings of 2^-24 against the largest value; bf16 products: the framework's own bound for them
        tol = 1e-4 if matmul == "fp32" else 3e-2
        for name, got, want in (("h2", dev.download(h2), out), ("dx", dev.download(ds1), t["x"].grad), ("dr", dev.download(ds1), t["r"].grad), ("dg1", dev.download(dg1), t["g1"].grad),
                                ("dg2", dev.download(dg2), t["g2"].grad), ("dwo", dev.numpy(wo.grad), t["wo"].grad), ("dwqkv", dev.numpy(wqkv.grad), t["wqkv"].grad)):
            want = want.detach().numpy()
            assert np.abs(got - want).max() <= tol * np.abs(want).max(), (name, np.abs(got - want).max() / np.abs(want).max())

        params, grads = [wqkv, wo, g1, g2], [wqkv.grad, wo.grad, dg1, dg2]
        states = [[ops.zeros(dev, p.shape) for p in params] for _ in range(2)]
        before = [dev.download(p.data if isinstance(p, G.Node) else p) for p in params]
        gh = [dev.download(g.data if isinstance(g, G.Node) else g) for g in grads]
        ops.AdamW(dev, params, grads, *states, weight_decay=[0.1, 0.1, 0.0, 0.0]).step(lr=0.01)
        for p, old, g, wd in zip(params, before, gh, (0.1, 0.1, 0.0, 0.0)):
            want = old.astype(np.float64) * (1 - 0.01 * wd) - 0.01 * g / (np.abs(g.astype(np.float64)) + 1e-8)      # the first step: m / sqrt(v) is the sign
            got = dev.download(p.data if isinstance(p, G.Node) else p)
            assert np.abs(got - want).max() < 1e-5
        # the next forward product sees the new weights (in "bf16" arithmetic through the copy that the optimizer rewrote)
        again = G.matmul(leaf(h1), wqkv)
        got = dev.numpy(again)
        want = dev.download(h1).astype(np.float64) @ dev.download(wqkv.data).astype(np.float64)
        assert np.abs(got - want).max() <= (1e-5 if matmul == "fp32" else 2e-2) * np.abs(want).max()
    finally:
        dev.close()


def mlp(seed=3, B=96, D=64, F=128):
    rng = np.random.default_rng(seed)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)      # noqa: E731
    return f(B, D), f(B, D), f(D, F) / D ** 0.5, f(F) * 0.1, f(F, D) / F ** 0.5, f(D) * 0.1


def mlp_grads(x, t, w1, b1, w2, b2):
    p = [torch.tensor(v, dtype=F8, requires_grad=True) for v in (w1, b1, w2, b2)]
    z = torch.tensor(x, dtype=F8) @ p[0] + p[1]
    h = 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    loss = ((h @ p[2] + p[3] - torch.tensor(t, dtype=F8)) ** 2).sum() / (x.shape[0] * t.shape[1])
    loss.backward()
    return float(loss.detach()), [v.grad.numpy() for v in p]


@gpu
@pytest.mark.parametrize("matmul, sharded", [("fp32", False), ("bf16", False), ("fp32", True)])
def test_mlp_trainer_with_adamw(matmul, sharded, monkeypatch):
    """Four steps of the training loop against AdamW in 64 bits.  `sharded`: the schedule of several ranks, run by one whose sums
    over ranks are its own."""
    from ormi_b200.runtime import Device
    from ormi_b200.train_step import MLPTrainer
    if sharded:
        monkeypatch.setattr(MLPTrainer, "_allreduce", lambda self, entries, slot: None)
        monkeypatch.setattr(MLPTrainer, "_wait", lambda self, slot: None)
    dev = Device(0)
    dev.set_option("matmul", matmul)
    try:
        x, t, *params = mlp()
        lr, b1, b2, eps, wd = 0.01, 0.9, 0.99, 1e-3, 0.1
        tr = MLPTrainer(dev, x, t, *params, lr=lr, world=2 if sharded else 1, global_batch=x.shape[0], optimizer="adamw", adamw=dict(betas=(b1, b2), eps=eps, weight_decay=wd))
        p, m, v = [q.astype(np.float64) for q in params], [0.0] * 4, [0.0] * 4
        for step in range(1, 5):
            tr.step()
            loss, grads = mlp_grads(x, t, *p)
            assert abs(tr.loss() - loss) <= (1e-4 if matmul == "fp32" else 3e-2) * loss
            for i, g in enumerate(grads):
                m[i] = b1 * m[i] + (1 - b1) * g
                v[i] = b2 * v[i] + (1 - b2) * g * g
                p[i] = p[i] - lr * (wd if i in (0, 2) else 0.0) * p[i] - lr * (m[i] / (1 - b1 ** step)) / (np.sqrt(v[i] / (1 - b2 ** step)) + eps)
        # an update is at most lr; relative errors of the gradients (1e-5 of the largest; bf16 products: 2e-2) pass through it against eps
        tol = 4 * lr * (1e-3 if matmul == "fp32" else 0.3)
        for name, want, old in zip(("w1", "b1", "w2", "b2"), p, params):
            got = tr.parameter(name).reshape(want.shape)
            assert np.abs(got - want).max() <= tol, name
            assert np.abs(got - old).max() > lr
    finally:
        dev.close()


@gpu
def test_mlp_trainer_with_adamw_in_8_bits_stays_near_32(device):
    from ormi_b200.train_step import MLPTrainer
    x, t, *params = mlp()
    lr, steps, got = 0.003, 10, {}
    for bits in (32, 8):
        tr = MLPTrainer(device, x, t, *params, lr=lr, optimizer="adamw", adamw=dict(state_bits=bits, betas=(0.9, 0.99)))
        for _ in range(steps):
            tr.step()
        got[bits] = [tr.parameter(k) for k in ("w1", "b1", "w2", "b2")]
    for p8, p32, old in zip(got[8], got[32], params):
        # a code is off by a step (1/8 of the value) at most and by less on average, so an update m / sqrt(v) of size lr is off by
        # 1/4 at most to first order; the mean over a tensor and ten steps stays below that
        assert np.abs(p8 - p32).mean() < 0.25 * steps * lr
        assert np.isfinite(p8).all() and np.abs(p8 - old.ravel()).mean() > lr


def test_mlp_trainer_refuses_unknown_optimizers():
    from ormi_b200.train_step import MLPTrainer
    with pytest.raises(ValueError, match="optimizer"):
        MLPTrainer(NODEV, *mlp(), lr=0.1, optimizer="adam")


@gpu
@no_guard_zones
def test_captured_block_replays_with_new_inputs_and_weights():
    """A captured forward and backward pass with an AdamW step: replays read the buffers' new contents, update in place, and a bf16
    copy made of a captured output outside is not used after a replay."""
    from ormi_b200.runtime import Device
    dev = Device(0)
    try:
        b, n, h, d = 1, 200, 4, 64
        q, k, v = qkv(b, n, n, h, h, d, BF)
        out, lse, dout = torch.empty_like(q), torch.empty(b, h, n, device="cuda"), randn(b, n, h, d, dtype=BF, seed=9)
        grads = [torch.empty_like(q) for _ in range(3)]
        w = torch.randn(n * h * d, device="cuda")
        m, s2 = torch.zeros_like(w), torch.zeros_like(w)
        count = torch.zeros(1, dtype=torch.int64, device="cuda")
        opt = ops.AdamW(dev, [w], [grads[0].view(-1)], [m], [s2])

        def step():
            ops.attention(dev, q, k, v, out, lse, causal=True)
            ops.attention_backward(dev, dout, q, k, v, out, lse, *grads, causal=True)
            opt.step(lr=0.01, device_step=count)
        torch.cuda.synchronize()
        step()
        dev.sync()
        with dev.capture() as one:
            step()
        step()                                           # the first graph keeps its scratch: a second one needs a plain run of its own
        dev.sync()
        with dev.capture() as two:
            step()
        q.copy_(randn(b, n, h, d, dtype=BF, seed=77))
        torch.cuda.synchronize()
        one.launch()
        two.launch()
        dev.sync()
        assert int(count) == 4
        ref = Attention(q, k, v, causal=True)
        want, bound, _, _ = ref.forward()
        close("out", out, want, bound)
        for (name, (want, bound)), got in zip(ref.backward(dout, out, lse).items(), grads):
            close(name, got, want, bound)
        one.destroy()
        two.launch()
        dev.sync()
        assert int(count) == 5
        two.destroy()
    finally:
        dev.close()
