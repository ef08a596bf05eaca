"""Transformer-block operators at the edges of what their documentation allows."""
import ctypes
import math

import numpy as np
import pytest

from ormi_b200 import graph as G
from ormi_b200 import ops
from ormi_b200 import workloads as W
from ormi_b200._lib import BackendError, check, lib
from test_transformer_ops import ACC, Attention, BF, F8, FP, NODEV, V, accepted, attn_args, close, done, gpu, ints, no_guard_zones, norm_args, norm_back, randn, refused, run_attention, torch


# ---- attention

UNSEEN = {
    # most of every row behind its length, one row without any key
    "key_len": lambda b, nq, nk: (dict(key_len=ints(*[nk // 9, 0, 130, 1][:b])), torch.tensor([nk // 9, 0, 130, 1][:b])),
    # the queries stand at the first positions of a longer row of keys
    "before": lambda b, nq, nk: (dict(causal=True, q_start=ints(*[0, 5, 100, 64][:b])), torch.tensor([nq + s for s in (0, 5, 100, 64)[:b]])),
    # every key from the 200th on is of a document that has no query
    "docs": lambda b, nq, nk: (dict(q_docs=torch.zeros(b, nq, dtype=torch.int32, device="cuda"),
                                    k_docs=(torch.arange(nk, device="cuda") >= 200).int().mul(7).repeat(b, 1)), torch.full((b,), 200)),
}


@gpu
@pytest.mark.parametrize("mask", sorted(UNSEEN))
@pytest.mark.parametrize("d", [64, 128])
# blocks of the key kernel and heads of a group decide how many blocks share a key/value head: 1, 2 and 4 of them, alone and with documents
@pytest.mark.parametrize("b, nk, h, hk", [(4, 20000, 24, 8), (4, 20000, 16, 8), (2, 4000, 2, 1), (1, 1100, 8, 1), (1, 1100, 6, 2), (1, 900, 3, 1)])
def test_attention_gradients_of_keys_that_nobody_sees(device, mask, d, b, nk, h, hk):
    """Exactly zero, every time: the keys and values of such a tile are still on their way when its zeros are written.  The caches
    are emptied between the calls (by a fill of 256 MB), so that they come from far."""
    nq = 128
    q, k, v = randn(b, nq, h, d, dtype=BF, seed=1), randn(b, nk, hk, d, dtype=BF, seed=2), randn(b, nk, hk, d, dtype=BF, seed=3)
    masks, first = UNSEEN[mask](b, nq, nk)
    unseen = torch.arange(nk)[None, :] >= first[:, None]
    unseen = unseen.cuda()
    if mask == "key_len":
        k[unseen], v[unseen] = float("nan"), float("inf")
    dout, out, lse = randn(b, nq, h, d, dtype=BF, seed=4), torch.empty_like(q), torch.empty(b, h, nq, device="cuda")
    grads = [torch.empty_like(x) for x in (q, k, v)]
    flush = torch.empty(64 << 20, device="cuda")
    torch.cuda.synchronize()
    ops.attention(device, q, k, v, out, lse, **masks)
    done(device)
    seen = None
    for turn in range(12):
        for x in grads:
            x.fill_(3.0)
        flush.fill_(float(turn))
        torch.cuda.synchronize()
        ops.attention_backward(device, dout, q, k, v, out, lse, *grads, **masks)
        done(device)
        for name, x in zip(("dk", "dv"), grads[1:]):
            assert bool((x[unseen] == 0).all()), f"{name}, call {turn}: {int((x[unseen] != 0).sum())} values of unseen keys are not zero"
            assert bool(torch.isfinite(x).all()), name
        if seen is None:
            seen = [x.clone() for x in grads]
        assert all(torch.equal(x, y) for x, y in zip(grads, seen)), f"call {turn} differs from the first"


@gpu
@pytest.mark.parametrize("nq, nk, d", [(1, 700, 64), (3, 1500, 128), (16, 90, 64), (200, 300, 64)])
@pytest.mark.parametrize("cap", [1e4, 1e6, 1e9, 1e30])
@pytest.mark.parametrize("scale", [None, -0.2])
def test_attention_under_a_cap_far_above_the_scores(device, nq, nk, d, cap, scale):
    """Such a cap changes nothing: |z - cap tanh(z / cap)| < |z|^3 / (3 cap^2) < 1e-5 for |z| < 30 and caps from 1e4 on, so the bounds
    are those of the call without a cap, which do not grow with it.  Few queries and many, either sign of the scale."""
    b, h, hk = 2, 4, 2
    q, k, v = randn(b, nq, h, d, dtype=BF, seed=1), randn(b, nk, hk, d, dtype=BF, seed=2), randn(b, nk, hk, d, dtype=BF, seed=3)
    out, lse = torch.empty_like(q), torch.empty(b, h, nq, device="cuda")
    torch.cuda.synchronize()
    ops.attention(device, q, k, v, out, lse, causal=True, cap=cap, scale=scale)
    done(device)
    ref = Attention(q, k, v, causal=True, scale=scale)
    want, bound, want_lse, lse_bound = ref.forward()
    size = float(ref.z[ref.seen].abs().max())
    assert size < 30
    off = size ** 3 / (3 * cap ** 2)
    close("lse", lse, want_lse, lse_bound + off)
    close("out", out, want, bound + 3 * off * float(v.abs().max()))


@gpu
@pytest.mark.parametrize("nq, nk", [(1, 700), (5, 300), (200, 300)])
@pytest.mark.parametrize("cap, scale", [(0.5, 0.3), (3.0, -0.4), (20.0, 2.0), (5.0, 0.0)])
def test_attention_caps_of_either_sign_that_scores_reach(device, nq, nk, cap, scale):
    """Scores on both sides of the border between the polynomial and the exponential form of the cap."""
    run_attention(device, randn(2, nq, 4, 64, dtype=BF, seed=1), randn(2, nk, 2, 64, dtype=BF, seed=2), randn(2, nk, 2, 64, dtype=BF, seed=3), causal=True, cap=cap, scale=scale)


@gpu
@pytest.mark.parametrize("nq, nk", [(2, 400), (200, 300)])
@pytest.mark.parametrize("cap", [3e6, 1e7, 1e8, 1e12])
def test_attention_large_caps_that_scores_reach(device, nq, nk, cap):
    """Scores up to 0.4 of a cap whose sixth power leaves fp32 against the scale: capped scores to 2^-16 (the exponential form is off by
    5e-7 of the cap, on scores from a tenth of it on; below, the polynomial's terms are worth less than 2^-24)."""
    b, h, d = 2, 2, 64
    q, k, v = (randn(b, n, h, d, dtype=BF, seed=i) for i, n in ((1, nq), (2, nk), (3, nk)))
    scale = 0.125
    size = (q.float().transpose(1, 2) @ k.float().permute(0, 2, 3, 1)).abs().max().item() * scale
    q = (q * (0.4 * cap / size) ** 0.5).to(BF)
    k = (k * (0.4 * cap / size) ** 0.5).to(BF)
    out, lse = torch.empty_like(q), torch.empty(b, h, nq, device="cuda")
    torch.cuda.synchronize()
    ops.attention(device, q, k, v, out, lse, cap=cap, scale=scale)
    done(device)
    want = Attention(q, k, v, cap=cap, scale=scale).lse
    close("lse", lse, want, 2.0 ** -16 * want.abs() + 2.0 ** -20 * math.log(nk))


@gpu
@pytest.mark.parametrize("nq, nk", [(1, 400), (8, 90), (200, 300)])
@pytest.mark.parametrize("cap", [1e-6, 1e-8, 1e-14, 1e-20, 1e-37])
@pytest.mark.parametrize("scale", [0.125, -3.0])
def test_attention_caps_far_below_the_scores(device, nq, nk, cap, scale):
    """Capped scores are all but equal; queries of zeros have scores of zero, whatever power of scale / cap leaves fp32."""
    q, k, v = randn(2, nq, 4, 64, dtype=BF, seed=1), randn(2, nk, 2, 64, dtype=BF, seed=2), randn(2, nk, 2, 64, dtype=BF, seed=3)
    q[0] = 0.0
    k[1, 5] = 0.0
    run_attention(device, q, k, v, causal=True, cap=cap, scale=scale)


@pytest.mark.parametrize("call", [
    # as many rows as 2^64 is zero of: an output whose rows all lie on one another is not an empty one
    lambda: norm_args(x=V(0x1000, (1 << 30, 1 << 30, 16, 64), "bf16", (0, 0, 0, 1)), out=V(0x8000, (1 << 30, 1 << 30, 16, 64), "bf16", (0, 0, 0, 1))),
    lambda: attn_args(b=16, nq=1 << 30, h=1 << 30, hk=1, q=V(0x100000, (16, 1 << 30, 1 << 30, 32), "bf16", (0, 0, 0, 1)), out=V(0x400000, (16, 1 << 30, 1 << 30, 32), "bf16", (0, 0, 0, 1))),
    # spans beyond 63 bits
    lambda: norm_args(x=V(0x1000, ((1 << 31) - 1, 64), "bf16", ((1 << 40) - 1, 1)), out=V(0x8000, ((1 << 31) - 1, 64), "bf16", ((1 << 40) - 1, 1))),
    lambda: attn_args(b=1, nk=1 << 30, k=V(0x200000, (1, 1 << 30, 2, 32), "bf16", (0, (1 << 40) - 8, 32, 1)), v=V(0x300000, (1, 1 << 30, 2, 32), "bf16", (0, (1 << 40) - 8, 32, 1))),
])
def test_views_beyond_the_address_space_are_refused(call):
    refused(call(), "too large")


def test_attention_refuses_caps_without_an_inverse():
    for cap in (1e-39, 1e-45):
        refused(attn_args(cap=cap), "cap")
    accepted(attn_args(cap=1e-37))


@gpu
@pytest.mark.parametrize("n", [(1 << 19) + 77, (1 << 20) - 5])
def test_attention_of_documents_up_to_the_longest_row(device, n):
    """Up to the 2^20 positions that the tensor-core kernels take, in documents of 200."""
    h, d, size = 1, 64, 200
    q, k, v, dout = (randn(1, n, h, d, dtype=BF, seed=i) for i in range(4))
    docs = (torch.arange(n, device="cuda") // size).int()[None]
    out, lse = torch.empty_like(q), torch.empty(1, h, n, device="cuda")
    g = [torch.full_like(q, 3.0) for _ in range(3)]
    torch.cuda.synchronize()
    ops.attention(device, q, k, v, out, lse, causal=True, q_docs=docs, k_docs=docs)
    ops.attention_backward(device, dout, q, k, v, out, lse, *g, causal=True, q_docs=docs, k_docs=docs)
    done(device)
    for first in (0, 400, (1 << 18) // size * size, (1 << 19) // size * size - size, (1 << 19) // size * size, n // size * size - size, n // size * size):
        cut = slice(first, min(first + size, n))
        ref = Attention(q[:, cut], k[:, cut], v[:, cut], causal=True)
        want, bound, want_lse, lse_bound = ref.forward()
        close("out", out[:, cut], want, bound)
        close("lse", lse[:, :, cut], want_lse, lse_bound)
        for (name, (want, bound)), got in zip(ref.backward(dout[:, cut], out[:, cut], lse[:, :, cut]).items(), g):
            close(name, got[:, cut], want, bound)
    assert all(bool(torch.isfinite(x).all()) and not bool((x == 3.0).all(-1).any()) for x in g)


# ---- buffers

class _Elsewhere:
    """A device of another GPU, as far as buffers know one."""
    index, handle = 1, None

    def alloc(self, nbytes):
        return 0x700000

    def free(self, ptr, nbytes):
        pass


def test_buffers_of_another_gpu_are_refused():
    far = _Elsewhere()
    buf = G.Buffer((4, 64))
    buf.dev_ptr, buf._release = far.alloc(buf.nbytes), far.free
    node = G.Node(G.OpEnum.LEAF, data=buf)
    for x in (ops.empty(far, (4, 64)), buf, node):
        refused(norm_args(x=x, out=V(0x8000, (4, 64))), "cuda:1")
    near = G.Buffer((4, 64))
    near.dev_ptr = 0x1000
    accepted(norm_args(x=near, out=V(0x8000, (4, 64))))


# ---- RMS norm

def test_norm_refuses_rows_whose_columns_pass_an_int():
    """(The kernels step past the last column in 32 bits.)"""
    at = lambda address, cols: V(address << 36, (2, cols), "bf16", (1 << 33, 1))      # noqa: E731
    for cols in ((1 << 30) + 1, (1 << 31) - 1):
        refused(norm_args(x=at(1, cols), weight=None, out=at(2, cols)), "2^30 columns")
        refused(norm_back(dout=at(1, cols), s=at(2, cols), weight=None, dx=at(3, cols), rstd=V(0x4000, (2,)), dweight=None), "2^30 columns")
    accepted(norm_args(x=at(1, 1 << 30), weight=None, out=at(2, 1 << 30)))

@gpu
@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("cols", [100, 256, 1111, 4096, 40000])
@pytest.mark.parametrize("group", [0, 128])
def test_norm_to_eight_bits_of_tiny_groups(device, dtype, cols, group):
    """Maxima down to 1e-39, where 448 / maximum is not an fp32 number: codes follow the values, zeros stay zeros."""
    sizes = [1e-30, 3e-36, 1e-37, 2e-39]
    x = randn(len(sizes) + 1, cols, seed=5).to(F8) * torch.tensor([*sizes, 0.0], dtype=F8, device="cuda")[:, None]     # (and a row of zeros)
    x[:, ::3] = 0.0
    x = x.to(dtype)
    # rstd = 1 / sqrt(eps) = 2^10 exactly, since s^2 vanishes against eps, and the weight takes that back
    weight, groups = torch.full((cols,), 2.0 ** -10, device="cuda"), 1 if not group else -(-cols // group)
    out, scales = torch.empty(x.shape, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(len(x), groups, device="cuda")
    torch.cuda.synchronize()
    ops.rmsnorm(device, x, weight, out, scales=scales, group=group, eps=2.0 ** -20)
    done(device)
    y = torch.nn.functional.pad(x.to(F8), (0, groups * (group or cols) - cols)).view(len(x), groups, -1)
    got = torch.nn.functional.pad(out.to(F8), (0, groups * (group or cols) - cols)).view(len(x), groups, -1)
    top = y.abs().amax(-1, keepdim=True)
    # y may be off by half of the smallest fp32 number, and relatively by a few roundings
    off = (2.0 ** -149 + 2.0 ** -20 * y.abs()) * torch.where(top > 0, 448 / top, 0.0)
    want = y * torch.where(top > 0, 448 / top, 0.0)
    # half a step of e4m3: 2^-4 of the value, 2^-10 below 2^-6
    bound = (want.abs() * 2.0 ** -4).clamp_min(2.0 ** -10) + 2 * off
    assert bool(torch.isfinite(got).all())
    assert bool(((got - want).abs() <= bound).all())
    assert bool((got[y == 0] == 0).all())
    assert bool(((scales.to(F8) - top[..., 0] / 448).abs() <= 2.0 ** -149 + 2.0 ** -22 * top[..., 0] / 448).all())


# ---- AdamW

def test_a_refused_adamw_step_does_not_count():
    """Refused for its rate, its gradient, its step number or its scalars: the next step is still the one that comes after the last good one."""
    opt = ops.AdamW(NODEV, [V(0x10000, (300,))], [V(0x20000, (300,))], [V(0x30000, (300,))], [V(0x40000, (300,))])
    for bad in (dict(lr=float("nan")), dict(lr=0.1, grads=[V(0x10000, (300,))]), dict(lr=0.1, grads=[]), dict(lr=0.1, step=0), dict(lr=0.1, step=-3), dict(lr=0.1, grad_scale=0x8002)):
        with pytest.raises((BackendError, ValueError)):
            opt.step(**bad)
        assert opt.steps_done == 0, bad


def test_adamw_refuses_device_scalars_inside_what_it_writes():
    """The blocks of a launch would read them while others write there."""
    def opt(**more):
        return ops.AdamW(NODEV, [V(0x10000, (300,))], [V(0x20000, (300,))], [V(0x30000, (300,))], [V(0x40000, (300,))], **more)
    refused(lambda: opt().step(lr=0.1, grad_scale=0x10004), "overlaps")
    refused(lambda: opt().step(device_lr=0x30000 + 1196), "overlaps")
    refused(lambda: opt().step(lr=0.1, device_step=0x40008), "overlaps")
    refused(lambda: opt().step(lr=0.1, device_step=0x20008), "overlaps")
    refused(lambda: opt().step(lr=0.1, device_step=0x80000, grad_scale=0x80004), "overlaps")
    accepted(lambda: opt().step(grad_scale=0x20004, device_lr=0x20004, device_step=0x80000))


def test_adamw_refuses_an_eps_that_its_reciprocal_takes_for_zero():
    """The quotient is m times an approximate reciprocal that flushes numbers below 2^-126: an element without a gradient would be 0 * inf."""
    def opt(eps):
        return ops.AdamW(NODEV, [V(0x10000, (300,))], [V(0x20000, (300,))], [V(0x30000, (300,))], [V(0x40000, (300,))], eps=eps)
    for eps in (1e-38, 1e-45, 1e-60):
        refused(lambda: opt(eps).step(lr=0.1), "eps")
    for eps in (0.0, 1.2e-38, 1e-8):
        accepted(lambda: opt(eps).step(lr=0.1))


@gpu
def test_adamw_goes_on_after_a_refused_step(device):
    n = 500
    g = randn(n, seed=8)
    got = []
    for refuse in (False, True):
        p, m, v = torch.ones(n, device="cuda"), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        opt = ops.AdamW(device, [p], [g], [m], [v])
        torch.cuda.synchronize()
        for _ in range(3):
            if refuse:
                with pytest.raises(BackendError):
                    opt.step(lr=float("inf"))
            opt.step(lr=0.1)
        done(device)
        assert opt.steps_done == 3
        got.append((p, m, v))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@gpu
@pytest.mark.parametrize("size", [1e-30, 1e-35, 1e-37])
def test_adamw_8_bit_states_of_tiny_gradients(device, size):
    """m far below 1e-36, where 448 / maximum is not an fp32 number: what was zero stays zero, the rest keeps its size.  9000 elements:
    two whole chunks and a part of one."""
    n, b1 = 9000, 0.75
    g = randn(n, seed=6) * size
    g[::3] = 0.0
    p, m, v = torch.zeros(n, device="cuda"), *(torch.zeros(n, device="cuda").to(torch.float8_e4m3fn) for _ in range(2))
    scales = [torch.zeros(-(-n // 128), device="cuda") for _ in range(2)]
    opt = ops.AdamW(device, [p], [g], [m], [v], m_scales=[scales[0]], v_scales=[scales[1]], betas=(b1, 0.9))
    torch.cuda.synchronize()
    opt.step(lr=0.1)
    done(device)
    want = (1 - b1) * g.to(F8)
    tops = torch.nn.functional.pad(want, (0, -n % 128)).view(-1, 128).abs().amax(1)
    top = tops.repeat_interleave(128)[:n]
    got = m.to(F8) * scales[0].to(F8).repeat_interleave(128)[:n]
    # rounded up or down by less than a step: 2^-3 of the value, 2^-9 of a code below 2^-6; codes are at most 448, and a
    # scale (or an m) may be off by the smallest fp32 number
    bound = torch.maximum(want.abs() * 2.0 ** -3, 2.0 ** -9 * top / 448) * 1.01 + 450 * 2.0 ** -149 + 2.0 ** -20 * top
    assert bool(torch.isfinite(m.to(F8)).all()) and bool((m.to(F8)[::3] == 0).all())
    assert bool(((got - want).abs() <= bound).all())


# ---- captured steps over weights that have a bf16 copy

class Steps:
    """A context in "bf16" arithmetic with y = x w (the products read bf16 copies that the context keeps of x and w) and an
    optimizer of w.  `check` compares y with the product of the weights as they stood before the call."""
    N = 128                                                     # the smallest cube that takes the path with copies

    def __init__(self):
        from ormi_b200.runtime import Device
        self.dev = Device(0)
        self.dev.set_option("matmul", "bf16")
        n = self.N
        self.x, self.w, self.g = (ops.upload(self.dev, W.normal(seed, (n, n))) for seed in (1, 2, 3))
        self.y, self.z = ops.empty(self.dev, (n, n)), ops.empty(self.dev, (n, n))
        self.opt = ops.AdamW(self.dev, [self.w], [self.g], [ops.zeros(self.dev, (n, n))], [ops.zeros(self.dev, (n, n))], betas=(0.0, 0.0))
        self.count = ops.zeros(self.dev, (2,), "i32")           # a 64-bit counter

    def product(self, y=None, w=None):
        n = self.N
        dims, strides = (ctypes.c_int32 * 2)(n, n), (ctypes.c_int32 * 2)(n, 1)
        check(lib.ormi_b200_matmul(self.dev.handle, self.x.ptr, 2, dims, strides, (w or self.w).ptr, 2, dims, strides, (y or self.y).ptr, 2, dims))

    def update(self):
        """Every weight moves by about 1 (betas of 0: the update is lr times the gradient's sign)."""
        self.opt.step(lr=1.0, device_step=self.count.ptr)

    def put(self, seed):
        self.dev.h2d(self.w.ptr, W.normal(seed, (self.N, self.N)))

    def check(self, what, call, y=None):
        y = y or self.y
        rounded = lambda a: torch.from_numpy(a.numpy()).to(BF).to(F8)      # noqa: E731
        x, w = rounded(self.x), rounded(self.w)
        check(lib.ormi_b200_memset(self.dev.handle, y.ptr, 0, y.nbytes))
        call()
        got = torch.from_numpy(y.numpy()).to(F8)
        bound = ACC * (self.N + 4) * (x.abs() @ w.abs())        # fp32 sums of exact products
        assert bool(((got - x @ w).abs() <= bound).all()), f"{what}: y is not the product of the weights, off by {float((got - x @ w).abs().max()):.3g}"


@pytest.fixture
def steps():
    s = Steps()
    yield s
    s.dev.close()


def outside(s):
    """Ways in which a weight changes between two replays."""
    other = ops.upload(s.dev, W.normal(77, (s.N, s.N)))
    return [("nothing", lambda: None), ("an update", s.update), ("an upload", lambda: s.put(50)), ("a copy", lambda: check(lib.ormi_b200_memcpy_d2d(s.dev.handle, s.w.ptr, other.ptr, other.nbytes))),
            ("an upload and an update", lambda: (s.put(51), s.update())), ("an upload and a product", lambda: (s.put(52), s.product(s.z))), ("nothing again", lambda: None)]


@gpu
@no_guard_zones
@pytest.mark.parametrize("trains", [False, True])
def test_captured_product_follows_its_weights(steps, trains):
    """A replay multiplies with the weights as they are, whatever changed them; and so does a plain product after a replay."""
    s = steps

    def step():
        s.product()
        if trains:
            s.update()
    s.check("plain", step)
    with s.dev.capture() as one:
        step()
    for what, change in outside(s):
        change()
        s.check(f"replay after {what}", one.launch)
        s.check(f"replay after a replay after {what}", one.launch)
        s.check(f"product after {what} and a replay", s.product)
        s.check(f"product again after {what}", s.product)
    one.destroy()
    s.check("product after the graph", s.product)
    s.check("step after the graph", step)


@gpu
@no_guard_zones
@pytest.mark.parametrize("first, second", [("both", "both"), ("both", "product"), ("product", "both"), ("product", "update"), ("update", "product")])
def test_two_captured_steps_share_their_weights(steps, first, second):
    s = steps
    parts = {"both": lambda: (s.product(), s.update()), "product": s.product, "update": s.update}
    s.check("plain", parts["both"])
    with s.dev.capture() as one:
        parts[first]()
    with s.dev.capture() as two:
        parts[second]()
    graphs = [(g, name != "update") for g, name in ((one, first), (two, second))]

    def run(order):
        for i in order:
            g, multiplies = graphs[i]
            if multiplies:
                s.check(f"graph {i} of {order}", g.launch)
            else:
                g.launch()
    run([0, 0, 1, 1, 0, 1])
    for what, change in outside(s):
        change()
        run([1, 0, 1])
        s.check(f"product after {what}", s.product)
    one.destroy()                                               # the second one's copies stay its own
    junk = [ops.zeros(s.dev, (s.N, s.N), "bf16") for _ in range(6)]
    for j in junk:
        check(lib.ormi_b200_memset(s.dev.handle, j.ptr, 0x55, j.nbytes))
    graphs[0] = (two, second != "update")
    run([1, 0])
    s.put(60)
    run([1, 1])
    two.destroy()
    s.check("product after both", s.product)


@gpu
@no_guard_zones
def test_a_copy_that_a_capture_recorded_is_not_taken_for_made(steps):
    """The weight's copy is dropped before the capture, so its conversion is recorded: a plain product between the capture and the
    first replay does not read a copy that nothing has written yet."""
    s = steps
    s.check("plain", s.product)
    s.put(40)
    with s.dev.capture() as one:
        s.product(s.z)
    s.check("product before the first replay", s.product)
    s.put(41)
    s.check("replay", one.launch, s.z)
    s.check("product", s.product)
    one.destroy()


@gpu
@no_guard_zones
def test_writes_inside_a_capture_make_copies_stale_at_every_replay(steps):
    """A captured fill of the weight: copies that plain products made between two replays are not used after the second."""
    s = steps
    s.check("plain", s.product)
    with s.dev.capture() as one:
        check(lib.ormi_b200_fill_u32(s.dev.handle, s.w.ptr, int(np.float32(0.5).view(np.uint32)), s.N * s.N))
    for seed in (30, 31):
        s.put(seed)
        s.check("product between", s.product)
        one.launch()
        s.check("product after the fill", s.product)
    one.destroy()


@gpu
@no_guard_zones
def test_results_of_a_captured_realize_are_multiplied_as_they_are(steps):
    """A plain product with a captured result as its weight makes a copy of it, which the next replay overtakes."""
    s = steps
    a = s.dev.leaf(W.normal(20, (s.N, s.N)))
    for _ in range(2):
        kept = G.add(a, a)
        s.dev.realize([kept])
        del kept
    with s.dev.capture() as one:
        kept = G.add(a, a)
        s.dev.realize([kept])
    for seed in (21, 22, 23):
        s.dev.h2d(a.data.dev_ptr, W.normal(seed, (s.N, s.N)))
        one.launch()
        s.w, w = ops.view(kept.data.dev_ptr, (s.N, s.N)), s.w
        want = torch.from_numpy(2 * W.normal(seed, (s.N, s.N))).to(BF).to(F8)
        x = torch.from_numpy(s.x.numpy()).to(BF).to(F8)
        s.product()
        s.w = w
        got = torch.from_numpy(s.y.numpy()).to(F8)
        assert bool(((got - x @ want).abs() <= ACC * (s.N + 4) * (x.abs() @ want.abs())).all()), seed
    one.destroy()


@gpu
@pytest.mark.parametrize("writer", ["matmul", "sum", "gemm_bf16", "gemm_bf16_kmajor", "memset", "copy"])
def test_raw_results_make_the_copies_of_their_buffer_stale(steps, writer):
    """A buffer that was multiplied with (so that the context has a bf16 copy of it) is written by a raw call and multiplied with again."""
    s, n = steps, steps.N
    two, one = (ctypes.c_int32 * 2)(n, n), (ctypes.c_int32 * 1)(0)
    many = ops.upload(s.dev, W.normal(9, (2, n, n)))
    half = [ops.upload(s.dev, W.normal(seed, (n, n)), "bf16") for seed in (4, 5)]
    shape3, strides3 = (ctypes.c_int32 * 3)(2, n, n), (ctypes.c_int32 * 3)(n * n, n, 1)
    calls = {
        "matmul": lambda: lib.ormi_b200_matmul(s.dev.handle, s.x.ptr, 2, two, (ctypes.c_int32 * 2)(n, 1), s.g.ptr, 2, two, (ctypes.c_int32 * 2)(n, 1), s.w.ptr, 2, two),
        "sum": lambda: lib.ormi_b200_sum(s.dev.handle, many.ptr, 3, shape3, strides3, one, 1, s.w.ptr),
        "gemm_bf16": lambda: lib.ormi_b200_gemm_bf16(s.dev.handle, half[0].ptr, 0, half[1].ptr, 0, s.w.ptr, n, n, n),
        "gemm_bf16_kmajor": lambda: lib.ormi_b200_gemm_bf16_kmajor(s.dev.handle, half[0].ptr, half[1].ptr, s.w.ptr, n, n, n),
        "memset": lambda: lib.ormi_b200_memset(s.dev.handle, s.w.ptr, 0x3f, s.w.nbytes),
        "copy": lambda: lib.ormi_b200_memcpy_d2d(s.dev.handle, s.w.ptr, s.g.ptr, s.w.nbytes),
    }
    before = s.w.numpy()
    s.check("before", s.product)
    check(calls[writer]())
    assert np.abs(s.w.numpy() - before).max() > 0.5
    s.check(f"after {writer}", s.product)
