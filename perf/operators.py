"""Measured cases of the transformer-block operators: RMS norm with the residual's addition, attention with capped scores,
distance bias, document and prefix masks, and AdamW over many tensors.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once at the end) or, where
``own`` is true, through ormi_b200.ops.  ``exact`` evaluates the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 128          # elements of an optimizer state that share a scale when it is held in 8 bits
E4M3_MAX = 448.0
_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # one decoding step of eight sequences: the smallest call of the norm, in front of an 8-bit product
        dict(name="norm_token", op="norm", direction="forward", type="bf16", rows=8, cols=4096, residual=True, out="e4m3", group=0),
        # a training batch of 16384 tokens, width 4096 (the shape of the softmax / layernorm benchmark)
        dict(name="norm_forward", op="norm", direction="forward", type="bf16", rows=16384, cols=4096, residual=True, out="bf16", group=0),
        # its backward pass: gradient of the stream, of the weight, with the gradient that skips the norm added
        dict(name="norm_backward", op="norm", direction="backward", type="bf16", rows=16384, cols=4096, residual=True, out="bf16", group=0),
        # an odd width in the framework's default type: nothing is aligned
        dict(name="norm_odd", op="norm", direction="forward", type="fp32", rows=3001, cols=1111, residual=True, out="fp32", group=0),
        # training on packed documents, q / k / v as slices of one product, heads shared four to one
        dict(name="attn_packed", op="attention", direction="forward", type="bf16", batch=2, q_len=4096, k_len=4096, heads=16,
             kv_heads=4, head_dim=128, causal=True, cap=0.0, bias=False, docs=6, prefix=False, ragged=False, packed=True),
        # its backward pass, with capped scores
        dict(name="attn_packed_backward", op="attention", direction="backward", type="bf16", batch=2, q_len=4096, k_len=4096, heads=16,
             kv_heads=4, head_dim=128, causal=True, cap=30.0, bias=False, docs=6, prefix=False, ragged=False, packed=True),
        # one long sequence with distance bias: the largest product
        dict(name="attn_long", op="attention", direction="forward", type="bf16", batch=1, q_len=8192, k_len=8192, heads=16,
             kv_heads=16, head_dim=128, causal=True, cap=0.0, bias=True, docs=0, prefix=False, ragged=False, packed=False),
        # odd lengths and head size in the default type, a prefix seen by everybody, both directions' gradients
        dict(name="attn_odd_backward", op="attention", direction="backward", type="fp32", batch=2, q_len=333, k_len=333, heads=4,
             kv_heads=2, head_dim=40, causal=True, cap=20.0, bias=False, docs=0, prefix=True, ragged=False, packed=False),
        # serving: one new token of 32 sequences over a padded cache
        dict(name="attn_decode", op="attention", direction="forward", type="bf16", batch=32, q_len=1, k_len=8192, heads=32,
             kv_heads=8, head_dim=128, causal=True, cap=50.0, bias=False, docs=0, prefix=False, ragged=True, packed=False),
        # the parameters of a 2048 x 8192 MLP with the bf16 copies that its products read
        dict(name="adamw_mlp", op="adamw", states=32, grads="fp32", width=2048, hidden=8192, layers=1, copies=True),
        # four of them with the states in 8 bits
        dict(name="adamw_8bit", op="adamw", states=8, grads="fp32", width=2048, hidden=8192, layers=4, copies=False),
        # many small tensors: the launches cost more than the data
        dict(name="adamw_small", op="adamw", states=32, grads="bf16", width=68, hidden=260, layers=12, copies=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "attention", "attention", "adamw"])
    if op == "norm":
        cols = _log_int(rng, 64, 12000)
        if rng.random() < 0.6:
            cols = (cols + 15) // 16 * 16
        t = rng.choice(["bf16", "fp32"])
        direction = rng.choice(["forward", "backward"])
        out = rng.choice([t, "e4m3"]) if direction == "forward" else t
        return dict(op=op, direction=direction, type=t, rows=_log_int(rng, 1, max(2, min(16384, 60_000_000 // cols))), cols=cols,
                    residual=rng.random() < 0.7, out=out, group=rng.choice([0, 128]) if out == "e4m3" else 0)
    if op == "adamw":
        width = _log_int(rng, 16, 2048)
        return dict(op=op, states=rng.choice([32, 8]), grads=rng.choice(["fp32", "bf16"]), width=width, hidden=width * rng.choice([2, 3, 4]) + rng.choice([0, 0, 7]),
                    layers=rng.randint(1, 3), copies=rng.random() < 0.5)
    kind = rng.choice(["train", "train", "serve"])
    group = rng.choice([1, 2, 4, 8])
    kv_heads = rng.choice([1, 2, 4])
    t = rng.choice(["bf16", "bf16", "fp32"])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128] if t == "bf16" else [24, 64, 100, 128])
    c = dict(op=op, type=t, heads=kv_heads * group, kv_heads=kv_heads, head_dim=dim, cap=rng.choice([0.0, 0.0, 15.0, 50.0]),
             bias=rng.random() < 0.3)
    if kind == "serve":
        q_len, k_len = rng.choice([1, 1, 1, 2, 5]), _log_int(rng, 16, 16384)
        return dict(c, direction="forward", batch=rng.randint(1, 16), q_len=q_len, k_len=max(k_len, q_len), causal=True, docs=0, prefix=False,
                    ragged=rng.random() < 0.6, packed=False)
    most = 3000 if t == "bf16" else 900
    n = _log_int(rng, 40, most)
    return dict(c, direction=rng.choice(["forward", "backward"]), batch=rng.randint(1, 3), q_len=n, k_len=n, causal=rng.random() < 0.75,
                docs=rng.choice([0, 0, 3, 7]), prefix=rng.random() < 0.3, ragged=rng.random() < 0.3, packed=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs

def _bounds(case):
    """What the masks of an attention case are made of, as host arrays: first positions, lengths, prefixes, document ids."""
    b, nq, nk = case["batch"], case["q_len"], case["k_len"]
    length = np.full(b, nk)
    if case["ragged"]:
        length = np.array([max(nq, nk - (nk * 3 // 4) * ((5 * i + 2) % b) // max(1, b)) for i in range(b)])
    start = np.array(length - nq) if nq < nk else np.zeros(b, dtype=np.int64)
    prefix = np.array([(nk // 5 + 3 * i) % (nk + 1) for i in range(b)]) if case["prefix"] else np.zeros(b, dtype=np.int64)
    docs = np.zeros((b, nk), dtype=np.int64)
    if case["docs"]:
        cuts = [int(nk * ((i + 1) / case["docs"]) ** 1.5) for i in range(case["docs"] - 1)]
        for i in range(b):
            docs[i] = np.searchsorted(np.array(cuts), np.arange(nk) - 2 * i, side="right")
    return start, length, prefix, docs


def _pairs(case):
    """Visible (query, key) pairs of one head, over the whole batch."""
    start, length, prefix, docs = _bounds(case)
    total = 0
    for b in range(case["batch"]):
        pos = start[b] + np.arange(case["q_len"])
        reach = np.maximum(pos + 1, prefix[b]) if case["causal"] else np.full(case["q_len"], case["k_len"])
        first, last = np.zeros_like(pos), np.full_like(pos, case["k_len"])
        if case["docs"]:
            first = np.searchsorted(docs[b], docs[b][pos], side="left")
            last = np.searchsorted(docs[b], docs[b][pos], side="right")
        total += int(np.maximum(0, np.minimum(np.minimum(last, length[b]), reach) - first).sum())
    return total


def _sizes(case):
    """Element counts of the optimizer's tensors: per layer two matrices and two biases."""
    w, h = case["width"], case["hidden"]
    return [w * h, h, h * w, w] * case["layers"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1 + seed)
    dt = _TYPES.get(case.get("type"), torch.float32)

    def normal(*shape, scale=1.0, dtype=None):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype or dt)

    s = {"case": case}
    if case["op"] == "norm":
        n, c = case["rows"], case["cols"]
        s["eps"] = 1e-6
        s["weight"] = (1 + 0.2 * torch.randn(c, generator=g, device="cuda")).to(dt)
        if case["direction"] == "forward":
            s["x"] = normal(n, c)
            s["residual"] = normal(n, c, scale=3.0) if case["residual"] else None
            s["out"] = torch.empty(n, c, device="cuda", dtype=_TYPES[case["out"]])
            s["stream"] = torch.empty(n, c, device="cuda", dtype=dt) if case["residual"] else None
            s["rstd"] = torch.empty(n, device="cuda")
            groups = 1 if not case["group"] else -(-c // case["group"])
            s["scales"] = torch.empty(n, groups, device="cuda") if case["out"] == "e4m3" else None
        else:
            s["stream"] = normal(n, c, scale=3.0)
            s["rstd"] = torch.rsqrt(s["stream"].float().square().mean(-1) + s["eps"])
            s["dout"] = normal(n, c)
            s["dstream"] = normal(n, c) if case["residual"] else None
            s["dx"] = torch.empty(n, c, device="cuda", dtype=dt)
            s["dweight"] = torch.empty(c, device="cuda", dtype=dt)
    elif case["op"] == "attention":
        b, nq, nk, h, hk, d = (case[k] for k in ("batch", "q_len", "k_len", "heads", "kv_heads", "head_dim"))
        if case["packed"]:
            joint = normal(b, nq, h + 2 * hk, d)
            s["q"], s["k"], s["v"] = joint[:, :, :h], joint[:, :, h:h + hk], joint[:, :, h + hk:]
        else:
            s["q"] = normal(b, nq, h, d)
            s["k"], s["v"] = (normal(b, hk, nk, d).transpose(1, 2) for _ in range(2))
        start, length, prefix, docs = _bounds(case)
        ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        s["scale"] = 1.0 / math.sqrt(d)
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, h + 1, device="cuda").float() / h) if case["bias"] else None
        s["q_start"] = ints(start) if nq < nk else None
        s["key_len"] = ints(length) if case["ragged"] else None
        s["prefix"] = ints(prefix) if case["prefix"] else None
        s["docs"] = ints(docs) if case["docs"] else None
        if case["direction"] == "forward":
            s["out"] = torch.empty(b, nq, h, d, device="cuda", dtype=dt)
            s["lse"] = torch.empty(b, h, nq, device="cuda")
        else:
            s["out"], s["lse"] = _attention(s)
            s["dout"] = normal(b, nq, h, d)
            s["dq"] = torch.empty(b, nq, h, d, device="cuda", dtype=dt)
            s["dk"], s["dv"] = (torch.empty(b, nk, hk, d, device="cuda", dtype=dt) for _ in range(2))
    else:
        sizes = _sizes(case)
        room = [-(-n // BLOCK) * BLOCK for n in sizes]
        total = sum(room)
        # every tensor starts on a whole block of one flat buffer; what lies behind its end is zero
        at = torch.arange(total, device="cuda")
        starts = torch.tensor(np.concatenate([[0], np.cumsum(room)[:-1]]), device="cuda")
        which = torch.repeat_interleave(torch.arange(len(room), device="cuda"), torch.tensor(room, device="cuda"))
        live = (at - starts[which]) < torch.tensor(sizes, device="cuda")[which]
        del at, which
        s["sizes"], s["room"] = sizes, room
        s["p"] = normal(total, scale=0.02, dtype=torch.float32) * live
        s["grad"] = (normal(total, scale=1e-3, dtype=torch.float32) * live).to(_TYPES[case["grads"]])
        m, r = normal(total, scale=3e-4, dtype=torch.float32) * live, (normal(total, scale=1e-3, dtype=torch.float32) * live).abs() + 1e-4 * live
        if case["states"] == 8:
            s["m_scale"], s["r_scale"] = (x.view(-1, BLOCK).abs().amax(1) / E4M3_MAX for x in (m, r))
            s["m"], s["r"] = ((x.view(-1, BLOCK) / y[:, None].clamp_min(1e-30)).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(-1)
                              for x, y in ((m, s["m_scale"]), (r, s["r_scale"])))
        else:
            s["m"], s["v"] = m, r * r
        s["copy"] = s["p"].to(torch.bfloat16) if case["copies"] else None
        s["decay"] = [0.1 if n == case["width"] * case["hidden"] else 0.0 for n in sizes]
        s.update(lr=3e-4, betas=(0.9, 0.95), eps=1e-8, grad_scale=torch.full((1,), 0.5, device="cuda"), step=100 + seed % 50, seed=seed & 0xffff, handle=None)
    return s


# ------------------------------------------------------------------------------------------------ plain forms

def _norm_forward(s):
    case = s["case"]
    x = s["x"].float()
    if s["residual"] is not None:
        x = (x + s["residual"].float()).to(s["x"].dtype).float()
    rstd = torch.rsqrt((x * x).mean(-1) + s["eps"])
    y = x * rstd[:, None] * s["weight"].float()
    got = {"rstd": rstd}
    if s["residual"] is not None:
        got["stream"] = x.to(s["x"].dtype)
    if case["out"] == "e4m3":
        n, c = y.shape
        width = case["group"] or c
        groups = -(-c // width)
        z = torch.nn.functional.pad(y, (0, groups * width - c)).view(n, groups, width)
        top = z.abs().amax(-1)
        up = torch.where(top > 0, E4M3_MAX / top, torch.zeros_like(top))
        got["scales"] = top / E4M3_MAX
        got["out"] = (z * up[..., None]).clamp(-E4M3_MAX, E4M3_MAX).reshape(n, -1)[:, :c].to(torch.float8_e4m3fn)
    else:
        got["out"] = y.to(_TYPES[case["out"]])
    return got


def _norm_backward(s):
    x, dy, rstd = s["stream"].float(), s["dout"].float(), s["rstd"][:, None]
    dyw = dy * s["weight"].float()
    c = (dyw * x).mean(-1, keepdim=True) * rstd * rstd
    dx = rstd * (dyw - x * c)
    if s["dstream"] is not None:
        dx = dx + s["dstream"].float()
    return {"dx": dx.to(s["stream"].dtype), "dweight": (dy * x * rstd).sum(0).to(s["weight"].dtype)}


def _scores(s):
    """Scores before and after the bias and the mask, [batch, kv head, head of the group, query, key]."""
    case = s["case"]
    b, nq, nk, h, hk, d = (case[k] for k in ("batch", "q_len", "k_len", "heads", "kv_heads", "head_dim"))
    q = (s["q"].float() * s["scale"]).permute(0, 2, 1, 3).reshape(b, hk, h // hk, nq, d)
    k = s["k"].float().permute(0, 2, 3, 1).reshape(b, hk, 1, d, nk)
    z = q @ k
    if case["cap"]:
        z = case["cap"] * torch.tanh(z / case["cap"])
    pos = torch.arange(nq, device="cuda")[None, :, None] + (s["q_start"].long()[:, None, None] if s["q_start"] is not None else 0)
    key = torch.arange(nk, device="cuda")[None, None, :]
    seen = torch.ones(b, nq, nk, dtype=torch.bool, device="cuda")
    if case["causal"]:
        reach = key <= pos
        if s["prefix"] is not None:
            reach = reach | (key < s["prefix"][:, None, None])
        seen = seen & reach
    if s["key_len"] is not None:
        seen = seen & (key < s["key_len"][:, None, None])
    if s["docs"] is not None:
        seen = seen & (s["docs"][:, :, None] == s["docs"][:, None, :])
    biased = z
    if s["slopes"] is not None:
        biased = z - s["slopes"].view(1, hk, h // hk, 1, 1) * (pos - key).abs().float()[:, None, None]
    return z, biased.masked_fill(~seen[:, None, None], -math.inf)


def _attention(s):
    case = s["case"]
    b, nq, h, d = (case[k] for k in ("batch", "q_len", "heads", "head_dim"))
    z = _scores(s)[1]
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(z - top)
    total = p.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).reshape(b, h, nq)
    v = s["v"].float().permute(0, 2, 1, 3)[:, :, None]
    out = (p @ v) / torch.where(total > 0, total, torch.ones_like(total))
    return out.reshape(b, h, nq, d).permute(0, 2, 1, 3).contiguous().to(s["q"].dtype), lse


def _attention_backward(s):
    case = s["case"]
    b, nq, nk, h, hk, d = (case[k] for k in ("batch", "q_len", "k_len", "heads", "kv_heads", "head_dim"))
    capped, z = _scores(s)
    lse = s["lse"].view(b, hk, h // hk, nq, 1)
    p = torch.where(z > -math.inf, torch.exp(z - lse), torch.zeros_like(z))
    q, do, o = (s[n].float().permute(0, 2, 1, 3).reshape(b, hk, h // hk, nq, d) for n in ("q", "dout", "out"))
    k, v = (s[n].float().permute(0, 2, 1, 3)[:, :, None] for n in ("k", "v"))
    dv = (p.transpose(-1, -2) @ do).sum(2)
    dz = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
    if case["cap"]:
        dz = dz * (1 - (capped / case["cap"]) ** 2)
    dq = (dz @ k) * s["scale"]
    dk = (dz.transpose(-1, -2) @ q).sum(2) * s["scale"]
    t = s["q"].dtype
    return {"dq": dq.reshape(b, h, nq, d).permute(0, 2, 1, 3).to(t), "dk": dk.permute(0, 2, 1, 3).to(t), "dv": dv.permute(0, 2, 1, 3).to(t)}


def _mix(x):
    """A 32-bit integer hash (two rounds of xor-shift and multiply), on int64 tensors or numbers that hold 32 bits."""
    x = x ^ (x >> 16)
    x = (x * 0x7feb352d) & 0xffffffff
    x = x ^ (x >> 15)
    x = (x * 0x846ca68b) & 0xffffffff
    return x ^ (x >> 16)


def _to_e4m3(x, u):
    """|x| <= 448 rounded to an e4m3 value, up with the probability of what it is above the value below (u in [0, 1))."""
    a = x.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6)))) / 8
    step = torch.where(a < step * 8, step / 2, step).clamp_min(2.0 ** -9)      # log2 next to a power of two may be rounded up
    return torch.copysign(torch.floor(a / step + u) * step, x).clamp(-E4M3_MAX, E4M3_MAX)


def _adamw(s):
    b1, b2 = s["betas"]
    t = s["step"]
    n = s["p"].numel()
    room = torch.tensor(s["room"], device="cuda")
    g = s["grad"].float() * s["grad_scale"]
    if s["case"]["states"] == 8:
        m = (s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        v = (s["r"].float().view(-1, BLOCK) * s["r_scale"][:, None]).view(-1).square()
    else:
        m, v = s["m"], s["v"]
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    rate = s["lr"] * torch.repeat_interleave(torch.tensor(s["decay"], device="cuda"), room)
    s["p"].sub_(rate * s["p"] + s["lr"] * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + s["eps"]))
    if s["case"]["states"] == 8:
        which = torch.repeat_interleave(torch.arange(len(s["room"]), device="cuda"), room)
        first = (torch.cumsum(room, 0) - room)[which]
        h = _mix((torch.arange(n, device="cuda") - first) ^ _mix((_mix(s["seed"] ^ t) + which) & 0xffffffff))
        del which, first
        r = torch.sqrt(v)
        tops = [x.view(-1, BLOCK).abs().amax(1) for x in (m, r)]
        ups = [torch.where(x > 0, E4M3_MAX / x, torch.zeros_like(x))[:, None] for x in tops]
        a = (m.view(-1, BLOCK) * ups[0]).clamp(-E4M3_MAX, E4M3_MAX).view(-1)
        s["m"].copy_(_to_e4m3(a, (h & 0xffff).float() / 65536))
        a = (r.view(-1, BLOCK) * ups[1]).clamp(0, E4M3_MAX).view(-1)
        a = torch.where(r > 0, a.clamp_min(2.0 ** -9), a)
        s["r"].copy_(_to_e4m3(a, (h >> 16).float() / 65536))
        s["m_scale"].copy_(tops[0] / E4M3_MAX)
        s["r_scale"].copy_(tops[1] / E4M3_MAX)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    if s["copy"] is not None:
        s["copy"].copy_(s["p"])


# ------------------------------------------------------------------------------------------------ the framework's operators

_device = None


def _dev():
    global _device
    if _device is None:
        from ormi_b200.runtime import Device
        _device = Device(torch.cuda.current_device())
    return _device


def _masks(s):
    return dict(scale=s["scale"], causal=s["case"]["causal"], cap=s["case"]["cap"], slopes=s["slopes"], q_docs=s["docs"], k_docs=s["docs"],
                prefix=s["prefix"], key_len=s["key_len"], q_start=s["q_start"])


def _optimizer(s):
    """The optimizer object over the slices of the flat buffers, as a program makes it once."""
    from ormi_b200 import ops
    cut = lambda x: [y[:n] for y, n in zip(torch.split(x, s["room"]), s["sizes"])]  # noqa: E731
    more = {}
    if s["case"]["states"] == 8:
        blocks = [n // BLOCK for n in s["room"]]
        more = dict(m_scales=list(torch.split(s["m_scale"], blocks)), v_scales=list(torch.split(s["r_scale"], blocks)))
    return ops.AdamW(_dev(), cut(s["p"]), cut(s["grad"]), cut(s["m"]), cut(s["r"] if more else s["v"]), weight_decay=s["decay"], betas=s["betas"],
                     eps=s["eps"], copies=cut(s["copy"]) if s["copy"] is not None else None, seed=s["seed"], **more)


def _run_own(s):
    from ormi_b200 import ops
    case = s["case"]
    if case["op"] == "norm" and case["direction"] == "forward":
        ops.rmsnorm(_dev(), s["x"], s["weight"], s["out"], residual=s["residual"], residual_out=s["stream"], rstd=s["rstd"], scales=s["scales"],
                    group=case["group"], eps=s["eps"])
    elif case["op"] == "norm":
        ops.rmsnorm_backward(_dev(), s["dout"], s["stream"], s["weight"], s["rstd"], s["dx"], s["dweight"], dresidual=s["dstream"])
    elif case["op"] == "attention" and case["direction"] == "forward":
        ops.attention(_dev(), s["q"], s["k"], s["v"], s["out"], s["lse"], **_masks(s))
    elif case["op"] == "attention":
        ops.attention_backward(_dev(), s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], s["dq"], s["dk"], s["dv"], **_masks(s))
    else:
        if s["handle"] is None:
            s["handle"] = _optimizer(s)
        s["handle"].step(lr=s["lr"], step=s["step"], grad_scale=s["grad_scale"])
    return _outputs(s)


def _outputs(s):
    """The buffers of the state that an operator writes."""
    case = s["case"]
    if case["op"] == "adamw":
        names = ["p", "m", "r", "m_scale", "r_scale"] if case["states"] == 8 else ["p", "m", "v"]
        names += ["copy"] if s["copy"] is not None else []
    elif case["op"] == "norm":
        names = ["out", "rstd", "stream", "scales"] if case["direction"] == "forward" else ["dx", "dweight"]
    else:
        names = ["out", "lse"] if case["direction"] == "forward" else ["dq", "dk", "dv"]
    return {n: s[n] for n in names if s[n] is not None}


def run(s):
    case = s["case"]
    if own:
        return _run_own(s)
    if case["op"] == "norm":
        return _norm_forward(s) if case["direction"] == "forward" else _norm_backward(s)
    if case["op"] == "attention":
        if case["direction"] == "backward":
            return _attention_backward(s)
        out, lse = _attention(s)
        return {"out": out, "lse": lse}
    _adamw(s)
    return _outputs(s)


# ------------------------------------------------------------------------------------------------ work

def work(case):
    size = {"fp32": 4, "bf16": 2, "e4m3": 1}
    if case["op"] == "norm":
        n, c, w = case["rows"], case["cols"], size[case["type"]]
        if case["direction"] == "forward":
            groups = 0 if case["out"] != "e4m3" else 1 if not case["group"] else -(-c // case["group"])
            return {"bytes": n * c * (w * (3 if case["residual"] else 1) + size[case["out"]]) + c * w + 4 * n * (1 + groups), "flops": 5 * n * c}
        return {"bytes": n * c * w * (4 if case["residual"] else 3) + 2 * c * w + 4 * n, "flops": 9 * n * c}
    if case["op"] == "attention":
        b, nq, nk, h, hk, d = (case[k] for k in ("batch", "q_len", "k_len", "heads", "kv_heads", "head_dim"))
        w = size[case["type"]]
        keys = int(_bounds(case)[1].sum())                         # key positions that some query may see
        pairs = _pairs(case) * h
        if case["direction"] == "forward":
            return {"bytes": w * d * (2 * b * nq * h + 2 * keys * hk) + 4 * b * h * nq, "flops": 4 * d * pairs}
        # q, out, dout in, dq out; k, v in; dk, dv out; the five products of the backward pass
        return {"bytes": w * d * (4 * b * nq * h + 2 * keys * hk + 2 * b * nk * hk) + 4 * b * h * nq, "flops": 10 * d * pairs}
    n = sum(_sizes(case))
    each = 8 + size[case["grads"]] + (16 if case["states"] == 32 else 4 + 16 / BLOCK) + (2 if case["copies"] else 0)
    return {"bytes": int(n * each), "flops": 14 * n}


# ------------------------------------------------------------------------------------------------ 64 bits

def _exact_norm(s):
    f8 = torch.float64
    w = s["weight"].to(f8)
    if s["case"]["direction"] == "backward":
        x, dy, inv = s["stream"].to(f8), s["dout"].to(f8), s["rstd"].to(f8).unsqueeze(1)
        xh = x * inv
        gw = dy * w
        dx = (gw - xh * (gw * xh).mean(1, keepdim=True)) * inv
        return {"dx": dx if s["dstream"] is None else dx + s["dstream"].to(f8), "dweight": torch.einsum("nc,nc->c", dy, xh)}
    # the stream is rounded to its type before it is normalised: that rounding is part of the definition
    x = s["x"].to(f8) if s["residual"] is None else (s["x"].to(f8) + s["residual"].to(f8)).to(s["x"].dtype).to(f8)
    inv = 1.0 / torch.sqrt(torch.linalg.vector_norm(x, dim=1) ** 2 / x.shape[1] + s["eps"])
    y = x * (inv.unsqueeze(1) * w)
    got = {"rstd": inv, "out": y}
    if s["residual"] is not None:
        got["stream"] = x
    if s["scales"] is not None:
        parts = y.split(s["case"]["group"] or y.shape[1], dim=1)
        got["scales"] = torch.stack([p.abs().max(dim=1).values / E4M3_MAX for p in parts], 1)
        got["out"] = None
    return got


def _exact_attention(s):
    case = s["case"]
    f8 = torch.float64
    b, nq, nk, h, hk = (case[k] for k in ("batch", "q_len", "k_len", "heads", "kv_heads"))
    per = h // hk
    j = torch.arange(nk, device="cuda")
    made = {}
    for i in range(b):
        at = torch.arange(nq, device="cuda") + (int(s["q_start"][i]) if s["q_start"] is not None else 0)
        hidden = torch.zeros(nq, nk, dtype=torch.bool, device="cuda")
        if case["causal"]:
            last = at if s["prefix"] is None else torch.clamp(at, min=int(s["prefix"][i]) - 1)
            hidden |= j.unsqueeze(0) > last.unsqueeze(1)
        if s["key_len"] is not None:
            hidden[:, int(s["key_len"][i]):] = True
        if s["docs"] is not None:
            hidden |= s["docs"][i].unsqueeze(0) != s["docs"][i].unsqueeze(1)
        distance = (at.unsqueeze(1) - j.unsqueeze(0)).abs().to(f8)
        rows = []
        dks = torch.zeros(2, hk, nk, case["head_dim"], dtype=f8, device="cuda")
        for n in range(h):
            q, k, v = s["q"][i, :, n].to(f8), s["k"][i, :, n // per].to(f8), s["v"][i, :, n // per].to(f8)
            z = torch.mm(q, k.T) * s["scale"]
            slope = 1.0
            if case["cap"]:
                th = torch.tanh(z / case["cap"])
                z, slope = th * case["cap"], 1.0 - th * th
            if s["slopes"] is not None:
                z = z - distance * s["slopes"][n].to(f8)
            z[hidden] = -math.inf
            if case["direction"] == "forward":
                lse = torch.logsumexp(z, 1)
                p = torch.exp(z - torch.where(lse == -math.inf, 0.0, lse).unsqueeze(1))
                rows.append((torch.mm(p, v), lse))
                continue
            lse, do, o = s["lse"][i, n].to(f8), s["dout"][i, :, n].to(f8), s["out"][i, :, n].to(f8)
            p = torch.exp(z - torch.where(lse == -math.inf, 0.0, lse).unsqueeze(1))
            dz = p * (torch.mm(do, v.T) - torch.einsum("qd,qd->q", do, o).unsqueeze(1)) * slope * s["scale"]
            rows.append((torch.mm(dz, k),))
            dks[0, n // per] += torch.mm(dz.T, q)
            dks[1, n // per] += torch.mm(p.T, do)
        if case["direction"] == "forward":
            made.setdefault("out", []).append(torch.stack([r[0] for r in rows], 1))
            made.setdefault("lse", []).append(torch.stack([r[1] for r in rows]))
        else:
            made.setdefault("dq", []).append(torch.stack([r[0] for r in rows], 1))
            made.setdefault("dk", []).append(dks[0].transpose(0, 1))
            made.setdefault("dv", []).append(dks[1].transpose(0, 1))
    return {k: torch.stack(v) for k, v in made.items()}


def _exact_adamw(s):
    f8 = torch.float64
    b1, b2 = s["betas"]
    eight = s["case"]["states"] == 8
    got = {"p": [], "m": [], "v": [], "m_scale": [], "r_scale": []}
    at = 0
    for room, decay in zip(s["room"], s["decay"]):
        cut = slice(at, at + room)
        blocks = slice(at // BLOCK, (at + room) // BLOCK)
        at += room
        p, g = s["p"][cut].to(f8), s["grad"][cut].to(f8) * s["grad_scale"].to(f8)
        m, v = s["m"][cut].to(f8), (s["r"] if eight else s["v"])[cut].to(f8)
        if eight:
            m = m * s["m_scale"][blocks].to(f8).repeat_interleave(BLOCK)
            v = (v * s["r_scale"][blocks].to(f8).repeat_interleave(BLOCK)) ** 2
        m, v = m + (g - m) * (1 - b1), v + (g * g - v) * (1 - b2)
        ahead = m / (1 - math.pow(b1, s["step"]))
        spread = torch.sqrt(v / (1 - math.pow(b2, s["step"]))) + s["eps"]
        got["p"].append(p * (1 - s["lr"] * decay) - s["lr"] * ahead / spread)
        if eight:
            got["m_scale"].append(m.view(-1, BLOCK).abs().max(1).values / E4M3_MAX)
            got["r_scale"].append(v.view(-1, BLOCK).max(1).values.sqrt() / E4M3_MAX)
        else:
            got["m"].append(m)
            got["v"].append(v)
    got = {k: torch.cat(x) if x else None for k, x in got.items()}
    if eight:
        got["m"], got["r"] = None, None
        del got["v"]
    else:
        del got["m_scale"], got["r_scale"]
    if s["copy"] is not None:
        got["copy"] = got["p"]
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "attention": _exact_attention, "adamw": _exact_adamw}[case["op"]](s)
