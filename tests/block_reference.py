"""Plain 64-bit evaluations of the transformer-block operators for the tests, with elementwise error bounds.

Bounds come from the arithmetic of the kernels: r = half a step of the output's type, products accumulated in fp32 (unit 2^-24,
doubled twice for the tensor cores, whose accumulators do not round to nearest), and for bf16 the probabilities and score
gradients rounded to bf16 (half a step 2^-8) before they are multiplied.
"""
import math

import torch

F8 = torch.float64
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
ACC = 2.0 ** -22


def visible(b, nq, nk, causal, prefix, key_len, q_start, q_docs, k_docs, device):
    pos = torch.arange(nq, device=device)[None, :, None] + (q_start.long()[:, None, None] if q_start is not None else nk - nq)
    key = torch.arange(nk, device=device)[None, None, :]
    seen = torch.ones(b, nq, nk, dtype=torch.bool, device=device)
    if causal:
        reach = key <= pos
        if prefix is not None:
            reach = reach | (key < prefix[:, None, None])
        seen = seen & reach
    if key_len is not None:
        seen = seen & (key < key_len[:, None, None])
    if q_docs is not None:
        seen = seen & (q_docs[:, :, None] == k_docs[:, None, :])
    return seen, (pos - key).abs().expand(b, nq, nk)


class Attention:
    """Everything about one call, [batch, heads, query, key] in 64 bits."""

    def __init__(self, q, k, v, scale=None, causal=False, cap=0.0, slopes=None, q_docs=None, k_docs=None, prefix=None, key_len=None, q_start=None):
        b, nq, h, d = q.shape
        nk, hk = k.shape[1], k.shape[2]
        self.type, self.group, self.cap = q.dtype, h // hk, cap
        self.scale = d ** -0.5 if scale is None else scale
        seen, dist = visible(b, nq, nk, causal, prefix, key_len, q_start, q_docs, k_docs, q.device)
        self.seen = seen[:, None].expand(b, h, nq, nk)
        if key_len is not None:                                   # what lies behind key_len is not part of the call
            gone = torch.arange(nk, device=q.device)[None, :] >= key_len[:, None]
            k, v = (x.masked_fill(gone[:, :, None, None], 0) for x in (k, v))
        self.q = q.to(F8).transpose(1, 2)
        self.k, self.v = (x.to(F8).transpose(1, 2).repeat_interleave(self.group, 1) for x in (k, v))
        z = self.q @ self.k.transpose(2, 3) * self.scale
        err = ACC * (d + 4) * (self.q.abs() @ self.k.abs().transpose(2, 3)) * abs(self.scale) + 2.0 ** -22 * z.abs()
        self.dcap = torch.ones_like(z)
        if cap:
            th = torch.tanh(z / cap)
            self.dcap = 1 - th * th
            z = cap * th
            err = err + cap * 2.0 ** -21
        if slopes is not None:
            bias = slopes.to(F8)[None, :, None, None] * dist[:, None].to(F8)
            z = z - bias
            err = err + 2.0 ** -21 * bias.abs()
        self.z = z.masked_fill(~self.seen, -math.inf)
        self.err = torch.where(self.seen, err + 2.0 ** -22 * z.abs(), torch.zeros_like(err)).amax(-1, keepdim=True) if nk else z.new_zeros(b, h, nq, 1)
        self.lse = torch.logsumexp(self.z, -1) if nk else z.new_full((b, h, nq), -math.inf)

    def probabilities(self, lse):
        lse = lse.to(F8)[..., None]
        return torch.where(self.seen, torch.exp(self.z - torch.where(lse == -math.inf, 0.0, lse)), torch.zeros_like(self.z))

    def forward(self):
        """out, bound, lse, bound."""
        p = self.probabilities(self.lse)
        out, size = p @ self.v, p @ self.v.abs()
        r = HALF[self.type]
        inner = (2.0 ** -8 if self.type == torch.bfloat16 else 0.0) + 3 * self.err + (self.z.shape[-1] + 64) * 2.0 ** -24 + 2.0 ** -20
        bound = r * out.abs() * 1.01 + 1.01 * inner * size + 1e-30
        lse_bound = 2 * self.err[..., 0] + (self.z.shape[-1] + 64) * 2.0 ** -24 + 2.0 ** -22 * self.lse.abs().nan_to_num(posinf=0.0) + 2.0 ** -20
        return out.transpose(1, 2), bound.transpose(1, 2), self.lse, lse_bound

    def _shared(self, x):
        b, h, nk, d = x.shape
        return x.view(b, h // self.group, self.group, nk, d).sum(2).transpose(1, 2)

    def backward(self, dout, out, lse):
        """{name: (gradient, bound)} for dq, dk, dv from the `out` and `lse` that the call is given."""
        do, o = dout.to(F8).transpose(1, 2), out.to(F8).transpose(1, 2)
        r, u = HALF[self.type], 2.0 ** -8 if self.type == torch.bfloat16 else 0.0
        d, nq, nk = do.shape[-1], do.shape[2], self.k.shape[2]
        p = self.probabilities(lse)
        # base-2 arithmetic: the exponent's own rounding, 2^-24 of the numbers that are subtracted
        e = self.err + 2.0 ** -22 * lse.to(F8).abs().nan_to_num(posinf=0.0)[..., None] + 2.0 ** -20
        gap = do @ self.v.transpose(2, 3) - (do * o).sum(-1, keepdim=True)
        gap_err = ACC * (d + 4) * (do.abs() @ self.v.abs().transpose(2, 3) + (do * o).abs().sum(-1, keepdim=True))
        dz = p * gap * self.dcap * self.scale
        dz_err = abs(self.scale) * p * (gap_err * self.dcap + gap.abs() * (self.dcap * (2 * e + u) + (2.0 ** -20 + 2 * e / max(self.cap, 1.0) if self.cap else 0.0)))
        got = {}
        for name, w, werr, x, shared in (("dq", dz, dz_err, self.k, False), ("dk", dz.transpose(2, 3), dz_err.transpose(2, 3), self.q, True),
                                         ("dv", p.transpose(2, 3), (p * (2 * e + u)).transpose(2, 3), do, True)):
            value, size = w @ x, (werr + w.abs() * ACC * (max(nq, nk) + 8)) @ x.abs()
            if shared:
                value, size = self._shared(value), self._shared(size)
            else:
                value, size = value.transpose(1, 2), size.transpose(1, 2)
            got[name] = (value, 1.01 * (r * value.abs() + size) + 1e-30)
        return got


def close(name, got, want, bound):
    """Every element within its bound; infinities and NaN in the same places."""
    got = got.to(F8)
    same = (got == want) | ((got - want).abs() <= bound)
    bad = ~same
    if bool(bad.any()):
        i = tuple(int(x) for x in bad.nonzero()[0])
        worst = float(((got - want).abs() / bound).nan_to_num(posinf=1e9).max())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} out of bounds, first at {i}: got {float(got[i])}, want {float(want[i])} "
                             f"+- {float(bound.expand_as(want)[i])}; worst {worst:.3g} bounds")


def mix32(x):
    """The rounding hash on int64 tensors that hold 32 bits."""
    x = x ^ (x >> 16)
    x = (x * 0x7feb352d) & 0xffffffff
    x = x ^ (x >> 15)
    x = (x * 0x846ca68b) & 0xffffffff
    return x ^ (x >> 16)
