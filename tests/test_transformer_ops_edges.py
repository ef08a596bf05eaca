"""Transformer-block operators at the edges of what their documentation allows."""
import pytest

from ormi_b200 import ops
from test_transformer_ops import BF, done, gpu, ints, randn, torch


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
