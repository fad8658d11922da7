"""Attention of many continuations of one prompt on the CPU: the formulas against a softmax by hand, gradients, and what is refused."""

import math

import pytest
import torch

from kempnerforge_b200.ops import functional as F

NAN = float("nan")


def by_hand(q, k, v, own_k, own_v, lens=None, rows=None, scale=None):
    """(attention, the same of the values' magnitudes) in 64 bits, continuation by continuation and head by head."""
    b, w, h, hd = q.shape
    p, group, s = k.shape[1], h // k.shape[2], own_k.shape[2]
    scale = hd**-0.5 if scale is None else scale
    q, k, v, own_k, own_v = (t.double() for t in (q, k, v, own_k, own_v))
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(b):
        n = p if lens is None else min(max(int(lens[i]), 0), p)
        for j in range(w):
            slots = [j] * s if rows is None else rows[i, j].tolist()
            at = [t for t in range(s) if slots[t] < w]
            own = [slots[t] for t in at]
            keys = torch.cat([k[i, :n], own_k[i, own, at]])
            values = torch.cat([v[i, :n], own_v[i, own, at]])
            if keys.shape[0] == 0:
                continue
            for x in range(h):
                weights = torch.softmax(keys[:, x // group] @ q[i, j, x] * scale, 0)
                out[i, j, x] = weights @ values[:, x // group]
                size[i, j, x] = weights @ values[:, x // group].abs()
    return out, size


def make(b, w, p, s, h, hkv, hd, dtype=torch.float32, table=False, ragged=False, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    q, k, v, ok, ov = (torch.randn(*shape, generator=g).to(dtype) for shape in (
        (b, w, h, hd), (b, p, hkv, hd), (b, p, hkv, hd), (b, w, s, hkv, hd), (b, w, s, hkv, hd)))
    lens = torch.randint(0, p + 1, (b,), generator=g).int() if ragged else None
    rows = torch.randint(0, w, (b, w, s), generator=g).to(torch.uint8) if table else None
    return [None if t is None else t.to(device) for t in (q, k, v, ok, ov, lens, rows)]


@pytest.mark.parametrize("b,w,p,s,h,hkv,hd", [(1, 1, 1, 1, 1, 1, 4), (2, 3, 9, 4, 4, 2, 8), (2, 2, 0, 3, 2, 1, 4), (1, 3, 5, 0, 2, 2, 4), (1, 2, 0, 0, 2, 2, 4)])
@pytest.mark.parametrize("table", [False, True])
@pytest.mark.parametrize("ragged", [False, True])
def test_formulas(b, w, p, s, h, hkv, hd, table, ragged):
    args = make(b, w, p, s, h, hkv, hd, table=table, ragged=ragged)
    want, _ = by_hand(*args)
    got = F.shared_prefix_attention(*args)
    assert got.dtype == torch.float32 and torch.allclose(got.double(), want, rtol=1e-5, atol=1e-5)
    want, _ = by_hand(*args, scale=0.3)
    assert torch.allclose(F.shared_prefix_attention(*args, scale=0.3).double(), want, rtol=1e-5, atol=1e-5)


def test_what_is_hidden_may_hold_anything():
    q, k, v, ok, ov, _, _ = make(2, 3, 6, 4, 4, 2, 8)
    lens = torch.tensor([4, 0])
    rows = torch.tensor([[0, 0, 0, 0], [0, 1, 1, 255], [0, 0, 7, 0]], dtype=torch.uint8).repeat(2, 1, 1)
    rows[1, 2] = 255          # the last continuation of the second prompt sees nothing at all
    for t in (k, v):
        t[0, 4:] = NAN
        t[1] = NAN
    for t in (ok, ov):
        t[:, 2] = NAN         # nobody has the third continuation's cache
    want, _ = by_hand(q, k, v, ok, ov, lens, rows)
    got = F.shared_prefix_attention(q, k, v, ok, ov, lens, rows)
    assert torch.isfinite(got).all() and torch.allclose(got.double(), want, rtol=1e-5, atol=1e-5)
    assert (got[1, 2] == 0).all()


def test_gradients():
    args = make(2, 2, 3, 3, 4, 2, 4, dtype=torch.float64, table=True)
    lens = torch.tensor([3, 2])
    leaves = [t.requires_grad_() for t in args[:5]]
    assert torch.autograd.gradcheck(lambda *a: F.shared_prefix_attention(*a, lens, args[6]), leaves)


def test_refuses():
    q, k, v, ok, ov, lens, rows = make(2, 3, 5, 4, 4, 2, 8, table=True, ragged=True)
    for bad in ((q[0], k, v, ok, ov), (q, k[0], v, ok, ov), (q, k, v, ok[0], ov), (q, k, v[:, :3], ok, ov), (q, k, v, ok, ov[:, :, :2]),
                (q, k[:1], v[:1], ok, ov), (q[..., :4], k, v, ok, ov), (q[:, :, :3], k, v, ok, ov), (q, k, v, ok[:, :2], ov[:, :2]),
                (q, k.double(), v, ok, ov), (q, k, v, ok, ov, lens[:1]), (q, k, v, ok, ov, lens.float()), (q, k, v, ok, ov, lens, rows[:, :2]),
                (q, k, v, ok, ov, lens, rows.int()), (q, k, v, ok, ov, lens, rows, 0.0), (q, k, v, ok, ov, lens, rows, -1.0),
                (q, k, v, ok, ov, lens, rows, math.inf), (q, k, v, ok, ov, lens, rows, NAN)):
        with pytest.raises(ValueError):
            F.shared_prefix_attention(*bad)
