"""Attention over a shared prompt, derivatives of the formulas: what is hidden has none, and none come from what it holds."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from kempnerforge_b200.ops import functional as F
from tests.test_shared_prefix import NAN, make

LENS = [4, 0]
ROWS = [[0, 0, 0, 0], [0, 1, 1, 255], [0, 0, 7, 0]]


def inputs(fill):
    q, k, v, ok, ov, _, _ = make(2, 3, 6, 4, 4, 2, 8, dtype=torch.float64)
    lens, rows = torch.tensor(LENS), torch.tensor(ROWS, dtype=torch.uint8).repeat(2, 1, 1)
    rows[1, 2] = 255
    for t in (k, v):
        t[0, 4:] = fill
        t[1] = fill
    for t in (ok, ov):
        t[:, 2] = fill
    return [q, k, v, ok, ov], lens, rows


@pytest.mark.parametrize("fill", [NAN, float("inf")])
def test_gradients_next_to_anything(fill):
    grads = []
    for x in (0.0, fill):
        args, lens, rows = inputs(x)
        leaves = [t.requires_grad_() for t in args]
        out = F.shared_prefix_attention(*leaves, lens, rows)
        (out * torch.linspace(-1, 1, out.numel(), dtype=out.dtype).view_as(out)).sum().backward()
        grads.append([t.grad for t in leaves])
    for want, got in zip(*grads):
        assert torch.isfinite(got).all() and torch.allclose(got, want, rtol=1e-12, atol=1e-14)
    for g in grads[1][1:3]:
        assert (g[0, 4:] == 0).all() and (g[1] == 0).all()
    for g in grads[1][3:]:
        assert (g[:, 2] == 0).all()


def test_tangents_next_to_anything():
    args, lens, rows = inputs(NAN)
    g = torch.Generator().manual_seed(1)
    along = [torch.randn(t.shape, generator=g, dtype=t.dtype) for t in args]
    with fwd.dual_level():
        out = F.shared_prefix_attention(*(fwd.make_dual(t, d) for t, d in zip(args, along)), lens, rows)
        got = fwd.unpack_dual(out).tangent
    step = 1e-6
    up, down = (F.shared_prefix_attention(*(t + s * d for t, d in zip(args, along)), lens, rows) for s in (step, -step))
    want = (up - down) / (2 * step)
    assert torch.isfinite(got).all() and torch.allclose(got, want, rtol=1e-6, atol=1e-7)
