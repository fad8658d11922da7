"""Reordering on a GPU of states with tangents."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from kempnerforge_b200.ops import beam

pytestmark = pytest.mark.gpu

PARENTS = [[2, 0, 0, 3], [1, 0, 3, 2]]


@pytest.mark.parametrize("own", [False, True])
def test_tangents_follow(native_lib, own):
    """No tangent stays with the beam that has gone."""
    parents = torch.tensor(PARENTS, device="cuda")
    at = torch.arange(2, device="cuda")[:, None]
    x, t = torch.randn(2, 4, 6, device="cuda"), torch.randn(2, 4, 6, device="cuda")
    want_x, want_t = x[at, parents], t[at, parents]
    with torch.no_grad(), fwd.dual_level():
        state = fwd.make_dual(x, t)
        out = fwd.make_dual(torch.zeros_like(x), torch.zeros_like(t)) if own else None
        got = fwd.unpack_dual(beam.reorder([state], parents, out=None if out is None else [out])[0])
        assert torch.equal(got.primal, want_x) and torch.equal(got.tangent, want_t)
