"""Attention over a shared prompt on a GPU: derivatives in forward mode and batched tensors take the formulas."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from kempnerforge_b200.ops import functional as F
from tests.test_shared_prefix import make
from tests.test_shared_prefix_gpu import near

pytestmark = pytest.mark.gpu


def test_tangents(native_lib):
    args = make(2, 3, 40, 5, 4, 2, 64, torch.bfloat16, table=True, ragged=True, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    along = [torch.randn(t.shape, generator=g, device="cuda").bfloat16() for t in args[:5]]
    with fwd.dual_level():
        got = fwd.unpack_dual(F.shared_prefix_attention(*(fwd.make_dual(t, d) for t, d in zip(args[:5], along)), *args[5:]))
        wide = fwd.unpack_dual(F.shared_prefix_attention(*(fwd.make_dual(t.double(), d.double()) for t, d in zip(args[:5], along)), *args[5:]))
        near(F.shared_prefix_attention(*args), args)
    near(got.primal, args)
    # rounded once to bf16; fp32 in between, of sums of some 45 x 64 products of a few units
    assert got.tangent is not None and ((got.tangent.double() - wide.tangent).abs() <= 2.0**-8 * wide.tangent.abs() + 1e-3).all()
    jvp = torch.func.jvp(lambda q: F.shared_prefix_attention(q, *args[1:]), (args[0],), (along[0],))[1]
    with fwd.dual_level():
        alone = fwd.unpack_dual(F.shared_prefix_attention(fwd.make_dual(args[0], along[0]), *args[1:])).tangent
    assert torch.equal(jvp, alone)


def test_batched_tensors(native_lib):
    sets = [make(2, 3, 40, 5, 4, 2, 64, torch.bfloat16, seed=i, device="cuda") for i in range(3)]
    stacked = [torch.stack(t) for t in list(zip(*sets))[:5]]
    got = torch.vmap(F.shared_prefix_attention)(*stacked)
    for out, args in zip(got, sets):
        near(out, args)
    # some arguments alone
    q = stacked[0]
    got = torch.vmap(lambda x: F.shared_prefix_attention(x, *sets[0][1:5]))(q)
    for i in range(3):
        near(got[i], [q[i], *sets[0][1:5]])
    lens = torch.tensor([[40, 3], [0, 1], [17, 40]], device="cuda")
    got = torch.vmap(lambda n: F.shared_prefix_attention(*sets[0][:5], n))(lens)
    for i in range(3):
        near(got[i], [*sets[0][:5], lens[i]])
    rows = torch.randint(0, 3, (3, 2, 3, 5), device="cuda").to(torch.uint8)
    got = torch.vmap(lambda r: F.shared_prefix_attention(*sets[0][:5], None, r))(rows)
    for i in range(3):
        near(got[i], [*sets[0][:5], None, rows[i]])
    grad = torch.func.grad(lambda x: F.shared_prefix_attention(x, *sets[0][1:5]).float().sum())(q[0])
    leaf = q[0].clone().requires_grad_()
    F.shared_prefix_attention(leaf, *sets[0][1:5]).float().sum().backward()
    assert torch.equal(grad, leaf.grad)
