"""Attention over a shared prompt on a GPU: scores of any size that 32 bits hold."""

import pytest
import torch

from kempnerforge_b200.ops import functional as F
from tests.test_shared_prefix import NAN

pytestmark = pytest.mark.gpu


def far_apart(b, w, p, s, h, hkv, hd, exponent, lens=None):
    """Keys are whole multiples of one direction and queries powers of two of it, so every score is exact, and one key is ahead by a fifth:
    its value is the result, to the last bit."""
    g = torch.Generator().manual_seed(p + s + h)
    sign = torch.where(torch.rand(hd, generator=g) < 0.5, -1.0, 1.0)
    c = torch.where(torch.rand(b, w, h, generator=g) < 0.5, -1.0, 1.0) * 2.0**exponent
    many, few = torch.randint(-200, 201, (b, p, hkv), generator=g).float(), torch.randint(-200, 201, (b, w, s, hkv), generator=g).float()
    v, ov = torch.randn(b, p, hkv, hd, generator=g).bfloat16(), torch.randn(b, w, s, hkv, hd, generator=g).bfloat16()
    want = torch.empty(b, w, h, hd, dtype=torch.bfloat16)
    for i in range(b):
        n = p if lens is None else lens[i]
        for kv in range(hkv):
            ahead = {1: None, -1: None}   # which position of the prompt is ahead for queries of either sign
            if n > 1:
                at = torch.randperm(n, generator=g)[:2].tolist()
                ahead = {1: at[0], -1: at[1]}
                many[i, at[0], kv], many[i, at[1], kv] = 250.0, -250.0
            for j in range(w):
                own = {1: None, -1: None}
                if s > 1 and (n < 2 or (i + j + kv) % 2):   # one of its own is further ahead
                    at = torch.randperm(s, generator=g)[:2].tolist()
                    own = {1: at[0], -1: at[1]}
                    few[i, j, at[0], kv], few[i, j, at[1], kv] = 256.0, -256.0
                for x in range(kv * (h // hkv), (kv + 1) * (h // hkv)):
                    d = int(torch.sign(c[i, j, x]))
                    want[i, j, x] = ov[i, j, own[d], kv] if own[d] is not None else v[i, ahead[d], kv]
    q, k, ok = (t[..., None] * sign for t in (c, many, few))
    return [t.bfloat16().cuda() for t in (q, k, v, ok, ov)], want.cuda()


SIZES = [(1, 2, 100, 5, 4, 2, 64, None), (2, 5, 300, 40, 8, 2, 128, None), (3, 3, 260, 20, 4, 4, 64, [260, 129, 0]), (2, 40, 600, 130, 8, 2, 128, [600, 77])]


@pytest.mark.parametrize("b,w,p,s,h,hkv,hd,lens", SIZES)
@pytest.mark.parametrize("exponent,scale", [(12, None), (24, None), (30, None), (36, None), (60, None), (100, None), (0, 2.0**24), (0, 2.0**40), (0, 2.0**100)])
def test_scores_of_any_size(native_lib, b, w, p, s, h, hkv, hd, lens, exponent, scale):
    args, want = far_apart(b, w, p, s, h, hkv, hd, exponent, lens)
    if lens is not None:
        for i, n in enumerate(lens):
            args[1][i, n:], args[2][i, n:] = NAN, float("inf")
        lens = torch.tensor(lens, device="cuda", dtype=torch.int32)
    before = native_lib.LAUNCH_COUNT
    assert torch.equal(F.shared_prefix_attention(*args, lens, scale=scale), want)
    assert native_lib.LAUNCH_COUNT > before
    for direct in (0, 1):
        assert torch.equal(native_lib.shared_prefix_attn(*args, lens, None, hd**-0.5 if scale is None else scale, direct), want)


# many tiles a CTA in many registers, and two row tiles that share the keys
@pytest.mark.parametrize("b,w,p,s,h,hkv,hd", [(1, 2, 40_001, 140, 8, 8, 128), (1, 17, 43_011, 5, 64, 8, 128)])
@pytest.mark.parametrize("exponent", [24, 33, 90])
def test_scores_of_any_size_in_other_forms(native_lib, b, w, p, s, h, hkv, hd, exponent):
    args, want = far_apart(b, w, p, s, h, hkv, hd, exponent)
    assert torch.equal(F.shared_prefix_attention(*args), want)
    assert native_lib.read_status() == 0
