"""Attention over a shared prompt on a GPU: one prompt for a whole batch."""

import pytest
import torch

from kempnerforge_b200.ops import functional as F
from tests.test_shared_prefix import make
from tests.test_shared_prefix_gpu import near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("p,s", [(60, 5), (300, 20), (2000, 20)])
def test_one_prompt_for_a_batch(native_lib, p, s):
    """A prompt that is expanded over the batch is read where it lies."""
    b, w, h, hkv, hd = 6, 3, 8, 2, 128
    q, _, _, ok, ov, _, rows = make(b, w, 1, s, h, hkv, hd, torch.bfloat16, table=True, device="cuda")
    one = [t.expand(b, -1, -1, -1) for t in make(1, 1, p, 1, h, hkv, hd, torch.bfloat16, device="cuda")[1:3]]
    lens = torch.tensor([p, 1, 0, p - 1, p // 2, p], device="cuda", dtype=torch.int32)
    for n in (None, lens):
        got = native_lib.shared_prefix_call(q, *one, ok, ov, n, rows, None)
        assert got is not None
        near(got, (q, *one, ok, ov, n, rows))
        for direct in (0, 1):
            near(native_lib.shared_prefix_attn(q, *one, ok, ov, n, rows, hd**-0.5, direct), (q, *one, ok, ov, n, rows))
        # one of the two alone
        near(F.shared_prefix_attention(q, one[0], one[1].contiguous(), ok, ov, n, rows), (q, *one, ok, ov, n, rows))
        near(F.shared_prefix_attention(q, one[0].contiguous(), one[1], ok, ov, n, rows), (q, *one, ok, ov, n, rows))


def test_one_long_prompt_for_a_batch(native_lib):
    """Two row tiles that share the keys."""
    b, w, p, h, hkv, hd = 3, 40, 14_500, 32, 8, 128
    q, _, _, ok, ov, _, _ = make(b, w, 1, 5, h, hkv, hd, torch.bfloat16, device="cuda")
    one = [torch.randn(1, p, hkv, hd, device="cuda").bfloat16().expand(b, -1, -1, -1) for _ in range(2)]
    got = native_lib.shared_prefix_call(q, *one, ok, ov, None, None, None)
    assert got is not None and torch.equal(got, F.shared_prefix_attention(q, *(t.contiguous() for t in one), ok, ov))
