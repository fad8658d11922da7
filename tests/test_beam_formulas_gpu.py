"""The formulas of selection on a GPU (more than 32 beams, other types than the kernel's): equal beams come in their order."""

import math

import pytest
import torch

from kempnerforge_b200.ops import beam
from tests.test_beam_order_gpu import best_of_equal_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,w,vocab", [(1, 40, 50257), (9, 33, 999), (20, 40, 1001), (20, 64, 2003), (3, 33, 128255), (1, 40, 17)])
def test_equal_rows(native_lib, b, w, vocab, dtype):
    # one logit at zero, the others' exponentials add up to about as much: the logarithm and the scores are small, and show a sum's last bit
    rows = 0.5 * torch.randn(b, 1, vocab, generator=torch.Generator().manual_seed(vocab), dtype=torch.float64) - math.log(vocab)
    rows[:, :, 5] = 0.0
    rows = rows.to(dtype)
    logits, scores = rows.cuda().expand(b, w, vocab), torch.zeros(b, w, device="cuda")
    for x in (logits, logits.contiguous()):
        got = beam.select(x, scores)
        for i in range(b):
            parents, tokens = best_of_equal_rows(rows[i, 0], w)
            assert torch.equal(got.parents[i].cpu(), parents) and torch.equal(got.tokens[i].cpu(), tokens)
