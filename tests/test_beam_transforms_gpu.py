"""Steps of beam search on a GPU under transforms."""

import pytest
import torch

from kempnerforge_b200.ops import beam

pytestmark = pytest.mark.gpu


def test_selection_of_batched_tensors(native_lib):
    logits, scores = torch.randn(3, 2, 4, 500, device="cuda"), -torch.rand(3, 2, 4, device="cuda")
    got = torch.vmap(lambda x, s: tuple(beam.select(x, s, eos_id=5)))(logits, scores)
    for i in range(3):
        want = beam.select(logits[i], scores[i], eos_id=5)
        assert torch.equal(got[1][i], want.parents) and torch.equal(got[2][i], want.tokens) and torch.equal(got[3][i], want.finished)
        assert ((got[0][i] - want.scores).abs() <= 4e-6 + 2.0**-23 * want.scores.abs()).all()
