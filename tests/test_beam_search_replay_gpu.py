"""Whole searches in bf16 on a GPU, replayed from the logits that the model gave: which beams go on, in which order, with which tokens."""

import pytest
import torch

from kempnerforge_b200.config import ModelConfig
from kempnerforge_b200.models import Transformer
from kempnerforge_b200.models.generate import beam_search
from tests.test_beam import NONE, by_hand

pytestmark = pytest.mark.gpu


class Recorded(Transformer):
    """Keeps the last position's logits of every call."""

    def forward(self, tokens, **kw):
        logits = super().forward(tokens, **kw)
        self.__dict__.setdefault("seen", []).append((tokens.cpu(), logits[:, -1].cpu()))
        return logits


@pytest.mark.parametrize("dim,heads,kv,w,eos,penalty", [(256, 4, 2, 5, None, 1.0), (256, 2, 1, 8, 7, 0.5)])
def test_search(native_lib, dim, heads, kv, w, eos, penalty):
    torch.manual_seed(1)
    b, steps, vocab = 3, 12, 501
    model = Recorded(ModelConfig(dim=dim, n_layers=2, n_heads=heads, n_kv_heads=kv, vocab_size=vocab, max_seq_len=256)).bfloat16().cuda().eval()
    with torch.no_grad():
        if eos is not None:
            model.output_head.proj.weight[eos] *= 3.0   # some end early
    prompt = torch.randint(0, vocab, (b, 100), device="cuda")
    tokens, scores = beam_search(model, prompt, steps, w, eos, penalty)
    pad = 0 if eos is None else eos
    total, finished = torch.full((b, w), NONE), torch.zeros(b, w, dtype=torch.bool)
    total[:, 0] = 0.0
    histories = [[[] for _ in range(w)] for _ in range(b)]
    for n, (given, logits) in enumerate(model.seen):
        if n:   # the tokens of the step before, beam by beam
            assert given.view(b, w).tolist() == [[h[-1] for h in row] for row in histories]
        logits = (logits[:, None].expand(b, w, vocab) if n == 0 else logits.view(b, w, vocab)).contiguous()
        best, parents, chosen, finished = by_hand(logits, total, finished, -1 if eos is None else eos, pad)
        total = best.float()
        histories = [[histories[i][int(parents[i, j])] + [int(chosen[i, j])] for j in range(w)] for i in range(b)]
    for i in range(b):
        lengths = [h.index(eos) + 1 if eos in h else len(h) for h in histories[i]]
        ranked = sorted(range(w), key=lambda j: -float(total[i, j]) / lengths[j] ** penalty)
        assert tokens[i, :, 100:].tolist() == [histories[i][j] for j in ranked]
        want = torch.tensor([float(total[i, j]) / lengths[j] ** penalty for j in ranked])
        # a step leaves 4e-6 and a rounding in a sum
        assert ((scores[i].cpu() - want).abs() <= steps * (4e-6 + 2.0**-23 * total[i].abs().max())).all()
    assert eos is None or any(eos in h[:-1] for row in histories for h in row)
