"""Where a beam search ends."""

import torch

from kempnerforge_b200.config import ModelConfig
from kempnerforge_b200.models import Transformer
from kempnerforge_b200.models.generate import beam_search

NONE = float("-inf")
EOS, OTHER = 3, 6


class TwoAnswers(Transformer):
    """After the prompt the end or one other token, after that the end."""

    calls = 0

    def forward(self, tokens, **kw):
        logits = super().forward(tokens, **kw)
        allowed = [EOS, OTHER] if self.calls == 0 else [EOS]
        self.calls += 1
        masked = torch.full_like(logits, NONE)
        masked[..., allowed] = logits[..., allowed]
        return masked


def test_places_without_a_continuation_do_not_keep_the_search_going():
    torch.manual_seed(0)
    model = TwoAnswers(ModelConfig(dim=64, n_layers=1, n_heads=4, n_kv_heads=2, vocab_size=11, max_seq_len=48)).eval()
    tokens, scores = beam_search(model, torch.tensor([[1, 2, 4], [5, 5, 0]]), 20, 5, EOS)
    assert model.calls == 2 and tokens.shape == (2, 5, 5)
    for b in range(2):
        assert sorted(tokens[b, :2, 3:].tolist()) == [[EOS, EOS], [OTHER, EOS]]
        assert torch.isfinite(scores[b, :2]).all() and (scores[b, 2:] == NONE).all()


def test_without_an_end_the_search_ends_where_nothing_goes_on():
    """No token may follow: all that could come are more places without a score."""
    torch.manual_seed(0)
    model = TwoAnswers(ModelConfig(dim=64, n_layers=1, n_heads=4, n_kv_heads=2, vocab_size=11, max_seq_len=48)).eval()
    tokens, scores = beam_search(model, torch.tensor([[1, 2, 4]]), 6, 5)   # no end: two answers, of six tokens each
    assert tokens.shape == (1, 5, 9) and torch.isfinite(scores[0, :2]).all() and (scores[0, 2:] == NONE).all()
