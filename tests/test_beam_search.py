"""Beam search through a model: against a search by hand with whole forward passes, and against all continuations there are."""

import itertools

import pytest
import torch

from kempnerforge_b200.config import ModelConfig
from kempnerforge_b200.models import KVCache, SharedPrefixCache, Transformer
from kempnerforge_b200.models.generate import beam_search, generate


def make_model(vocab=11, **kw):
    torch.manual_seed(0)
    model = Transformer(ModelConfig(dim=64, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=vocab, max_seq_len=48, **kw)).double().eval()
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() == 2:
                p.normal_(0.0, 0.3)   # probabilities that differ
    return model


@torch.no_grad()
def by_hand(model, prompt, steps, w, eos, penalty):
    """One prompt: every beam's whole sequence through the model at every step."""
    beams = [(0.0, (), False)]
    for _ in range(steps):
        found = []
        for j, (score, seq, done) in enumerate(beams):
            if done:
                found.append((score, -j, 0, seq, True))
                continue
            logits = model(torch.tensor([prompt + list(seq)]))[0, -1].double()
            logp = torch.log_softmax(logits, 0).tolist()
            found += [(score + lp, -j, -t, (*seq, t), t == eos) for t, lp in enumerate(logp)]
        found.sort(reverse=True, key=lambda f: f[:3])
        beams = [(f[0], f[3], f[4]) for f in found[:w]]
        if all(b[2] for b in beams):
            break
    ranked = sorted(((score / len(seq) ** penalty, seq) for score, seq, _ in beams), key=lambda f: -f[0])
    longest = max(len(seq) for _, seq in ranked)
    return [s for s, _ in ranked], [list(seq) + [eos or 0] * (longest - len(seq)) for _, seq in ranked]


@pytest.mark.parametrize("w,steps,eos,penalty", [(1, 5, None, 1.0), (3, 6, None, 1.0), (4, 8, 3, 1.0), (4, 8, 3, 0.0), (6, 7, 5, 2.0)])
def test_search(w, steps, eos, penalty):
    model = make_model()
    prompts = [[1, 5, 2, 9], [7, 7, 0, 3]]
    tokens, scores = beam_search(model, torch.tensor(prompts), steps, w, eos, penalty)
    for b, prompt in enumerate(prompts):
        want_scores, want = by_hand(model, prompt, steps, w, eos, penalty)
        n = len(want[0])
        assert tokens[b, :, :4].tolist() == [prompt] * w
        assert tokens[b, :, 4 : 4 + n].tolist() == want
        assert (tokens[b, :, 4 + n :] == (eos or 0)).all()
        assert torch.allclose(scores[b].double(), torch.tensor(want_scores, dtype=torch.float64), rtol=1e-5, atol=1e-5)


def test_search_over_everything_finds_the_best():
    model = make_model(vocab=5)
    prompt = [1, 4, 2]
    tokens, scores = beam_search(model, torch.tensor([prompt]), 3, 25)
    best = []
    with torch.no_grad():
        for seq in itertools.product(range(5), repeat=3):
            logp = torch.log_softmax(model(torch.tensor([prompt + list(seq)]))[0].double(), -1)
            best.append((sum(float(logp[2 + i, t]) for i, t in enumerate(seq)) / 3, list(seq)))
    best.sort(reverse=True)
    assert tokens[0, 0, 3:].tolist() == best[0][1] and abs(float(scores[0, 0]) - best[0][0]) < 1e-5


def test_one_beam_is_greedy():
    model = make_model()
    prompt = torch.tensor([[1, 2, 3], [4, 5, 6]])
    assert torch.equal(beam_search(model, prompt, 6, 1)[0][:, 0], generate(model, prompt, 6, temperature=0.0))


def test_more_beams_than_continuations():
    model = make_model(vocab=3)
    tokens, scores = beam_search(model, torch.tensor([[1, 2]]), 1, 5)
    assert torch.isfinite(scores[0, :3]).all() and (scores[0, 3:] == float("-inf")).all()
    assert sorted(tokens[0, :3, 2].tolist()) == [0, 1, 2]


def test_arguments():
    model = make_model()
    prompt = torch.tensor([[1, 2, 3]])
    for bad in (lambda: beam_search(model, prompt, 46), lambda: beam_search(model, prompt, 2, 0), lambda: beam_search(model, prompt, 2, 257),
                lambda: beam_search(model, prompt[:, :0], 2)):
        with pytest.raises(ValueError):
            bad()
    assert torch.equal(beam_search(model, prompt, 0, 2)[0], prompt[:, None].expand(1, 2, 3))
    model.train()
    beam_search(model, prompt, 2, 2)
    assert model.training


def test_cache():
    prefix = KVCache(2, 8, 2, 4, torch.float32, torch.device("cpu"))
    prefix.update(torch.randn(2, 3, 2, 4), torch.randn(2, 3, 2, 4))
    cache = SharedPrefixCache(prefix, 3, 2)
    assert cache.seq_len == 3 and cache.k.shape == (2, 3, 2, 4) and cache.own_k.shape == (2, 3, 2, 2, 4)
    q, k, v = torch.randn(6, 1, 4, 4), torch.randn(6, 1, 2, 4), torch.randn(6, 1, 2, 4)
    assert cache.attend(q, k, v).shape == (6, 1, 4, 4) and cache.seq_len == 4
    assert torch.equal(cache.own_k[1, 2, 0], k[5, 0])
    with pytest.raises(ValueError):
        cache.attend(q[:5], k[:5], v[:5])
    with pytest.raises(ValueError):
        cache.attend(q.expand(6, 2, 4, 4), k, v)
    cache.attend(q, k, v)
    with pytest.raises(ValueError, match="overflow"):
        cache.attend(q, k, v)
    rows = SharedPrefixCache.new_rows(2, 3, 5, "cpu")
    assert rows.shape == (2, 3, 5) and rows.dtype == torch.uint8 and (rows == torch.arange(3, dtype=torch.uint8)[:, None]).all()
    with pytest.raises(ValueError):
        SharedPrefixCache.new_rows(1, 257, 1, "cpu")


def test_masks_are_refused():
    model = make_model()
    prefix = KVCache(1, 8, 2, 16, torch.float64, torch.device("cpu"))
    att = model.layers["0"].attention
    cos, sin = model.rope_tables(torch.device("cpu"), 0, 1)
    with pytest.raises(ValueError):
        att(torch.randn(2, 1, 64, dtype=torch.float64), cos, sin, kv_cache=SharedPrefixCache(prefix, 2, 4), doc_ids=torch.zeros(2, 1))


def test_script(tmp_path, capsys, monkeypatch):
    import importlib.util
    import pathlib

    path = pathlib.Path(__file__).resolve().parent.parent / "scripts" / "generate.py"
    spec = importlib.util.spec_from_file_location("generate_script", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    cfg = path.parent.parent / "configs" / "train" / "debug.toml"
    assert mod.main([str(cfg), "--prompt", "1 2 3", "--max-new-tokens", "4", "--num-beams", "3", "--device", "cpu"]) == 0
    assert len(capsys.readouterr().out.split()[-7:]) == 7
