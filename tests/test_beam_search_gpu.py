"""Beam search on a GPU: its three operators step after step against the formulas, and whole searches through models."""

import pytest
import torch

from kempnerforge_b200.config import ModelConfig
from kempnerforge_b200.models import KVCache, SharedPrefixCache, Transformer
from kempnerforge_b200.models.generate import beam_search, generate
from kempnerforge_b200.ops import beam
from kempnerforge_b200.ops import functional as F
from tests.test_beam_search import by_hand as search_by_hand
from tests.test_beam_search import make_model
from tests.test_shared_prefix import by_hand
from tests.test_shared_prefix_gpu import RESULT, WEIGHT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("b,w,h,hkv,hd", [(1, 4, 4, 4, 64), (3, 5, 8, 2, 128)])
def test_steps(native_lib, b, w, h, hkv, hd):
    """Twenty steps: choice, exchange of histories and rows, attention through the rows.  Beside them run the formulas on states that
    are moved as a whole, so a row that points to the wrong cache is seen."""
    g = torch.Generator(device="cuda").manual_seed(w)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    steps, vocab, p = 20, 999, 150
    prefix = KVCache(b, p, hkv, hd, torch.bfloat16, torch.device("cuda"))
    prefix.update(rand(b, p, hkv, hd).bfloat16(), rand(b, p, hkv, hd).bfloat16())
    rows = SharedPrefixCache.new_rows(b, w, steps, "cuda")
    cache = SharedPrefixCache(prefix, w, steps, rows)
    tokens = torch.zeros(b, w, steps, dtype=torch.int64, device="cuda")
    scores, finished = torch.zeros(b, w, device="cuda"), torch.zeros(b, w, dtype=torch.bool, device="cuda")
    moved_k, moved_v = (torch.zeros(b, w, steps, hkv, hd, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    moved_tokens, at = tokens.clone(), torch.arange(b, device="cuda")[:, None]
    for n in range(steps):
        logits = (2.5 * rand(b, w, vocab)).bfloat16()
        step = beam.select(logits, scores, finished, eos_id=3, pad_id=3)
        with F.force_reference():
            want = beam.select(logits, scores, finished, eos_id=3, pad_id=3)
        assert torch.equal(step.parents, want.parents) and torch.equal(step.tokens, want.tokens) and torch.equal(step.finished, want.finished)
        assert ((step.scores - want.scores).abs() <= 4e-6 + 2.0**-23 * want.scores.abs()).all()
        beam.reorder([tokens, rows], step.parents, n)
        moved_tokens, moved_k, moved_v = (t[at, step.parents] for t in (moved_tokens, moved_k, moved_v))
        tokens[:, :, n] = moved_tokens[:, :, n] = step.tokens
        assert torch.equal(tokens, moved_tokens)
        scores, finished = step.scores, step.finished
        q, k, v = (rand(b * w, 1, x, hd).bfloat16() for x in (h, hkv, hkv))
        moved_k[:, :, n], moved_v[:, :, n] = k.view(b, w, hkv, hd), v.view(b, w, hkv, hd)
        got = cache.attend(q, k, v).view(b, w, h, hd)
        exact, size = by_hand(q.view(b, w, h, hd), prefix.k, prefix.v, moved_k[:, :, : n + 1], moved_v[:, :, : n + 1])
        assert not ((got.double() - exact).abs() - (WEIGHT * size + RESULT * exact.abs()) > 1e-30).any()


@pytest.mark.parametrize("w,steps,eos", [(1, 5, None), (4, 8, 3)])
def test_search_in_fp32(native_lib, w, steps, eos):
    """The search by hand runs in 64 bits on the CPU; probabilities of this model differ by far more than fp32 rounds."""
    model = make_model()
    prompts = [[1, 5, 2, 9], [7, 7, 0, 3]]
    gpu = make_model().float().cuda()
    tokens, scores = beam_search(gpu, torch.tensor(prompts, device="cuda"), steps, w, eos)
    for b, prompt in enumerate(prompts):
        want_scores, want = search_by_hand(model, prompt, steps, w, eos, 1.0)
        assert tokens[b, :, 4 : 4 + len(want[0])].tolist() == want
        assert torch.allclose(scores[b].cpu().double(), torch.tensor(want_scores, dtype=torch.float64), rtol=1e-3, atol=1e-3)


@pytest.mark.parametrize("dim,heads,kv", [(256, 4, 2), (256, 2, 1)])
def test_search_in_bf16(native_lib, dim, heads, kv):
    torch.manual_seed(1)
    model = Transformer(ModelConfig(dim=dim, n_layers=2, n_heads=heads, n_kv_heads=kv, vocab_size=500, max_seq_len=256)).bfloat16().cuda().eval()
    prompt = torch.randint(0, 500, (3, 100), device="cuda")
    before = native_lib.LAUNCH_COUNT
    tokens, scores = beam_search(model, prompt, 12, 5)
    # 12 choices, 11 reorderings, 11 steps of two layers of two attention kernels, and the models' own
    assert native_lib.LAUNCH_COUNT - before >= 12 + 11 + 44
    assert tokens.shape == (3, 5, 112) and torch.isfinite(scores).all() and (scores[:, :-1] >= scores[:, 1:]).all()
    assert all(len({tuple(row) for row in t.tolist()}) == 5 for t in tokens)
    # The scores are those of the sequences.  A logit is a sum over `dim` of a normed state, off by some 30 roundings of 2^-8 in all,
    # and a weight; random errors of each element add up to 30 * 2^-8 * |w| at most, and a log-probability moves by twice that.
    exact = model.double().cpu()
    logp = torch.log_softmax(exact(tokens.cpu().view(15, 112)), -1)[:, 99:-1]
    own = logp.gather(2, tokens.cpu().view(15, 112)[:, 100:, None])[..., 0].mean(1).view(3, 5)
    largest = exact.output_head.proj.weight.norm(dim=1).max()
    assert ((scores.cpu() - own).abs() <= 2 * 30 * 2.0**-8 * float(largest)).all()


def test_one_beam_is_greedy(native_lib):
    torch.manual_seed(2)
    model = Transformer(ModelConfig(dim=256, n_layers=1, n_heads=4, n_kv_heads=2, vocab_size=300, max_seq_len=64)).float().cuda().eval()
    prompt = torch.randint(0, 300, (2, 9), device="cuda")
    assert torch.equal(beam_search(model, prompt, 6, 1)[0][:, 0], generate(model, prompt, 6, temperature=0.0))
