"""Selection on a GPU where candidates of different beams lie next to each other: the order is that of 64-bit scores, equal ones go to the
lower beam and then to the lower token, wherever rows begin and whichever threads read them."""

import math

import pytest
import torch

from kempnerforge_b200.ops import beam
from tests.test_beam import NONE, by_hand, same

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def best_of_equal_rows(row, w):
    """Beams with this row and one score: every beam's best token, and where several are the best, all of a beam's before the next beam's."""
    ties = torch.nonzero(row == row.max())[:, 0].tolist()
    found = [(j, t) for j in range(w) for t in ties][:w]
    return torch.tensor([f[0] for f in found]), torch.tensor([f[1] for f in found])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,w,vocab", [(1, 4, 50257), (3, 5, 50257), (1, 2, 32001), (20, 6, 10007), (2, 32, 9001), (1, 8, 128256), (4, 3, 17)])
def test_equal_rows(native_lib, b, w, vocab, dtype):
    g = torch.Generator().manual_seed(vocab + w)
    rows = (2.5 * torch.randn(b, 1, vocab, generator=g)).to(dtype)
    scores = torch.full((b, w), -3.25)
    for logits in (rows.cuda().expand(b, w, vocab), rows.cuda().expand(b, w, vocab).contiguous()):
        got = beam.select(logits, scores.cuda())
        for i in range(b):
            parents, tokens = best_of_equal_rows(rows[i, 0], w)
            assert torch.equal(got.parents[i].cpu(), parents) and torch.equal(got.tokens[i].cpu(), tokens)


def close(b, w, vocab, dtype, seed, shuffled):
    """Rows of one prompt are the same, or the same in another order; scores are a few that lie a rounding apart."""
    g = torch.Generator().manual_seed(seed)
    row = (2.5 * torch.randn(b, 1, vocab, generator=g)).to(dtype)
    logits = row.expand(b, w, vocab).clone()
    if shuffled:
        for i in range(b):
            for j in range(w):
                logits[i, j] = row[i, 0, torch.randperm(vocab, generator=g)]
    base = torch.full((), -9.0)
    steps = [base]
    for _ in range(w):
        steps.append(torch.nextafter(steps[-1], torch.zeros(())))
    # beams of another order have a score each: of equal ones rounding decides, in the formulas as well
    scores = torch.stack([torch.stack(steps)[torch.randperm(w, generator=g) if shuffled else torch.randint(0, 2, (w,), generator=g)] for _ in range(b)])
    return logits, scores


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shuffled", [False, True])
@pytest.mark.parametrize("b,w,vocab", [(1, 4, 5003), (3, 5, 10007), (20, 8, 1001), (1, 32, 2003)])
def test_scores_a_rounding_apart(native_lib, b, w, vocab, dtype, shuffled):
    logits, scores = close(b, w, vocab, dtype, w, shuffled)
    same(beam.select(logits.cuda(), scores.cuda(), eos_id=5), by_hand(logits, scores, None, 5, 0))
    # some of them at their end, some without a score, tokens that must not appear
    done = torch.rand(b, w, generator=torch.Generator().manual_seed(1)) < 0.3
    scores[:, 1:2] = NONE
    logits[:, :, ::7] = NONE
    same(beam.select(logits.cuda(), scores.cuda(), done.cuda(), 5, 5), by_hand(logits, scores, done, 5, 5))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("up", [False, True])
def test_a_finished_beam_beside_a_live_one(native_lib, dtype, up):
    """The finished beam's score is the 32-bit number next to the live one's best."""
    g = torch.Generator().manual_seed(3)
    logits = (2.5 * torch.randn(1, 3, 20011, generator=g)).to(dtype)
    x = logits[0, 0].double()
    best = -2.0 + float(x.max() - torch.logsumexp(x, 0))
    beside = torch.tensor(best, dtype=torch.float64).float()
    if (float(beside) > best) != up:
        beside = torch.nextafter(beside, torch.tensor(math.inf if up else -math.inf))
    scores = torch.tensor([[-2.0, float(beside), -50.0]])
    done = torch.tensor([[False, True, False]])
    want = by_hand(logits, scores, done, 7, 7)
    assert want[1][0, 0] == (1 if up else 0)
    same(beam.select(logits.cuda(), scores.cuda(), done.cuda(), 7, 7), want)


def test_the_last_place_goes_to_the_lower_beam(native_lib):
    """Two beams, equal in all, and one place for them; and what lies behind the last place by less than a rounding."""
    g = torch.Generator().manual_seed(4)
    far = 2.5 * torch.randn(1, 1, 50257, generator=g)
    far[0, 0, 100] = 40.0   # takes the first place, and nothing else of this beam is near
    near = 2.5 * torch.randn(1, 1, 50257, generator=g)
    near[0, 0, 9] = 30.0
    logits = torch.cat([near, far, near], 1)
    for scores in ([-4.0, -1.0, -4.0], [-4.0, -1.0, float(torch.nextafter(torch.tensor(-4.0), torch.tensor(0.0)))]):
        scores = torch.tensor([scores])
        same(beam.select(logits.cuda(), scores.cuda()), by_hand(logits, scores, None, -1, 0))


def test_captured(native_lib):
    """What decides whether the sums are taken again is on the device: a graph captured where it is not needed replays where it is."""
    logits, scores = close(2, 6, 30011, torch.float32, 2, False)
    apart = torch.randn(2, 6, 30011, generator=torch.Generator().manual_seed(5)), -torch.arange(12.0).view(2, 6)
    buffers = [t.cuda() for t in apart]
    beam.select(*buffers)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = beam.select(*buffers)
    for inputs in (apart, (logits, scores), apart):
        for src, dst in zip(inputs, buffers):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        same(got, by_hand(*inputs, None, -1, 0))
