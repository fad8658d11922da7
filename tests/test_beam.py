"""Steps of beam search on the CPU: the formulas against a search by hand, what is refused, and which memory may be shared."""

import math

import pytest
import torch

from kempnerforge_b200.ops import beam

NONE = float("-inf")


def by_hand(logits, scores, finished, eos, pad):
    """Candidate by candidate in Python floats."""
    b, w, vocab = logits.shape
    largest = torch.finfo(torch.float32).max
    rows = []
    for i in range(b):
        found = []
        for j in range(w):
            s = float(scores[i, j])
            if not s > NONE:
                continue
            if finished is not None and bool(finished[i, j]):
                found.append((-s, j, 0, 0, pad, True))
                continue
            x = [min(v, largest) if v > NONE else NONE for v in logits[i, j].tolist()]
            top = max(x)
            if top == NONE:
                continue
            lse = top + math.log(math.fsum(math.exp(v - top) for v in x if v > NONE))
            found += [(-(s + (v - lse)), j, -v, t, t, False) for t, v in enumerate(x) if v > NONE]
        found.sort()
        rows.append([(-f[0], f[1], f[4], f[5] or f[4] == eos) for f in found[:w]]
                    + [(NONE, j, pad, False) for j in range(min(len(found), w), w)])
    pick = lambda n: [[r[n] for r in row] for row in rows]  # noqa: E731
    return (torch.tensor(pick(0), dtype=torch.float64), torch.tensor(pick(1)), torch.tensor(pick(2)), torch.tensor(pick(3)))


def same(got, want):
    assert torch.equal(got.parents.cpu(), want[1])
    assert torch.equal(got.tokens.cpu(), want[2])
    assert torch.equal(got.finished.cpu(), want[3])
    none = want[0] == NONE
    assert torch.equal(got.scores.cpu() == NONE, none)
    # 64 bits rounded to 32 once; sums of fp32 exponentials leave about 1e-6 in the logarithm
    assert ((got.scores.cpu().double() - want[0])[~none].abs() <= 2.0**-24 * want[0][~none].abs() + 4e-6).all()


def make(b, w, vocab, dtype, seed, finished=True):
    g = torch.Generator().manual_seed(seed)
    logits = (2.5 * torch.randn(b, w, vocab, generator=g)).to(dtype)
    scores = -20 * torch.rand(b, w, generator=g)
    done = torch.rand(b, w, generator=g) < 0.3 if finished else None
    return logits, scores, done


SIZES = [(1, 1, 1), (1, 4, 7), (2, 3, 2), (3, 5, 101), (2, 32, 40), (1, 8, 8)]


@pytest.mark.parametrize("b,w,vocab", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_select(b, w, vocab, dtype):
    logits, scores, done = make(b, w, vocab, dtype, b + w)
    same(beam.select(logits, scores, done, eos_id=vocab - 1, pad_id=3), by_hand(logits, scores, done, vocab - 1, 3))
    same(beam.select(logits, scores), by_hand(logits, scores, None, -1, 0))


def extremes(dtype):
    """Rows of what a mask leaves and of numbers at the ends of the type."""
    low, big = torch.finfo(dtype).min, torch.finfo(dtype).max
    inf, nan = float("inf"), float("nan")
    rows = [[1.0, NONE, 2.0, nan, 2.0, 0.5], [NONE] * 6, [low] * 6, [low, low, 1.0, NONE, 0.0, -0.0], [inf, 1.0, inf, 2.0, NONE, 0.0],
            [nan] * 6, [big, big, 1.0, low, 0.0, 2.0], [0.0, -0.0, 0.0, -0.0, 0.0, -0.0]]
    return torch.tensor(rows, dtype=torch.float64).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_select_extremes(dtype):
    rows = extremes(dtype)
    logits = torch.stack([rows, rows.flip(0)])
    scores = torch.tensor([-1.0, -2.0, -3.0, -4.0, -5.0, -6.0, -7.0, -8.0]).repeat(2, 1)
    same(beam.select(logits, scores, eos_id=2), by_hand(logits, scores, None, 2, 0))
    # a search's first step: one beam counts; and beams without a score
    first = torch.full((2, 8), NONE)
    first[:, 0] = 0.0
    same(beam.select(logits, first, eos_id=2, pad_id=9), by_hand(logits, first, None, 2, 9))
    first[1, 0] = float("nan")
    same(beam.select(logits, first, eos_id=2, pad_id=9), by_hand(logits, first, None, 2, 9))


def test_select_ties_go_to_the_lower_beam_and_token():
    logits = torch.zeros(1, 3, 5)
    got = beam.select(logits, torch.zeros(1, 3))
    assert got.parents.tolist() == [[0, 0, 0]] and got.tokens.tolist() == [[0, 1, 2]]


def test_select_refuses():
    logits, scores, done = make(2, 3, 5, torch.float32, 0)
    for bad in ((logits[0], scores, done), (logits.long(), scores, done), (logits[:, :, :0], scores, done), (logits, scores[:1], done),
                (logits, scores.double(), done), (logits, scores, done.int()), (logits, scores, done[:, :2])):
        with pytest.raises(ValueError):
            beam.select(*bad)


def states(b, w, room, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1000, (b, w, room), generator=g), torch.randint(0, 255, (b, w, room), generator=g, dtype=torch.uint8),
            torch.randn(b, w, room, 3, generator=g), torch.randn(b, w, room, 2, 8, generator=g).bfloat16()]


@pytest.mark.parametrize("b,w,room,length", [(1, 1, 1, 1), (2, 4, 9, 5), (3, 5, 7, None), (2, 3, 4, 0), (2, 40, 3, 2)])
@pytest.mark.parametrize("out", [False, True])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_reorder(b, w, room, length, out, dtype):
    parents = torch.randint(-1, w + 1, (b, w), generator=torch.Generator().manual_seed(1)).to(dtype)   # some are no beams
    old = states(b, w, room)
    new = [torch.full_like(x, 7) for x in old] if out else [x.clone() for x in old]
    want = [x.clone() for x in new]
    n = room if length is None else length
    for x, y in zip(old, want):
        for i in range(b):
            for j in range(w):
                p = int(parents[i, j])
                if 0 <= p < w:
                    y[i, j, :n] = x[i, p, :n]
    kept = [x.clone() for x in old]
    got = beam.reorder(old, parents, length, out=new) if out else beam.reorder(new, parents, length)
    assert all(a is b for a, b in zip(got, new))
    assert all(torch.equal(x, y) for x, y in zip(new, want))
    assert all(torch.equal(x, y) for x, y in zip(old, kept))


def test_reorder_refuses():
    parents = torch.zeros(2, 4, dtype=torch.int64)
    x = torch.zeros(2, 4, 8)
    wide = torch.zeros(2, 4, 16)
    for bad in (lambda: beam.reorder([x], parents[0]), lambda: beam.reorder([x], parents.float()), lambda: beam.reorder([x], parents, -1),
                lambda: beam.reorder([x], parents, 9), lambda: beam.reorder([x[:, :, 0]], parents, 1), lambda: beam.reorder([x[:1]], parents),
                lambda: beam.reorder([x], parents, out=[]), lambda: beam.reorder([x], parents, out=[x.double()]),
                lambda: beam.reorder([x], parents, out=[x[:, :, :4]]), lambda: beam.reorder([x, x], parents),
                lambda: beam.reorder([wide[:, :, :8]], parents, out=[wide[:, :, 4:12]]),
                lambda: beam.reorder([x.clone().requires_grad_()], parents)):
        with pytest.raises(ValueError):
            bad()


def test_reorder_takes_states_that_lie_between_each_other():
    both = torch.arange(2 * 3 * 8.0).view(2, 3, 8).clone()
    parents = torch.tensor([[1, 0, 0], [2, 2, 1]])
    want = torch.stack([both[i, parents[i]] for i in range(2)])
    beam.reorder([both[:, :, :4], both[:, :, 4:]], parents)
    assert torch.equal(both, want)


def test_reorder_moves_the_version():
    x = torch.randn(1, 2, 4)
    before = x._version
    beam.reorder([x], torch.tensor([[1, 0]]))
    assert x._version > before


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_reorder_refuses_to_write_its_parents(dtype):
    parents = torch.tensor([[1, 0, 2]], dtype=dtype)
    room = torch.tensor([[0, 2, 1, 1]], dtype=dtype)
    for bad in (lambda: beam.reorder([parents], parents), lambda: beam.reorder([torch.zeros(1, 3), room[:, 1:]], room[:, :3]),
                lambda: beam.reorder([torch.zeros(1, 3, dtype=dtype)], parents, out=[parents])):
        with pytest.raises(ValueError):
            bad()
    assert parents.tolist() == [[1, 0, 2]]
    assert beam.reorder([parents], parents, out=[torch.zeros(1, 3, dtype=dtype)])[0].tolist() == [[0, 1, 2]]
