"""Beam search's kernels: selection against a search by hand, reordering against indexing, captured, on other streams and twice at once."""

import pytest
import torch

from kempnerforge_b200.ops import beam
from tests.test_beam import NONE, by_hand, extremes, make, same, states

pytestmark = pytest.mark.gpu

SIZES = [(1, 1, 1), (1, 4, 7), (2, 3, 2), (3, 5, 101), (2, 32, 40), (1, 8, 8), (1, 4, 32000), (3, 5, 50257), (70, 2, 1000), (1, 32, 9001)]


@pytest.mark.parametrize("b,w,vocab", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_select(native_lib, b, w, vocab, dtype):
    logits, scores, done = make(b, w, vocab, dtype, b + w)
    before = native_lib.LAUNCH_COUNT
    same(beam.select(logits.cuda(), scores.cuda(), done.cuda(), eos_id=vocab - 1, pad_id=3), by_hand(logits, scores, done, vocab - 1, 3))
    assert native_lib.LAUNCH_COUNT > before
    same(beam.select(logits.cuda(), scores.cuda()), by_hand(logits, scores, None, -1, 0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("copies", [1, 300])
def test_select_extremes(native_lib, dtype, copies):
    rows = extremes(dtype).repeat(1, copies)
    logits = torch.stack([rows, rows.flip(0)])
    scores = torch.tensor([-1.0, -2.0, -3.0, -4.0, -5.0, -6.0, -7.0, -8.0]).repeat(2, 1)
    same(beam.select(logits.cuda(), scores.cuda(), eos_id=2), by_hand(logits, scores, None, 2, 0))
    first = torch.full((2, 8), NONE)
    first[:, 0] = 0.0
    same(beam.select(logits.cuda(), first.cuda(), eos_id=2, pad_id=9), by_hand(logits, first, None, 2, 9))
    first[1, 0] = float("nan")
    same(beam.select(logits.cuda(), first.cuda(), eos_id=2, pad_id=9), by_hand(logits, first, None, 2, 9))


@pytest.mark.parametrize("order", ["rising", "falling", "equal", "tiny"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select_orders(native_lib, order, dtype):
    """Every logit above the ones before, below them, all alike; and numbers below the smallest normal one."""
    n = 20011
    ramp = torch.arange(n, dtype=torch.float64) / n
    rows = {"rising": ramp, "falling": -ramp, "equal": 0 * ramp, "tiny": ramp * 1e-39}[order].to(dtype)
    logits = rows.repeat(1, 8, 1)
    scores = -torch.arange(8.0)[None] / 64
    same(beam.select(logits.cuda(), scores.cuda()), by_hand(logits, scores, None, -1, 0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("start", [0, 1, 3])
def test_select_strides(native_lib, dtype, start):
    """Rows that begin anywhere, one row for all beams, the last position of a longer tensor."""
    wide, scores, done = make(2, 4, 1031, dtype, 3)
    part = wide.cuda()[:, :, start : start + 1000]
    same(beam.select(part, scores.cuda(), done.cuda(), 5), by_hand(part.cpu(), scores, done, 5, 0))
    one = wide.cuda()[:, :1].expand(2, 4, 1031)
    same(beam.select(one, scores.cuda(), done.cuda(), 5), by_hand(one.cpu(), scores, done, 5, 0))
    steps = wide.cuda().transpose(0, 1)
    same(beam.select(steps, scores.cuda().t(), done.cuda().t(), 5), by_hand(steps.cpu(), scores.t(), done.t(), 5, 0))


def test_select_reads_nothing_of_beams_that_are_done(native_lib):
    logits, scores, _ = make(2, 4, 5000, torch.bfloat16, 1)
    done = torch.tensor([[True, False, False, True], [True] * 4])
    logits[done] = float("nan")
    same(beam.select(logits.cuda(), scores.cuda(), done.cuda(), 7, 7), by_hand(logits, scores, done, 7, 7))


def test_select_takes_more_beams_by_the_formulas(native_lib):
    logits, scores, done = make(1, 40, 50, torch.float32, 2)
    same(beam.select(logits.cuda(), scores.cuda(), done.cuda(), 7, 7), by_hand(logits, scores, done, 7, 7))


def test_select_captured_and_on_two_streams(native_lib):
    logits, scores, done = (t.cuda() for t in make(2, 6, 30001, torch.bfloat16, 4))
    want = by_hand(logits.cpu(), scores.cpu(), done.cpu(), 9, 9)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s in side:
            with torch.cuda.stream(s):
                got.append(beam.select(logits, scores, done, 9, 9))
    torch.cuda.synchronize()
    for x in got:
        same(x, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = beam.select(logits, scores, done, 9, 9)
    other = make(2, 6, 30001, torch.bfloat16, 5)
    for src, dst in zip(other, (logits, scores, done)):
        dst.copy_(src)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    same(kept, by_hand(*other, 9, 9))


@pytest.mark.parametrize("b,w,room,length", [(1, 1, 1, 1), (2, 4, 9, 5), (3, 5, 7, None), (2, 3, 4, 0), (2, 32, 33, 31), (2, 40, 3, 2), (3, 8, 700, 333),
                                             (40, 16, 65, 64)])
@pytest.mark.parametrize("out", [False, True])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_reorder(native_lib, b, w, room, length, out, dtype):
    parents = torch.randint(-1, w + 1, (b, w), generator=torch.Generator().manual_seed(1)).to(dtype)
    old = states(b, w, room)
    new = [torch.full_like(x, 7) for x in old] if out else [x.clone() for x in old]
    want = [x.clone() for x in new]
    beam.reorder(old, parents, length, out=want) if out else beam.reorder(want, parents, length)   # tested on the CPU
    gpu_old, gpu_new = [x.cuda() for x in old], [x.cuda() for x in new]
    if out:
        beam.reorder(gpu_old, parents.cuda(), length, out=gpu_new)
        assert all(torch.equal(x.cpu(), y) for x, y in zip(gpu_old, old))
    else:
        beam.reorder(gpu_new, parents.cuda(), length)
    assert all(torch.equal(x.cpu(), y) for x, y in zip(gpu_new, want))
    # one state alone takes the widest words that its own steps allow
    for x, y, z in zip(old, new, want):
        alone = y.cuda()
        beam.reorder([x.cuda()], parents.cuda(), length, out=[alone]) if out else beam.reorder([alone], parents.cuda(), length)
        assert torch.equal(alone.cpu(), z)


def test_reorder_many_states_views_and_versions(native_lib):
    parents = torch.tensor([[2, 0, 0, 3], [1, 0, 3, 2]], device="cuda")
    rows = torch.arange(2, device="cuda")[:, None]
    many = [torch.randn(2, 4, 5, device="cuda") for _ in range(130)]
    want = [x[rows, parents] for x in many]
    versions = [x._version for x in many]
    beam.reorder(many, parents)
    assert all(torch.equal(x, y) for x, y in zip(many, want))
    assert all(x._version > v for x, v in zip(many, versions))
    # keys and values of a layer side by side, beams first or prompts first, and entries that are not dense
    both = torch.randn(2, 4, 6, 16, device="cuda")
    want = both[rows, parents]
    beam.reorder([both[:, :, :3], both[:, :, 3:]], parents)
    assert torch.equal(both, want)
    turned = torch.randn(4, 2, 10, device="cuda").transpose(0, 1)
    want = turned[rows, parents]
    beam.reorder([turned], parents)
    assert torch.equal(turned, want)
    sparse = torch.randn(2, 4, 6, 16, device="cuda")[..., ::2]
    want = sparse[rows, parents]
    beam.reorder([sparse], parents)
    assert torch.equal(sparse, want)


def test_reorder_captured_and_behind_4_gb(native_lib):
    x = torch.randint(0, 100, (1, 4, 64), device="cuda")
    parents = torch.tensor([[1, 2, 3, 0]], device="cuda")
    want = x.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        beam.reorder([x], parents, 40)
    for _ in range(3):
        graph.replay()
        want[:, :, :40] = want[:, [1, 2, 3, 0], :40]
    assert torch.equal(x, want)
    big = torch.empty(1, 3, (1 << 31) + 40, dtype=torch.uint8, device="cuda")
    big[0, :, -40:] = torch.randint(0, 255, (3, 40), device="cuda", dtype=torch.uint8)
    want = big[0, [2, 0, 1], -40:].clone()
    beam.reorder([big], torch.tensor([[2, 0, 1]], device="cuda"))
    assert torch.equal(big[0, :, -40:], want)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_reorder_refuses_to_write_its_parents(native_lib, dtype):
    parents = torch.tensor([[1, 0, 2]], dtype=dtype, device="cuda")
    room = torch.tensor([[0, 2, 1, 1]], dtype=dtype, device="cuda")
    for bad in (lambda: beam.reorder([parents], parents), lambda: beam.reorder([torch.zeros(1, 3, device="cuda"), room[:, 1:]], room[:, :3]),
                lambda: beam.reorder([torch.zeros_like(parents)], parents, out=[parents])):
        with pytest.raises(ValueError):
            bad()
    assert parents.tolist() == [[1, 0, 2]]
    assert beam.reorder([parents], parents, out=[torch.zeros_like(parents)])[0].tolist() == [[0, 1, 2]]


def test_in_inference_mode(native_lib):
    logits = torch.randn(2, 3, 1000, device="cuda")
    scores = torch.randn(2, 3, device="cuda")
    history = torch.randint(0, 99, (2, 3, 8), device="cuda")
    want = beam.select(logits, scores, eos_id=5)
    moved = torch.stack([history[i, want.parents[i]] for i in range(2)])
    with torch.inference_mode():
        for x in (history.clone(), history):
            got = beam.select(logits, scores, eos_id=5)
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and got.scores.is_inference()
            got.scores.add_(1.0)
            assert torch.equal(got.parents, want.parents)
            beam.reorder([x], got.parents)
            assert torch.equal(x, moved)
