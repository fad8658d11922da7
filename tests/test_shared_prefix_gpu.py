"""Attention of many continuations of one prompt: the kernels against 64 bits at the sizes and masks where they can go wrong."""

import pytest
import torch

from kempnerforge_b200.ops import functional as F
from tests.test_shared_prefix import NAN, by_hand, make

pytestmark = pytest.mark.gpu

# bf16 rounds by up to 2^-8: each weight before the second product (in relation to the sum of weights times magnitudes) and the result.
# Scores are fp32 sums of up to 128 products of about 7 in all: 128 * 2^-24 * 7 < 6e-5 each, twice that in a normalised weight; the
# exponential adds 2^-22.
WEIGHT, RESULT = 2.0**-8 + 2.0**-12, 2.0**-8


def near(got, args, **kw):
    want, size = by_hand(*args, **kw)
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    off = (got.double() - want).abs() - (WEIGHT * size + RESULT * want.abs())
    assert not (off > 1e-30).any() and torch.isfinite(got).all(), f"{float(off.max())} over the bound"


SIZES = [
    (1, 1, 1, 1, 1, 1, 64), (1, 1, 1, 1, 2, 1, 128), (1, 2, 127, 0, 2, 2, 128), (1, 2, 128, 1, 2, 2, 64), (1, 2, 129, 63, 4, 2, 128),
    (2, 3, 0, 5, 4, 2, 128), (2, 3, 0, 0, 4, 2, 64), (1, 4, 300, 20, 12, 12, 64), (2, 5, 257, 65, 10, 2, 128), (1, 40, 500, 7, 8, 2, 128),
    (3, 17, 200, 130, 8, 1, 64), (1, 7, 140, 66, 20, 1, 128), (2, 3, 260, 9, 128, 1, 64), (1, 130, 150, 3, 1, 1, 128), (5, 2, 1000, 300, 4, 4, 128),
    (1, 8, 9000, 700, 8, 2, 64), (37, 3, 130, 2, 4, 4, 64),
]


@pytest.mark.parametrize("b,w,p,s,h,hkv,hd", SIZES)
@pytest.mark.parametrize("table", [False, True])
@pytest.mark.parametrize("ragged", [False, True])
def test_sizes(native_lib, b, w, p, s, h, hkv, hd, table, ragged):
    args = make(b, w, p, s, h, hkv, hd, torch.bfloat16, table, ragged, seed=p + s, device="cuda")
    before = native_lib.LAUNCH_COUNT
    got = F.shared_prefix_attention(*args)
    assert native_lib.LAUNCH_COUNT > before
    near(got, args)
    assert torch.equal(got, F.shared_prefix_attention(*args))
    for direct in (0, 1):   # the prompts once for all, and for every continuation again
        got = native_lib.shared_prefix_attn(*args, hd**-0.5, direct)
        near(got, args)
        assert torch.equal(got, native_lib.shared_prefix_attn(*args, hd**-0.5, direct))
    assert native_lib.read_status() == 0


def test_lengths(native_lib):
    """Prompts of every kind in one batch: empty, one key, a whole tile, one more, all."""
    q, k, v, ok, ov, _, _ = make(9, 3, 400, 4, 4, 2, 128, torch.bfloat16, device="cuda")
    lens = torch.tensor([0, 1, 400, 128, 0, 0, 129, 256, 5], device="cuda")
    k[0], v[0] = NAN, NAN
    for i, n in enumerate(lens.tolist()):
        k[i, n:], v[i, n:] = NAN, float("inf")
    for kind in (torch.int32, torch.int64):
        near(F.shared_prefix_attention(q, k, v, ok, ov, lens.to(kind)), (q, k, v, ok, ov, lens))
    for direct in (0, 1):
        near(native_lib.shared_prefix_attn(q, k, v, ok, ov, lens.int(), None, 128**-0.5, direct), (q, k, v, ok, ov, lens))
    # lengths that are none are taken to the nearest one
    past = torch.tensor([-5, 1, 4000, 128, -1, 0, 129, 256, 5], device="cuda", dtype=torch.int32)
    near(F.shared_prefix_attention(q, k, v, ok, ov, past), (q, k, v, ok, ov, lens))


def test_all_prompts_empty(native_lib):
    args = make(3, 2, 200, 3, 4, 2, 64, torch.bfloat16, device="cuda")
    args[5] = torch.zeros(3, dtype=torch.int32, device="cuda")
    near(F.shared_prefix_attention(*args), args)
    args[6] = torch.full((3, 2, 3), 255, dtype=torch.uint8, device="cuda")
    assert (F.shared_prefix_attention(*args) == 0).all()
    for direct in (0, 1):
        assert (native_lib.shared_prefix_attn(*args, 0.125, direct) == 0).all()


def test_what_is_hidden_may_hold_anything(native_lib):
    q, k, v, ok, ov, _, _ = make(2, 3, 140, 70, 4, 2, 128, torch.bfloat16, device="cuda")
    lens = torch.tensor([133, 0], device="cuda", dtype=torch.int32)
    rows = torch.zeros(2, 3, 70, dtype=torch.uint8, device="cuda")
    rows[:, 1, 3:] = 1
    rows[:, 2, ::2] = 9
    rows[1, 2] = 255
    for t in (k, v):
        t[0, 133:] = NAN
        t[1] = float("inf")
    for t in (ok, ov):
        t[:, 2] = NAN
        t[:, 1, :3] = NAN
    calls = [F.shared_prefix_attention] + [lambda *a, d=d: native_lib.shared_prefix_attn(*a, 128**-0.5, d) for d in (0, 1)]
    for call in calls:
        got = call(q, k, v, ok, ov, lens, rows)
        near(got, (q, k, v, ok, ov, lens, rows))
        assert (got[1, 2] == 0).all()
    # what one continuation sees stays with it
    ov[0, 1, 10] = NAN
    for call in calls:
        got = call(q, k, v, ok, ov, lens, rows)
        assert torch.isnan(got[0, 1]).all() and torch.isfinite(got[0, 0]).all() and torch.isfinite(got[0, 2]).all() and torch.isfinite(got[1]).all()


def test_large_scores(native_lib):
    """Scores of hundreds, in rising order, so that maxima move from tile to tile."""
    args = make(1, 40, 700, 150, 4, 2, 128, torch.bfloat16, device="cuda")   # so many that the prompt is read once for all
    ramp = torch.linspace(0.2, 30.0, 700, device="cuda")[None, :, None, None]
    args[1] = (args[1].float().abs() * ramp).bfloat16()
    args[0] = args[0].abs()
    # fp32 sums of 128 products of up to 4000 in all: 128 * 2^-24 * 4000 / 11 = 2.8e-3 worst in a score, twice that in a weight
    want, size = by_hand(*args)
    got = F.shared_prefix_attention(*args)
    off = (got.double() - want).abs() - ((WEIGHT + 2 * 128 * 2.0**-24 * float((args[0][0].double() @ args[1][0, -1].double().transpose(0, 1)).max()) / 11.3) * size
                                         + RESULT * want.abs())
    assert not (off > 1e-30).any()
    near(F.shared_prefix_attention(*args, scale=1e-3), args, scale=1e-3)


def test_views(native_lib):
    """Heads of a fused projection, caches with room behind, layers side by side, and what 16-byte copies cannot take."""
    b, w, p, s, h, hkv, hd = 2, 3, 150, 20, 4, 2, 128
    q, k, v, ok, ov, _, rows = make(b, w, p, s, h, hkv, hd, torch.bfloat16, table=True, device="cuda")
    want = F.shared_prefix_attention(q, k, v, ok, ov, None, rows)
    fused = torch.randn(b, w, h + 2 * hkv, hd, device="cuda").bfloat16()
    fused[:, :, :h] = q
    layers = torch.full((b, p + 30, 2, 3, hkv, hd), NAN, device="cuda", dtype=torch.bfloat16)
    layers[:, :p, 0, 1], layers[:, :p, 1, 1] = k, v
    own = torch.full((2, w, b, s + 9, hkv, hd), NAN, device="cuda", dtype=torch.bfloat16)
    own[0, :, :, :s], own[1, :, :, :s] = ok.transpose(0, 1), ov.transpose(0, 1)
    room = torch.full((b, w, s + 5), 200, dtype=torch.uint8, device="cuda")
    room[:, :, :s] = rows
    got = F.shared_prefix_attention(fused[:, :, :h], layers[:, :p, 0, 1], layers[:, :p, 1, 1], own[0].transpose(0, 1)[:, :, :s],
                                    own[1].transpose(0, 1)[:, :, :s], None, room[:, :, :s])
    assert torch.equal(got, want)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)] + [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (ok, ov)]
    assert torch.equal(F.shared_prefix_attention(q, *heads_first, None, rows), want)
    odd = [torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t) for t in (q, k, v, ok, ov)]
    assert torch.equal(F.shared_prefix_attention(*odd, None, rows), want)
    wide = [torch.empty(*t.shape[:-1], hd + 1, dtype=t.dtype, device="cuda")[..., :hd].copy_(t) for t in (q, k, v, ok, ov)]
    assert torch.equal(F.shared_prefix_attention(*wide, None, rows.transpose(1, 2).contiguous().transpose(1, 2)), want)
    one = k[:1].expand(b, -1, -1, -1), v[:1].expand(b, -1, -1, -1)
    near(F.shared_prefix_attention(q, *one, ok, ov, None, rows), (q, *one, ok, ov, None, rows))


def test_other_types_sizes_and_gradients_take_the_formulas(native_lib):
    before = native_lib.LAUNCH_COUNT
    for dtype, hd in ((torch.float32, 64), (torch.bfloat16, 32), (torch.float16, 64)):
        args = make(1, 2, 40, 5, 4, 2, hd, dtype, device="cuda")
        want, size = by_hand(*args)
        assert ((F.shared_prefix_attention(*args).double() - want).abs() <= 2.0**-8 * size + 1e-5).all()
    args = make(1, 2, 40, 5, 4, 2, 64, torch.bfloat16, device="cuda")
    leaves = [t.requires_grad_() for t in args[:5]]
    F.shared_prefix_attention(*args).sum().backward()
    assert all(t.grad is not None for t in leaves) and native_lib.LAUNCH_COUNT == before


def test_captured_and_on_two_streams(native_lib):
    sets = [make(2, 4, 900, 30, 8, 2, 128, torch.bfloat16, table=True, ragged=True, seed=i, device="cuda") for i in range(2)]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s, args in zip(side, sets):
            with torch.cuda.stream(s):
                got.append((F.shared_prefix_attention(*args), args))
    torch.cuda.synchronize()
    for out, args in got:
        near(out, args)
    graphs, kept = [], []
    for _ in range(2):   # two graphs over the same tensors
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept.append(F.shared_prefix_attention(*sets[0]))
        graphs.append(graph)
    for src, dst in zip(sets[1], sets[0]):
        dst.copy_(src)
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for out in kept:
        near(out, sets[1])


def test_prompts_behind_4_gb(native_lib):
    b, p, hkv, hd = 2, 70, 1, 64
    room = torch.empty(b, 1 << 25, hkv, hd, dtype=torch.bfloat16, device="cuda")   # the second prompt starts behind 4 GB
    q, k, v, ok, ov, _, _ = make(b, 2, p, 3, 2, hkv, hd, torch.bfloat16, device="cuda")
    room[:, :p] = k
    got = F.shared_prefix_attention(q, room[:, :p], v, ok, ov)
    near(got, (q, k, v, ok, ov))


# prompts of over 168 MB, which two row tiles read together: two tiles, three, an odd one of one row, lengths that end in any tile
@pytest.mark.parametrize("b,w,p,h,hkv,hd,lens", [
    (1, 17, 43_011, 64, 8, 128, None), (3, 40, 14_500, 32, 8, 128, [14_499, 1, 9000]), (3, 33, 14_500, 64, 8, 128, [0, 14_337, 130]),
    (5, 129, 58_000, 3, 3, 64, [58_000, 3, 0, 129, 10_001]),
])
def test_prompts_that_outlast_the_cache(native_lib, b, w, p, h, hkv, hd, lens):
    args = make(b, w, p, 5, h, hkv, hd, torch.bfloat16, device="cuda")
    if lens is not None:
        for i, n in enumerate(lens):
            args[1][i, n:], args[2][i, n:] = NAN, float("inf")
        args[5] = torch.tensor(lens, device="cuda", dtype=torch.int32)
    got = F.shared_prefix_attention(*args)
    # a prompt at a time, by what of it counts: the whole in 64 bits would be large
    for i in range(b):
        n = p if lens is None else lens[i]
        near(got[i : i + 1], (args[0][i : i + 1], args[1][i : i + 1, :n], args[2][i : i + 1, :n], args[3][i : i + 1], args[4][i : i + 1], None, None))
    assert torch.equal(got, F.shared_prefix_attention(*args))
    assert native_lib.read_status() == 0


@pytest.mark.parametrize("p,s", [(130, 0), (0, 130), (5, 17)])
def test_scales_that_leave_32_bits_take_the_formulas(native_lib, p, s):
    args = make(1, 2, p, s, 4, 2, 64, torch.bfloat16, device="cuda")
    before = native_lib.LAUNCH_COUNT
    near(F.shared_prefix_attention(*args, scale=1e-50), args, scale=1e-50)
    assert native_lib.LAUNCH_COUNT == before
    with torch.inference_mode():
        got = F.shared_prefix_attention(*args, scale=2.0**-100)
        near(got, args, scale=2.0**-100)
    assert native_lib.LAUNCH_COUNT > before


# sizes at which the kernels take other forms: narrow rings (10 warps an SM) with and without the prompts, many tiles of keys a CTA in few
# and in many registers, prompts of one tile by one kernel where they are many, and by two
@pytest.mark.parametrize("b,w,p,s,h,hkv,hd", [
    (3, 32, 20, 70, 16, 8, 128), (8, 16, 140, 40, 12, 12, 64), (1, 2, 40_001, 9, 8, 8, 128), (1, 2, 40_001, 140, 8, 8, 128),
    (40, 4, 60, 17, 16, 8, 128), (9, 16, 128, 17, 8, 8, 128), (70, 8, 3, 16, 4, 4, 64),
])
def test_forms(native_lib, b, w, p, s, h, hkv, hd):
    args = make(b, w, p, s, h, hkv, hd, torch.bfloat16, table=True, ragged=b > 1, seed=s, device="cuda")
    before = native_lib.LAUNCH_COUNT
    got = F.shared_prefix_attention(*args)
    assert native_lib.LAUNCH_COUNT > before
    near(got, args)
    assert torch.equal(got, F.shared_prefix_attention(*args))
    assert native_lib.read_status() == 0
