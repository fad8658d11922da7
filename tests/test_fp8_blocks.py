"""fp8 with a scale for each block of 128 on a CPU: the definition of the form, the emulated products, refusals."""

import pytest
import torch

from kempnerforge_b200.ops import fp8_blocks as fb

HALF_BF16 = 2.0**-8   # half a step of bf16 (7 fraction bits), relative


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)


@pytest.mark.parametrize("e5m2, top, fraction, least", [(False, 448.0, 3, -6), (True, 57344.0, 2, -14)], ids=["e4m3", "e5m2"])
@pytest.mark.parametrize("square", [False, True], ids=["rows", "squares"])
def test_values_are_the_nearest_and_scales_the_least(e5m2, top, fraction, least, square):
    x = (torch.randn(200, 300) * torch.exp(4 * torch.randn(200, 1))).bfloat16()
    row, t = fb.quantize(x, e5m2, square, True, True)
    for q, v in ((row, x.double()), (t, x.t().double())):
        rows, k = v.shape
        scale = torch.exp2(q.scales.double().t() - 127).repeat_interleave(128, 1)[:, :k]
        blocks = torch.nn.functional.pad(v, (0, -k % 128)).view(rows, -1, 128).abs().amax(2)
        if square:
            blocks = torch.nn.functional.pad(blocks, (0, 0, 0, -rows % 128)).view(-1, 128, blocks.shape[1]).amax(1).repeat_interleave(128, 0)[:rows]
        largest = blocks.repeat_interleave(128, 1)[:, :k]
        assert bool((largest <= top * scale).all()) and bool((largest > top * scale / 2).all())
        # half a step: of the value, or of the smallest numbers
        half = torch.maximum(torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(1e-300))) - fraction - 1), scale * 2.0 ** (least - fraction - 1))
        assert bool(((fb._values(q).double() - v).abs() <= half).all())
        assert torch.equal(q.dequantize().float(), fb._values(q))


def test_not_finite_and_zero_blocks():
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    x[0, 3], x[0, 4], x[1, 200], x[2, 5] = float("inf"), 3.0, float("nan"), 2.0**-133
    q, _ = fb.quantize(x)
    v = fb._values(q)
    assert v[0].isnan().nonzero().flatten().tolist() == [3] and v[0, 4] == 3 and v[1].isnan().nonzero().flatten().tolist() == [200]
    assert q.scales[:, 3].tolist() == [127, 127] and q.scales[0, 2] == 1


def test_products_against_64_bits():
    a, b = torch.randn(5, 300).bfloat16(), torch.randn(70, 300).bfloat16()
    qa, qb = fb.quantize(a, True)[0], fb.quantize(b, square=True)[0]
    av, bv = fb._values(qa).double(), fb._values(qb).double()
    want, mag = av @ bv.t(), av.abs() @ bv.abs().t()
    close = lambda got, w: bool(((got.double() - w).abs() <= HALF_BF16 * w.abs() * (1 + 2**-7) + 302 * 2.0**-24 * mag).all())   # noqa: E731
    got = fb.mm(qa, qb)
    assert close(got, want)
    assert bool(((fb.mm(qa, qb, dtype=torch.float32).double() - want).abs() <= 302 * 2.0**-24 * mag).all())
    out = torch.ones(5, 70, dtype=torch.bfloat16)
    assert close(fb.mm(qa, qb, out=out, accumulate=True), want + 1) and torch.equal(fb.mm(qa, qb, out=out), got)


def test_layer_gradients_of_the_formulas():
    """Against autograd of the same arithmetic in 64 bits, where each cast hands its gradient through."""
    x, r, gain, w = (torch.randn(*s).bfloat16().requires_grad_() for s in ((3, 50, 264), (3, 50, 264), (264,), (72, 264)))
    dt, dy = torch.randn(3, 50, 264).bfloat16(), torch.randn(3, 50, 72).bfloat16()
    t, y = fb.norm_linear(x, r, gain, [w])
    got = torch.autograd.grad((t, y), (x, r, gain, w), (dt, dy))
    x64, r64, g64 = (p.detach().double().requires_grad_() for p in (x, r, gain))
    total = x64 + r64
    t64 = total + (total.detach().bfloat16().double() - total.detach())
    h = t64 * (t64.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * g64
    w8 = fb._values(fb._cast_rows(w.detach().float(), False, True)).double()
    g8 = fb._values(fb._cast_rows(dy.view(150, 72).float(), False)).double().view(3, 50, 72)
    (h * (g8 @ w8)).sum().backward(retain_graph=True)   # dh = q(dy) q(W)
    total.backward(dt.double())
    for a, b in zip(got, (x64.grad, r64.grad, g64.grad)):
        # one rounding
        assert ((a.double() - b).norm() / b.norm()).item() <= HALF_BF16
    ht = fb._values(fb._cast_rows((h.detach().view(150, 264).t()).float().contiguous(), False)).double()
    gt = fb._values(fb._cast_rows(dy.view(150, 72).t().float().contiguous(), False)).double()
    dw = gt @ ht.t()
    assert ((got[3].double() - dw).norm() / dw.norm()).item() <= 2 * HALF_BF16


def test_a_graph_goes_one_way_only():
    x, w = torch.randn(4, 64).bfloat16().requires_grad_(), torch.randn(8, 64).bfloat16().requires_grad_()
    (g,) = torch.autograd.grad(fb.linear(x, [w]).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_kept_weights_follow_writes():
    w = torch.randn(32, 64).bfloat16().requires_grad_()
    row, t = fb.quantized_weight([w], want_t=True)
    assert fb.quantized_weight([w], want_t=False)[0] is row and fb.quantized_weight([w], want_t=True)[1] is t
    with torch.no_grad():
        w.mul_(2)
    new, _ = fb.quantized_weight([w], want_t=False)
    assert torch.equal(fb._values(new), 2 * fb._values(row))
    import copy

    assert copy.deepcopy(w)._kf_fp8_block_cache is None if hasattr(copy.deepcopy(w), "_kf_fp8_block_cache") else True


def _ok(k=200, rows=6):
    return fb.quantize(torch.randn(rows, k).bfloat16())[0]


@pytest.mark.parametrize("call", [
    lambda: fb.quantize(torch.randn(4, 8)),                                                       # fp32
    lambda: fb.quantize(torch.randn(4, 8, 2).bfloat16()),
    lambda: fb.mm(_ok(200), _ok(128)),                                                            # inner dimensions
    lambda: fb.mm(fb.BlockScaled(_ok().values.float(), _ok().scales), _ok()),
    lambda: fb.mm(fb.BlockScaled(_ok().values, _ok().scales.t()), _ok()),                         # scales of another shape
    lambda: fb.mm(fb.BlockScaled(_ok().values, _ok().scales[:1]), _ok()),
    lambda: fb.mm(fb.BlockScaled(_ok(6, 6).values.t(), _ok(6, 6).scales), _ok(6)),                # columns not contiguous
    lambda: fb.mm(_ok(), _ok(), out=torch.empty(6, 6, dtype=torch.float16)),
    lambda: fb.mm(_ok(), _ok(), dtype=torch.float64),
    lambda: fb.mm(_ok(), _ok(), out=torch.empty(6, 6), dtype=torch.bfloat16),
    lambda: fb.mm(_ok(), _ok(), out=torch.empty(6, 7, dtype=torch.bfloat16)),
    lambda: fb.mm(_ok(), _ok(), out=torch.empty(6, 6, dtype=torch.bfloat16).t()),
    lambda: fb.mm(_ok(), _ok(), out=torch.empty(1, 6, dtype=torch.bfloat16).expand(6, 6)),        # rows on one another
    lambda: fb.mm(_ok(), fb.BlockScaled(*(t.to("meta") for t in _ok()[:2]))),                     # another device
    lambda: fb.BlockScaled(_ok().values, _ok().scales.int()).dequantize(),
    lambda: fb.BlockScaled(*(torch.empty(s, device="meta", dtype=torch.uint8) for s in ((2**31, 1), (1, 2**31)))).dequantize(),   # too many rows
    lambda: fb.quantize(torch.empty(1, 2**32 + 1, device="meta", dtype=torch.bfloat16)),
    lambda: fb.add_rmsnorm(torch.empty(2**32 + 1, 8, device="meta", dtype=torch.bfloat16), None, torch.empty(8, device="meta", dtype=torch.bfloat16)),
    lambda: fb.add_rmsnorm(torch.randn(4, 12).bfloat16(), None, torch.ones(12).bfloat16()),       # rows of 12
    lambda: fb.add_rmsnorm(torch.randn(4, 32776).bfloat16(), None, torch.ones(32776).bfloat16()),
    lambda: fb.add_rmsnorm(torch.randn(2, 4, 16).bfloat16(), None, torch.ones(16).bfloat16()),
    lambda: fb.add_rmsnorm(torch.randn(4, 16).bfloat16(), torch.randn(16).bfloat16(), torch.ones(16).bfloat16()),
    lambda: fb.add_rmsnorm(torch.randn(4, 16).bfloat16(), None, torch.ones(16)),
    lambda: fb.linear(torch.randn(4, 16).bfloat16(), []),
    lambda: fb.linear(torch.randn(4, 16).bfloat16(), [torch.randn(8, 24).bfloat16()]),
    lambda: fb.linear(torch.randn(4, 16), [torch.randn(8, 16)]),
    lambda: fb.linear(torch.randn(4, 16).bfloat16(), [torch.randn(8, 16)]),
    lambda: fb.norm_linear(torch.randn(4, 20).bfloat16(), None, torch.ones(20).bfloat16(), [torch.randn(8, 20).bfloat16()]),
    lambda: fb.norm_linear(torch.randn(4, 16).bfloat16(), torch.randn(1, 16).bfloat16(), torch.ones(16).bfloat16(), [torch.randn(8, 16).bfloat16()]),
])
def test_refusals(call):
    with pytest.raises(ValueError):
        call()


def test_no_rows():
    x, gain, w = torch.randn(0, 16).bfloat16().requires_grad_(), torch.ones(16).bfloat16().requires_grad_(), torch.randn(8, 16).bfloat16().requires_grad_()
    t, y = fb.norm_linear(x, None, gain, [w])
    y.float().sum().backward()
    assert y.shape == (0, 8) and w.grad.shape == (8, 16) and not w.grad.any() and not gain.grad.any()
    assert fb.mm(fb.quantize(torch.randn(3, 0).bfloat16())[0], fb.quantize(torch.randn(2, 0).bfloat16())[0]).tolist() == [[0, 0]] * 3


def test_without_gradients_nothing_is_made_for_a_backward(monkeypatch):
    """A transposed copy serves a gradient only: weights that want one do not bring it where none is recorded."""
    wanted, real = [], fb.quantize
    monkeypatch.setattr(fb, "quantize", lambda x2, *a, **kw: wanted.append(kw.get("want_t", False)) or real(x2, *a, **kw))
    x, gain = torch.randn(4, 64).bfloat16().requires_grad_(), torch.ones(64).bfloat16().requires_grad_()
    for quiet in (torch.no_grad, torch.inference_mode):
        ws = [torch.randn(8, 64).bfloat16().requires_grad_() for _ in range(2)]
        with quiet():
            fb.linear(x, ws[:1])
            fb.norm_linear(x, None, gain, ws[1:])
        assert len(wanted) == 3 and not any(wanted) and all(w._kf_fp8_block_cache.transposed is None for w in ws)
        wanted.clear()
    y, (_, z) = fb.linear(x, ws[:1]), fb.norm_linear(x, None, gain, ws[1:])
    assert wanted == [True, True, True]        # x, and the transposed copies of the kept weights
    (y.float().sum() + z.float().sum()).backward()
    assert all(p.grad is not None and bool(p.grad.any()) for p in (x, gain, *ws))


def test_kept_weights_of_another_device_go_by_its_stream(monkeypatch):
    """The stream that copies belong to, and whether a graph is captured, are asked of the weights' device, not of the current one."""
    import contextlib
    import types

    current = [0]

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], d.index
        yield
        current[0] = before

    seen = []
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(fb.fp8, "weights_state", lambda ws: seen.append(current[0]))
    monkeypatch.setattr(fb, "quantize", lambda *a, **kw: seen.append(current[0]) or (None, None))
    monkeypatch.setattr(fb, "_others", lambda: (None, types.SimpleNamespace(_stack_weight_rows=lambda ws: torch.empty(1, 1))))
    for index in (0, 1):
        w = types.SimpleNamespace(is_cuda=True, device=torch.device("cuda", index))
        fb.quantized_weight([w], want_t=False)
        assert seen == [index, index] and current == [0]
        seen.clear()
