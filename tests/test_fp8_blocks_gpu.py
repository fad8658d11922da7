"""The kernels of fp8 with a scale for each block of 128 against plain arithmetic in 64 bits."""

import pytest
import torch

from kempnerforge_b200.ops import fp8_blocks as fb

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALF_BF16 = 2.0**-8        # bf16 has 7 fraction bits: a step at 1 is 2^-7 (torch.finfo(torch.bfloat16).eps), a rounding is off by half of it


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _spread(rows, cols, seed, dtype=torch.bfloat16):
    """Rows of very different size, some columns large, zeros among them."""
    g = _gen(seed)
    x = torch.randn(rows, cols, device=DEV, generator=g) * torch.exp(4 * torch.randn(rows, 1, device=DEV, generator=g))
    x[:, :: max(2, cols // 3)] *= 50
    x[torch.rand(rows, cols, device=DEV, generator=g) < 0.05] = 0
    if rows > 2:
        x[rows // 2] = 0
    return x.to(dtype)


def _same(a, b):
    return torch.equal(a.values, b.values) and torch.equal(a.scales, b.scales)


def _plain(x2, e5m2, square):
    return fb._cast_rows(x2.float(), e5m2, square)


SHAPES = [(1, 1), (1, 128), (3, 129), (127, 40), (128, 128), (130, 1000), (257, 776), (1, 4096), (1000, 264)]


@pytest.mark.parametrize("square", [False, True], ids=["rows", "squares"])
@pytest.mark.parametrize("e5m2", [False, True], ids=["e4m3", "e5m2"])
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_cast_gives_the_defined_bytes_both_ways(native_lib, rows, cols, e5m2, square):
    x = _spread(rows, cols, rows + cols)
    row, t = fb.quantize(x, e5m2, square, True, True)
    assert _same(row, _plain(x, e5m2, square)) and _same(t, _plain(x.t().contiguous(), e5m2, square))
    assert _same(fb.quantize(x, e5m2, square)[0], row) and _same(fb.quantize(x, e5m2, square, False, True)[1], t)
    if square:
        assert torch.equal(row.values, t.values.t())
    exact = fb._values(row)
    assert torch.equal(row.dequantize(), exact.bfloat16()) and torch.equal(row.dequantize().float(), exact)


def test_cast_reads_pitched_rows_and_writes_nothing_else(native_lib):
    frame = _spread(70, 400, 1)
    for view in (frame[:, 8:285], frame[3:, 5:300], frame.t()[:, 1:60], frame[:1].expand(40, 400)):
        row, t = fb.quantize(view, want_t=True)
        assert _same(row, _plain(view, False, False)) and _same(t, _plain(view.t().contiguous(), False, False))


@pytest.mark.parametrize("e5m2", [False, True], ids=["e4m3", "e5m2"])
def test_cast_at_borders_of_scales_and_at_the_ends_of_the_range(native_lib, e5m2):
    top = 57344.0 if e5m2 else 448.0
    x = torch.zeros(12, 128, device=DEV, dtype=torch.bfloat16)
    x[0, 5], x[1, 5], x[2, 5] = top, top * (1 + 2**-7), -top * 2.0**-20      # just fits; the next bf16 value does not
    x[3], x[4, 0] = 2.0**-130, 2.0**-133                                     # subnormal numbers only
    x[5, 0], x[5, 1] = 3.3e38, 1e-38
    x[6, 3], x[6, 4] = float("inf"), 2.0
    x[7, 9], x[7, 8] = float("nan"), -3.0
    x[8] = float("-inf")
    x[9] = -0.0
    x[10, ::2], x[11, 127] = 1.0, 2.0**-140
    row, t = fb.quantize(x, e5m2, want_t=True)
    want, want_t = _plain(x, e5m2, False), _plain(x.t().contiguous(), e5m2, False)
    for got, ref in ((row, want), (t, want_t)):
        assert torch.equal(got.scales, ref.scales)
        a, b = fb._values(got), fb._values(ref)
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
    assert row.scales[0, 0] == 127 and row.scales[0, 1] == 128 and row.scales[0, 9] == 127
    assert fb._values(row)[6].isnan().sum() == 1 and fb._values(row)[6, 4] == 2 and fb._values(row)[7, 8] == -3


def _mm_case(m, n, k, ea, eb, seed=0):
    a = fb.quantize(_spread(m, k, seed + 1), ea)[0]
    b = fb.quantize(_spread(n, k, seed + 2), eb)[0]
    return a, b, fb._values(a).double(), fb._values(b).double()


def _mm_close(got, want, mag, k):
    """One rounding to bf16, and a sum in 32 bits of k terms (2^-23 of the terms' sum each, for hardware that truncates)."""
    err = (got.double() - want).abs()
    return bool((err <= HALF_BF16 * want.abs() * (1 + 2**-7) + (k + 2) * 2.0**-23 * mag + 1e-38).all())


MM = [(1, 1, 1), (1, 4096, 512), (2, 24, 136), (16, 128, 128), (17, 1001, 777), (64, 256, 2048), (100, 136, 40), (128, 224, 640),
      (129, 225, 129), (200, 512, 1536), (256, 448, 256), (257, 300, 1000), (333, 1001, 777), (513, 96, 384), (700, 1792, 520),
      (300, 200, 4096), (260, 1000, 8200), (2001, 72, 2048), (72, 2001, 2048), (1300, 1304, 900), (5000, 40, 1000), (3000, 2999, 136),
      (5, 4096, 4097), (619, 1080, 5316), (200, 4096, 14300), (1300, 190, 6000)]


@pytest.mark.parametrize("ea, eb", [(False, False), (True, False), (False, True), (True, True)], ids=["e4m3", "e5m2xe4m3", "e4m3xe5m2", "e5m2"])
@pytest.mark.parametrize("m, n, k", MM)
def test_product(native_lib, m, n, k, ea, eb):
    a, b, av, bv = _mm_case(m, n, k, ea, eb)
    want, mag = av @ bv.t(), av.abs() @ bv.abs().t()
    got = fb.mm(a, b)
    assert got.is_contiguous() and got.shape == (m, n)
    assert _mm_close(got, want, mag, k)
    assert torch.equal(got, fb.mm(a, b))
    assert native_lib.read_status() == 0


@pytest.mark.parametrize("m, n, k", [(1, 1000, 700), (9, 129, 4096), (20, 256, 300), (300, 521, 384), (300, 200, 4096), (72, 2001, 2048), (700, 1792, 520)])
def test_product_in_32_bits(native_lib, m, n, k):
    a, b, av, bv = _mm_case(m, n, k, False, True, 5)
    want, mag = av @ bv.t(), av.abs() @ bv.abs().t()
    got = fb.mm(a, b, dtype=torch.float32)
    bound = (k + 2) * 2.0**-23 * mag + 1e-38
    assert got.dtype == torch.float32 and bool(((got.double() - want).abs() <= bound).all())
    frame = torch.full((m + 1, n + 5), 7.0, device=DEV)
    old = _spread(m, n, 3, torch.float32)
    frame[:m, 1 : n + 1] = old
    fb.mm(a, b, out=frame[:m, 1 : n + 1], accumulate=True)
    assert bool(((frame[:m, 1 : n + 1].double() - want - old.double()).abs() <= bound + 2.0**-23 * (old.double().abs() + want.abs())).all())
    assert bool((frame[m] == 7).all()) and bool((frame[:, 0] == 7).all()) and bool((frame[:, n + 1 :] == 7).all())
    assert native_lib.read_status() == 0


@pytest.mark.parametrize("m, n, k", [(5, 200, 300), (64, 129, 256), (300, 520, 384), (300, 521, 384), (264, 1000, 4096), (261, 1000, 4096), (1304, 296, 4096), (1300, 297, 2048)])
def test_product_adds_into_a_pitched_output_and_leaves_the_rest(native_lib, m, n, k):
    a, b, av, bv = _mm_case(m, n, k, False, False, 7)
    want, mag = av @ bv.t(), av.abs() @ bv.abs().t()
    for first, pitch in ((0, -(-n // 8) * 8 + 8), (1, n + 3)):
        frame = torch.full((m + 2, pitch), 7.0, dtype=torch.bfloat16, device=DEV)
        out = frame[1 : m + 1, first : first + n]
        assert fb.mm(a, b, out=out).data_ptr() == out.data_ptr()
        assert torch.equal(out, fb.mm(a, b))
        old = _spread(m, n, 3)
        out.copy_(old)
        fb.mm(a, b, out=out, accumulate=True)
        assert _mm_close(out, want + old.double(), mag + old.double().abs(), k)
        out.fill_(7.0)
        assert bool((frame == 7.0).all())
    assert native_lib.read_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("m, n, k", [(40, 4104, 300), (300, 520, 384), (1304, 296, 4096), (72, 2008, 2048), (2008, 72, 520), (1800, 7256, 136)])
def test_product_adds_into_a_contiguous_output(native_lib, m, n, k, dtype):
    a, b, av, bv = _mm_case(m, n, k, False, False, 17)
    want, mag = av @ bv.t(), av.abs() @ bv.abs().t()
    old = _spread(m, n, 3, dtype)
    out = fb.mm(a, b, out=old.clone(), accumulate=True)
    total, size = want + old.double(), mag + old.double().abs()
    if dtype == torch.bfloat16:
        assert _mm_close(out, total, size, k)
    else:
        assert bool(((out.double() - total).abs() <= (k + 4) * 2.0**-23 * size + 1e-38).all())
    assert native_lib.read_status() == 0


def test_product_of_slices_and_of_scales_at_the_ends(native_lib):
    a, b, av, bv = _mm_case(40, 72, 512, False, False, 9)
    part = fb.mm(fb.BlockScaled(a.values[3:20, 128:384], a.scales[1:3, 3:20]), fb.BlockScaled(b.values[5:, 128:384], b.scales[1:3, 5:]))
    want = av[3:20, 128:384] @ bv[5:, 128:384].t()
    assert _mm_close(part, want, av[3:20, 128:384].abs() @ bv[5:, 128:384].abs().t(), 256)
    for rows in (1, 9, 40, 300):                                              # of each kernel
        one = torch.full((rows, 128), 0x38, dtype=torch.uint8, device=DEV)    # 1.0 in e4m3
        s = lambda v, pitch=-(-rows // 16) * 16: torch.full((1, pitch), v, dtype=torch.uint8, device=DEV)[:, :rows]   # noqa: E731, B023
        for sa, sb in ((127, 127), (254, 1), (1, 254), (254, 0), (0, 254), (1, 200), (60, 194), (194, 60), (100, 100), (254, 100), (120, 120)):
            for a8, b8 in ((False, False), (False, True), (True, False)):
                v = one if not a8 else torch.full_like(one, 0x3C), one if not b8 else torch.full_like(one, 0x3C)      # 1.0 in e5m2
                got = fb.mm(fb.BlockScaled(v[0], s(sa), a8), fb.BlockScaled(v[1], s(sb), b8))
                assert bool((got.double() == 128 * 2.0 ** (sa + sb - 254)).all()), (rows, sa, sb, got)
        for sa, sb in ((255, 127), (127, 255), (255, 0)):
            assert fb.mm(fb.BlockScaled(one, s(sa)), fb.BlockScaled(one, s(sb))).isnan().all()


def test_what_is_not_finite_stays_in_its_row_and_column(native_lib):
    x, w = _spread(40, 300, 3), _spread(50, 300, 4)
    clean = fb.mm(fb.quantize(x)[0], fb.quantize(w)[0])
    x2, w2 = x.clone(), w.clone()
    x2[7, 200], w2[11, 5] = float("inf"), float("nan")
    got = fb.mm(fb.quantize(x2)[0], fb.quantize(w2)[0])
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[7], bad[:, 11] = True, True
    assert torch.equal(got.isnan(), bad)
    assert torch.equal(got[~bad], clean[~bad])


def _cast64(v):
    """Bytes and block-major scales of finite `v` (rows, k) in 64 bits, e4m3, from the definition."""
    rows, k = v.shape
    blocks = torch.nn.functional.pad(v, (0, -k % 128)).view(rows, -1, 128)
    mant, ex = torch.frexp(blocks.abs().amax(2))
    e = torch.where(mant > 0, (ex - 9 + (mant > 0.875)).clamp_min(-126), 0)
    q = blocks * torch.exp2(-e.double())[:, :, None]
    step = torch.exp2((torch.frexp(q)[1] - 1).clamp_min(-6).double() - 3)
    return (torch.round(q / step) * step).view(rows, -1)[:, :k].float().to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).t().to(torch.uint8)


NORM = [(1, 8), (1, 4096), (3, 136), (5, 1024), (130, 1032), (64, 4104), (33, 8200), (50, 2056), (700, 2560), (700, 2056), (20, 5128), (70, 4864), (2000, 6144), (8200, 264), (2, 16392), (2, 32768), (1000, 776)]


@pytest.mark.parametrize("with_residual", [False, True], ids=["alone", "residual"])
@pytest.mark.parametrize("rows, d", NORM)
def test_norm(native_lib, rows, d, with_residual):
    x, gain = _spread(rows, d, d), (1 + 0.2 * torch.randn(d, device=DEV, generator=_gen(1))).bfloat16()
    residual = _spread(rows, d, d + 1) if with_residual else None
    t, rstd, h = fb.add_rmsnorm(x, residual, gain, 1e-5)
    assert torch.equal(t, x if residual is None else (x.float() + residual.float()).bfloat16())
    want = (t.double().square().mean(1) + 1e-5).rsqrt()
    # a sum of d squares (2^-24 each, at most d of them one after another) under a square root, and an approximate one (2^-22)
    assert bool(((rstd.double() - want).abs() <= want * (d * 2.0**-25 + 2.0**-21)).all())
    q, scales = _cast64(t.double() * gain.double() / (t.double().square().mean(1) + 1e-5).sqrt()[:, None])
    assert torch.equal(h.scales, scales) and torch.equal(h.values, q)
    normed = fb._normed_t(t, rstd, gain)
    assert _same(normed, fb._cast_rows((t.float() * gain.float() * rstd[:, None]).t().contiguous(), False))
    again = fb.add_rmsnorm(x, residual, gain, 1e-5)
    assert torch.equal(again[1], rstd) and _same(again[2], h)


def test_norm_of_rows_with_infinities_and_zeros(native_lib):
    x = torch.randn(6, 264, device=DEV, generator=_gen(0)).bfloat16()
    x[1, 3], x[2, 200], x[3] = float("inf"), float("nan"), 0
    gain = torch.ones(264, device=DEV, dtype=torch.bfloat16)
    t, rstd, h = fb.add_rmsnorm(x, None, gain)
    v = fb._values(h)
    assert rstd[1] == 0 and rstd[2].isnan() and v[1].isnan().sum() == 1 and v[2].isnan().all() and not v[3].any()
    assert v[[0, 3, 4, 5]].isfinite().all()
    gain[5] = float("inf")                                       # of one column: NaN there, the rest of its block scaled as without it
    got = fb.add_rmsnorm(x[4:], None, gain)[2]
    assert _same(got, fb._cast_rows(x[4:].float() * gain.float() * fb.add_rmsnorm(x[4:], None, gain)[1][:, None], False))
    assert fb._values(got).isnan().sum() == 2


def test_norm_of_rows_at_the_ends_of_the_types(native_lib):
    one = lambda *s: torch.ones(*s, device=DEV, dtype=torch.bfloat16)   # noqa: E731
    # rstd a power of two: products are exact, and halfway between two 8-bit numbers they go to the even one
    gain = torch.tensor([1, 1.0625, 1.1875, 1.9375, 448, 416, 1.4375, -1.0625], device=DEV).bfloat16()
    for size in (1.0, 2.0**-12, 2.0**30):
        t, rstd, h = fb.add_rmsnorm(size * one(3, 8), None, gain, 0.0)
        assert bool((rstd == 1 / size).all())
        assert fb._values(h).tolist() == [[1, 1, 1.25, 2, 448, 416, 1.5, -1]] * 3
    # a product that 32 bits do not hold is NaN, the rest of its block scaled as if it were not there
    x, big = 2.0**-10 * one(1, 8), torch.full((8,), 3.3e38, device=DEV).bfloat16()
    x[0, 2], big[5] = 2.0**-8, 0
    v = fb._values(fb.add_rmsnorm(x, None, big, 0.0)[2])[0]
    want = big.double()[0] / (x.double().square().mean()).sqrt() * 2.0**-10
    assert v[2].isnan() and v[5] == 0 and bool(((v[[0, 1, 3, 4, 6, 7]].double() - want).abs() <= want * 2.0**-4).all())
    # squares that 32 bits do not hold: rstd is 0, and so are the finite values; a row of zeros without eps has none
    t, rstd, h = fb.add_rmsnorm(torch.cat([1e30 * one(1, 8), -1e30 * one(1, 8), 0 * one(1, 8)]), None, one(8), 0.0)
    assert rstd[:2].tolist() == [0, 0] and not fb._values(h)[:2].any() and h.scales[:, :2].tolist() == [[127, 127]]
    assert rstd[2].isinf() and fb._values(h)[2].isnan().all()
    assert native_lib.read_status() == 0


def _layer(tokens, d, outs, seed=0, grads=True):
    g = _gen(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, device=DEV, generator=g) * std).bfloat16()   # noqa: E731
    x, residual, gain = r(*tokens, d), r(*tokens, d), 1 + r(d, std=0.1)
    ws = [r(n, d, std=d**-0.5) for n in outs]
    if grads:
        for p in (x, residual, gain, *ws):
            p.requires_grad_()
    return x, residual, gain, ws, r(*tokens, d, std=0.1), r(*tokens, sum(outs), std=0.1)


def _norm_grads64(dh, t, gain, dt, eps):
    t, gain, dh = t.double(), gain.double(), dh.double()
    r = (t.square().mean(1, keepdim=True) + eps).rsqrt()
    g = dh * gain
    mean = (g * t).mean(1, keepdim=True)
    mag = (r * g).abs() + t.abs() * r**3 * (g * t).abs().mean(1, keepdim=True) + dt.double().abs()
    return r * g - t * r**3 * mean + dt.double(), mag, (dh * t * r).sum(0), (dh * t * r).abs().sum(0)


@pytest.mark.parametrize("with_residual", [False, True], ids=["alone", "residual"])
@pytest.mark.parametrize("tokens, d, outs", [((1,), 64, (40,)), ((3, 77), 264, (128, 40, 40)), ((257,), 768, (776,)), ((2, 300), 1024, (512, 512)), ((3,), 8200, (72,))])
def test_layer_and_its_gradients(native_lib, tokens, d, outs, with_residual):
    x, residual, gain, ws, dt, dy = _layer(tokens, d, outs)
    if not with_residual:
        residual = None
    t, y = fb.norm_linear(x, residual, gain, ws, 1e-5)
    leaves = [p for p in (x, residual, gain, *ws) if p is not None]
    got = dict(zip(["x"] + ["r"] * with_residual + ["gain"] + [f"w{i}" for i in range(len(ws))], torch.autograd.grad((t, y), leaves, (dt, dy))))
    rows = x.numel() // d
    t2, dy2, dt2 = t.detach().view(rows, d), dy.view(rows, -1), dt.view(rows, d)
    h, w = fb.add_rmsnorm(x.detach().view(rows, d), None if residual is None else residual.detach().view(rows, d), gain.detach()), torch.cat([p.detach() for p in ws])
    assert torch.equal(t2, h[0])
    hv, wv, gv = fb._values(h[2]).double(), fb._values(_plain(w, False, True)).double(), fb._values(_plain(dy2, False, False)).double()
    assert _mm_close(y.detach().view(rows, -1), hv @ wv.t(), hv.abs() @ wv.abs().t(), d)
    # dh stays in 32 bits, but for rows too wide for the kernel of the norm's gradients
    dh, dh_mag = gv @ wv, gv.abs() @ wv.abs()
    dh_err = (w.shape[0] + 2) * 2.0**-23 * dh_mag + (HALF_BF16 * dh.abs() * (1 + 2**-7) if d > 8192 else 0)
    dx, mag, dgain, dgain_mag = _norm_grads64(dh, t2, gain.detach(), dt2, 1e-5)
    _, err, _, gain_err = _norm_grads64(dh_err, t2, gain.detach().abs(), dt2 * 0, 1e-5)
    # 32-bit sums of d terms and of `rows` terms
    assert bool(((got["x"].view(rows, d).double() - dx).abs() <= err + HALF_BF16 * (dx.abs() + err) + d * 2.0**-22 * mag + 2.0**-20 * mag).all())
    if with_residual:
        assert torch.equal(got["r"], got["x"])
    assert bool(((got["gain"].double() - dgain).abs() <= gain_err + HALF_BF16 * (dgain.abs() + gain_err) + (rows + 8) * 2.0**-21 * dgain_mag).all())
    ht = fb._values(fb._cast_rows((t2.float() * gain.detach().float() * h[1][:, None]).t().contiguous(), False)).double()
    gt = fb._values(_plain(dy2.t().contiguous(), False, False)).double()
    dw = torch.cat([got[f"w{i}"] for i in range(len(ws))])
    assert _mm_close(dw, gt @ ht.t(), gt.abs() @ ht.abs().t(), rows)
    assert native_lib.read_status() == 0


@pytest.mark.parametrize("rows, d", [(1, 8), (3, 136), (3000, 1024), (130, 1032), (1000, 4096), (70, 4104), (33, 8192), (20, 8200)])
def test_gradients_of_the_norm(native_lib, rows, d):
    g = _gen(d)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)   # noqa: E731
    t, gain, dt, dh = (2 * r(rows, d)).bfloat16(), (1 + 0.2 * r(d)).bfloat16(), r(rows, d).bfloat16(), r(rows, d)
    rstd = (t.double().square().mean(1) + 1e-5).rsqrt().float()
    # rows too wide for the kernel of 32 bits: a rounding of dh to bf16, and a kernel that rounds less carefully
    err = dh.double().abs() * (HALF_BF16 if d > 8192 else 0)
    for with_dt in (dt, None):
        dx, dgain = fb._norm_grads(dh, t, gain, rstd, with_dt)
        want, mag, want_gain, gain_mag = _norm_grads64(dh, t, gain, dt if with_dt is not None else dt * 0, 1e-5)
        _, more, _, more_gain = _norm_grads64(err, t, gain.abs(), dt * 0, 1e-5)
        assert bool(((dx.double() - want).abs() <= more + HALF_BF16 * (want.abs() + more) + d * 2.0**-22 * mag).all())
        assert bool(((dgain.double() - want_gain).abs() <= more_gain + HALF_BF16 * (want_gain.abs() + more_gain) + (rows + 8) * 2.0**-22 * gain_mag).all())
        again = fb._norm_grads(dh, t, gain, rstd, with_dt)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dgain)


@pytest.mark.parametrize("lead", [(5,), (2, 150)])
def test_linear_and_its_gradients(native_lib, lead):
    d, outs = 200, (136, 48)
    x, _, _, ws, _, dy = _layer(lead, d, outs, 3)
    y = fb.linear(x, ws)
    dx, *dws = torch.autograd.grad(y, (x, *ws), dy)
    x2, dy2, w = x.detach().view(-1, d), dy.view(-1, sum(outs)), torch.cat([p.detach() for p in ws])
    v = lambda m, sq=False: fb._values(_plain(m, False, sq)).double()   # noqa: E731
    for got, a, b in ((y.detach().view(-1, sum(outs)), v(x2), v(w, True)), (dx.view(-1, d), v(dy2), v(w, True).t()),
                      (torch.cat(dws), v(dy2.t().contiguous()), v(x2.t().contiguous()))):
        assert _mm_close(got, a @ b.t(), a.abs() @ b.abs().t(), a.shape[1])


def test_gradients_of_a_linear_agree_with_differences(native_lib):
    """Small whole numbers are exact in 8 bits, so that all that differences of the loss are off by is the rounding of the outputs that the
    step changes (a row or a column of them; up to 136 * 49, so not all are exact in bf16): half a step of each, times its |c|."""
    g = _gen(5)
    whole = lambda *s, top: torch.randint(-top, top + 1, s, device=DEV, generator=g).bfloat16()   # noqa: E731
    x, w, c = whole(130, 136, top=7).requires_grad_(), whole(72, 136, top=7).requires_grad_(), whole(130, 72, top=2)
    dx, dw = torch.autograd.grad(fb.linear(x, [w]), (x, w), c)
    with torch.no_grad():
        for leaf, grad, other, at in ((x, dx, w, (3, 5)), (x, dx, w, (129, 135)), (w, dw, x, (71, 130)), (w, dw, x, (0, 0))):
            up, down = leaf.clone(), leaf.clone()
            up[at] += 1
            down[at] -= 1
            ys = [fb.linear(*((v, [other]) if leaf is x else (other, [v]))).double() for v in (up, down)]
            moved = (lambda v: v[at[0]]) if leaf is x else (lambda v: v[:, at[0]])
            slope = ((ys[0] - ys[1]) * c.double()).sum().item() / 2
            off = HALF_BF16 * sum((moved(v).abs() * (1 + 2**-7) * moved(c).double().abs()).sum().item() for v in ys) / 2
            assert abs(slope - grad[at].item()) <= off + HALF_BF16 * abs(grad[at].item()), (slope, grad[at], off)


def test_gradients_of_the_layer_agree_with_differences(native_lib):
    """Along a gradient the loss changes by its length; what the casts of two calls add to a difference is random: off by at most 2^-4 of
    a value, 0.03 of it in the mean square, which over the 512 x 256 outputs, each a sum, is 0.05 |c| |y| / sqrt(n) for one of them."""
    x, residual, gain, ws, _, c = _layer((512,), 256, (256,), 8)
    loss = lambda a, b, s: (fb.norm_linear(a, b, s, ws)[1].double() * c.double()).sum()   # noqa: E731
    t, y = fb.norm_linear(x, residual, gain, ws)
    grads = torch.autograd.grad(y, (x, residual, gain), c)
    noise = 0.05 * c.double().norm() * y.detach().double().norm() / y.numel() ** 0.5
    with torch.no_grad():
        for i, grad in enumerate(grads):
            leaves = [x, residual, gain]
            step = 0.05 * leaves[i].double().norm() / grad.double().norm()
            ends = []
            for sign in (1, -1):
                moved = list(leaves)
                moved[i] = (leaves[i].double() + sign * step * grad.double()).bfloat16()
                ends.append(loss(*moved))
            slope = ((ends[0] - ends[1]) / 2).item()
            want = (step * grad.double().square().sum()).item()
            # five deviations, and 5 % for the curvature over a step of 5 %
            assert abs(slope - want) <= 5 * noise.item() + 0.05 * want, (i, slope, want, noise)


def test_half_of_the_graph(native_lib):
    x, residual, gain, ws, dt, dy = _layer((40,), 264, (48,), 2)
    t, y = fb.norm_linear(x, residual, gain, ws)
    assert torch.equal(torch.autograd.grad(t, x, dt, retain_graph=True)[0], dt)          # the sum alone
    both = torch.autograd.grad((t, y), (x, gain, ws[0]), (dt, dy), retain_graph=True)
    only = torch.autograd.grad(y, (x, gain, ws[0]), dy, retain_graph=True)
    assert torch.equal(both[1], only[1]) and torch.equal(both[2], only[2])
    assert torch.equal(torch.autograd.grad(y, ws[0], dy)[0], both[2])
    for need in range(4):                                                                # one leaf at a time
        args = [p.detach().requires_grad_(i == need) for i, p in enumerate((x, residual, gain, ws[0]))]
        t, y = fb.norm_linear(args[0], args[1], args[2], args[3:])
        got = torch.autograd.grad(y, args[need], dy)[0]
        assert torch.equal(got, [only[0], only[0], only[1], only[2]][need])
    with torch.no_grad():
        quiet = fb.norm_linear(x, residual, gain, ws)
    assert torch.equal(quiet[1], y) and not quiet[1].requires_grad


def test_saved_on_the_host_and_expanded_gradients(native_lib):
    x, residual, gain, ws, _, dy = _layer((37,), 264, (40,), 4)
    want = torch.autograd.grad(fb.linear(x, ws), (x, *ws), dy)
    with torch.autograd.graph.save_on_cpu():
        y = fb.linear(x, ws)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, *ws), dy), want))
    y = fb.linear(x, ws)
    ones = torch.autograd.grad(y.float().sum(), (x, *ws))
    y = fb.linear(x, ws)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, *ws), torch.ones_like(y)), ones))


def test_no_tokens(native_lib):
    x, residual, gain, ws, _, _ = _layer((0,), 264, (40,), 4)
    t, y = fb.norm_linear(x, residual, gain, ws)
    grads = torch.autograd.grad((t.float().sum() + y.float().sum()), (x, residual, gain, *ws))
    assert y.shape == (0, 40) and grads[0].shape == x.shape and not grads[2].any() and not grads[3].any()
    y = fb.linear(x, ws)
    assert y.shape == (0, 40) and not torch.autograd.grad(y.float().sum(), ws[0])[0].any()


def test_captured_and_replayed_on_new_inputs_and_weights(native_lib):
    x, residual, gain, ws, _, _ = _layer((50,), 264, (136,), 6, grads=False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fb.norm_linear(x, residual, gain, ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t, y = fb.norm_linear(x, residual, gain, ws)
    for seed in (11, 12):
        new = _layer((50,), 264, (136,), seed, grads=False)
        for old, value in zip((x, residual, gain, *ws), (*new[:3], *new[3])):
            old.copy_(value)
        graph.replay()
        want = fb.norm_linear(*new[:3], new[3])
        assert torch.equal(t, want[0]) and torch.equal(y, want[1])
    assert native_lib.read_status() == 0


def test_two_streams_at_once(native_lib):
    cases = [_layer((300,), 512, (520,), s, grads=False) for s in (1, 2)]
    want = [fb.norm_linear(*c[:3], c[3]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(20):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(fb.norm_linear(*c[:3], c[3]))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_a_captured_step_gives_the_gradients_of_each_replay(native_lib):
    d, outs = 264, (136, 48)
    x, residual, gain, ws, dt, dy = _layer((70,), d, outs, 6)
    leaves = (x, residual, gain, *ws)

    def step():
        t, y = fb.norm_linear(x, residual, gain, ws)
        return t, y, *torch.autograd.grad((t, y), leaves, (dt, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                     # two graphs of the same step share nothing but their inputs
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got))
    for seed in (21, 22):
        new = _layer((70,), d, outs, seed)
        with torch.no_grad():
            for old, value in zip((*leaves, dt, dy), (*new[:3], *new[3], *new[4:])):
                old.copy_(value)
        for graph, got in graphs:
            for v in got:
                v.detach().fill_(7.0)
        for graph, _ in graphs:
            graph.replay()
        want = step()
        for _, got in graphs:
            for a, b in zip(got, want):
                assert torch.equal(a, b)
    assert native_lib.read_status() == 0


@pytest.mark.parametrize("m", [3, 70, 700])
def test_products_right_after_what_they_read_and_before_what_overwrites_it(native_lib, m):
    """Launches that overlap their predecessor's end: each cast, product and overwrite in a row sees what stands before it in the stream."""
    n, k, rounds = 520, 1040, 12
    xs, w = [_spread(m, k, s) for s in range(rounds)], fb.quantize(_spread(n, k, 99), square=True)[0]
    want = [fb.mm(fb.quantize(x)[0], w) for x in xs]
    torch.cuda.synchronize()
    x, out = torch.empty_like(xs[0]), torch.empty_like(want[0])
    a = fb.quantize(xs[0])[0]
    kept = []
    for v in xs:
        x.copy_(v)
        q = fb.quantize(x)[0]
        a.values.copy_(q.values)
        a.scales.copy_(q.scales)
        fb.mm(a, w, out=out)
        kept.append(out.clone())
        a.values.fill_(0x7F)                              # NaN: nothing may read it any more
        x.fill_(float("nan"))
        out.fill_(float("nan"))
    assert all(torch.equal(p, q) for p, q in zip(kept, want))
    assert native_lib.read_status() == 0


def test_the_checks_in_python_lead_to_the_same_kernels(native_lib, monkeypatch):
    x, residual, gain, ws, dt, dy = _layer((77,), 264, (128, 40), 12)

    def all_of():
        t, y = fb.norm_linear(x, residual, gain, ws)
        grads = torch.autograd.grad((t, y), (x, residual, gain, *ws), (dt, dy))
        z = fb.linear(x, ws)
        more = torch.autograd.grad(z, (x, *ws), dy)
        q, qt = fb.quantize(x.detach(), want_t=True)
        return [t, y, z, *grads, *more, *q[:2], *qt[:2], q.dequantize(), *fb.add_rmsnorm(x, None, gain)[:2], fb.mm(qt, qt, dtype=torch.float32)]

    native = all_of()
    before = native_lib.LAUNCH_COUNT
    all_of()
    launches = native_lib.LAUNCH_COUNT - before
    monkeypatch.setattr(native_lib, "_steps", False)
    before = native_lib.LAUNCH_COUNT
    plain = all_of()
    assert native_lib.LAUNCH_COUNT - before == launches > 0
    assert all(torch.equal(a, b) for a, b in zip(native, plain))


def test_refusals_on_a_gpu(native_lib):
    q = fb.quantize(torch.randn(6, 200, device=DEV).bfloat16())[0]
    host = fb.quantize(torch.randn(6, 200).bfloat16())[0]
    bf = lambda *s: torch.randn(*s, device=DEV).bfloat16()   # noqa: E731
    for call in (lambda: fb.mm(q, host), lambda: fb.mm(host, q), lambda: fb.mm(q, fb.quantize(bf(6, 199))[0]),
                 lambda: fb.mm(fb.BlockScaled(q.values, q.scales[:1]), q), lambda: fb.mm(fb.BlockScaled(q.values, host.scales), q),
                 lambda: fb.mm(q, q, out=bf(6, 7)), lambda: fb.mm(q, q, out=bf(1, 6).expand(6, 6)), lambda: fb.mm(q, q, out=torch.empty(6, 6, dtype=torch.bfloat16)),
                 lambda: fb.mm(fb.BlockScaled(q.values.float(), q.scales), q), lambda: fb.BlockScaled(q.values, q.scales.t()).dequantize(),
                 lambda: fb.quantize(torch.randn(4, 8, device=DEV)), lambda: fb.add_rmsnorm(bf(4, 12), None, bf(12)),
                 lambda: fb.add_rmsnorm(bf(4, 16), bf(4, 16).cpu(), bf(16)), lambda: fb.add_rmsnorm(bf(4, 16), None, bf(16).cpu()),
                 lambda: fb.norm_linear(bf(4, 16), None, bf(16), [bf(8, 16).cpu()]), lambda: fb.linear(bf(4, 16), [bf(8, 24)]),
                 lambda: fb.linear(bf(4, 16), [bf(8, 16).float()])):
        with pytest.raises(ValueError):
            call()
    assert native_lib.read_status() == 0


def test_operands_in_odd_places_of_memory(native_lib):
    """Bases and pitches that the kernels do not take are copied; what a view leaves out is not read into a result."""
    x, residual, gain, ws, _, _ = _layer((9,), 264, (40,), 14, grads=False)
    want = fb.norm_linear(x, residual, gain, ws)

    def moved(t, by=1):
        flat = torch.full((t.numel() + 64,), float("nan"), dtype=t.dtype, device=DEV)
        out = flat[by : by + t.numel()].view(t.shape)
        return out.copy_(t)

    got = fb.norm_linear(moved(x), moved(residual, 3), moved(gain, 5), [moved(ws[0])])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    wide = torch.full((9, 300), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 20:284] = x
    assert torch.equal(fb.norm_linear(wide[:, 20:284], residual, gain, [ws[0].t().contiguous().t()])[1], want[1])
    a, b = fb.quantize(x)[0], fb.quantize(ws[0])[0]
    odd = lambda q: fb.BlockScaled(torch.nn.functional.pad(q.values, (3, 2), value=0x7F)[:, 3:267], torch.nn.functional.pad(q.scales, (1, 1), value=255)[:, 1:-1])   # noqa: E731
    assert torch.equal(fb.mm(odd(a), odd(b)), fb.mm(a, b)) and torch.equal(odd(a).dequantize(), a.dequantize())


def test_offsets_past_32_bits(native_lib):
    rows, d = (1 << 20) + 1030, 4096                              # 4.3 G values: matrices of 2, 1 and 4 bytes a value all end behind 2^32 bytes
    tail, last = slice(rows - 300, rows), 300
    x = torch.zeros(rows, d, device=DEV, dtype=torch.bfloat16)
    x[tail], x[:300] = _spread(last, d, 1), _spread(last, d, 2)
    gain = (1 + 0.2 * torch.randn(d, device=DEV, generator=_gen(1))).bfloat16()
    q, qt = fb.quantize(x, want_t=True)
    assert _same(fb.BlockScaled(q.values[tail], q.scales[:, tail]), fb.quantize(x[tail])[0])
    first = (rows - 300) // 128 * 128                             # transposed blocks of whole 128 rows start there
    part = fb.quantize(x[first:], want_row=False, want_t=True)[1]
    assert torch.equal(qt.values[:, first:], part.values) and torch.equal(qt.scales[first // 128 :], part.scales)
    assert torch.equal(q.dequantize()[tail], fb.BlockScaled(q.values[tail], q.scales[:, tail]).dequantize())
    del qt, part
    t, rstd, h = fb.add_rmsnorm(x, x, gain)
    want = fb.add_rmsnorm(x[tail], x[tail], gain)
    assert torch.equal(t[tail], want[0]) and torch.equal(rstd[tail], want[1]) and _same(fb.BlockScaled(h.values[tail], h.scales[:, tail]), want[2])
    del t, h
    # a tall operand, in either place, and an output whose rows lie far apart
    w, _, wv, _ = _mm_case(40, 40, d, False, False, 3)
    qv = fb._values(fb.BlockScaled(q.values[tail], q.scales[:, tail])).double()
    exact, mag = qv @ wv.t(), qv.abs() @ wv.abs().t()
    assert _mm_close(fb.mm(q, w)[tail], exact, mag, d) and _mm_close(fb.mm(w, q)[:, tail], exact.t(), mag.t(), d)
    frame = torch.zeros(rows, d, device=DEV, dtype=torch.bfloat16)
    fb.mm(q, w, out=frame[:, 8:48])
    assert _mm_close(frame[tail, 8:48], exact, mag, d) and not frame[tail, :8].any() and not frame[tail, 48:].any()
    del q, frame
    dh = torch.zeros(rows, d, device=DEV)
    dh[tail] = _spread(last, d, 4, torch.float32)
    dx, dgain = fb._norm_grads(dh, x, gain, rstd, x)
    small, small_gain = fb._norm_grads(dh[tail].clone(), x[tail].clone(), gain, rstd[tail].clone(), x[tail].clone())
    assert torch.equal(dx[tail], small)
    # sums of the same 300 terms and zeros, in another order (2^-24 a term) before the rounding
    size = (dh[tail].double() * x[tail].double() * rstd[tail].double()[:, None]).abs().sum(0)
    assert bool(((dgain.double() - small_gain.double()).abs() <= 2 * HALF_BF16 * dgain.double().abs() + 600 * 2.0**-24 * size).all())
    assert native_lib.read_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64, torch.int32])
def test_products_of_other_types_are_refused(native_lib, dtype):
    q = fb.quantize(torch.randn(6, 200, device=DEV).bfloat16())[0]
    for out in (None, torch.full((6, 6), 7.0, dtype=torch.bfloat16, device=DEV), torch.full((6, 6), 7.0, device=DEV)):
        with pytest.raises(ValueError):
            fb.mm(q, q, out=out, dtype=dtype)
        assert out is None or bool((out == 7).all())
    for out, other in ((torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)):
        with pytest.raises(ValueError):
            fb.mm(q, q, out=torch.empty(6, 6, dtype=out, device=DEV), dtype=other)


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
@pytest.mark.parametrize("m, n, k", [(6, 40, 200), (300, 264, 200)])
def test_a_product_moves_the_version_of_what_it_writes(native_lib, monkeypatch, m, n, k, native):
    if not native:
        monkeypatch.setattr(native_lib, "_steps", False)
    a, b = fb.quantize(_spread(m, k, 1))[0], fb.quantize(_spread(n, k, 2))[0]
    for accumulate in (False, True):
        out = torch.ones(m, n, device=DEV, dtype=torch.bfloat16)
        other = torch.ones(m, n, device=DEV, dtype=torch.bfloat16, requires_grad=True)
        y = out * other                                      # keeps `out` for its gradient
        fb.mm(a, b, out=out, accumulate=accumulate)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    # a weight that is written so has 8-bit copies of its new values
    w = torch.nn.Parameter(torch.randn(m, n, device=DEV).bfloat16())
    fb.quantized_weight([w], want_t=True)
    with torch.no_grad():
        fb.mm(a, b, out=w)
    kept, fresh = fb.quantized_weight([w], want_t=True), fb.quantize(w.detach(), square=True, want_t=True)
    assert all(_same(p, q) for p, q in zip(kept, fresh))
    with torch.inference_mode():
        quiet = torch.empty(m, n, device=DEV, dtype=torch.bfloat16)    # has no version
    assert torch.equal(fb.mm(a, b, out=quiet), w)


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
def test_more_tiles_than_one_dimension_of_a_grid_holds(native_lib, monkeypatch, native):
    if not native:
        monkeypatch.setattr(native_lib, "_steps", False)
    first = 128 * 65535 + 256                                  # of the rows that are not zero: further tiles than 65 535
    rows, last = first + 300, slice(first, first + 300)
    x = torch.zeros(rows, 24, device=DEV, dtype=torch.bfloat16)
    x[last] = _spread(300, 24, 1)
    for square in (False, True):
        q, qt = fb.quantize(x, square=square, want_t=True)
        want, want_t = fb.quantize(x[last], square=square, want_t=True)
        assert _same(fb.BlockScaled(q.values[last], q.scales[:, last]), want)
        assert torch.equal(qt.values[:, last], want_t.values) and torch.equal(qt.scales[first // 128 :], want_t.scales)
        assert not q.values[:first].any() and bool((q.scales[:, :first] == 127).all())
        assert not qt.values[:, :first].any() and bool((qt.scales[: first // 128] == 127).all())
        alone = fb.quantize(x, square=square, want_row=False, want_t=True)[1]
        assert _same(alone, qt)
        del q, qt, alone
    # a layer's gradients cast as many rows; small whole numbers are exact in 8 bits and in sums of 32, in any order
    g = _gen(2)
    whole = lambda *s: torch.randint(-7, 8, s, device=DEV, generator=g).bfloat16()   # noqa: E731
    gain, w = torch.ones(24, device=DEV, dtype=torch.bfloat16), whole(16, 24).requires_grad_()
    dy = torch.zeros(rows, 16, device=DEV, dtype=torch.bfloat16)
    x[last], dy[last] = whole(300, 24), whole(300, 16)
    x.requires_grad_()
    small = x.detach()[last].clone().requires_grad_()
    for normed in (False, True):
        layer = (lambda v: fb.norm_linear(v, None, gain, [w])[1]) if normed else (lambda v: fb.linear(v, [w]))   # noqa: B023
        dx, dw = torch.autograd.grad(layer(x), (x, w), dy)
        want, want_w = torch.autograd.grad(layer(small), (small, w), dy[last])
        assert torch.equal(dx[last], want) and not dx[:first].any()
        # normalised values: the same 300 terms, at most 7 * sqrt(24) each, in another order, and a rounding of both
        off = 2 * HALF_BF16 * want_w.double().abs() + 302 * 2.0**-23 * 300 * 35 if normed else 0
        assert bool(((dw.double() - want_w.double()).abs() <= off).all())
        del dx, dw
    assert native_lib.read_status() == 0


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
def test_values_of_more_columns_than_one_dimension_of_a_grid_holds(native_lib, monkeypatch, native):
    if not native:
        monkeypatch.setattr(native_lib, "_steps", False)
    first = 256 * 65535 + 512
    x = torch.zeros(3, first + 300, device=DEV, dtype=torch.bfloat16)
    x[:, first:] = _spread(3, 300, 4)
    x[1, :300] = 1.0
    q = fb.quantize(x)[0]
    v = q.dequantize()
    part = fb.BlockScaled(q.values[:, first:], q.scales[first // 128 :])
    assert torch.equal(v[:, first:].float(), fb._values(part)) and bool((v[1, :300] == 1).all())
    assert not v[0, :first].any() and not v[2, :first].any() and not v[1, 300:first].any()
    assert native_lib.read_status() == 0


@pytest.mark.parametrize("d", [8192, 8200, 16392, 32768])
def test_gradients_of_a_norm_keep_their_32_bits_at_any_width(native_lib, d):
    """256 and 257 in turn, of changing sign from row to row: all sums are exact in 32 bits, and 16 bits have no 257."""
    rows, dev = 300, dict(device=DEV)
    r, c = torch.arange(rows, **dev)[:, None], torch.arange(d, **dev)[None]
    dh = (256.0 + (r + c) % 2) * (1 - 2 * (r % 2))
    one = torch.ones(rows, d, dtype=torch.bfloat16, **dev)
    dx, dgain = fb._norm_grads(dh, one, one[0].clone(), torch.ones(rows, **dev), None)
    assert torch.equal(dx.float(), dh - dh.mean(1, keepdim=True)) and bool((dx.float().abs() == 0.5).all())
    assert torch.equal(dgain.float(), dh.sum(0)) and bool((dgain.float().abs() == rows / 2).all())


@pytest.mark.parametrize("rows, d", [(1, 8200), (20, 8200), (700, 8200), (33, 12296), (150, 16392), (449, 20000), (7, 24584), (2, 32768), (320, 32768)])
def test_gradients_of_wide_norms(native_lib, rows, d):
    g = _gen(d)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)   # noqa: E731
    t, gain, dt, dh = (2 * r(rows, d)).bfloat16(), (1 + 0.2 * r(d)).bfloat16(), r(rows, d).bfloat16(), r(rows, d)
    rstd = (t.double().square().mean(1) + 1e-5).rsqrt().float()
    for with_dt in (dt, None):
        dx, dgain = fb._norm_grads(dh, t, gain, rstd, with_dt)
        want, mag, want_gain, gain_mag = _norm_grads64(dh, t, gain, dt if with_dt is not None else dt * 0, 1e-5)
        assert bool(((dx.double() - want).abs() <= HALF_BF16 * want.abs() + d * 2.0**-22 * mag).all())
        assert bool(((dgain.double() - want_gain).abs() <= HALF_BF16 * want_gain.abs() + (rows + 8) * 2.0**-22 * gain_mag).all())
        again = fb._norm_grads(dh, t, gain, rstd, with_dt)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dgain)


@pytest.mark.parametrize("d", [8200, 32768])
def test_a_wide_layer_through_both_ways_of_checks(native_lib, monkeypatch, d):
    x, residual, gain, ws, dt, dy = _layer((40,), d, (72,), 3)

    def step():
        t, y = fb.norm_linear(x, residual, gain, ws)
        return torch.autograd.grad((t, y), (x, gain, ws[0]), (dt, dy))

    native, before = step(), native_lib.LAUNCH_COUNT
    step()
    launches = native_lib.LAUNCH_COUNT - before
    # the product before the norm's gradients is in 32 bits: all that dx and the gain's gradient are off by is its sums and one rounding
    t, rstd, _ = fb.add_rmsnorm(x.detach(), residual.detach(), gain.detach())
    gv, wv = fb._values(fb.quantize(dy)[0]).double(), fb._values(fb.quantize(ws[0].detach(), square=True)[0]).double()
    dh, dh_err = gv @ wv, 74 * 2.0**-23 * (gv.abs() @ wv.abs())
    want, mag, want_gain, gain_mag = _norm_grads64(dh, t, gain.detach(), dt, 1e-5)
    _, err, _, gain_err = _norm_grads64(dh_err, t, gain.detach().abs(), dt * 0, 1e-5)
    assert bool(((native[0].double() - want).abs() <= err + HALF_BF16 * (want.abs() + err) + d * 2.0**-22 * mag).all())
    assert bool(((native[1].double() - want_gain).abs() <= gain_err + HALF_BF16 * (want_gain.abs() + gain_err) + 48 * 2.0**-21 * gain_mag).all())
    monkeypatch.setattr(native_lib, "_steps", False)
    before = native_lib.LAUNCH_COUNT
    plain = step()
    assert native_lib.LAUNCH_COUNT - before == launches > 0
    assert all(torch.equal(a, b) for a, b in zip(native, plain))
    assert native_lib.read_status() == 0


@pytest.mark.parametrize("with_residual", [False, True], ids=["alone", "residual"])
@pytest.mark.parametrize("rows, d", NORM)
def test_rstd_is_the_nearest_32_bit_number(native_lib, rows, d, with_residual):
    """The sum has 64 bits and rstd about 48 before it is rounded: half a step of 32 bits (2^-24 of the value at most) and 2^-40 for what is
    before it, whatever the width."""
    x, gain = _spread(rows, d, d), torch.ones(d, device=DEV, dtype=torch.bfloat16)
    t, rstd, _ = fb.add_rmsnorm(x, _spread(rows, d, d + 1) if with_residual else None, gain, 1e-5)
    want = (t.double().square().mean(1) + 1e-5).rsqrt()
    assert bool(((rstd.double() - want).abs() <= want * (2.0**-24 + 2.0**-40)).all())
