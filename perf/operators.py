"""Operators of fp8 training with a scale for each block of 128: what is measured, in plain form and through the framework.

A matrix (rows, k) in this form is a byte per value (e4m3 or e5m2) and a byte per row and 128 columns, block-major: (ceil(k / 128), rows);
a value is its 8-bit number times two to the power of (byte - 127).

``product``  two such matrices (m, k) and (n, k) -> bf16 (m, n)
``norm``     t = x + residual, RMSNorm of t with a gain, in 8 bits with block scales -> t and the values that the bytes stand for
``layer``    a training step through the two and the casts between them: t = x + residual, y = RMSNorm(t) Wᵀ with 8-bit operands,
             and the gradients of x, residual, gain and W
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BLOCK = 128
EPS = 1e-5


def listed() -> list[dict]:
    return [
        # generation, one sequence: the fused q | k | v projection of a 7B block
        dict(name="product_1x6144x4096", kind="product", m=1, n=6144, k=4096, e5m2=False),
        # generation, a batch: gate | up of a 7B feed-forward
        dict(name="product_24x28672x4096", kind="product", m=24, n=28672, k=4096, e5m2=False),
        # a short prompt through a 7B down projection
        dict(name="product_200x4096x14336", kind="product", m=200, n=4096, k=14336, e5m2=False),
        # a small, odd projection: no size a multiple of 16
        dict(name="product_333x1001x777", kind="product", m=333, n=1001, k=777, e5m2=False),
        # an uneven prompt through a 13B q | k | v projection
        dict(name="product_1554x7168x5120", kind="product", m=1554, n=7168, k=5120, e5m2=False),
        # the training step: gate | up of a 7B feed-forward over 2 x 4096 tokens
        dict(name="product_8192x28672x4096", kind="product", m=8192, n=28672, k=4096, e5m2=False),
        # a weight gradient: e5m2 gradients, reduction over an uneven number of tokens
        dict(name="product_14336x4096x8190", kind="product", m=14336, n=4096, k=8190, e5m2=True),
        # generation: the norm before a projection
        dict(name="norm_1x4096", kind="norm", rows=1, dim=4096, residual=True),
        # a prompt of uneven length
        dict(name="norm_777x5120", kind="norm", rows=777, dim=5120, residual=True),
        # a training batch of 4 x 4096 tokens
        dict(name="norm_16384x4096", kind="norm", rows=16384, dim=4096, residual=True),
        # a small model's training step on a ragged batch
        dict(name="layer_999x768x2304", kind="layer", rows=999, dim=768, out=2304),
        # a 7B block's q | k | v projection in training, 4096 tokens
        dict(name="layer_4096x4096x6144", kind="layer", rows=4096, dim=4096, out=6144),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["product", "product", "product", "norm", "norm", "layer"])
    if kind == "product":
        while True:
            m, n, k = _log_int(rng, 1, 14336), _log_int(rng, 64, 28672), _log_int(rng, 64, 14336)
            if rng.random() < 0.5:   # the widths of projections, any number of rows
                n, k = -(-n // 64) * 64, -(-k // 64) * 64
            if m * n * k <= 8192 * 28672 * 4096:
                return dict(kind=kind, m=m, n=n, k=k, e5m2=rng.random() < 0.3)
    if kind == "norm":
        return dict(kind=kind, rows=_log_int(rng, 1, 16384), dim=8 * _log_int(rng, 16, 1024), residual=rng.random() < 0.7)
    return dict(kind=kind, rows=_log_int(rng, 16, 4096), dim=8 * _log_int(rng, 32, 640), out=8 * _log_int(rng, 32, 768))


# --------------------------------------------------------------------------- the 8-bit form
def _scale_bytes(largest: torch.Tensor, e5m2: bool) -> torch.Tensor:
    """Exponent byte of the least power of two that brings `largest` (float) to at most 448 (e4m3) or 57344 (e5m2), both 1.75 times
    a power of two; blocks of zeros have 127."""
    mant, ex = torch.frexp(largest)
    e = (ex - 1 - (15 if e5m2 else 8) + (mant > 0.875)).clamp_min(-126)
    return torch.where(largest > 0, e + 127, torch.full_like(e, 127))


def _cast(v: torch.Tensor, e5m2: bool = False, square: bool = False):
    """(the 8-bit values scaled back, as floats; the 8-bit values; scale bytes (rows, blocks)) of `v` (rows, k), 32 or 64 bits."""
    rows, k = v.shape
    nb, rb = -(-k // BLOCK), -(-rows // BLOCK)
    p = torch.nn.functional.pad(v, (0, nb * BLOCK - k)).view(rows, nb, BLOCK)
    largest = p.abs().amax(2)
    if square:
        sq = torch.nn.functional.pad(largest, (0, 0, 0, rb * BLOCK - rows)).view(rb, BLOCK, nb).amax(1)
        largest = sq.repeat_interleave(BLOCK, 0)[:rows]
    s = _scale_bytes(largest, e5m2)
    step = torch.exp2((s - 127).to(v.dtype))[:, :, None]
    q8 = (p / step).to(torch.float32 if v.dtype == torch.float32 else torch.float64)
    q8 = _round8(q8, e5m2)
    back = (q8 * step).reshape(rows, nb * BLOCK)[:, :k]
    return back, q8.reshape(rows, nb * BLOCK)[:, :k], s


def _round8(v: torch.Tensor, e5m2: bool) -> torch.Tensor:
    """`v` (at most the largest number of the type in size) to the nearest number of the type, ties to even, as floats."""
    bits, low = (2, -14) if e5m2 else (3, -6)
    _, ex = torch.frexp(v)
    ulp = torch.exp2((ex - 1).clamp_min(low).to(v.dtype) - bits)
    return torch.round(v / ulp) * ulp


def _bytes(q8: torch.Tensor, e5m2: bool) -> torch.Tensor:
    """The bytes of 8-bit values, each row on 16 bytes."""
    rows, k = q8.shape
    b = torch.zeros(rows, -(-k // 16) * 16, dtype=torch.uint8, device=q8.device)
    b[:, :k] = q8.float().to(torch.float8_e5m2 if e5m2 else torch.float8_e4m3fn).view(torch.uint8)
    return b[:, :k]


def _scale_rows(s: torch.Tensor) -> torch.Tensor:
    """(rows, blocks) -> (blocks, rows) bytes, each row on 16 bytes."""
    rows, nb = s.shape
    b = torch.zeros(nb, -(-rows // 16) * 16, dtype=torch.uint8, device=s.device)
    b[:, :rows] = s.t().to(torch.uint8)
    return b[:, :rows]


def _values(b: torch.Tensor, s: torch.Tensor, e5m2: bool, dtype) -> torch.Tensor:
    rows, k = b.shape
    v = b.contiguous().view(torch.float8_e5m2 if e5m2 else torch.float8_e4m3fn).to(dtype)
    return v * torch.exp2(s.t().to(dtype) - 127).repeat_interleave(BLOCK, 1)[:, :k]


# --------------------------------------------------------------------------- inputs
def _normal(g, *shape, std=1.0):
    return torch.empty(shape, device=DEV).normal_(0.0, std, generator=g)


def _activations(g, rows, dim):
    """Hidden states: a few channels are much larger than the others."""
    x = _normal(g, rows, dim)
    big = torch.randint(0, dim, (max(1, dim // 200),), device=DEV, generator=g)
    x[:, big] *= 20.0
    return x.bfloat16()


def _gradients(g, rows, dim):
    """Gradients: small, and of very different size from token to token."""
    return (_normal(g, rows, dim, std=1e-4) * torch.exp(_normal(g, rows, 1))).bfloat16()


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    if case["kind"] == "product":
        m, n, k, e5m2 = case["m"], case["n"], case["k"], case["e5m2"]
        a = _gradients(g, k, m).t().float() if e5m2 else _activations(g, m, k).float()
        b = _activations(g, k, n).t().float() if e5m2 else _normal(g, n, k, std=0.02).bfloat16().float()
        _, qa, sa = _cast(a, e5m2)
        _, qb, sb = _cast(b, False, square=not e5m2)
        return dict(kind="product", a=_bytes(qa, e5m2), sa=_scale_rows(sa), b=_bytes(qb, False), sb=_scale_rows(sb), e5m2=e5m2)
    rows, dim = case["rows"], case["dim"]
    st = dict(kind=case["kind"], x=_activations(g, rows, dim), gain=(1.0 + _normal(g, dim, std=0.1)).bfloat16())
    st["residual"] = _activations(g, rows, dim) if case.get("residual", True) else None
    if case["kind"] == "layer":
        st["w"] = _normal(g, case["out"], dim, std=0.02).bfloat16()
        st["dt"], st["dy"] = _gradients(g, rows, dim), _gradients(g, rows, case["out"])
        for name in ("x", "residual", "gain", "w"):
            st[name].requires_grad_()
    return st


# --------------------------------------------------------------------------- one pass
def run(state: dict):
    if own:
        return _run_own(state)
    with torch.no_grad():
        if state["kind"] == "product":
            a = _values(state["a"], state["sa"], state["e5m2"], torch.float32)
            b = _values(state["b"], state["sb"], False, torch.float32)
            return torch.matmul(a, b.t()).bfloat16()
        t, rstd = _add_norm(state["x"], state["residual"])
        normed = t.float() * rstd * state["gain"].float()
        h = _cast(normed)[0]
        if state["kind"] == "norm":
            return dict(t=t, h=h.bfloat16())
        w8 = _cast(state["w"].float(), square=True)[0]
        y = torch.matmul(h, w8.t())
        dy = state["dy"].float()
        dh = torch.matmul(_cast(dy)[0], w8)
        dx, dgain = _norm_gradients(dh, t.float(), rstd, state["gain"].float())
        dx = (dx + state["dt"].float()).bfloat16()
        dw = torch.matmul(_cast(dy.t().contiguous())[0], _cast(normed.t().contiguous())[0].t())
        return dict(t=t, y=y.bfloat16(), dx=dx, dresidual=dx, dgain=dgain.bfloat16(), dw=dw.bfloat16())


def _add_norm(x, residual):
    t = x if residual is None else (x.float() + residual.float()).bfloat16()
    return t, torch.rsqrt(t.float().square().mean(1, keepdim=True) + EPS)


def _norm_gradients(dh, t, rstd, gain):
    g = dh * gain
    return rstd * g - t * (rstd * rstd * rstd * (g * t).mean(1, keepdim=True)), (dh * t * rstd).sum(0)


def _run_own(state: dict):
    from kempnerforge_b200.ops import fp8_blocks

    if state["kind"] == "product":
        return fp8_blocks.mm(fp8_blocks.BlockScaled(state["a"], state["sa"], state["e5m2"]),
                             fp8_blocks.BlockScaled(state["b"], state["sb"], False))
    if state["kind"] == "norm":
        t, _, h = fp8_blocks.add_rmsnorm(state["x"], state["residual"], state["gain"], EPS)
        return dict(t=t, h=h.dequantize())
    x, residual, gain, w = leaves = [state[name] for name in ("x", "residual", "gain", "w")]
    # a step follows the optimizer's write of the weights: their 8-bit copies are made anew
    torch.autograd.graph.increment_version(w)
    t, y = fp8_blocks.norm_linear(x, residual, gain, [w], EPS)
    dx, dresidual, dgain, dw = torch.autograd.grad((t, y), leaves, (state["dt"], state["dy"]))
    return dict(t=t.detach(), y=y.detach(), dx=dx, dresidual=dresidual, dgain=dgain, dw=dw)


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case: dict) -> dict:
    if case["kind"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return dict(bytes=(m + n) * (k + -(-k // BLOCK)) + 2 * m * n, flops=2 * m * n * k)
    rows, dim = case["rows"], case["dim"]
    if case["kind"] == "norm":
        ins = 2 if case["residual"] else 1   # x and the residual in, t and the values out, the gain
        return dict(bytes=2 * rows * dim * (ins + 2) + 2 * dim, flops=8 * rows * dim)
    out = case["out"]
    # x, residual, dt and t, dx; dy and y; w and dw
    return dict(bytes=2 * rows * dim * 5 + 2 * rows * out * 2 + 2 * out * dim * 2 + 4 * dim, flops=6 * rows * dim * out)


# --------------------------------------------------------------------------- 64 bits, from the definition
def _exact_scale(block: torch.Tensor, top: float) -> torch.Tensor:
    """The least power of two that brings every value of the last axis to at most `top`."""
    a = block.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(a / top)).clamp(-126, 120)
    e = torch.where(torch.exp2(e) * top < a, e + 1, e)            # next to a border the logarithm is not decisive
    e = torch.where((torch.exp2(e - 1) * top >= a) & (e > -126), e - 1, e)
    return torch.where(a > 0, torch.exp2(e), torch.ones_like(a))


def _exact_numbers(e5m2: bool) -> torch.Tensor:
    """All non-negative finite numbers of the type, in order."""
    codes = torch.arange(0, 0x7C if e5m2 else 0x7F, dtype=torch.uint8, device=DEV)
    return codes.view(torch.float8_e5m2 if e5m2 else torch.float8_e4m3fn).double()


def _exact_cast(v: torch.Tensor, e5m2: bool, square: bool = False) -> torch.Tensor:
    """What the 8-bit form of `v` stands for, by search among the numbers of the type."""
    numbers = _exact_numbers(e5m2)
    top = float(numbers[-1])
    out = torch.empty_like(v)
    for r in range(0, v.shape[0], BLOCK):
        rows = v[r : r + BLOCK]
        pad = torch.nn.functional.pad(rows, (0, -rows.shape[1] % BLOCK))
        blocks = pad.view(rows.shape[0], -1, BLOCK)
        if square:
            scale = _exact_scale(blocks.transpose(0, 1).reshape(blocks.shape[1], -1), top).view(1, -1, 1)
        else:
            scale = _exact_scale(blocks, top)
        q = (blocks / scale).abs()
        hi = torch.searchsorted(numbers, q.contiguous()).clamp_max(len(numbers) - 1)
        lo = (hi - 1).clamp_min(0)
        up, down = numbers[hi] - q, q - numbers[lo]
        near = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), numbers[hi], numbers[lo])
        out[r : r + BLOCK] = (near * torch.sign(blocks) * scale).reshape(rows.shape[0], -1)[:, : rows.shape[1]]
    return out


@torch.no_grad()
def exact(case: dict, seed: int):
    st = prepare(case, seed)
    if case["kind"] == "product":
        def numbers(values, scales, e5m2):
            kind = torch.float8_e5m2 if e5m2 else torch.float8_e4m3fn
            v = values.contiguous().view(kind).double()
            for i in range(scales.shape[0]):
                v[:, i * BLOCK : (i + 1) * BLOCK] *= torch.exp2(scales[i].double() - 127)[:, None]
            return v

        return numbers(st["a"], st["sa"], st["e5m2"]) @ numbers(st["b"], st["sb"], False).t()
    x, gain = st["x"].double(), st["gain"].double()
    t = x if st["residual"] is None else x + st["residual"].double()
    seen = t.bfloat16().double()      # the sum is stored in 16 bits, and the norm is taken of what is stored
    inverse = 1.0 / torch.sqrt((seen * seen).sum(1) / case["dim"] + EPS)
    normed = seen * inverse[:, None] * gain
    h = _exact_cast(normed, False)
    if case["kind"] == "norm":
        return dict(t=t, h=h)
    w8, dy = _exact_cast(st["w"].double(), False, square=True), st["dy"].double()
    dh = _exact_cast(dy, False) @ w8
    inner = (dh * gain * seen).sum(1) / case["dim"]
    dx = st["dt"].double() + inverse[:, None] * (dh * gain - seen * (inverse * inverse * inner)[:, None])
    dw = _exact_cast(dy.t().contiguous(), False) @ _exact_cast(normed.t().contiguous(), False).t()
    return dict(t=t, y=h @ w8.t(), dx=dx, dresidual=dx, dgain=(dh * seen * inverse[:, None]).sum(0), dw=dw)
