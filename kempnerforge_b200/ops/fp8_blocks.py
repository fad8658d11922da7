"""FP8 with a scale for each block of 128 values, for training and generation.

:mod:`kempnerforge_b200.ops.fp8` scales a tensor by one factor, so one outlier costs every other value its bits, and a cast has to wait for
the maximum of the whole tensor.  Here 128 neighbouring values along the reduction share a factor (activations and gradients; weights share
one over 128 x 128), a power of two:

    X[r, k] = q[r, k] * 2^(s[k // 128, r] - 127)          q: e4m3 or e5m2 bytes, s: bytes

of a block whose largest finite magnitude is a, the least power of two (at least 2^-126) that brings a to 448 or less (57 344 for e5m2); q
rounds to the nearest, ties to even.  A block of zeros has s = 127.  An infinity or a NaN is stored as NaN, the other values of its block as
if it were not there.

    quantize       bf16 matrix -> :class:`BlockScaled`, row-major and / or transposed
    add_rmsnorm    x + residual, its RMSNorm in 8 bits
    mm             product of two BlockScaled matrices (tcgen05 kind::mxf8f6f4 on a GPU)
    linear         differentiable Linear: e4m3 operands and gradients, bf16 weights, fp32 accumulation
    norm_linear    differentiable x + residual -> RMSNorm -> Linear, the normalised activation in 8 bits only

    forward   y  = q(h) q(W)ᵀ                 q over 128 values of k, W over squares
    backward  dh = q(dy) q(W)                 q over 128 values of n; of a norm_linear kept in 32 bits for the norm's gradients
              dW = q(dyᵀ) q(hᵀ)ᵀ              q over 128 tokens

``train.fp8_scaling = "block128"`` has the fp8 Linear layers take this path.  CUDA tensors run the kernels of ``csrc/fp8_blocks.cu`` and
``csrc/gemm_fp8_blocks_tcgen05.cu``; CPU tensors (tests) the same arithmetic with ``torch.float8_*`` dtypes.
"""

from __future__ import annotations

import contextlib
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from kempnerforge_b200.ops import fp8

BLOCK = 128
_LARGEST = 2**31 - 2**16  # rows or columns: indices of kernels have 32 bits, and a few blocks are added to them
_BF16 = torch.bfloat16
_NOTHING = contextlib.nullcontext()


_modules = None


def _others():
    """(ops.cuda, ops.functional), imported when first wanted."""
    global _modules
    if _modules is None:
        from kempnerforge_b200.ops import cuda, functional

        _modules = cuda, functional
    return _modules


def _cuda():
    return _others()[0]


def _on(t: torch.Tensor):
    """The device of ``t`` as the current one: a launch goes to the current device's stream."""
    return torch.cuda.device(t.device) if t.device.index != torch._C._cuda_getDevice() else _NOTHING


class BlockScaled(NamedTuple):
    """A (rows, k) matrix in 8 bits.  ``values``: uint8 (rows, k), ``scales``: uint8 (ceil(k / 128), rows); rows may be
    pitched (what is not on 16 bytes is copied before a product)."""

    values: torch.Tensor
    scales: torch.Tensor
    e5m2: bool = False

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    def dequantize(self) -> torch.Tensor:
        """The values as bf16, which has them exactly (down to 2^-133)."""
        if self.values.is_cuda and (out := _cuda()._step("fp8_values", *self)) is not None:
            return out
        _check_operand(self, "matrix")
        if self.values.numel() == 0:
            return torch.empty(self.values.shape, dtype=_BF16, device=self.values.device)
        if self.values.is_cuda:
            with _on(self.values):
                return _cuda().fp8_blocks_values(*self)
        return _values(self).to(_BF16)


def _check_operand(a: BlockScaled, name: str) -> None:
    q, s = a.values, a.scales
    if q.dtype != torch.uint8 or s.dtype != torch.uint8 or q.dim() != 2 or s.dim() != 2 or q.device != s.device:
        raise ValueError(f"{name}: values and scales are uint8 matrices on one device")
    rows, k = q.shape
    if max(rows, k) > _LARGEST:
        raise ValueError(f"{name}: {rows} rows of {k} values, at most {_LARGEST} of either are covered")
    if s.shape != (-(-k // BLOCK), rows):
        raise ValueError(f"{name}: {rows} rows of {k} values have scales of shape {(-(-k // BLOCK), rows)}, got {tuple(s.shape)}")
    if q.numel() and ((k > 1 and q.stride(1) != 1) or (rows > 1 and s.stride(1) != 1)):
        raise ValueError(f"{name}: the columns of values and scales must be contiguous")


def _check_matrix(x2: torch.Tensor, name: str = "x") -> None:
    if x2.dim() != 2 or x2.dtype != _BF16:
        raise ValueError(f"{name}: a bf16 matrix is wanted, got {x2.dtype} of shape {tuple(x2.shape)}")
    if max(x2.shape) > _LARGEST:
        raise ValueError(f"{name}: shape {tuple(x2.shape)}, at most {_LARGEST} rows or columns are covered")


# --------------------------------------------------------------------------- plain arithmetic (CPU)
def _block_max(v: torch.Tensor, square: bool) -> torch.Tensor:
    """(rows, blocks) largest finite magnitudes."""
    rows, k = v.shape
    nb, rb = -(-k // BLOCK), -(-rows // BLOCK)
    a = torch.nn.functional.pad(torch.where(v.isfinite(), v.abs(), 0.0), (0, nb * BLOCK - k)).view(rows, nb, BLOCK).amax(2)
    if square:
        a = torch.nn.functional.pad(a, (0, 0, 0, rb * BLOCK - rows)).view(rb, BLOCK, nb).amax(1).repeat_interleave(BLOCK, 0)[:rows]
    return a


def _cast_rows(v: torch.Tensor, e5m2: bool, square: bool = False) -> BlockScaled:
    """fp32 matrix -> 8 bits, on any device, in torch operations."""
    a = _block_max(v, square)
    mant, ex = torch.frexp(a)
    s = (ex - 1 - (15 if e5m2 else 8) + (mant > 0.875)).clamp_min(-126) + 127
    s = torch.where(a > 0, s, torch.full_like(s, 127))
    inv = torch.ldexp(torch.ones_like(a), 127 - s).repeat_interleave(BLOCK, 1)[:, : v.shape[1]]
    q = (torch.where(v.isfinite(), v, float("nan")) * inv).to(torch.float8_e5m2 if e5m2 else torch.float8_e4m3fn)
    return BlockScaled(q.view(torch.uint8), s.t().to(torch.uint8).contiguous(), e5m2)


def _values(a: BlockScaled) -> torch.Tensor:
    """The values as fp32."""
    v = a.values.contiguous().view(torch.float8_e5m2 if a.e5m2 else torch.float8_e4m3fn).float()
    f = torch.ldexp(torch.ones(a.scales.shape, device=v.device), a.scales.int() - 127)
    f = torch.where(a.scales == 255, float("nan"), f)
    return v * f.t().repeat_interleave(BLOCK, 1)[:, : v.shape[1]]


# --------------------------------------------------------------------------- operators
def _empty(rows: int, k: int, device, e5m2: bool) -> BlockScaled:
    return BlockScaled(torch.empty((rows, k), dtype=torch.uint8, device=device), torch.empty((-(-k // BLOCK), rows), dtype=torch.uint8, device=device), e5m2)


def quantize(x2: torch.Tensor, e5m2: bool = False, square: bool = False, want_row: bool = True,
             want_t: bool = False) -> tuple[BlockScaled | None, BlockScaled | None]:
    """(``x2`` in 8 bits or None, its transpose in 8 bits or None) of a bf16 matrix.  ``square``: blocks of 128 x 128, so that both hold
    the same values; else each has blocks of 128 along its own columns."""
    if x2.is_cuda and (r := _cuda()._step("fp8_cast", x2, e5m2, square, want_row, want_t, None, None)) is not None:
        q, s, qt, st = r
        return None if q is None else BlockScaled(q, s, e5m2), None if qt is None else BlockScaled(qt, st, e5m2)
    _check_matrix(x2)
    rows, cols = x2.shape
    if not (want_row or want_t):
        return None, None
    if x2.numel() == 0:
        return _empty(rows, cols, x2.device, e5m2) if want_row else None, _empty(cols, rows, x2.device, e5m2) if want_t else None
    if x2.is_cuda:
        if x2.stride(1) != 1 and cols > 1 or x2.stride(0) < cols and rows > 1:
            x2 = x2.contiguous()
        with _on(x2):
            row, t = _cuda().fp8_blocks_cast(x2, e5m2, square, want_row, want_t)
        return row and BlockScaled(*row, e5m2), t and BlockScaled(*t, e5m2)
    v = x2.float()
    return _cast_rows(v, e5m2, square) if want_row else None, _cast_rows(v.t().contiguous(), e5m2, square) if want_t else None


def mm(a: BlockScaled, b: BlockScaled, out: torch.Tensor | None = None, accumulate: bool = False, dtype: torch.dtype | None = None) -> torch.Tensor:
    """(M, N) = a (M, K) @ b (N, K)ᵀ, accumulated in fp32 and rounded once to ``dtype``: that of ``out``, else bf16 unless fp32 is asked for;
    with ``accumulate`` added to ``out`` before the rounding.  A write of ``out`` moves its version, as a tensor operation's does."""
    if dtype is None:
        dtype = _BF16 if out is None else out.dtype
    if dtype is not _BF16 and dtype is not torch.float32:   # first: the native call knows these two only
        raise ValueError(f"products are bf16 or fp32, got {dtype}")
    if a.values.is_cuda and (y := _cuda().fp8_blocks_mm(a, b, out, accumulate, dtype is torch.float32)) is not None:
        return y
    _check_operand(a, "a")
    _check_operand(b, "b")
    (m, k), n = a.values.shape, b.values.shape[0]
    if b.values.shape[1] != k:
        raise ValueError(f"inner dimensions differ: {k} and {b.values.shape[1]}")
    dev = a.values.device
    if b.values.device != dev:
        raise ValueError(f"operands on {dev} and {b.values.device}")
    if out is None:
        out, accumulate = torch.empty((m, n), dtype=dtype, device=dev), False
    elif out.shape != (m, n) or out.dtype != dtype or out.device != dev or (n > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < n):
        raise ValueError(f"out: a {dtype} ({m}, {n}) matrix on {dev} with contiguous columns is wanted")
    if m == 0 or n == 0 or k == 0:
        return out if accumulate else out.zero_()
    if not a.values.is_cuda:
        y = _values(a) @ _values(b).t()
        return out.copy_(out.float() + y if accumulate else y)
    with _on(out):
        _cuda().gemm_fp8_blocks(_pitched(a.values), _pitched(a.scales), _pitched(b.values), _pitched(b.scales), a.e5m2, b.e5m2, out, accumulate)
    torch.autograd.graph.increment_version(out)   # which a kernel's write does not do
    return out


def _pitched(t: torch.Tensor) -> torch.Tensor:
    """``t``, or a copy with the rows and the base on the 16 bytes that the kernels' bulk copies need (what was saved on the host and
    returns, a slice)."""
    if t.data_ptr() % 16 == 0 and t.stride(0) % 16 == 0 and t.stride(0) >= t.shape[1] and t.stride(1) == 1:
        return t
    rows, cols = t.shape
    out = torch.empty((rows, -(-cols // 16) * 16), dtype=t.dtype, device=t.device)[:, :cols]
    return out.copy_(t)


def add_rmsnorm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-5):
    """(t, rstd, h) of bf16 matrices (rows, d), d a multiple of 8 up to 32 768: t = x + residual rounded to bf16 (x itself without one),
    rstd = 1 / sqrt(mean(t²) + eps) as fp32 (rows,), h = (t * weight) * rstd in 8 bits, never rounded to 16 (on a GPU not to 32
    either: rstd has more bits there than are returned, and h is the 8-bit number next to the formula's value).  Not differentiable by
    itself: :func:`norm_linear` is."""
    if x.is_cuda and (r := _cuda()._step("fp8_add_rmsnorm", x, residual, weight, eps)) is not None:
        t, rstd, q, s = r
        return x.detach() if t is None else t, rstd, BlockScaled(q, s)
    _check_norm(x, residual, weight)
    _check_matrix(x)
    x, residual, weight = x.detach(), None if residual is None else residual.detach(), weight.detach()
    rows, d = x.shape
    if rows == 0:
        return x if residual is None else x + residual, torch.empty(0, device=x.device), _empty(0, d, x.device, False)
    if not x.is_cuda:
        t = x if residual is None else (x.float() + residual.float()).to(_BF16)
        rstd = torch.rsqrt(t.float().square().mean(1) + eps)
        return t, rstd, _cast_rows(t.float() * weight.float() * rstd[:, None], False)
    x, residual, weight = _aligned(x), residual if residual is None else _aligned(residual), _aligned(weight)
    with _on(x):
        t, rstd, h = _cuda().add_rmsnorm_fp8_blocks(x, residual, weight, eps)
    return x if t is None else t, rstd, BlockScaled(*h)


def _check_norm(x, residual, weight) -> None:
    d, device = x.size(-1) if x.dim() else 0, x.device
    if x.dtype is not _BF16 or weight.dtype is not _BF16 or (residual is not None and residual.dtype is not _BF16):
        raise ValueError("x, residual and weight are bf16")
    if weight.dim() != 1 or weight.size(0) != d or (residual is not None and residual.shape != x.shape):
        raise ValueError(f"shapes: x {tuple(x.shape)}, residual {None if residual is None else tuple(residual.shape)}, weight {tuple(weight.shape)}")
    if weight.device != device or (residual is not None and residual.device != device):
        raise ValueError("x, residual and weight are on one device")
    if d % 8 or not 0 < d <= 32768:
        raise ValueError(f"rows of {d} values: a multiple of 8 up to 32768 is wanted")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t``, contiguous and on 16 bytes."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


# --------------------------------------------------------------------------- weights
def quantized_weight(weights, want_t: bool) -> tuple[BlockScaled, BlockScaled | None]:
    """(the weights stacked along the output dimension in 8 bits, the transpose of that or None), in squares of 128 x 128.  Kept on the
    first weight and reused under the conditions of :func:`kempnerforge_b200.ops.fp8.quantized_weight`."""
    first = weights[0]
    if first.is_cuda and first.device.index != torch._C._cuda_getDevice():
        # the stream that copies belong to, and whether it is captured, are asked of the current device
        with torch.cuda.device(first.device):
            return quantized_weight(weights, want_t)
    stacked = lambda: _others()[1]._stack_weight_rows(weights).detach()  # noqa: E731
    state = fp8.weights_state(weights)
    if state is None:
        return quantize(stacked(), square=True, want_t=want_t)
    cached = getattr(first, "_kf_fp8_block_cache", None)
    if not fp8.still_those_of(cached, state):
        row, t = quantize(stacked(), square=True, want_t=want_t)
        cached = first._kf_fp8_block_cache = fp8.copies_of(weights, state, row)
        cached.transposed = t
    elif want_t and cached.transposed is None:
        cached.transposed = quantize(stacked(), square=True, want_row=False, want_t=True)[1]
    return cached.row, cached.transposed if want_t else None


def _check_weights(x: torch.Tensor, weights) -> None:
    if x.dtype is not _BF16 or not x.dim() or not weights:
        raise ValueError("x is bf16 and has at least one weight")
    k, device = x.size(-1), x.device
    for w in weights:
        if w.dtype is not _BF16 or w.dim() != 2 or w.size(1) != k or w.device != device:
            raise ValueError(f"weights are bf16 (out, {k}) matrices on {device}, got {w.dtype} {tuple(w.shape)} on {w.device}")


def _rows(x: torch.Tensor) -> torch.Tensor:
    x2 = x if x.dim() == 2 else x.reshape(-1, x.size(-1))
    return x2 if x2.is_contiguous() else x2.contiguous()


class _BlocksLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, recording, *weights):
        # what a backward reads is made where one is recorded: needs_input_grad tells of the leaves only
        x8, x8t = quantize(_rows(x), want_t=recording and any(ctx.needs_input_grad[2:]))
        w8, _ = quantized_weight(weights, want_t=recording and ctx.needs_input_grad[0])
        y = mm(x8, w8)
        # the transposed copy is all that the gradient of the weights reads of x: half of its bytes
        ctx.save_for_backward(*(x8t[:2] if x8t is not None else (None, None)), *weights)
        ctx.x_shape = x.shape
        return y.view(*x.shape[:-1], y.shape[1])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        q8t, s8t, *weights = ctx.saved_tensors
        need_dx, need_dw = ctx.needs_input_grad[0], any(ctx.needs_input_grad[2:])
        dy2 = _rows(dy)
        w8t = quantized_weight(weights, want_t=True)[1] if need_dx else None
        dx = None

        def run(out=None, accumulate=False):
            nonlocal dx
            if dy2.is_cuda:
                r = _cuda()._step("fp8_linear_grads", dy2, *(w8t[:2] if need_dx else (None, None)), q8t, s8t, out, accumulate, _cuda().sm_count(),
                                  launches=1 + need_dx + need_dw)
                if r is not None:
                    dx = r if need_dx else None
                    return
            g8, g8t = quantize(dy2, want_row=need_dx, want_t=need_dw)
            if need_dx:
                dx = mm(g8, w8t)
            if need_dw:
                mm(g8t, BlockScaled(q8t, s8t), out=out, accumulate=accumulate)

        wgrads = [None] * len(weights)
        if need_dw:
            wgrads = _others()[1]._deposit_stacked_weight_grads(weights, ctx.needs_input_grad[2:], run)
        elif need_dx:
            run()
        return dx.view(ctx.x_shape) if need_dx else None, None, *wgrads


def linear(x: torch.Tensor, weights) -> torch.Tensor:
    """x (..., K) bf16 against one or several (out_i, K) bf16 weights stacked along the output: y (..., sum out_i)."""
    weights = list(weights)
    _check_weights(x, weights)
    return _BlocksLinearFn.apply(x, torch.is_grad_enabled(), *weights)


class _NormLinearFn(torch.autograd.Function):
    """(x + residual, Linear(RMSNorm(x + residual))).  Saved: the sum, a scale per row, the weights; the gradient of the weights casts the
    normalised activation once more, along the tokens."""

    @staticmethod
    def forward(ctx, x, residual, gain, eps, recording, *weights):
        ctx.set_materialize_grads(False)
        x2, r2 = _rows(x), None if residual is None else _rows(residual)
        w8, _ = quantized_weight(weights, want_t=recording and any(ctx.needs_input_grad[:3]))
        r = _cuda()._step("fp8_norm_linear", x2, r2, gain, eps, *w8[:2], _cuda().sm_count(), launches=2) if x.is_cuda else None
        if r is not None:
            t, rstd, y = r
            t = x2.detach() if t is None else t
        else:
            t, rstd, h8 = add_rmsnorm(x2, r2, gain, eps)
            y = mm(h8, w8)
        ctx.save_for_backward(t, rstd, gain, *weights)
        ctx.x_shape = x.shape
        # without a residual the sum is x itself: its gradient comes in here and is added where the norm's is written
        return x.view_as(x) if residual is None else t.view(x.shape), y.view(*x.shape[:-1], y.shape[1])

    @staticmethod
    @once_differentiable
    def backward(ctx, dt, dy):
        t, rstd, gain, *weights = ctx.saved_tensors
        need_x, need_r, need_g, _, _, *need_w = ctx.needs_input_grad
        dx = dgain = None
        wgrads = [None] * len(weights)
        if dy is None:
            dx = dt
        else:
            need_h, any_w = need_x or need_r or need_g, any(need_w)
            dy2, dt2 = _rows(dy), None if dt is None else _rows(dt)
            w8t = quantized_weight(weights, want_t=True)[1] if need_h else None

            def run(out=None, accumulate=False):
                nonlocal dx, dgain
                if dy2.is_cuda:
                    r = _cuda()._step("fp8_norm_linear_grads", dy2, dt2, t, gain, rstd, *(w8t[:2] if need_h else (None, None)), out, accumulate,
                                      _cuda().sm_count(), launches=1 + 3 * need_h + 2 * any_w)
                    if r is not None:
                        dx, dgain = r
                        return
                g8, g8t = quantize(dy2, want_row=need_h, want_t=any_w)
                if need_h:
                    dx, dgain = _norm_grads(mm(g8, w8t, dtype=torch.float32), t, gain, rstd, dt2)
                if any_w:
                    mm(g8t, _normed_t(t, rstd, gain), out=out, accumulate=accumulate)

            if any_w:
                wgrads = _others()[1]._deposit_stacked_weight_grads(weights, need_w, run)
            elif need_h:
                run()
            if need_h:
                dx = dx.view(ctx.x_shape)
                dgain = _gain_grad(gain, dgain) if need_g else None
        return dx if need_x else None, dx if need_r else None, dgain, None, None, *wgrads


def _norm_grads(dh, t, gain, rstd, dt):
    """(gradient of t, dt included, bf16; gradient of the gain)."""
    if t.numel() == 0:
        return torch.empty_like(t), torch.zeros_like(gain)
    if t.is_cuda:
        with _on(t):
            return _cuda().norm_grads(dh, t, _aligned(gain), rstd, None if dt is None else _aligned(dt))
    tf, g, r = t.float(), dh * gain.float(), rstd[:, None]
    d = r * g - tf * (r * r * r * (g * tf).mean(1, keepdim=True))
    return (d if dt is None else d + dt.float()).to(_BF16), (dh * tf * r).sum(0).to(gain.dtype)


def _gain_grad(gain, dgain):
    """What autograd gets: None where the flat gradient buffer took it."""
    slot = getattr(gain, "_kf_grad", None)
    if slot is None:
        return dgain.to(gain.dtype)
    if getattr(gain, "_kf_grad_live", False):
        slot.add_(dgain)
    else:
        slot.copy_(dgain)
        gain._kf_grad_live = True
    return None


def _normed_t(t, rstd, gain) -> BlockScaled:
    """The transpose of (t * gain) * rstd in 8 bits, by way of 32: about one value in 1.5 million is the neighbour of the one that
    :func:`add_rmsnorm` gives."""
    if t.numel() == 0:
        return _empty(t.shape[1], t.shape[0], t.device, False)
    if t.is_cuda:
        r = _cuda()._step("fp8_cast", t, False, False, False, True, rstd, gain)
        if r is not None:
            return BlockScaled(r[2], r[3])
        with _on(t):
            return BlockScaled(*_cuda().fp8_blocks_cast(t, False, False, False, True, rstd, _aligned(gain))[1])
    return _cast_rows((t.float() * gain.float() * rstd[:, None]).t().contiguous(), False)


def norm_linear_of(norm, x: torch.Tensor, residual: torch.Tensor | None, weights):
    """:func:`norm_linear` in place of the module ``norm`` and the product with ``weights``, or None where that is something else: another
    norm, hooks that want its output, weights that are not tagged for block scales."""
    from torch.nn.modules import module

    from kempnerforge_b200.models.norm import RMSNorm

    if (type(norm) is not RMSNorm or norm._forward_hooks or norm._forward_pre_hooks or norm._backward_hooks or norm._backward_pre_hooks
            or "forward" in norm.__dict__ or module._has_any_global_hook() or not fp8.supported(x, weights)
            or not fp8.has_block_scales(weights[0])):
        return None
    d = x.shape[-1]
    if d % 8 or not 0 < d <= 32768 or norm.weight.dtype != _BF16 or norm.weight.device != x.device or (residual is not None and residual.dtype != _BF16):
        return None
    return norm_linear(x, residual, norm.weight, weights, norm.eps)


def norm_linear(x: torch.Tensor, residual: torch.Tensor | None, norm_weight: torch.Tensor, weights, eps: float = 1e-5):
    """(t, y): t = x + residual (x where there is none), y = RMSNorm(t) * norm_weight through a Linear of one or several weights stacked
    along the output; x (..., K) bf16, K a multiple of 8 up to 32 768.  The gradient of t is added to the norm's in one pass."""
    weights = list(weights)
    _check_weights(x, weights)
    _check_norm(x, residual, norm_weight)
    return _NormLinearFn.apply(x, residual, norm_weight, eps, torch.is_grad_enabled(), *weights)
