"""Steps of beam search: the choice of the beams that go on, and the states that follow them.

    select    the W best of a prompt's (beam, token) pairs, by log-probability added to the beam's score
    reorder   every beam's state becomes its parent's, for a list of states at once

A step of a search over W beams of B prompts:

    step = beam.select(logits, scores, finished, eos_id=eos)          # logits (B, W, V)
    beam.reorder([tokens, rows], step.parents, length)                # histories, tables, caches: (B, W, length, ..)
    tokens[:, :, length] = step.tokens

``models.generate.beam_search`` is that search.  CUDA tensors run the kernels of ``csrc/beam.cu``; CPU tensors, and more than 32 beams,
the formulas of ``ops.ref``.  No gradient passes through either.
"""

from __future__ import annotations

import contextlib
from typing import NamedTuple

import torch

from kempnerforge_b200.ops import functional as F
from kempnerforge_b200.ops import ref

_NOTHING = contextlib.nullcontext()
_cuda = F._cuda


class Selected(NamedTuple):
    """(B, W) each, the best beam first."""

    scores: torch.Tensor     # fp32
    parents: torch.Tensor    # int64: the beam that is continued
    tokens: torch.Tensor     # int64: with what
    finished: torch.Tensor   # bool


def _on(t: torch.Tensor):
    """Kernels run on the current device's stream: that of `t` has to be current."""
    return _NOTHING if not t.is_cuda or t.device.index == torch._C._cuda_getDevice() else torch.cuda.device(t.device)


def _native(t: torch.Tensor) -> bool:
    return t.is_cuda and not F._FORCE_REF


def select(logits: torch.Tensor, scores: torch.Tensor, finished: torch.Tensor | None = None, eos_id: int | None = None,
           pad_id: int = 0) -> Selected:
    """The W best continuations of each prompt's W beams: logits (B, W, V), scores (B, W) fp32, finished (B, W) bool.

    A beam's candidates are its tokens, with its score plus the token's log-probability; logits of -inf or NaN are no candidates, +inf
    counts as the largest fp32 number.  A finished beam has one candidate: itself, with ``pad_id`` and its score; a beam whose score is
    -inf or NaN has none (a search starts with the scores 0, -inf, -inf, ..).  Best first; ties go to the lower beam, then to the lower
    token.  A beam that takes ``eos_id`` is finished.  Where there are fewer than W candidates the places left have the score -inf, their
    own beam as parent and ``pad_id``.

    The order is that of scores in 64 bits, s + (x - (top + log of the sum)).  (Beside logits of 1e16 and more 64 bits hold no logarithm: all of
    a row of the lowest fp32 value have the log-probability 0.)  On a GPU exponentials have 32, which leaves up to 4e-6 in a score before it
    is rounded to 32 bits.  Where candidates of different beams are closer than that can tell, these beams' sums are taken again in 64: one prompt's
    beams of 128 256 tokens take 57 us longer each, or 28 if their logits are the same.
    """
    eos, pad = -1 if eos_id is None else int(eos_id), int(pad_id)
    if logits.is_cuda and not F._FORCE_REF:
        done = _cuda().beam_select_call(logits, scores, finished, eos, pad)
        if done is not None:
            return Selected._make(done)
    if logits.dim() != 3 or not logits.is_floating_point() or logits.shape[1] == 0 or logits.shape[2] == 0:
        raise ValueError(f"logits are (prompts, beams, vocabulary) in a floating type, not {tuple(logits.shape)} {logits.dtype}")
    if scores.shape != logits.shape[:2] or scores.dtype != torch.float32 or scores.device != logits.device:
        raise ValueError(f"scores are fp32 {tuple(logits.shape[:2])} on {logits.device}, not {scores.dtype} {tuple(scores.shape)} on {scores.device}")
    if finished is not None and (finished.shape != scores.shape or finished.dtype != torch.bool or finished.device != logits.device):
        raise ValueError(f"finished is bool {tuple(scores.shape)} on {logits.device}, not {finished.dtype} {tuple(finished.shape)} on "
                         f"{finished.device}")
    logits, scores = logits.detach(), scores.detach().contiguous()
    finished = None if finished is None else finished.contiguous()
    if logits.shape[0] and _native(logits) and F._plain(logits, scores, finished) and _cuda().beam_select_supported(logits):
        with _on(logits):
            return Selected(*_cuda().beam_select(logits, scores, finished, eos, pad))
    return Selected(*ref.beam_select(logits, scores, finished, eos, pad))


def _dense_beams(t: torch.Tensor) -> bool:
    """What a beam holds lies side by side."""
    step = 1
    for size, stride in zip(reversed(t.shape[2:]), reversed(t.stride()[2:])):
        if size != 1 and stride != step:
            return False
        step *= size
    return True


def _apart(t: torch.Tensor) -> bool:
    """No two beams of what is written share memory."""
    step = t[0, 0].numel()
    return all(n == 1 or abs(s) >= step for n, s in zip(t.shape[:2], t.stride()[:2])) and (
        t.shape[0] == 1 or t.shape[1] == 1 or t.stride(0) >= t.shape[1] * t.stride(1) or t.stride(1) >= t.shape[0] * t.stride(0))


def _span(t: torch.Tensor) -> tuple[int, int]:
    return t.data_ptr(), t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def _interleaved(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Tensors of one shape and stepping whose values lie between each other's: no value of the one shares memory with one of the other."""
    if a.shape != b.shape or a.stride() != b.stride() or a.element_size() != b.element_size():
        return False
    size = a.element_size()
    steps = sorted(((s * size, n) for n, s in zip(a.shape, a.stride()) if n > 1), reverse=True)
    if any(s < (inner[0] * inner[1] if inner else size) for (s, _), inner in zip(steps, [*steps[1:], None])):
        return False   # a step that is shorter than what it steps over: not looked into

    def met(apart: int, level: int) -> bool:
        """Whether steps from `level` on, so many forwards or backwards as there are entries, come within a value's size of `apart`."""
        if level == len(steps):
            return abs(apart) < size
        s, n = steps[level]   # what is left is less than a step
        return any(abs(k) < n and met(apart - k * s, level + 1) for k in (apart // s, apart // s + 1))

    return not met(a.data_ptr() - b.data_ptr(), 0)


def reorder(states: list[torch.Tensor], parents: torch.Tensor, length: int | None = None,
            out: list[torch.Tensor] | None = None) -> list[torch.Tensor]:
    """state[b, w] = state[b, parents[b, w]] for states (B, W, ..) of any types, in place, or into ``out``: tensors like the states that
    share no memory with them.

    States that are written share no memory with each other or with ``parents``.
    ``length``: only the first ``length`` entries of the third dimension move, and what lies behind them stays as it is.  parents (B, W)
    int64 or int32, any selection of beams; where one is no beam (outside 0 .. W - 1) that place stays as it is.  Returns what was written.
    """
    states, to = list(states), None if out is None else list(out)
    native = _native(parents) and torch.autograd.forward_ad._current_level < 0   # the formulas move tangents with the states
    if native and _cuda().beam_reorder_call(states, parents, length, to):
        return states if to is None else to
    if parents.dim() != 2 or parents.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"parents are (prompts, beams) in int64 or int32, not {tuple(parents.shape)} {parents.dtype}")
    if length is not None and length < 0:
        raise ValueError(f"length {length} is negative")
    to = states if to is None else to
    if len(to) != len(states):
        raise ValueError(f"{len(to)} tensors to write for {len(states)} states")
    for x, y in zip(states, to):
        if x.dim() < 2 or x.shape[:2] != parents.shape or x.device != parents.device:
            raise ValueError(f"a state is {(*parents.shape, '..')} on {parents.device}, not {tuple(x.shape)} on {x.device}")
        if length is not None and (x.dim() < 3 or x.shape[2] < length):
            raise ValueError(f"a state of shape {tuple(x.shape)} does not hold {length} entries")
        if y.shape != x.shape or y.dtype != x.dtype or y.device != x.device:
            raise ValueError(f"what is written for a state is {tuple(x.shape)} {x.dtype} on {x.device}, not {tuple(y.shape)} {y.dtype} on {y.device}")
        if torch.is_grad_enabled() and (x.requires_grad or y.requires_grad):
            raise ValueError("no gradient passes through a reordering: call it under no_grad")
    spans = [(*_span(y), 1, y) for y in to if y.numel()]
    if out is not None:
        spans += [(*_span(x), 0, x) for x in states if x.numel()]
    if parents.numel():
        spans.append((*_span(parents), 0, parents))
    spans.sort(key=lambda s: s[0])
    for n, (_, end, writes, x) in enumerate(spans):
        for begin, _, written, y in spans[n + 1 :]:
            if begin >= end:
                break
            if (writes or written) and not _interleaved(x, y):
                raise ValueError("a state that is written shares memory with another or with the parents")
    if parents.numel() == 0 or not states:
        return to
    with torch.no_grad():
        if not (native and parents.shape[1] <= 32 and parents.shape[0] <= 65535):
            ref.beam_reorder(states, parents, length, to)
        else:
            _reorder_native(states, parents, length, to)
    return to


def _reorder_native(states, parents, length, to):
    moves, later = [], []
    for x, y in zip(states, to):
        if length is not None:
            x, y = x[:, :, :length], y[:, :, :length]
        if x.numel() == 0:
            continue
        inner = x[0, 0].numel()
        if inner * x.element_size() > 1 << 37 or not _dense_beams(x) or not _dense_beams(y) or not _apart(y):
            later.append((x, y))
            continue
        moves.append((x, y, inner * x.element_size()))
    with _on(parents):
        parents = parents.contiguous()
        if moves:
            _cuda().beam_reorder(moves, parents)
            for _, y, _ in moves:
                if not y.is_inference():
                    torch.autograd.graph.increment_version(y)
        for x, y in later:
            ref.beam_reorder([x], parents, None, [y])
