"""Plain PyTorch implementations of every hot op.

They serve three purposes: the CPU execution path (tests, gloo runs), the fp32
oracle that each CUDA kernel is checked against, and the definition of the
numerics the kernels must reproduce.

Semantics follow the reference model code:
  RMSNorm fp32 compute then cast back ... kempnerforge/model/norm.py:11-27
  RoPE half-split rotation ............... kempnerforge/model/position.py:12-71
  GQA causal / document-masked attention . kempnerforge/model/attention.py:116-236
  SwiGLU .................................. kempnerforge/model/mlp.py:12-26
  cross entropy (ignore_index=-100) ....... kempnerforge/training/loss.py:19-102
  Newton-Schulz quintic ................... kempnerforge/training/optimizer.py:291-318
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

IGNORE_INDEX = -100


# --------------------------------------------------------------------------- norm
def _wide(x: torch.Tensor) -> torch.Tensor:
    """fp32 for the arithmetic of half-precision inputs; float64 stays float64 (gradient checks run in double)."""
    return x if x.dtype == torch.float64 else x.float()


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    xf = _wide(x)
    inv = torch.rsqrt(xf.pow(2).mean(dim=-1, keepdim=True) + eps)
    return (xf * inv * weight.to(xf.dtype)).to(x.dtype)


# --------------------------------------------------------------------------- rope
def rope_tables(head_dim: int, max_seq_len: int, theta: float = 10000.0, device=None):
    """(cos, sin), each (max_seq_len, head_dim // 2) in fp32."""
    half = head_dim // 2
    inv_freq = theta ** (-torch.arange(0, half, dtype=torch.float32, device=device) * 2.0 / head_dim)
    ang = torch.outer(torch.arange(max_seq_len, dtype=torch.float32, device=device), inv_freq)
    return ang.cos(), ang.sin()


def apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Rotate pairs (x[..., i], x[..., i + hd/2]).  x: (B, S, H, hd); cos/sin: (S, hd/2) or (B, S, hd/2)."""
    half = x.shape[-1] // 2
    x1, x2 = x[..., :half], x[..., half:]
    if cos.dim() == 2:
        c, s = cos[None, :, None, :], sin[None, :, None, :]
    else:
        c, s = cos[:, :, None, :], sin[:, :, None, :]
    c, s = c.to(x.dtype), s.to(x.dtype)
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)


# --------------------------------------------------------------------------- attention
def attention_mask(
    s_q: int,
    s_k: int,
    causal: bool,
    doc_ids: torch.Tensor | None = None,
    key_padding_mask: torch.Tensor | None = None,
    device=None,
) -> torch.Tensor | None:
    """Boolean (B or 1, 1, s_q, s_k) mask, True = may attend; None when nothing is masked."""
    mask = None
    if causal:
        offset = s_k - s_q
        i = torch.arange(s_q, device=device)[:, None]
        j = torch.arange(s_k, device=device)[None, :]
        mask = (j <= i + offset)[None, None]
    if doc_ids is not None:
        same = (doc_ids[:, :, None] == doc_ids[:, None, :])[:, None]
        mask = same if mask is None else (mask & same)
    if key_padding_mask is not None:
        keep = key_padding_mask[:, None, None, :].bool()
        mask = keep if mask is None else (mask & keep)
        # rows with no visible key would produce NaN; let them see everything instead
        dead = ~mask.any(dim=-1, keepdim=True)
        mask = mask | dead
    return mask


def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    causal: bool = True,
    doc_ids: torch.Tensor | None = None,
    key_padding_mask: torch.Tensor | None = None,
    scale: float | None = None,
    return_weights: bool = False,
):
    """softmax(q kᵀ * scale + mask) v with grouped KV heads.

    q: (B, Sq, H, hd); k, v: (B, Sk, Hkv, hd) with H % Hkv == 0.  Query head h
    reads KV head h // (H // Hkv).  Returns (B, Sq, H, hd).
    """
    b, sq, h, hd = q.shape
    sk, hkv = k.shape[1], k.shape[2]
    group = h // hkv
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    qf = _wide(q.transpose(1, 2)).reshape(b, hkv, group, sq, hd)
    kf = _wide(k.transpose(1, 2))[:, :, None]
    vf = _wide(v.transpose(1, 2))[:, :, None]
    scores = torch.matmul(qf, kf.transpose(-1, -2)) * scale  # (B, Hkv, G, Sq, Sk)
    mask = attention_mask(sq, sk, causal, doc_ids, key_padding_mask, device=q.device)
    if mask is not None:
        scores = scores.masked_fill(~mask[:, :, None], float("-inf"))
    probs = torch.softmax(scores, dim=-1)
    out = torch.matmul(probs, vf).reshape(b, h, sq, hd).transpose(1, 2).to(q.dtype)
    if return_weights:
        return out, probs.reshape(b, h, sq, sk)
    return out


def shared_prefix_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    own_k: torch.Tensor,
    own_v: torch.Tensor,
    prefix_lens: torch.Tensor | None = None,
    own_rows: torch.Tensor | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """One new token of each of W continuations of B prompts.  q (B, W, H, hd); k, v (B, P, Hkv, hd) and own_k, own_v
    (B, W, S, Hkv, hd); ``own_rows[b, w, s]``: the continuation whose own cache holds position s of continuation w (a value that is
    none: nowhere).  What is not visible takes no part, whatever it holds; a row that sees nothing is zero."""
    b, w, h, hd = q.shape
    p, hkv, s = k.shape[1], k.shape[2], own_k.shape[2]
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    qf = _wide(q).reshape(b, w, hkv, h // hkv, hd)
    kf, vf, okf, ovf = _wide(k), _wide(v), _wide(own_k), _wide(own_v)
    sees = torch.ones(b, 1, 1, 1, p, dtype=torch.bool, device=q.device)
    if prefix_lens is not None:
        sees = (torch.arange(p, device=q.device) < prefix_lens[:, None])[:, None, None, None]
        kf, vf = (torch.where(sees[:, 0, 0, 0, :, None, None], t, 0.0) for t in (kf, vf))   # gradients multiply by what keys hold, too
    own_sees = torch.ones(b, w, 1, 1, s, dtype=torch.bool, device=q.device)
    if own_rows is not None:
        own_sees = (own_rows < w)[:, :, None, None]
        at = torch.arange(b, device=q.device)[:, None, None], own_rows.long().clamp_max(w - 1), torch.arange(s, device=q.device)
        okf, ovf = (torch.where(own_sees[:, :, 0, 0, :, None, None], t[at], 0.0) for t in (okf, ovf))
    scores = torch.cat([torch.einsum("bwkgd,bpkd->bwkgp", qf, kf).masked_fill(~sees, float("-inf")),
                        torch.einsum("bwkgd,bwskd->bwkgs", qf, okf).masked_fill(~own_sees, float("-inf"))], dim=-1) * scale
    some = torch.cat([sees.expand(b, w, 1, 1, p), own_sees], dim=-1).any(-1, keepdim=True)
    probs = torch.softmax(scores, dim=-1) if p + s else scores
    probs = torch.where(some, probs, 0.0)
    out = torch.einsum("bwkgp,bpkd->bwkgd", probs[..., :p], vf) + torch.einsum("bwkgs,bwskd->bwkgd", probs[..., p:], ovf)
    return out.reshape(b, w, h, hd).to(q.dtype)


# --------------------------------------------------------------------------- beam search
def beam_select(logits: torch.Tensor, scores: torch.Tensor, finished: torch.Tensor | None, eos_id: int, pad_id: int):
    """(scores, parents, tokens, finished), each (B, W): the W best of a prompt's candidates, in 64 bits.  A beam's candidates are ordered
    by logit, then by token; all by score, then by beam.  NaN logits count as -inf, +inf as the largest fp32 number."""
    b, w, vocab = logits.shape
    x = logits.double()
    x = torch.where(x > float("-inf"), x.clamp_max(torch.finfo(torch.float32).max), float("-inf"))
    top = x.amax(-1, keepdim=True)
    shifted = torch.where(x > float("-inf"), x - top, float("-inf"))
    shifted = torch.nn.functional.pad(shifted, (0, -vocab % 16), value=float("-inf"))   # rows that begin alike are added up alike
    lse = top + shifted.exp().sum(-1, keepdim=True).log()
    x, token = torch.sort(x, dim=-1, descending=True, stable=True)
    x, token = x[..., :w], token[..., :w]
    total = torch.where(x > float("-inf"), scores.double()[..., None] + (x - lse), float("-inf"))
    done = torch.zeros_like(scores, dtype=torch.bool) if finished is None else finished
    only = torch.full_like(total, float("-inf"))
    only[..., 0] = scores.double()
    total = torch.where(done[..., None], only, total)
    total = torch.where((scores > float("-inf"))[..., None], total, float("-inf"))
    token = torch.where(done[..., None], pad_id, token)
    width = total.shape[-1]
    total, at = torch.sort(total.flatten(1), dim=-1, descending=True, stable=True)
    total, at = total[:, :w], at[:, :w]
    none = total == float("-inf")
    parents = torch.where(none, torch.arange(w, device=logits.device), at // width)
    tokens = torch.where(none, pad_id, torch.gather(token.flatten(1), 1, at))
    ended = torch.gather(done, 1, parents)
    return total.float(), parents, tokens, ~none & (ended | (tokens == eos_id))


def beam_reorder(states, parents: torch.Tensor, length: int | None, out) -> None:
    """out[b, w, :length] = state[b, parents[b, w], :length]; where the parent is no beam, out stays."""
    w = parents.shape[1]
    ok = (parents >= 0) & (parents < w)
    rows = torch.arange(parents.shape[0], device=parents.device)[:, None]
    for x, y in zip(states, out):
        n = x.shape[2] if length is None and x.dim() > 2 else length
        src, dst = (x, y) if n is None else (x[:, :, :n], y[:, :, :n])
        new = src[rows, parents.clamp(0, w - 1).long()]
        dst.copy_(torch.where(ok.view(*ok.shape, *([1] * (x.dim() - 2))), new, dst))


# --------------------------------------------------------------------------- mlp
def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    return F.silu(gate) * up


# --------------------------------------------------------------------------- loss
def cross_entropy_parts(logits: torch.Tensor, labels: torch.Tensor):
    """Returns (sum of nll over valid tokens, sum of logsumexp², valid count), all fp32 scalars."""
    lf = _wide(logits)
    lse = torch.logsumexp(lf, dim=-1)
    valid = labels != IGNORE_INDEX
    safe = labels.clamp_min(0)
    picked = lf.gather(-1, safe[..., None]).squeeze(-1)
    nll = torch.where(valid, lse - picked, torch.zeros_like(lse))
    z = torch.where(valid, lse * lse, torch.zeros_like(lse))
    return nll.sum(), z.sum(), valid.sum()


def cross_entropy(logits: torch.Tensor, labels: torch.Tensor, z_loss_weight: float = 0.0):
    """Mean NLL over labels != -100 (0 when all are ignored) + z_loss_weight * mean(lse²)."""
    nll, z, n = cross_entropy_parts(logits.reshape(-1, logits.shape[-1]), labels.reshape(-1))
    denom = n.clamp_min(1).float()
    loss = nll / denom
    if z_loss_weight:
        loss = loss + z_loss_weight * z / denom
    return loss


# --------------------------------------------------------------------------- optimizers
def adamw_step_(p, g, m, v, step: int, lr: float, b1: float, b2: float, eps: float, wd: float):
    """In-place decoupled-weight-decay Adam, same update order as ``torch.optim.AdamW``."""
    gf = g.float()
    pf = p.float() * (1.0 - lr * wd)
    mf = m.float().mul_(b1).add_(gf, alpha=1.0 - b1)
    vf = v.float().mul_(b2).addcmul_(gf, gf, value=1.0 - b2)
    bc1 = 1.0 - b1**step
    bc2 = 1.0 - b2**step
    denom = (vf.sqrt() / math.sqrt(bc2)).add_(eps)
    pf.addcdiv_(mf, denom, value=-lr / bc1)
    p.copy_(pf)
    m.copy_(mf)
    v.copy_(vf)


NS_COEFFS = (3.4445, -4.7750, 2.0315)


def newton_schulz(g: torch.Tensor, steps: int = 5, eps: float = 1e-7) -> torch.Tensor:
    """Quintic Newton-Schulz orthogonalisation of a 2-D matrix in fp32 (no transpose for tall inputs)."""
    a, b, c = NS_COEFFS
    x = g.float()
    x = x / (x.norm() + eps)
    for _ in range(steps):
        gram = x @ x.T
        poly = b * gram + c * (gram @ gram)
        x = a * x + poly @ x
    return x


# --------------------------------------------------------------------------- moe
def grouped_swiglu_experts(
    x_sorted: torch.Tensor,
    counts: torch.Tensor,
    gate_w: torch.Tensor,
    up_w: torch.Tensor,
    down_w: torch.Tensor,
) -> torch.Tensor:
    """Ragged expert SwiGLU.  x_sorted rows are grouped by expert; counts[e] rows go to expert e.

    gate_w/up_w: (E, D, H); down_w: (E, H, D).
    """
    out = torch.empty_like(x_sorted)
    start = 0
    for e, n in enumerate(counts.tolist()):
        if n == 0:
            continue
        seg = x_sorted[start : start + n]
        hid = F.silu(seg @ gate_w[e]) * (seg @ up_w[e])
        out[start : start + n] = hid @ down_w[e]
        start += n
    return out
