"""Sampling and autoregressive generation with per-layer KV caches.

``sample``: temperature -> top-k -> top-p (nucleus) -> multinomial; temperature 0 is greedy.
``generate``: one prefill pass over the prompt, then one token per step against the caches.
``beam_search``: the most likely continuations; the beams of a prompt share its cache and exchange no keys.

Parity: kempnerforge/model/generate.py:15-131 (``beam_search`` has no counterpart there).
"""

from __future__ import annotations

import torch

from kempnerforge_b200.models.attention import KVCache, SharedPrefixCache
from kempnerforge_b200.ops import beam


def sample(logits: torch.Tensor, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
           generator: torch.Generator | None = None) -> torch.Tensor:
    """logits (batch, vocab) -> token ids (batch,); greedy at temperature 0."""
    if temperature <= 0:
        return logits.argmax(dim=-1)
    logits = logits.float() / temperature
    if top_k and top_k > 0:
        k = min(top_k, logits.shape[-1])
        kth = torch.topk(logits, k, dim=-1).values[..., -1:]
        logits = logits.masked_fill(logits < kth, float("-inf"))
    if top_p < 1.0:
        sorted_logits, order = torch.sort(logits, descending=True, dim=-1)
        probs = torch.softmax(sorted_logits, dim=-1)
        cum = probs.cumsum(dim=-1)
        drop = cum - probs >= top_p  # a token is kept while the mass before it is still below the threshold
        sorted_logits = sorted_logits.masked_fill(drop, float("-inf"))
        logits = torch.full_like(logits, float("-inf")).scatter(-1, order, sorted_logits)
    probs = torch.softmax(logits, dim=-1)
    return torch.multinomial(probs, 1, generator=generator).squeeze(-1)


@torch.no_grad()
def generate(model, prompt_tokens: torch.Tensor, max_new_tokens: int, temperature: float = 1.0, top_k: int = 0,
             top_p: float = 1.0, eos_token_id: int | None = None, generator: torch.Generator | None = None) -> torch.Tensor:
    cfg = model.config
    b, plen = prompt_tokens.shape
    total = plen + max_new_tokens
    if total > cfg.max_seq_len:
        raise ValueError(f"prompt ({plen}) + max_new_tokens ({max_new_tokens}) = {total} exceeds model max_seq_len "
                         f"({cfg.max_seq_len})")
    if max_new_tokens <= 0:
        return prompt_tokens
    param = next(model.parameters())
    hd = cfg.head_dim
    caches = [KVCache(b, total, layer.attention.k_proj.weight.shape[0] // hd, hd, param.dtype, param.device)
              for layer in model.layers.values()]
    was_training = model.training
    model.eval()
    logits = model(prompt_tokens, kv_caches=caches)
    out = prompt_tokens
    done = torch.zeros(b, dtype=torch.bool, device=prompt_tokens.device)
    for _ in range(total - plen):
        nxt = sample(logits[:, -1], temperature, top_k, top_p, generator)[:, None]
        if eos_token_id is not None:
            nxt = torch.where(done[:, None], torch.full_like(nxt, eos_token_id), nxt)
            done |= nxt.squeeze(-1) == eos_token_id
        out = torch.cat([out, nxt], dim=1)
        if out.shape[1] >= total or (eos_token_id is not None and bool(done.all())):
            break
        logits = model(nxt, kv_caches=caches)
    if was_training:
        model.train()
    return out


@torch.no_grad()
def beam_search(model, prompt_tokens: torch.Tensor, max_new_tokens: int, num_beams: int = 4, eos_token_id: int | None = None,
                length_penalty: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """The ``num_beams`` best continuations that a beam search finds for each prompt (batch, prompt length): (token ids
    (batch, num_beams, prompt length + new), scores (batch, num_beams) fp32), best first.

    A score is the sum of the new tokens' log-probabilities divided by their number to the power ``length_penalty`` (an
    ``eos_token_id`` counts, what follows it does not, and is filled with it).  During the search beams compete by their sums; a finished
    one keeps its place as long as its sum does.  The search ends when all beams that there are have finished, or at ``max_new_tokens``.
    """
    cfg = model.config
    b, plen = prompt_tokens.shape
    w, total = int(num_beams), plen + max_new_tokens
    if w < 1 or w > 256:
        raise ValueError(f"num_beams {num_beams} is not between 1 and 256")
    if plen < 1:
        raise ValueError("a search needs a prompt of at least one token")
    if total > cfg.max_seq_len:
        raise ValueError(f"prompt ({plen}) + max_new_tokens ({max_new_tokens}) = {total} exceeds model max_seq_len "
                         f"({cfg.max_seq_len})")
    dev = prompt_tokens.device
    if max_new_tokens <= 0 or b == 0:
        return prompt_tokens[:, None].expand(b, w, plen).clone(), torch.zeros(b, w, device=dev)
    param = next(model.parameters())
    hd = cfg.head_dim
    caches = [KVCache(b, plen, layer.attention.k_proj.weight.shape[0] // hd, hd, param.dtype, param.device)
              for layer in model.layers.values()]
    was_training = model.training
    model.eval()
    logits = model(prompt_tokens, kv_caches=caches)[:, -1:].expand(b, w, -1)
    rows = SharedPrefixCache.new_rows(b, w, max_new_tokens, dev)
    caches = [SharedPrefixCache(c, w, max_new_tokens, rows) for c in caches]
    pad = 0 if eos_token_id is None else eos_token_id
    scores = torch.full((b, w), float("-inf"), device=dev)
    scores[:, 0] = 0.0   # the beams of a prompt are one until the first choice
    finished = torch.zeros(b, w, dtype=torch.bool, device=dev)
    tokens = torch.full((b, w, max_new_tokens), pad, dtype=torch.int64, device=dev)
    for n in range(max_new_tokens):
        step = beam.select(logits, scores, finished, eos_token_id, pad)
        if n:
            beam.reorder([tokens, rows], step.parents, n)
        tokens[:, :, n] = step.tokens
        scores, finished = step.scores, step.finished
        # a place without a continuation stays one: where the others have finished, nothing can come
        if n + 1 == max_new_tokens or (eos_token_id is not None and bool((finished | scores.isneginf()).all())):
            break
        logits = model(step.tokens.view(b * w, 1), kv_caches=caches)[:, -1].view(b, w, -1)
    if was_training:
        model.train()
    tokens = tokens[:, :, : n + 1]
    ends = (tokens == eos_token_id) if eos_token_id is not None else torch.zeros_like(tokens, dtype=torch.bool)
    lengths = (ends.cumsum(2) - ends.long() == 0).sum(2)
    scores, order = (scores / lengths**length_penalty).sort(dim=1, descending=True, stable=True)
    tokens = tokens.gather(1, order[:, :, None].expand_as(tokens))
    return torch.cat([prompt_tokens[:, None].expand(b, w, plen), tokens], dim=2), scores
