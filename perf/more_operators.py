"""Operators of beam search and of many continuations of one prompt: what is measured, in plain form and through the framework.

``attend``   attention of one new token for each of `beams` continuations of a prompt: over the prompt's keys, which all of them share,
             and over the keys of their own tokens; with `table` a continuation's own keys lie where its ancestors wrote them
``select``   a step of beam search: the best `beams` of all (beam, token) pairs, by log-probability added to the beam's score
``reorder``  every beam's state becomes its parent's: histories of tokens, tables, caches
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
NONE = float("-inf")

# heads, key heads and head dim of the presets: the 125 M benchmark model, moe_small, llama_7b, llama_13b, llama_70b
HEADS = {"125m": (12, 12, 64), "small": (16, 4, 128), "7b": (32, 8, 128), "13b": (40, 8, 128), "70b": (64, 8, 128)}
VOCABS = (32000, 50257, 102400, 128256)


def listed() -> list[dict]:
    return [
        # interactive beam search with the 125 M model, a short prompt: latency
        dict(name="attend_125m_1x4", kind="attend", model="125m", prompts=1, beams=4, prefix=300, steps=20, ragged=False, table=True),
        # beam search over a long prompt with a 7B model
        dict(name="attend_7b_1x8", kind="attend", model="7b", prompts=1, beams=8, prefix=4000, steps=96, ragged=False, table=True),
        # a batch of short prompts
        dict(name="attend_small_24x8", kind="attend", model="small", prompts=24, beams=8, prefix=512, steps=31, ragged=False, table=True),
        # a padded batch of uneven prompts, 13B, an odd number of beams
        dict(name="attend_13b_8x5_ragged", kind="attend", model="13b", prompts=8, beams=5, prefix=1777, steps=65, ragged=True, table=True),
        # sampling: 64 answers to each of two long prompts, each with its own tokens
        dict(name="attend_7b_2x64_sampled", kind="attend", model="7b", prompts=2, beams=64, prefix=8000, steps=257, ragged=False, table=False),
        # beam search over whole documents, 70B heads
        dict(name="attend_70b_4x8_long", kind="attend", model="70b", prompts=4, beams=8, prefix=32768, steps=200, ragged=False, table=True),
        # interactive beam search, one prompt
        dict(name="select_1x4x32000", kind="select", prompts=1, beams=4, vocab=32000, half=True, finished=0),
        # scores in 32 bits, an odd vocabulary, one beam at its end
        dict(name="select_3x5x50257_fp32", kind="select", prompts=3, beams=5, vocab=50257, half=False, finished=1),
        # translating a data set: a large batch
        dict(name="select_64x8x128256", kind="select", prompts=64, beams=8, vocab=128256, half=True, finished=1),
        # what every step of beam search moves: tokens so far and the table of ancestors
        dict(name="reorder_histories_16x8", kind="reorder", prompts=16, beams=8, room=2048, length=777, width=0, states=2),
        # caches of all layers of the 125 M model, keys and values
        dict(name="reorder_caches_125m_2x4", kind="reorder", prompts=2, beams=4, room=512, length=333, width=768, states=24),
        # caches of eight layers of a 7B model
        dict(name="reorder_caches_7b_4x8", kind="reorder", prompts=4, beams=8, room=1024, length=1000, width=1024, states=16),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["attend", "attend", "attend", "select", "select", "reorder"])
    while kind == "attend":
        c = dict(kind=kind, model=rng.choice(sorted(HEADS)), prompts=_log_int(rng, 1, 24), beams=_log_int(rng, 2, 64),
                 prefix=_log_int(rng, 1, 32768), steps=_log_int(rng, 1, 300), ragged=rng.random() < 0.4, table=rng.random() < 0.6)
        if c["table"]:
            c["beams"] = min(c["beams"], 32)
        heads, kv, dim = HEADS[c["model"]]
        rows = c["prompts"] * c["beams"]
        if c["prompts"] * c["prefix"] <= 4 * 32768 and rows * c["steps"] * kv * dim <= 1 << 26 and rows * heads * c["prefix"] <= 1 << 27:
            return c
    if kind == "select":
        return dict(kind=kind, prompts=_log_int(rng, 1, 64), beams=rng.randint(2, 8), vocab=rng.choice(VOCABS) if rng.random() < 0.5 else _log_int(rng, 500, 128256),
                    half=rng.random() < 0.6, finished=rng.randint(0, 1))
    while True:
        c = dict(kind=kind, prompts=_log_int(rng, 1, 16), beams=_log_int(rng, 2, 16), room=_log_int(rng, 64, 2048), length=0,
                 width=rng.choice([0, 0, 256, 768, 1024]), states=2)
        c["length"] = _log_int(rng, 1, c["room"])
        if c["width"]:
            c["states"] = 2 * rng.randint(1, 12)
        if c["prompts"] * c["beams"] * c["room"] * c["width"] * c["states"] <= 1 << 29:
            return c


# --------------------------------------------------------------------------- inputs
def _normal(g, *shape, std=1.0):
    return torch.empty(shape, device=DEV).normal_(0.0, std, generator=g)


def _lengths(case) -> list[int]:
    """Prompt lengths: down to half of the longest where the batch is ragged."""
    n, p = case["prompts"], case["prefix"]
    return [max(1, p - i * p // (2 * n)) if case["ragged"] else p for i in range(n)]


def _ancestors(rng, beams: int, steps: int) -> list[list[int]]:
    """Row w, entry s: the slot in which the ancestor of beam w was when it wrote position s (the newest position is the beam's own)."""
    at, table = list(range(beams)), []
    for _ in range(steps):
        table.append(at)
        parents = sorted(rng.randrange(beams) for _ in range(beams))   # a step before: who came from whom
        at = [parents[a] for a in at]
    return [list(row) for row in zip(*reversed(table))]


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    rng = random.Random(int(seed))
    n, w = case["prompts"], case["beams"]
    if case["kind"] == "attend":
        heads, kv, dim = HEADS[case["model"]]
        p, s = case["prefix"], case["steps"]
        lean = _normal(g, 1, 1, kv, dim)                              # keys have a mean, queries a few large channels
        st = dict(kind="attend", q=_normal(g, n, w, heads, dim), k=(_normal(g, n, p, kv, dim) + lean).bfloat16(), v=_normal(g, n, p, kv, dim).bfloat16())
        st["q"][..., torch.randint(0, dim, (3,), device=DEV, generator=g)] *= 4.0
        st["q"] = st["q"].bfloat16()
        # the continuations' caches have room for more tokens than there are so far
        room = s + 64
        keys, values = (_normal(g, n, w, room, kv, dim) + lean).bfloat16(), _normal(g, n, w, room, kv, dim).bfloat16()
        st["own_k"], st["own_v"] = keys[:, :, :s], values[:, :, :s]
        lens = _lengths(case)
        rng.shuffle(lens)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV) if case["ragged"] else None
        st["table"] = None
        if case["table"]:
            table = torch.zeros(n, w, -(-room // 16) * 16, dtype=torch.uint8, device=DEV)
            table[:, :, :s] = torch.tensor([_ancestors(rng, w, s) for _ in range(n)], dtype=torch.uint8, device=DEV)
            st["table"] = table[:, :, :s]
        return st
    if case["kind"] == "select":
        v = case["vocab"]
        logits = _normal(g, n, w, v, std=2.5)
        logits[:, :, torch.randint(0, v, (max(1, v // 100),), device=DEV, generator=g)] = NONE   # tokens that must not appear
        st = dict(kind="select", logits=logits.bfloat16() if case["half"] else logits, eos=v - 1)
        st["scores"] = -torch.sort(torch.empty(n, w, device=DEV).uniform_(5.0, 30.0, generator=g), 1).values
        st["finished"] = torch.zeros(n, w, dtype=torch.bool, device=DEV)
        if case["finished"]:
            st["finished"].scatter_(1, torch.randint(0, w, (n, 1), device=DEV, generator=g), True)
        return st
    st = dict(kind="reorder", length=case["length"], parents=torch.sort(torch.randint(0, w, (n, w), device=DEV, generator=g), 1).values)
    if case["width"]:
        st["states"] = [_normal(g, n, w, case["room"], case["width"]).bfloat16() for _ in range(case["states"])]
    else:
        st["states"] = [torch.randint(0, 32000, (n, w, case["room"]), device=DEV, generator=g),
                        torch.randint(0, w, (n, w, case["room"]), device=DEV, generator=g, dtype=torch.uint8)]
    st["out"] = [torch.zeros_like(x) for x in st["states"]]           # two sets of states that change places
    return st


# --------------------------------------------------------------------------- one pass
def run(state: dict):
    if own:
        return _run_own(state)
    with torch.no_grad():
        if state["kind"] == "attend":
            return _attend(state)
        if state["kind"] == "select":
            return _select(state["logits"], state["scores"], state["finished"], state["eos"])
        return [_take(x, out, state["parents"], state["length"]) for x, out in zip(state["states"], state["out"])]


def _attend(st):
    q, k, v, own_k, own_v = (st[name].float() for name in ("q", "k", "v", "own_k", "own_v"))
    n, w, heads, dim = q.shape
    kv, p, s = k.shape[2], k.shape[1], own_k.shape[2]
    q = q.view(n, w, kv, heads // kv, dim) / math.sqrt(dim)
    shared = torch.einsum("nwkgd,npkd->nwkgp", q, k)
    if st["lens"] is not None:
        hidden = torch.arange(p, device=q.device) >= st["lens"][:, None]
        shared = shared.masked_fill(hidden[:, None, None, None], NONE)
        v = v.masked_fill(hidden[:, :, None, None], 0.0)
    if st["table"] is not None:
        rows = st["table"].long()[..., None, None].expand(n, w, s, kv, dim)
        own_k, own_v = torch.gather(own_k, 1, rows), torch.gather(own_v, 1, rows)
    mine = torch.einsum("nwkgd,nwskd->nwkgs", q, own_k)
    top = torch.maximum(shared.amax(-1), mine.amax(-1))[..., None]
    shared, mine = torch.exp(shared - top), torch.exp(mine - top)
    out = torch.einsum("nwkgp,npkd->nwkgd", shared, v) + torch.einsum("nwkgs,nwskd->nwkgd", mine, own_v)
    out = out / (shared.sum(-1) + mine.sum(-1))[..., None]
    return out.reshape(n, w, heads, dim).bfloat16()


def _select(logits, scores, finished, eos):
    """In 64 bits: the order of candidates of different beams hangs on the sums over the vocabulary."""
    n, w, vocab = logits.shape
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    total = scores.double()[..., None] + (x - top) - torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    stays = torch.full_like(total, NONE)
    stays[..., eos] = scores.double()
    total = torch.where(finished[..., None], stays, total).view(n, w * vocab)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :w], at[:, :w]
    parents, tokens = at // vocab, at % vocab
    return dict(scores=best.float(), parents=parents, tokens=tokens, finished=torch.gather(finished, 1, parents) | (tokens == eos))


def _take(x, out, parents, length):
    out[:, :, :length] = x[torch.arange(x.shape[0], device=x.device)[:, None], parents, :length]
    return out


def _run_own(st: dict):
    from kempnerforge_b200.ops import beam
    from kempnerforge_b200.ops import functional as F

    if st["kind"] == "attend":
        return F.shared_prefix_attention(st["q"], st["k"], st["v"], st["own_k"], st["own_v"], prefix_lens=st["lens"], own_rows=st["table"])
    if st["kind"] == "select":
        return beam.select(st["logits"], st["scores"], st["finished"], eos_id=st["eos"], pad_id=st["eos"])._asdict()
    return beam.reorder(st["states"], st["parents"], st["length"], out=st["out"])


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case: dict) -> dict:
    n, w = case["prompts"], case["beams"]
    if case["kind"] == "attend":
        heads, kv, dim = HEADS[case["model"]]
        shared, s = sum(_lengths(case)), case["steps"]
        mine = n * w * s
        if case["table"]:   # own keys that some beam still has, for one course of events
            mine = n * sum(len(set(column)) for column in zip(*_ancestors(random.Random(1), w, s)))
        # keys and values once, q in and the result out, the table's bytes
        return dict(bytes=4 * (shared + mine) * kv * dim + 4 * n * w * heads * dim + (n * w * s if case["table"] else 0),
                    flops=4 * w * heads * dim * (shared + n * s))
    if case["kind"] == "select":
        values = n * (w - case["finished"]) * case["vocab"]
        return dict(bytes=values * (2 if case["half"] else 4) + n * w * 26, flops=4 * values)
    unit = 2 * case["width"] * case["states"] if case["width"] else 9
    parents = w * (1 - (1 - 1 / w) ** w)      # how many different ones, on the average
    return dict(bytes=n * case["length"] * unit * (parents + w) + 8 * n * w, flops=0)


# --------------------------------------------------------------------------- 64 bits, from the definition
@torch.no_grad()
def exact(case: dict, seed: int):
    st = prepare(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(st)
    if case["kind"] == "select":
        return _exact_select(st)
    n, w = case["prompts"], case["beams"]
    results = []
    for x in st["states"]:
        y = torch.zeros_like(x)
        for b in range(n):
            y[b, :, : case["length"]] = x[b].index_select(0, st["parents"][b])[:, : case["length"]]
        results.append(y)
    return results


def _exact_attend(st):
    """Prompt by prompt and continuation by continuation: softmax over the keys that it sees, side by side."""
    n, w, heads, dim = st["q"].shape
    group = heads // st["k"].shape[2]
    out = torch.empty(n, w, heads, dim, dtype=torch.float64, device=DEV)
    for b in range(n):
        length = st["k"].shape[1] if st["lens"] is None else int(st["lens"][b])
        k, v = st["k"][b, :length].double(), st["v"][b, :length].double()
        for i in range(w):
            if st["table"] is None:
                mine_k, mine_v = st["own_k"][b, i], st["own_v"][b, i]
            else:
                at = torch.arange(st["own_k"].shape[2], device=DEV)
                mine_k, mine_v = st["own_k"][b, st["table"][b, i].long(), at], st["own_v"][b, st["table"][b, i].long(), at]
            keys, values = torch.cat([k, mine_k.double()]).transpose(0, 1), torch.cat([v, mine_v.double()]).transpose(0, 1)
            q = st["q"][b, i].double().view(-1, group, dim)
            weights = torch.softmax(q @ keys.transpose(1, 2) * dim ** -0.5, -1)
            out[b, i] = (weights @ values).reshape(heads, dim)
    return out


def _exact_select(st):
    """The largest candidate, `beams` times over."""
    logits, scores, finished, eos = st["logits"].double(), st["scores"].double(), st["finished"], st["eos"]
    n, w, vocab = logits.shape
    total = torch.log_softmax(logits, -1) + scores[..., None]
    for b, i in torch.nonzero(finished).tolist():
        total[b, i] = NONE
        total[b, i, eos] = scores[b, i]
    total = total.view(n, w * vocab)
    picked = dict(scores=[], parents=[], tokens=[], finished=[])
    for _ in range(w):
        at = total.argmax(1, keepdim=True)
        picked["scores"].append(total.gather(1, at))
        picked["parents"].append(at // vocab)
        picked["tokens"].append(at % vocab)
        picked["finished"].append(finished.gather(1, at // vocab) | (at % vocab == eos))
        total.scatter_(1, at, NONE)
    return {name: torch.cat(parts, 1) for name, parts in picked.items()}
