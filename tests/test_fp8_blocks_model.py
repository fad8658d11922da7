"""Models whose fp8 Linear layers have a scale for each block of 128: configuration, the norms that write 8 bits, training and generation."""

import pytest
import torch

from kempnerforge_b200.config import ModelConfig, TrainConfig, config_from_dict
from kempnerforge_b200.models import Transformer
from kempnerforge_b200.models.generate import generate
from kempnerforge_b200.ops import fp8, fp8_blocks as fb
from kempnerforge_b200.ops import functional as F

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]


def _model(device, scaling="block128", ac="none", **kw):
    torch.manual_seed(0)
    cfg = ModelConfig(**{**dict(dim=128, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=256, ffn_hidden_dim=272, max_seq_len=64, init_std=0.1), **kw})
    model = Transformer(cfg).to(device=device, dtype=torch.bfloat16)
    if scaling is not None:
        fp8.convert_model(model, scaling=scaling)
    for block in model.layers.values():
        block.ac_mode = ac
    tokens = torch.randint(0, 256, (3, 38), generator=torch.Generator().manual_seed(1)).to(device)
    return model, tokens


def _count(monkeypatch):
    calls, real = [], fb.norm_linear
    monkeypatch.setattr(fb, "norm_linear", lambda *a: calls.append(a[1] is not None) or real(*a))
    return calls


def test_configuration():
    assert TrainConfig().fp8_scaling == "tensor" and TrainConfig(mixed_precision="fp8", fp8_scaling="block128").fp8_scaling == "block128"
    with pytest.raises(ValueError):
        TrainConfig(fp8_scaling="row")
    with pytest.raises(ValueError):
        fp8.convert_model(torch.nn.Linear(16, 16), scaling="row")
    with pytest.raises(ValueError):   # as with a scale per tensor
        config_from_dict({"model": dict(dim=64, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=128, max_seq_len=32), "distributed": {"tp": 2},
                          "train": dict(mixed_precision="fp8", fp8_scaling="block128", batch_size=1, seq_len=32)}).validate(2)


def test_a_model_tagged_again_takes_the_other_scaling():
    model, tokens = _model("cpu")
    fp8.convert_model(model)
    again, _ = _model("cpu", "tensor")
    assert torch.equal(model(tokens), again(tokens))


def _by_hand(block, x, cos, sin):
    """A block written out in the operators."""
    att, mlp = block.attention, block.mlp
    b, s, _ = x.shape
    t, qkv = fb.norm_linear(x, None, block.attention_norm.weight, [att.q_proj.weight, att.k_proj.weight, att.v_proj.weight], block.attention_norm.eps)
    h, hkv, hd = att.n_heads, att.n_kv_heads, att.head_dim
    qkv = F.rope(qkv.view(b, s, h + 2 * hkv, hd), cos, sin, n_rot_heads=h + hkv)
    out = F.attention(qkv[:, :, :h], qkv[:, :, h : h + hkv], qkv[:, :, h + hkv :])
    t, gu = fb.norm_linear(t, fb.linear(out.reshape(b, s, h * hd), [att.o_proj.weight]), block.mlp_norm.weight,
                           [mlp.gate_proj.weight, mlp.up_proj.weight], block.mlp_norm.eps)
    return t + fb.linear(F.swiglu_stacked(gu), [mlp.down_proj.weight])


@pytest.mark.parametrize("device", DEVICES)
def test_a_block_is_the_operators_in_a_row(device, monkeypatch):
    model, tokens = _model(device)
    block = model.layers["1"]
    x = torch.randn(3, 37, 128, generator=torch.Generator().manual_seed(2)).to(device, torch.bfloat16).requires_grad_()
    dy = torch.randn(3, 37, 128, generator=torch.Generator().manual_seed(3)).to(device, torch.bfloat16)
    cos, sin = model.rope_tables(x.device, 0, 37)
    leaves = [x, *block.parameters()]
    calls = _count(monkeypatch)
    y = block(x, cos, sin)
    assert calls == [False, True]
    want = _by_hand(block, x, cos, sin)
    assert torch.equal(y, want)
    names = ["x", *(n for n, _ in block.named_parameters())]
    for name, a, b in zip(names, torch.autograd.grad(y, leaves, dy), torch.autograd.grad(want, leaves, dy)):
        assert bool((a != 0).any())
        # the attention's backward kernel adds in the order in which its blocks finish
        assert torch.equal(a, b) or (device == "cuda" and name.startswith(("x", "attention.q", "attention.k", "attention.v", "attention_norm"))), name


@pytest.mark.parametrize("device", DEVICES)
def test_a_product_is_as_near_as_its_operands(device):
    """Both operands are off by 2^-4 of a value at most (and of what is 2^-16 of its block's largest, by that), the output by half a step of
    bf16: a bound for every element."""
    model, _ = _model(device)
    w = model.layers["0"].mlp.down_proj.weight.detach()
    x = torch.randn(50, w.shape[1], generator=torch.Generator().manual_seed(2)).to(device, torch.bfloat16)
    got = fb.linear(x, [w])
    xa, wa = x.double().abs(), w.double().abs()
    off = lambda v: v * 2**-4 + v.max() * 2**-16   # noqa: E731
    bound = off(xa) @ wa.t() + xa @ off(wa).t() + off(xa) @ off(wa).t()
    want = x.double() @ w.double().t()
    assert bool(((got.double() - want).abs() <= bound + 2**-8 * (want.abs() + bound)).all())


@pytest.mark.parametrize("device", DEVICES)
def test_hooks_and_other_norms_see_what_they_would(device, monkeypatch):
    model, tokens = _model(device)
    calls = _count(monkeypatch)
    plain = model(tokens)
    assert len(calls) == 4
    seen = []
    handles = [b.mlp_norm.register_forward_hook(lambda m, i, o: seen.append(o)) for b in model.layers.values()]
    handles.append(model.layers["0"].attention.register_forward_pre_hook(lambda m, i: seen.append(i[0])))
    watched = model(tokens)
    assert len(calls) == 5 and len(seen) == 3                                 # the second block's first norm is watched by none
    assert seen[0].float().square().mean(-1).sub(1).abs().max() < 0.05        # normalised, and rounded to bf16
    for h in handles:
        h.remove()
    assert torch.equal(model(tokens), plain)
    real = fb.norm_linear_of
    skip = {id(model.layers["0"].attention_norm), *(id(b.mlp_norm) for b in model.layers.values())}
    monkeypatch.setattr(fb, "norm_linear_of", lambda norm, *a: None if id(norm) in skip else real(norm, *a))
    assert torch.equal(model(tokens), watched)
    odd, _ = _model(device, norm_type="layernorm")
    k = len(calls)
    assert odd(tokens).isfinite().all() and len(calls) == k


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("ac", ["full", "selective"])
def test_recomputation_gives_the_same_gradients(device, ac, monkeypatch):
    grads = []
    if ac == "selective":   # recomputes the attention branch, whose norm is not in one node with the residual
        monkeypatch.setattr(type(_model(device)[0].layers["0"]), "_fp8_qkv", lambda self, x: None)
    for mode in ("none", ac):
        model, tokens = _model(device, ac=mode)
        model.compute_loss(tokens[:, :-1], tokens[:, 1:]).backward()
        grads.append({n: p.grad for n, p in model.named_parameters()})
    # the attention's and the embedding's backward kernels add in the order in which their blocks finish: on a GPU the last block's
    # gradients up to its attention are the ones that have the same bits every time
    for name, g in grads[0].items():
        if device == "cpu" or name.startswith(("layers.1.mlp", "layers.1.attention.o_proj", "norm", "output_head")):
            assert torch.equal(g, grads[1][name]), name


@pytest.mark.parametrize("device", DEVICES)
def test_generation_one_token_at_a_time(device, monkeypatch):
    model, tokens = _model(device)
    calls = _count(monkeypatch)
    out = generate(model, tokens[:, :5], 7, temperature=0)
    assert out.shape == (3, 12) and torch.equal(out[:, :5], tokens[:, :5]) and len(calls) == 7 * 4
    # the same weights and rows in another number of rows: greedy tokens of the whole sequence, where they are clear
    logits = model(out[:, :-1]).float()
    best = logits[:, 4:].topk(2, -1)
    clear = best.values[..., 0] - best.values[..., 1] > 0.05 * logits.abs().max()
    assert clear.any() and torch.equal(best.indices[..., 0][clear], out[:, 5:][clear])


@pytest.mark.parametrize("device", DEVICES)
def test_training_steps_through_flat_buffers(device):
    from kempnerforge_b200.parallel.flat import FlatParamGroup
    from kempnerforge_b200.training.optimizer import FusedAdamW

    model, tokens = _model(device)
    plain, _ = _model(device)
    groups = [FlatParamGroup(name, block.named_parameters()) for name, block in model.layers.items()]
    opt = FusedAdamW(model.parameters(), lr=1e-2)
    opt.attach_flat_groups(groups)
    for step in range(3):
        for _ in range(2):                                    # two micro-batches add up
            model.compute_loss(tokens[:, :-1], tokens[:, 1:]).backward()
        for g in groups:
            g.finalize_grads()
        if step == 0:
            for _ in range(2):
                plain.compute_loss(tokens[:, :-1], tokens[:, 1:]).backward()
            for (name, p), q in zip(model.layers.named_parameters(), plain.layers.parameters()):
                got = p._kf_grad if hasattr(p, "_kf_grad") else p.grad
                # the second gradient is added before its rounding, or after it
                assert bool(((got - q.grad).double().abs() <= 2**-7 * (got.double().abs() + q.grad.double().abs()).clamp_min(q.grad.double().abs().max() * 2**-8)).all())
        before = model(tokens).detach()
        opt.step()
        w = model.layers["0"].mlp.gate_proj.weight, model.layers["0"].mlp.up_proj.weight
        kept, fresh = fb.quantized_weight(w, True), fb.quantize(torch.cat([v.detach() for v in w]), square=True, want_t=True)
        assert all(torch.equal(a.values, b.values) and torch.equal(a.scales, b.scales) for a, b in zip(kept, fresh))
        assert not torch.equal(before, model(tokens))
        opt.zero_grad()
        for g in groups:
            g.zero_grad()


def test_a_mixture_of_experts_keeps_its_experts_in_bf16():
    model, tokens = _model("cpu", num_experts=4, moe_top_k=2, moe_frequency=2)
    tagged = {n for n, p in model.named_parameters() if fp8.has_block_scales(p)}
    assert tagged and not any("experts" in n or "router" in n for n in tagged)
    model.compute_loss(tokens[:, :-1], tokens[:, 1:]).backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in model.parameters() if p.requires_grad and p.grad is not None)


def test_the_trainer_builds_and_steps_it(tmp_path):
    from kempnerforge_b200.training.trainer import Trainer

    cfg = config_from_dict({
        "model": dict(dim=64, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=128, max_seq_len=32, ffn_hidden_dim=128),
        "train": dict(mixed_precision="fp8", fp8_scaling="block128", batch_size=2, seq_len=32, max_steps=2, activation_checkpointing="full"),
        "scheduler": dict(name="constant", warmup_steps=0), "checkpoint": dict(dir=str(tmp_path)),
    })
    trainer = Trainer(cfg)
    assert fp8.has_block_scales(trainer.model.layers["0"].mlp.gate_proj.weight)
    tok = torch.randint(0, 128, (2, 33))
    before = trainer.model.layers["0"].mlp.gate_proj.weight.detach().clone()
    trainer.train_step([{"input_ids": tok[:, :-1], "labels": tok[:, 1:]}])
    assert not torch.equal(before, trainer.model.layers["0"].mlp.gate_proj.weight)


@pytest.mark.parametrize("device", DEVICES)
def test_selective_recomputation_takes_the_same_norms(device, monkeypatch):
    """The attention's norm writes 8 bits inside of a recomputed branch too: outputs and losses are those of the other modes."""
    losses, grads = [], []
    for mode in ("none", "selective", "full"):
        model, tokens = _model(device, ac=mode)
        calls = _count(monkeypatch)
        loss = model.train().compute_loss(tokens[:, :-1], tokens[:, 1:])
        assert len(calls) == 4
        loss.backward()
        losses.append(loss.detach())
        grads.append({n: p.grad for n, p in model.named_parameters()})
        logits = model(tokens)
        with torch.no_grad():
            assert torch.equal(logits, model.eval()(tokens))
        monkeypatch.undo()
    assert torch.equal(losses[0], losses[1]) and torch.equal(losses[0], losses[2])
    # the gradient of the last block's first norm is added to the residual's in another node: what is behind it has the same bits
    for name, g in grads[0].items():
        assert grads[1][name].isfinite().all()
        if name.startswith(("layers.1.mlp", "layers.1.attention.o_proj", "norm", "output_head")):
            assert torch.equal(g, grads[1][name]) and torch.equal(g, grads[2][name]), name
