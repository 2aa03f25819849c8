"""Positions scaled for long contexts as a part of a model, and prompts taken from a step's rows instead of the cache."""

from __future__ import annotations

import pytest
import torch

H, NQ, NKV, VOCAB, LAYERS = 96, 4, 2, 83, 2
YARN = {"factor": 8.0, "original": 64, "fast": 32.0, "slow": 1.0}
WAVES = {"factor": 8.0, "low": 1.0, "high": 4.0, "original": 64}


def build(dtype, position, head_dim=64, whole_prompts=False, norm_eps=None):
    from edgerag_b200.cache.device import DevicePools
    from edgerag_b200.cache.manager import CacheManager
    from edgerag_b200.engine.step import ModelRunner
    from edgerag_b200.models.decoder import DecoderModel
    from edgerag_b200.parts.base import LayerCall, LayerSpec, ModelPlan, PartSpec

    norm = lambda p: PartSpec("rmsnorm", {"size": H, "eps": 1e-5}, p)   # noqa: E731
    how = {"hidden": H, "n_q_heads": NQ, "n_kv_heads": NKV, "head_dim": head_dim, "position": position}
    how |= {"whole_prompts": True} if whole_prompts else {}
    how |= {"qk_norm_eps": norm_eps} if norm_eps else {}
    specs = [LayerSpec(f"layers.{i}.", PartSpec("prenorm"), norm("ln1."), PartSpec("attention", how, "self_attn."), norm("ln2."),
                       PartSpec("swiglu", {"hidden": H, "intermediate": 64}, "mlp.")) for i in range(LAYERS)]
    plan = ModelPlan(H, VOCAB, PartSpec("table", {"vocab": VOCAB, "hidden": H}, "embed."), specs, [LayerCall(i, i) for i in range(LAYERS)], norm("norm."),
                     PartSpec("linear", {"vocab": VOCAB, "hidden": H, "tied_to": None}, "lm_head."))
    device = torch.device("cuda")
    model = DecoderModel(plan, dtype, device)
    g = torch.Generator().manual_seed(7)
    tensors = {s.name: 1 + 0.1 * torch.randn(s.shape, generator=g) if "norm" in s.name or "ln" in s.name else 0.15 * torch.randn(s.shape, generator=g)
               for s in model.weight_specs()}
    model.load_weights(tensors)
    cache = CacheManager(model.cache_layout, 16, 64, 8)
    return ModelRunner(model, cache, DevicePools(model.cache_layout, 16, [64], 8, dtype, device), 512, check_status=True)


def walk(runner, sequences, portions):
    """The logits of every token, each sequence cut into `portions` of its length, step by step beside the others."""
    from edgerag_b200.engine.step import StepEntry

    got, fed = {i: [] for i in range(len(sequences))}, [0] * len(sequences)
    for i in range(len(sequences)):
        runner.admit(i)
    for cut in range(max(len(p) for p in portions)):
        entries = [(i, sequences[i][fed[i]: fed[i] + p[cut]]) for i, p in enumerate(portions) if cut < len(p)]
        logits = runner.step([StepEntry(i, tokens=list(t), want=list(range(len(t)))) for i, t in entries]).float().cpu()
        row = 0
        for i, t in entries:
            got[i].append(logits[row: row + len(t)].clone())
            row += len(t)
            fed[i] += len(t)
    for i in range(len(sequences)):
        runner.release(i)
    return [torch.cat(got[i]) for i in range(len(sequences))]


def spec(**how):
    from edgerag_b200.parts.base import PartSpec

    return PartSpec("rope_scaled", {"theta": 1000.0, **how})


SEQUENCES = [[(7 * i + 3 * j) % VOCAB for j in range(n)] for i, n in enumerate((70, 33, 5))]


@pytest.mark.gpu
@pytest.mark.parametrize("head_dim,how", [(64, {}), (64, {"rot_dim": 32}), (128, {}), (48, {"rot_dim": 16})])
def test_unscaled_it_is_the_plain_rotation(head_dim, how):
    from edgerag_b200.parts.base import PartSpec

    plain = build(torch.float32, PartSpec("rope_halves", {"head_dim": head_dim, "theta": 1000.0, "precise": True, **how}), head_dim)
    scaled = build(torch.float32, spec(head_dim=head_dim, **how), head_dim)
    portions = [[70], [20, 13], [1, 4]]
    for a, b in zip(walk(plain, SEQUENCES, portions), walk(scaled, SEQUENCES, portions)):
        assert (a - b).abs().max() <= 2e-4 + 2e-4 * b.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("head_dim,how,norm_eps", [(64, {"scaling": YARN}, None), (128, {"scaling": WAVES, "pairs": True}, 1e-5), (64, {"scaling": YARN, "rot_dim": 32}, 1e-6)])
def test_prompts_from_their_rows_as_from_the_cache(dtype, head_dim, how, norm_eps):
    """Whole prompts, portions behind a past, single tokens beside new prompts: one way and the other."""
    position = spec(head_dim=head_dim, **how)
    cached, rows = (build(dtype, position, head_dim, whole, norm_eps) for whole in (False, True))
    for portions in ([[70], [33], [5]], [[40, 30], [1] * 33, [5]], [[69, 1], [30, 3], [1, 4]]):
        for a, b in zip(walk(cached, SEQUENCES, portions), walk(rows, SEQUENCES, portions)):
            scale = a.abs().max()
            assert torch.isfinite(b).all()
            assert (a - b).abs().max() <= (2e-4 + 2e-4 * scale if dtype == torch.float32 else 0.02 * scale)


@pytest.mark.gpu
def test_captured_steps_know_whole_prompts_from_portions():
    """The same layout of tokens, once at a prompt's beginning and once behind a past: two graphs."""
    from edgerag_b200.engine.step import StepEntry

    runner = build(torch.bfloat16, spec(head_dim=64, scaling=YARN), 64, True)
    runner.graphs_enabled = True
    runner._meta_dev = torch.empty(1 << 20, dtype=torch.int32, device="cuda")
    eager = build(torch.bfloat16, spec(head_dim=64, scaling=YARN), 64, True)
    for turn in range(4):
        tokens = [(5 * j + turn) % VOCAB for j in range(40)]
        for r in (runner, eager):
            r.admit("a")
        for part in (tokens[:20], tokens[20:]):
            a, b = (r.step([StepEntry("a", tokens=part, want=[19])]).float().cpu().clone() for r in (runner, eager))
            assert torch.equal(a, b)
        for r in (runner, eager):
            r.release("a")
    assert runner.graph_replays >= 4 and len(runner._graphs) == 2


def test_what_does_not_go_together_is_refused():
    from edgerag_b200.parts.attention import Attention
    from edgerag_b200.parts.base import PartSpec, build_part

    make = lambda position, **how: Attention(64, 4, 2, 16, position, torch.float32, torch.device("cpu"), **how)   # noqa: E731
    scaled, plain = PartSpec("rope_scaled", {"head_dim": 16, "theta": 100.0}), PartSpec("rope_halves", {"head_dim": 16, "theta": 100.0})
    make(scaled, whole_prompts=True, qk_norm_eps=1e-5)
    make(PartSpec("none"), whole_prompts=True)
    for position, how in ((plain, {"whole_prompts": True}), (scaled, {"whole_prompts": True, "window": 8}), (scaled, {"whole_prompts": True, "softcap": 2.0}),
                          (scaled, {"qk_bias": True}), (scaled, {"values_are_keys": True}), (scaled, {"all_bias": True}), (scaled, {"v_dim": 8}),
                          (scaled, {"whole_prompts": True, "own_kv": False}), (PartSpec("none"), {"whole_prompts": True, "qk_norm_eps": 1e-5}),
                          (scaled, {"whole_prompts": True, "penalty": ("a", "b")}), (scaled, {"whole_prompts": True, "chunk": 8})):
        with pytest.raises(ValueError):
            make(position, **how)
    for how in ({"rot_dim": 15}, {"rot_dim": 18}, {"scaling": {"factor": -1.0, "original": 8, "fast": 2.0, "slow": 1.0}}):
        with pytest.raises(ValueError):
            build_part("position", PartSpec("rope_scaled", {"head_dim": 16, "theta": 100.0, **how}), torch.float32, torch.device("cpu"))


@pytest.mark.parametrize("scaling", [None, YARN, WAVES])
def test_frequencies_and_multiplier(scaling):
    from edgerag_b200.ops import kernels
    from edgerag_b200.parts.base import build_part
    from edgerag_b200.parts.rope import rotary_frequencies, rotary_multiplier

    part = build_part("position", spec(head_dim=64, rot_dim=32, scaling=scaling), torch.float32, torch.device("cpu"))
    assert torch.equal(part.turns, kernels.rotary_turns(rotary_frequencies(1000.0, 32, scaling))) and part.multiplier == rotary_multiplier(scaling)
