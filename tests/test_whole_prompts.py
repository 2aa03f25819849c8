"""When the attention part may take prompts from a step's rows instead of the cache, and when it may not."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from edgerag_b200.ops import kernels
from edgerag_b200.parts import attention, rope
from edgerag_b200.parts.base import LayerCall, LayerSpec, ModelPlan, PartSpec
from test_rope_scaled import H, NKV, NQ, SEQUENCES, VOCAB, YARN, walk

POSITIONS = {"scaled": PartSpec("rope_scaled", {"head_dim": 64, "theta": 1000.0, "scaling": YARN}), "none": PartSpec("none")}


class Recorder:
    """Stands in for the module of kernels: launches are recorded in their order, everything else is the module's own."""

    LAUNCHES = ("linear", "rotary_append", "rope_cache_write", "attention_prompt", "attention_prefill_tc", "attention_rows")

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if name == "linear_parts_count":
            return lambda *a: 0
        if name in self.LAUNCHES:
            return lambda *a, **k: self.calls.append((name, a, k))
        return getattr(kernels, name)


def launches(monkeypatch, position, call, dtype=torch.float32, batch_invariant=False, whole_portions=True, n=40):
    """What the part launches for one prompt of `n` tokens (CPU: nothing runs)."""
    seen, cpu = Recorder(), torch.device("cpu")
    monkeypatch.setattr(attention, "kernels", seen)
    monkeypatch.setattr(rope, "kernels", seen)
    monkeypatch.setattr(kernels, "_sms", lambda device: 148)
    part = attention.Attention(H, NQ, NKV, 64, position, dtype, cpu, whole_prompts=True)
    part.w_o = torch.zeros(H, NQ * 64, dtype=dtype)
    pool = torch.zeros(4, NKV, 16, 64, dtype=dtype)
    ints = torch.zeros(n + 1, dtype=torch.int32)
    ctx = SimpleNamespace(batch_invariant=batch_invariant, whole_portions=whole_portions, host_q_len=[n], host_positions_last=[n - 1], n_seqs=1, n_decode=0, n_tokens=n,
                          page_size=16, slots=[ints[:n]], block_tables=[torch.zeros(1, 4, dtype=torch.int32)], seq_starts=torch.tensor([0, n], dtype=torch.int32),
                          seq_of_token=ints[:n], positions=ints[:n], status=ints[:1], max_keys_bound=lambda: 64, pages_of=lambda layer: (pool, pool),
                          group_of=lambda layer: 0, buf=lambda name, shape, kind: torch.zeros(shape, dtype=kind))
    part.forward(torch.zeros(n, H, dtype=dtype), ctx, call)
    return seen.calls


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("position", POSITIONS)
def test_a_call_that_reads_anothers_cache_takes_its_keys_from_there(position, dtype, monkeypatch):
    """Such a call turns and writes no keys: those of its rows are none that any token may see."""
    names = [c[0] for c in launches(monkeypatch, POSITIONS[position], LayerCall(0, 0, writes_cache=False), dtype)]
    assert "attention_prompt" not in names and ("attention_rows" in names or "attention_prefill_tc" in names)
    assert "attention_prompt" in [c[0] for c in launches(monkeypatch, POSITIONS[position], LayerCall(0, 0), dtype)]


def build(dtype, position, whole_prompts, schedule, batch_invariant=False):
    from edgerag_b200.cache.device import DevicePools
    from edgerag_b200.cache.manager import CacheManager
    from edgerag_b200.engine.step import ModelRunner
    from edgerag_b200.models.decoder import DecoderModel

    norm = lambda p: PartSpec("rmsnorm", {"size": H, "eps": 1e-5}, p)   # noqa: E731
    how = {"hidden": H, "n_q_heads": NQ, "n_kv_heads": NKV, "head_dim": 64, "position": position, "whole_prompts": whole_prompts}
    specs = [LayerSpec(f"layers.{i}.", PartSpec("prenorm"), norm("ln1."), PartSpec("attention", how, "self_attn."), norm("ln2."),
                       PartSpec("swiglu", {"hidden": H, "intermediate": 64}, "mlp.")) for i in range(2)]
    plan = ModelPlan(H, VOCAB, PartSpec("table", {"vocab": VOCAB, "hidden": H}, "embed."), specs, schedule, norm("norm."),
                     PartSpec("linear", {"vocab": VOCAB, "hidden": H, "tied_to": None}, "lm_head."))
    device, g = torch.device("cuda"), torch.Generator().manual_seed(7)
    model = DecoderModel(plan, dtype, device)
    model.load_weights({s.name: 1 + 0.1 * torch.randn(s.shape, generator=g) if "norm" in s.name or "ln" in s.name else 0.15 * torch.randn(s.shape, generator=g)
                        for s in model.weight_specs()})
    cache = CacheManager(model.cache_layout, 16, 64, 8)
    pools = DevicePools(model.cache_layout, 16, [64], 8, dtype, device)
    return ModelRunner(model, cache, pools, 512, check_status=True, batch_invariant=batch_invariant)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("position", POSITIONS)
def test_a_layer_called_twice_reads_its_own_cache(position, dtype):
    """The second time without writing: with and without the option the logits agree, as far as the bounds of the same prompts in test_rope_scaled.py go."""
    schedule = [LayerCall(0, 0), LayerCall(0, 0, writes_cache=False), LayerCall(1, 1)]
    cached, rows = (build(dtype, POSITIONS[position], whole, schedule) for whole in (False, True))
    for portions in ([[70], [33], [5]], [[40, 30], [1] * 33, [5]]):
        for a, b in zip(walk(cached, SEQUENCES, portions), walk(rows, SEQUENCES, portions)):
            assert (a - b).abs().max() <= (2e-4 + 2e-4 * a.abs().max() if dtype == torch.float32 else 0.02 * a.abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("position", POSITIONS)
def test_pinned_launch_shapes_do_not_look_at_other_requests(position, dtype, monkeypatch):
    """`batch_invariant`: whether another request's portion has a past does not change the kernel that takes a prompt."""
    seen = [[c[0] for c in launches(monkeypatch, POSITIONS[position], LayerCall(0, 0), dtype, True, whole)] for whole in (True, False)]
    assert seen[0] == seen[1] and "attention_prompt" not in seen[0]


@pytest.mark.gpu
@pytest.mark.parametrize("position", POSITIONS)
def test_a_prompt_has_its_bits_whatever_shares_its_step(position):
    """32-bit portions under `batch_invariant`: beside another prompt, and beside as many tokens of another one's second portion (the products
    of the two steps have the same shapes)."""
    from edgerag_b200.engine.step import StepEntry

    runner = build(torch.float32, POSITIONS[position], True, [LayerCall(0, 0), LayerCall(1, 1)], batch_invariant=True)
    prompt, other, got = SEQUENCES[0], SEQUENCES[1], []
    for parts in ((other[:20],), (other[:13], other[13:])):
        for name in ("a", "b"):
            runner.admit(name)
        for part in parts[:-1]:
            runner.step([StepEntry("b", tokens=list(part), want=[0])])
        step = [StepEntry("a", tokens=list(prompt), want=list(range(len(prompt)))), StepEntry("b", tokens=list(parts[-1]), want=[0])]
        got.append(runner.step(step)[: len(prompt)].float().cpu().clone())
        for name in ("a", "b"):
            runner.release(name)
    assert torch.equal(got[0], got[1])


@pytest.mark.parametrize("how,word", [({"head_dim": 272}, "256"), ({"scale": 0.0}, "scale"), ({"scale": -0.125}, "scale"), ({"scale": float("nan")}, "scale")])
def test_what_the_first_prompt_would_refuse_is_refused_at_once(how, word):
    """Head sizes and scales that attention over rows does not take."""
    make = lambda **more: attention.Attention(**{"hidden": 64, "n_q_heads": 4, "n_kv_heads": 2, "head_dim": 64, "position": PartSpec("none"),   # noqa: E731
                                                 "dtype": torch.float32, "device": torch.device("cpu"), **how, **more})
    make()
    with pytest.raises(ValueError, match=word):
        make(whole_prompts=True)
