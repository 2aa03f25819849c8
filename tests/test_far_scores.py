"""Scores whose scaled value a float rounds by more than a power of two of weight: the highest one still has the weight, none becomes infinite or is lost."""

from __future__ import annotations

import pytest
import torch

from edgerag_b200.ops import kernels as K
from test_packed_attention import prompt_call, run_prompt, run_shared, shared_call

KINDS = [("bfloat16", 64), ("bfloat16", 128), ("float32", 64), ("bfloat16", 40)]


def alone(q, k, v, scale, limits):
    """Rows whose highest score leads the next by 2^-10 of itself or more (64 roundings and more of a float's sums of up to 128 products of bfloat16
    entries, and at these sizes more than 128 in the exponent): the definition is the value of that key alone.  Which rows, and what they get.  A result
    is off by half a step, and by half of one more where the highest score is small and its weight is a power of two that bfloat16 rounds."""
    z = q.double() @ k.double().T * scale
    z[torch.arange(k.shape[0])[None, :] >= limits[:, None]] = -float("inf")
    top, where = z.topk(min(2, z.shape[1]), 1)
    clear = limits > 0
    if z.shape[1] > 1:
        clear &= (limits == 1) | (top[:, 0] - top[:, 1] >= 2.0**-10 * (q.double().abs() @ k.double().abs().T).amax(1) * scale)
    return clear, v[where[:, 0]].double()


def check(got, want, clear, what):
    assert torch.isfinite(got).all(), what
    assert clear.float().mean() > 0.5 and ((got.double() - want).abs() <= want.abs() * torch.finfo(got.dtype).eps * 1.0001)[clear].all(), what


@pytest.mark.gpu
@pytest.mark.parametrize("elem,dim", KINDS)
@pytest.mark.parametrize("power", [30, 36, 60, 100])
def test_prompts_of_far_scores(elem, dim, power):
    rows, starts, scale = prompt_call(elem, (300,), 4, 2, dim, seed=2)
    rows[:, : 6 * dim] = (rows[:, : 6 * dim].float() * 2.0 ** (power / 2)).to(rows.dtype)
    out, status = run_prompt(rows, starts, 4, 2, dim, scale)
    assert status == 0
    for h in range(4):
        g = h // 2
        q, k, v = (rows[:, i * dim: (i + 1) * dim] for i in (h, 4 + g, 6 + g))
        clear, want = alone(q, k, v, scale, torch.arange(1, 301))
        check(out[:, h * dim: (h + 1) * dim], want, clear, f"2^{power}, head {h}")


@pytest.mark.gpu
@pytest.mark.parametrize("elem,dim", KINDS)
@pytest.mark.parametrize("power", [30, 36, 60, 100])
@pytest.mark.parametrize("own", [K.OWN_MANY, K.OWN_TOKEN, K.OWN_ROWS])
def test_far_scores_behind_a_prefix(elem, dim, power, own):
    c = shared_call(elem, 200, (1, 3, 20), (90, 5, 60), 4, 2, dim, 16)
    c["q"], c["k"] = ((c[x].float() * 2.0 ** (power / 2)).to(c[x].dtype) for x in "qk")
    out, status = run_shared(c, K.SharedPrefixPlan(2, 2, 64, 24 * 4 * 4 * (dim + 2), K.packed_tc_supported(c["q"].dtype, dim, 2), own))
    assert status == 0
    for s, (a, b) in enumerate(zip(c["starts"][:-1].tolist(), c["starts"][1:].tolist())):
        limits = c["positions"][a:b].long() + 1
        at = torch.arange(int(limits.max()))
        pages = torch.cat((c["prefix_pages"][:13], c["tables"][s, 12:])).long()
        index = torch.where(at < 200, at // 16, at // 16 - 12 + 13)
        for h in range(4):
            k, v = (c[x][pages[index], h // 2, at % 16] for x in "kv")
            clear, want = alone(c["q"][a:b, h * dim: (h + 1) * dim], k, v, c["scale"], limits)
            assert torch.isfinite(out[a:b]).all()
            got = out[a:b, h * dim: (h + 1) * dim].double()
            assert ((got - want).abs() <= want.abs() * torch.finfo(c["q"].dtype).eps * 1.0001)[clear].all(), f"2^{power}, request {s}, head {h}"
