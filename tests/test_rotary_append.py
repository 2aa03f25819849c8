"""Head norms, rotary positions scaled for long contexts and the append to the cache in one pass, against the formulas in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from edgerag_b200.ops import kernels as K

ELEM = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def formula(x, heads, dim, positions, freq, m, pairs, norm, eps):
    """Rows of heads in 64 bits: normed, the first 2 len(freq) entries turned; and the size of the terms of each entry."""
    x = x.double().reshape(-1, heads, dim)
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * norm.double()
    out, size, half = x.clone(), x.abs(), len(freq)
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if pairs else (i, i + half)
        angle = positions.double() * float(freq[i])
        c, s = m * torch.cos(angle)[:, None], m * torch.sin(angle)[:, None]
        out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        size[..., a] = size[..., b] = m * (x[..., a].abs() + x[..., b].abs())
    return out.flatten(1), size.flatten(1)


def near(got, want, size, dim, what):
    """One rounding at the store, and float arithmetic before it: the sum of squares (dim + 8 roundings, halved by the root), the norm's two
    products, cosine and sine within 2^-21 of the multiplier (an angle within 2^-24 of an eighth turn, the function's and the
    multiplier's roundings), two products and a sum."""
    bound = want.abs() * torch.finfo(got.dtype).eps / 2 + size * ((dim + 8) / 2 + 8 + 8) * 2.0**-24
    off = (got.double().cpu() - want).abs() - bound * 1.0001
    assert off.max() <= 0, f"{what}: {off.max():.3g} over the bound"


CASES = [
    # tokens, query heads, kv heads, head size, turned entries, pairs, multiplier, norm, first position, page size (0: no cache), pad of the rows
    (1, 4, 2, 64, 64, False, 1.0, False, 0, 16, 0),
    (7, 9, 3, 64, 32, True, 1.3, True, 1048570, 8, 0),
    (33, 32, 8, 128, 128, False, 1.2772588722239781, True, 2147480000, 16, 0),
    (5, 2, 1, 80, 20, True, 1.0, False, 1000, 16, 3),
    (6, 3, 3, 12, 6, False, 0.5, True, 77, 5, 1),
    (130, 16, 2, 128, 64, True, 1.0, False, 500000, 32, 8),
    (40, 5, 5, 256, 64, False, 1.0, True, 31, 0, 0),
    (64, 15, 5, 64, 0, False, 1.0, True, 9, 16, 0),
    (3, 1, 1, 1, 0, False, 1.0, False, 0, 0, 0),
    (9, 4, 1, 96, 96, True, 2.0, False, 123456, 0, 5),
    (300, 8, 8, 64, 16, False, 1.0, False, 4000, 64, 0),
    (2, 2, 2, 1024, 1024, False, 1.0, True, 5, 4, 0),
    (470, 32, 8, 128, 128, False, 1.0, True, 5, 16, 0),
    (460, 6, 2, 64, 32, True, 1.2, True, 90000, 8, 8),
    (500, 64, 8, 128, 64, False, 1.0, True, 3, 32, 0),
    (2500, 20, 6, 128, 32, False, 1.1, False, 0, 16, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("elem", ["float32", "bfloat16"])
@pytest.mark.parametrize("tokens,nq,nkv,dim,rot,pairs,m,norm,first,page,pad", CASES)
def test_rows_are_the_formula(elem, tokens, nq, nkv, dim, rot, pairs, m, norm, first, page, pad):
    g, t = torch.Generator().manual_seed(tokens + dim), ELEM[elem]
    rows = torch.randn(tokens, (nq + 2 * nkv) * dim + pad, generator=g).to(t).cuda()
    q, k, v = rows[:, : nq * dim], rows[:, nq * dim: (nq + nkv) * dim], rows[:, (nq + nkv) * dim: (nq + 2 * nkv) * dim]
    before = rows.cpu()
    freq = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) / max(rot // 2, 1))
    positions = (first + torch.arange(tokens)).to(torch.int32)
    wq, wk = (1 + 0.2 * torch.randn(dim, generator=g), 1 + 0.2 * torch.randn(dim, generator=g)) if norm else (None, None)
    how = {"q_norm": wq.cuda(), "k_norm": wk.cuda(), "eps": 1e-5} if norm else {}
    turns = K.rotary_turns(freq).cuda() if rot else None
    if page:
        n_pages = -(-tokens // page) + 3
        pools = torch.full((2, n_pages, nkv, page, dim), -7.0, dtype=t).cuda()
        slots = torch.randperm(n_pages * page, generator=g)[:tokens].to(torch.int32)
        slots[tokens // 2] = -1 if tokens > 1 else slots[0]
        status = torch.zeros(1, dtype=torch.int32).cuda()
        how |= {"v": v, "slots": slots.cuda(), "k_pages": pools[0], "v_pages": pools[1], "status": status}
    K.rotary_append(q, positions.cuda(), turns, nq, nkv, dim, k=k, pairs=pairs, multiplier=m, **how)
    want_q, size_q = formula(before[:, : nq * dim], nq, dim, positions, freq, m, pairs, wq, 1e-5)
    want_k, size_k = formula(before[:, nq * dim: (nq + nkv) * dim], nkv, dim, positions, freq, m, pairs, wk, 1e-5)
    near(q.cpu(), want_q, size_q, dim, "q")
    after = rows.cpu()
    assert torch.equal(after[:, (nq + nkv) * dim:], before[:, (nq + nkv) * dim:])               # values and what lies behind the rows
    if not page:
        near(k.cpu(), want_k, size_k, dim, "k")
        return
    assert torch.equal(after[:, nq * dim: (nq + nkv) * dim], before[:, nq * dim: (nq + nkv) * dim]) and int(status) == 0
    flat_k, flat_v = (p.cpu().transpose(1, 2).reshape(n_pages * page, nkv * dim) for p in pools)
    here = slots >= 0
    near(flat_k[slots[here].long()], want_k[here], size_k[here], dim, "cached k")
    assert torch.equal(flat_v[slots[here].long()], before[here][:, (nq + nkv) * dim: (nq + 2 * nkv) * dim])
    untouched = torch.ones(n_pages * page, dtype=torch.bool)
    untouched[slots[here].long()] = False
    assert (flat_k[untouched] == -7).all() and (flat_v[untouched] == -7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,pairs", [(64, False), (128, True), (24, False)])
def test_other_rows_than_the_inputs(dim, pairs):
    """Results into rows of their own, and a slot behind the pool that is reported and left alone."""
    g = torch.Generator().manual_seed(dim)
    q, k, v = (torch.randn(6, h * dim, generator=g).bfloat16().cuda() for h in (4, 2, 2))
    q_out, k_out = torch.zeros(6, 8 * dim).bfloat16().cuda()[:, : 4 * dim], torch.zeros(6, 2 * dim).bfloat16().cuda()
    kept = q.cpu(), k.cpu()
    freq = 100.0 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))
    positions, status = torch.arange(6, dtype=torch.int32), torch.zeros(1, dtype=torch.int32).cuda()
    pools = torch.zeros(2, 2, 2, 8, dim).bfloat16().cuda()
    slots = torch.tensor([0, 3, 16, 9, -1, 15], dtype=torch.int32).cuda()
    K.rotary_append(q, positions.cuda(), K.rotary_turns(freq).cuda(), 4, 2, dim, k=k, v=v, pairs=pairs, q_out=q_out, k_out=k_out, slots=slots,
                    k_pages=pools[0], v_pages=pools[1], status=status)
    assert torch.equal(q.cpu(), kept[0]) and torch.equal(k.cpu(), kept[1])
    near(q_out.cpu(), *formula(kept[0], 4, dim, positions, freq, 1.0, pairs, None, 0.0), dim, "q")
    near(k_out.cpu(), *formula(kept[1], 2, dim, positions, freq, 1.0, pairs, None, 0.0), dim, "k")
    assert int(status) == 3                                                     # token 2
    cached = pools[0].cpu().transpose(1, 2).reshape(16, -1)
    assert torch.equal(cached[[0, 3, 9, 15]], k_out.cpu()[[0, 1, 3, 5]]) and int((cached != 0).any(1).sum()) == 4


@pytest.mark.gpu
def test_queries_alone_no_tokens_and_captured():
    q = torch.randn(5, 128).cuda()
    turns, positions = K.rotary_turns(torch.tensor([1.0, 0.1], dtype=torch.float64)).cuda(), torch.arange(5, dtype=torch.int32).cuda()
    out = torch.empty_like(q)
    K.rotary_append(q[:0], positions[:0], turns, 2, 0, 64)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            K.rotary_append(q, positions, turns, 2, 0, 64, q_out=out)
        q.copy_(torch.randn(5, 128))
        positions.add_(70000)
        graph.replay()
    torch.cuda.synchronize()
    near(out.cpu(), *formula(q.cpu(), 2, 64, positions.cpu(), [1.0, 0.1], 1.0, False, None, 0.0), 64, "replayed")


def test_turns_are_the_frequencies():
    """The fixed-point product with a position, modulo a turn, is the angle (a product of doubles loses 5e-10 radians of it at 2e9 * 0.001)."""
    freq = torch.tensor([1.0, 0.5, 1e-3, 0.0, -2.5, 7.0], dtype=torch.float64)
    turns = K.rotary_turns(freq)
    for f, u in zip(freq.tolist(), turns.tolist()):
        for p in (1, 77, 10**6, 2**31 - 1):
            got = (p * u) % 2**64 / 2.0**64 * 2 * math.pi
            assert abs(math.cos(got) - math.cos(p * f)) + abs(math.sin(got) - math.sin(p * f)) < 1e-8
    with pytest.raises(K.KernelError, match="finite"):
        K.rotary_turns(torch.tensor([math.inf]))


GOOD = dict(q=torch.zeros(4, 128), positions=torch.zeros(4, dtype=torch.int32), turns=torch.zeros(16, dtype=torch.int64), n_q_heads=2, n_kv_heads=1,
            head_dim=64)
KV = dict(k=torch.zeros(4, 64), v=torch.zeros(4, 64), slots=torch.zeros(4, dtype=torch.int32), k_pages=torch.zeros(3, 1, 8, 64),
          v_pages=torch.zeros(3, 1, 8, 64), status=torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("change,word", [
    (dict(q=torch.zeros(4, 128, dtype=torch.float16)), "float32 or bfloat16"),
    (dict(q=torch.zeros(4, 127)), "q must be"),
    (dict(q=torch.zeros(128, 4).t()), "contiguous"),
    (dict(q=torch.zeros(1, 128).expand(4, 128)), "overlap"),
    (dict(head_dim=2048), "at most 1024"),
    (dict(turns=torch.zeros(40, dtype=torch.int64)), "pairs do not fit"),
    (dict(turns=torch.zeros(16)), "turns must be"),
    (dict(positions=torch.zeros(3, dtype=torch.int32)), "positions must be"),
    (dict(positions=torch.zeros(4, dtype=torch.int64)), "positions must be"),
    (dict(q_norm=torch.zeros(63)), "q_norm must be"),
    (dict(k_norm=torch.zeros(64)), "need keys"),
    (dict(v=torch.zeros(4, 64)), "need keys"),
    (dict(q_out=torch.zeros(4, 64)), "q_out must be"),
    (dict(KV, v=None), "come together"),
    (dict(KV, k_pages=None, v_pages=None), "come together"),
    (dict(KV, k=torch.zeros(4, 128)), "k must be"),
    (dict(KV, k_pages=torch.zeros(3, 1, 16, 64)), "one shape"),
    (dict(KV, k_pages=torch.zeros(3, 2, 8, 64), v_pages=torch.zeros(3, 2, 8, 64)), "page layout"),
    (dict(KV, k_pages=torch.zeros(3, 1, 64, 8).transpose(2, 3), v_pages=torch.zeros(3, 1, 64, 8).transpose(2, 3)), "page layout"),
    (dict(KV, k_pages=torch.zeros(0, 1, 8, 64), v_pages=torch.zeros(0, 1, 8, 64)), "no page"),
    (dict(KV, slots=torch.zeros(3, dtype=torch.int32)), "slots must be"),
    (dict(KV, status=None), "status must be"),
    (dict(KV, k_out=torch.zeros(3, 64)), "k_out must be"),
    (dict(), "CUDA device"),
    (dict(KV), "CUDA device"),
])
def test_refusals(change, word):
    with pytest.raises(K.KernelError, match=word):
        K.rotary_append(**{**GOOD, **change})
