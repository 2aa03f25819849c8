"""Attention over packed whole prompts, and of batches behind a shared prefix, against the definition in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from edgerag_b200.ops import kernels as K

ELEM = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def define(q, k, v, scale, limits):
    """One head in 64 bits: rows over the keys below their limits; with it sum p |v| and the largest sum |q k| scale of each row."""
    q, k, v = q.double(), k.double(), v.double()
    out, weight, spread = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[0], 1, dtype=torch.float64)
    for r, n in enumerate(limits):
        if n <= 0:
            continue
        z = k[:n] @ q[r] * scale
        p = torch.softmax(z, 0)
        out[r], weight[r], spread[r] = p @ v[:n], p @ v[:n].abs(), float((k[:n].abs() @ q[r].abs()).max()) * scale
    return out, weight, spread


def near(got, want, weight, spread, dim, keys, what):
    """The bound: half a step of the stored result; half a step of its type for every weight before it meets its value (the weights and the
    values of the float kernels are floats); scores within (dim + 4) roundings of their terms, each an absolute error of an exponent, so
    a relative one of its weight; sums over `keys` weights in float, their exponentials (2^-21) and the joining of pieces."""
    half = torch.finfo(got.dtype).eps / 2
    bound = want.abs() * half + weight * (half + (2 * (dim + 4) * spread + 2 * keys + 64) * 2.0**-24)
    off = (got.double().cpu() - want).abs() - bound * 1.0001
    assert torch.isfinite(got).all(), what
    assert off.max() <= 0, f"{what}: {off.max():.3g} over the bound"


def prompt_call(elem, lengths, nq, nkv, dim, pad=0, behind=0, seed=0, scale=None, size=1.0):
    g, t = torch.Generator().manual_seed(seed + dim + sum(lengths)), ELEM[elem]
    n = sum(lengths)
    rows = (torch.randn(n + behind, (nq + 2 * nkv) * dim + pad, generator=g) * size).to(t)
    starts = torch.tensor([0, *lengths]).cumsum(0).to(torch.int32)
    return rows, starts, dim**-0.5 if scale is None else scale


def run_prompt(rows, starts, nq, nkv, dim, scale):
    dev = rows.cuda()
    out = torch.full((rows.shape[0], nq * dim), -7.0, dtype=rows.dtype).cuda()
    status = torch.zeros(1, dtype=torch.int32).cuda()
    K.attention_prompt(dev[:, : nq * dim], dev[:, nq * dim: (nq + nkv) * dim], dev[:, (nq + nkv) * dim: (nq + 2 * nkv) * dim], starts.cuda(), out, nq, nkv, scale, status)
    return out.cpu(), int(status)


def check_prompt(rows, starts, nq, nkv, dim, scale, out, sequences=None, some=None):
    for s, (a, b) in enumerate(zip(starts[:-1].tolist(), starts[1:].tolist())):
        if sequences is not None and s not in sequences or a == b:
            continue
        at = list(range(b - a)) if some is None else sorted({min(b - a - 1, x) for x in some})
        for h in range(nq):
            g = h // (nq // nkv)
            k, v = rows[a:b, (nq + g) * dim: (nq + g + 1) * dim], rows[a:b, (nq + nkv + g) * dim: (nq + nkv + g + 1) * dim]
            rel = [a + x for x in at]
            near(out[rel][:, h * dim: (h + 1) * dim], *define(rows[rel][:, h * dim: (h + 1) * dim], k, v, scale, [x + 1 for x in at]), dim, b - a, f"sequence {s}, head {h}")


PROMPTS = [
    # lengths, query heads, kv heads, head size, pad of the rows
    ((1,), 2, 2, 64, 0),
    ((0, 3, 0, 1, 17, 0), 4, 2, 64, 8),
    ((64, 65, 63, 128, 127, 129), 4, 1, 64, 0),
    ((300, 1, 2, 513), 6, 2, 128, 0),
    ((257,), 9, 3, 64, 0),
    ((31, 200), 8, 1, 128, 16),
    ((40, 130), 2, 1, 80, 0),
    ((70, 5), 3, 3, 12, 1),
    ((90,), 2, 2, 256, 0),
    ((33, 66), 2, 1, 96, 3),
    ((400,), 32, 1, 64, 0),
    (tuple([1] * 70 + [20] * 5), 3, 1, 128, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("elem", ["float32", "bfloat16"])
@pytest.mark.parametrize("lengths,nq,nkv,dim,pad", PROMPTS)
def test_prompts(elem, lengths, nq, nkv, dim, pad):
    rows, starts, scale = prompt_call(elem, lengths, nq, nkv, dim, pad, behind=5)
    rows[sum(lengths):] = float("nan")                                    # rows behind the last sequence
    out, status = run_prompt(rows, starts, nq, nkv, dim, scale)
    assert status == 0 and (out[sum(lengths):] == -7).all()
    check_prompt(rows, starts, nq, nkv, dim, scale, out)


@pytest.mark.gpu
@pytest.mark.parametrize("elem,dim,size", [("bfloat16", 64, 1.0), ("bfloat16", 128, 1.0), ("bfloat16", 128, 4.0), ("bfloat16", 64, 4.0), ("float32", 64, 2.0)])
def test_long_prompts(elem, dim, size):
    """Many tiles of keys; with large scores a row's maximum moves far along its keys."""
    rows, starts, scale = prompt_call(elem, (2100, 700), 4, 2, dim, size=size)
    out, status = run_prompt(rows, starts, 4, 2, dim, scale)
    assert status == 0
    check_prompt(rows, starts, 4, 2, dim, scale, out, some=(0, 63, 127, 128, 500, 699, 1023, 1500, 2047, 2048, 2099))


@pytest.mark.gpu
@pytest.mark.parametrize("elem,dim", [("bfloat16", 64), ("bfloat16", 128), ("float32", 64), ("bfloat16", 40)])
def test_scores_that_rise_and_fall(elem, dim):
    """Keys whose scores climb by hundreds along the sequence, and others that fall: no weight may overflow or vanish wrongly."""
    rows, starts, scale = prompt_call(elem, (600, 600), 2, 1, dim, scale=1.0)
    rows[:, : 2 * dim] = 1.0
    climb = torch.linspace(-300, 300, 600)[:, None] / dim
    rows[:600, 2 * dim: 3 * dim] = climb.expand(-1, dim).to(rows.dtype)
    rows[600:, 2 * dim: 3 * dim] = -climb.expand(-1, dim).to(rows.dtype)
    out, status = run_prompt(rows, starts, 2, 1, dim, 1.0)
    assert status == 0
    check_prompt(rows, starts, 2, 1, dim, 1.0, out, some=(0, 1, 100, 127, 128, 129, 300, 511, 512, 599))


@pytest.mark.gpu
@pytest.mark.parametrize("elem,dim", [("bfloat16", 64), ("bfloat16", 128), ("float32", 64), ("bfloat16", 24)])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_what_later_tokens_hold_stays_unseen(elem, dim, what):
    """A key or value that is no number reaches the rows that see it, and no other."""
    rows, starts, scale = prompt_call(elem, (150, 90), 4, 2, dim)
    clean = run_prompt(rows, starts, 4, 2, dim, scale)[0]
    for col, at in ((4 * dim + 3, 100), (6 * dim + 5, 133), (7 * dim + 2, 150 + 17)):     # a key, a value of head 0; a value of head 1
        rows[at, col] = what
    out, status = run_prompt(rows, starts, 4, 2, dim, scale)
    assert status == 0
    same = torch.ones(240, 4 * dim, dtype=torch.bool)
    same[100:150, : 2 * dim] = False
    same[133:150, 5] = same[133:150, dim + 5] = False
    same[150 + 17:, 2 * dim + 2] = same[150 + 17:, 3 * dim + 2] = False
    assert torch.equal(out[same], clean[same])
    assert not torch.isfinite(out[133:150][:, [5, dim + 5]]).any() and not torch.isfinite(out[150 + 17:][:, [2 * dim + 2, 3 * dim + 2]]).any()
    if math.isnan(what):
        assert torch.isnan(out[100:150, : 2 * dim]).all()


@pytest.mark.gpu
def test_prompt_starts_outside_the_rows_are_reported():
    rows, _, scale = prompt_call("bfloat16", (40,), 2, 1, 64)
    out, status = run_prompt(rows, torch.tensor([0, 10, 900], dtype=torch.int32), 2, 1, 64, scale)
    assert status == 9000002 and (out[10:] == -7).all()
    check_prompt(rows, torch.tensor([0, 10]), 2, 1, 64, scale, out)


def shared_call(elem, prefix, fresh, past, nq, nkv, dim, page, seed=0, pad=0, behind=0, sms=148, scale=None):
    """`past[s]` own keys of request s before its `fresh[s]` rows."""
    g, t = torch.Generator().manual_seed(seed + prefix + dim + sum(fresh)), ELEM[elem]
    n, own = sum(fresh), [a + b for a, b in zip(past, fresh)]
    per = -(-(prefix + max(own)) // page)
    shared, mine = -(-prefix // page), per - prefix // page
    pages = shared + mine * len(fresh) + 2
    order = torch.randperm(pages, generator=g).to(torch.int32)
    pools = torch.randn(2, pages, nkv, page, dim, generator=g).to(t)
    tables = torch.full((len(fresh), per), -5, dtype=torch.int32)               # entries of the prefix's pages are not read
    tables[:, prefix // page:] = order[shared: shared + mine * len(fresh)].view(len(fresh), mine)
    return {"q": torch.randn(n + behind, nq * dim + pad, generator=g).to(t), "k": pools[0], "v": pools[1], "prefix_pages": order[:shared], "prefix": prefix,
            "tables": tables, "starts": torch.tensor([0, *fresh]).cumsum(0).to(torch.int32),
            "positions": torch.cat([torch.arange(prefix + a, prefix + a + b) for a, b in zip(past, fresh)] + [torch.zeros(behind)]).to(torch.int32),
            "nq": nq, "scale": dim**-0.5 if scale is None else scale, "dim": dim, "sms": sms, "max_keys": prefix + max(own), "max_tokens": max(fresh)}


def run_shared(c, plan=None, stream=None):
    nkv, page, dim = c["k"].shape[1:]
    n, width = c["q"].shape[0], c["nq"] * dim
    plan = plan or K.shared_prefix_plan(n, c["tables"].shape[0], c["nq"], nkv, dim, c["q"].dtype, page, c["prefix"], c["max_keys"], c["max_tokens"], sms=c["sms"])
    out, status = torch.full((n, width), -7.0, dtype=c["q"].dtype).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    scratch = torch.full((max(plan.floats, 1),), float("nan")).cuda()
    K.attention_shared_prefix(c["q"].cuda()[:, :width], c["k"].cuda(), c["v"].cuda(), c["prefix_pages"].cuda(), c["prefix"], c["tables"].cuda(),
                              c["starts"].cuda(), c["positions"].cuda(), out, c["nq"], c["scale"], plan, scratch, status)
    return out.cpu(), int(status)


def check_shared(c, out, requests=None, rows_of=None):
    nkv, page, dim = c["k"].shape[1:]
    group, prefix = c["nq"] // nkv, c["prefix"]
    for s, (a, b) in enumerate(zip(c["starts"][:-1].tolist(), c["starts"][1:].tolist())):
        if a == b or requests is not None and s not in requests:
            continue
        limits = (c["positions"][a:b] + 1).tolist()
        at = torch.arange(max(max(limits), 0))
        pages = torch.cat((c["prefix_pages"][: -(-prefix // page)], c["tables"][s, prefix // page:])).long()
        index = torch.where(at < prefix, at // page, at // page - prefix // page + -(-prefix // page))
        for h in range(c["nq"]):
            k, v = (c[x][pages[index], h // group, at % page] for x in "kv")
            near(out[a:b, h * dim: (h + 1) * dim], *define(c["q"][a:b, h * dim: (h + 1) * dim], k, v, c["scale"], limits), dim, len(at), f"request {s}, head {h}")


SHARED = [
    # prefix, rows and earlier own keys of each request, query heads, kv heads, head size, page size
    (1, (1,), (0,), 2, 2, 64, 16),
    (64, (1, 1, 1), (0, 5, 200), 4, 2, 64, 16),
    (300, (1,) * 9, (0, 1, 2, 15, 16, 17, 127, 128, 400), 9, 3, 64, 16),
    (129, (1, 1), (3, 77), 8, 1, 128, 32),
    (1000, (1,) * 40, tuple(range(0, 400, 10)), 4, 2, 128, 64),
    (257, (3, 0, 40, 1, 0), (0, 0, 100, 30, 9), 6, 2, 64, 8),
    (500, (200, 1, 7), (20, 300, 1), 4, 4, 64, 16),
    (90, (5, 130), (60, 0), 4, 1, 128, 16),
    (0, (1, 1, 4), (0, 70, 3), 4, 2, 64, 16),
    (0, (150, 1), (0, 333), 4, 2, 128, 16),
    (77, (1, 2), (10, 40), 4, 2, 80, 12),
    (50, (1, 6), (4, 0), 3, 3, 12, 5),
    (333, (1, 1), (40, 9), 2, 1, 256, 16),
    (160, (1, 2, 1), (9, 0, 400), 32, 1, 64, 128),
    (700, (1, 1), (300, 20), 2, 1, 64, 256),
]


@pytest.mark.gpu
@pytest.mark.parametrize("elem", ["float32", "bfloat16"])
@pytest.mark.parametrize("prefix,fresh,past,nq,nkv,dim,page", SHARED)
def test_behind_a_prefix(elem, prefix, fresh, past, nq, nkv, dim, page):
    c = shared_call(elem, prefix, fresh, past, nq, nkv, dim, page, pad=8, behind=3)
    out, status = run_shared(c)
    assert status == 0 and (out[sum(fresh):] == -7).all()
    check_shared(c, out)


@pytest.mark.gpu
@pytest.mark.parametrize("elem", ["float32", "bfloat16"])
@pytest.mark.parametrize("plan", [(1, 1, 4096), (3, 2, 64), (64, 1, 64), (5, 64, 64), (2, 3, 128)])
def test_any_cut_gives_the_same(elem, plan):
    """Pieces without a key, a last piece that takes far more than the others, bounds that the batch does not keep."""
    c = shared_call(elem, 330, (1, 4, 1), (0, 260, 31), 4, 2, 64, 16)
    records = plan[0] + plan[1]
    out, status = run_shared(c, K.SharedPrefixPlan(*plan, 6 * 4 * records * 66))
    assert status == 0
    check_shared(c, out)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("plan", [(1, 1, 4096), (3, 2, 128), (2, 2, 4096), (64, 1, 128), (6, 64, 128), (4, 6, 64), (2, 3, 256), (1, 1, 64)])
@pytest.mark.parametrize("own", [K.OWN_MANY, K.OWN_TOKEN, K.OWN_ROWS])
def test_any_cut_gives_the_same_on_tensor_cores(dim, plan, own):
    c = shared_call("bfloat16", 330, (1, 4, 1, 40), (0, 260, 31, 500), 4, 2, dim, 16)
    records = plan[0] + plan[1]
    out, status = run_shared(c, K.SharedPrefixPlan(*plan, 46 * 4 * records * (dim + 2), True, own))
    assert status == 0
    check_shared(c, out)


@pytest.mark.gpu
def test_rows_off_16_bytes_take_the_other_kernel():
    """The plan may be the tensor cores'; rows whose stride they cannot take are computed all the same."""
    for pad in (8, 3):
        c = shared_call("bfloat16", 200, (1, 2), (10, 150), 4, 2, 64, 16, pad=pad)
        out, status = run_shared(c)
        assert status == 0
        check_shared(c, out)


@pytest.mark.gpu
@pytest.mark.parametrize("elem,dim", [("bfloat16", 64), ("bfloat16", 128), ("float32", 64), ("bfloat16", 40)])
def test_places_that_hold_no_keys_stay_unseen(elem, dim):
    """Slots behind a request's last key, behind the prefix in its last page and before the own keys in that page may hold anything."""
    c = shared_call(elem, 150, (1, 3, 1), (0, 40, 77), 4, 2, dim, 16)
    want, _ = run_shared(c)
    page = 16
    for x in "kv":
        c[x][int(c["prefix_pages"][-1]), :, 150 % page:] = float("nan")
        for s, own in enumerate((1, 43, 78)):
            table = c["tables"][s]
            c[x][int(table[150 // page]), :, : 150 % page] = float("inf")
            last = 150 + own
            if last % page:
                c[x][int(table[last // page]), :, last % page:] = float("nan")
            for later in table[last // page + 1:].tolist():
                c[x][later] = float("nan")
    out, status = run_shared(c)
    assert status == 0 and torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("elem,dim", [("bfloat16", 64), ("bfloat16", 128), ("float32", 64), ("float32", 20)])
def test_rows_that_see_nothing_and_rows_inside_the_prefix(elem, dim):
    c = shared_call(elem, 200, (1, 1, 1, 1, 2), (3, 3, 3, 3, 3), 4, 2, dim, 16)
    c["positions"][:4] = torch.tensor([-1, 0, 130, 199])
    out, status = run_shared(c)
    assert status == 0 and (out[0] == 0).all()
    check_shared(c, out)


@pytest.mark.gpu
@pytest.mark.parametrize("elem,dim", [("bfloat16", 64), ("bfloat16", 128), ("float32", 64)])
@pytest.mark.parametrize("where", ["prefix", "own", "behind", "starts"])
def test_bad_pages_are_reported(elem, dim, where):
    """Page numbers outside the pool, positions behind the table, starts outside the rows: nothing is read there, the status says so."""
    c = shared_call(elem, 100, (1, 1, 1), (20, 30, 50), 4, 2, dim, 16)
    if where == "prefix":
        c["prefix_pages"][3] = c["k"].shape[0]
    elif where == "own":
        c["tables"][1, 7] = -1
    elif where == "behind":
        c["positions"][2] = 100000
    else:
        c["starts"][3] = 50
    out, status = run_shared(c)
    assert status == (9000002 if where == "starts" else 9000001)
    if where == "own":
        check_shared(c, out, requests=(0, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("elem", ["float32", "bfloat16"])
def test_captured_together_and_replayed(elem):
    """The way of a step: rows turned and appended, then attention; captured once, replayed with other contents, two graphs on one scratch."""
    c = shared_call(elem, 130, (1, 1, 1), (5, 60, 17), 4, 2, 64, 16)
    t, nq, nkv, dim = ELEM[elem], 4, 2, 64
    dev = {x: c[x].cuda() for x in ("k", "v", "prefix_pages", "tables", "starts", "positions")}
    qkv = torch.randn(3, 8 * dim).to(t).cuda()
    plan = K.shared_prefix_plan(3, 3, nq, nkv, dim, t, 16, 130, 300, 1)
    scratch, status = torch.empty(plan.floats).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    outs = [torch.zeros(3, nq * dim, dtype=t).cuda() for _ in range(2)]
    freq = 1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)
    turns = K.rotary_turns(freq).cuda()
    slots = (dev["tables"].cpu()[torch.arange(3), c["positions"].long() // 16] * 16 + c["positions"] % 16).to(torch.int32).cuda()
    q_rows = torch.zeros(3, nq * dim, dtype=t).cuda()

    def step(out):
        K.rotary_append(qkv[:, : nq * dim], dev["positions"], turns, nq, nkv, dim, k=qkv[:, nq * dim: (nq + nkv) * dim], v=qkv[:, (nq + nkv) * dim:],
                        q_out=q_rows, slots=slots, k_pages=dev["k"], v_pages=dev["v"], status=status)
        K.attention_shared_prefix(q_rows, dev["k"], dev["v"], dev["prefix_pages"], 130, dev["tables"], dev["starts"], dev["positions"], out, nq, c["scale"],
                                  plan, scratch, status)

    step(outs[0])
    torch.cuda.synchronize()
    graphs = []
    for out in outs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            step(out)
    for turn in range(3):
        qkv.copy_(torch.randn(3, 8 * dim, generator=torch.Generator().manual_seed(turn)))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert int(status) == 0 and torch.equal(outs[0], outs[1])
        rows = qkv.cpu().double().view(3, 8, dim)
        a, b = rows[..., :32], rows[..., 32:]
        angle = c["positions"].double()[:, None] * freq
        cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        assert (q_rows.cpu().double().view(3, 4, dim) - turned[:, :4]).abs().max() <= turned.abs().max() * (torch.finfo(t).eps / 2 + 2.0**-20)
        now = {**c, "q": q_rows.cpu(), "k": dev["k"].cpu(), "v": dev["v"].cpu()}
        check_shared(now, outs[0].cpu())


@pytest.mark.gpu
def test_another_stream_and_two_calls_at_once():
    """Two calls side by side on streams of their own, each with its own scratch."""
    calls = [shared_call("bfloat16", 2000, (1,) * 20, tuple(range(20)), 8, 2, d, 16, seed=d) for d in (64, 128)]
    want = [run_shared(c)[0] for c in calls]
    streams, got, keep = [torch.cuda.Stream() for _ in calls], [], []
    torch.cuda.synchronize()
    for c, stream in zip(calls, streams):
        nkv, page, dim = c["k"].shape[1:]
        plan = K.shared_prefix_plan(20, 20, 8, nkv, dim, torch.bfloat16, page, 2000, c["max_keys"], 1)
        dev = [c[x].cuda() for x in ("q", "k", "v", "prefix_pages", "tables", "starts", "positions")]
        out, scratch, status = torch.zeros(20, 8 * dim).bfloat16().cuda(), torch.empty(plan.floats).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
        torch.cuda.synchronize()
        keep.append((dev, scratch, status))
        got.append(out)
        with torch.cuda.stream(stream):
            for _ in range(5):
                K.attention_shared_prefix(*dev[:4], 2000, *dev[4:], out, 8, c["scale"], plan, scratch, status)
    torch.cuda.synchronize()
    for w, o, c in zip(want, got, calls):
        check_shared(c, o.cpu(), requests=(0, 7, 19))
        assert (w.double() - o.cpu().double()).abs().max() < 0.02


ROWS = dict(q=torch.zeros(6, 256), k=torch.zeros(6, 128), v=torch.zeros(6, 128), seq_starts=torch.zeros(3, dtype=torch.int32), out=torch.zeros(6, 256), n_q_heads=4,
            n_kv_heads=2, scale=0.125, status=torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("change,word", [
    (dict(q=torch.zeros(6, 256, dtype=torch.float64)), "float32 or bfloat16"),
    (dict(n_kv_heads=3), "share"),
    (dict(n_q_heads=5), "share"),
    (dict(q=torch.zeros(6, 4 * 300), out=torch.zeros(6, 4 * 300)), "at most 256"),
    (dict(scale=0.0), "positive"),
    (dict(scale=float("nan")), "positive"),
    (dict(k=torch.zeros(5, 128)), "k must be"),
    (dict(v=torch.zeros(6, 128).bfloat16()), "v must be"),
    (dict(k=torch.zeros(128, 6).t()), "contiguous"),
    (dict(out=torch.zeros(1, 256).expand(6, 256)), "overlap"),
    (dict(out=torch.zeros(6, 255)), "out must be"),
    (dict(seq_starts=torch.zeros(3)), "seq_starts must be"),
    (dict(status=torch.zeros(0, dtype=torch.int32)), "status must be"),
    (dict(), "CUDA device"),
])
def test_prompt_refusals(change, word):
    with pytest.raises(K.KernelError, match=word):
        K.attention_prompt(**{**ROWS, **change})


PAGED = dict(q=torch.zeros(6, 256), k_pages=torch.zeros(9, 2, 16, 64), v_pages=torch.zeros(9, 2, 16, 64), prefix_pages=torch.zeros(3, dtype=torch.int32), prefix_len=40,
             block_tables=torch.zeros(6, 4, dtype=torch.int32), seq_starts=torch.zeros(7, dtype=torch.int32), positions=torch.zeros(6, dtype=torch.int32),
             out=torch.zeros(6, 256), n_q_heads=4, scale=0.125, plan=K.SharedPrefixPlan(1, 1, 64, 6 * 4 * 2 * 66), scratch=torch.zeros(6 * 4 * 2 * 66),
             status=torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("change,word", [
    (dict(n_q_heads=3), "share"),
    (dict(q=torch.zeros(6, 250)), "q must be"),
    (dict(k_pages=torch.zeros(9, 2, 16)), "pools"),
    (dict(v_pages=torch.zeros(9, 2, 8, 64)), "one shape"),
    (dict(v_pages=torch.zeros(9, 2, 16, 64).bfloat16()), "one shape"),
    (dict(k_pages=torch.zeros(9, 16, 2, 64).transpose(1, 2)), "contiguous"),
    (dict(prefix_len=-1), "prefix of"),
    (dict(prefix_len=50), "prefix_pages must be"),
    (dict(block_tables=torch.zeros(5, 4, dtype=torch.int32)), "block_tables"),
    (dict(block_tables=torch.zeros(6, 0, dtype=torch.int32)), "block_tables"),
    (dict(block_tables=torch.zeros(6, 4)), "block_tables"),
    (dict(positions=torch.zeros(5, dtype=torch.int32)), "positions must be"),
    (dict(scratch=torch.zeros(100)), "scratch must be"),
    (dict(scratch=torch.zeros(6 * 4 * 2 * 66).bfloat16()), "scratch must be"),
    (dict(plan=K.SharedPrefixPlan(0, 1, 64, 0)), "plan does not fit"),
    (dict(plan=K.SharedPrefixPlan(1, 0, 64, 0)), "plan does not fit"),
    (dict(prefix_len=0), "plan does not fit"),
    (dict(status=torch.zeros(1, dtype=torch.int64)), "status must be"),
    (dict(out=torch.zeros(6, 128)), "out must be"),
    (dict(), "CUDA device"),
])
def test_shared_refusals(change, word):
    with pytest.raises(K.KernelError, match=word):
        K.attention_shared_prefix(**{**PAGED, **change})


@pytest.mark.parametrize("rows,seqs,nq,nkv,dim,prefix,keys,fresh", [(1, 1, 2, 2, 64, 0, 1, 1), (64, 64, 32, 8, 128, 16384, 17384, 1), (4, 4, 9, 3, 64, 1024, 1084, 1),
                                                                  (600, 24, 32, 32, 64, 6000, 6060, 60), (256, 256, 32, 8, 128, 4007, 4307, 1), (5, 5, 4, 1, 96, 3, 3, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_plans_cover_the_keys(rows, seqs, nq, nkv, dim, prefix, keys, fresh, dtype):
    p = K.shared_prefix_plan(rows, seqs, nq, nkv, dim, dtype, 16, prefix, keys, fresh, sms=148)
    assert (p.prefix_pieces > 0) == (prefix > 0) and 1 <= p.own_pieces <= 64 and p.prefix_pieces <= 64
    assert p.own_pieces * p.piece_keys >= keys - prefix
    records = p.prefix_pieces + p.own_pieces
    assert p.floats >= (rows * nq * records * (dim + 2) if records > 1 else 0)


def test_plans_of_very_many_requests_stay_launchable():
    for rows, fresh in ((70000, 1), (70000, 2)):
        p = K.shared_prefix_plan(rows, rows // fresh, 8, 8, 64, torch.bfloat16, 16, 64, 96, fresh, sms=148)
        assert p.tensor_cores and (p.own == K.OWN_MANY or rows // fresh <= 65535 and p.own == K.OWN_ROWS and rows // 64 + rows // fresh <= 65535)


@pytest.mark.gpu
@pytest.mark.parametrize("elem", ["float32", "bfloat16"])
@pytest.mark.parametrize("shift", [0, 1, 2])
@pytest.mark.parametrize("dim", [5, 15, 64])
def test_records_at_any_place_of_the_scratch(elem, shift, dim):
    """An odd number of odd records, or a scratch that is a part of a larger buffer: maxima and sums then lie on no 8-byte boundary."""
    c = shared_call(elem, 200, (1,), (70,), 1, 1, dim, 16)
    plan = K.SharedPrefixPlan(2, 1, 4096, 3 * (dim + 2))
    n, width = c["q"].shape[0], c["nq"] * dim
    out, status = torch.zeros((n, width), dtype=c["q"].dtype).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    scratch = torch.full((shift + plan.floats,), float("nan")).cuda()[shift:]
    K.attention_shared_prefix(c["q"].cuda(), c["k"].cuda(), c["v"].cuda(), c["prefix_pages"].cuda(), c["prefix"], c["tables"].cuda(), c["starts"].cuda(),
                              c["positions"].cuda(), out, c["nq"], c["scale"], plan, scratch, status)
    assert int(status) == 0
    check_shared(c, out.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("elem,dim", [("bfloat16", 64), ("bfloat16", 128), ("float32", 64), ("bfloat16", 40)])
@pytest.mark.parametrize("fresh", [(1, 1), (1, 3), (150, 130)])
def test_the_last_position_of_all_is_reported(elem, dim, fresh):
    """Position 2^31 - 1, whose number of keys an int cannot hold, is behind every table."""
    c = shared_call(elem, 100, fresh, (20, 30), 4, 2, dim, 16)
    c["positions"][-1] = 2**31 - 1
    _, status = run_shared(c)
    assert status == 9000001


@pytest.mark.gpu
@pytest.mark.parametrize("elem", ["float32", "bfloat16"])
def test_one_row_of_queries_for_all(elem):
    """Queries whose rows have no stride between them (one row, expanded)."""
    rows, starts, scale = prompt_call(elem, (40, 130), 4, 2, 64)
    one = rows[:1, :256].clone().cuda()
    dev = rows.cuda()
    out, status = torch.zeros((170, 256), dtype=rows.dtype).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    K.attention_prompt(one.expand(170, 256), dev[:, 256:384], dev[:, 384:512], starts.cuda(), out, 4, 2, scale, status)
    rows[:, :256] = one.cpu()
    assert int(status) == 0
    check_prompt(rows, starts, 4, 2, 64, scale, out.cpu())
    c = shared_call(elem, 200, (1, 2), (10, 150), 4, 2, 64, 16)
    want, _ = run_shared({**c, "q": c["q"][:1].repeat(3, 1)})
    plan = K.shared_prefix_plan(3, 2, 4, 2, 64, c["q"].dtype, 16, 200, c["max_keys"], 2, sms=c["sms"])
    got, scratch = torch.zeros((3, 256), dtype=rows.dtype).cuda(), torch.zeros(max(plan.floats, 1)).cuda()
    K.attention_shared_prefix(c["q"][:1].cuda().expand(3, 256), c["k"].cuda(), c["v"].cuda(), c["prefix_pages"].cuda(), 200, c["tables"].cuda(), c["starts"].cuda(),
                              c["positions"].cuda(), got, 4, c["scale"], plan, scratch, status)
    c["q"] = c["q"][:1].repeat(3, 1)
    assert int(status) == 0 and torch.isfinite(want).all()
    check_shared(c, got.cpu())
