"""Timed cases of the operators that take a request's rows from its projections to its attention:

``rotary``   head norms, rotary positions scaled for long contexts, and the append to the paged cache in one pass
``prompt``   causal attention over whole prompts, packed one behind the other, with grouped heads
``shared``   attention of a batch whose requests share a long prefix in the cache: the prefix is read once for all of them

Each has its plain form in elementary torch operations (32-bit arithmetic, one rounding at the end), the calls a user makes of the
package's kernels (``own``), and its definition in 64 bits (``exact``).
"""

from __future__ import annotations

import math
import random

import torch

own = False

ELEM = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp32": 4}

#: (query heads, kv heads, head size): the heads of this package's measured decoders, and generic grouped ones of 128
HEADS = ((32, 32, 64), (9, 3, 64), (15, 5, 64), (32, 8, 128), (16, 2, 128), (8, 1, 128))


def listed() -> list[dict]:
    wide, many, few, odd = {"nq": 32, "nkv": 8, "d": 128}, {"nq": 32, "nkv": 32, "d": 64}, {"nq": 9, "nkv": 3, "d": 64}, {"nq": 15, "nkv": 5, "d": 64}
    return [
        # one decode step of 16 requests deep inside a long context: latency counts
        {"name": "rotary_decode", "op": "rotary", "elem": "bf16", **wide, "tokens": 16, "far": 900000, "layout": "halves", "part": 128,
         "scaling": "turns", "norm": True, "page": 16, "append": True},
        # a full step of prompt portions behind a past
        {"name": "rotary_prefill", "op": "rotary", "elem": "bf16", **wide, "tokens": 8192, "far": 120000, "layout": "halves", "part": 128,
         "scaling": "turns", "norm": False, "page": 16, "append": True},
        # the 32-bit path: neighbouring pairs in half of the head, norms, keys handed on instead of cached
        {"name": "rotary_pairs_fp32", "op": "rotary", "elem": "fp32", **odd, "tokens": 2501, "far": 30000, "layout": "pairs", "part": 32,
         "scaling": "waves", "norm": True, "page": 0, "append": False},
        # a lone short prompt: latency counts
        {"name": "prompt_short", "op": "prompt", "elem": "bf16", **wide, "n": 1, "longest": 48, "mix": 0},
        # prompts of a busy server in one step, lengths from one token on
        {"name": "prompt_ragged", "op": "prompt", "elem": "bf16", **many, "n": 23, "longest": 2001, "mix": 5},
        # one long document
        {"name": "prompt_long", "op": "prompt", "elem": "bf16", **wide, "n": 1, "longest": 8192, "mix": 0},
        # the 32-bit path with heads whose group is no power of two
        {"name": "prompt_fp32", "op": "prompt", "elem": "fp32", **odd, "n": 5, "longest": 701, "mix": 3},
        # a few chats behind one system prompt: latency counts
        {"name": "shared_few", "op": "shared", "elem": "bf16", **few, "n": 4, "prefix": 1024, "longest": 60, "mix": 1, "fresh": 1, "page": 16},
        # a decode step of 64 requests behind one long document
        {"name": "shared_document", "op": "shared", "elem": "bf16", **wide, "n": 64, "prefix": 16384, "longest": 1000, "mix": 2, "fresh": 1, "page": 16},
        # the largest batches behind a prompt that ends inside a page
        {"name": "shared_crowd", "op": "shared", "elem": "bf16", **wide, "n": 256, "prefix": 4007, "longest": 300, "mix": 4, "fresh": 1, "page": 32},
        # questions of several tokens each, all new in this step
        {"name": "shared_questions", "op": "shared", "elem": "bf16", **many, "n": 24, "prefix": 6000, "longest": 60, "mix": 6, "fresh": 60, "page": 16},
        # the 32-bit path
        {"name": "shared_fp32", "op": "shared", "elem": "fp32", **odd, "n": 16, "prefix": 2000, "longest": 120, "mix": 7, "fresh": 1, "page": 16},
    ]


def _log_between(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng) -> dict:
    nq, nkv, d = rng.choice(HEADS)
    op = rng.choice(("rotary", "prompt", "prompt", "shared", "shared"))
    elem = rng.choice(("bf16", "bf16", "bf16", "fp32"))
    case = {"op": op, "elem": elem, "nq": nq, "nkv": nkv, "d": d}
    if op == "rotary":
        append = rng.random() < 0.7
        return {**case, "tokens": _log_between(rng, 1, 8192), "far": _log_between(rng, 1, 1000000), "layout": rng.choice(("halves", "pairs")),
                "part": rng.choice((d, d, d // 2, d // 4)), "scaling": rng.choice(("none", "waves", "turns")), "norm": rng.random() < 0.5,
                "page": rng.choice((8, 16, 32, 64)) if append else 0, "append": append}
    if op == "prompt":
        longest = _log_between(rng, 1, 1500 if elem == "fp32" else 8192)
        most = int(32 * 8192**2 // (nq * longest**2))          # (the scores of the plain form stay within those of the longest prompt)
        return {**case, "n": _log_between(rng, 1, max(1, min(64, most))), "longest": longest, "mix": rng.randrange(1, 1000)}
    n = _log_between(rng, 1, 16 if elem == "fp32" else 256)
    prefix = _log_between(rng, 16, 4000 if elem == "fp32" else max(4000, min(32768, 64 * 16384 // n)))
    longest = _log_between(rng, 1, 1000 if n <= 64 else 300)
    fresh = 1 if n > 48 or rng.random() < 0.6 else min(longest, _log_between(rng, 2, 60))
    return {**case, "n": n, "prefix": prefix, "longest": longest, "mix": rng.randrange(1, 1000), "fresh": fresh, "page": rng.choice((8, 16, 32, 64))}


def _lengths(case: dict) -> list[int]:
    """The requests' lengths: the longest, and shorter ones spread over the logarithm down to a single token."""
    rng = random.Random(case["mix"])
    rest = [_log_between(rng, 1, case["longest"]) for _ in range(case["n"] - 1)]
    at = rng.randrange(case["n"])
    return rest[:at] + [case["longest"]] + rest[at:]


def _starts(lengths: list[int]) -> list[int]:
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    return starts


def _frequencies(case: dict) -> tuple[torch.Tensor, float]:
    """Radians a position turns each pair by (64 bits), and what cosines and sines are multiplied by.  ``waves``: wavelengths beyond
    the trained context stretched, those in between blended; ``turns``: pairs told apart by their turns within it (YaRN)."""
    dims, base, factor, original = case["part"], 500000.0, 16.0, 8192.0
    i = torch.arange(dims // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / dims)
    if case["scaling"] == "waves":
        s = ((original * f / (2.0 * math.pi) - 1.0) / 3.0).clamp(0.0, 1.0)
        return (1.0 - s) * f / factor + s * f, 1.0
    if case["scaling"] == "turns":
        lo, hi = (dims * math.log(original / (2.0 * math.pi * t)) / (2.0 * math.log(base)) for t in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), dims - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        return f / factor * ramp + f * (1.0 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    elem, nq, nkv, d = ELEM[case["elem"]], case["nq"], case["nkv"], case["d"]

    def rows(*shape, scale=1.0):
        return (torch.randn(shape, device="cuda", generator=g) * scale).to(elem)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    st = {"case": case}
    if case["op"] == "rotary":
        t, page = case["tokens"], case["page"]
        qkv = rows(t, (nq + 2 * nkv) * d)               # the projections' rows: q, k and v are views of them
        st["q"], st["k"], st["v"] = qkv[:, : nq * d], qkv[:, nq * d: (nq + nkv) * d], qkv[:, (nq + nkv) * d:]
        first = torch.randint(0, case["far"], (1,), device="cuda", generator=g)
        st["positions"] = (first + torch.arange(t, device="cuda")).to(torch.int32)
        freq, st["multiplier"] = _frequencies(case)
        st["freq"] = freq.cuda()
        if case["norm"]:
            st["q_norm"], st["k_norm"] = (1.0 + 0.2 * torch.randn(d, device="cuda", generator=g) for _ in range(2))
        st["q_out"] = torch.zeros((t, nq * d), dtype=elem, device="cuda")
        if case["append"]:
            pages = -(-t // page) + 2
            st["k_pages"], st["v_pages"] = (torch.zeros((pages, nkv, page, d), dtype=elem, device="cuda") for _ in range(2))
            order = torch.randperm(pages, device="cuda", generator=g)
            at = torch.arange(t, device="cuda")
            st["slots"] = (order[at // page] * page + at % page).to(torch.int32)
        else:
            st["k_out"] = torch.zeros((t, nkv * d), dtype=elem, device="cuda")
        if own:
            from edgerag_b200.ops import kernels
            st["turns"] = kernels.rotary_turns(freq).cuda()
            st["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        return st

    lengths = _lengths(case)
    st["scale"] = d**-0.5
    if case["op"] == "prompt":
        starts = _starts(lengths)
        qkv = rows(starts[-1], (nq + 2 * nkv) * d, scale=1.4)
        st["q"], st["k"], st["v"] = qkv[:, : nq * d], qkv[:, nq * d: (nq + nkv) * d], qkv[:, (nq + nkv) * d:]
        st["starts"] = ints(starts)
        st["out"] = torch.zeros((starts[-1], nq * d), dtype=elem, device="cuda")
        if own:
            st["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        else:
            st.update(_padded(lengths))
        return st

    page, prefix = case["page"], case["prefix"]
    new = [min(n, case["fresh"]) for n in lengths]           # tokens of this step: each request's last ones
    starts = _starts(new)
    st["starts"] = ints(starts)
    st["positions"] = ints([prefix + n - m + i for n, m in zip(lengths, new) for i in range(m)])
    st["q"] = rows(starts[-1], nq * d, scale=1.4)
    shared, per = -(-prefix // page), -(-(prefix + case["longest"]) // page)
    mine = per - prefix // page                              # a request's own pages, the one the prefix ends in among them
    pages = shared + case["n"] * mine
    st["k_pages"], st["v_pages"] = (rows(pages, nkv, page, d, scale=1.4) for _ in range(2))
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    st["prefix_pages"] = order[:shared].contiguous()
    tables = torch.zeros((case["n"], per), dtype=torch.int32, device="cuda")
    tables[:, : prefix // page] = order[: prefix // page]
    tables[:, prefix // page:] = order[shared:].view(case["n"], mine)
    st["tables"] = tables
    st["out"] = torch.zeros((starts[-1], nq * d), dtype=elem, device="cuda")
    if own:
        from edgerag_b200.ops import kernels
        st["plan"] = kernels.shared_prefix_plan(starts[-1], case["n"], nq, nkv, d, elem, page, prefix, prefix + case["longest"], max(new))
        st["scratch"] = torch.empty(max(st["plan"].floats, 1), dtype=torch.float32, device="cuda")
        st["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    else:
        st.update(_padded(new))
        st["own_len"] = case["longest"]
    return st


def _padded(lengths: list[int]) -> dict:
    """Where the packed rows lie in a batch padded to the longest: indices there and back."""
    longest, n = max(lengths), torch.tensor(lengths, device="cuda")
    at = torch.arange(longest, device="cuda")
    there = at[None, :] < n[:, None]
    first = torch.cumsum(n, 0) - n
    return {"there": there, "row": torch.where(there, first[:, None] + at[None, :], 0)}


def _turned(x, st, heads, norm):
    """Rows of heads, normed, turned by their position, in 32 bits (angles in 64)."""
    case = st["case"]
    t, d, half = x.shape[0], case["d"], case["part"] // 2
    x = x.float().view(t, heads, d)
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * norm
    angle = st["positions"].double()[:, None] * st["freq"][None, :]
    cos, sin = ((st["multiplier"] * f(angle)).float()[:, None, :] for f in (torch.cos, torch.sin))
    turned, rest = x[..., : 2 * half], x[..., 2 * half:]
    if case["layout"] == "pairs":
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _run_rotary(st):
    case = st["case"]
    nq, nkv, d, page = case["nq"], case["nkv"], case["d"], case["page"]
    if own:
        from edgerag_b200.ops import kernels
        kernels.rotary_append(st["q"], st["positions"], st["turns"], nq, nkv, d, k=st["k"], v=st["v"] if case["append"] else None,
                              pairs=case["layout"] == "pairs", multiplier=st["multiplier"], q_norm=st.get("q_norm"), k_norm=st.get("k_norm"),
                              eps=1e-6, q_out=st["q_out"], k_out=st.get("k_out"), slots=st.get("slots"), k_pages=st.get("k_pages"),
                              v_pages=st.get("v_pages"), status=st["status"])
    else:
        st["q_out"].copy_(_turned(st["q"], st, nq, st.get("q_norm")).flatten(1))
        k = _turned(st["k"], st, nkv, st.get("k_norm"))
        if case["append"]:
            at, offset = st["slots"].long() // page, st["slots"].long() % page
            st["k_pages"][at, :, offset] = k.to(st["q"].dtype)
            st["v_pages"][at, :, offset] = st["v"].reshape(-1, nkv, d)
        else:
            st["k_out"].copy_(k.flatten(1))
    return {n: st[n] for n in ("q_out", "k_out", "k_pages", "v_pages") if n in st}


def _run_prompt(st):
    case = st["case"]
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    if own:
        from edgerag_b200.ops import kernels
        kernels.attention_prompt(st["q"], st["k"], st["v"], st["starts"], st["out"], nq, nkv, st["scale"], st["status"])
        return st["out"]
    there, row = st["there"], st["row"]
    n, long = there.shape
    q = st["q"].float()[row].view(n, long, nkv, nq // nkv, d).permute(0, 2, 3, 1, 4).reshape(n, nkv, -1, d)
    k, v = (x.float()[row].view(n, long, nkv, d).transpose(1, 2) for x in (st["k"], st["v"]))
    s = torch.matmul(q, k.transpose(2, 3)).mul_(st["scale"]).view(n, nkv, nq // nkv, long, long)
    at = torch.arange(long, device=s.device)
    s.masked_fill_(at[None, :] > at[:, None], float("-inf"))
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(n, nkv, -1, long), v).view(n, nkv, nq // nkv, long, d) / total
    st["out"].copy_(o.permute(0, 3, 1, 2, 4)[there].flatten(1))
    return st["out"]


def _run_shared(st):
    case = st["case"]
    nq, nkv, d, page, prefix = case["nq"], case["nkv"], case["d"], case["page"], case["prefix"]
    if own:
        from edgerag_b200.ops import kernels
        kernels.attention_shared_prefix(st["q"], st["k_pages"], st["v_pages"], st["prefix_pages"], prefix, st["tables"], st["starts"],
                                        st["positions"], st["out"], nq, st["scale"], st["plan"], st["scratch"], st["status"])
        return st["out"]
    there, row, group = st["there"], st["row"], nq // nkv
    n, long = there.shape
    q = st["q"].float()[row].view(n, long, nkv, group, d)
    at = torch.arange(prefix, device=q.device)
    first, offset = st["prefix_pages"].long()[at // page], at % page
    kp, vp = (x[first, :, offset].float().transpose(0, 1) for x in (st["k_pages"], st["v_pages"]))            # [kv heads, prefix, d]
    own_at = prefix + torch.arange(st["own_len"], device=q.device)
    first, offset = st["tables"].long()[:, own_at // page], (own_at % page).expand(n, -1)
    ks, vs = (x[first, :, offset].float().permute(0, 2, 1, 3) for x in (st["k_pages"], st["v_pages"]))        # [n, kv heads, own, d]
    sp = torch.matmul(q.permute(2, 0, 1, 3, 4).reshape(nkv, -1, d), kp.transpose(1, 2)) * st["scale"]
    sp = sp.view(nkv, n, long, group, prefix).permute(1, 0, 2, 3, 4)
    so = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(n, nkv, -1, d), ks.transpose(2, 3)) * st["scale"]
    so = so.view(n, nkv, long, group, -1)
    hidden = own_at[None, None, :] > st["positions"].long()[row][:, :, None]
    so.masked_fill_(hidden[:, None, :, None, :], float("-inf"))
    top = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    sp, so = torch.exp(sp - top), torch.exp(so - top)
    total = sp.sum(-1, keepdim=True) + so.sum(-1, keepdim=True)
    o = torch.matmul(sp.transpose(0, 1).reshape(nkv, -1, prefix), vp).view(nkv, n, long, group, d).transpose(0, 1)
    o = (o + torch.matmul(so.reshape(n, nkv, long * group, -1), vs).view(n, nkv, long, group, d)) / total
    st["out"].copy_(o.permute(0, 2, 1, 3, 4)[there].flatten(1))
    return st["out"]


def run(st):
    op = st["case"]["op"]
    if op == "rotary":
        return _run_rotary(st)
    return _run_prompt(st) if op == "prompt" else _run_shared(st)


def work(case: dict) -> dict:
    nq, nkv, d, size = case["nq"], case["nkv"], case["d"], BYTES[case["elem"]]
    if case["op"] == "rotary":
        t, moved = case["tokens"], nq + (2 if case["append"] else 1) * nkv
        return {"bytes": t * (2 * moved * d * size + 8), "flops": t * (nq + nkv) * (3 * case["part"] + (4 * d if case["norm"] else 0))}
    lengths = _lengths(case)
    if case["op"] == "prompt":
        return {"bytes": sum(lengths) * 2 * (nq + nkv) * d * size, "flops": sum(4 * d * nq * n * (n + 1) // 2 for n in lengths)}
    new = [min(n, case["fresh"]) for n in lengths]
    keys = case["prefix"] + sum(lengths)
    seen = sum(m * (case["prefix"] + n) - m * (m - 1) // 2 for n, m in zip(lengths, new))
    return {"bytes": 2 * (keys * nkv + sum(new) * nq) * d * size, "flops": 4 * d * nq * seen}


def _exact_attention(q, k, v, scale, limit):
    """One head: rows ``q`` over keys ``k``; row ``r`` sees the first ``limit[r]``."""
    out = torch.empty_like(q)
    for r in range(0, q.shape[0], 2048):
        z = (q[r: r + 2048] @ k.T) * scale
        z[torch.arange(k.shape[0], device=z.device)[None, :] >= limit[r: r + 2048, None]] = -math.inf
        out[r: r + 2048] = torch.softmax(z, 1) @ v
    return out


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    if case["op"] == "rotary":
        result = {}
        for name, heads in (("q", nq), ("k", nkv)):
            x = st[name].double().reshape(-1, heads, d).clone()
            if case["norm"]:
                x = x / torch.sqrt((x**2).sum(-1, keepdim=True) / d + 1e-6) * st[name + "_norm"].double()
            for i in range(case["part"] // 2):
                i0, i1 = (2 * i, 2 * i + 1) if case["layout"] == "pairs" else (i, i + case["part"] // 2)
                turn = torch.polar(torch.full_like(st["positions"].double(), st["multiplier"]), st["positions"].double() * st["freq"][i])
                z = torch.complex(x[..., i0].clone(), x[..., i1].clone()) * turn[:, None]
                x[..., i0], x[..., i1] = z.real, z.imag
            result[name] = x
        found = {"q_out": result["q"].flatten(1)}
        if not case["append"]:
            return {**found, "k_out": result["k"].flatten(1)}
        for name, rows in (("k_pages", result["k"]), ("v_pages", st["v"].double().reshape(-1, nkv, d))):
            flat = torch.zeros((st[name].shape[0] * case["page"], nkv, d), dtype=torch.float64, device="cuda")
            flat[st["slots"].long()] = rows
            found[name] = flat.view(-1, case["page"], nkv, d).transpose(1, 2).contiguous()
        return found
    lengths = _lengths(case)
    new = lengths if case["op"] == "prompt" else [min(n, case["fresh"]) for n in lengths]
    starts = _starts(new)
    out = torch.empty((starts[-1], nq, d), dtype=torch.float64, device="cuda")
    for s, (a, b) in enumerate(zip(starts[:-1], starts[1:])):
        for g in range(nkv):
            if case["op"] == "prompt":
                k, v = (st[x][a:b, g * d: (g + 1) * d].double() for x in "kv")
                limit = torch.arange(1, b - a + 1, device="cuda")
            else:
                page, prefix, n = case["page"], case["prefix"], lengths[s]
                table = torch.cat((st["prefix_pages"][: -(-prefix // page)], st["tables"][s, prefix // page:])).long()
                at = torch.arange(prefix + n, device="cuda")
                index = torch.where(at < prefix, at // page, at // page - prefix // page + -(-prefix // page))
                k, v = (st[x][table[index], g, at % page].double() for x in ("k_pages", "v_pages"))
                limit = prefix + n - (b - a) + torch.arange(1, b - a + 1, device="cuda")
            for h in range(g * (nq // nkv), (g + 1) * (nq // nkv)):
                out[a:b, h] = _exact_attention(st["q"][a:b, h * d: (h + 1) * d].double(), k, v, st["scale"], limit)
    return out.flatten(1)
