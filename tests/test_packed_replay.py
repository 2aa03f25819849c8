"""Calls behind a shared prefix, captured once and replayed back to back: every kernel for the requests' own keys beside the prefix's."""

from __future__ import annotations

import pytest
import torch

from edgerag_b200.ops import kernels as K
from test_packed_attention import ELEM, check_shared, shared_call

FORMS = [("bfloat16", 64, own) for own in (K.OWN_MANY, K.OWN_TOKEN, K.OWN_ROWS)] + [("bfloat16", 128, own) for own in (K.OWN_MANY, K.OWN_TOKEN, K.OWN_ROWS)]
FORMS += [("float32", 64, None), ("bfloat16", 80, None)]


@pytest.mark.gpu
@pytest.mark.parametrize("elem,dim,own", FORMS)
@pytest.mark.parametrize("pieces", [(3, 1, 4096), (4, 3, 128)])
@pytest.mark.parametrize("fresh", [(1, 1, 1), (1, 40, 7)])
def test_replayed_without_a_pause(elem, dim, own, pieces, fresh):
    """Two captured calls on one scratch, one behind the other with other queries and positions, replayed three times without a wait in
    between: a block that began too early would read the other call's queries, or join the other call's records."""
    c = shared_call(elem, 400, fresh, (300, 20, 5), 4, 2, dim, 16)
    t, n, records = ELEM[elem], sum(fresh), pieces[0] + pieces[1]
    plan = K.SharedPrefixPlan(*pieces, n * 4 * records * (dim + 2), own is not None, own or 0)
    dev = {x: c[x].cuda() for x in ("k", "v", "prefix_pages", "tables", "starts")}
    g = torch.Generator().manual_seed(3)
    asked = [torch.randn(n, 4 * dim, generator=g).to(t) for _ in range(2)]
    at = [c["positions"], torch.clamp(c["positions"] - 3, min=0)]
    given = [(q.cuda(), p.cuda()) for q, p in zip(asked, at)]
    q, positions = torch.zeros(n, 4 * dim, dtype=t).cuda(), torch.zeros(n, dtype=torch.int32).cuda()
    outs = [torch.zeros(n, 4 * dim, dtype=t).cuda() for _ in range(2)]
    scratch, status = torch.full((plan.floats,), float("nan")).cuda(), torch.zeros(1, dtype=torch.int32).cuda()

    def both():
        for (rows, where), out in zip(given, outs):
            q.copy_(rows)
            positions.copy_(where)
            K.attention_shared_prefix(q, dev["k"], dev["v"], dev["prefix_pages"], 400, dev["tables"], dev["starts"], positions, out, 4, c["scale"], plan, scratch, status)

    both()
    torch.cuda.synchronize()
    want = [out.clone() for out in outs]
    for rows, where, out in zip(asked, at, want):
        check_shared({**c, "q": rows, "positions": where}, out.cpu())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for out in outs:
        out.zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert int(status) == 0 and all(torch.equal(a, b) for a, b in zip(want, outs))
