"""Sizes at which a count in an int, or the arithmetic on it, would overflow: refused before anything is launched (CPU)."""

from __future__ import annotations

import pytest
import torch

from edgerag_b200.ops import kernels as K
from test_packed_attention import PAGED


@pytest.mark.parametrize("piece_keys", [2**30 + 1, 2**31 - 127, 2**31 - 1, 2**32 + 64])
@pytest.mark.parametrize("plan", [(1, 1), (2, 3)])
def test_pieces_that_their_arithmetic_cannot_hold_are_refused(plan, piece_keys):
    """Rounded up to tiles, pieces of almost 2^31 keys were negative ones, and the last of several then walked tiles from far before the first key on."""
    for tensor_cores in (True, False):
        records = sum(plan)
        made = K.SharedPrefixPlan(*plan, piece_keys, 6 * 4 * records * 66, tensor_cores)
        with pytest.raises(K.KernelError, match="plan does not fit"):
            K.attention_shared_prefix(**{**PAGED, "plan": made, "scratch": torch.zeros(made.floats)})


@pytest.mark.parametrize("nq,nkv,dim,rows,fresh", [(32, 8, 128, 64, 1), (32, 8, 128, 6400, 100), (4, 2, 80, 6400, 100), (512, 512, 64, 600, 4), (2, 1, 64, 1, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("keys", [2**30 + 5, 2**31 - 257, 2**31 - 1])
def test_plans_for_the_longest_contexts_stay_within_that(nq, nkv, dim, rows, fresh, dtype, keys):
    for prefix in (0, 77, 4096):
        p = K.shared_prefix_plan(rows, rows // fresh, nq, nkv, dim, dtype, 16, prefix, keys, fresh, sms=148)
        assert p.piece_keys <= 2**30 and 1 <= p.own_pieces <= 64 and p.own_pieces * p.piece_keys >= keys - prefix


def test_contexts_that_a_walk_cannot_end_are_refused():
    """A walk whose last tile ends behind 2^31 - 1 would start again from below zero: the longest context and prefix lie a tile before that."""
    pools = {x: torch.empty(1, 2, 1 << 16, 64) for x in ("k_pages", "v_pages")}
    wide = {**PAGED, **pools, "prefix_len": 40, "prefix_pages": torch.zeros(1, dtype=torch.int32)}
    for entries, word in ((2**15 - 1, "CUDA device"), (2**15, "keys")):
        with pytest.raises(K.KernelError, match=word):
            K.attention_shared_prefix(**{**wide, "block_tables": torch.empty(6, entries, dtype=torch.int32)})
    pages = torch.empty(2**27, dtype=torch.int32)                     # (never touched)
    for prefix, word in ((2**31 - 256, "CUDA device"), (2**31 - 255, "prefix of"), (2**31 - 17, "prefix of"), (2**32 + 40, "prefix of")):
        with pytest.raises(K.KernelError, match=word):
            K.attention_shared_prefix(**{**PAGED, "prefix_len": prefix, "prefix_pages": pages})


def test_counts_that_an_int_cannot_hold_are_refused():
    """The kernels take rows, sequences, pages and their sizes as ints: 2^32 + 5 rows would be five.  (Tensors without memory: sizes are all that is looked at.)"""
    empty = lambda *shape, dtype=torch.bfloat16: torch.empty(shape, dtype=dtype, device="meta")       # noqa: E731
    ints = lambda *shape: empty(*shape, dtype=torch.int32)                                             # noqa: E731
    turned = lambda n, **more: K.rotary_append(empty(n, 8), ints(n), None, 1, 1, 8, **more)             # noqa: E731
    appended = lambda pages, size: turned(4, k=empty(4, 8), v=empty(4, 8), slots=ints(4), k_pages=empty(pages, 1, size, 8),      # noqa: E731
                                          v_pages=empty(pages, 1, size, 8), status=ints(1))
    prompt = lambda sequences: K.attention_prompt(empty(6, 256), empty(6, 128), empty(6, 128), ints(sequences + 1), empty(6, 256), 4, 2, 0.125, ints(1))   # noqa: E731
    behind = lambda pages: K.attention_shared_prefix(empty(6, 256), empty(pages, 2, 16, 64), empty(pages, 2, 16, 64), ints(3), 40, ints(6, 4), ints(7),      # noqa: E731
                                                     ints(6), empty(6, 256), 4, 0.125, K.SharedPrefixPlan(1, 1, 64, 6 * 4 * 2 * 66), empty(6 * 4 * 2 * 66, dtype=torch.float32), ints(1))
    for call, fits, word in ((turned, 2**31 - 1, "tokens"), (lambda n: appended(n, 16), 2**31 - 1, "pages"), (lambda n: appended(3, n), 2**31 - 1, "pages"),
                             (prompt, 2**31 - 1, "sequences"), (behind, 2**31 - 1, "pages")):
        with pytest.raises(K.KernelError, match="CUDA device"):
            call(fits)
        for n in (2**31, 2**32 + 5):
            with pytest.raises(K.KernelError, match=f"at most 2147483647.*{word}|{word}.*at most 2147483647"):
                call(n)
