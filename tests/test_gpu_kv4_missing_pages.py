"""Attention over the paged 4-bit cache: queries that see pages outside the cache alone give zeros, whatever they hold themselves."""
import math

import numpy as np
import pytest
import torch

from castforge_amd import ops
from test_gpu_kv4_attention import _cache, _reference, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("q_lens,kv_lens,hkv,ratio", [  # few rows, in one launch and split; two row tiles a wave; many rows
    ([1, 1, 1], [200, 64, 130], 2, 2), ([1, 1], [9000, 40], 2, 2), ([3, 1, 9], [200, 64, 130], 2, 2), ([40, 33], [300, 33], 2, 2),
    ([60, 70], [9000, 200], 2, 2), ([1700, 700], [1800, 900], 8, 4), ([2000], [4000], 8, 4)])
def test_a_query_of_nan_that_sees_nothing_gives_zeros(cuda, q_lens, kv_lens, hkv, ratio, d, group, value):
    """The padding of a batch: the last sequence, whose pages are all missing, and the first queries of the first, which see missing pages
    alone.  They reach neither their own rows nor others'."""
    page, b = 16, len(kv_lens) - 1
    need = [-(-kv // page) for kv in kv_lens]
    cache, table = _cache(1, sum(need), hkv, page, d, group, cuda), _table(1, need, sum(need), max(need), cuda)
    table[0, :3 if b else need[0]] = -1
    if b:
        table[b, :need[b]] = sum(need)
    q = torch.randn((sum(q_lens), hkv * ratio, d), generator=torch.Generator(device=cuda).manual_seed(2), device=cuda).bfloat16()
    lens = torch.tensor(kv_lens, dtype=torch.int32, device=cuda)
    cu = torch.tensor(np.cumsum([0] + q_lens), dtype=torch.int32, device=cuda) if any(n != 1 for n in q_lens) else None
    want, want_lse, bound, _ = _reference(q, cache, table, kv_lens, q_lens, True, d ** -0.5)
    empty = torch.isinf(want_lse)
    assert empty[-q_lens[b]:].all()
    q[empty] = value
    out, lse = ops.kv4_attention(q, cache, table, lens, cu_q=cu, return_lse=True)
    assert torch.all(out[empty] == 0) and torch.equal(lse == -math.inf, empty)
    assert not (~((out.double() - want).abs() <= bound)).any()
