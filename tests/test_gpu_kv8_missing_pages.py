"""Attention over the paged 8-bit cache where pages of a sequence are none of the cache's: their tokens are left out of outputs,
logarithms and weights, whatever lies in page 0, which is what the kernels read in their place, and whatever the queries hold
that see nothing else.  Every comparison is written so that a NaN fails it; the bounds are those of test_gpu_kv8_attention.py."""
import math

import numpy as np
import pytest
import torch

from castforge_amd import ops
from test_gpu_kv8_attention import _cache, _reference, _table

pytestmark = pytest.mark.gpu

# queries and lengths that take every form: few rows in one launch and split, with saved scores and without; many rows (of eight heads, see
# Case), by four waves, by eight, and split
FORMS = [
    ([1, 1, 1], [200, 64, 130]),
    ([1, 1], [9000, 40]),
    ([1] * 80, [2000] * 79 + [48]),
    ([2, 1, 2], [200, 64, 130]),
    ([3, 1, 1], [7000, 64, 130]),
    ([3, 1, 9], [200, 64, 130]),
    ([40, 33], [300, 33]),
    ([60, 4], [9000, 200]),
    ([900, 700], [1000, 900]),
    ([256], [6000]),
    ([128] * 8, [200] * 8),
    ([1000], [4000]),
]


class Case:
    """Sequences in pages 1 .. of a cache whose page 0 holds NaN, codes and scales; page ids of `missing` ([(sequence, first token,
    end)], whole pages) are outside the cache."""

    def __init__(self, cuda, q_lens, kv_lens, missing, d=128, page=16, seed=0, window=None, sinks=0, causal=True):
        self.q_lens, self.kv_lens, self.page = q_lens, kv_lens, page
        hkv, ratio = (8, 4) if sum(q_lens) > 300 else (2, 2)
        self.args = dict(causal=causal, window=window, sinks=sinks)
        need = [-(-kv // page) for kv in kv_lens]
        tensors = _cache(seed, sum(need) + 1, hkv, page, d, cuda)
        self.table = _table(seed, need, sum(need), max(need), cuda)
        self.table[self.table < sum(need)] += 1
        bad = [-1, sum(need) + 1, 2**31 - 1, -2**31]
        self.gone = torch.zeros((len(kv_lens), max(need) * page), dtype=torch.bool, device=cuda)
        for i, (b, first, end) in enumerate(missing):
            for c in range(first // page, -(-end // page)):
                self.table[b, c] = bad[(i + c) % 4]
                self.gone[b, c * page:(c + 1) * page] = True
        self.clean = ops.Kv8Cache(*[t.clone() for t in tensors])
        tensors[0][0], tensors[2][0] = 0x7F, 0xFF
        tensors[1][0], tensors[3][0] = math.nan, math.nan
        self.cache = ops.Kv8Cache(*tensors)
        g = torch.Generator(device=cuda).manual_seed(seed + 1)
        self.q = (1.5 * torch.randn((sum(q_lens), hkv * ratio, d), generator=g, device=cuda)).bfloat16()
        self.lens = torch.tensor(kv_lens, dtype=torch.int32, device=cuda)
        self.cu = torch.tensor(np.cumsum([0] + q_lens), dtype=torch.int32, device=cuda) if any(n != 1 for n in q_lens) else None
        self.before = torch.rand((len(kv_lens), hkv, max(need) * page), generator=g, device=cuda)

    def call(self, cache=None, q=None):
        weights = self.before.clone()
        out, lse = ops.kv8_attention(self.q if q is None else q, cache or self.cache, self.table, self.lens, cu_q=self.cu, return_lse=True, weights=weights, **self.args)
        return out, lse, weights

    def check(self, got=None, but=None):
        """Against float64; returns the call's results and which rows see nothing, [T, q heads].  but: (row, query head of the first sequence) that
        is not compared, nor the weights that it has a share in."""
        out, lse, weights = got = got or self.call()
        a = self.args
        want, want_lse, bound, slack, given = _reference(self.q, self.clean, self.table, self.kv_lens, self.q_lens, a["causal"], self.cache.head_dim ** -0.5, a["window"], a["sinks"])
        held = torch.ones_like(lse, dtype=torch.bool)
        if but:
            held[but] = False
        far = ~((out.double() - want).abs() <= bound)[held]
        assert not far.any(), f"{far.sum().item()} of {far.numel()} outputs past the bound"
        empty = torch.isinf(want_lse)
        assert torch.equal((lse == -math.inf)[held], empty[held]) and torch.all(out[empty & held] == 0)
        assert torch.all(((lse.double() - want_lse).abs() <= slack)[held & ~empty])
        for b, (w, off) in enumerate(given):
            n = w.shape[1]
            expect = self.before[b].double()
            expect[:, :n] += w
            tol = 2.0 ** -24 * expect
            tol[:, :n] += off
            far = ~((weights[b].double() - expect).abs() <= tol)
            if but and b == 0:
                far = far[torch.arange(far.shape[0], device=far.device) != but[1] * far.shape[0] // self.q.shape[1]]
            assert not far.any(), (b, far.sum().item(), torch.isnan(weights[b]).sum().item())
            assert torch.equal(weights[b][:, self.gone[b]], self.before[b][:, self.gone[b]])
        return got, empty


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_lens,kv_lens", FORMS)
def test_sequences_of_missing_pages_alone(cuda, q_lens, kv_lens, d):
    """The last sequence of a batch: zeros, -inf, and its weights as they were."""
    b = len(kv_lens) - 1
    case = Case(cuda, q_lens, kv_lens, [(b, 0, kv_lens[b])], d=d, seed=d)
    (out, lse, weights), empty = case.check()
    n = q_lens[b]
    assert empty[-n:].all() and torch.all(out[-n:] == 0) and torch.all(lse[-n:] == -math.inf)
    assert torch.equal(weights[b], case.before[b])


@pytest.mark.parametrize("q_lens,kv_lens", FORMS)
def test_some_missing_pages(cuda, q_lens, kv_lens):
    """At a sequence's start (a prompt's first queries see nothing else), inside it, and at its end."""
    kv = kv_lens[0]
    for missing in ([(0, 0, 32)], [(0, 64, 80), (0, 112, 144)], [(0, kv - kv % 16 - 16, kv)], [(0, 0, 16), (len(kv_lens) - 1, 16, 32)]):
        Case(cuda, q_lens, kv_lens, missing, seed=3).check()


@pytest.mark.parametrize("q_lens,kv_lens", FORMS)
@pytest.mark.parametrize("sinks", [0, 20])
def test_windows_over_missing_pages(cuda, q_lens, kv_lens, sinks):
    """Of the tokens that the last queries see, those of the window are gone, and with sinks the first ones are not."""
    kv = kv_lens[0]
    case = Case(cuda, q_lens, kv_lens, [(0, max(kv - 128, 0) // 16 * 16, kv)], seed=5, window=60, sinks=sinks)
    _, empty = case.check()
    assert empty[q_lens[0] - 1].all() == (sinks == 0)


@pytest.mark.parametrize("q_lens,kv_lens", FORMS)
def test_what_page_0_holds_is_not_read(cuda, q_lens, kv_lens):
    missing = [(0, 32, 48), (0, 80, 112), (len(kv_lens) - 1, 0, 16)]
    case = Case(cuda, q_lens, kv_lens, missing, seed=7)
    for a, b in zip(case.call(), case.call(case.clean)):
        assert torch.equal(a, b)
    case = Case(cuda, q_lens, kv_lens, missing, seed=7, causal=False)
    for a, b in zip(case.call(), case.call(case.clean)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("q_lens,kv_lens", FORMS)
def test_a_query_of_nan_leaves_missing_tokens_alone(cuda, q_lens, kv_lens, value):
    """The last query of a sequence whose start is missing: its own outputs and the weights of the tokens that it sees, no others."""
    case = Case(cuda, q_lens, kv_lens, [(0, 0, 32), (0, 48, 64)], seed=9)
    q, row = case.q.clone(), q_lens[0] - 1
    q[row, 1] = value
    case.check(case.call(q=q), but=(row, 1))


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("q_lens,kv_lens", FORMS)
def test_a_query_of_nan_that_sees_nothing_gives_zeros(cuda, q_lens, kv_lens, value):
    """The padding of a batch holds anything: the last sequence, whose pages are all missing, and the first queries of the first, or those whose
    window is missing.  Their queries reach nothing: neither their rows nor others'."""
    b, kv = len(kv_lens) - 1, kv_lens[0]
    for missing, window in (((0, 0, 48 if b else kv), None), ((0, max(kv - 128, 0) // 16 * 16, kv), 60)):
        case = Case(cuda, q_lens, kv_lens, [missing, (b, 0, kv_lens[b])] if b else [missing], seed=11, window=window)
        want, empty = case.check()
        q = case.q.clone()
        q[empty] = value
        for x, y in zip(case.call(q=q), want):
            assert torch.equal(x, y)
        assert empty[-q_lens[b] if b or not window else -1:].all()


@pytest.mark.parametrize("q_lens,kv_lens", FORMS)
def test_queries_whose_scores_are_all_minus_infinity(cuda, q_lens, kv_lens):
    """-inf times positive keys: as if they saw nothing, for the weights too."""
    case = Case(cuda, q_lens, kv_lens, [], seed=13)
    k = case.cache.k_codes
    k.copy_((k & 0x7F).clamp(1, 0x7E))
    want = case.call()
    q, n = case.q.clone(), q_lens[0]
    q[:n] = -math.inf
    out, lse, weights = case.call(q=q)
    assert torch.all(out[:n] == 0) and torch.all(lse[:n] == -math.inf) and torch.equal(weights[0], case.before[0])
    assert torch.equal(out[n:], want[0][n:]) and torch.equal(lse[n:], want[1][n:]) and torch.equal(weights[1:], want[2][1:])
    q = case.q.clone()
    q[n - 1] = -math.inf  # beside others
    out, lse, weights = case.call(q=q)
    assert torch.all(out[n - 1] == 0) and torch.all(lse[n - 1] == -math.inf) and torch.isfinite(out).all() and torch.isfinite(weights).all()
    if n == 1:
        assert torch.equal(weights[0], case.before[0])
