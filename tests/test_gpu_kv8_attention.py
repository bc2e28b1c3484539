"""Attention over the paged 8-bit cache, over all tokens and over a window with sinks, and the weights that the tokens got,
against float64 over the cache's own numbers.

Bound of an output: weights are rounded to f16, 2^-11 of each term, so 2^-11 of sum p |v|; f16 holds no number below
2^-25, where the largest weights times their values' scale are above 2^7: 448 2^-32 of the largest p s a token, s the scale of
its values; scores are f32 sums of d exact products and a scale, (d + 8) 2^-24 of scale * sum |q k| each, which moves a weight by
as much of itself, and so the output by twice that of sum p |v|, and the logarithm of the sum by as much; a bf16
output rounds by 2^-8 of itself.  Sums of n f32 terms add n 2^-24 of themselves, the logarithm 2^-22 of itself and 1.  A weight is off by
twice what its score is, and by what the logarithm is; its sum over the rows by 2^-24 of itself a row."""
import math

import numpy as np
import pytest
import torch

from castforge_amd import ffi, ops

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _cache(seed, pages, heads, page, d, cuda, power=True, spread=2, base=-8):
    g, t = torch.Generator(device=cuda).manual_seed(seed), []
    for _ in range(2):
        c = torch.randint(0, 256, (pages, heads, page, d), generator=g, device=cuda, dtype=torch.uint8)
        t.append(torch.where(c & 0x7F == 0x7F, torch.zeros_like(c), c))
        s = torch.randint(-spread, spread + 1, (pages, heads), generator=g, device=cuda).float() + base
        t.append(torch.exp2(s if power else s + torch.rand((pages, heads), generator=g, device=cuda)))
    return t


def _numbers(codes, scales):
    return codes.view(F8).double() * scales.double()[..., None, None]


def _reference(q, cache, table, kv_lens, q_lens, causal, scale, window, sinks):
    """(out, lse, their bounds, [weights and their bounds of each sequence, [H, kv]]) in float64, a sequence at a time."""
    hq, hkv, page, d = q.shape[1], cache.kv_heads, cache.page_size, cache.head_dim
    ratio, first = hq // hkv, 0
    outs, lses, bounds, slack, given = [], [], [], [], []
    for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        kv = min(max(kv, 0), table.shape[1] * page) if cache.num_pages else 0
        ids = table[b, :-(-kv // page)].long()
        ok = ((ids >= 0) & (ids < cache.num_pages)).repeat_interleave(page)[:kv]
        ids = ids.clamp(0, max(cache.num_pages - 1, 0))
        k, v = (torch.where(ok[:, None], _numbers(c[ids], s[ids]).transpose(0, 1).flatten(1, 2)[:, :kv], 0.0)
                for c, s in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)))
        x = q[first:first + n].double().transpose(0, 1).unflatten(0, (hkv, ratio))  # [H, ratio, n, D]
        first += n
        t, place = torch.arange(kv, device=q.device), torch.arange(n, device=q.device)[:, None] + kv - n
        seen = ok[None].expand(n, kv).clone()
        if causal:
            seen &= t <= place
        if window:
            seen &= (t > place - window) | (t < sinks)
        kk, vv = k[:, None], v[:, None]
        if kv:
            s = (x @ kk.transpose(2, 3) * scale).masked_fill(~seen, -math.inf)
            lse = torch.logsumexp(s, -1)
            p = torch.where(seen, torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse)[..., None]), 0.0)
            mag = (x.abs() @ kk.abs().transpose(2, 3) * abs(scale)).masked_fill(~seen, 0)
        else:
            p = mag = torch.zeros((hkv, ratio, n, 0), dtype=torch.float64, device=q.device)
            lse = torch.full((hkv, ratio, n), -math.inf, dtype=torch.float64, device=q.device)
        o, pv = p @ vv, p @ vv.abs()
        one = (d + 8) * 2.0 ** -24
        most = mag.amax(-1) if kv else torch.zeros_like(lse)
        under = kv * 448 * 2.0 ** -32 * (p * vv.abs().amax(-1)[:, :, None]).amax(-1, keepdim=True) if kv else torch.zeros_like(o[..., :1])
        off = one * most + 2.0 ** -22 * (1 + torch.where(torch.isinf(lse), 0.0, lse).abs()) + (kv / 4 + 64) * 2.0 ** -24
        outs.append(o), lses.append(lse), slack.append(off)
        bounds.append((2.0 ** -11 + 2 * one * most[..., None] + 2 * 2.0 ** -20) * pv * 1.01 + under + 2.0 ** -8 * o.abs() + 1e-30)
        w = p.sum((1, 2))
        given.append((w, (p * (2 * one * mag + off[..., None] + 2.0 ** -21)).sum((1, 2)) + (n * ratio + 2) * 2.0 ** -24 * w + 1e-30))
    flat = [torch.cat([t.flatten(0, 1).transpose(0, 1) for t in part]) if part else None for part in (outs, lses, bounds, slack)]
    return (*flat, given)


def _table(seed, need, pages, cols, cuda):
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    t = torch.full((len(need), cols), 2**31 - 1, dtype=torch.int32)  # entries past the last page are never read
    i = 0
    for b, n in enumerate(need):
        t[b, :n] = perm[i:i + n]
        i += n
    return t.to(cuda)


def _check(q, cache, table, kv_lens, q_lens, lens, cu, causal, scale, window, sinks, weights_cols=None):
    d = cache.head_dim
    args = dict(cu_q=cu, causal=causal, scale=scale, window=window, sinks=sinks)
    cols = table.shape[1] * cache.page_size if weights_cols is None else weights_cols
    g = torch.Generator(device=q.device).manual_seed(len(kv_lens))
    before = torch.rand((len(kv_lens), cache.kv_heads, cols), generator=g, device=q.device)
    weights = before.clone()
    got, lse = ops.kv8_attention(q, cache, table, lens, return_lse=True, weights=weights, **args)
    want, want_lse, bound, slack, given = _reference(q, cache, table, kv_lens, q_lens, causal, d ** -0.5 if scale is None else scale, window, sinks)
    got, lse = got[:want.shape[0]], lse[:want.shape[0]]
    far = ~((got.double() - want).abs() <= bound)
    assert not far.any(), f"{far.sum().item()} of {want.numel()} outputs past the bound, worst {((got.double() - want).abs() / bound).max().item():.2f}"
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty) and torch.all(got[empty] == 0)
    assert torch.all(((lse.double() - want_lse).abs() <= slack)[~empty])
    for b, (w, off) in enumerate(given):
        n = min(w.shape[1], cols)
        expect = before[b].double()
        expect[:, :n] += w[:, :n]
        tol = 2.0 ** -24 * expect
        tol[:, :n] += off[:, :n]
        far = (weights[b].double() - expect).abs() > tol
        assert not far.any(), (b, far.sum().item(), ((weights[b].double() - expect).abs() / tol.clamp(min=1e-30)).max().item())
        assert torch.equal(weights[b, :, n:], before[b, :, n:])
    assert torch.equal(ops.kv8_attention(q, cache, table, lens, **args)[:want.shape[0]], got)
    return got


def _run(cuda, q_lens, kv_lens, hkv, ratio, d, page, causal=True, seed=0, scale=None, extra_cols=0, varlen=None, q_scale=1.5, window=None, sinks=0,
         weights_cols=None, **cache_args):
    need = [-(-max(kv, 0) // page) for kv in kv_lens]
    pages = sum(need) + 2
    tensors = _cache(seed, pages, hkv, page, d, cuda, **cache_args)
    table = _table(seed, need, pages, max(need + [0]) + extra_cols, cuda)
    # places past a sequence's end, and pages of none: NaN
    ends = torch.zeros(pages, dtype=torch.int64, device=cuda)
    for b, (kv, n) in enumerate(zip(kv_lens, need)):
        for c in range(n):
            ends[table[b, c].long()] = min(kv - c * page, page)
    off = (torch.arange(page, device=cuda) >= ends[:, None])[:, None, :, None]
    for i in (0, 2):
        tensors[i] = torch.where(off, torch.full_like(tensors[i], 0x7F), tensors[i])
        tensors[i + 1] = torch.where((ends == 0)[:, None], torch.full_like(tensors[i + 1], math.nan), tensors[i + 1])
    cache = ops.Kv8Cache(*tensors)
    g = torch.Generator(device=cuda).manual_seed(seed + 1)
    q = (q_scale * torch.randn((sum(q_lens), hkv * ratio, d), generator=g, device=cuda)).bfloat16()
    lens = torch.tensor(kv_lens, dtype=torch.int32, device=cuda)
    if varlen is None:
        varlen = any(n != 1 for n in q_lens)
    cu = torch.tensor(np.cumsum([0] + q_lens), dtype=torch.int32, device=cuda) if varlen else None
    # the reference reads NaN places too, times nothing
    clean = ops.Kv8Cache(*[torch.where(t & 0x7F == 0x7F, torch.zeros_like(t), t) if t.dtype == torch.uint8 else torch.nan_to_num(t, nan=1.0) for t in tensors])
    got = _check(q, cache, table, kv_lens, q_lens, lens, cu, causal, scale, window, sinks, weights_cols)
    assert torch.equal(ops.kv8_attention(q, clean, table, lens, cu_q=cu, causal=causal, scale=scale, window=window, sinks=sinks), got)
    return q, cache, table, lens, cu, got


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kv", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 500, 1000])
def test_single_queries(cuda, d, kv):
    _run(cuda, [1, 1], [kv, max(1, kv // 2)], 2, 4, d, 16, seed=kv)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (1, 1), (16, 4), (33, 0), (100, 64), (128, 3), (700, 5), (5000, 40)])
def test_windows_and_pages(cuda, page, window, sinks):
    _run(cuda, [1, 1, 1, 1], [777, 100, 3, 701], 2, 3, 128, page, window=window, sinks=sinks, seed=page)
    _run(cuda, [5, 40, 3, 129], [777, 100, 3, 701], 1, 2, 64, page, window=window, sinks=sinks, seed=page + 1)


@pytest.mark.parametrize("ratio", [1, 2, 3, 5, 7, 8, 16, 17, 33, 64])
def test_head_layouts(cuda, ratio):
    _run(cuda, [1, 1, 1], [300, 41, 1], 2, ratio, 64, 16, seed=ratio)
    _run(cuda, [3, 17, 1], [300, 41, 1], 1, ratio, 128, 32, seed=ratio, window=37, sinks=2)


@pytest.mark.parametrize("d,hkv,ratio,q_lens,kv_lens,page", [
    (128, 2, 4, [65, 300, 1, 17], [65, 700, 900, 17], 64),
    (64, 4, 2, [257, 31], [257, 1031], 16),
    (128, 1, 8, [130], [1130], 256),
    (128, 8, 4, [700], [700], 64),
    (64, 8, 8, [333, 400], [333, 2000], 32),
    (128, 8, 4, [1500, 900], [1500, 1700], 64),
    (64, 8, 4, [2048, 700], [2048, 800], 32),
    (128, 32, 1, [1700], [2100], 128),
])
@pytest.mark.parametrize("window,sinks", [(None, 0), (200, 4)])
def test_prompts(cuda, d, hkv, ratio, q_lens, kv_lens, page, window, sinks):
    _run(cuda, q_lens, kv_lens, hkv, ratio, d, page, window=window, sinks=sinks, seed=d + hkv)


@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 1), (64, 0), (129, 33), (1023, 64), (3000, 4)])
@pytest.mark.parametrize("d", [64, 128])
def test_prompts_through_windows_of_every_kind(cuda, window, sinks, d):
    _run(cuda, [1601, 700], [1601, 2222], 8, 4, d, 64, window=window, sinks=sinks, seed=window)


def test_without_causal_order(cuda):
    _run(cuda, [5, 1, 40], [100, 7, 40], 2, 3, 128, 16, causal=False, seed=2)
    _run(cuda, [2000], [1100], 8, 4, 64, 64, causal=False, seed=2)


def test_more_queries_than_tokens_and_none(cuda):
    """Rows that see nothing: zeros and -inf, and no weights."""
    _run(cuda, [5, 3, 4, 1], [3, 0, -2, 1], 2, 2, 128, 16, seed=1)
    _run(cuda, [1, 1, 1], [0, 5, -1], 2, 2, 64, 16, seed=1)
    _run(cuda, [1900, 300], [700, 0], 8, 4, 128, 64, seed=1)
    _run(cuda, [1900, 300], [700, 0], 8, 4, 64, 64, seed=1, window=50, sinks=3)


def test_many_sequences(cuda):
    kv = [1 + (i * 37) % 200 for i in range(150)]
    _run(cuda, [1] * 150, kv, 2, 4, 64, 16, seed=4)
    _run(cuda, [i % 4 for i in range(150)], kv, 1, 3, 128, 16, seed=4, window=60, sinks=2)


def test_long_sequences_are_split(cuda):
    _run(cuda, [1], [40000], 2, 4, 128, 64, seed=1)
    _run(cuda, [1], [33333], 1, 1, 64, 16, seed=1, window=20000, sinks=10)
    _run(cuda, [3, 1], [20000, 9], 2, 7, 128, 256, seed=2)


@pytest.mark.parametrize("causal", [True, False])
def test_scales_that_are_no_powers_of_two(cuda, causal):
    _run(cuda, [1, 1], [700, 90], 2, 4, 128, 16, seed=3, power=False, causal=causal)
    _run(cuda, [1500], [1600], 8, 4, 128, 64, seed=3, power=False, causal=causal)


@pytest.mark.parametrize("base,spread", [(-30, 30), (-68, 2), (28, 2), (-20, 50)])
def test_scales_of_the_whole_range(cuda, base, spread):
    """Pages' scales of values 2^100 apart, those of keys such that scores stay in range."""
    q_lens, kv_lens, page = [1, 1, 1], [600, 33, 1000], 16
    for q_lens, kv_lens, hkv in (([1, 1, 1], [600, 33, 1000], 2), ([1600], [1600], 8)):
        need = [-(-kv // page) for kv in kv_lens]
        t = _cache(5, sum(need), hkv, page, 128, cuda)
        t[3] = _cache(6, sum(need), hkv, page, 128, cuda, spread=spread, base=base)[3]
        cache, table = ops.Kv8Cache(*t), _table(5, need, sum(need), max(need), cuda)
        q = torch.randn((sum(q_lens), 4 * hkv, 128), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda).bfloat16()
        lens = torch.tensor(kv_lens, dtype=torch.int32, device=cuda)
        cu = torch.tensor(np.cumsum([0] + q_lens), dtype=torch.int32, device=cuda)
        _check(q, cache, table, kv_lens, q_lens, lens, cu, True, None, None, 0)


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [900, 300]), ([1500], [1500])])
def test_large_scores(cuda, q_lens, kv_lens):
    """Softmaxes of one token, and references that move by thousands."""
    _run(cuda, q_lens, kv_lens, 8, 4, 128, 64, seed=8, q_scale=300.0)
    _run(cuda, q_lens, kv_lens, 8, 4, 64, 64, seed=8, q_scale=300.0, scale=-0.1)
    _run(cuda, q_lens, kv_lens, 8, 4, 64, 64, seed=8, scale=0.0)


def test_bad_pages_are_left_out_and_lengths_cut(cuda):
    for q_lens, kv_lens in (([1, 1, 1], [200, 64, 130]), ([3, 1, 9], [200, 64, 130]), ([900, 700], [1000, 900])):
        q, cache, table, lens, cu, ref = _run(cuda, q_lens, kv_lens, 8, 4, 128, 16, seed=3)
        bad = table.clone()
        bad[0, 2], bad[0, 5], bad[1, 0], bad[-1, 1] = -1, cache.num_pages, 2**31 - 1, -2**31
        tensors = [torch.where(t & 0x7F == 0x7F, torch.zeros_like(t), t) if t.dtype == torch.uint8 else torch.nan_to_num(t, nan=1.0) for t in
                   (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
        _check(q, ops.Kv8Cache(*tensors), bad, kv_lens, q_lens, lens, cu, True, None, None, 0)
        tensors[0][0], tensors[2][0] = 0x7F, 0xFF  # what a page id that is none reads instead
        used = (table == 0).any()
        if not used:
            assert torch.isfinite(ops.kv8_attention(q, ops.Kv8Cache(*tensors), bad, lens, cu_q=cu)).all()
        page = table.shape[1] * 16
        over = torch.where(lens == lens.max(), lens + 1000, lens)
        exact = torch.where(lens == lens.max(), torch.full_like(lens, page), lens)
        full = torch.where((table >= 0) & (table < cache.num_pages), table, 0)
        clean = ops.Kv8Cache(*[torch.where(t & 0x7F == 0x7F, torch.zeros_like(t), t) if t.dtype == torch.uint8 else torch.nan_to_num(t, nan=1.0) for t in tensors])
        assert torch.equal(ops.kv8_attention(q, clean, full, over, cu_q=cu), ops.kv8_attention(q, clean, full, exact, cu_q=cu))


def test_nan_of_one_query_stays_with_it(cuda):
    for q_lens, kv_lens in (([1, 1], [100, 50]), ([1000], [1000])):
        q, cache, table, lens, cu, ref = _run(cuda, q_lens, kv_lens, 8, 4, 128, 64, seed=3)
        q[0, 3] = math.nan
        got = ops.kv8_attention(q, cache, table, lens, cu_q=cu)
        assert torch.isnan(got[0, 3]).all()
        got[0, 3] = ref[0, 3]
        assert torch.equal(got, ref)


def test_rows_of_no_sequence_are_left_alone(cuda):
    for n in (4, 1100):
        q, cache, table, lens, cu, ref = _run(cuda, [3, n], [40, n], 8, 4, 64, 16, seed=3)
        padded = torch.cat([q, torch.full((5, *q.shape[1:]), math.nan, dtype=q.dtype, device=cuda)])
        t, hq, d = padded.shape
        out, lse = torch.full_like(padded, 7.0), torch.full((t, hq), 7.0, device=cuda)
        size = ops._kv8_workspace(0, 8, 16, 64, t, hq, 2, table.shape[1], 1, 0, 0, 0)
        ws = torch.empty(max(size, 1), dtype=torch.uint8, device=cuda)
        ffi.call("castforge_hip_kv8_attention", cache._ref, padded.data_ptr(), hq * d, t, hq, 2, cu.data_ptr(), table.data_ptr(), table.shape[1],
                 lens.data_ptr(), 1, 0, 0, d ** -0.5, out.data_ptr(), lse.data_ptr(), None, 0, ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
        assert torch.equal(out[:-5], ref) and torch.all(out[-5:] == 7.0) and torch.all(lse[-5:] == 7.0)


def test_strided_queries_and_other_streams(cuda):
    q, cache, table, lens, cu, ref = _run(cuda, [3, 5], [100, 60], 2, 3, 128, 16, seed=3)
    wide = torch.zeros((8, 11, 128), dtype=torch.bfloat16, device=cuda)
    wide[:, 2:8] = q
    assert torch.equal(ops.kv8_attention(wide[:, 2:8], cache, table, lens, cu_q=cu), ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.kv8_attention(q, cache, table, lens, cu_q=cu)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref)


def test_captured_calls_follow_their_lists_and_share_no_workspace(cuda):
    q, cache, table, lens, cu, ref = _run(cuda, [1, 1], [3000, 1700], 2, 4, 128, 64, seed=3)
    weights = torch.zeros((2, 2, table.shape[1] * 64), device=cuda)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.kv8_attention(q, cache, table, lens, weights=weights.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.kv8_attention(q, cache, table, lens, weights=weights)
        y2 = ops.kv8_attention(-q, cache, table, lens, window=200, sinks=4)
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        z = ops.kv8_attention(q, cache, table, lens, window=100)
    for cut in (0, 1, 900, 1690):
        lens.copy_(torch.tensor([3000 - cut, 1700 - cut], dtype=torch.int32))
        weights.zero_()
        graph.replay(), other.replay()
        torch.cuda.synchronize()
        w = torch.zeros_like(weights)
        assert torch.equal(y, ops.kv8_attention(q, cache, table, lens, weights=w)) and torch.equal(w, weights)
        assert torch.equal(y2, ops.kv8_attention(-q, cache, table, lens, window=200, sinks=4))
        assert torch.equal(z, ops.kv8_attention(q, cache, table, lens, window=100))


def test_weights_shorter_and_longer_than_the_table(cuda):
    for cols in (0, 1, 33, 64, 500):
        _run(cuda, [1, 1], [300, 20], 2, 4, 64, 16, seed=3, weights_cols=cols)
        _run(cuda, [3, 9], [300, 20], 2, 4, 128, 16, seed=3, weights_cols=cols, window=40, sinks=20)


def test_a_cache_of_more_than_2_32_bytes(cuda):
    """Offsets past 32 bits, in the codes and in the table."""
    page, hkv, d = 256, 4, 128
    pages = 2**32 // (page * hkv * d) + 40
    t = [torch.empty((pages, hkv, page, d), dtype=torch.uint8, device=cuda) for _ in range(2)]
    for x in t:
        x.fill_(0x7F)
    kv = [1000, 515]
    need = [-(-n // page) for n in kv]
    small = _cache(1, sum(need), hkv, page, d, cuda)
    far = torch.tensor([[pages - 1, 7, pages - 3, pages - 4], [pages - 5, 1, pages - 9, 0]], dtype=torch.int32, device=cuda)
    table = torch.tensor([[0, 1, 2, 3], [4, 5, 6, 0]], dtype=torch.int32, device=cuda)
    s = [torch.ones((pages, hkv), device=cuda) for _ in range(2)]
    for b, n in enumerate(need):
        for c in range(n):
            for i in range(2):
                t[i][far[b, c].long()] = small[2 * i][table[b, c].long()]
                s[i][far[b, c].long()] = small[2 * i + 1][table[b, c].long()]
    big, near = ops.Kv8Cache(t[0], s[0], t[1], s[1]), ops.Kv8Cache(*small)
    lens = torch.tensor(kv, dtype=torch.int32, device=cuda)
    for n in ([1, 1], [900, 500]):
        q = torch.randn((sum(n), 16, d), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda).bfloat16()
        cu = torch.tensor(np.cumsum([0] + n), dtype=torch.int32, device=cuda)
        w = [torch.zeros((2, hkv, 1024), device=cuda) for _ in range(2)]
        assert torch.equal(ops.kv8_attention(q, big, far, lens, cu_q=cu, weights=w[0]), ops.kv8_attention(q, near, table, lens, cu_q=cu, weights=w[1]))
        assert torch.equal(*w)


def test_refusals_and_empty_calls(cuda):
    cache = ops.Kv8Cache.empty(4, 2, 16, 128, device=cuda)
    i32 = dict(dtype=torch.int32, device=cuda)
    q, table, lens = torch.zeros((3, 8, 128), dtype=torch.bfloat16, device=cuda), torch.zeros((3, 2), **i32), torch.ones(3, **i32)
    good = dict(q=q, cache=cache, page_table=table, kv_lens=lens)
    ops.kv8_attention(**good)
    for bad in (dict(q=q.float()), dict(q=q[..., :64]), dict(q=q[:, :7]), dict(q=q[:2]), dict(q=q.cpu()), dict(page_table=table.long()), dict(page_table=table[0]),
                dict(kv_lens=lens[:2]), dict(kv_lens=lens.long()), dict(cu_q=torch.zeros(3, **i32)), dict(window=0), dict(window=-3),
                dict(weights=torch.zeros((3, 2, 5), dtype=torch.float64, device=cuda)), dict(weights=torch.zeros((3, 8, 5), device=cuda)),
                dict(weights=torch.zeros((3, 2, 5))), dict(weights=torch.zeros((3, 2, 10), device=cuda)[..., ::2])):
        with pytest.raises(ValueError):
            ops.kv8_attention(**{**good, **bad})
    for bad, needle in ((dict(window=4, causal=False), "causal"), (dict(window=2**31), "window"), (dict(window=4, sinks=-1), "sinks"),
                        (dict(window=4, sinks=2**31), "sinks")):
        with pytest.raises(ffi.CastForgeHipError, match=needle):
            ops.kv8_attention(**{**good, **bad})
    assert ops.kv8_attention(q[:0], cache, table[:0], lens[:0]).shape == (0, 8, 128)
    w = torch.ones((3, 2, 8), device=cuda)
    assert torch.all(ops.kv8_attention(q, cache, table[:, :0], lens, weights=w) == 0) and torch.all(w == 1)
    nothing = ops.Kv8Cache.empty(0, 2, 16, 128, device=cuda)
    assert torch.all(ops.kv8_attention(q, nothing, table, lens, weights=w) == 0) and torch.all(w == 1)
