"""Attention over the paged 4-bit cache against float64 over the cache's own numbers.

Bound of an output: weights are rounded to f16 after their scale, two roundings of 2^-11 of each term, so
2^-10 of sum p |v|; f16 holds no number below 2^-25, where the largest weights are above 2^7 times their scale's
mantissa: up to 15 2^-31 of the largest p s a token, s the scale of its values; scores are f32 sums of d exact products and a scale, (d + 8) 2^-24 of scale * sum |q k| each,
which moves a weight by as much of itself, and so the output by twice that of sum p |v|, and the logarithm of
the sum by as much; a bf16 output rounds by 2^-9 of itself."""
import ctypes
import math

import numpy as np
import pytest
import torch

from castforge_amd import ffi, ops

pytestmark = pytest.mark.gpu


def _cache(seed, pages, heads, page, d, group, cuda, spread=0.3, base=0.25):
    g = torch.Generator(device=cuda).manual_seed(seed)
    shape, t = (pages, heads, page), []
    for _ in range(2):
        t.append(torch.randint(-2**31, 2**31, shape + (d // 8,), generator=g, device=cuda, dtype=torch.int32))
        s = (base * torch.exp(spread * torch.randn(shape + (d // group,), generator=g, device=cuda))).clamp(max=60000).half()
        z = torch.randint(4, 12, shape + (d // group,), generator=g, device=cuda, dtype=torch.int32)
        t.append((s.view(torch.int16).to(torch.int32) & 0xFFFF) | (z << 16))
    return ops.Kv4Cache(*t, group=group)


def _numbers(codes, groups, group):
    shift = 4 * torch.arange(8, device=codes.device, dtype=torch.int32)
    q = ((codes[..., None] >> shift) & 15).flatten(-2).double()
    s = groups.to(torch.int16).view(torch.float16).double().repeat_interleave(group, -1)
    return (q - ((groups >> 16) & 15).double().repeat_interleave(group, -1)) * s


def _reference(q, cache, table, kv_lens, q_lens, causal, scale):
    """(out, lse, bound) in float64, a sequence at a time."""
    ratio = q.shape[1] // cache.kv_heads
    outs, lses, bounds, moved, first = [], [], [], [], 0
    page = cache.page_size
    for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        kv = min(max(kv, 0), table.shape[1] * page)
        ids = table[b, :-(-kv // page)].long()
        ok = ((ids >= 0) & (ids < cache.num_pages)).repeat_interleave(page)[:kv]
        ids = ids.clamp(0, max(cache.num_pages - 1, 0))
        k, v = (_numbers(c[ids], g[ids], cache.group).transpose(0, 1).flatten(1, 2)[:, :kv]
                for c, g in ((cache.k_codes, cache.k_groups), (cache.v_codes, cache.v_groups)))
        x = q[first:first + n].double()
        first += n
        seen = torch.arange(kv, device=q.device)[None] <= (torch.arange(n, device=q.device)[:, None] + kv - n if causal else kv)
        seen = seen & ok[None]
        for h in range(q.shape[1]):
            kk, vv = k[h // ratio], v[h // ratio]
            vv = torch.where(ok[:, None], vv, 0.0)
            kk = torch.where(ok[:, None], kk, 0.0)
            s = (x[:, h] @ kk.t() * scale).masked_fill(~seen, -math.inf)
            lse = torch.logsumexp(s, 1) if kv else torch.full((n,), -math.inf, dtype=torch.float64, device=q.device)
            p = torch.where(seen, torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse)[:, None]), 0.0)
            o = p @ vv
            mag = (x[:, h].abs() @ kk.abs().t() * abs(scale)).masked_fill(~seen, 0).amax(1) if kv else torch.zeros_like(lse)
            pv = p @ vv.abs()
            e = 2.0 ** -10 + 2 * (cache.head_dim + 8) * 2.0 ** -24 * mag[:, None]
            moved.append((cache.head_dim + 8) * 2.0 ** -24 * mag)
            under = kv * 15 * 2.0 ** -31 * (p * vv.abs().amax(1)).amax(1, keepdim=True) if kv else torch.zeros_like(pv)
            outs.append(o), lses.append(lse), bounds.append(e * pv * 1.1 + under + 2.0 ** -8 * o.abs() + 1e-30)
    hq = q.shape[1]

    def together(parts):
        res, i = [], 0
        for n in q_lens:
            res.append(torch.stack(parts[i:i + hq], 1))
            i += hq
        return torch.cat(res)

    return together(outs), together(lses), together(bounds), together(moved)


def _table(seed, need, pages, cols, cuda):
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    t = torch.full((len(need), cols), 2**31 - 1, dtype=torch.int32)  # entries past the last page are never read
    i = 0
    for b, n in enumerate(need):
        t[b, :n] = perm[i:i + n]
        i += n
    return t.to(cuda)


def _run(cuda, q_lens, kv_lens, hkv, ratio, d, group, page, causal=True, seed=0, scale=None, extra_cols=0, varlen=None, q_scale=1.5, **cache_args):
    need = [-(-max(kv, 0) // page) for kv in kv_lens]
    pages = sum(need) + 2
    cache = _cache(seed, pages, hkv, page, d, group, cuda, **cache_args)
    table = _table(seed, need, pages, max(need + [0]) + extra_cols, cuda)
    g = torch.Generator(device=cuda).manual_seed(seed + 1)
    q = (q_scale * torch.randn((sum(q_lens), hkv * ratio, d), generator=g, device=cuda)).bfloat16()
    lens = torch.tensor(kv_lens, dtype=torch.int32, device=cuda)
    if varlen is None:
        varlen = any(n != 1 for n in q_lens)
    cu = torch.tensor(np.cumsum([0] + q_lens), dtype=torch.int32, device=cuda) if varlen else None
    got, lse = ops.kv4_attention(q, cache, table, lens, cu_q=cu, causal=causal, scale=scale, return_lse=True)
    want, want_lse, bound, moved = _reference(q, cache, table, kv_lens, q_lens, causal, d ** -0.5 if scale is None else scale)
    far = ((got.double() - want).abs() > bound).sum().item()
    assert far == 0, f"{far} of {want.numel()} outputs past the bound, worst {((got.double() - want).abs() / bound).max().item():.2f}"
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty) and torch.all(got[empty] == 0)
    assert torch.all((lse.double() - want_lse)[~empty].abs() <= 1e-5 * (1 + want_lse[~empty].abs()) + moved[~empty])
    assert torch.equal(ops.kv4_attention(q, cache, table, lens, cu_q=cu, causal=causal, scale=scale), got)
    return q, cache, table, lens, cu, got


SHAPES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("hkv,ratio,page,kv_lens", [
    (8, 4, 16, [1]), (1, 1, 16, [15, 16, 17]), (2, 8, 64, [777, 1, 0, 64, 63, 65]), (4, 7, 32, [31, 32, 33, 500]),
    (1, 16, 128, [2000, 3]), (3, 20, 16, [130, 257]), (2, 3, 4096, [5000, 4096, 4095]), (8, 1, 16, [100] * 40)])
def test_one_query_each(cuda, d, group, hkv, ratio, page, kv_lens):
    _run(cuda, [1] * len(kv_lens), kv_lens, hkv, ratio, d, group, page, seed=hkv * 10 + ratio)


@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("q_lens,kv_lens", [([1] * 4, [100, 1, 0, 700]), ([1] * 3, [513, 1024, 97]), ([3, 1, 4], [300, 129, 1000])])
@pytest.mark.parametrize("cols", [0, 90])
def test_short_sequences(cuda, d, group, q_lens, kv_lens, cols):
    """In one launch or, with a table that has room for more, in splits and a join."""
    _run(cuda, q_lens, kv_lens, 4, 3, d, group, 16, seed=60, extra_cols=cols)


@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hkv,ratio,page,lens", [
    (2, 4, 16, [(5, 100), (1, 33), (3, 3)]), (1, 8, 32, [(17, 17), (64, 200), (2, 1000)]), (4, 1, 64, [(130, 130), (33, 65)]),
    (2, 3, 16, [(100, 612), (0, 50), (7, 7)]), (1, 7, 128, [(257, 300)])])
def test_several_queries(cuda, d, group, causal, hkv, ratio, page, lens):
    _run(cuda, [q for q, _ in lens], [kv for _, kv in lens], hkv, ratio, d, group, page, causal, seed=hkv + ratio)


@pytest.mark.parametrize("d,group", [(64, 32), (128, 128)])
@pytest.mark.parametrize("lens", [[(8, 3)], [(40, 7), (3, 0), (2, 5)], [(300, 100)], [(1, 0), (1, 4)]])
def test_rows_that_see_nothing(cuda, d, group, lens):
    """More queries than cached tokens: the first ones' masks leave nothing; so does an empty sequence."""
    _run(cuda, [q for q, _ in lens], [kv for _, kv in lens], 2, 4, d, group, 16, True, seed=3, varlen=True)
    _run(cuda, [q for q, _ in lens], [kv for _, kv in lens], 2, 4, d, group, 16, False, seed=4, varlen=True)


@pytest.mark.parametrize("d,group", SHAPES)
def test_long_context_and_prompt(cuda, d, group):
    _run(cuda, [1], [20011], 2, 4, d, group, 64, seed=5)
    _run(cuda, [1, 1, 1], [9000, 10, 4001], 1, 5, d, group, 16, seed=6, extra_cols=100)
    _run(cuda, [700, 129], [700, 1500], 2, 4, d, group, 64, seed=7)
    _run(cuda, [6, 2], [6000, 3000], 2, 4, d, group, 32, seed=8)


@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hkv,ratio,page,lens", [
    (8, 4, 64, [(1500, 1500), (700, 1203), (1, 65)]), (4, 8, 16, [(1637, 1637), (3, 1), (0, 9), (60, 20)]),
    (1, 40, 128, [(1301, 1400)]), (16, 1, 32, [(3100, 3112)]), (8, 3, 4096, [(1, 5000), (2100, 2099)])])
def test_whole_prompts(cuda, d, group, causal, hkv, ratio, page, lens):
    """Enough rows for every wave to have its own."""
    q, cache, table, kv, cu, ref = _run(cuda, [n for n, _ in lens], [k for _, k in lens], hkv, ratio, d, group, page, causal, seed=30 + hkv)
    last = lens[0][1] - 1
    if lens[0][1] % page:  # what lies past the first sequence's last token changes nothing
        at = table[0, last // page].item()
        for g in (cache.k_groups, cache.v_groups):
            g[at, :, lens[0][1] % page:] = torch.tensor([0x7E00] * (d // group), dtype=torch.int32, device=cuda)
        assert torch.equal(ops.kv4_attention(q, cache, table, kv, cu_q=cu, causal=causal), ref)
    t = table.clone()
    t[0, 0] = -1  # a page of no cache is left out
    got = ops.kv4_attention(q, cache, t, kv, cu_q=cu, causal=causal)
    want, _, bound, _ = _reference(q, cache, t, [k for _, k in lens], [n for n, _ in lens], causal, d ** -0.5)
    assert torch.all((got.double() - want).abs() <= bound)


@pytest.mark.parametrize("d,group", [(64, 64), (128, 32), (128, 128)])
@pytest.mark.parametrize("spread,base,q_scale", [(3.0, 0.25, 1.5), (0.3, 2000.0, 1e-5), (0.3, 1e-5, 1e4), (0.3, 0.25, 30.0)])
def test_whole_prompts_scales_of_any_size(cuda, d, group, spread, base, q_scale):
    _run(cuda, [1300, 300], [1300, 700], 8, 4, d, group, 16, seed=40, spread=spread, base=base, q_scale=q_scale)


@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
def test_prompts_of_many_heads(cuda, d, group, causal):
    """Enough row tiles for the largest workgroups."""
    _run(cuda, [1101, 30, 0, 300], [1101, 500, 9, 299], 8, 16, d, group, 16, causal, seed=50)


@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("q_lens,kv_lens", [([1637, 30], [1637, 500]), ([20, 9], [300, 700]), ([200, 9], [300, 700])])
@pytest.mark.parametrize("top", [0, 60, 120])
def test_rows_of_any_size(cuda, d, group, q_lens, kv_lens, top):
    """Queries of a tile from 2^-40 to 2^3, of zeros, and a few 2^top times that: a row's products do not suffer from a larger row's."""
    cache = _cache(51, 300, 8, 16, d, group, cuda)
    table = _table(51, [-(-n // 16) for n in kv_lens], 300, -(-max(kv_lens) // 16), cuda)
    g = torch.Generator(device=cuda).manual_seed(52)
    shape = (sum(q_lens), 32, 1)
    q = torch.randn((*shape[:2], d), generator=g, device=cuda) * torch.exp2(torch.randint(-40, 4, shape, generator=g, device=cuda).float())
    u = torch.rand(shape, generator=g, device=cuda)
    q = (q * (u > 0.1) * torch.where(u > 0.97, 2.0**top, 1.0)).bfloat16()
    lens = torch.tensor(kv_lens, dtype=torch.int32, device=cuda)
    cu = torch.tensor(np.cumsum([0] + q_lens), dtype=torch.int32, device=cuda)
    for scale in (d ** -0.5, 2.0 ** 20):  # the second makes scores of the small rows, and one heavy token of the large ones'
        got, lse = ops.kv4_attention(q, cache, table, lens, cu_q=cu, scale=scale, return_lse=True)
        want, want_lse, bound, moved = _reference(q, cache, table, kv_lens, q_lens, True, scale)
        near = 2 * moved < 1  # else the scores' own rounding decides which token is the heavy one
        assert torch.all(((got.double() - want).abs() <= bound)[near])
        assert torch.all(((lse.double() - want_lse).abs() <= 1e-5 * (1 + want_lse.abs()) + moved)[near])
        assert near.double().mean() > 0.5


@pytest.mark.parametrize("d,group", [(64, 64), (128, 32), (128, 128)])
@pytest.mark.parametrize("q_lens", [[1, 1], [40, 90]])
def test_scales_of_any_size(cuda, d, group, q_lens):
    """Values near f16's ends, scales that differ by orders of magnitude from token to token, sharp and flat scores,
    large and small queries."""
    kv = [300, 1111]
    _run(cuda, q_lens, kv, 2, 2, d, group, 16, seed=9, spread=3.0)
    _run(cuda, q_lens, kv, 2, 2, d, group, 16, seed=10, base=2000.0, q_scale=1e-5)
    _run(cuda, q_lens, kv, 2, 2, d, group, 16, seed=11, base=1e-5, q_scale=1e4)
    _run(cuda, q_lens, kv, 2, 2, d, group, 16, seed=12, q_scale=30.0)
    _run(cuda, q_lens, kv, 2, 2, d, group, 16, seed=13, q_scale=1e30, scale=1e-31)
    _run(cuda, q_lens, kv, 2, 2, d, group, 16, seed=14, scale=0.0)
    _run(cuda, q_lens, kv, 2, 2, d, group, 16, seed=15, scale=-0.2)


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [20, 3, 150]])
def test_masked_places_may_hold_anything(cuda, q_lens):
    """NaN and inf scales in the places past a sequence's length, and pages outside the cache, change nothing."""
    kv = [100, 37, 1000]
    q, cache, table, lens, cu, ref = _run(cuda, q_lens, kv, 2, 4, 128, 64, 64, seed=16, varlen=True)
    for b, n in enumerate(kv):
        last = table[b, n // 64].item() if n % 64 else None
        if last is not None:
            for g in (cache.k_groups, cache.v_groups):
                g[last, :, n % 64:] = torch.tensor([0x7E00, 0x7C00], dtype=torch.int32, device=cuda)  # NaN, inf
    assert torch.equal(ops.kv4_attention(q, cache, table, lens, cu_q=cu), ref)
    for bad in (-1, cache.num_pages, 2**31 - 1):
        t = table.clone()
        t[2, 3] = bad
        got = ops.kv4_attention(q, cache, t, lens, cu_q=cu)
        want, _, bound, _ = _reference(q, cache, t, kv, q_lens, True, 128 ** -0.5)
        assert torch.all((got.double() - want).abs() <= bound)


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [700, 129]), ([1, 1], [90, 3000]), ([500, 40], [700, 129]), ([900, 300], [900, 300])])
def test_offsets_past_32_bits(cuda, q_lens, kv_lens):
    """Pages at the ends of a cache of more than 2^32 words of codes give the bits of a small cache's."""
    heads, page, d, pages = 16, 128, 128, 140000  # 18 GB of codes each
    small = _cache(70, 40, heads, page, d, 128, cuda)
    big = ops.Kv4Cache(*(torch.empty((pages, *t.shape[1:]), dtype=torch.int32, device=cuda)
                         for t in (small.k_codes, small.k_groups, small.v_codes, small.v_groups)))
    at = torch.tensor([i if i % 2 else pages - 1 - i for i in range(40)], device=cuda)
    for a, b in ((big.k_codes, small.k_codes), (big.k_groups, small.k_groups), (big.v_codes, small.v_codes), (big.v_groups, small.v_groups)):
        a[at] = b
    table = _table(71, [-(-n // page) for n in kv_lens], 40, -(-max(kv_lens) // page), cuda)
    far = torch.where(table < 40, at[table.clamp(max=39).long()].int(), table)
    g = torch.Generator(device=cuda).manual_seed(72)
    q = torch.randn((sum(q_lens), 4 * heads, d), generator=g, device=cuda).bfloat16()
    lens = torch.tensor(kv_lens, dtype=torch.int32, device=cuda)
    cu = None if max(q_lens) == 1 else torch.tensor(np.cumsum([0] + q_lens), dtype=torch.int32, device=cuda)
    got = ops.kv4_attention(q, big, far, lens, cu_q=cu)
    assert torch.equal(got, ops.kv4_attention(q, small, table, lens, cu_q=cu)) and torch.isfinite(got).all()


def test_length_past_the_table_is_cut(cuda):
    q, cache, table, lens, _, _ = _run(cuda, [1], [160], 2, 4, 128, 128, 16, seed=17)
    assert torch.equal(ops.kv4_attention(q, cache, table, lens + 1000), ops.kv4_attention(q, cache, table, lens))
    assert torch.all(ops.kv4_attention(q, cache, table, lens - 1000) == 0)


@pytest.mark.parametrize("tokens", [3, 200])
def test_slices_of_a_projection(cuda, tokens):
    """Queries with a token stride of their own give the bits of contiguous ones."""
    q, cache, table, lens, cu, ref = _run(cuda, [tokens], [tokens + 50], 2, 3, 64, 32, 16, seed=18, varlen=True)
    wide = torch.full((tokens, 6 + 4, 64), float("nan"), device=cuda, dtype=torch.bfloat16)
    wide[:, :6] = q
    assert torch.equal(ops.kv4_attention(wide[:, :6], cache, table, lens, cu_q=cu), ref)


@pytest.mark.parametrize("q_lens,kv", [([1] * 5, [3000, 1, 77, 900, 12]), ([33, 200], [900, 200])])
def test_same_bits_other_stream_and_graph(cuda, q_lens, kv):
    q, cache, table, lens, cu, ref = _run(cuda, q_lens, kv, 4, 4, 128, 64, 16, seed=19)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = ops.kv4_attention(q, cache, table, lens, cu_q=cu)
        y2 = ops.kv4_attention(q, cache, table, lens, cu_q=cu)
    s.synchronize()
    assert torch.equal(y, ref) and torch.equal(y2, ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.kv4_attention(q, cache, table, lens, cu_q=cu)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
        assert torch.equal(ops.kv4_attention(q, cache, table, lens, cu_q=cu), ref)


def test_rows_of_no_sequence_are_left_alone(cuda):
    """cu_q that ends before the last row: that row is not written (its memory comes from a block set to ones)."""
    q, cache, table, lens, cu, ref = _run(cuda, [3, 2], [50, 60], 2, 4, 128, 128, 16, seed=20)
    more = torch.cat([q, q[:1]])
    got = ops.kv4_attention(more, cache, table, lens, cu_q=cu)
    assert torch.equal(got[:5], ref)


def test_refusals(cuda):
    q, cache, table, lens, _, _ = _run(cuda, [1, 1], [50, 60], 2, 4, 128, 128, 16, seed=21)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda)
    for bad in (dict(q=q.float()), dict(q=q[:, :7]), dict(q=q[..., :64]), dict(page_table=table.long()), dict(page_table=table[0]),
                dict(kv_lens=lens.long()), dict(kv_lens=lens[:1]), dict(cu_q=cu[:2]), dict(cu_q=cu.long()), dict(q=q[:1]),
                dict(q=q.cpu()), dict(q=torch.zeros((2, 8, 256), device=cuda, dtype=torch.bfloat16)[..., ::2])):
        with pytest.raises((ValueError, ffi.CastForgeHipError)):
            ops.kv4_attention(**{"q": q, "cache": cache, "page_table": table, "kv_lens": lens, **bad})
    many = torch.zeros((2, 130, 128), device=cuda, dtype=torch.bfloat16)
    with pytest.raises(ffi.CastForgeHipError, match="q_heads"):
        ops.kv4_attention(many, cache, table, lens)


def test_empty(cuda):
    _, cache, table, lens, _, _ = _run(cuda, [1], [50], 2, 4, 128, 128, 16, seed=22)
    q = torch.zeros((0, 8, 128), device=cuda, dtype=torch.bfloat16)
    assert ops.kv4_attention(q, cache, table[:0], lens[:0]).shape == (0, 8, 128)
    one = torch.ones((1, 8, 128), device=cuda, dtype=torch.bfloat16)
    assert torch.all(ops.kv4_attention(one, cache, table[:, :0], lens) == 0)


@pytest.mark.parametrize("heads,pages", [(1, 524272), (2, 524280), (4, 524284), (8, 524286), (1, 524287), (8, 524287)])
def test_lengths_up_to_the_limit(cuda, heads, pages):
    """Tables near 2^31 - 4096 tokens, whose entries but the last name a page of zero keys: the last page's keys, of score 60, take
    all of the weight but 2^31 exp(-60), and so the output is the mean of its values, for whichever split holds it."""
    page, d = 4096, 64
    cache = _cache(80, 2, heads, page, d, 64, cuda)
    cache.k_groups.fill_(0x3C00 | (7 << 16))  # scale 1, zero point 7
    cache.k_codes[0] = 0x77777777             # zeros
    cache.k_codes[1] = -0x77777778            # 0x88888888: ones
    table = torch.zeros((1, pages), dtype=torch.int32, device=cuda)
    table[0, -1] = 1
    q = torch.ones((1, heads, d), dtype=torch.bfloat16, device=cuda)
    lens = torch.tensor([pages * page], dtype=torch.int32, device=cuda)
    got, lse = ops.kv4_attention(q, cache, table, lens, scale=60 / 64, return_lse=True)
    v = _numbers(cache.v_codes[1], cache.v_groups[1], 64)
    want, mag = v.mean(1), v.abs().mean(1)
    # scores are exact here; the other bounds as above
    under = page * 15 * 2.0 ** -31 * (v.abs().amax() / page)
    assert torch.all((got[0].double() - want).abs() <= 1.1 * 2.0 ** -10 * mag + under + 2.0 ** -8 * want.abs())
    assert torch.all((lse.double() - (60 + math.log(page))).abs() <= 1e-5 * 70)


@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [777, 40]), ([3, 40], [300, 90]), ([1637, 30], [1637, 500])])
@pytest.mark.parametrize("sign", ["both", "below"])
def test_negative_scales(cuda, d, group, q_lens, kv_lens, sign):
    """Groups whose scale is negative, up to 2^9: some of a token's, or all of them."""
    pages, page = [-(-n // 16) for n in kv_lens], 16
    cache = _cache(81, sum(pages), 8, page, d, group, cuda, base=100.0, spread=0.5)
    g = torch.Generator(device=cuda).manual_seed(82)
    for t in (cache.k_groups, cache.v_groups):
        t |= 0x8000 if sign == "below" else torch.where(torch.rand(t.shape, generator=g, device=cuda) < 0.5, 0x8000, 0)
    table = _table(83, pages, sum(pages), max(pages), cuda)
    q = (1e-3 * torch.randn((sum(q_lens), 32, d), generator=g, device=cuda)).bfloat16()
    lens = torch.tensor(kv_lens, dtype=torch.int32, device=cuda)
    cu = torch.tensor(np.cumsum([0] + q_lens), dtype=torch.int32, device=cuda)
    got = ops.kv4_attention(q, cache, table, lens, cu_q=cu)
    want, _, bound, _ = _reference(q, cache, table, kv_lens, q_lens, True, d ** -0.5)
    assert torch.all((got.double() - want).abs() <= bound)


def test_more_sequences_than_a_launch_of_workgroups(cuda):
    """2^21 sequences and a few: with eight heads of keys more than 2^32 work-items."""
    b, heads, d = 2**21 + 5, 8, 64
    cache = _cache(84, 3, heads, 16, d, 64, cuda)
    table = torch.zeros((b, 1), dtype=torch.int32, device=cuda)
    lens = torch.zeros(b, dtype=torch.int32, device=cuda)
    at = torch.tensor([0, 12345, 2**21 - 1, 2**21, 2**21 + 4], device=cuda)
    table[at, 0] = torch.tensor([0, 1, 2, 1, 0], dtype=torch.int32, device=cuda)
    lens[at] = torch.tensor([3, 16, 9, 1, 15], dtype=torch.int32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(85)
    q = torch.ones((b, heads, d), dtype=torch.bfloat16, device=cuda)
    q[at] = torch.randn((5, heads, d), generator=g, device=cuda).bfloat16()
    got = ops.kv4_attention(q, cache, table, lens)
    assert torch.equal(got[at], ops.kv4_attention(q[at], cache, table[at], lens[at]))
    got[at] = 0
    assert not got.any()


@pytest.mark.parametrize("q_lens,kv_lens", [
    ([1, 1, 1], [300, 17, 777]),         # one launch
    ([3, 1, 2], [50, 5000, 300]),        # splits and their join
    ([900, 1, 700], [900, 40, 800])])    # rows of each wave's own
def test_rows_of_no_sequence_keep_what_they_hold(cuda, q_lens, kv_lens):
    """Rows of out and lse past the last of cu_q, and all of them without a sequence, are not written; a caller's own buffers show it."""
    q, cache, table, lens, cu, _ = _run(cuda, q_lens, kv_lens, 8, 4, 128, 128, 16, seed=23, varlen=True)
    t, more = len(q), 5
    wide = torch.cat([q, torch.ones((more, *q.shape[1:]), dtype=q.dtype, device=cuda)])
    for b in (len(q_lens), 0):
        out = torch.full_like(wide, 7.0)
        lse = torch.full(wide.shape[:2], 7.0, device=cuda)
        size = ctypes.c_int64()
        ffi.call("castforge_hip_kv4_attention_workspace", cache._ref, t + more, 32, b, table.shape[1], 1, ctypes.byref(size))
        ws = torch.empty(max(size.value, 1), dtype=torch.uint8, device=cuda)
        ffi.call("castforge_hip_kv4_attention", cache._ref, wide.data_ptr(), 32 * 128, t + more, 32, b, cu.data_ptr(), table.data_ptr(), table.shape[1],
                 lens.data_ptr(), 1, 128 ** -0.5, out.data_ptr(), lse.data_ptr(), ws.data_ptr(), size.value, torch.cuda.current_stream().cuda_stream)
        n = t if b else 0
        assert torch.all(out[n:] == 7) and torch.all(lse[n:] == 7)
        if b:
            want, want_lse, bound, moved = _reference(q, cache, table, kv_lens, q_lens, True, 128 ** -0.5)
            assert torch.all((out[:t].double() - want).abs() <= bound)
            assert torch.all((lse[:t].double() - want_lse).abs() <= 1e-5 * (1 + want_lse.abs()) + moved)


@pytest.mark.parametrize("q_lens,kv_lens", [([1], [131072]), ([1, 1], [99991, 70001]), ([5], [60013])])
def test_long_caches(cuda, q_lens, kv_lens):
    _run(cuda, q_lens, kv_lens, 4, 7, 128, 32, 64, seed=24)
