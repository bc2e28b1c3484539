"""Eviction from the paged 8-bit cache: which tokens stay, against a sort, and what their new pages hold, bit for bit against a
restatement in f32 on the CPU; all other pages keep their bits."""
import math

import pytest
import torch

from castforge_amd import ffi, ops

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _kept(w, kv, keep, sinks, recent):
    """w: a list of at least kv numbers."""
    if kv <= keep:
        return list(range(kv))
    always = set(range(sinks)) | set(range(kv - recent, kv))
    rest = sorted((t for t in range(kv) if t not in always), key=lambda t: (math.isnan(w[t]), 0.0 if math.isnan(w[t]) else -w[t], t))
    return sorted(always | set(rest[:keep - sinks - recent]))


def _moved(codes, scales, table, kept, page, h):
    """(codes, scale) of a page's kept tokens."""
    rows, s = [], []
    for t in kept:
        p = int(table[t // page])
        ok = 0 <= p < codes.shape[0]
        rows.append(codes[p, h, t % page] if ok else torch.zeros(codes.shape[3], dtype=torch.uint8))
        s.append(scales[p, h] if ok else torch.tensor(0.0))
    rows, s = torch.stack(rows), torch.stack(s)
    top = s.max() if s.max() > 0 else torch.tensor(1.0)
    new = (rows.view(F8).float() * (s / top)[:, None]).to(F8).view(torch.uint8)
    return torch.where((s == top)[:, None], rows, new), top


def _run(cuda, lens, keep, heads, d, page, sinks=0, recent=0, seed=0, weights=None, cols_of_weights=None, power=True, extra=0, bad=False):
    g = torch.Generator().manual_seed(seed)
    cols, new_cols = max([-(-max(kv, 0) // page) for kv in lens] + [0]) + extra, -(-keep // page) + extra
    b, need = len(lens), sum(-(-max(kv, 0) // page) for kv in lens)
    pages = need + b * new_cols + 2
    state = []
    for _ in range(2):
        c = torch.randint(0, 256, (pages, heads, page, d), generator=g, dtype=torch.uint8)
        s = torch.randint(-9, -5, (pages, heads), generator=g).float()
        state += [torch.where(c & 0x7F == 0x7F, torch.zeros_like(c), c), torch.exp2(s if power else s + torch.rand((pages, heads), generator=g))]
    at = torch.randperm(pages, generator=g).int()
    table, i = torch.full((b, cols), 2**31 - 1, dtype=torch.int32), 0
    for r, kv in enumerate(lens):
        n = -(-max(kv, 0) // page)
        table[r, :n] = at[i:i + n]
        i += n
    new = at[need:need + b * new_cols].view(b, new_cols).clone()
    if bad:
        table[0, 1], new[-1, 0] = -5, pages
    wcols = cols * page if cols_of_weights is None else cols_of_weights
    if weights is None:
        weights = torch.exp(2 * torch.randn((b, heads, wcols), generator=g))
        weights[torch.rand(weights.shape, generator=g) < 0.2] = 0.0
    else:
        weights = weights(b, heads, wcols, g)
    cache = ops.Kv8Cache(*[t.to(cuda) for t in state])
    kept, new_lens, new_weights = ops.kv8_evict(cache, table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda), weights.to(cuda), keep, new.to(cuda),
                                                sinks=sinks, recent=recent)
    want = [t.clone() for t in state]
    for r, kv in enumerate(lens):
        kv = min(max(kv, 0), cols * page)
        n = min(kv, keep)
        assert new_lens[r].item() == n
        for h in range(heads):
            w = (weights[r, h].tolist() + [0.0] * kv)[:max(kv, wcols)]
            mine = _kept(w, kv, keep, sinks, recent)
            assert kept[r, h].tolist() == mine + [-1] * (keep - n), (r, h)
            expect = torch.tensor([w[t] for t in mine] + [0.0] * (keep - n))
            assert torch.equal(torch.nan_to_num(new_weights[r, h].cpu(), nan=-3.0), torch.nan_to_num(expect, nan=-3.0))
            for c in range(-(-n // page)):
                to = int(new[r, c])
                if not 0 <= to < pages:
                    continue
                part = mine[c * page:(c + 1) * page]
                for k in (0, 2):
                    want[k][to, h, :len(part)], want[k + 1][to, h] = _moved(state[k], state[k + 1], table[r], part, page, h)
    for got, t in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), want):
        assert torch.equal(got.cpu(), t)
    return kept


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_pages_and_head_sizes(cuda, d, page):
    _run(cuda, [300, 100, 7, 513], 100, 2, d, page, sinks=4, recent=30, seed=page)


@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (2, 1, 1), (17, 0, 0), (17, 17, 0), (17, 0, 17), (64, 10, 54), (64, 0, 63), (128, 4, 20),
                                               (1000, 4, 20), (1023, 1000, 3), (2000, 0, 0)])
def test_budgets(cuda, keep, sinks, recent):
    _run(cuda, [1024, 1, 17, 65, 1025, 0, 999], keep, 2, 64, 16, sinks=sinks, recent=recent, seed=keep)


@pytest.mark.parametrize("kind", ["equal", "zero", "two", "rising", "falling", "tiny", "nan", "infinite", "negative", "few bits"])
def test_weights_of_every_kind(cuda, kind):
    def weights(b, h, n, g):
        t = torch.arange(n).float().expand(b, h, n).clone()
        r = torch.rand((b, h, n), generator=g)
        return {"equal": torch.full_like(t, 0.3), "zero": torch.where(r < 0.5, 0.0, -0.0), "two": torch.where(r < 0.3, 1.0, 2.0), "rising": t, "falling": -t,
                "tiny": r * 1e-40, "nan": torch.where(r < 0.8, math.nan, r), "infinite": torch.where(r < 0.4, math.inf, torch.where(r < 0.9, -math.inf, r)),
                "negative": r - 0.5, "few bits": 1 + torch.floor(r * 4) * 2.0 ** -23}[kind]

    _run(cuda, [3000, 700, 4100], 600, 2, 64, 64, sinks=2, recent=100, seed=1, weights=weights)
    _run(cuda, [3000, 700, 4100], 600, 1, 64, 64, seed=1, weights=weights)


def test_long_sequences(cuda):
    _run(cuda, [70000], 1000, 1, 64, 256, sinks=4, recent=64, seed=1)
    _run(cuda, [20000, 4097, 4096, 4095], 4000, 1, 64, 128, seed=2)


def test_many_sequences(cuda):
    _run(cuda, [(37 * i) % 90 for i in range(70)], 33, 3, 64, 16, sinks=1, recent=5, seed=3)


def test_lengths_past_the_table_and_weights_of_fewer_tokens(cuda):
    _run(cuda, [100, -3, 40], 20, 2, 64, 16, seed=1, cols_of_weights=50, extra=2)
    _run(cuda, [100, 64], 70, 2, 64, 16, seed=1, cols_of_weights=0, recent=10)
    _run(cuda, [100, 64], 70, 2, 64, 16, seed=1, cols_of_weights=1000, recent=10)


def test_scales_that_are_no_powers_of_two(cuda):
    _run(cuda, [200, 64], 70, 2, 128, 16, seed=1, power=False)


def test_pages_outside_the_cache(cuda):
    _run(cuda, [100, 64], 40, 2, 64, 16, seed=1, bad=True)


def test_a_table_shorter_than_the_lengths(cuda):
    cache = ops.Kv8Cache.empty(8, 1, 16, 64, device=cuda)
    i32 = dict(dtype=torch.int32, device=cuda)
    kept, lens, _ = ops.kv8_evict(cache, torch.tensor([[0, 1]], **i32), torch.tensor([1000], **i32), torch.arange(40.0, device=cuda).view(1, 1, 40), 20, torch.tensor([[2, 3]], **i32))
    assert kept[0, 0].tolist() == list(range(12, 32)) and lens.item() == 20
    kept, lens, w = ops.kv8_evict(cache, torch.empty((1, 0), **i32), torch.tensor([1000], **i32), torch.ones((1, 1, 40), device=cuda), 20, torch.tensor([[2, 3]], **i32))
    assert torch.all(kept == -1) and lens.item() == 0 and torch.all(w == 0)


def test_offsets_past_32_bits(cuda):
    page, heads, d = 256, 4, 128
    pages = 2**32 // (page * heads * d) + 8
    big = ops.Kv8Cache(*[t for _ in range(2) for t in (torch.empty((pages, heads, page, d), dtype=torch.uint8, device=cuda), torch.ones((pages, heads), device=cuda))])
    small = ops.Kv8Cache.empty(8, heads, page, d, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    for i, far in ((0, pages - 1), (1, 3)):
        for a, b in ((small.k_codes, big.k_codes), (small.v_codes, big.v_codes)):
            a[i] = torch.randint(0, 127, a[i].shape, generator=g, device=cuda, dtype=torch.uint8)
            b[far] = a[i]
    i32 = dict(dtype=torch.int32, device=cuda)
    w, lens = torch.rand((1, heads, 512), generator=g, device=cuda), torch.tensor([500], **i32)
    a = ops.kv8_evict(big, torch.tensor([[pages - 1, 3]], **i32), lens, w, 300, torch.tensor([[pages - 2, 4]], **i32))
    b = ops.kv8_evict(small, torch.tensor([[0, 1]], **i32), lens, w, 300, torch.tensor([[2, 3]], **i32))
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    for x, y in ((big.k_codes, small.k_codes), (big.v_codes, small.v_codes)):
        assert torch.equal(x[pages - 2], y[2]) and torch.equal(x[4, :, :44], y[3, :, :44])


def test_captured_evictions_follow_their_lists(cuda):
    g = torch.Generator(device=cuda).manual_seed(1)
    cache = ops.Kv8Cache.empty(40, 2, 16, 64, device=cuda)
    for t in (cache.k_codes, cache.v_codes):
        t.copy_(torch.randint(0, 127, t.shape, generator=g, device=cuda, dtype=torch.uint8))
    table, new = torch.arange(20, dtype=torch.int32, device=cuda).view(1, 20), torch.arange(20, 24, dtype=torch.int32, device=cuda).view(1, 4)
    other = torch.arange(30, 34, dtype=torch.int32, device=cuda).view(1, 4)
    w, lens = torch.rand((1, 2, 320), generator=g, device=cuda), torch.tensor([300], dtype=torch.int32, device=cuda)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.kv8_evict(cache, table, lens, w, 60, new)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.kv8_evict(cache, table, lens, w, 60, new)
    for kv in (300, 61, 60, 5, 320):
        lens.fill_(kv), w.copy_(torch.rand(w.shape, generator=g, device=cuda))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, ops.kv8_evict(cache, table, lens, w, 60, other)):
            assert torch.equal(a, b)
        n = -(-min(kv, 60) // 16)
        rows = torch.cat([torch.arange(min(16, min(kv, 60) - 16 * c), device=cuda) + 16 * c for c in range(n)])
        a, b = (ops.kv8_gather(cache, t[0, rows // 16].long() * 16 + rows % 16, torch.float32) for t in (new, other))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_refusals_and_empty_calls(cuda):
    cache = ops.Kv8Cache.empty(8, 2, 16, 64, device=cuda)
    i32 = dict(dtype=torch.int32, device=cuda)
    good = dict(cache=cache, page_table=torch.tensor([[0, 1]], **i32), kv_lens=torch.tensor([20], **i32), weights=torch.ones((1, 2, 32), device=cuda), keep=10,
                new_table=torch.tensor([[2]], **i32))
    ops.kv8_evict(**good)
    w = good["weights"]
    for bad in (dict(weights=w.double()), dict(weights=w[:, :1]), dict(weights=w[0]), dict(weights=w.cpu()), dict(weights=w.repeat(1, 1, 2)[..., ::2]), dict(keep=0),
                dict(new_table=good["new_table"].long()), dict(new_table=good["new_table"][0]), dict(kv_lens=torch.ones(2, **i32)), dict(page_table=torch.zeros((2, 2), **i32))):
        with pytest.raises(ValueError):
            ops.kv8_evict(**{**good, **bad})
    for bad, needle in ((dict(sinks=-1), "sinks"), (dict(recent=-1), "recent"), (dict(sinks=6, recent=5), "together"), (dict(keep=17), "new_table")):
        with pytest.raises(ffi.CastForgeHipError, match=needle):
            ops.kv8_evict(**{**good, **bad})
    none = ops.kv8_evict(cache, torch.empty((0, 2), **i32), torch.empty(0, **i32), torch.empty((0, 2, 5), device=cuda), 10, torch.empty((0, 1), **i32))
    assert none[0].shape == (0, 2, 10) and none[1].shape == (0,) and none[2].shape == (0, 2, 10)
    nothing = ops.Kv8Cache.empty(0, 2, 16, 64, device=cuda)
    kept, lens, _ = ops.kv8_evict(**{**good, "cache": nothing})
    assert lens.item() == 10 and kept[0, 0].tolist() == list(range(10))
