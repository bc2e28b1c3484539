"""The operators of the paged 8-bit cache one after another, as a server runs them: prompts appended, attended and observed, cut to
a budget, then tokens appended behind what was kept, each way against float64 over the cache's own numbers; and the example of a
layer that does so, by calls and by graph replay."""
import importlib.util
from pathlib import Path

import pytest
import torch

from castforge_amd import ops
from test_gpu_kv8_attention import _check, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,hkv,ratio,page,window,sinks", [(128, 2, 4, 16, None, 0), (64, 3, 1, 32, None, 0), (128, 1, 7, 64, 300, 4), (64, 2, 3, 16, 50, 20)])
def test_prompt_eviction_and_tokens(cuda, d, hkv, ratio, page, window, sinks):
    """After the eviction the cache holds exactly what it held of the kept tokens (scales of random numbers of one size are alike or a
    power of two apart, which rounds codes: so the attention is checked over what lies there now, and the kept rows against those before
    to a step of E4M3), and the attention over it is the softmax over those tokens."""
    prompts, keep, first, recent, tokens = [700, 37, 300], 128, 4, 24, 20
    g = torch.Generator(device=cuda).manual_seed(d + ratio)
    batch, hq, cols, new_cols = len(prompts), hkv * ratio, -(-max(prompts) // page), -(-(keep + tokens) // page)
    pages = torch.randperm(batch * (cols + new_cols), generator=g, device=cuda).int()
    table, new = pages[:batch * cols].view(batch, cols), pages[batch * cols:].view(batch, new_cols)
    cache = ops.Kv8Cache.empty(pages.numel(), hkv, page, d, device=cuda)
    angle = torch.arange(2048, device=cuda)[:, None] * 10000.0 ** (-torch.arange(d // 2, device=cuda) / (d // 2))
    cos, sin = angle.cos(), angle.sin()
    lens = torch.tensor(prompts, dtype=torch.int32, device=cuda)
    cu = torch.nn.functional.pad(lens.cumsum(0), (1, 0)).int()

    def rows(n):
        return (1.5 * torch.randn((n, hq + 2 * hkv, d), generator=g, device=cuda)).bfloat16().split((hq, hkv, hkv), 1)

    q, k, v = rows(sum(prompts))
    at = torch.cat([torch.arange(n, device=cuda) for n in prompts])
    turned = ops.kv8_append(cache, k, v, table, lens, cu_q=cu, positions=at, cos=cos, sin=sin, q=q)
    _check(turned, cache, table, prompts, prompts, lens, cu, True, None, window, sinks)
    weights = torch.zeros((batch, hkv, max(prompts)), device=cuda)
    ops.kv8_attention(turned, cache, table, lens, cu_q=cu, window=window, sinks=sinks, weights=weights)
    held = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    kept, new_lens, kept_weights = ops.kv8_evict(cache, table, lens, weights, keep, new, sinks=first, recent=recent)
    before = ops.Kv8Cache(*held)
    for b, n in enumerate(prompts):
        m = min(n, keep)
        assert new_lens[b].item() == m
        places = torch.arange(m, device=cuda)
        mine = ops.kv8_gather(cache, new[b, places // page].long() * page + places % page, torch.float32)
        for h in range(hkv):
            t = kept[b, h, :m].long()
            assert torch.equal(weights[b, h][t], kept_weights[b, h, :m])
            for x, y, s in zip(mine, ops.kv8_gather(before, table[b, t // page].long() * page + t % page, torch.float32), (cache.k_scales, cache.v_scales)):
                step = s[new[b, places // page].long(), h][:, None]  # below 2^-6 a code's step is 2^-9 of the scale: half a step, or 2^-4 of the number
                assert torch.all((x[:, h] - y[:, h]).abs() <= torch.maximum(y[:, h].abs() * 2.0 ** -4, step * 2.0 ** -10))

    # single tokens behind the kept ones: positions go on from the old lengths, places from the new ones
    live = torch.zeros((batch, hkv, new_cols * page), device=cuda)
    live[..., :keep] = kept_weights
    now = new_lens.clone()
    for i in range(tokens):
        q, k, v = rows(batch)
        now += 1
        turned = ops.kv8_append(cache, k, v, new, now, positions=lens.long() + i, cos=cos, sin=sin, q=q)
        if i in (0, 1, page - 1, tokens - 1):
            _check(turned, cache, new, now.tolist(), [1] * batch, now, None, True, None, window, sinks)
        ops.kv8_attention(turned, cache, new, now, window=window, sinks=sinks, weights=live)
    # a query's weights sum to 1: scores' magnitudes sum |q k| / sqrt(d) stay below 40, each of (d + 8) 2^-24 of which moves a weight by
    # three times as much of itself (twice by its score, once by the logarithm): 2^-10
    gained = live.sum((1, 2)) - kept_weights.sum((1, 2))
    assert torch.all((gained - hq * tokens).abs() <= 2.0 ** -9 * (hq * tokens + kept_weights.sum((1, 2))))
    # and cut again, into the pages of the prompts
    kept, lens2, _ = ops.kv8_evict(cache, new, now, live, keep, table, sinks=first, recent=recent)
    assert lens2.tolist() == [min(n, keep) for n in now.tolist()]
    assert torch.all(kept[:, :, :first] == torch.arange(first, device=cuda, dtype=torch.int32))
    _check(turned, cache, table, lens2.tolist(), [1] * batch, lens2, None, True, None, window, sinks)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_lens,kv_lens,window", [([100] * 16, [100] * 16, None), ([32] * 64, [32] * 64, None), ([24] * 48, [900] * 48, None), ([1000], [4000], None),
                                                   ([1000], [4000], 2500), ([300, 301, 299, 1], [2500, 2400, 300, 2000], None), ([256], [6000], None), ([512], [512], None),
                                                   ([2400], [2400], None), ([130, 2], [9000, 9000], None)])
def test_every_form_of_attention(cuda, d, q_lens, kv_lens, window):
    """Few rows, many, each with splits and without, as the sizes choose."""
    _run(cuda, q_lens, kv_lens, 4, 4, d, 32, seed=len(q_lens), window=window, sinks=4 if window else 0)


def test_sequences_that_share_pages(cuda):
    """A prefix that three sequences have in the same pages: attention, weights and eviction as with copies of their own."""
    q, cache, table, lens, cu, _ = _run(cuda, [3, 1, 20], [200, 180, 220], 2, 3, 64, 16, seed=5)
    shared = table.clone()
    shared[1:, :8] = table[0, :8]
    copies = ops.Kv8Cache(*[t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)])
    for t in (copies.k_codes, copies.k_scales, copies.v_codes, copies.v_scales):
        for b in (1, 2):
            t[table[b, :8].long()] = t[table[0, :8].long()]
    free = cache.num_pages
    both = []
    for c, tab in ((cache, shared), (copies, table)):
        more = ops.Kv8Cache(*[torch.cat([t, torch.zeros_like(t[:12])]) for t in (c.k_codes, c.k_scales, c.v_codes, c.v_scales)])
        w = torch.zeros((3, 2, 224), device=cuda)
        o = ops.kv8_attention(q, more, tab, lens, cu_q=cu, weights=w)
        new = torch.arange(free, free + 12, dtype=torch.int32, device=cuda).view(3, 4)
        kept, new_lens, kept_w = ops.kv8_evict(more, tab, lens, w, 64, new, sinks=4, recent=8)
        both.append((o, w, kept, new_lens, kept_w, more.k_codes[free:], more.k_scales[free:], more.v_codes[free:], more.v_scales[free:]))
    for a, b in zip(*both):
        assert torch.equal(a, b)


def test_calls_on_two_streams_at_once(cuda):
    """Two batches on pages of their own in one cache, appended, attended and cut on two streams at the same time."""
    g, d, page, keep = torch.Generator(device=cuda).manual_seed(1), 128, 32, 100
    lens = [torch.tensor([700, 90], dtype=torch.int32, device=cuda), torch.tensor([300, 800], dtype=torch.int32, device=cuda)]
    tables = [torch.arange(50, dtype=torch.int32, device=cuda).view(2, 25) + 50 * i for i in range(2)]
    news = [torch.arange(8, dtype=torch.int32, device=cuda).view(2, 4) + 100 + 8 * i for i in range(2)]
    rows = [torch.randn((int(n.sum()), 12, d), generator=g, device=cuda).bfloat16() for n in lens]
    cus = [torch.nn.functional.pad(n.cumsum(0), (1, 0)).int() for n in lens]

    def work(cache, i):
        q, k, v = rows[i].split((8, 2, 2), 1)
        q = ops.kv8_append(cache, k, v, tables[i], lens[i], cu_q=cus[i], q=q)
        w = torch.zeros((2, 2, 800), device=cuda)
        o = ops.kv8_attention(q, cache, tables[i], lens[i], cu_q=cus[i], weights=w)
        return (o, w, *ops.kv8_evict(cache, tables[i], lens[i], w, keep, news[i]))

    one, two = (ops.Kv8Cache.empty(116, 2, page, d, device=cuda) for _ in range(2))
    want = [work(one, i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(work(two, i))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            for x, y in zip(a, b):
                assert torch.equal(x, y)
        for a, b in ((one.k_codes, two.k_codes), (one.k_scales, two.k_scales), (one.v_codes, two.v_codes), (one.v_scales, two.v_scales)):
            assert torch.equal(a, b)


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "long_context.py"
    spec = importlib.util.spec_from_file_location("long_context", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("prompts,q_heads,kv_heads,head_dim", [((300, 17, 1), 8, 2, 128), ((40,), 4, 4, 64), ((900, 150), 12, 4, 64)])
def test_layer(cuda, example, prompts, q_heads, kv_heads, head_dim):
    """Where nothing is evicted, against float32.  E4M3 rounds numbers spread evenly over a binade by 0.026 of their root mean square.
    A product of two such operands is off by 0.037: the queries, keys and values, and the output; the cache's keys and values by 0.026
    more.  In the values, and in the output's product, that is the output's error; in queries and keys that of a score of
    about one sigma, and so of a weight.  Squared and added, queries 0.037, keys and values 0.037 and 0.026 each, the output 0.037: 0.083;
    twice that is not exceeded.  Where tokens are evicted, replays give what calls do."""
    called, replayed, plain, _ = example.run(prompts, 20, 1000, 32, 4, 16, 512, q_heads, kv_heads, head_dim)
    assert example.distance(called, plain) < 0.17
    for a, b in zip(called, replayed):
        assert torch.equal(a, b)
    called, replayed, _, _ = example.run(prompts, 20, 32, 6, 4, 16, 512, q_heads, kv_heads, head_dim)
    for a, b in zip(called, replayed):
        assert torch.isfinite(a).all() and torch.equal(a, b)
