"""Appending to the paged 8-bit cache and reading it back, bit for bit against a restatement in f32 on the CPU; rows
that no sequence has and pages that get no token keep their bits."""
import copy
import math

import numpy as np
import pytest
import torch

from castforge_amd import ffi, ops

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _rotate(x, cos, sin, rot, interleaved):
    """x [T, H, D] f32; each product and each sum rounded where it stands."""
    x = x.clone()
    c, s = cos[:, None], sin[:, None]
    one, two = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., one].clone(), x[..., two].clone()
    x[..., one], x[..., two] = a * c - b * s, b * c + a * s
    return x


def _least_power(amax):
    if amax == 0:
        return 2.0 ** -70
    if math.isinf(amax):
        return 2.0 ** 30
    m, e = math.frexp(amax)  # 448 = 0.875 * 2^9
    return 2.0 ** min(max(e - 9 + (m > 0.875), -70), 30)


def _codes(x):
    """E4M3 codes of f32 numbers: NaN as 0, past 448 as 448."""
    return torch.where(torch.isnan(x), torch.zeros_like(x), x).clamp(-448, 448).to(F8).view(torch.uint8)


def _append(codes, scales, x, table, lens, q_lens, page):
    """In place; codes [pages, H, page, D], x [T, H, D] f32."""
    first = 0
    for b, (n, kv) in enumerate(zip(q_lens, lens)):
        tokens = [(t, first + t - (kv - n)) for t in range(max(kv - n, 0), min(kv, table.shape[1] * page))]
        first += n
        for col in sorted({t // page for t, _ in tokens}):
            p = int(table[b, col])
            if not 0 <= p < codes.shape[0]:
                continue
            mine = [(t % page, r) for t, r in tokens if t // page == col]
            rows, lo = x[[r for _, r in mine]], mine[0][0]
            for h in range(codes.shape[1]):
                new = rows[:, h]
                amax = torch.where(torch.isnan(new), torch.zeros_like(new), new.abs()).max().item()
                old = float(scales[p, h]) if lo > 0 else 0.0
                scale = max(old, _least_power(amax))
                if scale > old and lo > 0:
                    codes[p, h, :lo] = _codes(codes[p, h, :lo].view(F8).float() * torch.tensor(old / scale))
                scales[p, h] = scale
                codes[p, h, lo:lo + len(mine)] = _codes(new / torch.tensor(scale))


def _state(seed, pages, heads, page, d):
    g = torch.Generator().manual_seed(seed)
    t = []
    for _ in range(2):
        c = torch.randint(0, 256, (pages, heads, page, d), generator=g, dtype=torch.uint8)
        t += [torch.where(c & 0x7F == 0x7F, torch.zeros_like(c), c), torch.ldexp(torch.ones(pages, heads), torch.randint(-12, -4, (pages, heads), generator=g))]
    return t


def _table(seed, need, pages, cols):
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    t, i = torch.full((len(need), cols), 2**31 - 1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        t[b, :n] = perm[i:i + n]
        i += n
    return t


def _case(cuda, q_lens, lens, heads, d, page, rot=0, interleaved=False, hq=0, seed=0, change=None, varlen=None, pad=0):
    need = [-(-max(kv, 0) // page) for kv in lens]
    pages, n = sum(need) + 2, sum(q_lens)
    state = _state(seed, pages, heads, page, d)
    table = _table(seed, need, pages, max(need + [0]))
    g = torch.Generator().manual_seed(seed + 1)
    rows = torch.randn((n + pad, hq + 2 * heads, d), generator=g) * torch.exp(2 * torch.randn((n + pad, 1, 1), generator=g))
    rows = rows.bfloat16()
    if change:
        change(rows)
    q, k, v = rows[:, :hq], rows[:, hq:hq + heads], rows[:, hq + heads:]
    pos = torch.randint(-3, 70, (n + pad,), generator=g)
    angle = torch.arange(64)[:, None] * 10000.0 ** (-torch.arange(max(rot // 2, 1)) / max(rot // 2, 1))
    cos, sin = angle.cos(), angle.sin()
    if varlen is None:
        varlen = any(x != 1 for x in q_lens) or pad > 0
    cu = torch.tensor(np.cumsum([0] + q_lens), dtype=torch.int32)
    cache = ops.Kv8Cache(*[t.to(cuda) for t in state])
    dev = rows.to(cuda)
    turn = dict(positions=pos.to(cuda), cos=cos.to(cuda), sin=sin.to(cuda), interleaved=interleaved) if rot else {}
    got = ops.kv8_append(cache, dev[:, hq:hq + heads], dev[:, hq + heads:], table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                         cu_q=cu.to(cuda) if varlen else None, q=dev[:, :hq] if hq else None, **turn)
    at = pos.clamp(0, 63)
    turned = [_rotate(x.float(), cos[at], sin[at], rot, interleaved) if rot else x.float() for x in (q, k)]
    _append(state[0], state[1], turned[1], table, lens, q_lens, page)
    _append(state[2], state[3], v.float(), table, lens, q_lens, page)
    for what, a, b in zip(("k codes", "k scales", "v codes", "v scales"), (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), state):
        assert torch.equal(a.cpu(), b), (what, (a.cpu() != b).sum().item())
    if hq:
        assert torch.equal(got[:n].cpu().view(torch.int16), turned[0][:n].bfloat16().view(torch.int16))
    return cache, table, state


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_prompts_of_every_page_size(cuda, d, page):
    _case(cuda, [page * 2 + 3, 1, page, 5], [page * 2 + 3, 1, page + 7, 2 * page + 1], 2, d, page, rot=d, hq=3, seed=page + d)


@pytest.mark.parametrize("d,rot,interleaved", [(128, 128, False), (128, 64, False), (128, 128, True), (128, 32, True), (64, 64, False), (64, 16, True), (64, 0, False)])
def test_rotations(cuda, d, rot, interleaved):
    _case(cuda, [9, 2, 17], [40, 2, 17], 3, d, 16, rot=rot, interleaved=interleaved, hq=5, seed=rot + d)


@pytest.mark.parametrize("page", [16, 64, 256])
def test_single_tokens(cuda, page):
    lens = [1, 2, page, page + 1, page - 1, 3 * page, 5, 17] * 9
    _case(cuda, [1] * len(lens), lens, 4, 128, page, rot=128, hq=8, seed=page)
    _case(cuda, [1] * len(lens), lens, 4, 64, page, seed=page, varlen=True)


def test_many_sequences_some_without_rows(cuda):
    q_lens = [i % 4 for i in range(150)]
    lens = [q + (7 * i) % 50 for i, q in enumerate(q_lens)]
    _case(cuda, q_lens, lens, 1, 64, 16, rot=64, hq=2, seed=5)


def test_lengths_that_tokens_and_tables_do_not_fill(cuda):
    # more rows than tokens (the first ones are left out), no tokens, a negative length
    _case(cuda, [5, 3, 2, 4], [3, 0, -7, 4], 2, 128, 16, rot=128, hq=2, seed=3)


def test_tokens_past_the_table_and_pages_outside_the_cache_are_left_out(cuda):
    state = _state(1, 4, 2, 16, 64)
    cache = ops.Kv8Cache(*[t.to(cuda) for t in state])
    table = torch.tensor([[0, -1], [2**31 - 1, 1]], dtype=torch.int32)
    lens, q_lens = [40, 32], [40, 32]
    x = torch.randn((72, 2, 64), generator=torch.Generator().manual_seed(2)).bfloat16()
    ops.kv8_append(cache, x.to(cuda), x.to(cuda), table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                   cu_q=torch.tensor([0, 40, 72], dtype=torch.int32, device=cuda))
    for i in (0, 2):
        _append(state[i], state[i + 1], x.float(), table, lens, q_lens, 16)
    for a, b in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), state):
        assert torch.equal(a.cpu(), b)


def test_rows_behind_the_last_sequence_are_left_out(cuda):
    cache, _, _ = _case(cuda, [3, 2], [20, 2], 2, 128, 16, rot=128, hq=2, seed=9, pad=7)


def test_numbers_at_the_borders(cuda):
    """Zeros, the largest and least numbers, infinities, NaN, and absmaxes around 448 * 2^e."""
    def change(rows):
        flat = rows.view(rows.shape[0], -1)
        flat[0] = 0.0
        flat[1, ::3] = float("nan")
        flat[2, 5] = float("inf")
        flat[3, 7] = float("-inf")
        flat[4] = 3.3e38
        flat[5] = 1e-38
        flat[6] = float("nan")
        for i, x in enumerate((448.0, 450.0, 446.0, 0.875, 0.8789, 0.87, 1.75 * 2.0 ** 38, 1.7578 * 2.0 ** 38, 2.0 ** -62, 1.75 * 2.0 ** -62, 1.7578 * 2.0 ** -62)):
            flat[7 + i] = torch.linspace(-1, 1, flat.shape[1]) * x
            flat[7 + i, 11] = -x

    lens = [1] * 18
    _case(cuda, lens, lens, 2, 64, 16, seed=4, change=change)
    _case(cuda, lens, [2] * 18, 2, 64, 16, seed=4, change=change)   # beside what a page held
    _case(cuda, [18], [18], 2, 64, 32, seed=4, change=change)       # all in one page


def test_a_page_grows_token_by_token_and_starts_anew(cuda):
    cache = ops.Kv8Cache.empty(1, 1, 16, 64, device=cuda)
    state = [t.cpu().clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    table = torch.zeros((1, 1), dtype=torch.int32)
    g = torch.Generator().manual_seed(1)
    for i in list(range(16)) + [0, 1, 7, 3]:  # at the end: the page in another sequence, a token written again after others
        x = (torch.randn((1, 1, 64), generator=g) * 4.0 ** (i % 5)).bfloat16()
        ops.kv8_append(cache, x.to(cuda), -x.to(cuda), table.to(cuda), torch.tensor([i + 1], dtype=torch.int32, device=cuda))
        _append(state[0], state[1], x.float(), table, [i + 1], [1], 16)
        _append(state[2], state[3], -x.float(), table, [i + 1], [1], 16)
        for a, b in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), state):
            assert torch.equal(a.cpu(), b), i


def test_scales_that_are_no_powers_of_two(cuda):
    state = _state(1, 3, 2, 16, 64)
    for i in (1, 3):
        state[i] *= 1.37
    cache = ops.Kv8Cache(*[t.to(cuda) for t in state])
    table = torch.tensor([[1, 2]], dtype=torch.int32)
    for factor in (1e-3, 1.0, 30.0):
        x = (factor * torch.randn((9, 2, 64), generator=torch.Generator().manual_seed(2))).bfloat16()
        ops.kv8_append(cache, x.to(cuda), x.to(cuda), table.to(cuda), torch.tensor([21], dtype=torch.int32, device=cuda),
                       cu_q=torch.tensor([0, 9], dtype=torch.int32, device=cuda))
        for i in (0, 2):
            _append(state[i], state[i + 1], x.float(), table, [21], [9], 16)
        for a, b in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), state):
            assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,n", [(1, 1), (3, 7), (8, 300), (32, 40), (40, 1)])
def test_gather(cuda, d, heads, n):
    state = _state(n, 9, heads, 32, d)
    cache = ops.Kv8Cache(*[t.to(cuda) for t in state])
    slots = torch.randint(-2, 9 * 32 + 2, (n,), generator=torch.Generator().manual_seed(n))
    inside = (slots >= 0) & (slots < 9 * 32)
    at = slots.clamp(0, 9 * 32 - 1)
    for dtype in (torch.float32, torch.bfloat16):
        for got, c, s in zip(ops.kv8_gather(cache, slots.to(cuda), dtype), state[::2], state[1::2]):
            want = c[at // 32, :, at % 32].view(F8).float() * s[at // 32][..., None]
            assert torch.equal(got.cpu(), torch.where(inside[:, None, None], want, torch.zeros_like(want)).to(dtype))


def test_every_code_is_read_exactly(cuda):
    codes = torch.arange(256, dtype=torch.uint8).view(1, 1, 16, 16).repeat(1, 1, 1, 4).contiguous()
    cache = ops.Kv8Cache(codes.to(cuda), torch.full((1, 1), 2.0 ** -3, device=cuda), codes.to(cuda), torch.full((1, 1), 2.0 ** 9, device=cuda))
    k, v = ops.kv8_gather(cache, torch.arange(16, device=cuda), torch.float32)
    want = codes[0, 0].view(F8).float()
    for got, s in ((k, 2.0 ** -3), (v, 2.0 ** 9)):
        assert torch.equal(torch.nan_to_num(got[:, 0].cpu(), nan=1e9), torch.nan_to_num(want * s, nan=1e9))


def test_more_than_2_31_elements(cuda):
    """A cache of 2^31 + bytes of keys: offsets past 32 bits."""
    pages, heads, page, d = 70000, 2, 128, 128
    cache = ops.Kv8Cache.empty(pages, heads, page, d, device=cuda)
    x = torch.randn((130, heads, d), generator=torch.Generator().manual_seed(2)).bfloat16()
    table = torch.tensor([[pages - 1, 65530]], dtype=torch.int32)
    ops.kv8_append(cache, x.to(cuda), -x.to(cuda), table.to(cuda), torch.tensor([130], dtype=torch.int32, device=cuda),
                   cu_q=torch.tensor([0, 130], dtype=torch.int32, device=cuda))
    small = [t.cpu() for t in (torch.zeros((2, heads, page, d), dtype=torch.uint8), torch.ones(2, heads))]
    _append(small[0], small[1], x.float(), torch.tensor([[1, 0]]), [130], [130], page)
    assert torch.equal(cache.k_codes[[65530, pages - 1]].cpu(), small[0]) and torch.equal(cache.k_scales[[65530, pages - 1]].cpu(), small[1])
    slots = torch.cat([torch.arange(128) + (pages - 1) * page, torch.tensor([65530 * page, 65530 * page + 1])]).to(cuda)
    k, v = ops.kv8_gather(cache, slots, torch.float32)
    assert torch.equal(k, -v) and torch.equal(k[128:].cpu(), small[0][0, :, :2].view(F8).float().transpose(0, 1) * small[1][0][:, None])


def test_empty_calls(cuda):
    cache = ops.Kv8Cache.empty(2, 2, 16, 64, device=cuda)
    none, i32 = torch.empty((0, 2, 64), dtype=torch.bfloat16, device=cuda), dict(dtype=torch.int32, device=cuda)
    assert ops.kv8_append(cache, none, none, torch.empty((0, 1), **i32), torch.empty(0, **i32), q=none).shape == (0, 2, 64)
    one = torch.ones((1, 2, 64), dtype=torch.bfloat16, device=cuda)
    ops.kv8_append(cache, one, one, torch.empty((1, 0), **i32), torch.ones(1, **i32))        # a table of no pages
    ops.kv8_append(cache, one, one, torch.empty((0, 1), **i32), torch.empty(0, **i32), cu_q=torch.zeros(1, **i32))  # rows of no sequence
    nothing = ops.Kv8Cache.empty(0, 2, 16, 64, device=cuda)
    ops.kv8_append(nothing, one, one, torch.zeros((1, 1), **i32), torch.ones(1, **i32))
    assert torch.all(ops.kv8_gather(nothing, torch.zeros(1, dtype=torch.int64, device=cuda))[0] == 0)
    assert torch.all(cache.k_codes == 0) and ops.kv8_gather(cache, torch.empty(0, dtype=torch.int64, device=cuda))[0].shape == (0, 2, 64)


def test_refusals(cuda):
    cache = ops.Kv8Cache.empty(2, 2, 16, 64, device=cuda)
    k, i32 = torch.ones((3, 2, 64), dtype=torch.bfloat16, device=cuda), dict(dtype=torch.int32, device=cuda)
    good = dict(cache=cache, k=k, v=k, page_table=torch.zeros((1, 2), **i32), kv_lens=torch.full((1,), 3, **i32), cu_q=torch.tensor([0, 3], **i32))
    ops.kv8_append(**good)
    angles = torch.ones((4, 32), device=cuda)
    for bad in (dict(k=k.float()), dict(k=k[:, :1]), dict(v=k[:2]), dict(k=k[..., :32]), dict(k=k.cpu()), dict(kv_lens=torch.ones(2, **i32)),
                dict(kv_lens=torch.ones(1, device=cuda)), dict(cu_q=None), dict(cu_q=torch.zeros(1, **i32)), dict(page_table=torch.zeros((1, 2), device=cuda)),
                dict(page_table=torch.zeros(2, **i32)), dict(cos=angles), dict(cos=angles, sin=angles), dict(q=k[:2]),
                dict(cos=angles, sin=angles[:3], positions=torch.zeros(3, dtype=torch.int64, device=cuda)), dict(k=k.transpose(0, 1).contiguous().transpose(0, 1))):
        with pytest.raises(ValueError):
            ops.kv8_append(**{**good, **bad})
    with pytest.raises(ffi.CastForgeHipError, match="rot"):
        ops.kv8_append(**good, cos=torch.ones((4, 40), device=cuda), sin=torch.ones((4, 40), device=cuda), positions=torch.zeros(3, dtype=torch.int64, device=cuda))
    slots = torch.zeros(3, dtype=torch.int64, device=cuda)
    for bad in ((cache, slots.int()), (cache, slots, torch.float16), (cache, slots[None])):
        with pytest.raises(ValueError):
            ops.kv8_gather(*bad)
    t = (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)
    for bad in ((t[0].int(), *t[1:]), (t[0], t[1].double(), *t[2:]), (t[0], t[1][:1], *t[2:]), (*t[:2], t[2][:1], t[3]), (t[0].cpu(), *t[1:]), (t[0][..., :32], *t[1:])):
        with pytest.raises(ValueError):
            ops.Kv8Cache(*bad)
    with pytest.raises(ffi.CastForgeHipError, match="page_size"):
        ops.kv8_append(**{**good, "cache": ops.Kv8Cache.empty(2, 2, 24, 64, device=cuda)})
    with pytest.raises(Exception):
        cache.k_codes = t[0]


def test_copies_have_their_own_memory(cuda):
    cache = ops.Kv8Cache.empty(1, 1, 16, 64, device=cuda)
    other = copy.deepcopy(cache)
    one, i32 = torch.ones((1, 1, 64), dtype=torch.bfloat16, device=cuda), dict(dtype=torch.int32, device=cuda)
    ops.kv8_append(other, one, one, torch.zeros((1, 1), **i32), torch.ones(1, **i32))
    assert torch.all(cache.k_codes == 0) and not torch.all(other.k_codes == 0)
    assert other.nbytes() == 2 * (16 * 64 + 4)


def test_a_captured_append_follows_its_lists(cuda):
    """A replay reads the lengths, the table and the rows that it finds."""
    d, page = 128, 16
    cache = ops.Kv8Cache.empty(8, 2, page, d, device=cuda)
    state = [t.cpu().clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    table = torch.tensor([[3, 1], [0, 6]], dtype=torch.int32)
    lens, dtable = torch.tensor([1, 1], dtype=torch.int32, device=cuda), table.to(cuda)
    rows = torch.zeros((2, 4, d), dtype=torch.bfloat16, device=cuda)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.kv8_append(cache, rows[:, :2], rows[:, 2:], dtable, lens)
    torch.cuda.synchronize()
    _append(state[0], state[1], torch.zeros(2, 2, d), table, [1, 1], [1, 1], page), _append(state[2], state[3], torch.zeros(2, 2, d), table, [1, 1], [1, 1], page)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.kv8_append(cache, rows[:, :2], rows[:, 2:], dtable, lens)
    g = torch.Generator().manual_seed(3)
    for kv in ([1, 5], [2, 6], [17, 16], [18, 17]):
        x = (torch.randn((2, 4, d), generator=g) * kv[0]).bfloat16()
        rows.copy_(x), lens.copy_(torch.tensor(kv, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        _append(state[0], state[1], x[:, :2].float(), table, kv, [1, 1], page), _append(state[2], state[3], x[:, 2:].float(), table, kv, [1, 1], page)
        for a, b in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), state):
            assert torch.equal(a.cpu(), b)
