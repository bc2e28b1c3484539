"""Appending to the paged 4-bit cache and reading it back, bit for bit against a numpy restatement in f32, and
the codes' own error against float64; rows that no slot names keep their bits."""
import copy
import dataclasses

import numpy as np
import pytest
import torch

from castforge_amd import ffi, ops

pytestmark = pytest.mark.gpu
F = np.float32


def _rotate(x, cos, sin, rot, interleaved):
    x = x.copy()
    c, s = cos[:, None], sin[:, None]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    u, v = a * c - b * s, b * c + a * s
    if interleaved:
        x[..., 0:rot:2], x[..., 1:rot:2] = u, v
    else:
        x[..., :rot // 2], x[..., rot // 2:rot] = u, v
    return x


def _quantize(x, group):
    """codes [.., D] 0..15, scale bits u16 and zero points [.., D / group]."""
    t = x.reshape(*x.shape[:-1], -1, group)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        lo = np.minimum(np.fmin.reduce(t, -1), F(0))
        hi = np.maximum(np.fmax.reduce(t, -1), F(0))
        lo, hi = np.where(np.isnan(lo), F(0), lo), np.where(np.isnan(hi), F(0), hi)
        r = hi - lo
        h = np.where(r >= F(1e-12), (r * F(1 / 15)).astype(np.float16), np.float16(1)).view(np.uint16)
        h = np.where(h == 0, 1, np.where(h == 0x7C00, 0x7BFF, h)).astype(np.uint16)
        s = h.view(np.float16).astype(F)
        z = np.rint(-lo / s)
        z = np.clip(np.where(np.isnan(z), 0, z), 0, 15)
        q = np.rint(t / s[..., None])
        q = np.clip(np.where(np.isnan(q), 0, q) + z[..., None], 0, 15)
    return q.astype(np.uint32).reshape(x.shape), h, z.astype(np.uint32)


def _pack(q, h, z):
    w = (q.reshape(*q.shape[:-1], -1, 8) << (4 * np.arange(8, dtype=np.uint32))).sum(-1, dtype=np.uint32)
    return w, h.astype(np.uint32) | (z << 16)


def _random_cache(seed, pages, heads, page, d, group, cuda):
    g = torch.Generator().manual_seed(seed)
    shape = (pages, heads, page)
    t = [torch.randint(-2**31, 2**31, shape + (w,), generator=g, dtype=torch.int64).to(torch.int32).to(cuda)
         for w in (d // 8, d // group) * 2]
    return ops.Kv4Cache(*t, group=group)


def _case(seed, tokens, hkv, hq, d, rot, max_pos=300):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn((tokens, hq + 2 * hkv, d), generator=g)
    qkv[:, :, ::37] *= 8
    qkv = qkv.bfloat16()
    angle = torch.arange(max_pos)[:, None] * 10000.0 ** (-torch.arange(rot // 2) / max(rot // 2, 1))
    pos = torch.randint(0, max_pos, (tokens,), generator=g)
    return qkv, pos, angle.cos(), angle.sin()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hkv,hq,d,group,page,rot", [
    (1, 1, 1, 64, 32, 16, 64), (1, 8, 32, 128, 128, 16, 128), (5, 3, 6, 64, 64, 32, 32), (17, 2, 10, 128, 32, 64, 128),
    (33, 8, 8, 128, 64, 16, 64), (130, 1, 7, 128, 128, 128, 16), (257, 4, 4, 64, 64, 16, 48), (40, 5, 5, 128, 64, 32, 0),
    (2048, 32, 1, 128, 32, 64, 128)])
def test_append_bits(cuda, tokens, hkv, hq, d, group, page, rot, interleaved):
    pages = tokens // page + 3
    cache = _random_cache(1, pages, hkv, page, d, group, cuda)
    before = [t.clone() for t in (cache.k_codes, cache.k_groups, cache.v_codes, cache.v_groups)]
    qkv, pos, cos, sin = _case(2, tokens, hkv, hq, d, rot)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(3))[:tokens]
    if tokens > 4:
        slots[3] = -1
        slots[4] = pages * page  # past the end
    dev = qkv.to(cuda)
    q, k, v = dev[:, :hq], dev[:, hq:hq + hkv], dev[:, hq + hkv:]
    table = (pos.to(cuda), cos.to(cuda), sin.to(cuda)) if rot else (None, None, None)
    got = ops.kv4_append(cache, k, v, slots.to(cuda), *table, q=q, interleaved=interleaved)
    f = qkv.float().numpy()
    c, s = cos.numpy()[pos.numpy()], sin.numpy()[pos.numpy()]
    turned = _rotate(f[:, :hq + hkv], c, s, rot, interleaved) if rot else f[:, :hq + hkv]
    assert torch.equal(got.cpu(), torch.from_numpy(turned[:, :hq]).bfloat16())
    kq, vq = _quantize(turned[:, hq:], group), _quantize(f[:, hq + hkv:], group)
    live = [i for i in range(tokens) if 0 <= slots[i] < pages * page]
    for (codes, groups), old, parts in (((cache.k_codes, cache.k_groups), before[:2], kq),
                                        ((cache.v_codes, cache.v_groups), before[2:], vq)):
        want = [o.cpu().numpy().view(np.uint32).copy() for o in old]
        for w, p in zip(want, _pack(*parts)):
            for i in live:
                w[slots[i] // page, :, slots[i] % page] = p[i]
        assert np.array_equal(codes.cpu().numpy().view(np.uint32), want[0])
        assert np.array_equal(groups.cpu().numpy().view(np.uint32), want[1])
    # read back: exact in f32, once rounded in bf16, zeros where there is no slot
    for out in (torch.float32, torch.bfloat16):
        for t, (qq, h, z) in zip(ops.kv4_gather(cache, slots.to(cuda), out), (kq, vq)):
            val = (qq.astype(F) - np.repeat(z.astype(F), group, -1)) * np.repeat(h.view(np.float16).astype(F), group, -1)
            val[[i for i in range(tokens) if i not in live]] = 0
            assert torch.equal(t.cpu(), torch.from_numpy(val).to(out))


def test_code_error_against_float64(cuda):
    """A code is within half a step of its number, and a step beyond at the range's ends, where the zero point's
    rounding cuts: |x - (q - z) s| <= s (1 + 2^-10)."""
    cache = ops.Kv4Cache.empty(20, 4, 16, 128, 64, device=cuda)
    qkv, pos, cos, sin = _case(5, 300, 4, 1, 128, 128)
    dev = qkv.to(cuda)
    slots = torch.arange(300, device=cuda)
    ops.kv4_append(cache, dev[:, 1:5], dev[:, 5:], slots, pos.to(cuda), cos.to(cuda), sin.to(cuda))
    k, v = ops.kv4_gather(cache, slots, torch.float32)
    f = qkv.double().numpy()
    turned = _rotate(f[:, 1:5], cos.double().numpy()[pos.numpy()], sin.double().numpy()[pos.numpy()], 128, False)
    for got, x in ((k, turned), (v, f[:, 5:])):
        t = x.reshape(300, 4, 2, 64)
        step = (np.maximum(t.max(-1), 0) - np.minimum(t.min(-1), 0))[..., None] / 15
        err = np.abs(got.cpu().numpy().reshape(t.shape) - t)
        assert np.all(err <= step * (1 + 2.0 ** -10) + 1e-6) and np.median(err / step) < 0.3


def test_special_groups(cuda):
    """Zeros, one sign only, tiny and huge ranges, infinities and NaN."""
    x = torch.zeros((8, 1, 64))
    g = torch.Generator().manual_seed(6)
    x[1] = 3 + torch.rand((1, 64), generator=g)
    x[2] = -5 * torch.rand((1, 64), generator=g)
    x[3] = 1e-30
    x[4] = 1e-7 * torch.randn((1, 64), generator=g)
    x[5] = 3e38 * (torch.rand((1, 64), generator=g) - 0.5)
    x[6] = torch.randn((1, 64), generator=g)
    x[6, 0, 5], x[6, 0, 40] = float("nan"), float("inf")
    x[7] = float("nan")
    x = x.bfloat16()
    cache = ops.Kv4Cache.empty(1, 1, 16, 64, 32, device=cuda)
    slots = torch.arange(8, device=cuda)
    ops.kv4_append(cache, x.to(cuda), x.to(cuda), slots)
    q, h, z = _quantize(x.float().numpy(), 32)
    w, gr = _pack(q, h, z)
    for codes, groups in ((cache.k_codes, cache.k_groups), (cache.v_codes, cache.v_groups)):
        assert np.array_equal(codes.cpu().numpy().view(np.uint32)[0, 0, :8], w[:, 0])
        assert np.array_equal(groups.cpu().numpy().view(np.uint32)[0, 0, :8], gr[:, 0])
    k, _ = ops.kv4_gather(cache, slots, torch.float32)
    assert torch.equal(k[0], torch.zeros_like(k[0])) and (k[1, 0] - x[1, 0].to(cuda).float()).abs().max() < 0.2


def test_positions_outside_the_table_take_its_ends(cuda):
    qkv, _, cos, sin = _case(7, 4, 1, 1, 64, 64, max_pos=10)
    dev, slots = qkv.to(cuda), torch.arange(4, device=cuda)
    res = []
    for pos in ([-7, 0, 9, 10 ** 12], [0, 0, 9, 9]):
        cache = ops.Kv4Cache.empty(1, 1, 16, 64, 64, device=cuda)
        q = ops.kv4_append(cache, dev[:, 1:2], dev[:, 2:], slots, torch.tensor(pos, device=cuda), cos.to(cuda), sin.to(cuda), q=dev[:, :1])
        res.append((q, cache.k_codes, cache.k_groups))
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_offsets_past_32_bits(cuda):
    """A cache of more than 2^32 bytes of codes: rows at its end are written and read where they belong."""
    pages, heads, page, d = 40000, 16, 128, 128  # 5.2 GB of key codes
    cache = ops.Kv4Cache.empty(pages, heads, page, d, 128, device=cuda)
    qkv, pos, cos, sin = _case(8, 3, heads, 1, d, d)
    dev = qkv.to(cuda)
    slots = torch.tensor([pages * page - 1, 5, 35000 * page + 7], device=cuda)
    ops.kv4_append(cache, dev[:, 1:1 + heads], dev[:, 1 + heads:], slots, pos.to(cuda), cos.to(cuda), sin.to(cuda))
    small = ops.Kv4Cache.empty(1, heads, page, d, 128, device=cuda)
    at = torch.arange(3, device=cuda)
    ops.kv4_append(small, dev[:, 1:1 + heads], dev[:, 1 + heads:], at, pos.to(cuda), cos.to(cuda), sin.to(cuda))
    for a, b in zip(ops.kv4_gather(cache, slots), ops.kv4_gather(small, at)):
        assert torch.equal(a, b)
    assert int((cache.v_groups != 0).sum()) == 3 * heads
    o1 = ops.kv4_attention(dev[:1, :1].expand(1, heads, d).contiguous(), cache, torch.tensor([[35000, pages - 1]], dtype=torch.int32, device=cuda),
                           torch.tensor([page + 128], dtype=torch.int32, device=cuda))
    assert torch.isfinite(o1).all() and o1.abs().max() > 0


def test_refusals(cuda):
    cache = ops.Kv4Cache.empty(2, 2, 16, 64, 32, device=cuda)
    k = torch.zeros((3, 2, 64), device=cuda, dtype=torch.bfloat16)
    slots, pos = torch.arange(3, device=cuda), torch.arange(3, device=cuda)
    cos = torch.zeros((8, 32), device=cuda)
    good = dict(cache=cache, k=k, v=k, slots=slots, positions=pos, cos=cos, sin=cos)
    wide = torch.zeros((3, 2, 65), device=cuda, dtype=torch.bfloat16)[..., :64]
    odd = torch.zeros((3, 131), device=cuda, dtype=torch.bfloat16)[:, :128].unflatten(1, (2, 64))  # stride 131
    for bad in (dict(k=k.float()), dict(k=k[:, :1]), dict(v=k[:2]), dict(slots=slots.int()), dict(slots=slots[:2]),
                dict(cos=None), dict(cos=cos[:, :24 // 2]), dict(cos=cos.double(), sin=cos.double()), dict(positions=pos.int()),
                dict(k=wide), dict(k=odd), dict(q=k[:2]), dict(q=k.float()), dict(k=k.cpu()), dict(cos=torch.zeros((8, 40), device=cuda), sin=torch.zeros((8, 40), device=cuda))):
        with pytest.raises((ValueError, ffi.CastForgeHipError)):
            ops.kv4_append(**{**good, **bad})
    with pytest.raises(ValueError):
        ops.kv4_gather(cache, slots.int())
    with pytest.raises(ValueError):
        ops.kv4_gather(cache, slots, torch.float16)
    z = torch.zeros
    i = dict(dtype=torch.int32, device=cuda)
    for bad in ((z((2, 2, 16, 8), **i), z((2, 2, 16, 1), **i), z((2, 2, 16, 8), **i), z((2, 2, 16, 2), **i), 64),
                (z((2, 2, 16, 12), **i), z((2, 2, 16, 3), **i), z((2, 2, 16, 12), **i), z((2, 2, 16, 3), **i), 32),
                (z((2, 2, 16, 8), **i), z((2, 2, 16, 1), **i), z((2, 2, 16, 8), **i), z((2, 2, 16, 1), **i), 128)):
        with pytest.raises(ValueError):
            ops.Kv4Cache(*bad[:4], group=bad[4])
    with pytest.raises(ffi.CastForgeHipError, match="page_size"):
        ops.kv4_append(ops.Kv4Cache.empty(2, 2, 24, 64, 32, device=cuda), k, k, slots)


def test_empty(cuda):
    cache = ops.Kv4Cache.empty(2, 2, 16, 64, 32, device=cuda)
    k = torch.zeros((0, 2, 64), device=cuda, dtype=torch.bfloat16)
    none = torch.zeros(0, dtype=torch.int64, device=cuda)
    assert ops.kv4_append(cache, k, k, none, q=k).shape == (0, 2, 64)
    assert ops.kv4_gather(cache, none)[0].shape == (0, 2, 64)
    nothing = ops.Kv4Cache.empty(0, 2, 16, 64, 32, device=cuda)
    one = torch.ones((1, 2, 64), device=cuda, dtype=torch.bfloat16)
    ops.kv4_append(nothing, one, one, torch.zeros(1, dtype=torch.int64, device=cuda))
    assert torch.equal(ops.kv4_gather(nothing, torch.zeros(1, dtype=torch.int64, device=cuda))[0], torch.zeros_like(one))


def test_more_tokens_than_a_launch_of_workgroups(cuda):
    """2^24 tokens and a few, each a workgroup of 256: more than 2^32 work-items.  Those with a slot come out as they do alone."""
    n, d = 2**24 + 5, 64
    cache, small = (ops.Kv4Cache.empty(1, 1, 16, d, 64, device=cuda) for _ in range(2))
    at = torch.tensor([0, 7654321, 2**23 - 1, 2**23, 2**24 - 1, 2**24, n - 1], device=cuda)
    qkv, pos, cos, sin = _case(11, 7, 1, 1, d, d)
    few = [qkv[:, i:i + 1].to(cuda).contiguous() for i in range(3)]
    q, k, v = (torch.zeros((n, 1, d), dtype=torch.bfloat16, device=cuda).index_copy_(0, at, t) for t in few)
    slots, positions = torch.full((n,), -1, device=cuda), torch.zeros(n, dtype=torch.int64, device=cuda)
    slots[at], positions[at] = torch.arange(7, device=cuda), pos.to(cuda)
    got = ops.kv4_append(cache, k, v, slots, positions, cos.to(cuda), sin.to(cuda), q=q)
    want = ops.kv4_append(small, few[1], few[2], torch.arange(7, device=cuda), pos.to(cuda), cos.to(cuda), sin.to(cuda), q=few[0])
    assert torch.equal(got[at], want)
    assert torch.equal(cache.k_codes, small.k_codes) and torch.equal(cache.v_groups, small.v_groups)
    for a, b in zip(ops.kv4_gather(cache, slots), ops.kv4_gather(small, torch.arange(7, device=cuda))):
        assert torch.equal(a[at], b)
        a[at] = 0
        assert not a.any()


def test_fields_stay_those_the_calls_use(cuda):
    """A cache's buffers and group cannot be exchanged behind the addresses that its calls take; another cache is made of others."""
    cache = _random_cache(9, 3, 2, 16, 64, 32, cuda)
    for name in ("k_codes", "k_groups", "v_codes", "v_groups"):
        with pytest.raises(AttributeError):
            setattr(cache, name, getattr(cache, name).clone())
        with pytest.raises(AttributeError):
            delattr(cache, name)
    for name, value in (("group", 64), ("num_pages", 2), ("kv_heads", 1), ("page_size", 32), ("head_dim", 128)):
        with pytest.raises(AttributeError):
            setattr(cache, name, value)
    larger = [torch.cat([t, t]) for t in (cache.k_codes, cache.k_groups, cache.v_codes, cache.v_groups)]
    grown = dataclasses.replace(cache, **dict(zip(("k_codes", "k_groups", "v_codes", "v_groups"), larger)))
    assert grown.num_pages == 6 and cache.num_pages == 3 and grown.nbytes() == 2 * cache.nbytes()
    slots = torch.arange(48, 96, device=cuda)
    for a, b in zip(ops.kv4_gather(grown, slots), ops.kv4_gather(cache, slots - 48)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))  # random words hold NaN


def test_copies_hold_their_own_rows(cuda):
    cache = _random_cache(10, 2, 2, 16, 64, 32, cuda)
    other, same = copy.deepcopy(cache), copy.copy(cache)
    assert same.k_codes is cache.k_codes and other.k_codes.data_ptr() != cache.k_codes.data_ptr()
    slots, one = torch.arange(3, device=cuda), torch.ones((3, 2, 64), device=cuda, dtype=torch.bfloat16)
    before = [t.clone() for t in ops.kv4_gather(cache, slots)]
    ops.kv4_append(other, one, one, slots)
    for a, b in zip(ops.kv4_gather(cache, slots), before):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    ops.kv4_append(same, one, one, slots)
    for a, b in zip(ops.kv4_gather(cache, slots), ops.kv4_gather(other, slots)):
        assert torch.equal(a, b)
