"""RMS norm with the residual's addition and E4M3 output, and the E4M3 block quantizer, against plain numpy:
h and the quantizer's codes and scales bit for bit, the norm's scales and codes against float64."""
import numpy as np
import pytest
import torch

from castforge_amd import ops

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def _randn(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


def _values(codes):
    return codes.cpu().view(F8).double().numpy()


def _blocks_up(s, block_rows, r, c):
    return np.repeat(np.repeat(s, block_rows, 0)[:r], 128, 1)[:, :c]


def _check_norm(x, r, w, eps, block, got, terms):
    """x, r, w as the f32 numbers that the inputs hold.  f32 sums of `terms` squares, a root and three products are
    within (terms + 8) / 2 ulp of f32 of the definition: that bounds the scale, and a code is at most half a
    step of E4M3 off its number (2^-4 of it, or half of 2^-9), widened by the scale's and the number's own error."""
    codes, scales, h = got
    hd = h.float().cpu().numpy().astype(np.float64)
    y = hd / np.sqrt((hd ** 2).mean(1, keepdims=True) + eps) * w.astype(np.float64)
    rel = (terms + 8) * 2.0 ** -24
    size = block or x.shape[1]
    runs = -(-x.shape[1] // size)
    amax = np.stack([np.abs(y[:, i * size:(i + 1) * size]).max(1) for i in range(runs)], 1)
    want = np.where(amax < 1e-12, 1.0, amax / 448)
    s = scales.cpu().numpy().astype(np.float64).reshape(len(x), runs)
    assert np.all(np.abs(s - want) <= rel * want)
    up = np.repeat(s, size, 1)[:, :x.shape[1]]
    err = np.abs(_values(codes) * up - y)
    assert np.all(err <= np.maximum(np.abs(y) * 2.0 ** -4, 2.0 ** -10 * up) * (1 + 2.0 ** -10) + rel * np.abs(y))


@pytest.mark.parametrize("block", [0, 128])
@pytest.mark.parametrize("m,k,dtype,wdtype,residual", [
    (1, 4096, "bfloat16", "bfloat16", True), (3, 128, "bfloat16", "float32", False), (5, 64, "float32", "float32", True),
    (2, 1, "bfloat16", "bfloat16", True), (7, 1000, "bfloat16", "bfloat16", True), (4, 1001, "float32", "bfloat16", True),
    (9, 8, "bfloat16", "bfloat16", False), (33, 520, "bfloat16", "bfloat16", True), (2, 2056, "float32", "float32", False),
    (3, 5001, "bfloat16", "float32", True), (2, 16384, "bfloat16", "bfloat16", True), (2, 16392, "bfloat16", "bfloat16", False),
    (130, 2048, "bfloat16", "bfloat16", True), (2, 40000, "float32", "float32", True)])
def test_norm_against_float64(cuda, m, k, dtype, wdtype, residual, block):
    dt, wt = getattr(torch, dtype), getattr(torch, wdtype)
    x = torch.from_numpy(_randn(1, m, k)).to(dt)
    x[:, ::97] *= 20
    r = torch.from_numpy(_randn(2, m, k)).to(dt) if residual else None
    w = (1 + 0.2 * torch.from_numpy(_randn(3, k))).to(wt)
    got = ops.rms_norm_fp8(x.to(cuda), w.to(cuda), eps=1e-5, residual=None if r is None else r.to(cuda), block=block)
    h = x if r is None else (x.float() + r.float()).to(dt)
    assert torch.equal(got[2].cpu(), h)
    _check_norm(x.float().numpy(), r, w.float().numpy(), 1e-5, block, got, k)


def test_norm_in_place_and_same_as_out_of_place(cuda):
    x = torch.from_numpy(_randn(4, 6, 1024)).to(cuda).bfloat16()
    r = torch.from_numpy(_randn(5, 6, 1024)).to(cuda).bfloat16()
    w = torch.ones(1024, device=cuda)
    ref = ops.rms_norm_fp8(x, w, residual=r, block=128)
    for which in (0, 1):
        a, b = x.clone(), r.clone()
        got = ops.rms_norm_fp8(a, w, residual=b, block=128, out=(a, b)[which])
        assert got[2] is (a, b)[which]
        assert all(torch.equal(p, q) for p, q in zip(ref, got))


@pytest.mark.parametrize("k", [1000, 1024, 1003])
@pytest.mark.parametrize("block", [0, 128])
def test_norm_zero_rows_and_non_finite(cuda, k, block):
    """A row of zeros (eps > 0) gives zeros with scale 1; NaN and inf stay in their rows."""
    x = torch.from_numpy(_randn(6, 5, k)).bfloat16()
    x[1] = 0
    x[2, 17] = float("nan")
    x[3, 400] = float("inf")
    w = torch.ones(k)
    codes, scales, h = ops.rms_norm_fp8(x.to(cuda), w.to(cuda), block=block)
    v, s = _values(codes), scales.cpu().numpy().reshape(5, -1)
    assert np.all(v[1] == 0) and np.all(s[1] == 1)
    assert np.all(np.isnan(v[2])) and np.all(s[2] == 1)
    assert np.isnan(v[3, 400]) and np.all(v[3, np.arange(k) != 400] == 0)
    clean = ops.rms_norm_fp8(x[[0, 4]].contiguous().to(cuda), w.to(cuda), block=block)
    assert torch.equal(clean[0].cpu(), codes.cpu()[[0, 4]]) and torch.equal(clean[1].cpu(), scales.cpu()[[0, 4]])


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,cols,br", [(1, 128, 1), (1, 4096, 1), (5, 200, 1), (3, 1, 1), (130, 1100, 1), (64, 256, 1),
                                          (7, 8, 1), (256, 384, 128), (200, 130, 128), (1, 5, 128), (129, 4096, 128)])
def test_block_quantizer_codes(cuda, rows, cols, br, dtype):
    v = torch.from_numpy(_randn(7, rows, cols)).to(getattr(torch, dtype))
    v[:, ::61] *= 30
    v[0] = -0.0
    codes, scales = ops.quantize_fp8_block(v.to(cuda), br)
    f = v.float().numpy()
    pad = np.zeros((-(-rows // br) * br, -(-cols // 128) * 128), np.float32)
    pad[:rows, :cols] = np.abs(f)
    amax = pad.reshape(-(-rows // br), br, -1, 128).max((1, 3))
    s = np.where(amax < 1e-12, np.float32(1), amax * np.float32(1 / 448))
    assert np.array_equal(scales.cpu().numpy(), s)
    up = _blocks_up(s, br, rows, cols)
    assert np.array_equal(codes.cpu().numpy(), torch.from_numpy(f / up).to(F8).view(torch.uint8).numpy())
    assert np.array_equal(ops.dequantize_fp8_block(codes, scales, br).cpu().numpy(),
                          (_values(codes).astype(np.float32) * up))


def test_block_quantizer_non_finite(cuda):
    v = torch.from_numpy(_randn(8, 4, 512))
    v[0, 3] = float("nan")
    v[1, 200] = float("inf")
    codes, scales = ops.quantize_fp8_block(v.to(cuda))
    c, s = _values(codes), scales.cpu().numpy()
    assert np.isnan(c[0, 3]) and np.isfinite(np.delete(c[0], 3)).all()
    assert np.isinf(s[1, 1]) and np.isnan(c[1, 200]) and np.all(np.delete(c[1, 128:256], 72) == 0)
    assert np.isfinite(c[2:]).all()


def test_offsets_past_32_bits(cuda):
    """Rows at the end of more than 2^32 bytes come out as they do alone."""
    m, k = 65600, 32768
    x = torch.zeros((m, k), dtype=torch.bfloat16, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(30)
    x[-3:] = torch.randn((3, k), generator=g, device=cuda).bfloat16()
    w = torch.ones(k, dtype=torch.bfloat16, device=cuda)
    for part, whole in ((ops.rms_norm_fp8(x[-3:], w, residual=x[-3:], block=128), ops.rms_norm_fp8(x, w, residual=x, block=128)),
                        (ops.quantize_fp8_block(x[-3:]), ops.quantize_fp8_block(x))):
        for a, b in zip(part, whole):
            assert torch.equal(a, b[-3:])


def test_refusals(cuda):
    x, w = torch.zeros((2, 128), device=cuda, dtype=torch.bfloat16), torch.zeros(128, device=cuda)
    for bad in (dict(weight=w[:64]), dict(block=64), dict(residual=x.float()), dict(residual=x[:1]), dict(out=x),
                dict(weight=w.half()), dict(eps=-1.0), dict(x=x.half()), dict(x=x.t()), dict(x=x.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            ops.rms_norm_fp8(**{"x": x, "weight": w, **bad})
    for args in ((x, 2), (x.half(), 1), (x[0], 1)):
        with pytest.raises(ValueError):
            ops.quantize_fp8_block(*args)
    c, s = ops.quantize_fp8_block(x)
    for args in ((c, s, 128), (c.float(), s, 1), (c, s.double(), 1)):
        with pytest.raises(ValueError):
            ops.dequantize_fp8_block(*args)


def test_empty(cuda):
    for shape in ((0, 128), (3, 0)):
        x = torch.zeros(shape, device=cuda, dtype=torch.bfloat16)
        codes, scales, h = ops.rms_norm_fp8(x, torch.zeros(shape[1], device=cuda), residual=x, block=128)
        assert codes.shape == shape and h.shape == shape
        assert ops.quantize_fp8_block(x)[0].shape == shape


@pytest.mark.parametrize("k", [1032, 7])
def test_more_rows_than_a_launch_of_workgroups(cuda, k):
    """2^24 rows and a few, each a workgroup of 256: more than 2^32 work-items.  Rows come out as they do alone."""
    m = 2**24 + 5
    x = torch.zeros((m, k), dtype=torch.bfloat16, device=cuda)
    at = torch.tensor([0, 1, 2**23, 2**24 - 1, 2**24, m - 1], device=cuda)
    g = torch.Generator(device=cuda).manual_seed(31)
    x[at] = torch.randn((6, k), generator=g, device=cuda).bfloat16()
    w = torch.ones(k, dtype=torch.bfloat16, device=cuda)
    part = ops.rms_norm_fp8(x[at], w, residual=x[at], block=128)
    for a, b in zip(part, ops.rms_norm_fp8(x, w, residual=x, block=128, out=x)):
        assert torch.equal(a, b[at])


def test_more_blocks_than_a_launch_of_workgroups(cuda):
    """2^24 blocks and a few of the quantizer's plain kernel, as rows of seven elements and as one long row of 128 x 128 blocks."""
    g = torch.Generator(device=cuda).manual_seed(32)
    rows = torch.zeros((2**24 + 5, 7), dtype=torch.bfloat16, device=cuda)
    rows[-9:] = torch.randn((9, 7), generator=g, device=cuda).bfloat16()
    for a, b in zip(ops.quantize_fp8_block(rows), ops.quantize_fp8_block(rows[-9:])):
        assert torch.equal(a[-9:], b)
    del rows
    row = torch.zeros((1, 2**31 + 300), dtype=torch.bfloat16, device=cuda)
    row[:, -700:] = torch.randn((1, 700), generator=g, device=cuda).bfloat16()
    (codes, scales), tail = ops.quantize_fp8_block(row, 128), ops.quantize_fp8_block(row[:, -(6 * 128 + 44):], 128)
    assert torch.equal(codes[:, -(6 * 128 + 44):], tail[0]) and torch.equal(scales[:, -7:], tail[1])
    assert torch.all(scales[:, :2**24 - 10] == 1)


def test_rows_of_no_elements_have_a_scale(cuda):
    """The greatest of nothing is zero, and the scale of zeros one; with runs of 128 there is none to give."""
    x = torch.empty((5, 0), device=cuda, dtype=torch.bfloat16)
    held = torch.full((5,), 7.0, device=cuda)  # what the scales' memory may hold before
    del held
    codes, scales, h = ops.rms_norm_fp8(x, torch.empty(0, device=cuda))
    assert codes.shape == (5, 0) and h is x and torch.equal(scales, torch.ones(5, device=cuda))
    assert ops.rms_norm_fp8(x, torch.empty(0, device=cuda), residual=x, block=128)[1].shape == (5, 0)
