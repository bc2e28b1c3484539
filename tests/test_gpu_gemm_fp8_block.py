"""The block-scaled FP8 product against a float64 product of the dequantized operands.

exact=True: products of E4M3 codes are exact in f32, and a sum of K of them is within K 2^-24 of the sum of
their magnitudes; scaling rounds twice more.  exact=False adds the fp8 MFMA's adder, which keeps at least 12
bits below the largest product of a 64-wide step (so 64 * 2^-12 of it, summed over the steps).  A bf16 output
rounds by 2^-9 of itself."""
import numpy as np
import pytest
import torch

from castforge_amd import ffi, ops

pytestmark = pytest.mark.gpu


def _inputs(seed, m, n, k, cuda, outliers=True):
    g = torch.Generator().manual_seed(seed)
    a, w = torch.randn((m, k), generator=g), torch.randn((n, k), generator=g) * 0.02
    if outliers:
        a[:, torch.rand(k, generator=g) < 0.01] *= 20
        w[:, torch.rand(k, generator=g) < 0.005] *= 30
    a[:, : min(k, 128)] *= 1e-3  # blocks of very different scales
    w[: min(n, 128)] *= 50
    return ops.quantize_fp8_block(a.to(cuda)), ops.quantize_fp8_block(w.to(cuda), 128)


def _up(s, block_rows, r, c):
    return s.double().repeat_interleave(block_rows, 0)[:r].repeat_interleave(128, 1)[:, :c]


def _check(y, qa, sa, qw, sw, exact):
    (m, k), n = qa.shape, qw.shape[0]
    f8 = torch.float8_e4m3fn
    a = qa.view(f8).float().double() * _up(sa, 1, m, k)
    w = qw.view(f8).float().double() * _up(sw, 128, n, k)
    ref, mag = a @ w.t(), a.abs() @ w.abs().t()
    bound = (k + 4) * 2.0 ** -24 * mag + 1e-30
    if not exact:
        steps = torch.zeros_like(ref)
        for k0 in range(0, k, 64):
            x, z = a[:, k0:k0 + 64].abs(), w[:, k0:k0 + 64].abs()
            for i in range(0, m, 64):
                for j in range(0, n, 256):
                    steps[i:i + 64, j:j + 256] += (x[i:i + 64, None] * z[None, j:j + 256]).amax(2)
        bound += 64 * 2.0 ** -12 * steps
    if y.dtype == torch.bfloat16:
        bound += 2.0 ** -8 * (ref.abs() + bound)
    far = ((y.double() - ref).abs() > bound).sum().item()
    assert far == 0, f"{far} of {y.numel()} outputs past the bound"
    rel = ((y.double() - ref).norm() / ref.norm().clamp(min=1e-300)).item()
    assert rel <= (2.5e-3 if y.dtype == torch.bfloat16 else 2e-6 if exact else 5e-4), rel


@pytest.mark.parametrize("exact,out", [(True, torch.float32), (True, torch.bfloat16), (False, torch.bfloat16),
                                       (False, torch.float32)])
@pytest.mark.parametrize("m,n,k", [(1, 16, 128), (1, 4096, 1024), (2, 33, 64), (5, 7, 100), (17, 129, 192), (16, 256, 4096),
                                   (33, 5001, 256), (64, 384, 320), (300, 200, 384), (129, 257, 1984), (256, 512, 2048),
                                   (4, 1, 1), (3, 130, 130), (100, 1000, 16), (512, 300, 576)])
def test_against_float64(cuda, m, n, k, exact, out):
    (qa, sa), (qw, sw) = _inputs(m * 7 + n, m, n, k, cuda)
    _check(ops.gemm_fp8_block(qa, sa, qw, sw, out_dtype=out, exact=exact), qa, sa, qw, sw, exact)


@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("m,n,k", [(1, 11008, 4096), (16, 8333, 2064), (40, 5001, 1552), (3, 16000, 784), (100, 4100, 912)])
def test_tiles_of_64_by_32(cuda, m, n, k, exact):
    """Few rows of many outputs: K over six waves, more than one turn of each wave's ring."""
    (qa, sa), (qw, sw) = _inputs(m + n, m, n, k, cuda)
    y = ops.gemm_fp8_block(qa, sa, qw, sw, out_dtype=torch.float32 if exact else torch.bfloat16, exact=exact)
    _check(y, qa, sa, qw, sw, exact)


@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("m,n,k", [(700, 4096, 4096), (1500, 1408, 1024), (2048, 2049, 512), (4096, 2048, 1088)])
def test_large(cuda, m, n, k, exact):
    (qa, sa), (qw, sw) = _inputs(5, m, n, k, cuda)
    y = ops.gemm_fp8_block(qa, sa, qw, sw, exact=exact)
    f8 = torch.float8_e4m3fn
    ref = (qa.view(f8).float().double() * _up(sa, 1, m, k)) @ (qw.view(f8).float().double() * _up(sw, 128, n, k)).t()
    assert ((y.double() - ref).norm() / ref.norm()).item() <= 2.5e-3
    # rows and columns of every tile edge by themselves
    rows = sorted({0, 1, 31, 32, 63, 64, 127, 128, 191, 192, 255, 256, m - 2, m - 1})
    cols = sorted({0, 1, 31, 32, 63, 64, 127, 128, 191, 192, 255, 256, n - 2, n - 1})
    _check_part = (y.double() - ref)[rows][:, cols].abs()
    scale = ref.abs().mean().item()
    assert _check_part.max().item() <= 0.03 * max(scale, ref[rows][:, cols].abs().max().item())


@pytest.mark.parametrize("m", [1, 40, 700])
def test_rows_do_not_depend_on_each_other(cuda, m):
    """NaN in a row of x, or in a row of w, stays in its row, or column, of the product."""
    n, k = 300, 512
    (qa, sa), (qw, sw) = _inputs(9, m, n, k, cuda)
    ref = ops.gemm_fp8_block(qa, sa, qw, sw)
    qa2, qw2 = qa.clone(), qw.clone()
    qa2[m // 2, 77] = 0x7F
    qw2[123, 400] = 0x7F
    y = ops.gemm_fp8_block(qa2, sa, qw2, sw)
    bad = torch.zeros_like(ref, dtype=torch.bool)
    bad[m // 2] = bad[:, 123] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], ref[~bad])


def test_unaligned_operands(cuda):
    """Operands that start anywhere take another kernel, with the same result up to rounding."""
    (qa, sa), (qw, sw) = _inputs(10, 9, 70, 256, cuda)
    hold = torch.empty(9 * 256 + 3, dtype=torch.uint8, device=cuda)
    qa2 = hold[3:].view(9, 256).copy_(qa)
    _check(ops.gemm_fp8_block(qa2, sa, qw, sw, out_dtype=torch.float32, exact=True), qa, sa, qw, sw, True)
    big = torch.empty(9 * 70 + 1, dtype=torch.bfloat16, device=cuda)
    out = big[1:].view(9, 70)
    assert torch.equal(ops.gemm_fp8_block(qa, sa, qw, sw, out=out), ops.gemm_fp8_block(qa, sa, qw, sw))
    shifted = torch.empty(sw.numel() + 1, device=cuda)[1:].view(sw.shape).copy_(sw)
    assert torch.equal(ops.gemm_fp8_block(qa, sa, qw, shifted), ops.gemm_fp8_block(qa, sa, qw, sw))


def test_other_stream_and_graph(cuda):
    (qa, sa), (qw, sw) = _inputs(11, 60, 512, 1024, cuda)
    ref = ops.gemm_fp8_block(qa, sa, qw, sw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = ops.gemm_fp8_block(qa, sa, qw, sw)
    s.synchronize()
    assert torch.equal(y, ref)
    out = torch.empty_like(ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.gemm_fp8_block(qa, sa, qw, sw, out=out)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)


def test_refusals(cuda):
    (qa, sa), (qw, sw) = _inputs(12, 4, 130, 256, cuda)
    for bad in (dict(qa=qa[:, :128]), dict(sa=sa[:, :1]), dict(sw=sw[:1]), dict(sw=sw.t()), dict(qw=qw.float()),
                dict(sa=sa.double()), dict(out=torch.empty((4, 129), device=cuda)), dict(out_dtype=torch.float16),
                dict(qa=qa.cpu()), dict(sa=sa.view(-1))):
        with pytest.raises(ValueError):
            ops.gemm_fp8_block(**{"qa": qa, "sa": sa, "qw": qw, "sw": sw, **bad})


def test_empty(cuda):
    (qa, sa), (qw, sw) = _inputs(13, 4, 130, 256, cuda)
    assert ops.gemm_fp8_block(qa[:0], sa[:0], qw, sw).shape == (0, 130)
    e = torch.empty((3, 0), dtype=torch.uint8, device=cuda)
    z = torch.empty((3, 0), device=cuda)
    assert torch.equal(ops.gemm_fp8_block(e, z, e, z[:1]), torch.zeros((3, 3), device=cuda, dtype=torch.bfloat16))


def test_more_outputs_than_a_launch_of_work_items(cuda):
    """2^32 outputs and some of the plain kernel (K is no multiple of 16): rows come out as they do alone."""
    m, n, k = 2**16 + 3, 2**16, 8
    g = torch.Generator(device=cuda).manual_seed(33)
    qa, qw = (torch.randint(0, 120, (r, k), generator=g, device=cuda, dtype=torch.uint8) for r in (m, n))
    sa, sw = torch.rand((m, 1), generator=g, device=cuda), torch.rand((n // 128, 1), generator=g, device=cuda)
    y = ops.gemm_fp8_block(qa, sa, qw, sw)
    for r in (slice(0, 3), slice(2**15 - 1, 2**15 + 2), slice(2**16 - 2, m)):
        assert torch.equal(y[r], ops.gemm_fp8_block(qa[r].contiguous(), sa[r].contiguous(), qw, sw))


def test_refuses_more_tiles_than_a_launch(cuda):
    n, k = 2**30, 16
    qw, sw = torch.zeros((n, k), dtype=torch.uint8, device=cuda), torch.zeros((n // 128, 1), device=cuda)
    with pytest.raises(ffi.CastForgeHipError, match="too many tiles"):
        ops.gemm_fp8_block(qw[:1], sw[:1], qw, sw)


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(3600, 4104, 592), (3700, 4099, 400), (3300, 3500, 912)])
def test_tiles_of_256(cuda, m, n, k, out):
    """The tiles of the largest products, cut in M, N and K: more than a round of 128 x 128 ones, at most one of 256 x 256."""
    (qa, sa), (qw, sw) = _inputs(m + k, m, n, k, cuda)
    _check(ops.gemm_fp8_block(qa, sa, qw, sw, out_dtype=out), qa, sa, qw, sw, False)


@pytest.mark.parametrize("m,n,k,exact", [(1000, 4100, 400, False), (1000, 4100, 400, True), (3600, 4104, 400, False), (3700, 4099, 592, False)])
def test_large_tiles_keep_rows_apart(cuda, m, n, k, exact):
    """NaN in a row of x, or in a row of w, stays in its row, or column, of a product by 128 x 128 and 256 x 256 tiles."""
    (qa, sa), (qw, sw) = _inputs(14, m, n, k, cuda)
    ref = ops.gemm_fp8_block(qa, sa, qw, sw, exact=exact)
    qa2, qw2 = qa.clone(), qw.clone()
    rows, cols = [5, m // 2, m - 1], [0, 1234, n - 1]
    for i, (r, c) in enumerate(zip(rows, cols)):
        qa2[r, 130 * i] = 0x7F
        qw2[c, k - 1 - 100 * i] = 0x7F
    y = ops.gemm_fp8_block(qa2, sa, qw2, sw, exact=exact)
    bad = torch.zeros_like(ref, dtype=torch.bool)
    bad[rows] = True
    bad[:, cols] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], ref[~bad])
