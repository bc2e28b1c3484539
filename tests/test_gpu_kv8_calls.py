"""Calls over the paged 8-bit cache that test_gpu_kv8_attention.py does not make, and what its comparison of weights lets through: NaN."""
import pytest
import torch

import test_gpu_kv8 as append
import test_gpu_kv8_attention as attention
from castforge_amd import ffi, ops
from test_gpu_kv8_missing_pages import FORMS, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", [
    lambda cuda: attention.test_windows_and_pages(cuda, 16, 33, 0),
    lambda cuda: attention.test_windows_and_pages(cuda, 256, 128, 3),
    lambda cuda: attention.test_head_layouts(cuda, 7),
    lambda cuda: attention.test_prompts(cuda, 128, 8, 4, [1500, 900], [1500, 1700], 64, None, 0),
    lambda cuda: attention.test_prompts(cuda, 64, 8, 4, [2048, 700], [2048, 800], 32, 200, 4),
    lambda cuda: attention.test_prompts_through_windows_of_every_kind(cuda, 129, 33, 128),
    lambda cuda: attention.test_without_causal_order(cuda),
    lambda cuda: attention.test_more_queries_than_tokens_and_none(cuda),
    lambda cuda: attention.test_many_sequences(cuda),
    lambda cuda: attention.test_long_sequences_are_split(cuda),
    lambda cuda: attention.test_scales_of_the_whole_range(cuda, -20, 50),
    lambda cuda: attention.test_large_scores(cuda, [1500], [1500]),
    lambda cuda: attention.test_large_scores(cuda, [1, 1], [900, 300]),
    lambda cuda: attention.test_weights_shorter_and_longer_than_the_table(cuda),
], ids=str)
def test_weights_are_numbers(cuda, monkeypatch, case):
    """Those tests' caches hold NaN wherever no token lies."""
    call, calls = ops.kv8_attention, []

    def checked(*args, **kw):
        got = call(*args, **kw)
        if kw.get("weights") is not None:
            assert torch.isfinite(kw["weights"]).all()
            calls.append(1)
        return got

    monkeypatch.setattr(ops, "kv8_attention", checked)
    case(cuda)
    assert calls


@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 20)])
@pytest.mark.parametrize("q_lens,kv_lens", FORMS)
def test_what_a_workspace_held_is_not_read(cuda, q_lens, kv_lens, window, sinks):
    """And the same call gives the same bits again."""
    case = Case(cuda, q_lens, kv_lens, [(0, 16, 32)], seed=1, window=window, sinks=sinks)
    want = case.call()
    t, hq, d = case.q.shape
    b, cols = case.table.shape
    size = ops._kv8_workspace(0, case.cache.kv_heads, case.page, d, t, hq, b, cols, 0 if case.cu is None else 1, window or 0, sinks, 1)
    for byte in (0xFF, 0x00, 0x7F):
        ws = torch.full((max(size, 1),), byte, dtype=torch.uint8, device=cuda)
        out, lse, weights = torch.full_like(case.q, 7.0), torch.full((t, hq), 7.0, device=cuda), case.before.clone()
        ffi.call("castforge_hip_kv8_attention", case.cache._ref, case.q.data_ptr(), hq * d, t, hq, b, None if case.cu is None else case.cu.data_ptr(),
                 case.table.data_ptr(), cols, case.lens.data_ptr(), 1, window or 0, sinks, d ** -0.5, out.data_ptr(), lse.data_ptr(), weights.data_ptr(),
                 weights.shape[2], ws.data_ptr() if size else None, size, torch.cuda.current_stream().cuda_stream)
        for x, y in zip((out, lse, weights), want):
            assert torch.equal(x, y)


def test_caches_of_no_heads_are_refused(cuda):
    q, i32 = torch.zeros((1, 4, 64), dtype=torch.bfloat16, device=cuda), dict(dtype=torch.int32, device=cuda)
    table, lens = torch.zeros((1, 1), **i32), torch.ones(1, **i32)
    for call, cache in ((ops.kv8_attention, ops.Kv8Cache.empty(1, 0, 16, 64, device=cuda)), (ops.kv4_attention, ops.Kv4Cache.empty(1, 0, 16, 64, 32, device=cuda))):
        with pytest.raises(ValueError, match="heads"):
            call(q, cache, table, lens)


def test_a_table_of_no_dimensions_is_refused(cuda):
    cache, i32 = ops.Kv8Cache.empty(1, 1, 16, 64, device=cuda), dict(dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError, match="page_table"):
        ops.kv8_evict(cache, torch.tensor(0, **i32), torch.ones(1, **i32), torch.ones((1, 1, 16), device=cuda), 4, torch.zeros((1, 1), **i32))


@pytest.mark.parametrize("interleaved", [False, True])
def test_queries_of_nan_and_infinity_are_rotated_as_others(cuda, interleaved):
    """NaN wherever f32 gives it (whatever its bits), every other number bit for bit, where the cache holds what it holds without queries."""
    g = torch.Generator().manual_seed(1)
    rows = torch.randn((40, 7, 128), generator=g)
    at = torch.rand(rows.shape, generator=g)
    for i, value in enumerate((float("nan"), float("inf"), -float("inf"), 3e38, 1e-38, -0.0)):
        rows[:, :5][(at[:, :5] > 0.03 * i) & (at[:, :5] < 0.03 * i + 0.01)] = value
    rows = rows.bfloat16()
    angle = torch.arange(50)[:, None] * 10000.0 ** (-torch.arange(64) / 64)
    i32, dev = dict(dtype=torch.int32, device=cuda), rows.to(cuda)
    caches, lists = [ops.Kv8Cache.empty(3, 1, 16, 128, device=cuda) for _ in range(2)], (torch.tensor([[2, 0, 1]], **i32), torch.tensor([40], **i32))
    turn = dict(cu_q=torch.tensor([0, 40], **i32), positions=torch.arange(40, device=cuda), cos=angle.cos().to(cuda), sin=angle.sin().to(cuda), interleaved=interleaved)
    got = ops.kv8_append(caches[0], dev[:, 5:6], dev[:, 6:], *lists, q=dev[:, :5], **turn).cpu()
    assert ops.kv8_append(caches[1], dev[:, 5:6], dev[:, 6:], *lists, **turn) is None
    want = append._rotate(rows[:, :5].float(), angle.cos()[:40], angle.sin()[:40], 128, interleaved).bfloat16()
    nan = torch.isnan(want)
    assert nan.any() and torch.equal(torch.isnan(got), nan)
    assert torch.equal(got.view(torch.int16)[~nan], want.view(torch.int16)[~nan])
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        assert torch.equal(getattr(caches[0], name), getattr(caches[1], name))


@pytest.mark.parametrize("extra", [60, 250, 2040])
@pytest.mark.parametrize("q_lens,kv_lens", [([1], [1009]), ([1] * 24, [500] * 24), ([1, 1], [0, 1]), ([5, 2], [300, 9]), ([512], [512]), ([900, 3], [1600, 3])])
def test_tables_wider_than_the_lengths(cuda, monkeypatch, q_lens, kv_lens, extra):
    """Which form a call takes goes by the table's width; what it gives, by the lengths."""
    def case(cuda):
        attention._run(cuda, q_lens, kv_lens, 8, 4, 128, 64, seed=extra, extra_cols=extra)
        attention._run(cuda, q_lens, kv_lens, 2, 3, 64, 64, seed=extra, extra_cols=extra, window=100, sinks=4)

    test_weights_are_numbers(cuda, monkeypatch, case)
