"""Refusals of the decoder layer's entry points (status 1 and a message, before the device is touched) and
their empty calls; no GPU needed."""
import ctypes

import pytest

from castforge_amd import ffi
from test_abi import _status


def _cache(**kw):
    f = dict(num_pages=4, kv_heads=2, page_size=16, head_dim=128, group=64, k_codes=16, k_groups=16, v_codes=16, v_groups=16)
    f.update(kw)
    return ctypes.byref(ffi.Kv4CacheStruct(**f))


NORM = "castforge_hip_rms_norm_fp8"
APPEND, GATHER, ATTN, SIZE = (f"castforge_hip_kv4_{n}" for n in ("append", "gather", "attention", "attention_workspace"))


@pytest.mark.parametrize("call,needle", [
    ((NORM, 16, 7, None, 16, 0, 1e-6, 1, 128, 0, None, 16, 16, None), "x_dtype"),
    ((NORM, 16, 1, None, 16, 9, 1e-6, 1, 128, 0, None, 16, 16, None), "weight_dtype"),
    ((NORM, 16, 1, None, 16, 0, 1e-6, 1, 128, 64, None, 16, 16, None), "block"),
    ((NORM, 16, 1, 16, 16, 0, 1e-6, 1, 128, 0, None, 16, 16, None), "residual"),
    ((NORM, 16, 1, None, 16, 0, -1.0, 1, 128, 0, None, 16, 16, None), "eps"),
    ((NORM, 16, 1, None, 16, 0, float("nan"), 1, 128, 0, None, 16, 16, None), "eps"),
    ((NORM, None, 1, None, 16, 0, 1e-6, 1, 128, 0, None, 16, 16, None), "NULL"),
    ((NORM, 16, 1, None, 16, 0, 1e-6, -1, 128, 0, None, 16, 16, None), "non-negative"),
    (("castforge_hip_quantize_fp8_block", 16, 1, 2, 128, 2, 16, 16, None), "block_rows"),
    (("castforge_hip_quantize_fp8_block", 16, 3, 2, 128, 1, 16, 16, None), "src_dtype"),
    (("castforge_hip_quantize_fp8_block", None, 1, 2, 128, 1, 16, 16, None), "NULL"),
    (("castforge_hip_dequantize_fp8_block", 16, 16, 2, 128, 3, 16, None), "block_rows"),
    (("castforge_hip_gemm_fp8_block", 16, 16, 1, 16, 16, 16, 128, 16, 5, 0, None), "y_dtype"),
    (("castforge_hip_gemm_fp8_block", 16, 16, 1, 16, 16, 16, 128, 16, 0, 2, None), "exact"),
    (("castforge_hip_gemm_fp8_block", 16, 16, -1, 16, 16, 16, 128, 16, 0, 0, None), "non-negative"),
    (("castforge_hip_gemm_fp8_block", 16, None, 1, 16, 16, 16, 128, 16, 0, 0, None), "NULL"),
    ((APPEND, None, 16, 256, 16, 256, 1, 16, 16, 16, 16, 8, 128, 0, None, 0, 0, None, None), "cache"),
    ((APPEND, _cache(head_dim=96), 16, 256, 16, 256, 1, 16, 16, 16, 16, 8, 128, 0, None, 0, 0, None, None), "head_dim"),
    ((APPEND, _cache(group=48), 16, 256, 16, 256, 1, 16, 16, 16, 16, 8, 128, 0, None, 0, 0, None, None), "group"),
    ((APPEND, _cache(page_size=20), 16, 256, 16, 256, 1, 16, 16, 16, 16, 8, 128, 0, None, 0, 0, None, None), "page_size"),
    ((APPEND, _cache(k_codes=None), 16, 256, 16, 256, 1, 16, 16, 16, 16, 8, 128, 0, None, 0, 0, None, None), "NULL"),
    ((APPEND, _cache(v_groups=20), 16, 256, 16, 256, 1, 16, 16, 16, 16, 8, 128, 0, None, 0, 0, None, None), "aligned"),
    ((APPEND, _cache(), 16, 256, 16, 256, 1, 16, 16, 16, 16, 8, 24, 0, None, 0, 0, None, None), "rot"),
    ((APPEND, _cache(), 16, 256, 16, 256, 1, 16, 16, 16, 16, 8, 128, 3, None, 0, 0, None, None), "interleaved"),
    ((APPEND, _cache(), 16, 100, 16, 256, 2, 16, 16, 16, 16, 8, 128, 0, None, 0, 0, None, None), "stride"),
    ((APPEND, _cache(), 18, 256, 16, 256, 1, 16, 16, 16, 16, 8, 128, 0, None, 0, 0, None, None), "aligned"),
    ((APPEND, _cache(), 16, 256, 16, 256, 1, 16, None, 16, 16, 8, 128, 0, None, 0, 0, None, None), "positions"),
    ((APPEND, _cache(), 16, 256, 16, 256, 1, 16, 16, 16, 16, 8, 128, 0, 16, 256, 2, None, None), "q_out"),
    ((GATHER, _cache(), 16, 3, 16, 16, 4, None), "out_dtype"),
    ((GATHER, _cache(), 16, 3, 8, 16, 1, None), "aligned"),
    ((GATHER, _cache(), 16, -3, 16, 16, 1, None), "tokens"),
    ((ATTN, _cache(), 16, 512, 1, 3, 1, None, 16, 4, 16, 1, 0.1, 16, None, 16, 1 << 30, None), "q_heads"),
    ((ATTN, _cache(), 16, 512, 1, 4, 2, None, 16, 4, 16, 1, 0.1, 16, None, 16, 1 << 30, None), "batch"),
    ((ATTN, _cache(), 16, 512, 1, 4, 1, None, 16, 4, 16, 2, 0.1, 16, None, 16, 1 << 30, None), "causal"),
    ((ATTN, _cache(), 16, 512, 1, 4, 1, None, 16, 4, None, 1, 0.1, 16, None, 16, 1 << 30, None), "NULL"),
    ((ATTN, _cache(), 20, 512, 1, 4, 1, None, 16, 4, 16, 1, 0.1, 16, None, 16, 1 << 30, None), "aligned"),
    ((ATTN, _cache(), 16, 200, 2, 4, 2, None, 16, 4, 16, 1, 0.1, 16, None, 16, 1 << 30, None), "stride"),
    ((ATTN, _cache(), 16, 512, 1, 4, 1, None, 16, 1 << 28, 16, 1, 0.1, 16, None, 16, 1 << 30, None), "2^31"),
    ((SIZE, _cache(), 1, 4, 1, 4, 0, None), "out_bytes"),
])
def test_invalid_arguments_report_status_1(call, needle):
    rc, msg = _status(*call)
    assert rc == 1 and msg and needle in msg, (rc, msg)


def test_empty_calls_are_noops():
    assert _status(NORM, None, 1, None, None, 0, 1e-6, 0, 128, 0, None, None, None, None)[0] == 0
    assert _status("castforge_hip_quantize_fp8_block", None, 1, 0, 128, 1, None, None, None)[0] == 0
    assert _status("castforge_hip_gemm_fp8_block", None, None, 0, None, None, 16, 128, None, 0, 0, None)[0] == 0
    assert _status(APPEND, _cache(), None, 0, None, 0, 0, None, None, None, None, 0, 0, 0, None, 0, 0, None, None)[0] == 0
    assert _status(GATHER, _cache(), None, 0, None, None, 1, None)[0] == 0
    assert _status(ATTN, _cache(), None, 0, 0, 4, 0, None, None, 0, None, 1, 0.1, None, None, None, 0, None)[0] == 0
