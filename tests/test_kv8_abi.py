"""Refusals of the 8-bit cache's entry points (status 1 and a message, before the device is touched) and their empty
calls; no GPU needed."""
import ctypes

import pytest

from castforge_amd import ffi
from test_abi import _status


def _cache(**kw):
    f = dict(num_pages=4, kv_heads=2, page_size=16, head_dim=128, k_codes=16, k_scales=16, v_codes=16, v_scales=16)
    f.update(kw)
    return ctypes.byref(ffi.Kv8CacheStruct(**f))


def _append(cache=None, k=16, ks=256, v=16, vs=256, n=1, b=1, cu=None, table=16, cols=4, lens=16, pos=16, cos=16, sin=16, max_pos=8, rot=128,
            interleaved=0, q=None, qs=0, hq=0, q_out=None):
    return ("castforge_hip_kv8_append", cache or _cache(), k, ks, v, vs, n, b, cu, table, cols, lens, pos, cos, sin, max_pos, rot, interleaved, q, qs, hq,
            q_out, None)


def _gather(cache=None, slots=16, n=3, k=16, v=16, dtype=1):
    return ("castforge_hip_kv8_gather", cache or _cache(), slots, n, k, v, dtype, None)


def _attention(cache=None, q=16, qs=512, n=1, hq=4, b=1, cu=None, table=16, cols=4, lens=16, causal=1, window=0, sinks=0, out=16, lse=None, weights=None,
               wcols=0, ws=16, size=1 << 30):
    return ("castforge_hip_kv8_attention", cache or _cache(), q, qs, n, hq, b, cu, table, cols, lens, causal, window, sinks, 0.1, out, lse, weights, wcols,
            ws, size, None)


def _evict(cache=None, table=16, cols=4, lens=16, b=1, w=16, wcols=64, keep=20, sinks=0, recent=0, new=16, ncols=2, kept=16, nlens=16, nw=None):
    return ("castforge_hip_kv8_evict", cache or _cache(), table, cols, lens, b, w, wcols, keep, sinks, recent, new, ncols, kept, nlens, nw, None)


@pytest.mark.parametrize("call,needle", [
    (("castforge_hip_kv8_append", None, *_append()[2:]), "cache"),
    (_append(_cache(head_dim=96)), "head_dim"),
    (_append(_cache(page_size=20)), "page_size"),
    (_append(_cache(page_size=8)), "page_size"),
    (_append(_cache(page_size=512)), "page_size"),
    (_append(_cache(kv_heads=0)), "kv_heads"),
    (_append(_cache(num_pages=-1)), "num_pages"),
    (_append(_cache(k_codes=None)), "NULL"),
    (_append(_cache(v_scales=None)), "NULL"),
    (_append(_cache(v_codes=20)), "aligned"),
    (_append(_cache(k_scales=18)), "aligned"),
    (_append(rot=24), "rot"),
    (_append(rot=144), "rot"),
    (_append(interleaved=3), "interleaved"),
    (_append(n=2, b=2, ks=100), "stride"),
    (_append(n=2, b=2, vs=260), "stride"),
    (_append(k=18), "aligned"),
    (_append(pos=None), "positions"),
    (_append(cos=20), "aligned"),
    (_append(q=16, qs=256, hq=2), "q_out"),
    (_append(q=16, q_out=16, hq=0), "q_heads"),
    (_append(q=16, qs=256, hq=2, q_out=8), "aligned"),
    (_append(n=2, ks=256), "batch"),
    (_append(n=-1), "tokens"),
    (_append(b=-1, cu=16), "batch"),
    (_append(cols=1 << 28), "2^31"),
    (_append(lens=None), "NULL"),
    (_append(table=None), "NULL"),
    (_append(v=None), "NULL"),
    (_gather(dtype=4), "out_dtype"),
    (_gather(k=8), "aligned"),
    (_gather(n=-3), "tokens"),
    (_gather(slots=None), "NULL"),
    (_attention(hq=3), "q_heads"),
    (_attention(hq=130), "q_heads"),
    (_attention(b=2), "batch"),
    (_attention(causal=2), "causal"),
    (_attention(causal=0, window=4), "causal"),
    (_attention(window=-1), "window"),
    (_attention(window=1 << 31), "window"),
    (_attention(sinks=-1), "sinks"),
    (_attention(sinks=1 << 31), "sinks"),
    (_attention(lens=None), "NULL"),
    (_attention(out=None), "NULL"),
    (_attention(weights=16, wcols=4), "lse"),
    (_attention(weights=16, lse=16, wcols=-1), "weights_cols"),
    (_attention(q=20), "aligned"),
    (_attention(n=2, b=2, qs=200), "stride"),
    (_attention(cols=1 << 28), "2^31"),
    (_attention(n=1 << 30, b=1 << 30), "2^31"),
    (_evict(_cache(page_size=20)), "page_size"),
    (_evict(b=-1), "batch"),
    (_evict(cols=1 << 28), "2^31"),
    (_evict(wcols=-1), "weights_cols"),
    (_evict(keep=0), "keep"),
    (_evict(keep=1 << 31), "keep"),
    (_evict(sinks=-1), "sinks"),
    (_evict(sinks=11, recent=10), "together"),
    (_evict(keep=33), "new_table"),
    (_evict(ncols=1 << 28), "new_table"),
    (_evict(lens=None), "NULL"),
    (_evict(w=None), "NULL"),
    (_evict(kept=None), "NULL"),
    (_evict(nlens=None), "NULL"),
    (("castforge_hip_kv8_attention_workspace", _cache(), 1, 4, 1, 4, 0, 0, 0, 0, None), "out_bytes"),
])
def test_invalid_arguments_report_status_1(call, needle):
    rc, msg = _status(*call)
    assert rc == 1 and msg and needle in msg, (rc, msg)


def test_empty_calls_are_noops():
    nothing = dict(n=0, b=0, lens=None, table=None)
    for call in (_append(**nothing, k=None, v=None, rot=0), _append(n=0, b=3, cu=16), _append(n=3, b=0, cu=16, ks=256), _gather(n=0, slots=None, k=None, v=None),
                 _attention(**nothing, q=None, out=None), _attention(n=0, b=3, cu=16), _attention(n=3, b=0, cu=16), _evict(b=0, lens=None, table=None, kept=None)):
        assert _status(*call)[0] == 0
