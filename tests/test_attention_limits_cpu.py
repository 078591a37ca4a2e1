"""Attention calls whose launch would hold 2^32 threads or more are refused (such a
grid wraps without an error); checked on the host, before anything is launched."""

import ctypes

import pytest

from mlx_batch_invariant_amd import _lib

P = ctypes.c_void_p(256)                                 # never dereferenced
BIG = 1 << 62                                            # workspace bytes that are enough
ST = (ctypes.c_int64 * 9)(*([128] * 9))


def _error(rc):
    assert rc == -2, rc
    return _lib.load().bi_last_error().decode()


def _prefill(B, Hq, Hkv, Tq, L, D, scored=False, docs=False, causal=0):
    lib = _lib.load()
    if not scored:
        return lib.bi_attn_prefill(P, P, P, None, P, B, Hq, Hkv, Tq, L, D, ST, causal, 1.0, 0, None)
    m = _lib.ScoreMod(softcap=0.0 if docs else 5.0, doc_ids=256 if docs else None, doc_stride=L)
    return lib.bi_attn_scored(P, P, P, None, 0, 0, 0, None, P, B, Hq, Hkv, Tq, L, D, ST, causal, 1.0, ctypes.byref(m), 0,
                              P, BIG, None)


@pytest.mark.parametrize("scored", [False, True])
def test_prefill_rows(scored):
    # 64 rows a workgroup, 256 threads each
    for B, Hq, Hkv, Tq in ((1024, 16, 16, 1 << 16), (1, 64, 1, 1 << 24), (65535, 512, 512, 64)):
        assert "grid too large" in _error(_prefill(B, Hq, Hkv, Tq, 1 << 17, 32, scored))


def test_document_ranges():
    assert "grid too large" in _error(_prefill(1024, 1, 1, 64, 1 << 24, 32, True, docs=True))


@pytest.mark.parametrize("per_key", [False, True])
def test_decode_merge(per_key):
    lib, a = _lib.load(), (P, P, P, None, P, 65535, 1025, 1025, 300, 64, ST, 1.0, 0)
    if per_key:
        rc = lib.bi_attn_decode_per_key(*a[:10], ST, 1.0, 256, 0, P, BIG, None)
    else:
        rc = lib.bi_attn_decode(*a, P, BIG, None)
    assert "grid too large" in _error(rc)
    if not per_key:
        m = _lib.ScoreMod(softcap=5.0)
        rc = lib.bi_attn_scored(P, P, P, None, 0, 0, 0, None, P, 65535, 1025, 1025, 1, 300, 64, ST, 0, 1.0,
                                ctypes.byref(m), 0, P, BIG, None)
        assert "grid too large" in _error(rc)
