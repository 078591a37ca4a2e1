"""What attention with changed scores and masks refuses, on the host."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mlx_batch_invariant_amd as bi
from mlx_batch_invariant_amd import _lib


def _qkv(B=2, Hq=4, Hkv=2, T=3, L=8, D=64):
    return torch.zeros(B, Hq, T, D), torch.zeros(B, Hkv, L, D), torch.zeros(B, Hkv, L, D)


@pytest.mark.parametrize("kw,match", [
    (dict(softcap=5.0), "GPU"), (dict(softcap=5.0, order="per_key"), "matrix-core order"),
    (dict(softcap=5.0, split_size=128), "matrix-core order"), (dict(softcap=5.0, mask="prefix"), "mask must be")])
def test_contiguous_arguments(kw, match):
    with pytest.raises(ValueError, match=match):
        bi.batch_invariant_attention(*_qkv(), **kw)


def test_shapes():
    q, k, v = _qkv()
    for bad in ((q, k, v[:, :1]), (q, k[:1], v[:1]), (q[:, :3], k, v), (q, k[..., :32], v[..., :32])):
        with pytest.raises(ValueError, match="unsupported shapes"):
            bi.batch_invariant_attention(*bad, softcap=5.0)
    q, k, v = _qkv(D=160)
    with pytest.raises(ValueError, match="matrix-core order"):
        bi.batch_invariant_attention(q, k, v, softcap=5.0)
    q, k, v = _qkv(T=9)
    with pytest.raises(ValueError, match="T_q <= L"):
        bi.batch_invariant_attention(q, k, v, mask="causal", softcap=5.0)


def _scored(q, **kw):
    """The checks behind the device check, which CPU tensors do not pass."""
    from mlx_batch_invariant_amd.kernels.attention import _scored
    a = dict(softcap=None, slopes=None, doc_ids=None, prefix_lens=None) | kw
    return _scored("x", q, *_qkv()[1:], None, 0, 0, 8, None, 1.0, a.pop("causal", True), **a)


@pytest.mark.parametrize("kw,match", [
    (dict(softcap=0.0), "softcap"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("inf")), "softcap"),
    (dict(softcap=float("nan")), "softcap"), (dict(slopes=[1.0, 2.0]), "slopes"),
    (dict(slopes=torch.zeros(4, 1)), "slopes"), (dict(doc_ids=torch.zeros(2, 8)), "doc_ids"),
    (dict(doc_ids=torch.zeros(2, 7, dtype=torch.int32)), "doc_ids"),
    (dict(doc_ids=torch.zeros(8, dtype=torch.int32)), "doc_ids"),
    (dict(doc_ids=torch.zeros(2, 8, dtype=torch.int32)), "GPU"),
    (dict(prefix_lens=[1, 2], causal=False), "causal"), (dict(prefix_lens=[1, 2, 3]), "entries")])
def test_modifiers(kw, match):
    with pytest.raises(ValueError, match=match):
        _scored(_qkv()[0], **kw)


def test_abi():
    lib = _lib.load()
    p = ctypes.c_void_p(256)                             # never dereferenced: validation fails first
    st = (ctypes.c_int64 * 9)(*([128] * 9))
    M = _lib.ScoreMod

    def call(mod, **k):
        return lib.bi_attn_scored(*(k.get(n, d) for n, d in (
            ("q", p), ("k", p), ("v", p), ("table", None), ("stride", 0), ("page", 0), ("pages", 0), ("lens", None),
            ("out", p), ("B", 1), ("Hq", 4), ("Hkv", 2), ("Tq", 4), ("L", 300), ("D", 128), ("st", st), ("causal", 1),
            ("scale", 1.0))), None if mod is None else ctypes.byref(mod), k.get("dt", 2), k.get("ws"), k.get("n", 0),
            None)

    assert call(None) == -1
    for bad in (M(softcap=-1.0), M(softcap=float("nan")), M(softcap=float("inf")), M(doc_ids=256, doc_stride=299)):
        assert call(bad) == -1
    assert call(M(prefix_lens=256), causal=0) == -1
    assert call(M(softcap=1.0), Tq=0) == -1 and call(M(softcap=1.0), Tq=301) == -1 and call(M(softcap=1.0), q=None) == -1
    assert call(M(softcap=1.0), D=160) == -2 and call(M(softcap=1.0), dt=3) == -2
    assert call(M(slopes=256), L=(1 << 24) + 1) == -2
    assert call(M(softcap=1.0), table=p, page=12, pages=9, stride=99) == -1
    docs = M(doc_ids=256, doc_stride=300)
    size = lib.bi_attn_scored_workspace_bytes
    need = size(1, 4, 2, 4, 300, 128, 1, 1, 2)           # few rows: partials of 16 rows and 2 splits
    assert need == (2 * 32 + 32 * 128) * 4 and call(docs) == -3 and call(docs, ws=p, n=need - 1) == -3
    assert call(docs, ws=ctypes.c_void_p(264), n=need) == -3
    assert size(3, 4, 2, 1, 300, 128, 0, 1, 2) == lib.bi_attn_decode_workspace_bytes(3, 4, 300, 128)
    assert size(1, 4, 2, 4, 256, 128, 1, 1, 2) == 8 and size(1, 4, 2, 4, 256, 128, 1, 0, 2) == 0     # one split
    assert size(4, 32, 8, 2048, 2048, 128, 1, 1, 2) == 4 * 8 * 8 and size(4, 32, 8, 2048, 2048, 128, 1, 0, 2) == 0
    assert size(1, 32, 8, 16, 1 << 20, 128, 1, 0, 0) == 0                   # partials over 256 MB
    assert size(1, 4, 3, 4, 300, 128, 1, 1, 2) == 0
    assert call(docs, Tq=1) == -3 and call(M(softcap=1.0), B=0) == 0 and call(M(softcap=1.0), B=0, Tq=1) == 0


def test_operators_are_registered():
    for name in ("scored_attention", "scored_paged_attention"):
        assert str(getattr(torch.ops.mlx_bi, name).default._schema).startswith(f"mlx_bi::{name}(")
    with FakeTensorMode():
        q, k, v = _qkv()
        assert torch.ops.mlx_bi.scored_attention(q, k, v, 1.0, True, None, 5.0, None, None, None).shape == q.shape
        t = torch.empty(2, 3, dtype=torch.int32)
        pool = torch.empty(9, 2, 16, 64)
        assert torch.ops.mlx_bi.scored_paged_attention(q, pool, pool, t, None, 1.0, True, 5.0, None, None,
                                                       None).shape == q.shape
