"""What the quantized cache's calls and shared-prefix attention refuse, on the host
(nothing is launched), their workspaces, and the library operators' fake shapes."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mlx_batch_invariant_amd as bi
from mlx_batch_invariant_amd import _lib

I32 = torch.int32
P = ctypes.c_void_p(256)                                 # never dereferenced
BIG = 1 << 62                                            # workspace bytes that are enough


def _pool(n=5, H=2, page=8, D=64, **kw):
    return bi.quantized_pages(n, H, page, D, device="cpu", dtype=torch.float32, **kw)


def _write(**change):
    B, T, Hq, Hkv, D = 2, 3, 4, 2, 64
    q, k, v = (torch.zeros(B, T, h, D) for h in (Hq, Hkv, Hkv))
    cs, pos = torch.zeros(9, D // 2), torch.zeros(B, T, dtype=I32)
    return dict(q=q, k=k, v=v, cos=cs, sin=cs.clone(), positions=pos, slots=pos.long(), k_pages=_pool(), v_pages=_pool()) | change


def test_pools():
    p = bi.quantized_pages(3, 2, 16, 128, bits=4, group_size=32, dtype=torch.float16, device="cpu")
    assert p.codes.shape == (3, 2, 16, 64) and p.groups.shape == (3, 2, 16, 4, 2) and p.head_dim == 128
    assert p.codes.view(torch.uint32).shape == (3, 2, 16, 16)
    for kw in (dict(bits=3), dict(group_size=16), dict(group_size=128), dict(dtype=torch.int32)):
        with pytest.raises(ValueError):
            bi.quantized_pages(1, 1, 16, 64, device="cpu", **kw)
    with pytest.raises(ValueError, match="page size"):
        bi.quantized_pages(1, 1, 12, 64, device="cpu")


@pytest.mark.parametrize("change,match", [
    (dict(k=torch.zeros(2, 3, 2, 32)), "shapes"), (dict(v=torch.zeros(2, 3, 1, 64)), "shapes"),
    (dict(k_pages=_pool(H=3), v_pages=_pool(H=3)), "heads"), (dict(k_pages=_pool(D=128), v_pages=_pool(D=128)), "heads"),
    (dict(v_pages=_pool(n=4)), "pools"), (dict(v_pages=_pool(bits=4)), "pools"), (dict(v_pages=_pool(group_size=32)), "pools"),
    (dict(k_pages=torch.zeros(5, 2, 8, 64)), "QuantizedPages"), (dict(q=torch.zeros(2, 3, 4, 64).half()), "type"),
    (dict(k_pages=_pool()._replace(codes=torch.zeros(5, 2, 8, 64))), "uint8"),
    (dict(k_pages=_pool()._replace(groups=torch.zeros(5, 2, 8, 1, 2).half())), "pairs"),
    (dict(k_pages=_pool()._replace(groups=torch.zeros(5, 2, 8, 2, 2))), "pools"),
    (dict(k_pages=_pool(group_size=32)._replace(group_size=64), v_pages=_pool(group_size=32)._replace(group_size=64)), "groups"),
    (dict(k_pages=_pool(page=6 + 2)._replace(codes=torch.zeros(5, 2, 8, 72, dtype=torch.uint8)[..., 4:68])), "aligned"),
    (dict(k_pages=_pool()._replace(groups=torch.zeros(5, 2, 8, 1, 3)[..., :2])), "aligned"),
    (dict(cos=torch.zeros(9, 12), sin=torch.zeros(9, 12)), "multiple of 8"), (dict(cos=torch.zeros(8, 32)), "tables"),
    (dict(slots=torch.zeros(2, 3)), "slots"), (dict(sections=(8, 9)), "sections"), ({}, "GPU")])
def test_write_arguments(change, match):
    with pytest.raises(ValueError, match=match):
        bi.rope_quantized_cache(**_write(**change))


def test_page_sizes():
    odd = _pool()
    odd = [odd._replace(codes=odd.codes[:, :, :6], groups=odd.groups[:, :, :6]) for _ in range(2)]
    with pytest.raises(ValueError, match="page size"):
        bi.rope_quantized_cache(**_write(k_pages=odd[0], v_pages=odd[1]))


def test_read_arguments():
    t = torch.zeros(2, 3, dtype=I32)
    for bad in (t[0], t.float()):
        with pytest.raises(ValueError, match="block table"):
            bi.read_quantized_cache(_pool(), _pool(), bad)
    with pytest.raises(ValueError, match="GPU"):
        bi.read_quantized_cache(_pool(), _pool(), t)
    with pytest.raises(ValueError, match="pools"):
        bi.read_quantized_cache(_pool(), _pool(n=3), t)


def test_attention_arguments():
    call, t = bi.batch_invariant_quantized_paged_attention, torch.zeros(2, 3, dtype=I32)
    q = torch.zeros(2, 4, 1, 64)
    for bad, match in ((q[0], "q"), (q[..., :32], "heads of"), (q.half(), "type"), (q[:, :3], "query heads")):
        with pytest.raises(ValueError, match=match):
            call(bad, _pool(), _pool(), t)
    with pytest.raises(ValueError, match="mask"):
        call(q, _pool(), _pool(), t, mask="sliding")
    with pytest.raises(ValueError, match="block table"):
        call(q, _pool(), _pool(), t[:1])
    with pytest.raises(ValueError, match="GPU"):
        call(q, _pool(), _pool(), t)


def test_shared_arguments():
    call, t = bi.batch_invariant_shared_prefix_attention, torch.zeros(2, 3, dtype=I32)
    q, kp = torch.zeros(2, 4, 1, 64), torch.zeros(5, 2, 8, 64)
    for bad in (kp[0], kp[..., :32], torch.zeros(4, 2, 8, 64)):
        with pytest.raises(ValueError, match="shapes"):
            call(q, kp, bad, t, shared_lens=256)
    with pytest.raises(ValueError, match="type"):
        call(q, kp.half(), kp.half(), t, shared_lens=256)
    with pytest.raises(ValueError, match="shared_lens"):
        call(q, kp, kp, t, shared_lens=None)
    with pytest.raises(ValueError, match="aligned"):
        call(q, torch.zeros(5, 2, 8, 66)[..., :64], kp, t, shared_lens=256)
    with pytest.raises(ValueError, match="page size"):
        call(q, kp[:, :, :6], kp[:, :, :6], t, shared_lens=256)
    with pytest.raises(ValueError, match="GPU"):
        call(q, kp, kp, t, shared_lens=256)


def test_groups_of():
    from mlx_batch_invariant_amd.kernels.quantized_cache import _groups_of
    d, of = torch.device("cpu"), lambda *a: _groups_of("call", 4, *a)
    assert of(None, None, d) == (0, None, None, 0) and of(None, 700, d) == (1, None, None, 700)
    assert of(None, 1 << 40, d)[3] == 0x7fffffff
    n, s, l, x = of([0, 2, 4], [300, 400], d)
    assert (n, s.tolist(), l.tolist(), x) == (2, [0, 2, 4], [300, 400], 0)
    for starts, lens in (([0, 4], None), ([0, 4], 300), (None, [1, 2]), ([0, 4], [1, 2]), ([0, 1, 4], [[1, 2]]), (None, -1),
                         ([0.0, 4.0, 5.0], torch.zeros(2)), (None, torch.zeros(65536, dtype=I32))):
        with pytest.raises(ValueError):
            of(starts, lens, d)


def _pages_call(B=2, Hq=4, Hkv=2, Tq=1, L=512, D=64, bits=8, gs=64, groups=0, starts=None, lens=None, shared=0, page=16,
                pages=9, stride=None, causal=1, dtype=0, strides=(64,) * 15, ws=P, n=BIG, q=P, kg=P):
    st = None if strides is None else (ctypes.c_int64 * 15)(*strides)
    return _lib.load().bi_attn_pages(q, P, kg, P, P, bits, gs, P, L // page if stride is None else stride, page, pages, None,
                                     starts, lens, shared, groups, P, B, Hq, Hkv, Tq, L, D, st, causal, 1.0, dtype, ws, n,
                                     None)


@pytest.mark.parametrize("code,change", [
    (-1, dict(Hq=5)), (-1, dict(B=-1)), (-1, dict(Tq=0)), (-1, dict(L=0)), (-2, dict(D=48)), (-2, dict(D=160)), (-2, dict(dtype=3)),
    (-2, dict(B=65536)), (-1, dict(Tq=513)), (-1, dict(page=24)), (-1, dict(page=0, stride=99)), (-1, dict(pages=0)),
    (-1, dict(pages=1 << 31)), (-1, dict(stride=31)), (-1, dict(groups=2)), (-1, dict(groups=2, starts=P)),
    (-1, dict(groups=1, shared=-1)), (-1, dict(q=None)), (-1, dict(q=ctypes.c_void_p(264))), (-1, dict(strides=None)),
    (-1, dict(strides=(3,) * 15)), (-1, dict(strides=(64,) * 9 + (3,) * 6)), (-1, dict(kg=None)), (-2, dict(bits=2)),
    (-2, dict(gs=16)), (-1, dict(gs=128)), (-3, dict(ws=None)), (-3, dict(n=64)), (-3, dict(ws=ctypes.c_void_p(264))),
    (-2, dict(B=65535, Hq=1 << 20, Hkv=4)), (-2, dict(B=60000, Hq=60000, Hkv=60000, L=1 << 20)), (-1, dict(groups=-1))])
def test_c_attention_refusals(code, change):
    assert _pages_call(**change) == code, _lib.load().bi_last_error()
    assert b"bi_attn_pages" in _lib.load().bi_last_error()


def test_c_empty_batch():
    assert _pages_call(B=0) == 0


def test_c_write_and_read_refusals():
    lib = _lib.load()
    st, sec = (ctypes.c_int64 * 12)(*([64] * 12)), (ctypes.c_int64 * 4)(32, 0, 0, 0)

    def write(page=16, T=3, D=64, rows=9, tdt=0, sections=sec, axes=1, pools=(P, ctypes.c_void_p(512), ctypes.c_void_p(768), ctypes.c_void_p(1024)),
              B=2, bits=8, gs=64, strides=st, dtype=0, q=P):
        return lib.bi_rope_quantized_cache(q, 256, P, 128, P, 128, P, P, rows, tdt, P, sections, axes, P, P, *pools, 9, page, B, T, 4,
                                           2, D, bits, gs, strides, dtype, None)

    def read(page=16, L=64, pools=(P, P, P, P), B=2, bits=8, gs=64, strides=st, dtype=0, D=64, pages=9, table=P, stride=4, out=P, H=2):
        return lib.bi_read_quantized_cache(*pools, strides, table, stride, page, pages, None, out, P, B, H, L, D, bits, gs, 1, dtype,
                                           None)

    bad = (ctypes.c_int64 * 12)(*([8] * 12))
    odd = (ctypes.c_int64 * 12)(*([64, 64, 64, 3, 2, 2] * 2))
    for code, change in ((-1, dict(page=24)), (-1, dict(D=0)), (-1, dict(D=48)), (-1, dict(rows=0)), (-2, dict(tdt=2)), (-2, dict(axes=5)),
                         (-1, dict(sections=None)), (-1, dict(sections=(ctypes.c_int64 * 4)(12, 0, 0, 0))),
                         (-1, dict(sections=(ctypes.c_int64 * 4)(40, 0, 0, 0))), (-1, dict(pools=(P, P, P, P))), (-1, dict(pools=(None, P, P, P))),
                         (-2, dict(bits=5)), (-2, dict(gs=256)), (-1, dict(gs=128)), (-1, dict(strides=bad)), (-1, dict(strides=odd)),
                         (-1, dict(strides=None)), (-2, dict(dtype=7)), (-1, dict(q=None)), (-1, dict(q=ctypes.c_void_p(260))),
                         (-2, dict(B=1 << 20, T=1 << 12))):
        assert write(**change) == code, (change, lib.bi_last_error())
    assert write(B=0, pools=(None,) * 4) == 0 and write(T=0) == 0
    for code, change in ((-1, dict(page=3)), (-1, dict(B=-1)), (-1, dict(D=48)), (-1, dict(pools=(P, None, P, P))), (-2, dict(bits=16)),
                         (-2, dict(gs=8)), (-1, dict(strides=bad)), (-1, dict(strides=None)), (-2, dict(dtype=7)), (-1, dict(pages=0)),
                         (-1, dict(stride=3)), (-1, dict(table=None)), (-1, dict(out=None)), (-1, dict(out=ctypes.c_void_p(264))),
                         (-2, dict(B=65536)), (-2, dict(L=1 << 24, stride=1 << 20, B=60, H=512))):
        assert read(**change) == code, (change, lib.bi_last_error())
    assert read(B=0) == 0 and read(L=0) == 0


def test_workspaces():
    f = _lib.load().bi_attn_pages_workspace_bytes
    for bad in ((0, 4, 2, 1, 512, 64, 0), (1, 5, 2, 1, 512, 64, 0), (1, 4, 2, 0, 512, 64, 0), (1, 4, 2, 1, 0, 64, 0), (1, 4, 2, 1, 512, 64, -1)):
        assert f(*bad, 8, 1, 2) == 0
    # partials of every row and split, and the plan
    assert f(2, 4, 2, 1, 512, 64, 0, 8, 1, 2) >= 4 * (2 * 4 * 2) * (64 + 2)
    # many rows: the sequences read back, up to 2 GiB of them
    one = 2 * 2 * 65536 * 128 * 2
    assert f(3, 8, 2, 4096, 65536, 128, 0, 8, 1, 2) >= 3 * one
    assert 2 << 30 <= f(300, 8, 2, 4096, 65536, 128, 0, 8, 1, 2) < (2 << 30) + one
    assert f(3, 8, 2, 4096, 65536, 128, 0, 0, 1, 2) < one


def test_fake_shapes():
    ops, dt = torch.ops.mlx_bi, torch.bfloat16
    with FakeTensorMode():
        i = lambda *s: torch.empty(s, dtype=I32)
        q, kv = torch.empty(2, 3, 4, 64, dtype=dt), torch.empty(2, 3, 2, 64, dtype=dt)
        codes, groups, table = torch.empty(9, 2, 16, 32, dtype=torch.uint8), torch.empty(9, 2, 16, 2, 2, dtype=dt), torch.empty(50, 32)
        out = ops.rope_quantized_cache(q, kv, kv, table, table, i(2, 3), i(2, 3).long(), codes, groups, codes.clone(), groups.clone(),
                                       4, 32, None)
        assert out.shape == (2, 4, 3, 64) and out.dtype == dt
        assert ops.read_quantized_cache(codes, groups, codes, groups, i(2, 5), None, 4, 32).shape == (2, 2, 2, 80, 64)
        assert ops.quantized_paged_attention(out, codes, groups, codes, groups, i(2, 5), i(2), 4, 32, 0.125, True, None,
                                             None).shape == out.shape
        pool = torch.empty(9, 2, 16, 64, dtype=dt)
        assert ops.shared_prefix_attention(out, pool, pool, i(2, 5), i(2), 0.125, True, None, i(1)).shape == out.shape


def test_shared_pages_of_several_splits():
    """Many rows behind shared prefixes over plain pages of more than a split: one ratio of strides
    for K and V, page numbers that stay below 2^31."""
    lib = _lib.load()
    q = (1 << 20, 1 << 12, 64)

    def call(k, v, pages=9, page=512, n=BIG):
        return _pages_call(B=32, Hq=8, Hkv=2, Tq=200, L=4096, bits=0, groups=1, shared=512, page=page, pages=pages,
                           strides=(*q, *k, *v, *(0,) * 6), n=n)

    heads_out, rows_out = (2 * 512 * 64, 512 * 64, 64), (512 * 128, 64, 128)      # heads around rows, rows around heads
    assert call(heads_out, rows_out) == -2 and b"layout" in lib.bi_last_error()
    assert call((1 << 20, 64, 64), (1 << 20, 64, 64), pages=(1 << 31) - 1) == -2
    assert call((1 << 20, 64, 1 << 51), heads_out) == -2
    # (what is enough otherwise is a workspace, asked for last)
    for k, v in ((heads_out, heads_out), (rows_out, rows_out), ((2 * 512 * 64 + 8, 512 * 64, 64), (2 * 512 * 64 + 8, 512 * 64, 64)),
                 ((1 << 19, 1 << 18, 8), (1 << 21, 64, 32))):
        assert call(k, v, n=0) == -3, lib.bi_last_error()
    assert call(heads_out, rows_out, pages=1, n=0) == -3          # one page: its stride does not matter
    assert call(heads_out, rows_out, page=256, n=0) == -3         # pages of one split


def test_workspaces_of_shared_prefixes():
    lib = _lib.load()
    f, g = lib.bi_attn_pages_workspace_bytes, lib.bi_attn_pages_workspace_bytes_paged
    shape = (32, 8, 2, 200, 4096, 64)
    none = f(*shape, 0, 0, 1, 2)
    # a table of every sequence's pages (of at most 256 keys), or two words a sequence
    for page, cols in ((1, 4096), (16, 256), (256, 16), (512, 16), (1 << 20, 16)):
        assert g(*shape, 0, 0, 1, 2, page) == none
        assert g(*shape, 3, 0, 1, 2, page) == none + 4 * 32 * cols
        assert g(*shape, 3, 8, 1, 2, page) == f(*shape, 0, 8, 1, 2) + 8 * 32
    assert f(*shape, 3, 0, 1, 2) == g(*shape, 3, 0, 1, 2, 1) and g(*shape, 3, 0, 1, 2, 0) == 0
    assert g(32, 8, 2, 1, 4096, 64, 3, 0, 1, 2, 16) == f(32, 8, 2, 1, 4096, 64, 3, 0, 1, 2)


def test_workspaces_of_refused_shapes():
    """Shapes that the call refuses need nothing; none of their products wraps."""
    lib = _lib.load()
    for f, more in ((lib.bi_attn_pages_workspace_bytes, ()), (lib.bi_attn_pages_workspace_bytes_paged, (16,))):
        for bits in (0, 8):
            for dtype in (0, 1, 2):                       # 2^63 and 2^64 bytes read back
                assert f(1, 32768, 32768, 4096, 1 << 30, 65536, 0, bits, 1, dtype, *more) == 0
            for D in (16, 48, 160, 512, 65536):
                assert f(1, 4, 2, 200, 512, D, 1, bits, 1, 2, *more) == 0
            assert f(1, 4, 2, 200, 512, 64, 1, bits, 1, 7, *more) == 0                        # no such type
            assert f(65535, 1 << 26, 1 << 10, 1, (1 << 31) - 257, 256, 0, bits, 1, 2, *more) == 0   # 2^65 partials
            assert f(60000, 60000, 60000, 1, 1 << 20, 64, 0, bits, 1, 2, *more) == 0
    assert _pages_call(B=65535, Hq=1 << 26, Hkv=1 << 10, L=(1 << 31) - 4096, D=256, stride=1 << 28) == -2
    assert b"grid too large" in lib.bi_last_error()


@pytest.mark.parametrize("change,match", [
    (dict(codes=None), "tensors"), (dict(codes=[[0]]), "tensors"), (dict(groups=1.0), "tensors"), (dict(bits="8"), "bits"),
    (dict(bits=[8]), "bits"), (dict(bits=8.0), "bits"), (dict(group_size=64.0), "bits"), (dict(group_size=None), "bits")])
def test_pools_of_other_things(change, match):
    """Fields of the wrong kind are named, also after pools of the same layout have passed."""
    t, q = torch.zeros(2, 3, dtype=I32), torch.zeros(2, 4, 1, 64)
    good = [_pool() for _ in range(2)]
    for calls in range(2):
        bad = [p._replace(**change) for p in good]
        for kp, vp in (bad, (bad[0], good[1]), (good[0], bad[1])):
            with pytest.raises(ValueError, match=match + "|pools"):
                bi.rope_quantized_cache(**_write(k_pages=kp, v_pages=vp))
            with pytest.raises(ValueError, match=match + "|pools"):
                bi.read_quantized_cache(kp, vp, t)
            with pytest.raises(ValueError, match=match + "|pools"):
                bi.batch_invariant_quantized_paged_attention(q, kp, vp, t)
        with pytest.raises(ValueError, match="GPU"):      # (the layout is remembered now)
            bi.read_quantized_cache(*good, t)
