"""What the paged-cache calls and the residual norms refuse, on the host (nothing
is launched), and the library operators' schemas and fake shapes."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mlx_batch_invariant_amd as bi
from mlx_batch_invariant_amd import _lib

I32 = torch.int32


def test_slots_arguments():
    t, l, f = torch.zeros(2, 4, dtype=I32), torch.zeros(2, dtype=I32), torch.zeros(5, dtype=I32)
    good = dict(page_size=16, max_new=3)
    with pytest.raises(ValueError, match="GPU"):
        bi.paged_slots(l, l, t, f, **good)
    for page in (0, -16, 24, 16.0, True):
        with pytest.raises(ValueError, match="page size"):
            bi.paged_slots(l, l, t, f, page_size=page, max_new=3)
    for T in (0, -1, 2.0, True):
        with pytest.raises(ValueError, match="max_new"):
            bi.paged_slots(l, l, t, f, page_size=16, max_new=T)
    for bad in (t.long(), t[0], t.float()):
        with pytest.raises(ValueError, match="block table"):
            bi.paged_slots(l, l, bad, f, **good)
    with pytest.raises(ValueError, match="columns"):
        bi.paged_slots(l, l, t[:, :0], f, **good)
    for bad in (t.t().contiguous().t(), t[:1].expand(2, 4)):
        with pytest.raises(ValueError, match="strides"):
            bi.paged_slots(l, l, bad, f, **good)


def _rope_operands(B=2, T=3, Hq=4, Hkv=2, D=32, P=5, page=8):
    q, k, v = (torch.zeros(B, T, h, D) for h in (Hq, Hkv, Hkv))
    cs = torch.zeros(9, D // 2)
    pos = torch.zeros(B, T, dtype=I32)
    kp, vp = torch.zeros(P, Hkv, page, D), torch.zeros(P, Hkv, page, D)
    return dict(q=q, k=k, v=v, cos=cs, sin=cs.clone(), positions=pos, slots=pos.long(), k_pages=kp, v_pages=vp)


@pytest.mark.parametrize("change,match", [
    (dict(k=torch.zeros(2, 3, 2, 16)), "shapes"), (dict(v=torch.zeros(2, 3, 1, 32)), "shapes"),
    (dict(q=torch.zeros(2, 4, 4, 32)), "shapes"), (dict(k_pages=torch.zeros(5, 3, 8, 32)), "pools"),
    (dict(v_pages=torch.zeros(4, 2, 8, 32)), "pools"), (dict(q=torch.zeros(2, 3, 4, 32).half()), "type"),
    (dict(k_pages=torch.zeros(5, 2, 8, 32).half()), "type"), (dict(cos=torch.zeros(9, 16).half()), "tables"),
    (dict(cos=torch.zeros(8, 16)), "tables"), (dict(cos=torch.zeros(9, 8), sin=torch.zeros(9, 8), sections=(16,)), "sections"),
    (dict(slots=torch.zeros(2, 3)), "slots"), (dict(slots=torch.zeros(6, dtype=torch.int64)), "slots"),
    (dict(sections=(8, 9)), "sections"), (dict(sections=(-8, 24)), "sections"), (dict(sections=()), "sections"),
    (dict(sections=(4, 4, 4, 2, 2)), "sections"), (dict(cos=torch.zeros(9, 12), sin=torch.zeros(9, 12)), "multiple of 8"),
    (dict(cos=torch.zeros(9, 24), sin=torch.zeros(9, 24)), "multiple of 8"),
    (dict(cos=torch.zeros(0, 16), sin=torch.zeros(0, 16)), "multiple of 8"),
    (dict(k_pages=torch.zeros(5, 2, 6, 32), v_pages=torch.zeros(5, 2, 6, 32)), "page size"), ({}, "GPU")])
def test_rope_arguments(change, match):
    with pytest.raises(ValueError, match=match):
        bi.rope_paged_cache(**(_rope_operands() | change))


def test_written_tensors():
    """What an in-place operation of torch refuses is refused."""
    t = torch.zeros(3, 4)
    _lib.in_place("x", t, t.t(), t[:, 1:], t[:1].expand(1, 4))
    with pytest.raises(ValueError, match="share memory"):
        _lib.in_place("x", t[:1].expand(3, 4))
    with torch.inference_mode():
        i = torch.zeros(3)
        _lib.in_place("x", i)
    with pytest.raises(ValueError, match="inference"):
        _lib.in_place("x", i)
    leaf = torch.zeros(3, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        _lib.in_place("x", leaf)
    with torch.no_grad():
        _lib.in_place("x", leaf)


def test_residual_norm_arguments():
    x = torch.zeros(2, 3, 16)
    w = torch.zeros(16)
    f = bi.batch_invariant_residual_rms_norm
    with pytest.raises(ValueError, match="GPU"):
        f(x, x, w, w, 1e-6)
    for a, b in ((x, x.half()), (x.double(), x.double()), (x.long(), x.long())):
        with pytest.raises(ValueError, match="dtypes"):
            f(a, b, w, w, 1e-6)
    with pytest.raises(ValueError, match="shapes"):
        f(x, x[0], w, w, 1e-6)
    with pytest.raises(ValueError, match="neither"):
        f(x, x, None, None, 1e-6, post_norm=False, pre_norm=False)
    for kw in (dict(post_norm=False), dict(pre_norm=False)):
        with pytest.raises(ValueError, match="not asked"):
            f(x, x, w, w, 1e-6, **kw)


@pytest.mark.parametrize("shape,want", [((16,), (0, 6)), ((2, 3, 16), (16, 1)), ((2, 1, 16), (16, 3)),
                                        ((1, 1, 16), (0, 6)), ((3, 16), (16, 1)), ((1, 3, 16), (16, 1))])
def test_gate_rows(shape, want):
    """Rows of x that share a gate row, and the values each row reads."""
    from mlx_batch_invariant_amd.kernels.residual_norm import _gate
    x, g = torch.zeros(2, 3, 16), torch.randn(shape)
    rows, stride, group = _gate("x", g, x)
    assert (stride, group) == want
    read = torch.stack([rows.flatten()[r // group * stride:][:16] for r in range(6)])
    assert torch.equal(read, g.expand(2, 3, 16).reshape(6, 16))
    for bad in ((15,), (1,), (4, 16), (3, 3, 16), (1, 2, 3, 16), ()):
        with pytest.raises(ValueError, match="broadcast"):
            _gate("x", torch.zeros(bad), x)


def _err(lib):
    return lib.bi_last_error().decode()


def test_abi_rejections():
    lib = _lib.load()
    p, o = ctypes.c_void_p(16), ctypes.c_void_p(32)      # never dereferenced: validation fails first
    slots = lambda **k: lib.bi_paged_slots(*(k.get(n, d) for n, d in (
        ("lens", p), ("news", p), ("table", p), ("stride", 4), ("max_pages", 4), ("free", p), ("nfree", 9),
        ("cursor", None), ("slots", p), ("pos", p), ("out", o), ("out_cursor", o), ("B", 2), ("T", 3), ("page", 16),
        ("stream", None))))
    for bad in (dict(page=24), dict(page=0), dict(page=1 << 25), dict(B=-1), dict(T=0), dict(max_pages=0),
                dict(stride=3), dict(nfree=-1), dict(lens=None), dict(slots=None), dict(free=None), dict(out=p),
                dict(out_cursor=None), dict(cursor=o)):
        assert slots(**bad) == -1, bad
    for bad in (dict(B=(1 << 20) + 1), dict(T=(1 << 24) + 1), dict(max_pages=1 << 27, stride=1 << 27)):
        assert slots(**bad) == -2, bad
    st = (ctypes.c_int64 * 6)(*([128] * 6))
    sec = lambda *s: (ctypes.c_int64 * 4)(*s, *([0] * (4 - len(s))))
    rope = lambda **k: lib.bi_rope_paged_cache(*(k.get(n, d) for n, d in (
        ("q", p), ("qr", 512), ("k", p), ("kr", 256), ("v", p), ("vr", 256), ("cos", p), ("sin", p), ("rows", 9),
        ("tdt", 0), ("pos", p), ("sec", sec(32)), ("axes", 1), ("slots", p), ("qo", p), ("kp", p), ("vp", p),
        ("pages", 5), ("page", 16), ("B", 2), ("T", 3), ("Hq", 4), ("Hkv", 2), ("D", 128), ("st", st), ("dt", 2),
        ("stream", None))))
    for bad in (dict(page=12), dict(D=120), dict(rows=0), dict(pages=0), dict(sec=sec(12)), dict(sec=sec(72)),
                dict(sec=sec(0)), dict(sec=sec(-8, 16), axes=2), dict(q=None), dict(kp=ctypes.c_void_p(24)),
                dict(qr=504), dict(kr=255), dict(st=(ctypes.c_int64 * 6)(*([100] * 6))), dict(B=-1)):
        assert rope(**bad) == -1, bad
    for bad in (dict(axes=5), dict(axes=0), dict(tdt=1), dict(dt=3), dict(B=1 << 20, T=1 << 12)):
        assert rope(**bad) == -2, bad
    assert rope(T=0) == 0
    norm = lambda **k: lib.bi_residual_rms_norm(*(k.get(n, d) for n, d in (
        ("x", p), ("xs", 16), ("res", p), ("rs", 16), ("gate", None), ("gs", 0), ("gg", 1), ("w1", p), ("w2", p),
        ("y", p), ("h", p), ("rows", 2), ("D", 16), ("eps", 1e-6), ("scale", 1.0), ("post", 1), ("pre", 1), ("dt", 2),
        ("stream", None))))
    for bad in (dict(rows=-1), dict(D=0), dict(post=0, pre=0), dict(x=None), dict(h=None), dict(xs=8), dict(rs=8),
                dict(gate=p, gg=0), dict(gate=p, gs=-1)):
        assert norm(**bad) == -1, bad
    assert norm(dt=5) == -2 and norm(rows=1 << 31) == -2 and norm(rows=0) == 0


def test_operators_are_registered():
    for name in ("residual_rms_norm", "paged_slots", "rope_paged_cache"):
        assert str(getattr(torch.ops.mlx_bi, name).default._schema).startswith(f"mlx_bi::{name}(")
    with FakeTensorMode():
        x = torch.empty(5, 7, 64, dtype=torch.bfloat16)
        y, h = torch.ops.mlx_bi.residual_rms_norm(x, x, None, None, 1e-6, None, 1.0)
        assert y.shape == h.shape == x.shape
        i = torch.empty(5, dtype=I32)
        s, pos, lens, cur = torch.ops.mlx_bi.paged_slots(i, i, torch.empty(5, 9, dtype=I32), i, None, 16, 3)
        assert s.shape == pos.shape == (5, 3) and s.dtype == torch.int64 and lens.shape == (5,) and cur.shape == (1,)
        o = _rope_operands()
        assert torch.ops.mlx_bi.rope_paged_cache(*o.values(), None).shape == (2, 4, 3, 32)


def test_bindings_agree():
    """The CPython binding and ctypes hand the same arguments over: each refuses
    what the other does, with the same text."""
    from mlx_batch_invariant_amd import _bi_pycall as fast
    lib = _lib.load()
    assert _lib.slots_call is fast.paged_slots and _lib.rope_paged_call is fast.rope_paged_cache
    assert _lib.scored_call is fast.attn_scored and _lib.residual_norm_call is fast.residual_rms_norm

    slots = [16, 16, 16, 4, 4, 16, 9, None, 16, 16, 32, 32, 2, 3, 24, None]
    rope = [16, 512, 16, 256, 16, 256, 16, 16, 9, 0, 16, 2, 16, 24, 7, 7, 16, 16, 16, 16, 5, 16, 2, 3, 4, 2, 128,
            *(128, 256, 384, 512, 640, 100), 2, None]
    scored = [256] * 3 + [None, 0, 0, 0, None, 256, 1, 4, 2, 4, 300, 128, *(128 * i for i in range(1, 10)), 1, 0.5, 2.0,
              None, 256, 299, None, 2, None, 0, None]
    norm = [16, 16, 16, 15, None, 0, 1, 16, 16, 16, 16, 2, 16, 1e-6, 2.0, 1, 1, 2, None]
    for calls in (((fast.paged_slots, lib.bi_paged_slots), slots), ((fast.residual_rms_norm, lib.bi_residual_rms_norm), norm),
                  ((fast.rope_paged_cache, lambda *a: lib.bi_rope_paged_cache(
                      *a[:11], (ctypes.c_int64 * 4)(*a[12:16]), a[11], *a[16:27], (ctypes.c_int64 * 6)(*a[27:33]),
                      *a[33:])), rope),
                  ((fast.attn_scored, lambda *a: lib.bi_attn_scored(
                      *a[:15], (ctypes.c_int64 * 9)(*a[15:24]), a[24], a[25], _lib.ScoreMod(*a[26:31]), *a[31:])),
                   scored)):
        (f, g), args = calls
        got = f(*args)
        text = _err(lib)
        assert got == g(*args) < 0 and _err(lib) == text and text
        with pytest.raises(TypeError, match="arguments"):
            f(*args, 0)
        with pytest.raises(TypeError):
            f("x", *args[1:])
