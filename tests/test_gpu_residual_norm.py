"""The norms around a block against the 64-bit formula, and their invariance."""

import pytest
import torch

import paged_ref as ref
from helpers import DT, bits, gen, randn

pytestmark = pytest.mark.gpu
EPS = 1e-5


def _f(*a, **k):
    import mlx_batch_invariant_amd as bi
    return bi.batch_invariant_residual_rms_norm(*a, **k)


def _check(dt, x, res, w1, w2, gate, scale, post, pre):
    """Half a step of each result, and fp32's share: a sum of D squares in D / 256
    + 9 additions is off by at most that many 2^-24 of itself, its root by half
    of that, and each of the up to 8 operations behind it by one 2^-24."""
    y, h = _f(x, res, w1, w2, EPS, gate=gate, scale=scale, post_norm=post, pre_norm=pre)
    c = lambda t: None if t is None else t.cpu()
    wy, wh = ref.residual_norm(c(x), c(res), c(w1), c(w2), EPS, c(gate), scale, post, pre)
    D = x.shape[-1]
    e = ((D / 256 + 9) / 2 + 8) * 2.0 ** -24
    add = (wy - res.cpu().double()).abs()
    dy = e * add + 2.0 ** -24 * wy.abs()                       # y before its rounding
    fi = torch.finfo(DT[dt])
    step = lambda w: fi.eps / 2 * w.abs() * (1 + 2.0 ** -20) + fi.smallest_normal * fi.eps
    assert ((y.double().cpu() - wy).abs() <= dy + step(wy)).all()
    assert (h is None) == (not pre)
    if pre:
        rel = dy.norm(dim=-1, keepdim=True) / wy.norm(dim=-1, keepdim=True).clamp(min=1e-30)
        dh = wh.abs() * (e + rel) + dy * (wh / wy).abs().nan_to_num(0.0)
        assert ((h.double().cpu() - wh).abs() <= dh + step(wh)).all()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [1, 7, 64, 129, 896, 2048, 4096, 4097, 8192, 9000])
def test_residual_norm(dt, D):
    g = gen(D)
    for n, (rows, gate, scale, post, pre) in enumerate((
            (1, None, 1.0, True, True), (5, "channel", 0.5, True, True), (3, "row", -2.0, True, False),
            (6, "group", 1.0, False, True))):
        x, res = randn((rows, D), DT[dt], g, 1.5), randn((rows, D), DT[dt], g, 4.0)
        w1, w2 = (1 + randn((D,), torch.float32, g, 0.1)).to(DT[dt]), (1 + randn((D,), torch.float32, g, 0.1)).to(DT[dt])
        gt = {None: None, "channel": (D,), "row": (rows, D), "group": (2, 1, D)}[gate]
        gt = None if gt is None else randn(gt, DT[dt], g)
        if gate == "group":
            x, res = x.reshape(2, 3, D), res.reshape(2, 3, D)
        _check(dt, x, res, w1 if post and n != 1 else None, w2 if pre and n != 3 else None, gt, scale, post, pre)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_residual_norm_layouts_and_invariance(dt):
    """Rows of a wider tensor, misaligned ones, weights of another type; a row's
    bits alone and in a batch."""
    g = gen(3)
    D = 896
    x, res, gate = (randn((37, D), DT[dt], g) for _ in range(3))
    w1, w2 = (randn((D,), DT[dt], g) for _ in range(2))
    y, h = _f(x, res, w1, w2, EPS, gate=gate)
    wide = torch.cat([x, res, gate], 1)
    for a in (wide.split(D, 1), torch.cat([x[:, :1], x, res, gate], 1)[:, 1:].split(D, 1),
              [t.t().contiguous().t() for t in (x, res, gate)]):
        y2, h2 = _f(a[0], a[1], w1, w2.double(), EPS, gate=a[2])
        assert bits(y2) == bits(y) and bits(h2) == bits(h)
    for r in (0, 17, 36):
        y1, h1 = _f(x[r], res[r], w1, w2, EPS, gate=gate[r])
        assert bits(y1) == bits(y[r]) and bits(h1) == bits(h[r])
        y1, h1 = _f(x[r:r + 1], res[r:r + 1], w1, w2, EPS, gate=gate[r:r + 1])
        assert bits(y1) == bits(y[r:r + 1]) and bits(h1) == bits(h[r:r + 1])
    one = gate.reshape(1, 37, D).expand(2, 37, D)       # a gate that broadcasts over the leading dim
    y2, h2 = _f(torch.stack([x, x]), torch.stack([res, res]), w1, w2, EPS, gate=gate.reshape(1, 37, D))
    assert bits(y2[1]) == bits(y) and bits(h2[0]) == bits(h) and one.shape == y2.shape


def test_residual_norm_edges():
    """No rows, no elements, rows of zeros, a NaN that stays in its row."""
    for shape in ((0, 64), (3, 0), (2, 0, 5)):
        x = torch.zeros(shape, device="cuda")
        y, h = _f(x, x, None, None, EPS)
        assert y.shape == h.shape == shape
    x = torch.zeros(3, 256, device="cuda")
    y, h = _f(x, x, None, None, EPS)
    assert not y.any() and not h.any()
    res = torch.ones_like(x)
    res[1, 7] = float("nan")
    y, h = _f(x, res, None, None, EPS)
    assert y[[0, 2]].eq(1).all() and h[[0, 2]].isfinite().all() and h[1].isnan().all()
    assert y[1].isnan().sum() == 1


def test_residual_norm_in_a_graph_and_by_the_dispatcher():
    g = gen(4)
    x, res = randn((4, 512), torch.bfloat16, g), randn((4, 512), torch.bfloat16, g)
    w, gate = randn((512,), torch.bfloat16, g), randn((4, 512), torch.bfloat16, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _f(x, res, w, w, EPS, gate=gate)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = _f(x, res, w, w, EPS, gate=gate)
    for i in range(3):
        x.copy_(randn(x.shape, x.dtype, gen(50 + i)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        a, b = _f(x, res, w, w, EPS, gate=gate)
        assert bits(y) == bits(a) and bits(h) == bits(b)
        a, b = torch.ops.mlx_bi.residual_rms_norm(x, res, w, w, EPS, gate, 1.0)
        assert bits(y) == bits(a) and bits(h) == bits(b)
    del graph
