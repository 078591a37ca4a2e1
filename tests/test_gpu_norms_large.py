"""Norms of more rows than one launch holds threads for (256 a row, 2^32 in all):
every row gets what it gets alone."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _rows(n, D, seed):
    """[n, D] whose row r is drawn by r alone (a repeated block, turned and scaled)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    base = torch.randn((4093, D), generator=g, device="cuda").to(torch.bfloat16)
    return base.repeat(-(-n // 4093), 1)[:n].contiguous()


def _same_as_alone(got, f, n, *xs):
    """``got[r]`` against f of some rows alone: the first, those around 2^24, the last."""
    for a, b in ((0, 100), (n // 3, n // 3 + 50), (2**24 - 60, 2**24 + 40), (n - 70, n)):
        if b <= n:
            assert torch.equal(got[a:b], f(*(x[a:b].contiguous() for x in xs))), (a, b)
    # every row: equal inputs, equal outputs
    assert torch.equal(got[4093:2 * 4093], got[:4093])
    step = 4093 * 64
    first = got[:step]
    for a in range(0, n - step, step):
        assert torch.equal(got[a:a + step], first), a


def test_residual_norm():
    """(Four rows a workgroup.)"""
    import mlx_batch_invariant_amd as bi
    D, n = 8, 2**26 + 300
    x = _rows(n, D, 1)
    w = torch.linspace(0.5, 2.0, D, device="cuda").to(torch.bfloat16)
    f = lambda a: torch.cat(bi.batch_invariant_residual_rms_norm(a, a, w, w, 1e-5, gate=w), 1)
    y, h = bi.batch_invariant_residual_rms_norm(x, x, w, w, 1e-5, gate=w)
    _same_as_alone(y, lambda a: f(a)[:, :D], n, x)
    _same_as_alone(h, lambda a: f(a)[:, D:], n, x)


def test_rms_norm():
    import mlx_batch_invariant_amd as bi
    D, n = 8, 2**24 + 300
    x = _rows(n, D, 2)
    w = torch.linspace(0.5, 2.0, D, device="cuda").to(torch.bfloat16)
    f = lambda a: bi.batch_invariant_rms_norm(a, w, 1e-5)
    _same_as_alone(f(x), f, n, x)


def test_layer_norm():
    import mlx_batch_invariant_amd as bi
    D, n = 8, 2**24 + 300
    x = _rows(n, D, 3)
    w = torch.linspace(0.5, 2.0, D, device="cuda").to(torch.bfloat16)
    f = lambda a: bi.batch_invariant_layer_norm(a, w, w, 1e-5)
    _same_as_alone(f(x), f, n, x)
