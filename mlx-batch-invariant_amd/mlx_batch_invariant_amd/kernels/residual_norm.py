"""The norms around a block in one pass over the residual stream, on gfx950.

``y = residual + norm(x) * w_post * gate * scale`` and ``h = norm(y) * w_pre``:
what a block's output adds to the residual stream, and the next block's input.
Both sums run in ``rms_norm``'s order (D alone fixes it, and how many waves a row
has), everything else per element in fp32; y and h are rounded once each, h from the
unrounded y. The reference norms only (mlx_batch_invariant/kernels/rmsnorm.py:1-79).
"""

from __future__ import annotations

import torch

from .. import _lib


def _weight(what: str, name: str, w, x):
    """A weight vector as contiguous elements of x's type (None stays None)."""
    if w is None or w.dtype == x.dtype and w.ndim == 1 and w.is_contiguous() and w.shape[0] == x.shape[-1]:
        return w
    if w.numel() != x.shape[-1]:
        raise ValueError(f"{what}: {name} has {w.numel()} elements, expected {x.shape[-1]}")
    w = w.reshape(-1)
    return (w if w.dtype == x.dtype else w.to(x.dtype)).contiguous()


def _gate(what: str, gate, x):
    """(gate rows, elements between them, rows of x that share one). A vector
    and a gate of x's shape are read in place, and so is one that is constant
    over the last token dims ([B, 1, D] for x [B, T, D]); other broadcasts are
    laid out first."""
    if gate is None:
        return None, 0, 1
    D, rows = x.shape[-1], x.numel() // x.shape[-1]
    if gate.ndim == 0 or gate.ndim > x.ndim or gate.shape[-1] != D or any(
            a != b and a != 1 for a, b in zip(reversed(gate.shape), reversed(x.shape))):
        raise ValueError(f"{what}: gate {tuple(gate.shape)} does not broadcast over rows of {tuple(x.shape)}")
    if gate.dtype != x.dtype:
        gate = gate.to(x.dtype)
    if gate.numel() == D:
        return gate.reshape(D).contiguous(), 0, max(rows, 1)
    lead = (1,) * (x.ndim - gate.ndim) + tuple(gate.shape[:-1])
    full = x.ndim - 1                                # dims [0, full) as in x, ones behind
    while full > 0 and lead[full - 1] == 1:
        full -= 1
    if lead[:full] == tuple(x.shape[:full]):
        g2 = gate.reshape(-1, D)
        if g2.stride(-1) != 1 or g2.stride(0) < D:
            g2 = g2.contiguous()
        return g2, g2.stride(0), rows // g2.shape[0]
    return gate.expand(x.shape).contiguous().reshape(rows, D), D, 1


def _rows(t, rows: int, D: int):
    """t as rows of D contiguous elements, and the elements between rows."""
    if t.is_contiguous():
        return t, D
    t = t.reshape(rows, D)
    if t.stride(1) != 1 and D > 1 or t.stride(0) < D and rows > 1:
        t = t.contiguous()
    return t, max(t.stride(0), D)


def batch_invariant_residual_rms_norm(x: torch.Tensor, residual: torch.Tensor, post_weight: torch.Tensor | None,
                                      pre_weight: torch.Tensor | None, eps: float, *,
                                      gate: torch.Tensor | None = None, scale: float = 1.0, post_norm: bool = True,
                                      pre_norm: bool = True) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``(y, h)``: the residual stream behind a block, and the next block's input.

    ``x`` (the block's output) and ``residual`` ``[..., D]`` of one shape and
    type; ``post_norm`` norms x with ``post_weight``, ``pre_norm`` norms y with
    ``pre_weight`` (weights None: ones; without ``pre_norm`` h is None). ``gate``
    broadcasts over x with its own last dim D (``[D]``, ``[B, 1, D]``, x's shape);
    weights and gate are converted to x's type. ``h`` is taken from y before its
    rounding, so it is not the bits of ``batch_invariant_rms_norm(y, ...)``."""
    what = "batch_invariant_residual_rms_norm"
    dt, shape = x.dtype, x.shape
    if dt not in _lib.FLOAT_DTYPES or residual.dtype != dt:
        raise ValueError(f"{what}: unsupported dtypes {x.dtype} and {residual.dtype}")
    if not shape or residual.shape != shape:
        raise ValueError(f"{what}: shapes {tuple(x.shape)} and {tuple(residual.shape)}")
    if not post_norm and not pre_norm:
        raise ValueError(f"{what}: neither post_norm nor pre_norm")
    if not post_norm and post_weight is not None or not pre_norm and pre_weight is not None:
        raise ValueError(f"{what}: a weight for a norm that is not asked for")
    dev = _lib.one_device(what, x, residual, post_weight, pre_weight, gate)
    D = shape[-1]
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    h = torch.empty_like(y) if pre_norm else None
    w1, w2 = _weight(what, "post_weight", post_weight, x), _weight(what, "pre_weight", pre_weight, x)
    n = x.numel()
    if n == 0:
        return y, h
    rows = n // D
    g, g_stride, g_group = _gate(what, gate, x)
    x2, x_stride = _rows(x, rows, D)
    r2, r_stride = _rows(residual, rows, D)
    rc = _lib.launch(dev, _lib.residual_norm_call, x2.data_ptr(), x_stride, r2.data_ptr(), r_stride, _lib.ptr(g),
                     g_stride, g_group, _lib.ptr(w1), _lib.ptr(w2), y.data_ptr(), _lib.ptr(h), rows, D, float(eps),
                     float(scale), bool(post_norm), bool(pre_norm), _lib.DTYPE_CODE[dt], _lib.stream_of(x))
    if rc:
        _lib.check(rc, "bi_residual_rms_norm")
    return y, h
