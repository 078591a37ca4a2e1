"""torch.ops.mlx_bi.* of the serving operators (CPU): schemas and fake-tensor
shape rules."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mlx_batch_invariant_amd  # noqa: F401  (registers the ops)

BF16, I32 = torch.bfloat16, torch.int32


def test_fake_shapes_and_dtypes():
    ops = torch.ops.mlx_bi
    with FakeTensorMode():
        x = torch.empty(2, 3, 64, dtype=BF16)
        w = torch.empty(64, dtype=BF16)
        y, h = ops.residual_rms_norm(x, x, w, w, 1e-6, None, 1.0)
        assert y.shape == h.shape == x.shape and y.dtype == h.dtype == BF16
        y, h = ops.residual_rms_norm(x, x, None, w, 1e-6, None, 1.0, False)
        assert y.shape == h.shape == x.shape
        y, h = ops.residual_rms_norm(x, x, w, None, 1e-6, None, 1.0, pre_norm=False)
        assert y.shape == x.shape and h.shape == (0,) and h.dtype == BF16
        i = lambda *s: torch.empty(s, dtype=I32)
        slots, pos, lens, cursor = ops.paged_slots(i(2), i(2), i(2, 5), i(9), None, 16, 3)
        assert slots.shape == pos.shape == (2, 3) and slots.dtype == torch.int64 and pos.dtype == I32
        assert lens.shape == (2,) and cursor.shape == (1,)
        q, kv = torch.empty(2, 3, 4, 64, dtype=BF16), torch.empty(2, 3, 2, 64, dtype=BF16)
        pool, table = torch.empty(9, 2, 16, 64, dtype=BF16), torch.empty(50, 32)
        out = ops.rope_paged_cache(q, kv, kv, table, table, pos, slots, pool, pool.clone(), None)
        assert out.shape == (2, 4, 3, 64) and out.dtype == BF16
        assert ops.scored_paged_attention(out, pool, pool, i(2, 5), lens, 0.125, True, 30.0, None, None,
                                          None).shape == out.shape


def test_residual_norm_arguments_default_to_both_norms():
    schema = str(torch.ops.mlx_bi.residual_rms_norm.default._schema)
    assert "bool post_norm=True, bool pre_norm=True" in schema
    x = torch.randn(3, 64)
    with pytest.raises(ValueError, match="neither"):
        torch.ops.mlx_bi.residual_rms_norm(x, x, None, None, 1e-6, None, 1.0, False, False)
