"""torch.ops.mlx_bi.* of the serving operators on the GPU: the Python functions'
bits, opcheck, and a compiled graph of the block before attention."""

import pytest
import torch

from helpers import bits, gen, randn

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _bi():
    import mlx_batch_invariant_amd as bi
    return bi


@pytest.mark.parametrize("post,pre", [(True, True), (False, True), (True, False)])
def test_residual_norm_with_either_norm_left_out(post, pre):
    """The add and norm of a plain block (no post norm), and a last block's add
    (no pre norm: h is empty)."""
    g = gen(61)
    x, res = randn((3, 5, 512), torch.bfloat16, g), randn((3, 5, 512), torch.bfloat16, g)
    w1, w2 = (randn((512,), torch.bfloat16, g) for _ in range(2))
    w1, w2 = w1 if post else None, w2 if pre else None
    y, h = _bi().batch_invariant_residual_rms_norm(x, res, w1, w2, 1e-5, scale=0.5, post_norm=post, pre_norm=pre)
    y2, h2 = torch.ops.mlx_bi.residual_rms_norm(x, res, w1, w2, 1e-5, None, 0.5, post, pre)
    assert bits(y) == bits(y2)
    assert bits(h) == bits(h2) if pre else h is None and h2.shape == (0,) and h2.dtype == x.dtype
    if not post:
        assert torch.equal(y, (res.float() + x.float() * 0.5).bfloat16())


def test_opcheck():
    g = gen(62)
    ops, tests = torch.ops.mlx_bi, ("test_schema", "test_faketensor")
    x, w = randn((4, 512), torch.bfloat16, g), randn((512,), torch.bfloat16, g)
    for post, pre in ((True, True), (False, True), (True, False)):
        torch.library.opcheck(ops.residual_rms_norm.default,
                              (x, x + 1, w if post else None, w if pre else None, 1e-5, None, 1.0, post, pre),
                              test_utils=tests)
    i = lambda *v: torch.tensor(v, dtype=I32, device="cuda")
    torch.library.opcheck(ops.paged_slots.default, (i(0, 5), i(3, 1), i(*range(8)).view(2, 4), i(8, 9), None, 4, 3),
                          test_utils=tests)
    q, k, v = randn((2, 3, 4, 64), x.dtype, g), randn((2, 3, 2, 64), x.dtype, g), randn((2, 3, 2, 64), x.dtype, g)
    kp, vp = randn((9, 2, 16, 64), x.dtype, g), randn((9, 2, 16, 64), x.dtype, g)
    cos, sin = randn((50, 32), torch.float32, g), randn((50, 32), torch.float32, g)
    pos, slots = i(0, 1, 2, 7, 8, 9).view(2, 3), torch.arange(6, device="cuda").view(2, 3) * 7
    torch.library.opcheck(ops.rope_paged_cache.default, (q, k, v, cos, sin, pos, slots, kp, vp, None), test_utils=tests)
    qh = q.transpose(1, 2).contiguous()
    table = i(*range(8)).view(2, 4)
    torch.library.opcheck(ops.scored_paged_attention.default,
                          (qh, kp, vp, table, i(50, 64), 0.125, True, 30.0, None, None, None), test_utils=tests)
    kc = randn((2, 2, 40, 64), x.dtype, g)
    docs = torch.zeros(2, 40, dtype=I32, device="cuda")
    torch.library.opcheck(ops.scored_attention.default,
                          (qh, kc, kc + 1, 0.125, True, None, None, torch.ones(4, device="cuda"), docs, i(3, 4)),
                          test_utils=tests)


def test_compiled_block_keeps_the_kernels():
    """Add and norm, positions and page writes in one compiled graph, in-place
    pools included: the eager calls' bits."""
    g = gen(63)
    dt = torch.bfloat16
    w = randn((256,), dt, g)
    cos, sin = randn((64, 32), torch.float32, g), randn((64, 32), torch.float32, g)
    table = torch.arange(8, dtype=I32, device="cuda").view(2, 4)
    pos = torch.tensor([[3, 4], [0, 1]], dtype=I32, device="cuda")
    slots = torch.tensor([[3, 4], [64, 65]], device="cuda")
    lens = torch.tensor([5, 2], dtype=I32, device="cuda")
    ops = torch.ops.mlx_bi

    def step(x, res, kp, vp):
        y, h = ops.residual_rms_norm(x, res, None, w, 1e-5, None, 1.0, False)
        h = h.view(2, 2, 4, 64)
        q = ops.rope_paged_cache(h, h[:, :, :2].contiguous(), h[:, :, 2:].contiguous(), cos, sin, pos, slots, kp, vp, None)
        return y, ops.scored_paged_attention(q, kp, vp, table, lens, 0.125, True, 20.0, None, None, None)

    x, res = randn((2, 2, 256), dt, g), randn((2, 2, 256), dt, g)
    pools = [randn((8, 2, 16, 64), dt, g) for _ in range(2)]
    a, b = [p.clone() for p in pools], [p.clone() for p in pools]
    want = step(x, res, *a)
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(x, res, *b)
    for u, v in zip((*want, *a), (*got, *b)):
        assert bits(u) == bits(v)
