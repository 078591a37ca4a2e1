"""Pages, slots and the rotary embedding with the write into a paged cache,
against plain forms (whole numbers exactly; rotated values in 64 bits)."""

import numpy as np
import pytest
import torch

import paged_ref as ref
from helpers import DT, bits, gen, randn

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _bi():
    import mlx_batch_invariant_amd as bi
    return bi


def _requests(B, T, cols, page, seed, spare=4, short=False):
    """Random counts within the table, its held pages, and the free ones."""
    r = np.random.default_rng(seed)
    news = r.integers(0, T + 1, B)
    lens = [int(r.integers(0, max(1, cols * page - n + 1))) for n in news]
    pool = r.permutation(B * cols + spare)
    table = pool[:B * cols].reshape(B, cols).copy()
    for b in range(B):
        table[b, -(-lens[b] // page):] = 0
    used = {int(p) for b in range(B) for p in table[b, :-(-lens[b] // page)]}
    free = [int(p) for p in pool if int(p) not in used]
    if short:
        free = free[:len(free) // 3]
    return lens, [int(n) for n in news], table.tolist(), free


def _run(lens, news, table, free, page, T, cursor=None):
    dev = lambda x: torch.tensor(x, dtype=I32, device="cuda")
    t = dev(table) if table else torch.zeros(0, 3, dtype=I32, device="cuda")
    p = _bi().paged_slots(dev(lens), dev(news), t, dev(free), page_size=page, max_new=T,
                          cursor=None if cursor is None else dev([cursor]))
    return p.slots.tolist(), p.positions.tolist(), p.kv_lens.tolist(), p.cursor.item(), t.tolist()


def _check(lens, news, table, free, page, T, cursor=None):
    want = ref.slots(lens, news, table, free, page, T, cursor or 0)
    got = _run(lens, news, table, free, page, T, cursor)
    for g, w, what in zip(got, want, ("slots", "positions", "lengths", "cursor", "table")):
        assert g == w, what


@pytest.mark.parametrize("B,T,cols,page", [(1, 1, 1, 1), (3, 5, 7, 4), (64, 1, 32, 16), (257, 1, 5, 2), (700, 3, 9, 8),
                                           (1500, 1, 3, 16), (2, 4100, 40, 256), (5, 2049, 70, 64), (33, 40, 4, 1024)])
@pytest.mark.parametrize("short", [False, True])
def test_slots(B, T, cols, page, short):
    _check(*_requests(B, T, cols, page, B + T, short=short), page, T)


@pytest.mark.parametrize("cursor", [-3, 0, 2, 5, 6, 99])
def test_slots_cursor_and_refusals(cursor):
    """Pages from the cursor on; requests that do not fit the table, the free
    list or the rows; counts out of range; free lists and tables with holes."""
    lens = [0, 16, 15, -4, 1 << 30, 30, 33, 0, 47, 7]
    news = [5, 1, 1, 2, 1, 0, 16, 9, 2, -7]
    table = [[100 + 3 * b + j for j in range(3)] for b in range(10)]
    table[6][2] = -1
    for free in ([11, 12, 13, 14, 15, 16], [11, -5], []):
        _check(lens, news, table, free, 16, 8, cursor)


def test_slots_empty_batch_and_list_arguments():
    _check([], [], [], [4, 5], 16, 3, 1)
    bi = _bi()
    t = torch.zeros(2, 3, dtype=I32, device="cuda")
    p = bi.paged_slots([0, 3], torch.tensor([2, 1]), t, [7, 8, 9], page_size=4, max_new=2)
    assert p.slots.tolist() == [[28, 29], [-1, 3]] and p.cursor.item() == 1 and t.tolist()[0] == [7, 0, 0]


def test_slots_of_a_table_slice_and_outputs_of_their_own():
    """A table with longer rows: columns behind the slice, and the inputs, stay."""
    bi = _bi()
    wide = torch.full((4, 9), -7, dtype=I32, device="cuda")
    lens, news = torch.tensor([0, 1, 2, 8], dtype=I32, device="cuda"), torch.full((4,), 3, dtype=I32, device="cuda")
    free, cur = torch.arange(50, 60, dtype=I32, device="cuda"), torch.tensor([1], dtype=I32, device="cuda")
    before = wide._version
    p = bi.paged_slots(lens, news, wide[:, 2:5], free, page_size=4, max_new=3, cursor=cur)
    assert wide._version > before
    assert wide[:, :2].eq(-7).all() and wide[:, 5:].eq(-7).all()
    assert wide[:, 2:5].tolist() == [[51, -7, -7], [-7] * 3, [-7, 52, -7], [-7, -7, 53]]
    assert lens.tolist() == [0, 1, 2, 8] and cur.item() == 1 and p.cursor.item() == 4
    again = bi.paged_slots(lens, news, wide[:, 2:5], free, page_size=4, max_new=3, cursor=cur)
    for a, b in zip(p, again):
        assert torch.equal(a, b)


def _rope_case(dt, tab, B, T, heads, D, sections, page, seed, token_major=False, rows=40):
    Hq, Hkv = heads
    g = gen(seed)
    q, k, v = (randn((B, T, h, D), DT[dt], g, 3.0) for h in (Hq, Hkv, Hkv))
    ang = torch.rand((rows, sum(sections)), generator=g, dtype=torch.float64) * 6.3
    cos, sin = (f(ang).to(DT[tab]).cuda() for f in (torch.cos, torch.sin))
    pos = torch.randint(-3, rows + 3, (len(sections), B, T), generator=g, dtype=I32).cuda()
    pages = -(-B * T // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:B * T].reshape(B, T)
    slots[torch.rand((B, T), generator=g) < 0.2] = -1
    shape = (pages, page, Hkv, D) if token_major else (pages, Hkv, page, D)
    pools = [randn(shape, DT[dt], g) for _ in range(2)]
    view = [p.permute(0, 2, 1, 3) if token_major else p for p in pools]
    return q, k, v, cos, sin, pos, slots.cuda(), view


def _rope_check(got, pools, before, q, k, v, cos, sin, pos, slots, sections, dt):
    """|error| <= half a step of the result + 3 fp32 roundings of the products."""
    def near(x, want, size):
        err = (x.double().cpu() - want).abs()
        allow = torch.finfo(DT[dt]).eps / 2 * want.abs() * (1 + 2e-7) + 3 * 2.0 ** -24 * size
        allow += torch.finfo(DT[dt]).smallest_normal * torch.finfo(DT[dt]).eps      # subnormal results
        assert (err <= allow).all(), float((err / allow).max())

    c = [t.cpu() for t in (cos, sin, pos)]
    turn = lambda x: ref.rope(x.cpu(), *c, sections)
    size = lambda x: ref.rope(x.cpu().abs(), c[0].abs(), -c[1].abs(), c[2], sections).abs() + x.cpu().double().abs()
    near(got.transpose(1, 2), turn(q), size(q))
    page = pools[0].shape[2]
    keep = ((slots >= 0) & (slots < pools[0].shape[0] * page)).cpu()
    at = slots.cpu()[keep]
    kp, vp = pools[0].cpu(), pools[1].cpu()
    near(kp[at // page, :, at % page], turn(k)[keep], size(k)[keep])
    assert bits(vp[at // page, :, at % page]) == bits(v.cpu()[keep])
    for p, b in zip((kp, vp), before):                  # every other row as it was
        rest = torch.ones(p.shape[0], page, dtype=torch.bool)
        rest[at // page, at % page] = False
        assert bits(p.transpose(1, 2)[rest]) == bits(b.transpose(1, 2)[rest])


@pytest.mark.parametrize("dt,tab", [("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("B,T,heads,D,sections,page", [
    (1, 1, (32, 8), 128, (64,), 16), (3, 5, (14, 2), 64, (6, 10), 8), (2, 37, (3, 1), 16, (8,), 1),
    (5, 1, (8, 8), 96, (16, 24, 8), 64), (2, 9, (5, 5), 256, (1, 0, 127, 0), 4), (1, 130, (4, 1), 32, (3, 2, 3), 256)])
def test_rope(dt, tab, B, T, heads, D, sections, page):
    for token_major in (False, True):
        q, k, v, cos, sin, pos, slots, pools = _rope_case(dt, tab, B, T, heads, D, sections, page, B + T + D, token_major)
        slots[0, 0] = pools[0].shape[0] * page          # behind the pool: nothing is written
        before = [p.cpu().clone() for p in pools]
        got = _bi().rope_paged_cache(q, k, v, cos, sin, pos, slots, *pools, sections=sections)
        _rope_check(got, pools, before, q, k, v, cos, sin, pos, slots, sections, dt)


def test_rope_of_a_joint_projection_and_odd_layouts():
    """Slices of one projection are read in place; other layouts give the same bits."""
    bi = _bi()
    q, k, v, cos, sin, pos, slots, pools = _rope_case("bf16", "f32", 3, 4, (6, 2), 64, (32,), 16, 5)
    run = lambda q, k, v, cos=cos: [(o := [p.clone() for p in pools]),
                                    bi.rope_paged_cache(q, k, v, cos, sin, pos[0], slots, *o)]
    joint = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1)
    a, b, c = joint.split([384, 128, 128], -1)
    sliced = [t.view(3, 4, -1, 64) for t in (a, b, c)]
    from mlx_batch_invariant_amd.kernels.paged_cache import _rows
    assert all(_rows(t) is t for t in sliced)
    odd = [torch.empty(*t.shape[:3], 65, dtype=t.dtype, device="cuda")[..., :64].copy_(t) for t in (q, k, v)]
    heads = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    want = run(q, k, v)
    for other in (run(*sliced), run(*odd), run(*heads), run(q, k, v, torch.cat([cos, cos], 1)[:, :32])):
        assert bits(other[1]) == bits(want[1])
        for x, y in zip(other[0], want[0]):
            assert bits(x) == bits(y)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_rope_batch_invariant(dt):
    """A token's bits alone and within a batch."""
    bi = _bi()
    q, k, v, cos, sin, pos, slots, pools = _rope_case(dt, "f32", 7, 9, (14, 2), 64, (12, 20), 16, 6)
    all_pools = [p.clone() for p in pools]
    out = bi.rope_paged_cache(q, k, v, cos, sin, pos, slots, *all_pools, sections=(12, 20))
    for b, t in ((0, 0), (6, 8), (3, 4)):
        one = [x[b:b + 1, t:t + 1] for x in (q, k, v)]
        mine = [p.clone() for p in pools]
        got = bi.rope_paged_cache(*one, cos, sin, pos[:, b:b + 1, t:t + 1], slots[b:b + 1, t:t + 1], *mine,
                                  sections=(12, 20))
        assert bits(got) == bits(out[b:b + 1, :, t:t + 1])
        s = int(slots[b, t])
        if s >= 0:
            for x, y in zip(mine, all_pools):
                assert bits(x[s // 16, :, s % 16]) == bits(y[s // 16, :, s % 16])


def test_rope_into_a_pool_past_32_bits():
    """Pages whose offsets pass 2^32 elements."""
    bi = _bi()
    stride = (1 << 32) + 512
    base = torch.empty(stride + 8 * 1024, dtype=torch.bfloat16, device="cuda")
    pool = base.as_strided((2, 2, 8, 64), (stride, 512, 64, 1))
    pool.zero_()
    q, k, v, cos, sin, pos, _, _ = _rope_case("bf16", "f32", 1, 2, (4, 2), 64, (32,), 8, 7)
    other = torch.zeros(2, 2, 8, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.tensor([[3, 13]], device="cuda")
    got = bi.rope_paged_cache(q, k, v, cos, sin, pos, slots, other, pool)
    want = [torch.zeros_like(other) for _ in range(2)]
    assert bits(got) == bits(bi.rope_paged_cache(q, k, v, cos, sin, pos, slots, *want))
    assert bits(other) == bits(want[0]) and bits(pool.contiguous()) == bits(want[1])


def test_rope_refuses_pools_it_cannot_write():
    o = [t for t in _rope_case("bf16", "f32", 1, 2, (4, 2), 64, (32,), 8, 8)]
    q, k, v, cos, sin, pos, slots, pools = o
    f = lambda kp, vp: _bi().rope_paged_cache(q, k, v, cos, sin, pos, slots, kp, vp)
    shape = tuple(pools[0].shape)
    skew = torch.zeros(*shape[:3], 68, dtype=torch.bfloat16, device="cuda")[..., :64]
    for bad, match in ((skew, "aligned"), (pools[0][:1].expand(shape), "share memory"),
                       (pools[0].clone().requires_grad_(), "gradient"), (pools[0].cpu(), "GPU")):
        with pytest.raises(ValueError, match=match):
            f(bad, pools[1])
        with pytest.raises(ValueError, match=match):
            f(pools[0], bad)
    before = pools[0]._version, pools[1]._version
    f(*pools)
    assert pools[0]._version > before[0] and pools[1]._version > before[1]
    f(pools[0], pools[1])
    assert _bi().rope_paged_cache(q[:, :0], k[:, :0], v[:, :0], cos, sin, pos[:, :, :0], slots[:, :0],
                                  *pools).shape == (1, 4, 0, 64)


def test_steps_captured_in_a_graph():
    """Plan and rotation of a decode step captured on a side stream and replayed:
    lengths and cursor handed on between the replays, each checked against the
    plain forms, with eager work in between."""
    bi = _bi()
    B, page, cols = 6, 4, 5
    q, k, v, cos, sin, _, _, pools = _rope_case("f16", "f32", B, 1, (4, 2), 32, (16,), page, 9)
    pools = [torch.zeros(B * cols, 2, page, 32, dtype=torch.float16, device="cuda") for _ in range(2)]
    lens = torch.tensor([0, 3, 4, 7, 8, 16], dtype=I32, device="cuda")
    news = torch.ones(B, dtype=I32, device="cuda")
    table = torch.zeros(B, cols, dtype=I32, device="cuda")
    free = torch.randperm(B * cols, generator=gen(1)).to(I32).cuda()
    first = bi.paged_slots(torch.zeros_like(lens), lens, table, free, page_size=page, max_new=16)
    cur = first.cursor.clone()
    shadow = ref.slots([0] * B, lens.tolist(), [[0] * cols] * B, free.tolist(), page, 16)

    def step():
        p = bi.paged_slots(lens, news, table, free, page_size=page, max_new=1, cursor=cur)
        return p, bi.rope_paged_cache(q, k, v, cos, sin, p.positions, p.slots, *pools)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()                                          # leaves lengths and cursor as they are
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, out = step()
    for i in range(4):
        before = [p.cpu().clone() for p in pools]
        q.copy_(randn(q.shape, q.dtype, gen(20 + i)))
        k.copy_(randn(k.shape, k.dtype, gen(30 + i)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = ref.slots(lens.tolist(), [1] * B, shadow[4], free.tolist(), page, 1, cur.item())
        assert [plan.slots.tolist(), plan.positions.tolist(), plan.kv_lens.tolist(), plan.cursor.item(),
                table.tolist()] == list(want)
        _rope_check(out, pools, before, q, k, v, cos, sin, plan.positions[None], plan.slots, (16,), "f16")
        shadow = want
        lens.copy_(plan.kv_lens)
        cur.copy_(plan.cursor)
    del graph


def test_operators_of_the_dispatcher():
    bi = _bi()
    q, k, v, cos, sin, pos, slots, pools = _rope_case("bf16", "f32", 2, 3, (4, 2), 64, (8, 24), 8, 11)
    other = [p.clone() for p in pools]
    a = bi.rope_paged_cache(q, k, v, cos, sin, pos, slots, *pools, sections=(8, 24))
    b = torch.ops.mlx_bi.rope_paged_cache(q, k, v, cos, sin, pos, slots, *other, [8, 24])
    assert bits(a) == bits(b) and all(bits(x) == bits(y) for x, y in zip(pools, other))
    i = lambda *x: torch.tensor(x, dtype=I32, device="cuda")
    t1, t2 = torch.zeros(2, 2, dtype=I32, device="cuda"), torch.zeros(2, 2, dtype=I32, device="cuda")
    p = bi.paged_slots(i(0, 5), i(3, 1), t1, i(8, 9), page_size=4, max_new=3)
    for x, y in zip(p, torch.ops.mlx_bi.paged_slots(i(0, 5), i(3, 1), t2, i(8, 9), None, 4, 3)):
        assert torch.equal(x, y)
    assert torch.equal(t1, t2)


def test_rope_refuses_one_pool_for_both():
    q, k, v, cos, sin, pos, slots, pools = _rope_case("bf16", "f32", 1, 2, (4, 2), 64, (32,), 8, 8)
    with pytest.raises(ValueError, match="one pool"):
        _bi().rope_paged_cache(q, k, v, cos, sin, pos, slots, pools[0], pools[0])
