"""The quantized cache and the attention behind shared prefixes as a server runs them:
a batch's prompts, chunks and decode steps with the planning of its pages, eager and
captured, on two streams, in pools whose offsets pass 32 bits, and as torch.ops."""

import pytest
import torch

from helpers import DT, bits, gen, randn
from test_gpu_quantized_cache import pack, quantize_rows, random_pool, values

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _bi():
    import mlx_batch_invariant_amd as bi
    return bi


def dev(x, dtype=I32):
    return torch.tensor(x, dtype=dtype, device="cuda")


class _Model:
    """One block's heads over a quantized pool and, beside it, over the plain one."""

    def __init__(self, nbits, gs, dt, B, Hq=6, Hkv=2, D=64, page=16, pages=120, cols=40, half=32):
        bi = _bi()
        self.bi, self.dt, self.B, self.Hq, self.Hkv, self.D, self.page = bi, DT[dt], B, Hq, Hkv, D, page
        ang = torch.rand(cols * page, half, generator=gen(5)) * 6
        self.cos, self.sin = ang.cos().cuda(), ang.sin().cuda()
        self.free = torch.randperm(pages, generator=gen(6)).to(I32).cuda()
        self.table = torch.zeros(B, cols, dtype=I32, device="cuda")
        self.lens, self.cursor = dev([0] * B), dev([0])
        self.quant = [bi.quantized_pages(pages, Hkv, page, D, bits=nbits, group_size=gs, dtype=self.dt) for _ in range(2)]
        self.plain = [torch.zeros(pages, Hkv, page, D, dtype=self.dt, device="cuda") for _ in range(2)]

    def tokens(self, T, g):
        return [randn((self.B, T, h, self.D), self.dt, g) for h in (self.Hq, self.Hkv, self.Hkv)]

    def step(self, q, k, v, news, plain=False):
        T = q.shape[1]
        plan = self.bi.paged_slots(self.lens, news, self.table, self.free, page_size=self.page, max_new=T, cursor=self.cursor)
        where = (self.cos, self.sin, plan.positions, plan.slots)
        if plain:
            self.bi.rope_paged_cache(q, k, v, *where, *self.plain)
        turned = self.bi.rope_quantized_cache(q, k, v, *where, *self.quant)
        self.lens, self.cursor = plan.kv_lens, plan.cursor
        return turned, self.bi.batch_invariant_quantized_paged_attention(turned, *self.quant, self.table, self.lens, mask="causal")


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nbits,gs", [(8, 64), (4, 32)])
def test_prompts_chunks_and_decode(dt, nbits, gs):
    """Padded prompts, chunks and decode steps leave the quantizer's codes and give the plain
    attention's bits over the values that the pages stand for."""
    m, g = _Model(nbits, gs, dt, 3), gen(9)
    for T, news in ((300, [37, 0, 300]), (40, [40, 11, 0]), (16, [16, 16, 9]), (1, [1, 1, 1]), (3, [3, 0, 2]), (1, [0, 1, 1])):
        before = m.lens.tolist()
        turned, got = m.step(*m.tokens(T, g), dev(news), plain=True)
        assert m.lens.tolist() == [a + b for a, b in zip(before, news)]
        for p, rows in zip(m.quant, m.plain):
            codes, groups = quantize_rows(rows.cpu(), nbits, gs)
            written = (rows != 0).any(-1, keepdim=True).cpu()        # (a page row without a token is all zeros)
            assert torch.equal(torch.where(written, p.codes.cpu(), 0), torch.where(written, pack(codes, nbits), 0))
            assert torch.equal(torch.where(written[..., None], p.groups.cpu(), 0), torch.where(written[..., None], groups, 0))
        dense = [values(p).cuda() for p in m.quant]
        want = m.bi.batch_invariant_paged_attention(turned, *dense, m.table, m.lens, mask="causal")
        assert torch.equal(got, want)
        for b in range(3):
            if T > int(m.lens[b]):
                assert (got[b, :, :T - int(m.lens[b])] == 0).all()     # rows in front of a short sequence


def test_captured_decode_steps():
    """A captured step that plans, writes and attends; replays between eager work continue the batch
    as eager steps do."""
    runs = []
    for captured in (False, True):
        m, g = _Model(8, 64, "bf16", 4), gen(21)
        m.step(*m.tokens(250, g), dev([250, 3, 0, 100]))
        held, news = m.tokens(1, g), dev([1, 1, 1, 1])
        lens, cursor = m.lens.clone(), m.cursor.clone()

        def step():
            m.lens, m.cursor = lens, cursor
            out = m.step(*held, news)[1]
            lens.copy_(m.lens)
            cursor.copy_(m.cursor)
            return out

        outs = []
        if captured:
            state = [t.clone() for t in (lens, cursor, m.table)]
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                step()
            torch.cuda.current_stream().wait_stream(stream)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
            for t, s in zip((lens, cursor, m.table), state):
                t.copy_(s)
        for i in range(9):                                       # (the first sequence passes a split and a page)
            for h, x in zip(held, m.tokens(1, gen(100 + i))):
                h.copy_(x)
            news.copy_(dev([1, i % 2, 1, 1]))
            if captured:
                graph.replay()
                torch.cuda.synchronize()
                outs.append(out.clone())
            else:
                outs.append(step())
        runs.append((outs, lens.tolist(), values(m.quant[0]), values(m.quant[1])))
    (a, la, ka, va), (b, lb, kb, vb) = runs
    assert la == lb and la[0] == 259
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert torch.equal(ka, kb) and torch.equal(va, vb)


@pytest.mark.parametrize("nbits", [0, 8, 4])
def test_branches_of_one_prompt(nbits):
    """Samples of one prompt: pages of the prompt in every row of the table, a token each into pages of their
    own, and the shared attention's bits are the plain one's."""
    bi, g = _bi(), gen(31)
    B, Hq, Hkv, D, page, P = 11, 8, 2, 64, 16, 600
    first = P // page
    n = first + 2 * B
    table = torch.cat([torch.arange(first).expand(B, first), first + torch.arange(2 * B).reshape(B, 2)], 1).to(I32).cuda()
    if nbits:
        pools = [random_pool(n, Hkv, page, D, nbits, 32, "bf16", g) for _ in range(2)]
    else:
        pools = [randn((n, Hkv, page, D), torch.bfloat16, g) for _ in range(2)]
    lens = dev([P // page * page + 1 + b for b in range(B)])         # (each in its first own page, to whose end it is filled at most)
    ang = torch.rand(1024, 16, generator=g)
    for T in (1, 1, 3):
        q, k, v = (randn((B, T, h, D), torch.bfloat16, g) for h in (Hq, Hkv, Hkv))
        plan = bi.paged_slots(lens, dev([T] * B), table, dev([]), page_size=page, max_new=T)
        write = bi.rope_quantized_cache if nbits else bi.rope_paged_cache
        q = write(q, k, v, ang.cos().cuda(), ang.sin().cuda(), plan.positions, plan.slots, *pools)
        lens = plan.kv_lens
        if nbits:
            call = lambda **kw: bi.batch_invariant_quantized_paged_attention(q, *pools, table, lens, mask="causal", **kw)
            want = call()
        else:
            call = lambda **kw: bi.batch_invariant_shared_prefix_attention(q, *pools, table, lens, mask="causal", **kw)
            want = bi.batch_invariant_paged_attention(q, *pools, table, lens, mask="causal")
        assert torch.equal(call(shared_lens=P), want)
        assert torch.equal(call(shared_starts=dev([0, 5, B]), shared_lens=dev([512, 300])), want)


def test_two_streams():
    """Calls of two streams at once keep to workspaces of their own."""
    bi = _bi()
    work = []
    for i in range(2):
        g = gen(40 + i)
        B, n = 6 + i, 400
        table = torch.randperm(n, generator=g)[:B * 50].reshape(B, 50).to(I32).cuda()
        lens = dev([800 - 90 * b for b in range(B)])
        pools = [random_pool(n, 2, 16, 64, 8 - 4 * i, 32, "bf16", g) for _ in range(2)]
        qs = [randn((B, 8, T, 64), torch.bfloat16, g) for T in (1, 2, 40)]
        work.append((qs, pools, table, lens))

    def calls(w):
        qs, pools, table, lens = w
        out = [bi.batch_invariant_quantized_paged_attention(q, *pools, table, lens, mask="causal") for q in qs]
        return out + [bi.batch_invariant_quantized_paged_attention(qs[0], *pools, table, lens, mask="causal", shared_lens=0)]

    want = [calls(w) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = [[], []]
    for _ in range(10):
        for i, (s, w) in enumerate(zip(streams, work)):
            with torch.cuda.stream(s):
                got[i].append(calls(w))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(out, want[i]))


@pytest.mark.parametrize("nbits", [8, 4])
def test_far_pages(nbits):
    """Pools whose pages lie 2 GiB apart: offsets past 32 bits in the write, the reading and every attention."""
    bi, g = _bi(), gen(50)
    Hkv, D, page, n, far = 2, 64, 16, 4, 1 << 31
    width = D * nbits // 8
    pools = []
    for _ in range(2):
        memory = torch.zeros((n - 1) * far + Hkv * page * width, dtype=torch.uint8, device="cuda")
        codes = memory.as_strided((n, Hkv, page, width), (far, page * width, width, 1))
        near = random_pool(n, Hkv, page, D, nbits, 32, "bf16", g)
        codes.copy_(near.codes)
        pools.append((bi.QuantizedPages(codes, near.groups.clone(), nbits, 32), near))
    far_p, near_p = [p[0] for p in pools], [p[1] for p in pools]
    q, k, v = (randn((2, 3, h, D), torch.bfloat16, g) for h in (8, Hkv, Hkv))
    ang = torch.rand(64, 16, generator=g)
    slots = dev([[3 * page + 1, 2, -1], [2 * page, 3 * page + 15, page + 3]], torch.int64)
    out = [bi.rope_quantized_cache(q, k, v, ang.cos().cuda(), ang.sin().cuda(), torch.zeros(2, 3, dtype=I32, device="cuda"),
                                   slots, *p) for p in (far_p, near_p)]
    assert bits(out[0]) == bits(out[1])
    for a, b in zip(far_p, near_p):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.groups, b.groups)
    table = torch.randint(0, n, (2, 40), generator=g).to(I32).cuda()
    table[:, 0], table[:, 39] = 3, 3
    lens = dev([640, 301])
    for x, y in zip(bi.read_quantized_cache(*far_p, table, lens), bi.read_quantized_cache(*near_p, table, lens)):
        assert torch.equal(x, y)
    for T in (1, 3, 9, 200):
        q = randn((2, 8, T, D), torch.bfloat16, g)
        for more in ({}, dict(shared_lens=300)):
            a, b = (bi.batch_invariant_quantized_paged_attention(q, *p, table, lens, mask="causal", **more) for p in (far_p, near_p))
            assert torch.equal(a, b), (T, more)
    # (of rows 2^32 or more apart a lane cannot tell the offset)
    memory = torch.zeros(2 * far + 16 * 32 * Hkv * D, dtype=torch.uint8, device="cuda")
    codes = memory.as_strided((2, Hkv, page, width), (2 * far, page * width, width, 1))
    wide = bi.QuantizedPages(codes, far_p[0].groups[:2], nbits, 32)
    with pytest.raises(NotImplementedError, match="2\\^32"):
        bi.batch_invariant_quantized_paged_attention(q, wide, wide, table, lens)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (6, 1)])
def test_rows_to_either_way(dt, Hq, Hkv):
    """Around the sizes from which rows are scored over all keys at a time, the bits stay."""
    bi, g = _bi(), gen(60)
    B, D, page, cols, groups = 20, 64, 16, 20, 2
    n = B * cols
    table = torch.randperm(n, generator=g).reshape(B, cols).to(I32)
    table[:, :16] = table[:1, :16]
    table, lens = table.cuda(), dev([300 - b for b in range(B)])
    quant = [random_pool(n, Hkv, page, D, 8, 64, dt, g) for _ in range(2)]
    plain = [values(p).cuda() for p in quant]
    share = dict(shared_starts=dev([0, 7, B]), shared_lens=dev([256, 256]))
    for rows in (12, 16, 20, 60, 64, 72):
        T = rows * Hkv // Hq
        q = randn((B, Hq, T, D), DT[dt], g)
        want = bi.batch_invariant_paged_attention(q, *plain, table, lens, mask="causal")
        for more in ({}, share):
            assert torch.equal(bi.batch_invariant_quantized_paged_attention(q, *quant, table, lens, mask="causal", **more), want)
        assert torch.equal(bi.batch_invariant_shared_prefix_attention(q, *plain, table, lens, mask="causal", **share), want)


@pytest.mark.parametrize("B,groups", [(140, 51), (140, 52), (140, 53), (200, 55), (200, 56), (200, 57), (2000, 100)])
def test_plans_of_many_segments(B, groups):
    """Plans that every workgroup makes, that one makes, and of more segments than LDS keeps."""
    bi, g = _bi(), gen(B + groups)
    page, cols, D = 64, 12, 32
    edges = torch.sort(torch.randint(0, B + 1, (groups + 1,), generator=g)).values
    table = torch.randint(0, 900, (B, cols), generator=g)
    shared = torch.randint(0, 700, (groups,), generator=g)
    lens = torch.randint(0, cols * page, (B,), generator=g)
    for n in range(groups):
        a, b = int(edges[n]), int(edges[n + 1])
        table[a:b, :int(shared[n]) // page + 1] = table[a:a + 1, :int(shared[n]) // page + 1]
        lens[a:b].clamp_(min=int(shared[n]))
    table, lens = table.to(I32).cuda(), lens.to(I32).cuda()
    pools = [randn((900, 1, page, D), torch.bfloat16, g) for _ in range(2)]
    q = randn((B, 3, 1, D), torch.bfloat16, g)
    got = bi.batch_invariant_shared_prefix_attention(q, *pools, table, lens, shared_starts=edges.to(I32).cuda(),
                                                     shared_lens=shared.to(I32).cuda())
    assert torch.equal(got, bi.batch_invariant_paged_attention(q, *pools, table, lens))


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (7, 7)])
def test_write_odd_heads_and_long_tokens(Hq, Hkv):
    bi, g = _bi(), gen(70 + Hq)
    B, T, D, page = 2, 77, 96, 16
    q, k, v = (randn((B, T, h, D), torch.float16, g) for h in (Hq, Hkv, Hkv))
    ang = torch.rand(128, 24, generator=g) * 6
    pos = torch.arange(T).expand(B, T).to(I32).cuda()
    slots = torch.randperm(12 * page, generator=g)[:B * T].reshape(B, T).cuda()
    plain = [torch.zeros(12, Hkv, page, D, dtype=torch.float16, device="cuda") for _ in range(2)]
    quant = [bi.quantized_pages(12, Hkv, page, D, bits=8, group_size=32, dtype=torch.float16) for _ in range(2)]
    where = (ang.cos().cuda(), ang.sin().cuda(), pos, slots)
    assert bits(bi.rope_quantized_cache(q, k, v, *where, *quant)) == bits(bi.rope_paged_cache(q, k, v, *where, *plain))
    put = torch.zeros(12 * page, 1, dtype=torch.bool)
    put[slots.cpu().flatten()] = True
    put = put.view(12, 1, page, 1)
    for p, rows in zip(quant, plain):
        codes, groups = quantize_rows(rows.cpu(), 8, 32)
        assert torch.equal(p.codes.cpu(), torch.where(put, codes, 0))
        assert torch.equal(p.groups.cpu(), torch.where(put[..., None], groups, 0))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nbits", [8, 4])
def test_codes_are_the_quotients(dt, nbits):
    """Groups of every magnitude, with values at and beside the middles between codes: each code is that of
    the IEEE quotient."""
    bi, g = _bi(), gen(80)
    D, gs, n, page = 128, 32, 64, 64
    top = 2 ** nbits - 1
    # (a range of 2 top steps of a random scale; the halves of a step are the middles)
    scale = torch.exp2(torch.rand(n * page, 4, 1, generator=g) * (200 if dt != "f16" else 12) - (110 if dt != "f16" else 10))
    v = torch.randint(0, 2 * top + 1, (n * page, 4, gs), generator=g) / 2 * scale
    v[..., 0], v[..., 1] = 0.0, top * scale[..., 0]
    v = (v * (1 + torch.randint(-1, 2, v.shape, generator=g) * torch.finfo(DT[dt]).eps)).to(DT[dt])
    v[..., 0] = 0.0
    v = v.reshape(1, n * page, 1, D).cuda()
    k, q = torch.zeros_like(v), torch.zeros_like(v)
    tab = torch.ones(1, 16, device="cuda")
    pools = [bi.quantized_pages(n, 1, page, D, bits=nbits, group_size=gs, dtype=DT[dt]) for _ in range(2)]
    zero = torch.zeros(1, n * page, dtype=I32, device="cuda")
    slots = torch.arange(n * page, device="cuda")[None]
    bi.rope_quantized_cache(q, k, v, tab, tab, zero, slots, *pools)
    codes, groups = quantize_rows(v.cpu().view(n, 1, page, D), nbits, gs)
    assert torch.equal(pools[1].groups.cpu(), groups)
    assert torch.equal(pools[1].codes.cpu(), pack(codes, nbits))


def test_library_ops():
    bi, g, ops = _bi(), gen(90), torch.ops.mlx_bi
    B, T, Hq, Hkv, D, page, n = 2, 3, 4, 2, 64, 16, 40
    table = torch.randperm(n, generator=g).reshape(2, 20).to(I32).cuda()
    lens = dev([300, 290])
    a, b = ([random_pool(n, Hkv, page, D, 4, 32, "bf16", gen(1 + i)) for i in range(2)] for _ in range(2))
    flat = lambda p: (p[0].codes, p[0].groups, p[1].codes, p[1].groups)
    q, k, v = (randn((B, T, h, D), torch.bfloat16, g) for h in (Hq, Hkv, Hkv))
    ang = torch.rand(512, 32, generator=g)
    cos, sin = ang.cos().cuda(), ang.sin().cuda()
    pos, slots = dev([[1, 2, 3]] * 2), dev([[5, 600, -1], [7, 8, 9]], torch.int64)
    want = bi.rope_quantized_cache(q, k, v, cos, sin, pos, slots, *a)
    got = ops.rope_quantized_cache(q, k, v, cos, sin, pos, slots, *flat(b), 4, 32, None)
    assert bits(got) == bits(want)
    for x, y in zip(flat(a), flat(b)):
        assert torch.equal(x, y)
    for x, y in zip(bi.read_quantized_cache(*a, table, lens), ops.read_quantized_cache(*flat(a), table, lens, 4, 32)):
        assert torch.equal(x, y)
    want = bi.batch_invariant_quantized_paged_attention(got, *a, table, lens, scale=0.2, mask="causal", shared_lens=dev([256]))
    assert torch.equal(want, ops.quantized_paged_attention(got, *flat(a), table, lens, 4, 32, 0.2, True, None, dev([256])))
    kd, vd = (values(p).cuda() for p in a)
    want = bi.batch_invariant_shared_prefix_attention(got, kd, vd, table, lens, scale=0.2, shared_starts=dev([0, 2]), shared_lens=dev([256]))
    assert torch.equal(want, ops.shared_prefix_attention(got, kd, vd, table, lens, 0.2, False, dev([0, 2]), dev([256])))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nbits,gs,D", [(4, 32, 64), (4, 64, 128), (4, 32, 256), (8, 64, 64)])
@pytest.mark.parametrize("which", ["k", "v", "kv"])
def test_scales_of_every_size(dt, nbits, gs, D, which):
    """Scales at both ends of their type, in a few keys or all of one wave's, beside ordinary ones."""
    bi, g = _bi(), gen(D + nbits)
    B, Hq, Hkv, page, L, n = 3, 4, 2, 16, 700, 150
    table = torch.randperm(n, generator=g)[:B * 44].reshape(B, 44).to(I32).cuda()
    lens = dev([L, 256, 65])
    high, low = (1e4, 6e-8) if dt == "f16" else (2.0 ** 118, 2.0 ** -130)
    for part in range(3):
        pools = [random_pool(n, Hkv, page, D, nbits, gs, dt, g) for _ in range(2)]
        for p, name in zip(pools, "kv"):
            if name not in which:
                continue
            pages = table.cpu().long()
            rows = (pages[0, 5:6], pages[:, 0:4].flatten(), torch.arange(n))[part]   # one page, the first wave of each, all
            for size, pick in ((high, rows), (low, pages[1, 9:11])):
                p.groups[pick.cuda(), :, ::3] *= size
        for t in ("k" in which and part == 2, False):
            for T in (1, 3):
                q = randn((B, Hq, T, D), DT[dt], g) * (2.0 / high if t else 1.0 / (1 + (high if "k" in which else 0)))
                got = bi.batch_invariant_quantized_paged_attention(q, *pools, table, lens, mask="causal")
                k, v = bi.read_quantized_cache(*pools, table, lens)
                want = bi.batch_invariant_attention(q, k, v, kv_lens=lens, mask="causal")
                assert torch.isfinite(want).all()
                assert torch.equal(got, want), (part, T)
