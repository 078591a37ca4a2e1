"""A paged cache in 8 or 4 bits: the rotary embedding with the quantized write, the
reading back, and attention over the codes. Codes, pairs and values are compared
exactly with the framework's quantizer on the rows that the plain write leaves;
attention bit for bit with the plain attention over the values read back, and with
the 64-bit formula."""

import numpy as np
import pytest
import torch

import paged_ref as ref
from helpers import DT, bits, gen, randn

pytestmark = pytest.mark.gpu
I32 = torch.int32
FORMATS = [(8, 64), (8, 32), (8, 128), (4, 64), (4, 32), (4, 128)]


def formats(*dims):
    """(bits, group size, head dim ...) for every format that divides the head dim; a dim may carry more."""
    return [(b, g, *d) for b, g in FORMATS for d in ((x if isinstance(x, tuple) else (x,)) for x in dims) if d[0] % g == 0]


def _bi():
    import mlx_batch_invariant_amd as bi
    return bi


def quantize_rows(x, nbits, gs):
    """Codes [..., D] and pairs [..., D / gs, 2] of x's type: the quantizer's rule in fp32."""
    top = 2 ** nbits - 1
    y = x.float().unflatten(-1, (-1, gs))
    low, high = y.amin(-1), y.amax(-1)
    s = ((high - low) / top).to(x.dtype).float()
    s = torch.where(s > 0, s, torch.ones_like(s))
    codes = ((y - low[..., None]) / s[..., None]).round().clamp(0, top)
    return codes.flatten(-2).to(torch.uint8), torch.stack([s, low], -1).to(x.dtype)


def pack(codes, nbits):
    return codes if nbits == 8 else codes[..., 0::2] | codes[..., 1::2] << 4


def unpack(codes, nbits):
    return codes if nbits == 8 else torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def values(pages):
    """What a pool stands for, rounded from 64 bits to 32 and to the pairs' type."""
    c = unpack(pages.codes.cpu(), pages.bits).double().unflatten(-1, (-1, pages.group_size))
    g = pages.groups.cpu().double()
    return (c * g[..., :1] + g[..., 1:]).float().to(pages.groups.dtype).flatten(-2)


def random_pool(n, H, page, D, nbits, gs, dt, g, layout="page"):
    """A pool with random codes; `layout` "row": heads inside rows in memory."""
    bi = _bi()
    shape = (n, H, page) if layout == "page" else (n, page, H)
    codes = torch.randint(0, 256, (*shape, D * nbits // 8), generator=g, dtype=torch.uint8).cuda()
    span = (3 + torch.rand((*shape, D // gs), generator=g)) / (2 ** nbits - 1)
    groups = torch.stack([span, -1.5 + 0.3 * torch.randn(span.shape, generator=g)], -1).to(DT[dt]).cuda()
    if layout == "row":
        codes, groups = codes.transpose(1, 2), groups.transpose(1, 2)
    return bi.QuantizedPages(codes, groups, nbits, gs)


# ---- the write -------------------------------------------------------------------

@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nbits,gs,D,half,sections,page", formats(
    (128, 64, None, 16), (256, 128, (40, 48, 40), 1), (64, 16, None, 64), (96, 24, (8, 16), 4), (192, 96, None, 8),
    (32, 16, None, 256)))
def test_write(dt, nbits, gs, D, half, sections, page):
    bi, g = _bi(), gen(D + gs + nbits)
    B, T, Hq, Hkv, P = 3, 7, 5, 2, 64 // page + 6
    q, k, v = (randn((B, T, h, D), DT[dt], g) for h in (Hq, Hkv, Hkv))
    A = 1 if sections is None else len(sections)
    pos = torch.randint(0, 40, (A, B, T), generator=g).to(I32).cuda()
    ang = torch.rand(40, half, generator=g) * 6
    cos, sin = ang.cos().cuda(), ang.sin().cuda()
    slots = torch.randperm(P * page, generator=g)[:B * T].reshape(B, T).cuda() if P * page >= B * T else None
    slots[0, :3], slots[1, 2], slots[2, 1] = -1, P * page, -(1 << 40)
    pools = [torch.zeros(P, Hkv, page, D, dtype=DT[dt], device="cuda") for _ in range(2)]
    qw = bi.rope_paged_cache(q, k, v, cos, sin, pos, slots, *pools, sections=sections)
    for layout in ("page", "row"):
        quant = [random_pool(P, Hkv, page, D, nbits, gs, dt, gen(1 + i), layout) for i in range(2)]
        before = [(p.codes.clone(), p.groups.clone()) for p in quant]
        qg = bi.rope_quantized_cache(q, k, v, cos, sin, pos, slots, *quant, sections=sections)
        assert bits(qg) == bits(qw)
        put = torch.zeros(P * page, dtype=torch.bool)
        put[slots[(slots >= 0) & (slots < P * page)].cpu()] = True
        put = put.view(P, 1, page, 1)
        for p, plain, (codes0, groups0) in zip(quant, pools, before):
            codes, groups = quantize_rows(plain.cpu(), nbits, gs)
            assert torch.equal(p.codes.cpu(), torch.where(put, pack(codes, nbits), codes0.cpu())), layout
            want = torch.where(put[..., None], groups, groups0.cpu())
            assert bits(p.groups) == bits(want), layout


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nbits", [8, 4])
def test_write_extremes(dt, nbits):
    """Constant groups, tiny ranges, ranges as large as the type's, infinities and NaN."""
    bi, fi = _bi(), torch.finfo(DT[dt])
    D, gs = 64, 32
    v = torch.randn(1, 9, 1, D, generator=gen(3))
    v[0, 0] = 2.5
    v[0, 1] = 0.0
    v[0, 2] *= fi.tiny * 4
    v[0, 3] = torch.tensor([fi.max, fi.min]).repeat(D // 2)
    v[0, 4, 0, 5] = float("inf")
    v[0, 5, 0, 40] = float("nan")
    v[0, 6, 0, :gs] = torch.linspace(fi.max / 2, fi.max, gs)
    v[0, 6, 0, gs:] = torch.linspace(fi.min, 0, gs)
    v[0, 7] = fi.smallest_normal * fi.eps * torch.arange(D)
    v[0, 8] = -7.0
    v[0, 8, 0, 0] = -6.875
    v = v.to(DT[dt])
    pools = [bi.quantized_pages(1, 1, 16, D, bits=nbits, group_size=gs, dtype=DT[dt]) for _ in range(2)]
    table = torch.ones(16, 8, device="cuda")
    one = v.cuda()
    bi.rope_quantized_cache(one, one, one, table, 0 * table, torch.zeros(1, 9, dtype=I32, device="cuda"),
                            torch.arange(9, device="cuda")[None], *pools)
    for pool in pools:                                   # (a turn by 0: keys are the same rows)
        got = values(pool)[0, 0, :9].double()
        gpu = bi.read_quantized_cache(pool, pool, torch.zeros(1, 1, dtype=I32, device="cuda"))[0][0, 0, :9].cpu().double()
        x = v[0, :, 0].double()
        for i in range(9):
            for n in range(2):
                y, z, w = (t[i, n * gs:(n + 1) * gs] for t in (got, gpu, x))
                if not torch.isfinite(w).all():
                    assert torch.isnan(y).all() and torch.isnan(z).all(), i
                    continue
                assert torch.isfinite(z).all() and torch.equal(y, z), i
                # a step at most: half from the code, the rest from the scale's rounding (eps / 2 of the range,
                # half a step of 8 bits in bf16 and less than that elsewhere), the type's own steps (results and scale)
                step = max((w.max() - w.min()).item() / (2 ** nbits - 1), 0.0)
                tiny = fi.smallest_normal * fi.eps
                slack = 2 ** nbits * tiny + fi.eps * w.abs().max().item()
                assert (z - w).abs().max().item() <= step + slack + fi.eps * (w.max() - w.min()).item(), i


def test_write_strided_operands_and_empty():
    """Slices of a joint projection, int32 slots, tables in the operands' type; no tokens."""
    bi, g = _bi(), gen(9)
    B, T, Hq, Hkv, D = 2, 3, 4, 2, 64
    qkv = randn((B, T, (Hq + 2 * Hkv) * D), torch.bfloat16, g)
    q, k, v = (t.view(B, T, -1, D) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], -1))
    cos, sin = (randn((9, D // 2), torch.bfloat16, g) for _ in range(2))
    pos, slots = torch.arange(T).repeat(B, 1).to(I32).cuda(), torch.arange(B * T).view(B, T).cuda()
    new = lambda: [bi.quantized_pages(3, Hkv, 4, D) for _ in range(2)]
    a, b = new(), new()
    assert bits(bi.rope_quantized_cache(q, k, v, cos, sin, pos, slots, *a)) == bits(
        bi.rope_quantized_cache(q.contiguous(), k.contiguous(), v.contiguous(), cos, sin, pos, slots.to(I32), *b))
    for x, y in zip(a, b):
        assert torch.equal(x.codes, y.codes) and bits(x.groups) == bits(y.groups)
    versions = [t._version for t in (a[0].codes, a[0].groups, a[1].codes, a[1].groups)]
    out = bi.rope_quantized_cache(q[:, :0], k[:, :0], v[:, :0], cos, sin, pos[:, :0], slots[:, :0], *a)
    assert out.shape == (B, Hq, 0, D)
    bi.rope_quantized_cache(q, k, v, cos, sin, pos, slots, *a)
    assert [t._version for t in (a[0].codes, a[0].groups, a[1].codes, a[1].groups)] == [x + 1 for x in versions]


# ---- the reading back ----------------------------------------------------------------

@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nbits,gs,D,page,layout", formats((128, 16, "page"), (96, 1, "row"), (256, 4, "page"),
                                                           (64, 64, "row")))
def test_read(dt, nbits, gs, D, page, layout):
    bi, g = _bi(), gen(D + page)
    B, H, cols, n = 4, 3, 150 // page + 1, 700 // page + 8
    kp, vp = (random_pool(n, H, page, D, nbits, gs, dt, g, layout) for _ in range(2))
    table = torch.randint(0, n, (B, cols), generator=g).to(I32)
    table[1, 0], table[2, -1] = -7, 1 << 30
    lens = torch.tensor([cols * page, 0, 77, -3], dtype=I32)
    for ls in (lens, None):
        got = bi.read_quantized_cache(kp, vp, table.cuda(), None if ls is None else ls.cuda())
        rows = table.clamp(0, n - 1).long()
        for x, p in zip(got, (kp, vp)):
            want = values(p)[rows].transpose(1, 2).reshape(B, H, cols * page, D)
            if ls is not None:
                want = want * (torch.arange(cols * page) < ls[:, None])[:, None, :, None]
            assert x.dtype == DT[dt] and torch.equal(x.cpu().double(), want.double())


# ---- attention ------------------------------------------------------------------------

def _requests(g, B, L, page, spare=5):
    cols = -(-L // page)
    table = torch.randperm(B * cols + spare, generator=g)[:B * cols].reshape(B, cols).to(I32)
    return table, B * cols + spare


def _check_bits(dt, nbits, gs, Hq, Hkv, D, T, L, lens, page, mask, seed, layout="page"):
    bi, g = _bi(), gen(seed)
    B = len(lens)
    table, n = _requests(g, B, L, page)
    kp, vp = (random_pool(n, Hkv, page, D, nbits, gs, dt, g, layout) for _ in range(2))
    q = randn((B, Hq, T, D), DT[dt], g, 2.0)
    lens = torch.tensor(lens, dtype=I32, device="cuda")
    table = table.cuda()
    got = bi.batch_invariant_quantized_paged_attention(q, kp, vp, table, lens, mask=mask)
    k, v = bi.read_quantized_cache(kp, vp, table, lens)
    want = bi.batch_invariant_attention(q, k, v, kv_lens=lens, mask=mask)
    assert torch.equal(got, want), (got.float() - want.float()).abs().max()
    return q, k, v, lens, got, (kp, vp, table)


LENS = [0, 1, 255, 256, 257, 700, 1023]


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nbits,gs,D", formats(32, 64, 96, 128, 192, 256))
def test_decode_bits(dt, nbits, gs, D):
    _check_bits(dt, nbits, gs, 8, 2, D, 1, 1024, LENS, 16, None, D + gs)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (6, 2), (7, 1), (16, 1), (20, 1), (34, 2), (8, 8)])
@pytest.mark.parametrize("page,layout", [(1, "page"), (2, "row"), (32, "row"), (256, "page"), (1024, "row")])
def test_decode_heads_and_pages(dt, Hq, Hkv, page, layout):
    _check_bits(dt, 8, 64, Hq, Hkv, 64, 1, 1024, LENS, page, "causal", Hq + page, layout)
    _check_bits(dt, 4, 32, Hq, Hkv, 64, 1, 300, [300, 0, 299], page, None, Hq + page + 1, layout)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nbits,gs,D", [(8, 64, 64), (4, 32, 96), (8, 128, 128), (4, 64, 192), (8, 32, 256)])
@pytest.mark.parametrize("T", [2, 5, 16, 33, 130, 400])
def test_chunks_bits(dt, nbits, gs, D, T):
    """From a few draft tokens to prompts read back first; rows in front of short sequences see nothing."""
    _check_bits(dt, nbits, gs, 6, 2, D, T, 1024, [1024, 3, 700, 0, 257], 16, "causal", T + D)
    _check_bits(dt, nbits, gs, 4, 4, D, T, 500, [500, 260], 4, None, T + D + 1)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_one_split(dt):
    """Caches of at most 256 keys: no merge."""
    for T in (1, 3, 40):
        _check_bits(dt, 8, 64, 8, 2, 64, T, 256, [256, 0, 1, 100], 16, "causal", T)
        _check_bits(dt, 4, 64, 40, 2, 64, T, 64, [64, 0, 7], 64, None, T)


def test_many_short_sequences():
    """More sequences than a wave has lanes, most of them empty or one token long."""
    g = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 3, (300,), generator=g) * torch.randint(0, 400, (300,), generator=g)
    for T in (1, 9):
        _check_bits("bf16", 8, 32, 4, 2, 32, T, 800, lens.tolist(), 16, "causal", 11 + T)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T", [1, 6, 260])
def test_values(dt, T):
    q, k, v, lens, got, _ = _check_bits(dt, 8, 64, 4, 2, 64, T, 600, [600, 290], 8, "causal", 5)
    want, absv, dot, bias = ref.attention(q.cpu(), k.cpu(), v.cpu(), 64 ** -0.5, lens.cpu(), True)
    allow = ref.attention_allowance(want, absv, dot, bias, DT[dt], 64, 3)
    assert ((got.cpu().double() - want).abs() <= allow).all()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 192, 256])
@pytest.mark.parametrize("T", [1, 4, 300])
def test_hidden_and_seen_nans(dt, D, T):
    """Rows behind a sequence, and rows that the causal mask hides, may hold anything; a NaN
    that a query sees in V comes out in its group of dims, one in K in the whole row."""
    bi, g = _bi(), gen(D + T)
    B, L, page, gs = 2, 512, 16, 64
    table, n = _requests(g, B, L, page)
    kp, vp = (random_pool(n, 2, page, D, 8, gs, dt, g) for _ in range(2))
    q = randn((B, 4, T, D), DT[dt], g)
    lens = torch.tensor([330, 301], dtype=I32)
    args = (table.cuda(), lens.cuda())
    clean = bi.batch_invariant_quantized_paged_attention(q, kp, vp, *args, mask="causal")
    assert torch.isfinite(clean).all()
    for b in range(B):                                   # behind the sequences
        for p in range(int(lens[b]), L):
            for pool in (kp, vp):
                pool.groups[table[b, p // page], :, p % page] = float("nan")
    again = bi.batch_invariant_quantized_paged_attention(q, kp, vp, *args, mask="causal")
    assert torch.equal(again, clean)
    if T > 1:                                            # sequence 0's last key: its last row alone sees it
        p = int(lens[0]) - 1
        vp.groups[table[0, p // page], 1, p % page, 0] = float("nan")
        got = bi.batch_invariant_quantized_paged_attention(q, kp, vp, *args, mask="causal")
        want = clean.clone()
        want[0, 2:, -1, :gs] = float("nan")
        assert torch.equal(torch.nan_to_num(got.float(), 1e4), torch.nan_to_num(want.float(), 1e4))
        kp.groups[table[0, p // page], 0, p % page, 0] = float("nan")
        got = bi.batch_invariant_quantized_paged_attention(q, kp, vp, *args, mask="causal")
        want[0, :2, -1] = float("nan")
        assert torch.equal(torch.nan_to_num(got.float(), 1e4), torch.nan_to_num(want.float(), 1e4))


def test_batch_and_chunk_invariance():
    """A sequence alone, in a batch, in chunks and token by token: the same bits."""
    dt, D, page, L = torch.bfloat16, 128, 16, 640
    bi, g = _bi(), gen(8)
    table, n = _requests(g, 6, L, page)
    kp, vp = (random_pool(n, 2, page, D, 4, 64, "bf16", g) for _ in range(2))
    lens = torch.tensor([640, 5, 300, 511, 640, 257], dtype=I32).cuda()
    table, T = table.cuda(), 250
    q = randn((6, 8, T, D), dt, g)
    call = bi.batch_invariant_quantized_paged_attention
    full = call(q, kp, vp, table, lens, mask="causal")
    for b in range(6):
        assert torch.equal(call(q[b:b + 1], kp, vp, table[b:b + 1], lens[b:b + 1], mask="causal"), full[b:b + 1])
    for t0, t1 in ((0, 3), (3, 103), (103, 104), (249, 250)):
        part = call(q[:, :, t0:t1], kp, vp, table, lens - (T - t1), mask="causal")
        assert torch.equal(part, full[:, :, t0:t1])


def test_slices_of_the_workspace(monkeypatch):
    """Chunks of many rows over a table so wide that its sequences are read back a few at a time."""
    bi, g = _bi(), gen(21)
    D, page, cols = 256, 256, 1 << 10                    # 2^18 keys: 2 x 128 MiB a head and sequence
    kp, vp = (random_pool(40, 4, page, D, 8, 64, "bf16", g) for _ in range(2))
    table = torch.randint(0, 40, (3, cols), generator=g).to(I32).cuda()
    lens = torch.tensor([900, 300, 1500], dtype=I32).cuda()
    q = randn((3, 16, 280, D), torch.bfloat16, g)
    got = bi.batch_invariant_quantized_paged_attention(q, kp, vp, table, lens, mask="causal")
    for b in range(3):
        want = bi.batch_invariant_quantized_paged_attention(q[b:b + 1], kp, vp, table[b:b + 1, :6], lens[b:b + 1], mask="causal")
        assert torch.equal(got[b:b + 1], want)


def test_noncontiguous_queries_and_lists():
    bi, g = _bi(), gen(31)
    table, n = _requests(g, 2, 300, 4)
    kp, vp = (random_pool(n, 2, 4, 64, 8, 64, "f16", g) for _ in range(2))
    q = randn((2, 3, 4, 64), torch.float16, g)
    args = (kp, vp, table.cuda(), [300, 17])
    want = bi.batch_invariant_quantized_paged_attention(q.transpose(1, 2).contiguous(), *args, mask="causal")
    assert torch.equal(bi.batch_invariant_quantized_paged_attention(q.transpose(1, 2), *args, mask="causal"), want)
    odd = torch.empty(2 * 4 * 3 * 64 + 1, dtype=torch.float16, device="cuda")[1:].view(2, 4, 3, 64)
    odd.copy_(q.transpose(1, 2))
    assert torch.equal(bi.batch_invariant_quantized_paged_attention(odd, *args[:2], table.long().cuda(), args[3], mask="causal"), want)
    assert bi.batch_invariant_quantized_paged_attention(odd[:0], kp, vp, table[:0].cuda(), []).shape == (0, 4, 3, 64)


def _seen_values(clean, v, lens, T, mask, G):
    """What comes out where rows see infinities and NaN of v [B, Hkv, L, D]: those, else `clean`."""
    B, _, L, _ = v.shape
    reach = lens[:, None] if mask is None else lens[:, None] - T + 1 + torch.arange(T, device=lens.device)
    seen = (torch.arange(L, device=lens.device) < reach[:, :, None]).expand(B, T, L).float()[:, None]      # [B, 1, T, L]
    v = v.repeat_interleave(G, 1)
    up, down, nan = (torch.matmul(seen, x.float()) > 0 for x in (v == float("inf"), v == -float("inf"), v.isnan()))
    want = clean.clone()
    want[up & ~down] = float("inf")
    want[down & ~up] = -float("inf")
    want[nan | up & down] = float("nan")
    return want


def _same(got, want):
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~got.isnan()], want[~want.isnan()])


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nbits,gs,D", [(8, 64, 64), (8, 32, 96), (4, 32, 64), (4, 64, 128), (4, 32, 256)])
@pytest.mark.parametrize("L", [256, 512])
@pytest.mark.parametrize("T,mask,shared", [(1, None, False), (4, "causal", False), (3, "causal", True), (150, "causal", False),
                                           (150, "causal", True)])
def test_not_finite_codes(dt, nbits, gs, D, L, T, mask, shared):
    """Infinite and NaN scales and biases, seen and hidden, of one split and several, few rows and
    many, behind a shared split too; a scale of 2^101 beside them where the type has it."""
    bi, g = _bi(), gen(D + T + L + nbits)
    B, Hq, Hkv, page, inf, nan = 3, 8, 2, 16, float("inf"), float("nan")
    table, n = _requests(g, B, L, page)
    if shared:
        table[1:, :256 // page] = table[0, :256 // page]
    kp, vp = (random_pool(n, Hkv, page, D, nbits, gs, dt, g) for _ in range(2))
    q = randn((B, Hq, T, D), DT[dt], g)
    lens = [256, 160, 230] if L == 256 else [512, 301, 330]
    at = lambda b, p: (int(table[b, p // page]), p % page)
    if dt != "f16":
        page0, row0 = at(0, 7)
        vp.groups[page0, 0, row0, 0, 0] = 2.0 ** 101
    lens = torch.tensor(lens, dtype=I32, device="cuda")
    args = (table.cuda(), lens)
    more = dict(mask=mask, **(dict(shared_lens=256) if shared else {}))
    clean = bi.batch_invariant_quantized_paged_attention(q, kp, vp, *args, **more)
    assert torch.isfinite(clean).all()
    last = D // gs - 1
    for b, p, h, group, pair in ((0, int(lens[0]) - 1, 0, 0, (0.01, inf)),       # seen by the last row alone
                                 (0, 5, 1, last, (0.02, -inf)), (0, 70, 1, 0, (inf, 1.0)), (1, 130, 0, last, (-inf, 0.5)),
                                 (1, int(lens[1]) - 2, 1, last, (nan, nan)), (2, 3, 1, last, (0.01, inf)),
                                 (1, int(lens[1]) + 1, 0, 0, (0.01, -inf)), (2, int(lens[2]), 1, 0, (inf, -inf)),   # behind sequences
                                 (2, int(lens[2]) + 9, 0, last, (nan, 1.0))):
        pg, row = at(b, p)
        vp.groups[pg, h, row, group] = torch.tensor(pair)
        kp_row = kp.groups[pg, h, row]
        if p >= int(lens[b]) and not shared:
            kp_row.fill_(nan)                             # K behind a sequence may hold anything too
    v = bi.read_quantized_cache(kp, vp, args[0])[1]
    want = _seen_values(clean, v, lens, T, mask, Hq // Hkv)
    got = bi.batch_invariant_quantized_paged_attention(q, kp, vp, *args, **more)
    assert not torch.isfinite(want).all() and _same(got, want)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("T", [1, 6, 200])
def test_not_finite_in_one_shared_split(dt, T):
    """Plain pages, a table of one split: the first sequence's hidden and seen values."""
    bi, g = _bi(), gen(T)
    B, D, page, inf = 4, 64, 16, float("inf")
    table, n = _requests(g, 1, 256, page)
    table = table.expand(B, -1).contiguous()
    kp, vp = (randn((n, 2, page, D), DT[dt], g) for _ in range(2))
    q = randn((B, 8, T, D), DT[dt], g)
    lens = torch.tensor([256, 90, 0, 255], dtype=I32, device="cuda")
    call = lambda: bi.batch_invariant_shared_prefix_attention(q, kp, vp, table.cuda(), lens, mask="causal", shared_lens=256)
    clean = call()
    for p, h, d, x in ((255, 0, 3, inf), (100, 1, 5, -inf), (4, 1, 5, inf), (89, 0, 9, float("nan"))):
        vp[table[0, p // page], h, p % page, d] = x
    v = vp[table.cuda().long()].transpose(1, 2).flatten(2, 3)
    want = _seen_values(clean, v, lens, T, "causal", 4)
    assert not torch.isfinite(want).all() and _same(call(), want)
