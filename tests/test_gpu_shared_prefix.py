"""Attention of sequences that share prefixes: the bits of the plain paged attention,
whatever the groups; the others' table entries of shared splits are not read."""

import pytest
import torch

import paged_ref as ref
from helpers import DT, gen, randn
from test_gpu_quantized_cache import random_pool

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _bi():
    import mlx_batch_invariant_amd as bi
    return bi


def _case(sizes, shared, own, page, g, lead=0, tail=0):
    """A table of groups of `sizes` sequences whose first shared[n] keys (rounded down to whole
    pages) are the same pages, `lead` and `tail` sequences in no group around them; `own`: each
    sequence's further keys. Returns table, lens, starts, pages."""
    B, rows, at = lead + sum(sizes) + tail, [], 0
    cols = (max(shared, default=0) + max(own)) // page + 2
    group = [-1] * lead + [n for n, s in enumerate(sizes) for _ in range(s)] + [-1] * tail
    first = {}
    lens = []
    for b in range(B):
        n = group[b]
        keep = shared[n] // page if n >= 0 else 0
        row = list(range(at, at + cols))
        at += cols
        if n >= 0:
            row[:keep] = first.setdefault(n, row)[:keep]
        rows.append(row)
        lens.append(keep * page + own[b % len(own)])
    order = torch.randperm(at, generator=g)
    starts = [lead]
    for s in sizes:
        starts.append(starts[-1] + s)
    whole = [s // page * page for s in shared]
    return order[torch.tensor(rows)].to(I32), torch.tensor(lens, dtype=I32), starts, whole, at


def _pools(n, Hkv, page, D, dt, g, nbits):
    if nbits:
        return [random_pool(n, Hkv, page, D, nbits, 32, dt, g) for _ in range(2)]
    return [randn((n, Hkv, page, D), DT[dt], g) for _ in range(2)]


def _calls(nbits, q, kp, vp, table, lens, mask, **shared):
    bi = _bi()
    if nbits:
        call = bi.batch_invariant_quantized_paged_attention
        return call(q, kp, vp, table, lens, mask=mask, **shared), call(q, kp, vp, table, lens, mask=mask)
    return (bi.batch_invariant_shared_prefix_attention(q, kp, vp, table, lens, mask=mask, **shared),
            bi.batch_invariant_paged_attention(q, kp, vp, table, lens, mask=mask))


dev = lambda x: torch.tensor(x, dtype=I32, device="cuda")


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nbits", [0, 8, 4])
@pytest.mark.parametrize("T", [1, 4])
@pytest.mark.parametrize("sizes,shared,lead,tail", [([9], [1024], 0, 0), ([2, 1, 5], [600, 900, 256], 1, 2), ([3, 0, 4], [255, 70, 1300], 0, 1),
                                                    ([40], [512], 3, 0)])
def test_bits(dt, nbits, T, sizes, shared, lead, tail):
    g = gen(sum(sizes) + T)
    page, D = 16, 64
    table, lens, starts, whole, n = _case(sizes, shared, [5, 300, 17, 256, 4], page, g, lead, tail)
    kp, vp = _pools(n, 2, page, D, dt, g, nbits)
    q = randn((len(lens), 6, T, D), DT[dt], g, 2.0)
    got, want = _calls(nbits, q, kp, vp, table.cuda(), lens.cuda(), "causal", shared_starts=dev(starts), shared_lens=dev(whole))
    assert torch.equal(got, want)
    got, want = _calls(nbits, q, kp, vp, table.cuda(), lens.cuda(), None, shared_starts=dev(starts), shared_lens=dev(whole))
    assert torch.equal(got, want)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [32, 96, 128, 192, 256])
@pytest.mark.parametrize("Hq,Hkv,page", [(4, 1, 64), (3, 3, 1), (34, 2, 256)])
def test_head_dims(dt, D, Hq, Hkv, page):
    g = gen(D + Hq)
    table, lens, starts, whole, n = _case([5], [768], [40, 1], page, g)
    kp, vp = _pools(n, Hkv, page, D, dt, g, 0)
    q = randn((5, Hq, 1, D), DT[dt], g)
    got, want = _calls(0, q, kp, vp, table.cuda(), lens.cuda(), None, shared_lens=whole[0])
    assert torch.equal(got, want)


@pytest.mark.parametrize("nbits", [0, 8])
def test_pages_of_others_are_not_read(nbits):
    """Only the group's first sequence needs the shared splits' table entries."""
    g = gen(77)
    page, D = 16, 64
    table, lens, starts, whole, n = _case([6], [700], [30, 200], page, g)
    kp, vp = _pools(n, 2, page, D, "bf16", g, nbits)
    q = randn((6, 8, 2, D), torch.bfloat16, g)
    _, want = _calls(nbits, q, kp, vp, table.cuda(), lens.cuda(), "causal", shared_lens=whole[0])
    table[1:, :512 // page] = -1
    got, _ = _calls(nbits, q, kp, vp, table.cuda(), lens.cuda(), "causal", shared_lens=dev([whole[0]]))
    assert torch.equal(got, want)


@pytest.mark.parametrize("starts,shared", [([0, 4, 2, 8], [512, 512, 512]), ([-5, 3, 99], [1 << 30, -4]), ([7, 7, 7], [512, 512]),
                                           ([3, 1], [512]), ([0, 8], [100000])])
def test_odd_groups(starts, shared):
    """Starts that fall, repeat or lie outside the batch, lengths past the keys: with tables that
    are the same everywhere, the plain bits."""
    g = gen(5)
    page, D = 16, 64
    table, lens, _, _, n = _case([8], [1024], [9, 100, 500], page, g)
    lens[2], lens[5] = 0, 300
    kp, vp = _pools(n, 2, page, D, "f16", g, 0)
    q = randn((8, 4, 3, D), torch.float16, g)
    got, want = _calls(0, q, kp, vp, table.cuda(), lens.cuda(), "causal", shared_starts=dev(starts), shared_lens=dev(shared))
    assert torch.equal(got, want)


def test_first_sequence_holds_less():
    """A first sequence shorter than the shared length: what it lacks comes from each one's own pages."""
    g = gen(6)
    page, D = 16, 64
    table, lens, _, whole, n = _case([4], [1024], [9, 100], page, g)
    lens[0] = 300
    kp, vp = _pools(n, 2, page, D, "bf16", g, 0)
    q = randn((4, 4, 1, D), torch.bfloat16, g)
    got, want = _calls(0, q, kp, vp, table.cuda(), lens.cuda(), None, shared_lens=1024)
    assert torch.equal(got, want)


def test_many_groups():
    """More groups and sequences than the plan's workgroup has threads."""
    g = gen(7)
    sizes = [1 + i % 3 for i in range(1300)]
    table, lens, starts, whole, n = _case(sizes, [256] * 1300, [3, 40], 256, g)
    table = table[:, :3].contiguous()
    kp, vp = _pools(n, 1, 256, 32, "bf16", g, 4)
    q = randn((len(lens), 2, 1, 32), torch.bfloat16, g)
    got, want = _calls(4, q, kp, vp, table.cuda(), lens.cuda(), None, shared_starts=dev(starts), shared_lens=dev(whole))
    assert torch.equal(got, want)


def test_many_rows():
    """Chunks of many rows: the kernels that walk, the same bits."""
    for nbits in (0, 8):
        g = gen(8)
        table, lens, starts, whole, n = _case([6], [1024], [500, 300], 16, g)
        kp, vp = _pools(n, 2, 16, 64, "bf16", g, nbits)
        q = randn((6, 8, 200, 64), torch.bfloat16, g)
        got, want = _calls(nbits, q, kp, vp, table.cuda(), lens.cuda(), "causal", shared_lens=whole[0])
        assert torch.equal(got, want)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_values(dt):
    g = gen(9)
    table, lens, starts, whole, n = _case([5], [512], [9, 100], 16, g)
    kp, vp = _pools(n, 2, 16, 64, dt, g, 0)
    q = randn((5, 4, 2, 64), DT[dt], g)
    got, _ = _calls(0, q, kp, vp, table.cuda(), lens.cuda(), "causal", shared_lens=whole[0])
    k, v = (p.cpu()[table.long()].transpose(1, 2).reshape(5, 2, -1, 64) for p in (kp, vp))
    want, absv, dot, bias = ref.attention(q.cpu(), k, v, 64 ** -0.5, lens, True)
    assert ((got.cpu().double() - want).abs() <= ref.attention_allowance(want, absv, dot, bias, DT[dt], 64, 3)).all()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 256])
def test_not_finite(dt, D):
    """Infinities and NaN behind sequences and in hidden keys take no part; seen ones come out in their dim."""
    bi, g = _bi(), gen(10)
    page, inf = 16, float("inf")
    table, lens, _, whole, n = _case([3], [512], [40, 60], page, g)
    kp, vp = _pools(n, 1, page, D, dt, g, 0)
    q = randn((3, 2, 4, D), DT[dt], g)
    call = lambda: bi.batch_invariant_shared_prefix_attention(q, kp, vp, table.cuda(), lens.cuda(), mask="causal", shared_lens=512)
    clean = call()
    for b in range(3):
        for p in range(int(lens[b]), table.shape[1] * page):
            kp[table[b, p // page], :, p % page] = float("nan")
            vp[table[b, p // page], :, p % page] = inf
    assert torch.equal(call(), clean)
    want = clean.clone()
    p = int(lens[1]) - 2                                  # seen by the last two of sequence 1's tokens
    vp[table[1, p // page], 0, p % page, 3] = -inf
    want[1, :, 2:, 3] = -inf
    p = int(lens[2]) - 1
    vp[table[2, p // page], 0, p % page, 5] = inf
    vp[table[2, 0], 0, 7, 5] = -inf                        # a shared key: every row sees it
    want[:, :, :, 5] = -inf
    want[2, :, 3, 5] = float("nan")
    got = call()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.float(), 0, 9, -9), torch.nan_to_num(want.float(), 0, 9, -9))
    q[0, 0, 1, 0] = float("nan")
    got = call()
    assert torch.isnan(got[0, 0, 1]).all() and not torch.isnan(got[0, 1]).any()


def test_graph_with_changing_groups():
    """One captured call serves other groups, lengths and tables; every replay has the eager bits."""
    bi, g = _bi(), gen(11)
    page, D, B = 16, 64, 8
    kp, vp = _pools(900, 2, page, D, "bf16", g, 0)
    qp = _pools(900, 2, page, D, "bf16", g, 8)
    q = randn((B, 8, 1, D), torch.bfloat16, g)
    cases = []
    for sizes, shared in (([8], [1024]), ([3, 5], [512, 768]), ([2, 2], [256, 1024])):
        table, lens, starts, whole, _ = _case(sizes, shared, [9, 100], page, g, tail=B - sum(sizes))
        starts, whole = (starts + [starts[-1]] * 2)[:3], (whole + [0])[:2]
        full = torch.zeros(B, 72, dtype=I32)
        full[:, :table.shape[1]] = table
        cases.append([full.cuda(), lens.cuda(), dev(starts), dev(whole)])
    held = [t.clone() for t in cases[0]]

    def step():
        more = dict(shared_starts=held[2], shared_lens=held[3])
        return (bi.batch_invariant_shared_prefix_attention(q, kp, vp, *held[:2], **more),
                bi.batch_invariant_quantized_paged_attention(q, *qp, *held[:2], **more),
                bi.batch_invariant_quantized_paged_attention(q, *qp, *held[:2]))

    step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for case in cases + cases[:2]:
        for h, c in zip(held, case):
            h.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, step()):
            assert torch.equal(x, y)
        want = bi.batch_invariant_paged_attention(q, kp, vp, *held[:2])
        assert torch.equal(out[0], want) and torch.equal(out[1], out[2])


# ---- whose pages are read --------------------------------------------------------------

def _rows_of(nbits, kp, vp, table):
    """K and V of every sequence through its own table row, [B, Hkv, L, D]."""
    if nbits:
        return _bi().read_quantized_cache(kp, vp, table)
    return [p[table.long()].transpose(1, 2).flatten(2, 3).contiguous() for p in (kp, vp)]


def _check_sources(dt, nbits, Hq, Hkv, D, T, page, sizes, shared, lens, mask, seed, lead=0, tail=0, layout="page"):
    """Sequences with pages all of their own: the shared splits' keys are those of the group's first
    sequence, the others' table entries of whole pages there are not read."""
    bi, g = _bi(), gen(seed)
    B = lead + sum(sizes) + tail
    L = max(max(lens), 1)
    cols = -(-L // page)
    lens = torch.tensor([lens[b % len(lens)] for b in range(B)], dtype=I32)
    n = B * cols
    table = torch.randperm(n, generator=g).reshape(B, cols).to(I32).cuda()
    kp, vp = _pools(n, Hkv, page, D, dt, g, nbits)
    if layout == "row":                                  # heads inside rows in memory
        kp, vp = (p.transpose(1, 2).contiguous().transpose(1, 2) for p in (kp, vp))
    q = randn((B, Hq, T, D), DT[dt], g, 2.0)
    k, v = _rows_of(nbits, kp, vp, table)
    starts = [lead]
    given = table.clone()
    for s, keys in zip(sizes, shared):
        lo = starts[-1]
        starts.append(lo + s)
        keys = min(keys, int(lens[lo])) // 256 * 256 if s > 1 else 0
        for b in range(lo + 1, lo + s):
            k[b, :, :keys], v[b, :, :keys] = k[lo, :, :keys], v[lo, :, :keys]
            given[b, :keys // page] = -1 if b % 2 else 1 << 30
    want = bi.batch_invariant_attention(q, k, v, kv_lens=lens.cuda(), mask=mask)
    call = bi.batch_invariant_quantized_paged_attention if nbits else bi.batch_invariant_shared_prefix_attention
    got = call(q, kp, vp, given, lens.cuda(), mask=mask, shared_starts=dev(starts), shared_lens=dev(shared))
    assert torch.equal(got, want), (got.float() - want.float()).abs().amax((1, 2, 3))
    return q, kp, vp, given, lens.cuda(), dev(starts), dev(shared), want


@pytest.mark.parametrize("nbits,dt", [(0, "bf16"), (8, "bf16"), (4, "f16"), (0, "f32"), (8, "f32")])
@pytest.mark.parametrize("page", [1, 16, 256, 512, 1024])
@pytest.mark.parametrize("T", [1, 4, 8, 100])
def test_pages_of_the_first_sequence(nbits, dt, page, T):
    """Any number of query tokens, pages that hold several splits, groups of one, none and many."""
    lens = [1030, 700, 40, 1100, 0, 900, 256, 511]
    _check_sources(dt, nbits, 8, 2, 64, T, page, [3, 1, 4], [600, 512, 1024], lens, "causal", 100 + T + page, lead=1, tail=1)
    _check_sources(dt, nbits, 3, 3, 64, T, page, [9], [768], lens, None, 200 + T + page)


@pytest.mark.parametrize("T", [4, 8, 16, 17])
@pytest.mark.parametrize("nbits", [0, 8])
def test_pages_of_the_first_sequence_whichever_kernel(T, nbits):
    """Token counts to either side of the rules on rows, many sequences."""
    _check_sources("bf16", nbits, 16, 4, 64, T, 16, [8, 8, 8, 8], [512, 600, 256, 300], [620, 700, 560, 800], "causal", T + nbits)


@pytest.mark.parametrize("layout", ["page", "row"])
@pytest.mark.parametrize("page", [512, 2048])
def test_splits_inside_pages(layout, page):
    """Many rows, a prefix that ends inside a page; heads inside rows in memory as well."""
    _check_sources("bf16", 0, 16, 2, 128, 200, page, [4], [1300], [1500, 2000, 1600, 1400], "causal", page, layout=layout)


@pytest.mark.parametrize("nbits,dt", [(0, "bf16"), (8, "f16"), (4, "bf16"), (0, "f32")])
@pytest.mark.parametrize("T", [1, 3, 8, 80])
def test_one_split_is_shared(nbits, dt, T):
    """A table of one split: the first sequence's pages too."""
    _check_sources(dt, nbits, 8, 2, 64, T, 16, [3, 4], [256, 300], [256, 100, 0, 256, 256, 255, 3], "causal", T)
    _check_sources(dt, nbits, 5, 1, 32, T, 64, [6], [256], [256, 100, 0, 256, 1], None, T + 1, tail=1)


@pytest.mark.parametrize("nbits", [0, 8])
def test_captured_many_rows(nbits):
    """A captured call of many rows with changing groups and tables: every replay has the eager bits."""
    bi = _bi()
    cases = [_check_sources("bf16", nbits, 8, 2, 64, 200, 16, sizes, shared, lens, "causal", 7) for sizes, shared, lens in (
        ([3, 3], [512, 700], [900, 800, 300]), ([6, 0], [256, 9], [900, 333]), ([1, 5], [900, 768], [900, 850, 870]))]
    q, kp, vp = cases[0][:3]
    call = bi.batch_invariant_quantized_paged_attention if nbits else bi.batch_invariant_shared_prefix_attention
    held = [t.clone() for t in cases[0][3:7]]
    step = lambda: call(q, kp, vp, held[0], held[1], mask="causal", shared_starts=held[2], shared_lens=held[3])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for case in cases + cases[:2]:
        for h, c in zip(held, case[3:7]):
            h.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step()) and torch.equal(out, case[7])


def test_empty_sequences_of_many_heads():
    """A sequence without keys, and more values in its rows than 31 bits count: zeros."""
    bi, g = _bi(), gen(12)
    kp, vp = _pools(4, 1, 16, 256, "bf16", g, 0)
    table = torch.zeros(1, 3, dtype=I32, device="cuda")
    for heads in (40, 5000, 1 << 23):
        q = torch.ones(1, heads, 1, 256, dtype=torch.bfloat16, device="cuda")
        torch.full_like(q, float("nan"))                  # (what the result's memory held before)
        out = bi.batch_invariant_shared_prefix_attention(q, kp, vp, table, dev([0]), shared_lens=300)
        assert not out.any()
        del q, out


def test_empty_and_short_sequences_of_many_heads():
    g = gen(13)
    table, lens, _, _, n = _case([7], [0], [0, 3, 40, 0, 31], 16, g)
    kp, vp = _pools(n, 1, 16, 64, "f16", g, 0)
    q = randn((7, 700, 1, 64), torch.float16, g)
    got, want = _calls(0, q, kp, vp, table.cuda(), lens.cuda(), None, shared_lens=256)
    assert torch.equal(got, want) and not want[0].any() and want[1].any()


def test_slices_behind_a_shared_prefix():
    """Codes of sequences so wide that they are read back a few at a time: every slice finds the first
    sequence's pages."""
    bi, g = _bi(), gen(22)
    D, page, cols = 256, 256, 1 << 10                    # 2^18 keys: 2 x 128 MiB a head and sequence
    kp, vp = (random_pool(40, 4, page, D, 8, 64, "bf16", g) for _ in range(2))
    table = torch.randint(0, 40, (5, cols), generator=g).to(I32)
    lens = dev([300, 900, 600, 1500, 500])
    q = randn((5, 16, 280, D), torch.bfloat16, g)
    given, whole = table.clone(), table.clone()
    given[2:5, :2] = -1                                   # group of sequences 1 to 4, 700 keys: two whole splits
    whole[2:5, :2] = table[1, :2]
    got = bi.batch_invariant_quantized_paged_attention(q, kp, vp, given.cuda(), lens, mask="causal", shared_starts=dev([1, 5]),
                                                       shared_lens=dev([700]))
    for b in range(5):
        want = bi.batch_invariant_quantized_paged_attention(q[b:b + 1], kp, vp, whole[b:b + 1, :6].cuda(), lens[b:b + 1], mask="causal")
        assert torch.equal(got[b:b + 1], want)


@pytest.mark.parametrize("B,groups,Hq,Hkv", [(300, 100, 4, 2), (600, 2, 64, 4), (64, 64, 8, 8)])
def test_one_split_of_many_sequences(B, groups, Hq, Hkv):
    """One split: plans that a launch of its own makes, items of several chunks, groups of one."""
    sizes = [B // groups] * groups
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 257, (B,), generator=g)
    lens[::max(sizes[0], 1)] = 256                        # first sequences hold the split, but for some
    lens[sizes[0] * (groups // 2)] = 255
    shared = [256] * groups
    _check_sources("bf16", 0, Hq, Hkv, 32, 1, 16, sizes, shared, lens.tolist(), "causal", B)
    _check_sources("f16", 8, Hq, Hkv, 64, 2, 64, sizes, shared, lens.tolist(), "causal", B + 1)
