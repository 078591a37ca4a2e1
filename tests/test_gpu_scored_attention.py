"""Attention with capped scores, a distance bias, a document mask and a prefix
mask against the 64-bit formula, over types, head sizes, caches and lengths; its
invariances; hidden infinities and NaN; refusals."""

import pytest
import torch

import paged_ref as ref
from helpers import DT, bits, gen, randn

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _bi():
    import mlx_batch_invariant_amd as bi
    return bi


def _pages(k, page, g, token_major=False):
    """The contiguous cache k [B, Hkv, L, D] as a pool of pages and its table."""
    B, H, L, D = k.shape
    per = -(-L // page)
    table = torch.randperm(B * per + 3, generator=g)[:B * per].reshape(B, per).to(I32)
    pool = torch.full((B * per + 3, page, H, D), 7.0, dtype=k.dtype, device="cuda")
    padded = torch.nn.functional.pad(k, (0, 0, 0, per * page - L))
    pool[table.long().flatten()] = padded.reshape(B, H, per, page, D).permute(0, 2, 3, 1, 4).reshape(-1, page, H, D)
    return (pool if token_major else pool.transpose(1, 2).contiguous().transpose(1, 2)).transpose(1, 2), table.cuda()


def _call(q, k, v, lens, causal, page=0, seed=0, token_major=False, **mods):
    bi = _bi()
    kw = dict(mask="causal" if causal else None, scale=q.shape[3] ** -0.5)
    dev = {n: m.cuda() if isinstance(m, torch.Tensor) else m for n, m in mods.items()}
    if lens is not None:
        lens = torch.tensor(lens, dtype=I32, device="cuda")
    if not page:
        return bi.batch_invariant_attention(q, k, v, kv_lens=lens, **kw, **dev)
    kp, table = _pages(k, page, gen(seed), token_major)
    vp, _ = _pages(v, page, gen(seed), token_major)
    if dev.get("doc_ids") is not None:
        d = dev["doc_ids"]
        dev["doc_ids"] = torch.nn.functional.pad(d, (0, max(0, table.shape[1] * page - d.shape[1])), value=-9)
    if lens is None:
        lens = torch.full((q.shape[0],), k.shape[2], dtype=I32, device="cuda")
    return bi.batch_invariant_paged_attention(q, kp, vp, table, lens, **kw, **dev)


def _check(got, q, k, v, lens, causal, softcap=None, slopes=None, doc_ids=None, prefix_lens=None):
    c = [t.cpu() for t in (q, k, v)]
    want, absv, dot, bias = ref.attention(*c, q.shape[3] ** -0.5, lens, causal, softcap, slopes, doc_ids, prefix_lens)
    allow = ref.attention_allowance(want, absv, dot, bias, q.dtype, q.shape[3], -(-k.shape[2] // 256), softcap)
    err = (got.double().cpu() - want).abs()
    assert (err <= allow).all(), float((err / allow.clamp(min=1e-300)).max())


def _case(dt, B, Hq, Hkv, T, L, D, seed, qscale=3.0):
    g = gen(seed)
    return randn((B, Hq, T, D), DT[dt], g, qscale), randn((B, Hkv, L, D), DT[dt], g), randn((B, Hkv, L, D), DT[dt], g)


def _mods(which, B, Hq, L, seed):
    g = gen(seed + 1000)
    m = {}
    if "c" in which:
        m["softcap"] = 5.0
    if "s" in which:
        m["slopes"] = 2.0 ** (-8.0 * torch.arange(1, Hq + 1) / Hq)
    if "d" in which:
        m["doc_ids"] = (torch.rand((B, L), generator=g) < 0.02).cumsum(1).to(I32)
    if "p" in which:
        m["prefix_lens"] = torch.randint(0, L, (B,), generator=g, dtype=I32)
    return m


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("which", ["c", "s", "d", "p", "csdp"])
@pytest.mark.parametrize("B,Hq,Hkv,T,L,D,page,causal", [
    (2, 4, 2, 37, 600, 64, 0, True), (1, 6, 1, 70, 70, 128, 0, True), (2, 4, 4, 19, 530, 64, 16, True),
    (2, 2, 1, 33, 300, 32, 4, True), (1, 3, 3, 21, 520, 96, 64, True), (2, 2, 2, 5, 3, 64, 0, False)])
def test_prefill(dt, which, B, Hq, Hkv, T, L, D, page, causal):
    if not causal:
        which = which.replace("p", "")
        if not which:
            pytest.skip("a prefix goes with the causal mask")
    for lens in (None, [L // 2, max(1, T // 2)][:B]):
        q, k, v = _case(dt, B, Hq, Hkv, T, L, D, B + T + L)
        m = _mods(which, B, Hq, L, L)
        _check(_call(q, k, v, lens, causal, page, **m), q, k, v, lens, causal, **m)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("which", ["c", "s", "d", "csdp"])
@pytest.mark.parametrize("B,Hq,Hkv,L,D,page", [(3, 8, 2, 1000, 128, 0), (2, 16, 1, 257, 64, 16), (3, 5, 5, 520, 96, 8),
                                               (2, 6, 3, 300, 256, 64), (1, 4, 2, 1, 32, 0)])
def test_decode(dt, which, B, Hq, Hkv, L, D, page):
    for lens in (None, [0, 256, L][:B] if B > 1 else None):
        q, k, v = _case(dt, B, Hq, Hkv, 1, L, D, B + L + D)
        m = _mods(which, B, Hq, L, L)
        _check(_call(q, k, v, lens, True, page, **m), q, k, v, lens, True, **m)


@pytest.mark.parametrize("dt,D", [("bf16", 128), ("bf16", 192), ("f16", 256), ("f16", 64), ("f32", 64), ("f32", 192),
                                  ("f32", 256), ("bf16", 32), ("f32", 128)])
@pytest.mark.parametrize("page", [0, 4, 32, 64])
def test_every_head_dim(dt, D, page):
    q, k, v = _case(dt, 1, 4, 2, 20, 300, D, D)
    for which in ("csdp", "d", "c", "s"):
        m = _mods(which, 1, 4, 300, D)
        _check(_call(q, k, v, None, True, page, **m), q, k, v, None, True, **m)
        last = _call(q[:, :, -1:], k, v, None, True, page, **m)
        assert bits(last) == bits(_call(q, k, v, None, True, page, **m)[:, :, -1:])


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("page", [0, 8, 16, 128])
def test_unchanged_scores_are_the_plain_bits(dt, page):
    """Slopes of 0, one document, a prefix of 0: the plain call, bit for bit, for
    prompts, a chunk of a longer one and decode."""
    for T, L, D in ((90, 90, 64), (40, 700, 128), (1, 600, 64)):
        q, k, v = _case(dt, 2, 6, 2, T, L, D, T)
        lens = [L, L - 20]
        plain = _call(q, k, v, lens, True, page)
        one = torch.full((2, L), 5, dtype=I32)
        for m in (dict(slopes=torch.zeros(6)), dict(doc_ids=one), dict(prefix_lens=torch.zeros(2, dtype=I32)),
                  dict(slopes=torch.zeros(6), doc_ids=one, prefix_lens=torch.tensor([-5, 0], dtype=I32))):
            assert bits(_call(q, k, v, lens, True, page, **m)) == bits(plain)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("which", ["c", "sd", "csdp"])
def test_invariances(dt, which):
    """A sequence alone and in a batch; chunked and whole prompts; the last token
    of a prompt and its decode step; contiguous and paged caches: one set of bits."""
    B, Hq, Hkv, T, L, D = 3, 6, 2, 300, 560, 64
    q, k, v = _case(dt, B, Hq, Hkv, T, L, D, 77)
    m = _mods(which, B, Hq, L, 77)
    lens = [L, 400, 311]
    whole = _call(q, k, v, lens, True, **m)
    for page in (4, 16, 64):
        assert bits(_call(q, k, v, lens, True, page, **m)) == bits(whole)
        assert bits(_call(q, k, v, lens, True, page, token_major=True, **m)) == bits(whole)
    for b in range(B):
        one = {n: (x[b:b + 1, :lens[b]] if n == "doc_ids" else x[b:b + 1] if n == "prefix_lens" else x)
               for n, x in m.items()}
        cut = [x[b:b + 1, :, :lens[b]] for x in (k, v)]
        assert bits(_call(q[b:b + 1], *cut, None, True, **one)) == bits(whole[b:b + 1])
        if "p" in which:
            continue                                    # (an earlier chunk sees no later prefix key)
        n = lens[b] - 100                               # the first T - 100 tokens as a chunk of their own
        first = [x[:, :, :n] for x in cut]
        early = {k2: (x[:, :n] if k2 == "doc_ids" else x) for k2, x in one.items()}
        assert bits(_call(q[b:b + 1, :, :T - 100], *first, None, True, **early)) == bits(whole[b:b + 1, :, :T - 100])
    assert bits(_call(q[:, :, -1:], k, v, lens, True, **m)) == bits(whole[:, :, -1:])


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("page", [0, 4, 16, 64])
def test_hidden_infinities_and_nan(dt, page):
    """Rows of K and V that a query does not see hold infinities and NaN: what it
    gets is what it got with zeros there. Queries that see one get it."""
    B, Hq, Hkv, T, L, D = 2, 4, 2, 150, 420, 64
    q, k, v = _case(dt, B, Hq, Hkv, T, L, D, 5)
    docs = torch.tensor([[j // 130 for j in range(L)], [7] * 200 + [j % 3 for j in range(220)]], dtype=I32)
    lens = [L, L - 30]
    bad = [(0, 3, "nan"), (0, 135, "inf"), (0, 300, "-inf"), (0, 419, "nan"), (1, 10, "inf"), (1, 310, "nan"),
           (1, 395, "nan"), (1, 389, "-inf")]
    for mods in (dict(doc_ids=docs), dict(softcap=4.0), dict(slopes=torch.full((Hq,), 0.1), doc_ids=docs)):
        clean, dirty = [k.clone(), v.clone()], [k.clone(), v.clone()]
        for b, j, x in bad:
            for i in range(2):
                clean[i][b, :, j, 5:40] = 0.0
                dirty[i][b, :, j, 5:40] = float(x)
        for TT in (T, 1):
            qq = q[:, :, T - TT:]
            got = _call(qq, *dirty, lens, True, page, **mods)
            base = _call(qq, *clean, lens, True, page, **mods)
            sees = torch.zeros(B, TT, dtype=torch.bool)
            for b in range(B):
                for t in range(TT):
                    p = lens[b] - TT + t
                    for bb, j, _ in bad:
                        if bb == b and j <= p and ("doc_ids" not in mods or docs[b, j] == docs[b, p]):
                            sees[b, t] = True
            sees = sees.cuda()
            # (decode and prefill, masked rows: the bits of the clean cache)
            blind = ~sees[:, None, :, None].expand(got.shape)
            assert torch.equal(got[blind], base[blind]) and got[blind].isfinite().all()
            assert got[~blind].isnan().any(-1).all() if (~blind).any() else True


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_visible_infinities_in_v_only(dt):
    """An infinity in V that a query sees comes out as it is, others' rows as with
    a finite value there; the dims beside it stay finite."""
    q, k, v = _case(dt, 1, 2, 1, 40, 300, 64, 6, 0.5)
    docs = torch.tensor([[0] * 280 + [1] * 20], dtype=I32)
    v[0, 0, 100, 3], v[0, 0, 275, 4], v[0, 0, 276, 4] = float("inf"), float("-inf"), float("inf")
    got = _call(q, k, v, None, True, doc_ids=docs)[0, :, :, :].cpu()
    first = got[:, :16]                                 # positions 260 .. 275
    assert (first[:, :, 3] == float("inf")).all()
    assert got[:, 15, 4].eq(float("-inf")).all() and got[:, 16:20, 4].isnan().all()
    assert got[:, 20:].isfinite().all()
    assert got[:, :15, 4].isfinite().all() and got[:, :20, [0, 1, 2, 5, 6]].isfinite().all()


def test_rows_that_see_nothing():
    """Queries in front of a padded prompt, sequences of length 0, prefixes and
    documents there: zeros."""
    q, k, v = _case("bf16", 3, 4, 2, 80, 100, 64, 9)
    lens = [0, 30, 100]
    for m in (dict(softcap=3.0), dict(doc_ids=torch.zeros(3, 100, dtype=I32)), dict(slopes=torch.ones(4)),
              dict(prefix_lens=torch.tensor([50, 50, 50], dtype=I32))):
        out = _call(q, k, v, lens, True, **m)
        assert not out[0].any() and not out[1, :, :50].any() and out[1, :, 50:].any() and out.isfinite().all()
        assert not _call(q[:, :, -1:], k, v, lens, True, **m)[0].any()
        _check(out, q, k, v, lens, True, **m)
    out = _call(q, k[:, :, :20], v[:, :, :20], None, False, doc_ids=torch.zeros(3, 20, dtype=I32))
    assert not out[:, :, :60].any() and out[:, :, 60:].any()


def test_many_documents_over_a_long_row():
    """More than 64 splits, unsorted document numbers (equal ones far apart), as
    well as sorted ones whose splits are skipped."""
    L, T, D = 20000, 64, 64
    q, k, v = _case("bf16", 1, 2, 1, T, L, D, 11)
    for docs in (torch.arange(L)[None] // 333 % 9 - 4, torch.arange(L)[None] // 150, torch.arange(L)[None] * 0 - 3):
        docs = docs.to(I32)
        docs[0, 5000:5003] = docs[0, -1]
        _check(_call(q, k, v, None, True, doc_ids=docs), q, k, v, None, True, doc_ids=docs)
        last = _call(q[:, :, -1:], k, v, None, True, doc_ids=docs)
        _check(last, q[:, :, -1:], k, v, None, True, doc_ids=docs)


def test_argument_forms_and_streams():
    """int64 document numbers, a slice of a wider table of them, slopes as a list;
    another stream; a captured call replayed with other contents."""
    q, k, v = _case("f16", 2, 4, 2, 30, 260, 64, 12)
    m = _mods("csdp", 2, 4, 260, 12)
    want = _call(q, k, v, None, True, **m)
    wide = torch.full((2, 300), -1, dtype=I32)
    wide[:, 7:267] = m["doc_ids"]
    other = dict(softcap=5, slopes=m["slopes"].tolist(), doc_ids=wide.cuda()[:, 7:267],
                 prefix_lens=m["prefix_lens"].tolist())
    assert bits(_call(q, k, v, None, True, **other)) == bits(want)
    other["doc_ids"] = m["doc_ids"].long()
    assert bits(_call(q, k, v, None, True, **other)) == bits(want)
    bi = _bi()
    dev = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in m.items()}
    for T in (30, 1):
        qq = q[:, :, :T].contiguous()
        f = lambda: bi.batch_invariant_attention(qq, k, v, mask="causal", **dev)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a = f()
        torch.cuda.current_stream().wait_stream(side)
        assert bits(a) == bits(f())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        for i in range(3):
            qq.copy_(randn(qq.shape, qq.dtype, gen(60 + i)))
            dev["doc_ids"].copy_(_mods("d", 2, 4, 260, 70 + i)["doc_ids"])
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert bits(out) == bits(f())
        del graph


def test_operators_of_the_dispatcher():
    q, k, v = _case("bf16", 2, 4, 2, 10, 64, 64, 13)
    m = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in _mods("csdp", 2, 4, 64, 13).items()}
    want = _bi().batch_invariant_attention(q, k, v, scale=0.125, mask="causal", **m)
    a = (m["softcap"], m["slopes"], m["doc_ids"], m["prefix_lens"])
    assert bits(torch.ops.mlx_bi.scored_attention(q, k, v, 0.125, True, None, *a)) == bits(want)
    table = torch.arange(8, dtype=I32, device="cuda").reshape(2, 4)
    kp, vp = (x.reshape(2, 2, 4, 16, 64).transpose(1, 2).reshape(8, 2, 16, 64) for x in (k, v))
    assert bits(torch.ops.mlx_bi.scored_paged_attention(q, kp, vp, table, None, 0.125, True, *a)) == bits(want)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("page,D", [(0, 64), (16, 128), (64, 64), (4, 32)])
@pytest.mark.parametrize("which", ["c", "s", "d", "p", "csdp"])
def test_many_rows_are_the_bits_of_few(dt, page, D, which):
    """A batch large enough for the workgroups that walk the splits against its
    sequences alone, which take a workgroup per split; hidden infinities in both."""
    B, Hq, Hkv, T, L = 6, 8, 4, 200, 600
    q, k, v = _case(dt, B, Hq, Hkv, T, L, D, 21)
    m = _mods(which, B, Hq, L, 21)
    lens = [L, 100, 257, 513, 31, 599]
    for b, n in enumerate(lens):
        k[b, :, n:], v[b, :, n:] = float("inf"), float("nan")
    if "d" in which:
        for b in range(B):                              # another document's rows, and the last token's own
            other = (m["doc_ids"][b] != m["doc_ids"][b, lens[b] - 1]).nonzero()[:, 0]
            v[b, :, other[other < 20].cuda(), 3] = float("nan")
    from mlx_batch_invariant_amd import _lib
    size = lambda n: _lib.load().bi_attn_scored_workspace_bytes(n, Hq, Hkv, T, L, D, 1, 0, _lib.DTYPE_CODE[DT[dt]])
    assert size(B) == 0 < size(1)
    got = _call(q, k, v, lens, True, page, **m)
    for b in range(B):
        one = {n: (x[b:b + 1] if n in ("doc_ids", "prefix_lens") else x) for n, x in m.items()}
        alone = _call(q[b:b + 1], k[b:b + 1], v[b:b + 1], lens[b:b + 1], True, page, **one)
        same = (alone == got[b:b + 1]) | (alone.isnan() & got[b:b + 1].isnan())
        assert same.all(), b
    clean = [x.clone() for x in (k, v)]
    for b, n in enumerate(lens):
        clean[0][b, :, n:], clean[1][b, :, n:] = 0.0, 0.0
    if which != "d" and "d" not in which:
        assert bits(_call(q, *clean, lens, True, page, **m)) == bits(got)
        _check(got[1:2], q[1:2], clean[0][1:2], clean[1][1:2], lens[1:2], True,
               **{n: (x[1:2] if n == "prefix_lens" else x) for n, x in m.items()})


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D,page", [(64, 0), (128, 16), (256, 0), (96, 4)])
def test_caches_of_one_split(dt, D, page):
    """Caches of at most 256 keys need no merge: the bits of the same lengths in a
    longer cache; empty sequences and negative zeros as there."""
    B, Hq, Hkv = 5, 8, 2
    lens = [256, 0, 1, 77, 255]
    for T in (1, 9, 60):
        q, k, v = _case(dt, B, Hq, Hkv, T, 256, D, 31)
        v[:, :, :, 0] = -0.0
        longer = [torch.nn.functional.pad(x, (0, 0, 0, 300), value=3.0) for x in (k, v)]
        for which in ("c", "sd", "csdp"):
            m = _mods(which, B, Hq, 256, 31)
            n = {a: torch.nn.functional.pad(x, (0, 300), value=-1) if a == "doc_ids" else x for a, x in m.items()}
            got = _call(q, k, v, lens, True, page, **m)
            assert bits(got) == bits(_call(q, *longer, lens, True, page, **n))
            assert not got[1].any()
            _check(got, q, k, v, lens, True, **m)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("cap", [1e-3, 128.0, 1000.0, 1e6, 1e30])
def test_caps_small_and_large(dt, cap):
    """Caps far below the scores and far above them (then the plain scores)."""
    q, k, v = _case(dt, 2, 4, 2, 24, 300, 64, 41)
    for T in (24, 1):
        qq = q[:, :, :T].contiguous()
        got = _call(qq, k, v, None, True, softcap=cap)
        c = [t.cpu() for t in (qq, k, v)]
        want, absv, dot, bias = ref.attention(*c, 0.125, None, True, cap)
        # past a cap of 128 (or in fp32) the error is 12 2^-24 of the score, not of the cap
        close = cap > 128 or dt == "f32"
        allow = ref.attention_allowance(want, absv, dot + (12 * dot if close else 0), bias, DT[dt], 64, 2,
                                        0.0 if close else cap)
        err = (got.double().cpu() - want).abs()
        assert (err <= allow).all(), float((err / allow).max())


def test_bias_of_any_sign_and_masks_at_their_ends():
    q, k, v = _case("bf16", 2, 4, 2, 40, 290, 64, 42)
    for m in (dict(slopes=torch.tensor([-0.01, 0.0, 3.0, 1e-6])),
              dict(prefix_lens=torch.tensor([1000, -7], dtype=I32)),
              dict(doc_ids=torch.tensor([[-2**31] * 250 + [2**31 - 1] * 40, list(range(290))], dtype=I32))):
        for T in (40, 1):
            qq = q[:, :, :T].contiguous()
            _check(_call(qq, k, v, None, True, **m), qq, k, v, None, True, **m)


def test_bias_over_a_long_cache():
    """Distances of hundreds of thousands of keys (exact in fp32 up to 2^24)."""
    L = 300_000
    q, k, v = _case("bf16", 1, 2, 1, 3, L, 32, 43)
    m = dict(slopes=torch.tensor([1e-5, 0.0]))
    for T in (3, 1):
        qq = q[:, :, :T].contiguous()
        _check(_call(qq, k, v, None, True, **m), qq, k, v, None, True, **m)


def test_caches_past_32_bits():
    """Pages and sequences that start behind 2^32 elements of their storage."""
    Hkv, D, page, L = 2, 64, 16, 300
    n = (1 << 21) + 64                                   # 2048 elements a page
    q, k, v = _case("bf16", 2, 4, Hkv, 40, L, D, 44)
    per = -(-L // page)
    pools, flats = [], []
    for x in (k, v):
        pool = torch.empty((n, Hkv, page, D), dtype=x.dtype, device="cuda")
        pad = torch.nn.functional.pad(x, (0, 0, 0, per * page - L))
        # the last pages in reverse order, then (contiguous) rows 2^32 elements apart
        at = torch.arange(n - 1, n - 1 - 2 * per, -1, device="cuda")
        pool[at] = pad.reshape(2, Hkv, per, page, D).transpose(1, 2).reshape(-1, Hkv, page, D)
        pools.append(pool)
        flat = torch.as_strided(pool, (2, Hkv, L, D), (1 << 32, L * D, D, 1))
        flats.append(flat)
    table = torch.arange(n - 1, n - 1 - 2 * per, -1, dtype=I32, device="cuda").view(2, per)
    lens = [L, 211]
    m = dict(softcap=30.0, slopes=torch.tensor([0.01, 0.1, 0.0, 0.5]).cuda(),
             doc_ids=(torch.arange(L) // 90).repeat(2, 1).cuda())
    mp = dict(m, doc_ids=torch.nn.functional.pad(m["doc_ids"], (0, per * page - L)))
    want = {}
    for T in (40, 1):
        qq = q[:, :, :T].contiguous()
        want[T] = bits(_call(qq, k, v, lens, True, **m))
        got = _bi().batch_invariant_paged_attention(qq, *pools, table, torch.tensor(lens, dtype=I32, device="cuda"),
                                                    scale=D ** -0.5, mask="causal", **mp)
        assert bits(got) == want[T]
    for flat, x in zip(flats, (k, v)):
        flat.copy_(x)
    for T in (40, 1):
        assert bits(_call(q[:, :, :T].contiguous(), *flats, lens, True, **m)) == want[T]
    many = q.repeat(1, 4, 8, 1)[:, :, :300].contiguous()  # rows enough for the kernel that walks the splits
    m["slopes"] = m["slopes"].repeat(4)
    assert bits(_call(many, *flats, lens, True, **m)) == bits(_call(many, k, v, lens, True, **m))


def test_calls_at_once_on_two_streams():
    """Every call has a workspace of its own."""
    q, k, v = _case("bf16", 2, 8, 2, 48, 1500, 64, 45)
    forms = [(q[:, :, :T].contiguous(), dict(softcap=20.0 + T, slopes=torch.full((8,), 0.01 * T))) for T in (1, 5, 48)]
    want = [bits(_call(x, k, v, None, True, **m)) for x, m in forms]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got += [_call(x, k, v, None, True, **m) for x, m in forms]
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert bits(g) == want[i % 3]


@pytest.mark.parametrize("page", [0, 16, 4])
@pytest.mark.parametrize("dt,D", [("bf16", 128), ("f16", 64), ("f32", 64), ("bf16", 256)])
def test_documents_that_begin_anywhere_in_a_split(dt, D, page):
    """Rows enough for the kernel that walks the splits; documents that begin in each
    64 keys of a split, some shorter than 64, against the formula and one call each."""
    L, at = 700, [0, 70, 130, 200, 256, 330, 450, 465, 480, 515, 640]
    q, k, v = _case(dt, 2, 8, 1, L, L, D, 46)
    doc = torch.zeros(2, L, dtype=I32)
    for i, b in enumerate(at):
        doc[0, b:] = i
        doc[1, b:] = len(at) - i                         # descending numbers
    lens = [L, 690]
    got = _call(q, k, v, lens, True, page, doc_ids=doc)
    _check(got, q, k, v, lens, True, doc_ids=doc)
    ends = at[1:] + [L]
    for b, e in zip(at, ends):
        # (a call of the document alone counts its splits from its own start, so only
        # those that begin a split have the same bits)
        if b % 256 == 0:
            alone = _call(q[:1, :, b:e].contiguous(), k[:1, :, b:e].contiguous(), v[:1, :, b:e].contiguous(), None, True)
            assert bits(alone) == bits(got[:1, :, b:e])
