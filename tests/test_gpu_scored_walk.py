"""Scored attention of many rows: the kernel whose workgroups walk a sequence's
splits (a batch of few rows takes a workgroup per split, so shapes here assert
which of the two runs)."""

import pytest
import torch

import paged_ref as ref
from helpers import DT, bits
from test_gpu_scored_attention import _call, _case, _check, _mods

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _walks(dt, B, Hq, Hkv, T, L, D, causal=True):
    """Whether a call without documents needs no workspace: the kernel that walks."""
    from mlx_batch_invariant_amd import _lib
    return _lib.load().bi_attn_scored_workspace_bytes(B, Hq, Hkv, T, L, D, int(causal), 0, _lib.DTYPE_CODE[DT[dt]]) == 0


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("page", [0, 4, 16, 64])
def test_documents_of_the_extreme_numbers(dt, page):
    """Document numbers -2^31 and 2^31 - 1 in one workgroup's rows, sorted and not,
    with lengths that end inside a split: only splits below the length are read."""
    B, Hq, Hkv, T, L, D = 8, 16, 8, 128, 300, 64
    assert _walks(dt, B, Hq, Hkv, T, L, D)
    q, k, v = _case(dt, B, Hq, Hkv, T, L, D, 51)
    lo, hi = -2**31, 2**31 - 1
    rows = [[lo] * 250 + [hi] * 50, [hi] * 250 + [lo] * 50, [lo, hi] * 150, [lo] * 100 + [0] * 100 + [hi] * 100,
            [hi] * 220 + [lo] * 80, [lo] * 300, [hi] * 300, list(range(150)) + [lo, hi] * 75]
    docs = torch.tensor(rows, dtype=I32)
    for lens in (None, [300, 260, 257, 256, 230, 129, 300, 1]):
        for causal in (True, False):
            _check(_call(q, k, v, lens, causal, page, doc_ids=docs), q, k, v, lens, causal, doc_ids=docs)


def _one(mods, b):
    """What changes sequence b's scores, for a call of it alone."""
    return {n: (x[b:b + 1] if n in ("doc_ids", "prefix_lens") else x) for n, x in mods.items()}


def _visible(lens, T, L, causal, doc_ids=None, prefix_lens=None, **_):
    """[B, T, L]: the keys that each query sees."""
    B, j = len(lens), torch.arange(L)
    see = torch.zeros(B, T, L, dtype=torch.bool)
    for b, n in enumerate(lens):
        for t in range(T):
            p = n - T + t
            if p < 0 and (causal or doc_ids is not None):
                continue
            s = j < n
            if causal:
                s &= (j <= p) | (j < (min(int(prefix_lens[b]), n) if prefix_lens is not None else 0))
            if doc_ids is not None:
                s &= doc_ids[b] == doc_ids[b, p]
            see[b, t] = s
    return see


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,page", [(64, 0), (128, 16), (64, 64), (96, 4), (256, 0), (192, 16)])
@pytest.mark.parametrize("which", ["c", "s", "d", "p", "csdp"])
def test_infinities_in_v_of_any_weight(dt, D, page, which):
    """Infinities and NaN in V, some of keys whose weight is far below the smallest
    number: a dim in which a query sees one is inf, -inf or NaN, every other element
    what it is with zeros there, and prompts of many rows, of few and decode steps
    agree."""
    B, Hq, Hkv, T, L = 8, 32 if dt == "f32" and D == 256 else 16, 8, 160, 700
    assert _walks(dt, B, Hq, Hkv, T, L, D) and not _walks(dt, 1, Hq, Hkv, T, L, D)
    q, k, v = _case(dt, B, Hq, Hkv, T, L, D, 52)
    lens = [700, 700, 513, 512, 640, 300, 200, 161]
    m = {}
    if "c" in which:
        m["softcap"] = 20.0
    if "s" in which:
        m["slopes"] = torch.full((Hq,), 0.5)            # exp(-0.5 * 300) is 0 in fp32
    if "d" in which:
        m["doc_ids"] = torch.arange(L).div(310, rounding_mode="floor").repeat(B, 1).to(I32)
        m["doc_ids"][1] = torch.arange(L) % 2
    if "p" in which:
        m["prefix_lens"] = torch.tensor([0, 600, 5, 512, 100, 290, 0, 161], dtype=I32)
    inf, nan = float("inf"), float("nan")
    put = [(0, 3, 1, inf), (0, 640, 2, -inf), (0, 100, 3, inf), (0, 690, 3, -inf), (0, 699, 4, nan), (1, 2, 0, inf),
           (1, 3, 0, -inf), (1, 520, 5, -inf), (2, 0, 7, -inf), (2, 511, 8, inf), (2, 512, 9, inf), (3, 255, 20, nan),
           (3, 300, 20, inf), (4, 600, 31, inf), (5, 299, 11, -inf), (5, 290, 11, inf), (7, 1, 30, inf)]
    clean = v.clone()
    kinds = torch.zeros(B, L, D, 3, dtype=torch.bool)   # inf, -inf, NaN
    for b, j, d, x in put:
        v[b, :, j, d], clean[b, :, j, d] = x, 0.0
        kinds[b, j, d, 2 if x != x else 0 if x > 0 else 1] = True
    see = _visible(lens, T, L, True, **m)
    has = torch.einsum("btl,bldk->btdk", see.float(), kinds.float()) > 0
    want = torch.where(has[..., 2] | (has[..., 0] & has[..., 1]), nan, torch.where(has[..., 0], inf, -inf))
    odd = has.any(-1)[:, None].expand(B, Hq, T, D).cuda()
    want = want[:, None].expand(B, Hq, T, D).to(DT[dt]).cuda()

    def check(got, base, odd, want):
        assert torch.equal(got[~odd], base[~odd]) and base.isfinite().all()
        a, b = got[odd], want[odd]
        assert ((a == b) | (a.isnan() & b.isnan())).all()

    check(_call(q, k, v, lens, True, page, **m), _call(q, k, clean, lens, True, page, **m), odd, want)
    for b in (0, 1, 2, 5, 7):                            # a workgroup per split
        check(_call(q[b:b + 1], k[b:b + 1], v[b:b + 1], lens[b:b + 1], True, page, **_one(m, b)),
              _call(q[b:b + 1], k[b:b + 1], clean[b:b + 1], lens[b:b + 1], True, page, **_one(m, b)), odd[b:b + 1],
              want[b:b + 1])
    # (a decode step sees every key of its sequence, as the last row of a prompt does)
    check(_call(q[:, :, -1:], k, v, lens, True, page, **m), _call(q[:, :, -1:], k, clean, lens, True, page, **m),
          odd[:, :, -1:], want[:, :, -1:])


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_infinities_in_v_beside_scores_that_are_not_finite(dt):
    """A query whose only visible score is -inf gets zeros, one with a NaN score NaN,
    whatever V holds, by every kernel; caches of one split and of several."""
    Hq, Hkv, T, D = 16, 8, 128, 64
    for L in (128, 600):
        B = 8
        assert _walks(dt, B, Hq, Hkv, T, L, D) and (L < 256 or not _walks(dt, 1, Hq, Hkv, T, L, D))
        q, k, v = _case(dt, B, Hq, Hkv, T, L, D, 53)
        q[..., 0] = 1.0
        lens = [128] * B
        docs = torch.zeros(B, L, dtype=I32)
        docs[:, 5] = 1                                   # a document of one key
        k[:, :, 5, 0], v[:, :, 5, 9], v[:, :, 5, 10] = float("-inf"), float("inf"), float("nan")
        docs[:, 50:] = 2
        k[:, :, 60, 0], v[:, :, 60, 3] = float("nan"), float("inf")
        m = dict(doc_ids=docs, slopes=torch.zeros(Hq))
        got = _call(q, k, v, lens, True, **m)
        assert not got[:, :, 5].any() and got[:, :, 60:].isnan().all()
        keep = torch.arange(T, device="cuda")
        assert got[:, :, (keep < 60) & (keep != 5)].isfinite().all()
        for b in (0, 3):
            one = _call(q[b:b + 1], k[b:b + 1], v[b:b + 1], lens[b:b + 1], True, **_one(m, b))
            assert ((one == got[b:b + 1]) | (one.isnan() & got[b:b + 1].isnan())).all()
        for n in (6, 59, 60, 61, 128):
            one = _call(q[:, :, n - 1:n], k, v, [n] * B, True, **m)
            a = got[:, :, n - 1:n]
            assert ((one == a) | (one.isnan() & a.isnan())).all(), n


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("T", [16, 1])
def test_short_sequences_in_a_wide_table(dt, T):
    """Tables that hold far more than the sequences, and whose entries behind them
    point anywhere: the bits of a narrow table."""
    import mlx_batch_invariant_amd as bi
    B, Hq, Hkv, D, page, used, wide = 4, 8, 2, 64, 16, 40, 4096
    q, k, v = _case(dt, B * used, Hq, Hkv, page, page, D, 54)
    q = q[:B, :, :T].contiguous()
    table = torch.full((B, wide), -7, dtype=I32)
    table[:, 100:] = 10**9
    table[:, :used] = torch.randperm(B * used, generator=torch.Generator().manual_seed(1)).view(B, used)
    lens = torch.tensor([300, 640, 17, 0], dtype=I32, device="cuda")
    m = dict(softcap=20.0, slopes=torch.full((Hq,), 0.01, device="cuda"))
    table = table.cuda()
    docs = (torch.arange(wide * page, device="cuda") // 200).to(I32).repeat(B, 1)
    for mods in (m, dict(m, doc_ids=docs), dict(prefix_lens=torch.tensor([100, 640, 5, 9], dtype=I32))):
        f = lambda n: bi.batch_invariant_paged_attention(q, k, v, table[:, :n], lens, mask="causal", **mods)
        assert torch.equal(f(wide), f(used))
        assert not f(wide)[3].any()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("page", [0, 4, 16, 64])
@pytest.mark.parametrize("which", ["d", "c", "s", "csdp"])
def test_every_head_dim_walked(dt, D, page, which):
    """Every head dim and type over two splits, the last one partial, against the
    formula and against the sequences alone, which take a workgroup per split."""
    B, Hq, Hkv, T, L = 8, 32 if dt == "f32" and D == 256 else 16, 8, 96, 400
    assert _walks(dt, B, Hq, Hkv, T, L, D) and not _walks(dt, 1, Hq, Hkv, T, L, D)
    q, k, v = _case(dt, B, Hq, Hkv, T, L, D, D + page)
    m = _mods(which, B, Hq, L, D)
    lens = [400, 257, 399, 256, 300, 97, 50, 0]
    got = _call(q, k, v, lens, True, page, token_major=page == 16, **m)
    for b in (0, 1, 6):
        s = slice(b, b + 1)
        _check(got[s], q[s], k[s], v[s], lens[s], True, **_one(m, b))
    for b in range(B):
        s = slice(b, b + 1)
        assert bits(_call(q[s], k[s], v[s], lens[s], True, page, **_one(m, b))) == bits(got[s]), b


@pytest.mark.parametrize("D", [64, 96, 256])
def test_wider_cap_and_no_mask_walked(D):
    """Caps above 128 (the closer tanh, in the kernel with both score terms) and no
    causal mask, with a bias and without."""
    B, Hq, Hkv, T, L = 8, 16, 8, 96, 400
    for dt in ("bf16", "f16"):
        assert _walks(dt, B, Hq, Hkv, T, L, D, causal=False)
        q, k, v = _case(dt, B, Hq, Hkv, T, L, D, 55)
        lens = [400, 257, 399, 256, 300, 97, 50, 0]
        for m in (dict(softcap=200.0), dict(softcap=200.0, slopes=torch.linspace(0.0, 0.1, Hq))):
            for causal in (True, False):
                got = _call(q, k, v, lens, causal, 0, **m)
                for b in (1, 5):
                    s = slice(b, b + 1)
                    # past a cap of 128 the error is 12 2^-24 of the score, not of the cap
                    c = [x[s].cpu() for x in (q, k, v)]
                    want, absv, dot, bias = ref.attention(*c, D ** -0.5, lens[s], causal, **m)
                    allow = ref.attention_allowance(want, absv, 13 * dot, bias, DT[dt], D, 2, 0.0)
                    assert ((got[s].double().cpu() - want).abs() <= allow).all()


@pytest.mark.parametrize("page", [0, 16, 4])
def test_documents_that_begin_anywhere_walked_fp32(page):
    """fp32 rows enough for the kernel that walks: documents that begin in each 64 keys
    of a split, some shorter than 64."""
    L, D, at = 700, 64, [0, 70, 130, 200, 256, 330, 450, 465, 480, 515, 640]
    assert _walks("f32", 4, 8, 1, L, L, D)
    q, k, v = _case("f32", 4, 8, 1, L, L, D, 56)
    doc = torch.zeros(4, L, dtype=I32)
    for i, b in enumerate(at):
        doc[0::2, b:], doc[1::2, b:] = i, len(at) - i
    lens = [L, 690, 300, 1]
    got = _call(q, k, v, lens, True, page, doc_ids=doc)
    for b in range(2):
        s = slice(b, b + 1)
        _check(got[s], q[s], k[s], v[s], lens[s], True, doc_ids=doc[s])
    for b in range(4):
        s = slice(b, b + 1)
        assert bits(_call(q[s], k[s], v[s], lens[s], True, page, doc_ids=doc[s])) == bits(got[s])


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("page", [0, 4, 16, 64])
def test_hidden_infinities_and_nan_walked(dt, page):
    """Rows of K and V that a query does not see hold infinities and NaN, in the kernel
    that walks: what it gets is what it got with zeros there."""
    B, Hq, Hkv, T, L, D = 8, 16, 8, 150, 420, 64
    assert _walks(dt, B, Hq, Hkv, T, L, D)
    q, k, v = _case(dt, B, Hq, Hkv, T, L, D, 57)
    docs = torch.arange(L).div(130, rounding_mode="floor").repeat(B, 1).to(I32)
    docs[1::2, 200:] = torch.arange(220) % 3
    lens = [L, L - 30] * 4
    bad = [(0, 3, "nan"), (0, 135, "inf"), (0, 300, "-inf"), (0, 419, "nan"), (1, 10, "inf"), (1, 310, "nan"),
           (3, 395, "nan"), (3, 389, "-inf"), (5, 400, "nan"), (5, 419, "inf")]
    clean, dirty = [k.clone(), v.clone()], [k.clone(), v.clone()]
    for b, j, x in bad:
        for i in range(2):
            clean[i][b, :, j, 5:40], dirty[i][b, :, j, 5:40] = 0.0, float(x)
    for m in (dict(doc_ids=docs), dict(softcap=4.0), dict(slopes=torch.full((Hq,), 0.1), doc_ids=docs)):
        see = _visible(lens, T, L, True, **m)
        sees = torch.zeros(B, T, dtype=torch.bool)
        for b, j, _ in bad:
            sees[b] |= see[b, :, j]
        got, base = _call(q, *dirty, lens, True, page, **m), _call(q, *clean, lens, True, page, **m)
        blind = ~sees[:, None, :, None].expand(got.shape).cuda()
        assert torch.equal(got[blind], base[blind]) and base.isfinite().all()
        assert got[~blind].isnan().any()
