"""Scored attention of many rows: the kernel whose workgroups walk a sequence's
splits (a batch of few rows takes a workgroup per split, so shapes here assert
which of the two runs)."""

import pytest
import torch

from helpers import DT
from test_gpu_scored_attention import _call, _case, _check

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
