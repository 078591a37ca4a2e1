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
