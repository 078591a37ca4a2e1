"""What fills a paged K/V cache: the pages and slots of a step's new tokens, and
the rotary embedding with the write of keys and values into the pages.

A serving step of one block, for requests padded to the same number T of new
tokens, the new ones last (as the bottom-right aligned causal attention counts):

    plan = bi.paged_slots(kv_lens, new_lens, block_table, free_pages, page_size=16, max_new=T, cursor=cursor)
    q = bi.rope_paged_cache(q, k, v, cos, sin, plan.positions, plan.slots, k_pages, v_pages)
    out = bi.batch_invariant_paged_attention(q, k_pages, v_pages, block_table, plan.kv_lens, mask="causal")

Every output element depends on its own request's data only, except the page
numbers, which follow from the requests before it (a page's number changes no
value). The reference's caches are contiguous
(mlx_batch_invariant/kernels/attention.py:87-254).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib

_INTS = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)


class PagedSlots(NamedTuple):
    """What ``paged_slots`` gives a step: see there."""
    slots: torch.Tensor
    positions: torch.Tensor
    kv_lens: torch.Tensor
    cursor: torch.Tensor


def _int32(what: str, name: str, t, device, shape=None) -> torch.Tensor:
    """``t`` (a tensor of whole numbers, or a list) as contiguous int32 on ``device``."""
    if not (isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.device == device and t.is_contiguous()):
        if isinstance(t, torch.Tensor) and t.dtype not in _INTS:
            raise ValueError(f"{what}: {name} must hold whole numbers; got {t.dtype}")
        if isinstance(t, torch.Tensor) and t.is_cuda and t.device != device:
            raise ValueError(f"{what}: {name} on {t.device}, expected {device}")
        t = torch.as_tensor(t, dtype=torch.int32, device=device).contiguous()
    if shape is not None and t.shape != shape:
        raise ValueError(f"{what}: {name} {tuple(t.shape)}, expected {tuple(shape)}")
    return t


def _page_size(what: str, page_size: int) -> None:
    if isinstance(page_size, bool) or not isinstance(page_size, int) or page_size <= 0 or page_size & (page_size - 1):
        raise ValueError(f"{what}: page size {page_size!r} is not a power of two")


def paged_slots(kv_lens, new_lens, block_table: torch.Tensor, free_pages, *, page_size: int, max_new: int,
                cursor=None) -> PagedSlots:
    """Pages and slots of a step's new tokens, planned on the GPU in one launch.

    ``kv_lens`` / ``new_lens``: int32 ``[B]``, the tokens request b holds and
    gets (0 .. ``max_new`` = T); ``block_table``: int32 ``[B, max_pages]``,
    changed in place: request b's new pages are written behind those that its
    ``kv_lens[b]`` tokens fill; ``free_pages``: int32 ``[F]``, of which the pages
    from ``cursor`` (int32 ``[1]``, None: the first) on are handed out, request
    by request in order.

    Returns ``slots`` int64 ``[B, T]`` (page * page_size + row of each new token,
    in the last ``new_lens[b]`` rows; -1 in the others), ``positions`` int32
    ``[B, T]`` (its place in the sequence; 0 in the others), ``kv_lens`` int32
    ``[B]`` (after the step) and ``cursor`` int32 ``[1]`` (behind the last page
    taken). The inputs other than the table are left as they are, so a step can
    be planned again with the same outcome; a loop hands the returned lengths and
    cursor to the next step.

    A request whose pages fit neither its table row nor the free list, or with
    more than T new tokens, is refused: no page, slots -1, its length stays
    (``plan.kv_lens[b] < kv_lens[b] + new_lens[b]`` tells). Behind a request that
    the free list cannot serve only those that need no page are served. Negative
    counts are 0, lengths past the table's reach are cut to it. (Wider whole numbers
    are taken modulo 2^32.)
    """
    what = "paged_slots"
    _page_size(what, page_size)
    if isinstance(max_new, bool) or not isinstance(max_new, int) or max_new < 1:
        raise ValueError(f"{what}: max_new must be a positive int; got {max_new!r}")
    if block_table.ndim != 2 or block_table.dtype != torch.int32:
        raise ValueError(f"{what}: block table must be int32 [B, max_pages]; got {block_table.dtype} "
                         f"{tuple(block_table.shape)}")
    B, max_pages = block_table.shape
    if B > 0 and max_pages == 0:
        raise ValueError(f"{what}: block table without columns")
    stride, one = block_table.stride()
    if one != 1 and max_pages > 1 or B > 1 and stride < max_pages:
        raise ValueError(f"{what}: block table rows must be contiguous and apart; got strides {block_table.stride()}")
    index = _lib.one_device(what, block_table)
    _lib.in_place(what, block_table)
    dev = block_table.device
    lens = _int32(what, "kv_lens", kv_lens, dev, (B,))
    news = _int32(what, "new_lens", new_lens, dev, (B,))
    free = _int32(what, "free_pages", free_pages, dev)
    if free.ndim != 1:
        raise ValueError(f"{what}: free_pages must be one list; got {tuple(free.shape)}")
    cur = None if cursor is None else _int32(what, "cursor", cursor, dev, (1,))
    slots = torch.empty((B, max_new), dtype=torch.int64, device=dev)
    positions = torch.empty_like(slots, dtype=torch.int32)
    out = torch.empty_like(lens)
    end = lens.new_empty(1) if cur is None else torch.empty_like(cur)
    max_pages = max(max_pages, 1)
    rc = _lib.launch(index, _lib.slots_call, lens.data_ptr(), news.data_ptr(), block_table.data_ptr(),
                     stride if B > 1 else max_pages, max_pages, free.data_ptr(), free.numel(), _lib.ptr(cur),
                     slots.data_ptr(), positions.data_ptr(), out.data_ptr(), end.data_ptr(), B, max_new, page_size,
                     _lib.stream_of(block_table))
    if rc:
        _lib.check(rc, "bi_paged_slots")
    _lib.written(block_table)
    return PagedSlots(slots, positions, out, end)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` [B, T, H, D] with contiguous heads and all tokens at one stride of
    whole 16-byte pieces (such as a slice of a joint projection), else a copy."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    B, T, H, D = t.shape
    unit = 16 // t.element_size()
    s = t.stride()
    ok = (s[3] == 1 and (H == 1 or s[2] == D) and t.data_ptr() % 16 == 0
          and (T == 1 or s[1] % unit == 0 and s[1] >= H * D)
          and (B == 1 or (s[0] == T * s[1] if T > 1 else s[0] % unit == 0 and s[0] >= H * D)))
    if not ok:
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _packed(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous and 16-byte aligned, or a copy that is."""
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _row_stride(t: torch.Tensor) -> int:
    B, T, H, D = t.shape
    return t.stride(1) if T > 1 else t.stride(0) if B > 1 else H * D


def rope_paged_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                     positions, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, *,
                     sections=None) -> torch.Tensor:
    """Rotate queries and keys by their positions and write keys and values into
    the pages of the cache, in one launch; returns the queries ``[B, Hq, T, D]``.

    ``q`` ``[B, T, Hq, D]``, ``k`` / ``v`` ``[B, T, Hkv, D]`` as the projections
    give them; ``k_pages`` / ``v_pages`` ``[num_pages, Hkv, page_size, D]``, the
    pools of ``batch_invariant_paged_attention``, changed in place; ``slots``
    int64 ``[B, T]`` as ``paged_slots`` gives them: one outside the pool (-1: a
    padding row) writes nothing, and each of the others should occur once (of
    rows written twice either one's values may stay, piece by piece).

    ``cos`` / ``sin`` ``[n, R]`` (fp32 or q's type): row p, column j turns the
    pair of dims (j, R + j) of a head at position p; dims from 2 R on are copied
    (R a multiple of 8, at most D / 2). ``positions`` ``[B, T]``, or ``[A, B, T]``
    for tokens placed along up to four axes (time, height, width), with
    ``sections`` the A numbers of pairs that turn with each axis, in order
    (their sum is R). A position outside the tables is clamped into them (int32;
    wider numbers are taken modulo 2^32). Each
    product and sum is in fp32, the result rounded once.
    """
    what = "rope_paged_cache"
    qs, ks, ps = q.shape, k.shape, k_pages.shape
    if len(qs) != 4 or len(ks) != 4 or ks != v.shape or qs[:2] != ks[:2] or qs[3] != ks[3]:
        raise ValueError(f"{what}: shapes q {tuple(q.shape)} k {tuple(k.shape)} v {tuple(v.shape)}")
    B, T, Hq, D = qs
    Hkv = ks[2]
    if len(ps) != 4 or ps != v_pages.shape or ps[1] != Hkv or ps[3] != D:
        raise ValueError(f"{what}: pools {tuple(k_pages.shape)} and {tuple(v_pages.shape)} for {Hkv} heads of {D}")
    dt = q.dtype
    if dt not in _lib.FLOAT_DTYPES or not dt == k.dtype == v.dtype == k_pages.dtype == v_pages.dtype:
        raise ValueError(f"{what}: q, k, v and the pools must have one type of {_lib.FLOAT_DTYPES}; got "
                         f"{[str(t.dtype) for t in (q, k, v, k_pages, v_pages)]}")
    if cos.ndim != 2 or cos.shape != sin.shape or cos.dtype != sin.dtype or cos.dtype not in (dt, torch.float32):
        raise ValueError(f"{what}: tables {cos.dtype} {tuple(cos.shape)} and {sin.dtype} {tuple(sin.shape)}; need "
                         f"one shape [n, R] in {dt} or float32")
    if slots.dtype not in (torch.int64, torch.int32) or tuple(slots.shape) != (B, T):
        raise ValueError(f"{what}: slots {slots.dtype} {tuple(slots.shape)}, expected int64 {(B, T)}")
    page_size = ps[2]
    _page_size(what, page_size)
    half = cos.shape[1]
    sections = (half,) if sections is None else tuple(map(int, sections))
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) != half:
        raise ValueError(f"{what}: sections {sections} of tables with {half} columns (1 to 4 axes)")
    if D % 16 or half % 8 or not 0 < half <= D // 2 or cos.shape[0] == 0:
        raise ValueError(f"{what}: head dim {D} with tables {tuple(cos.shape)}: need D % 16 == 0 and a positive "
                         "multiple of 8 columns, at most D / 2")
    index = _lib.one_device(what, q, k, v, cos, sin, slots, k_pages, v_pages)
    _lib.in_place(what, k_pages, v_pages)
    unit = 16 // q.element_size()
    kst, vst = k_pages.stride(), v_pages.stride()
    kp, vp = k_pages.data_ptr(), v_pages.data_ptr()
    if kp == vp and ps[0] > 0:
        raise ValueError(f"{what}: one pool for keys and values")
    for s, p in ((kst, kp), (vst, vp)):
        if s[3] != 1 or s[0] % unit or s[1] % unit or s[2] % unit or p % 16:
            raise ValueError(f"{what}: pool rows must be contiguous and 16-byte aligned; got strides {s}")
    A, dev = len(sections), q.device
    pos = _int32(what, "positions", positions, dev)
    if pos.shape != (A, B, T) and (A > 1 or pos.shape != (B, T)):
        raise ValueError(f"{what}: positions {tuple(pos.shape)}, expected {(A, B, T)}")
    out = torch.empty((B, Hq, T, D), dtype=dt, device=dev)
    if B == 0 or T == 0:
        return out
    if ps[0] == 0:
        raise ValueError(f"{what}: a pool without pages")
    q, k, v, cos, sin = _rows(q), _rows(k), _rows(v), _packed(cos), _packed(sin)
    if slots.dtype != torch.int64 or not slots.is_contiguous():
        slots = slots.to(torch.int64).contiguous()
    rc = _lib.launch(index, _lib.rope_paged_call, q.data_ptr(), _row_stride(q), k.data_ptr(), _row_stride(k),
                     v.data_ptr(), _row_stride(v), cos.data_ptr(), sin.data_ptr(), cos.shape[0],
                     _lib.DTYPE_CODE[cos.dtype], pos.data_ptr(), A, *sections, *(0,) * (4 - A), slots.data_ptr(),
                     out.data_ptr(), kp, vp, ps[0], page_size, B, T, Hq, Hkv, D, *kst[:3], *vst[:3],
                     _lib.DTYPE_CODE[dt], _lib.stream_of(q))
    if rc:
        _lib.check(rc, "bi_rope_paged_cache")
    _lib.written(k_pages, v_pages)
    return out
