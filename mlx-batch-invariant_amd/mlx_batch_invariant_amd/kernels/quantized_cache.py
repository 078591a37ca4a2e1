"""A paged K/V cache in 8 or 4 bits, and attention over it and behind shared prefixes.

A serving step of one block with such a cache:

    k_pages, v_pages = (bi.quantized_pages(n, Hkv, 16, D, bits=8, group_size=64) for _ in range(2))
    plan = bi.paged_slots(kv_lens, new_lens, block_table, free_pages, page_size=16, max_new=T, cursor=cursor)
    q = bi.rope_quantized_cache(q, k, v, cos, sin, plan.positions, plan.slots, k_pages, v_pages)
    out = bi.batch_invariant_quantized_paged_attention(q, k_pages, v_pages, block_table, plan.kv_lens, mask="causal")

The format is that of the quantized matmul's weights (MLX affine): a row of D values
is D codes of 8 or 4 bits, low to high within a 32-bit word, and one (scale, bias)
pair for each group of 32, 64 or 128 values; a code stands for ``T(fma(code, scale,
bias))``, T the type of q and of the pairs. Attention over the pages gives the bits of
``batch_invariant_paged_attention`` over the values that they stand for, so the
invariances of kernels/attention.py hold over a quantized cache too.

Sequences of a batch that begin with the same keys (an instruction, a document) may
say so: ``shared_lens`` and ``shared_starts``. The 256-key splits of the shared keys
are then those of the first sequence's pages, with the same bits as without, and calls
of few rows read them once for the whole group.

The reference quantizes weights only (mlx_batch_invariant/kernels/quantized.py:33-67)
and reads one contiguous cache for each sequence (kernels/attention.py:87-254).
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from .. import _lib
from .attention import MFMA_HEAD_DIMS, _aligned, _lens
from .paged_cache import _int32, _packed, _page_size, _row_stride, _rows
from .quantized import SUPPORTED_BITS, SUPPORTED_GROUPS


class QuantizedPages(NamedTuple):
    """One pool of a paged cache: ``codes`` uint8 ``[num_pages, Hkv, page_size, D *
    bits / 8]``, ``groups`` ``[num_pages, Hkv, page_size, D / group_size, 2]``, the
    (scale, bias) of every group. ``codes.view(torch.uint32)`` are MLX's words."""
    codes: torch.Tensor
    groups: torch.Tensor
    bits: int
    group_size: int

    @property
    def head_dim(self) -> int:
        return self.codes.shape[3] * 8 // self.bits


def quantized_pages(num_pages: int, kv_heads: int, page_size: int, head_dim: int, *, bits: int = 8,
                    group_size: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda") -> QuantizedPages:
    """An empty pool (zeros: every row reads as 0)."""
    _format("quantized_pages", bits, group_size, head_dim)
    _page_size("quantized_pages", page_size)
    if dtype not in _lib.FLOAT_DTYPES:
        raise ValueError(f"quantized_pages: unsupported dtype {dtype}")
    rows = (num_pages, kv_heads, page_size)
    return QuantizedPages(torch.zeros(*rows, head_dim * bits // 8, dtype=torch.uint8, device=device),
                          torch.zeros(*rows, head_dim // group_size, 2, dtype=dtype, device=device), bits, group_size)


def _format(what: str, bits, group_size, head_dim: int) -> None:
    whole = hasattr(bits, "__index__") and hasattr(group_size, "__index__")
    if not whole or bits not in SUPPORTED_BITS or group_size not in SUPPORTED_GROUPS:
        raise ValueError(f"{what}: bits={bits} group_size={group_size} (4 or 8 bits, groups of 32, 64 or 128)")
    if head_dim <= 0 or head_dim % group_size:
        raise ValueError(f"{what}: head dim {head_dim} is no whole number of groups of {group_size}")


_layouts: dict = {}


def _pools(what: str, k_pages: QuantizedPages, v_pages: QuantizedPages, dtype=None):
    """Checks a pair of pools; (num_pages, Hkv, page_size, D, the 12 strides). Shapes, strides and types
    that passed once are remembered (a lookup is cheaper than the checks on every step)."""
    key = None
    if type(k_pages) is QuantizedPages is type(v_pages):
        kc, kg, bits, gs = k_pages
        vc, vg, v_bits, v_gs = v_pages
        try:
            key = (kc.shape, kc.stride(), kg.shape, kg.stride(), vc.shape, vc.stride(), vg.shape, vg.stride(), kc.dtype, kg.dtype,
                   vc.dtype, vg.dtype, bits, gs, v_bits, v_gs, dtype)
            if not type(bits) is type(gs) is type(v_bits) is type(v_gs) is int:
                key = None                                # (8.0 would find what 8 left)
            seen = _layouts.get(key)
        except AttributeError:                            # a field that is no tensor: _check_pools names it
            seen = None
        if seen is not None and not (kc.data_ptr() | kg.data_ptr() | vc.data_ptr() | vg.data_ptr()) & 15:
            return seen
    seen = _check_pools(what, k_pages, v_pages, dtype)
    if key is not None:
        if len(_layouts) > 1024:
            _layouts.clear()
        _layouts[key] = seen
    return seen


def _check_pools(what: str, k_pages: QuantizedPages, v_pages: QuantizedPages, dtype):
    for p in (k_pages, v_pages):
        if not isinstance(p, QuantizedPages):
            raise ValueError(f"{what}: pools must be QuantizedPages; got {type(p).__name__}")
        if not isinstance(p.codes, torch.Tensor) or not isinstance(p.groups, torch.Tensor):
            raise ValueError(f"{what}: a pool's codes and groups must be tensors; got {type(p.codes).__name__} and "
                             f"{type(p.groups).__name__}")
    codes, groups, bits, gs = k_pages
    if (bits, gs) != v_pages[2:] or codes.shape != v_pages.codes.shape or groups.shape != v_pages.groups.shape:
        raise ValueError(f"{what}: pools of {bits} bits, groups of {gs}, {tuple(codes.shape)} and of "
                         f"{v_pages.bits}, {v_pages.group_size}, {tuple(v_pages.codes.shape)}")
    cs = codes.shape
    D = cs[3] * 8 // bits if len(cs) == 4 and bits in SUPPORTED_BITS else 0
    _format(what, bits, gs, D)
    _format(what, *v_pages[2:], D)
    if groups.shape != (*cs[:3], D // gs, 2):
        raise ValueError(f"{what}: groups {tuple(groups.shape)} for codes {tuple(cs)} of {bits} bits, groups of {gs}")
    _page_size(what, cs[2])
    if codes.dtype != torch.uint8 or v_pages.codes.dtype != torch.uint8:
        raise ValueError(f"{what}: codes must be uint8; got {codes.dtype} and {v_pages.codes.dtype}")
    dt = groups.dtype if dtype is None else dtype
    if dt not in _lib.FLOAT_DTYPES or groups.dtype != dt or v_pages.groups.dtype != dt:
        raise ValueError(f"{what}: the pools' pairs must be of one type of {_lib.FLOAT_DTYPES}, that of q; got "
                         f"{groups.dtype}, {v_pages.groups.dtype} and {dt}")
    strides = []
    for p in (k_pages, v_pages):
        c, g = p.codes.stride(), p.groups.stride()
        if (c[3] != 1 or (c[0] | c[1] | c[2] | p.codes.data_ptr() | p.groups.data_ptr()) & 15 or g[4] != 1
                or (groups.shape[3] > 1 and g[3] != 2) or (g[0] | g[1] | g[2]) & 1):
            raise ValueError(f"{what}: pool rows must be contiguous and 16-byte aligned; got strides {c} of codes, "
                             f"{g} of groups")
        strides += [*c[:3], *g[:3]]
    return cs[0], cs[1], cs[2], D, strides


def rope_quantized_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                         positions, slots: torch.Tensor, k_pages: QuantizedPages, v_pages: QuantizedPages, *,
                         sections=None) -> torch.Tensor:
    """``rope_paged_cache`` with quantized pools: rotate queries and keys, write
    keys and values in the pools' bits, in one launch; returns the queries ``[B, Hq,
    T, D]``. The arguments are as there.

    What ``rope_paged_cache`` would write (keys rounded to their type) is quantized
    by ``quantize``'s rule: per group of a row ``bias = min``, ``scale = (max - min) /
    (2^bits - 1)`` rounded to the type (1 where that is 0), ``code = round((y - bias) /
    scale)``, clamped. A code whose value the rounded scale would put past the type's
    largest number is not used. A group with an infinity or a NaN reads back as
    NaN. Of several tokens with one slot, each 16 values of the row keep some one's codes
    and each group some one's pair.
    """
    what = "rope_quantized_cache"
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or ks != v.shape or qs[:2] != ks[:2] or qs[3] != ks[3]:
        raise ValueError(f"{what}: shapes q {tuple(q.shape)} k {tuple(k.shape)} v {tuple(v.shape)}")
    B, T, Hq, D = qs
    Hkv, dt = ks[2], q.dtype
    if dt not in _lib.FLOAT_DTYPES or not dt == k.dtype == v.dtype:
        raise ValueError(f"{what}: q, k and v must have one type of {_lib.FLOAT_DTYPES}; got "
                         f"{[str(t.dtype) for t in (q, k, v)]}")
    num_pages, heads, page_size, dim, strides = _pools(what, k_pages, v_pages, dt)
    if heads != Hkv or dim != D:
        raise ValueError(f"{what}: pools of {heads} heads of {dim} for {Hkv} heads of {D}")
    if cos.ndim != 2 or cos.shape != sin.shape or cos.dtype != sin.dtype or cos.dtype not in (dt, torch.float32):
        raise ValueError(f"{what}: tables {cos.dtype} {tuple(cos.shape)} and {sin.dtype} {tuple(sin.shape)}; need "
                         f"one shape [n, R] in {dt} or float32")
    if slots.dtype not in (torch.int64, torch.int32) or tuple(slots.shape) != (B, T):
        raise ValueError(f"{what}: slots {slots.dtype} {tuple(slots.shape)}, expected int64 {(B, T)}")
    half = cos.shape[1]
    sections = (half,) if sections is None else tuple(map(int, sections))
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) != half:
        raise ValueError(f"{what}: sections {sections} of tables with {half} columns (1 to 4 axes)")
    if half % 8 or not 0 < half <= D // 2 or cos.shape[0] == 0:
        raise ValueError(f"{what}: head dim {D} with tables {tuple(cos.shape)}: need a positive multiple of 8 columns, "
                         "at most D / 2")
    written = (k_pages.codes, k_pages.groups, v_pages.codes, v_pages.groups)
    index = _lib.one_device(what, q, k, v, cos, sin, slots, *written)
    _lib.in_place(what, *written)
    kc, kg, vc, vg = (t.data_ptr() for t in written)
    if num_pages > 0 and (kc == vc or kg == vg):
        raise ValueError(f"{what}: one pool for keys and values")
    A, dev = len(sections), q.device
    pos = _int32(what, "positions", positions, dev)
    if pos.shape != (A, B, T) and (A > 1 or pos.shape != (B, T)):
        raise ValueError(f"{what}: positions {tuple(pos.shape)}, expected {(A, B, T)}")
    out = torch.empty((B, Hq, T, D), dtype=dt, device=dev)
    if B == 0 or T == 0:
        return out
    if num_pages == 0:
        raise ValueError(f"{what}: a pool without pages")
    q, k, v, cos, sin = _rows(q), _rows(k), _rows(v), _packed(cos), _packed(sin)
    if slots.dtype != torch.int64 or not slots.is_contiguous():
        slots = slots.to(torch.int64).contiguous()
    rc = _lib.launch(index, _lib.rope_quantized_call, q.data_ptr(), _row_stride(q), k.data_ptr(), _row_stride(k),
                     v.data_ptr(), _row_stride(v), cos.data_ptr(), sin.data_ptr(), cos.shape[0],
                     _lib.DTYPE_CODE[cos.dtype], pos.data_ptr(), A, *sections, *(0,) * (4 - A), slots.data_ptr(),
                     out.data_ptr(), kc, kg, vc, vg, num_pages, page_size, B, T, Hq, Hkv, D, k_pages.bits,
                     k_pages.group_size, *strides, _lib.DTYPE_CODE[dt], _lib.stream_of(q))
    if rc:
        _lib.check(rc, "bi_rope_quantized_cache")
    _lib.written(*written)
    return out


def _table(what: str, block_table: torch.Tensor) -> torch.Tensor:
    if block_table.ndim != 2 or block_table.is_floating_point():
        raise ValueError(f"{what}: block table must be int32 [B, max_pages]; got {block_table.dtype} "
                         f"{tuple(block_table.shape)}")
    if block_table.dtype == torch.int32 and block_table.is_contiguous():
        return block_table
    return block_table.to(torch.int32).contiguous()


def read_quantized_cache(k_pages: QuantizedPages, v_pages: QuantizedPages, block_table: torch.Tensor,
                         kv_lens=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of whole sequences out of quantized pools, in one launch: two
    contiguous ``[B, Hkv, max_pages * page_size, D]`` of the pairs' type, such as
    ``batch_invariant_attention`` takes. Row p of sequence b is what row ``p %
    page_size`` of page ``block_table[b, p // page_size]`` stands for, zeros from
    ``kv_lens[b]`` on (None: no row). Table entries outside the pool are clamped into
    it."""
    what = "read_quantized_cache"
    num_pages, Hkv, page_size, D, strides = _pools(what, k_pages, v_pages)
    table = _table(what, block_table)
    B, L = table.shape[0], table.shape[1] * page_size
    index = _lib.one_device(what, *k_pages[:2], *v_pages[:2], block_table)
    dev, dt = block_table.device, k_pages.groups.dtype
    kl = _lens(kv_lens, B, L, dev)
    out = torch.empty((2, B, Hkv, L, D), dtype=dt, device=dev)
    if B == 0 or L == 0:
        return out[0], out[1]
    if num_pages == 0:
        raise ValueError(f"{what}: a pool without pages")
    k, v = out.unbind(0)
    rc = _lib.launch(index, _lib.read_quantized_call, k_pages.codes.data_ptr(), k_pages.groups.data_ptr(),
                     v_pages.codes.data_ptr(), v_pages.groups.data_ptr(), *strides, table.data_ptr(), table.shape[1],
                     page_size, num_pages, _lib.ptr(kl), k.data_ptr(), v.data_ptr(), B, Hkv, L, D, k_pages.bits,
                     k_pages.group_size, 1, _lib.DTYPE_CODE[dt], _lib.stream_of(table))
    if rc:
        _lib.check(rc, "bi_read_quantized_cache")
    return k, v


def _groups_of(what: str, B: int, shared_starts, shared_lens, device):
    """(groups, starts, lens, the one length as a number)."""
    if shared_lens is None:
        if shared_starts is not None:
            raise ValueError(f"{what}: shared_starts without shared_lens")
        return 0, None, None, 0
    if isinstance(shared_lens, int) and not isinstance(shared_lens, bool):
        if shared_starts is not None:
            raise ValueError(f"{what}: one shared length goes without shared_starts (the whole batch shares it)")
        if shared_lens < 0:
            raise ValueError(f"{what}: shared length {shared_lens}")
        return 1, None, None, min(shared_lens, 0x7fffffff)
    lens = _int32(what, "shared_lens", shared_lens, device)
    n = lens.numel()
    if lens.ndim != 1 or (shared_starts is None and n != 1):
        raise ValueError(f"{what}: shared_lens {tuple(lens.shape)}; need one for each group, with shared_starts "
                         "[groups + 1] (None: one group)")
    if n > 65535:
        raise ValueError(f"{what}: {n} groups (at most 65535)")
    starts = None if shared_starts is None else _int32(what, "shared_starts", shared_starts, device, (n + 1,))
    return n, starts, lens, 0


def _attend(what, q, k, v, kg, vg, bits, gs, num_pages, Hkv, page_size, kv_strides, block_table, kv_lens, scale, mask,
            shared_starts, shared_lens) -> torch.Tensor:
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if mask is not None and mask != "causal":
        raise ValueError(f"{what}: mask must be None or 'causal'")
    B, Hq, Tq, D = q.shape
    if D not in MFMA_HEAD_DIMS or Hkv == 0 or Hq % Hkv:
        raise ValueError(f"{what}: {Hq} query heads of {D} on {Hkv}; need a multiple, and a head dim of {MFMA_HEAD_DIMS}")
    table = _table(what, block_table)
    if table.shape[0] != B:
        raise ValueError(f"{what}: block table {tuple(table.shape)} for batch {B}")
    index = _lib.one_device(what, q, k, v, kg, vg, block_table)
    dev, L, causal = q.device, table.shape[1] * page_size, mask == "causal"
    kl = _lens(kv_lens, B, L, dev)
    groups, starts, slens, shared = _groups_of(what, B, shared_starts, shared_lens, dev)
    if causal and Tq > L:
        raise ValueError(f"causal prefill needs T_q <= L (T_q={Tq}, L={L})")
    out = torch.empty((B, Hq, Tq, D), dtype=q.dtype, device=dev)
    if B == 0 or Tq == 0:
        return out
    if L == 0 or num_pages == 0:
        return out.zero_()
    if not _aligned(q) or max(q.stride()) >> 32:
        q = q.clone(memory_format=torch.contiguous_format)
    dt = _lib.DTYPE_CODE[q.dtype]
    n = _lib.ws_bytes("bi_attn_pages_workspace_bytes_paged", B, Hq, Hkv, Tq, L, D, groups, bits, int(causal), dt, page_size)
    ws = _lib.workspace(n, dev)
    rc = _lib.launch(index, _lib.pages_call, q.data_ptr(), k.data_ptr(), _lib.ptr(kg), v.data_ptr(), _lib.ptr(vg), bits, gs,
                     table.data_ptr(), table.shape[1], page_size, num_pages, _lib.ptr(kl), _lib.ptr(starts),
                     _lib.ptr(slens), shared, groups, out.data_ptr(), B, Hq, Hkv, Tq, L, D, *q.stride()[:3], *kv_strides,
                     int(causal), float(scale), dt, _lib.ptr(ws), n, _lib.stream_of(q))
    if rc:
        _lib.check(rc, "bi_attn_pages")
    return out


def batch_invariant_quantized_paged_attention(q: torch.Tensor, k_pages: QuantizedPages, v_pages: QuantizedPages,
                                              block_table: torch.Tensor, kv_lens=None, *, scale: float | None = None,
                                              mask=None, shared_starts=None, shared_lens=None) -> torch.Tensor:
    """Attention over a quantized paged cache: ``batch_invariant_paged_attention``
    (``q`` ``[B, Hq, T, D]`` of the pairs' type, ``block_table``, ``kv_lens``, ``scale``
    and ``mask`` as there) over the values that the pages stand for, bit for bit where
    they and q are finite. Keys that a query does not see take no part whatever their
    rows hold; one that sees none gets zeros; a NaN or infinity that it sees in V
    comes out in its dim.

    Single tokens and chunks of up to 64 rows (tokens x query heads of a kv head) read
    the codes; longer ones read them back first, into a workspace of up to 2 GiB (or
    one sequence).

    ``shared_lens`` / ``shared_starts``: as in ``batch_invariant_shared_prefix_attention``
    (None: no sequence shares its prefix). Read once where the codes are read, up to 64
    rows. Own keys take longer then: 64 sequences of up to 8192 keys of which none is
    shared 269 us instead of 150 in 8 bits, 242 instead of 98 in 4, so give them for
    prefixes that are long beside what follows.
    """
    what = "batch_invariant_quantized_paged_attention"
    if q.ndim != 4:
        raise ValueError(f"{what}: q {tuple(q.shape)}")
    num_pages, Hkv, page_size, D, s = _pools(what, k_pages, v_pages, q.dtype)
    if q.shape[3] != D:
        raise ValueError(f"{what}: q {tuple(q.shape)} for heads of {D}")
    return _attend(what, q, k_pages.codes, v_pages.codes, k_pages.groups, v_pages.groups, k_pages.bits, k_pages.group_size,
                   num_pages, Hkv, page_size, (*s[0:3], *s[6:9], *s[3:6], *s[9:12]), block_table, kv_lens, scale, mask,
                   shared_starts, shared_lens)


def batch_invariant_shared_prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                                            block_table: torch.Tensor, kv_lens=None, *, shared_lens,
                                            shared_starts=None, scale: float | None = None, mask=None) -> torch.Tensor:
    """``batch_invariant_paged_attention`` for sequences that share long prefixes; the
    same bits where q, K and V are finite. Single tokens read a prefix once for all
    of its group; so do the few rows (tokens x query heads of a kv head) of chunks whose
    batch does not fill the GPU otherwise, and up to 16 of them in 16-bit types with four sequences
    or more a group and 128 (sequence, kv head) pairs in the batch. Calls of more rows
    read it for every 64 rows of a sequence, from the first sequence's pages too.

    ``shared_lens`` int32 ``[N]`` and ``shared_starts`` int32 ``[N + 1]``, rising:
    sequences ``shared_starts[n]`` .. ``shared_starts[n + 1] - 1`` begin with the same
    ``shared_lens[n]`` keys. A number, or one length without ``shared_starts``: the
    whole batch. The whole 256-key splits of those keys, as far as the first sequence
    of the group holds them, come from that sequence's pages (the others' table
    entries there are not read), everything else from each sequence's own. Lengths
    and starts are read on the GPU, so one captured graph serves changing groups. Calls
    of many rows over pages of more than 256 keys need K and V pools whose page and row
    strides have one ratio, as pools of one layout have.

    The other arguments are those of ``batch_invariant_paged_attention``: pools
    ``[num_pages, Hkv, page_size, D]`` of q's type with contiguous rows at strides of
    whole 16 bytes. Hidden keys take no part whatever their rows hold; a query that
    sees no key gets zeros; infinities and NaN that a query sees in V come out in
    their dim.
    """
    what = "batch_invariant_shared_prefix_attention"
    if q.ndim != 4 or k_pages.ndim != 4 or k_pages.shape != v_pages.shape or k_pages.shape[3] != q.shape[3]:
        raise ValueError(f"{what}: unsupported shapes q {tuple(q.shape)} k {tuple(k_pages.shape)} v {tuple(v_pages.shape)}")
    if q.dtype not in _lib.FLOAT_DTYPES or not q.dtype == k_pages.dtype == v_pages.dtype:
        raise ValueError(f"{what}: q and the pools must have one type of {_lib.FLOAT_DTYPES}; got "
                         f"{[str(t.dtype) for t in (q, k_pages, v_pages)]}")
    if shared_lens is None:
        raise ValueError(f"{what}: shared_lens is needed")
    num_pages, Hkv, page_size, _ = k_pages.shape
    _page_size(what, page_size)
    unit = 16 // q.element_size()
    for t in (k_pages, v_pages):
        s = t.stride()
        if s[3] != 1 or any(x % unit for x in s[:3]) or t.data_ptr() % 16:
            raise ValueError(f"{what}: pool rows must be contiguous and 16-byte aligned; got strides {s}")
    return _attend(what, q, k_pages, v_pages, None, None, 0, 0, num_pages, Hkv, page_size,
                   (*k_pages.stride()[:3], *v_pages.stride()[:3], 0, 0, 0, 0, 0, 0), block_table, kv_lens, scale, mask,
                   shared_starts, shared_lens)
