"""The batch-invariant kernels as dispatcher operators: ``torch.ops.mlx_bi.*``.

Registered with ``torch.library.custom_op`` when the package is imported, each
with a fake (shape / dtype) implementation, so code that goes through the
dispatcher reaches the HIP kernels by name: ``torch.compile`` graphs (the op
stays one opaque node; no generated kernel replaces it), ``torch.export``, and
C++ code in the same process through ``c10::Dispatcher``
(``findSchemaOrThrow("mlx_bi::matmul", "")``). The mode's monkey-patching
cannot reach callers that captured the stock functions before it was entered
(the reference's limitation, README.md:252-253); an explicit
``torch.ops.mlx_bi.*`` call is bound to the kernel whatever the mode.

Operators (each the same computation, and bits, as the Python function named):

* ``matmul(a, b)``: ``batch_invariant_matmul`` for 2-D ``b``, else
  ``batch_invariant_bmm``;
* ``quantized_matmul(x, w, scales, biases, group_size, bits)``;
* ``rms_norm(x, weight, eps)``; ``layer_norm(x, weight, bias, eps)``;
* ``attention(q, k, v, scale, causal, kv_lens)``: decode for one query token,
  prefill otherwise (``mask="causal"`` is bottom-right aligned);
* ``paged_attention(q, k_pages, v_pages, block_table, kv_lens, scale, causal)``:
  the same over a paged K/V pool (``batch_invariant_paged_attention``);
* ``scored_attention(q, k, v, scale, causal, kv_lens, softcap, slopes, doc_ids,
  prefix_lens)`` and ``scored_paged_attention(q, k_pages, v_pages, block_table,
  kv_lens, scale, causal, softcap, ...)``: the two with capped scores, a distance
  bias, a document mask or a prefix mask;
* ``residual_rms_norm(x, residual, post_weight, pre_weight, eps, gate, scale,
  post_norm=True, pre_norm=True)``: ``batch_invariant_residual_rms_norm``; returns
  (y, h), h empty without ``pre_norm``;
* ``paged_slots(kv_lens, new_lens, block_table!, free_pages, cursor, page_size,
  max_new)``: (slots, positions, kv_lens, cursor), the table changed in place;
* ``rope_paged_cache(q, k, v, cos, sin, positions, slots, k_pages!, v_pages!,
  sections)``: the rotated queries, the pools changed in place.

* ``rope_quantized_cache(q, k, v, cos, sin, positions, slots, k_codes!, k_groups!,
  v_codes!, v_groups!, bits, group_size, sections)``, ``read_quantized_cache(k_codes,
  k_groups, v_codes, v_groups, block_table, kv_lens, bits, group_size)`` and
  ``quantized_paged_attention(q, k_codes, k_groups, v_codes, v_groups, block_table,
  kv_lens, bits, group_size, scale, causal, shared_starts, shared_lens)``: the pools of
  a quantized paged cache, tensor by tensor;
* ``shared_prefix_attention(q, k_pages, v_pages, block_table, kv_lens, scale, causal,
  shared_starts, shared_lens)``: ``batch_invariant_shared_prefix_attention``.

The ops have no autograd formula (inference kernels, as in the reference).
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import kernels as _k

NAMESPACE = "mlx_bi"


@torch.library.custom_op(f"{NAMESPACE}::matmul", mutates_args=())
def matmul(a: Tensor, b: Tensor) -> Tensor:
    return _k.batch_invariant_matmul(a, b) if b.ndim == 2 else _k.batch_invariant_bmm(a, b)


@matmul.register_fake
def _matmul_fake(a, b):
    dt = torch.result_type(a, b)
    if b.ndim == 2:
        return a.new_empty((*a.shape[:-1], b.shape[1]), dtype=dt)
    batch = torch.broadcast_shapes(a.shape[:-2], b.shape[:-2])
    return a.new_empty((*batch, a.shape[-2], b.shape[-1]), dtype=dt)


@torch.library.custom_op(f"{NAMESPACE}::quantized_matmul", mutates_args=())
def quantized_matmul(x: Tensor, w: Tensor, scales: Tensor, biases: Tensor, group_size: int, bits: int) -> Tensor:
    return _k.batch_invariant_quantized_matmul(x, w, scales, biases, group_size=group_size, bits=bits)


@quantized_matmul.register_fake
def _quantized_matmul_fake(x, w, scales, biases, group_size, bits):
    return x.new_empty((*x.shape[:-1], w.shape[0]))


@torch.library.custom_op(f"{NAMESPACE}::rms_norm", mutates_args=())
def rms_norm(x: Tensor, weight: Optional[Tensor], eps: float) -> Tensor:
    return _k.batch_invariant_rms_norm(x, weight, eps)


@rms_norm.register_fake
def _rms_norm_fake(x, weight, eps):
    return torch.empty_like(x)


@torch.library.custom_op(f"{NAMESPACE}::layer_norm", mutates_args=())
def layer_norm(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float) -> Tensor:
    return _k.batch_invariant_layer_norm(x, weight, bias, eps)


@layer_norm.register_fake
def _layer_norm_fake(x, weight, bias, eps):
    return torch.empty_like(x)


@torch.library.custom_op(f"{NAMESPACE}::attention", mutates_args=())
def attention(q: Tensor, k: Tensor, v: Tensor, scale: float, causal: bool, kv_lens: Optional[Tensor]) -> Tensor:
    return _k.batch_invariant_attention(q, k, v, scale=scale, mask="causal" if causal else None, kv_lens=kv_lens)


@attention.register_fake
def _attention_fake(q, k, v, scale, causal, kv_lens):
    return q.new_empty((*q.shape[:-1], v.shape[-1]))


@torch.library.custom_op(f"{NAMESPACE}::paged_attention", mutates_args=())
def paged_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, block_table: Tensor, kv_lens: Optional[Tensor],
                    scale: float, causal: bool) -> Tensor:
    return _k.batch_invariant_paged_attention(q, k_pages, v_pages, block_table, kv_lens, scale=scale,
                                              mask="causal" if causal else None)


@paged_attention.register_fake
def _paged_attention_fake(q, k_pages, v_pages, block_table, kv_lens, scale, causal):
    return q.new_empty((*q.shape[:-1], v_pages.shape[-1]))


@torch.library.custom_op(f"{NAMESPACE}::residual_rms_norm", mutates_args=())
def residual_rms_norm(x: Tensor, residual: Tensor, post_weight: Optional[Tensor], pre_weight: Optional[Tensor],
                      eps: float, gate: Optional[Tensor], scale: float, post_norm: bool = True,
                      pre_norm: bool = True) -> tuple[Tensor, Tensor]:
    y, h = _k.batch_invariant_residual_rms_norm(x, residual, post_weight, pre_weight, eps, gate=gate, scale=scale,
                                                post_norm=post_norm, pre_norm=pre_norm)
    return y, x.new_empty(0) if h is None else h


@residual_rms_norm.register_fake
def _residual_rms_norm_fake(x, residual, post_weight, pre_weight, eps, gate, scale, post_norm=True, pre_norm=True):
    return x.new_empty(x.shape), x.new_empty(x.shape if pre_norm else 0)


@torch.library.custom_op(f"{NAMESPACE}::paged_slots", mutates_args=("block_table",))
def paged_slots(kv_lens: Tensor, new_lens: Tensor, block_table: Tensor, free_pages: Tensor,
                cursor: Optional[Tensor], page_size: int, max_new: int) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    p = _k.paged_slots(kv_lens, new_lens, block_table, free_pages, page_size=page_size, max_new=max_new, cursor=cursor)
    return tuple(p)


@paged_slots.register_fake
def _paged_slots_fake(kv_lens, new_lens, block_table, free_pages, cursor, page_size, max_new):
    new = lambda dt, *shape: block_table.new_empty(shape, dtype=dt)
    B = block_table.shape[0]
    return new(torch.int64, B, max_new), new(torch.int32, B, max_new), new(torch.int32, B), new(torch.int32, 1)


@torch.library.custom_op(f"{NAMESPACE}::rope_paged_cache", mutates_args=("k_pages", "v_pages"))
def rope_paged_cache(q: Tensor, k: Tensor, v: Tensor, cos: Tensor, sin: Tensor, positions: Tensor, slots: Tensor,
                     k_pages: Tensor, v_pages: Tensor, sections: Optional[list[int]]) -> Tensor:
    return _k.rope_paged_cache(q, k, v, cos, sin, positions, slots, k_pages, v_pages, sections=sections)


@rope_paged_cache.register_fake
def _rope_paged_cache_fake(q, k, v, cos, sin, positions, slots, k_pages, v_pages, sections):
    B, T, H, D = q.shape
    return q.new_empty((B, H, T, D))


@torch.library.custom_op(f"{NAMESPACE}::scored_attention", mutates_args=())
def scored_attention(q: Tensor, k: Tensor, v: Tensor, scale: float, causal: bool, kv_lens: Optional[Tensor],
                     softcap: Optional[float], slopes: Optional[Tensor], doc_ids: Optional[Tensor],
                     prefix_lens: Optional[Tensor]) -> Tensor:
    return _k.batch_invariant_attention(q, k, v, scale=scale, mask="causal" if causal else None, kv_lens=kv_lens,
                                        softcap=softcap, slopes=slopes, doc_ids=doc_ids, prefix_lens=prefix_lens)


@scored_attention.register_fake
def _scored_attention_fake(q, k, v, scale, causal, kv_lens, softcap, slopes, doc_ids, prefix_lens):
    return q.new_empty(q.shape)


@torch.library.custom_op(f"{NAMESPACE}::scored_paged_attention", mutates_args=())
def scored_paged_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, block_table: Tensor,
                           kv_lens: Optional[Tensor], scale: float, causal: bool, softcap: Optional[float],
                           slopes: Optional[Tensor], doc_ids: Optional[Tensor],
                           prefix_lens: Optional[Tensor]) -> Tensor:
    return _k.batch_invariant_paged_attention(q, k_pages, v_pages, block_table, kv_lens, scale=scale,
                                              mask="causal" if causal else None, softcap=softcap, slopes=slopes,
                                              doc_ids=doc_ids, prefix_lens=prefix_lens)


@scored_paged_attention.register_fake
def _scored_paged_attention_fake(q, k_pages, v_pages, block_table, kv_lens, scale, causal, softcap, slopes, doc_ids,
                                 prefix_lens):
    return q.new_empty(q.shape)


@torch.library.custom_op(f"{NAMESPACE}::rope_quantized_cache", mutates_args=("k_codes", "k_groups", "v_codes", "v_groups"))
def rope_quantized_cache(q: Tensor, k: Tensor, v: Tensor, cos: Tensor, sin: Tensor, positions: Tensor, slots: Tensor,
                         k_codes: Tensor, k_groups: Tensor, v_codes: Tensor, v_groups: Tensor, bits: int,
                         group_size: int, sections: Optional[list[int]]) -> Tensor:
    return _k.rope_quantized_cache(q, k, v, cos, sin, positions, slots,
                                   _k.QuantizedPages(k_codes, k_groups, bits, group_size),
                                   _k.QuantizedPages(v_codes, v_groups, bits, group_size), sections=sections)


@rope_quantized_cache.register_fake
def _rope_quantized_cache_fake(q, k, v, cos, sin, positions, slots, k_codes, k_groups, v_codes, v_groups, bits,
                               group_size, sections):
    B, T, H, D = q.shape
    return q.new_empty((B, H, T, D))


@torch.library.custom_op(f"{NAMESPACE}::read_quantized_cache", mutates_args=())
def read_quantized_cache(k_codes: Tensor, k_groups: Tensor, v_codes: Tensor, v_groups: Tensor, block_table: Tensor,
                         kv_lens: Optional[Tensor], bits: int, group_size: int) -> Tensor:
    """Keys and values as one tensor [2, B, Hkv, L, D] (an operator's outputs share no memory)."""
    k, v = _k.read_quantized_cache(_k.QuantizedPages(k_codes, k_groups, bits, group_size),
                                   _k.QuantizedPages(v_codes, v_groups, bits, group_size), block_table, kv_lens)
    return k._base if k._base is not None else torch.stack([k, v])


@read_quantized_cache.register_fake
def _read_quantized_cache_fake(k_codes, k_groups, v_codes, v_groups, block_table, kv_lens, bits, group_size):
    _, H, page, W = k_codes.shape
    B, cols = block_table.shape
    return k_groups.new_empty((2, B, H, cols * page, W * 8 // bits))


@torch.library.custom_op(f"{NAMESPACE}::quantized_paged_attention", mutates_args=())
def quantized_paged_attention(q: Tensor, k_codes: Tensor, k_groups: Tensor, v_codes: Tensor, v_groups: Tensor,
                              block_table: Tensor, kv_lens: Optional[Tensor], bits: int, group_size: int,
                              scale: float, causal: bool, shared_starts: Optional[Tensor],
                              shared_lens: Optional[Tensor]) -> Tensor:
    return _k.batch_invariant_quantized_paged_attention(
        q, _k.QuantizedPages(k_codes, k_groups, bits, group_size), _k.QuantizedPages(v_codes, v_groups, bits, group_size),
        block_table, kv_lens, scale=scale, mask="causal" if causal else None, shared_starts=shared_starts,
        shared_lens=shared_lens)


@quantized_paged_attention.register_fake
def _quantized_paged_attention_fake(q, k_codes, k_groups, v_codes, v_groups, block_table, kv_lens, bits, group_size, scale,
                                    causal, shared_starts, shared_lens):
    return q.new_empty(q.shape)


@torch.library.custom_op(f"{NAMESPACE}::shared_prefix_attention", mutates_args=())
def shared_prefix_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, block_table: Tensor, kv_lens: Optional[Tensor],
                            scale: float, causal: bool, shared_starts: Optional[Tensor],
                            shared_lens: Tensor) -> Tensor:
    return _k.batch_invariant_shared_prefix_attention(q, k_pages, v_pages, block_table, kv_lens, scale=scale,
                                                      mask="causal" if causal else None, shared_starts=shared_starts,
                                                      shared_lens=shared_lens)


@shared_prefix_attention.register_fake
def _shared_prefix_attention_fake(q, k_pages, v_pages, block_table, kv_lens, scale, causal, shared_starts, shared_lens):
    return q.new_empty(q.shape)
