"""The hot-path ops registered as PyTorch operators: ``torch.ops.engpt_b200.*``.

Registering them with ``torch.library`` makes the CUDA kernels first-class
PyTorch operators (visible to ``torch.ops``, to the dispatcher and, through
the fake implementations below, to tracing and shape propagation) while the
computation still runs through the C ABI of ``libengpt_b200.so``.  The
operator signatures are those of the reference ops they replace:

* ``engpt_b200::qkv_postprocess_from_carried(qkv, rho, cos, sin, qk_scale, norm_eps) -> (q, k, v)``
  -- engpt/kernels.py:139-179
* ``engpt_b200::causal_sdpa(q, k, v, *, scale, dropout_p) -> o`` -- engpt/kernels.py:417-431
* ``engpt_b200::carried_residual_gauge(y, rho, branch, alpha, branch_eps, residual_eps, max_radius) -> (y, rho)``
  -- engpt/kernels.py:277-324

and those of the paged key-value cache (no counterpart in the reference; the arguments of ``engpt_b200.kernels``):

* ``engpt_b200::advance_block_tables(lengths, new_tokens, block_table, free_pages, free_count, finished=None, *,
  page_size, max_new) -> (slots, positions)`` (changes ``lengths``, ``block_table``, ``free_pages`` and ``free_count``)
* ``engpt_b200::qkv_append_from_carried(qkv, rho, cos, sin, qk_scale, norm_eps, positions, slots, k_pages, v_pages, *,
  qk_mult=1.0) -> q`` (changes ``k_pages`` and ``v_pages``)
* ``engpt_b200::write_kv_pages(k, v, slots, k_pages, v_pages)`` (the same)
* ``engpt_b200::paged_sdpa(q, k_pages, v_pages, block_table, lengths, *, scale) -> o``
* ``engpt_b200::write_kv_pages_q8``, ``qkv_append_from_carried_q8``, ``read_kv_pages_q8`` and ``paged_sdpa_q8``: the
  same on a cache of 8 bits (``k_pages, v_pages, k_scales, v_scales``; the writing ones change all four)

Only CUDA implementations are registered: a CPU tensor finds no kernel and
the dispatcher raises (there is no CPU fallback).  Like the underlying ops
they are forward-only.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from . import kernels as K

NAMESPACE = "engpt_b200"


@torch.library.custom_op(f"{NAMESPACE}::qkv_postprocess_from_carried", mutates_args=(), device_types="cuda")
def qkv_postprocess_from_carried(qkv: Tensor, rho: Tensor, cos: Tensor, sin: Tensor, qk_scale: Tensor,
                                 norm_eps: float) -> Tuple[Tensor, Tensor, Tensor]:
    return K.qkv_postprocess_from_carried(qkv, rho, cos, sin, qk_scale, norm_eps)


@qkv_postprocess_from_carried.register_fake
def _qkv_fake(qkv, rho, cos, sin, qk_scale, norm_eps):
    bsz, seq_len, _, n_head, head_dim = qkv.shape
    return tuple(qkv.new_empty(bsz, seq_len, n_head, head_dim) for _ in range(3))


@torch.library.custom_op(f"{NAMESPACE}::causal_sdpa", mutates_args=(), device_types="cuda")
def causal_sdpa(q: Tensor, k: Tensor, v: Tensor, *, scale: float, dropout_p: float) -> Tensor:
    return K.causal_sdpa(q, k, v, scale=scale, dropout_p=dropout_p)


@causal_sdpa.register_fake
def _sdpa_fake(q, k, v, *, scale, dropout_p):
    return q.new_empty(q.shape)


@torch.library.custom_op(f"{NAMESPACE}::carried_residual_gauge", mutates_args=(), device_types="cuda")
def carried_residual_gauge(y: Tensor, rho: Tensor, branch: Tensor, alpha: Tensor, branch_eps: float,
                           residual_eps: float, max_radius: float) -> Tuple[Tensor, Tensor]:
    return K.carried_residual_gauge(y, rho, branch, alpha, branch_eps, residual_eps, max_radius)


@carried_residual_gauge.register_fake
def _residual_fake(y, rho, branch, alpha, branch_eps, residual_eps, max_radius):
    dt = torch.promote_types(y.dtype, branch.dtype)
    return y.new_empty(y.shape, dtype=dt), rho.new_empty(rho.shape, dtype=dt)


@torch.library.custom_op(f"{NAMESPACE}::advance_block_tables",
                         mutates_args=("lengths", "block_table", "free_pages", "free_count"), device_types="cuda")
def advance_block_tables(lengths: Tensor, new_tokens: Tensor, block_table: Tensor, free_pages: Tensor,
                         free_count: Tensor, finished: Optional[Tensor] = None, *, page_size: int,
                         max_new: int) -> Tuple[Tensor, Tensor]:   # (a tensor argument cannot be keyword-only)
    return K.advance_block_tables(lengths, new_tokens, block_table, free_pages, free_count, page_size=page_size,
                                  max_new=max_new, finished=finished)


@advance_block_tables.register_fake
def _advance_fake(lengths, new_tokens, block_table, free_pages, free_count, finished=None, *, page_size, max_new):
    return tuple(lengths.new_empty(lengths.shape[0], max_new) for _ in range(2))


@torch.library.custom_op(f"{NAMESPACE}::qkv_append_from_carried", mutates_args=("k_pages", "v_pages"),
                         device_types="cuda")
def qkv_append_from_carried(qkv: Tensor, rho: Tensor, cos: Tensor, sin: Tensor, qk_scale: Tensor, norm_eps: float,
                            positions: Tensor, slots: Tensor, k_pages: Tensor, v_pages: Tensor, *,
                            qk_mult: float = 1.0) -> Tensor:
    return K.qkv_append_from_carried(qkv, rho, cos, sin, qk_scale, norm_eps, positions, slots, k_pages, v_pages,
                                     qk_mult=qk_mult)


@qkv_append_from_carried.register_fake
def _append_fake(qkv, rho, cos, sin, qk_scale, norm_eps, positions, slots, k_pages, v_pages, *, qk_mult=1.0):
    return qkv.new_empty(*qkv.shape[:-3], *qkv.shape[-2:])


@torch.library.custom_op(f"{NAMESPACE}::write_kv_pages", mutates_args=("k_pages", "v_pages"), device_types="cuda")
def write_kv_pages(k: Tensor, v: Tensor, slots: Tensor, k_pages: Tensor, v_pages: Tensor) -> None:
    K.write_kv_pages(k, v, slots, k_pages, v_pages)


@write_kv_pages.register_fake
def _write_fake(k, v, slots, k_pages, v_pages):
    return None


@torch.library.custom_op(f"{NAMESPACE}::paged_sdpa", mutates_args=(), device_types="cuda")
def paged_sdpa(q: Tensor, k_pages: Tensor, v_pages: Tensor, block_table: Tensor, lengths: Tensor, *,
               scale: float) -> Tensor:
    return K.paged_sdpa(q, k_pages, v_pages, block_table, lengths, scale=scale)


@paged_sdpa.register_fake
def _paged_sdpa_fake(q, k_pages, v_pages, block_table, lengths, *, scale):
    return q.new_empty(q.shape)


_Q8_CACHE = ("k_pages", "v_pages", "k_scales", "v_scales")


@torch.library.custom_op(f"{NAMESPACE}::write_kv_pages_q8", mutates_args=_Q8_CACHE, device_types="cuda")
def write_kv_pages_q8(k: Tensor, v: Tensor, slots: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Tensor,
                      v_scales: Tensor) -> None:
    K.write_kv_pages_q8(k, v, slots, k_pages, v_pages, k_scales, v_scales)


@write_kv_pages_q8.register_fake
def _write_q8_fake(k, v, slots, k_pages, v_pages, k_scales, v_scales):
    return None


@torch.library.custom_op(f"{NAMESPACE}::qkv_append_from_carried_q8", mutates_args=_Q8_CACHE, device_types="cuda")
def qkv_append_from_carried_q8(qkv: Tensor, rho: Tensor, cos: Tensor, sin: Tensor, qk_scale: Tensor, norm_eps: float,
                               positions: Tensor, slots: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Tensor,
                               v_scales: Tensor, *, qk_mult: float = 1.0) -> Tensor:
    return K.qkv_append_from_carried_q8(qkv, rho, cos, sin, qk_scale, norm_eps, positions, slots, k_pages, v_pages,
                                        k_scales, v_scales, qk_mult=qk_mult)


@qkv_append_from_carried_q8.register_fake
def _append_q8_fake(qkv, rho, cos, sin, qk_scale, norm_eps, positions, slots, k_pages, v_pages, k_scales, v_scales, *,
                    qk_mult=1.0):
    return qkv.new_empty(*qkv.shape[:-3], *qkv.shape[-2:])


@torch.library.custom_op(f"{NAMESPACE}::read_kv_pages_q8", mutates_args=(), device_types="cuda")
def read_kv_pages_q8(slots: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Tensor, v_scales: Tensor, *,
                     dtype: torch.dtype = torch.bfloat16) -> Tuple[Tensor, Tensor]:
    return K.read_kv_pages_q8(slots, k_pages, v_pages, k_scales, v_scales, dtype=dtype)


@read_kv_pages_q8.register_fake
def _read_q8_fake(slots, k_pages, v_pages, k_scales, v_scales, *, dtype=torch.bfloat16):
    return tuple(k_scales.new_empty(*slots.shape, k_pages.shape[1], k_pages.shape[3], dtype=dtype) for _ in range(2))


@torch.library.custom_op(f"{NAMESPACE}::paged_sdpa_q8", mutates_args=(), device_types="cuda")
def paged_sdpa_q8(q: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Tensor, v_scales: Tensor,
                  block_table: Tensor, lengths: Tensor, *, scale: float) -> Tensor:
    return K.paged_sdpa_q8(q, k_pages, v_pages, k_scales, v_scales, block_table, lengths, scale=scale)


@paged_sdpa_q8.register_fake
def _paged_sdpa_q8_fake(q, k_pages, v_pages, k_scales, v_scales, block_table, lengths, *, scale):
    return q.new_empty(q.shape)


OPS = ("qkv_postprocess_from_carried", "causal_sdpa", "carried_residual_gauge")
