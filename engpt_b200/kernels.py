"""``engpt.kernels``-compatible ops backed by the sm_100a kernels of ``libengpt_b200``.

Each function keeps the name, argument meaning and return shapes of the
reference op it replaces (cited per function, paths inside the
Pi-Willie/enGPT project) and launches CUDA kernels through the C ABI on the
current torch stream.  There is no CPU or library fallback: non-CUDA inputs,
float64, and autograd-tracked inputs raise.

Ownership differs from the reference in one place: the reference's no-grad
``qkv_postprocess_from_carried`` returns views into ``qkv`` after mutating it;
here ``qkv`` is read-only and fresh tensors are returned (callers in the
reference never reuse ``qkv``).
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _lib

__all__ = [
    "normalize_rows_",
    "normalize_columns_",
    "project_row_grad_",
    "project_column_grad_",
    "qkv_postprocess_from_carried",
    "causal_sdpa",
    "ngpt_attention_scale",
    "gpt_attention_scale",
    "carried_residual_gauge",
    "carried_residual",
    "rotary_frequencies",
    "carried_up_gate_swiglu",
    "scaled_logits_from_carried",
    "attention_strides",
    "advance_block_tables",
    "qkv_append_from_carried",
    "write_kv_pages",
    "paged_sdpa",
    "write_kv_pages_q8",
    "qkv_append_from_carried_q8",
    "read_kv_pages_q8",
    "paged_sdpa_q8",
]


def _require_cuda(*ts: Optional[Tensor]) -> torch.device:
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("engpt_b200 ops run on CUDA tensors only (no CPU fallback)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError("engpt_b200 ops: all tensors must be on the same device")
    return dev


def _forward_only(*ts: Optional[Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise NotImplementedError("engpt_b200 kernels are forward-only; call under torch.no_grad()")


def _f32c(t: Tensor) -> Tensor:
    return t.to(torch.float32).contiguous()


def ngpt_attention_scale(head_dim: int) -> float:
    """``sqrt(head_dim)`` -- engpt/kernels.py:434-435."""
    return math.sqrt(float(head_dim))


def gpt_attention_scale(head_dim: int) -> float:
    """``1/sqrt(head_dim)`` -- engpt/kernels.py:438-439."""
    return 1.0 / math.sqrt(float(head_dim))


def rotary_frequencies(seq_len: int, head_dim: int, *, device: torch.device, dtype: torch.dtype,
                       theta: float) -> Tuple[Tensor, Tensor]:
    """cos/sin tables ``[T, rd/2]`` -- engpt/kernels.py:355-374 (computed in fp32, cast to ``dtype``)."""
    device = torch.device(device)
    rd = head_dim - (head_dim % 2)
    if rd == 0:
        empty = torch.empty(seq_len, 0, device=device, dtype=dtype)
        return empty, empty
    if device.type != "cuda":
        raise RuntimeError("engpt_b200 ops run on CUDA tensors only (no CPU fallback)")
    cos = torch.empty(seq_len, rd // 2, device=device, dtype=torch.float32)
    sin = torch.empty_like(cos)
    with torch.cuda.device(device):
        _lib.call("engpt_rotary_tables", seq_len, head_dim, float(theta), cos.data_ptr(), sin.data_ptr(),
                  _lib.stream_handle(device))
    if dtype != torch.float32:
        return cos.to(dtype), sin.to(dtype)
    return cos, sin


def qkv_postprocess_into(qkv: Tensor, rho: Tensor, cos: Tensor, sin: Tensor, qk_scale: Tensor, qk_mult: float,
                         norm_eps: float, q: Tensor, k: Tensor, v: Tensor, head_major: bool) -> None:
    """Launch the fused epilogue into caller-owned ``q, k, v`` (no checks beyond the C ABI's)."""
    bsz, seq_len, _, n_head, head_dim = qkv.shape
    _lib.call("engpt_qkv_postprocess", qkv.data_ptr(), _lib.dtype_code(qkv.dtype), rho.data_ptr(),
              cos.data_ptr() if cos.numel() else None, sin.data_ptr() if sin.numel() else None, cos.shape[-1],
              qk_scale.data_ptr(), float(qk_mult), float(norm_eps), bsz, seq_len, n_head, head_dim,
              q.data_ptr(), k.data_ptr(), v.data_ptr(), _lib.QKV_BHTD if head_major else _lib.QKV_BTHD,
              _lib.stream_handle(qkv.device))


def qkv_postprocess_from_carried(qkv: Tensor, rho: Tensor, cos: Tensor, sin: Tensor, qk_scale: Tensor,
                                 norm_eps: float) -> Tuple[Tensor, Tensor, Tensor]:
    """Raw ``[B, T, 3, H, Dh]`` projection of carried ``Y`` -> nGPT attention inputs.

    engpt/kernels.py:139-179: q/k are L2-normalised per head (norm guarded by
    ``rho * eps``), rotated with interleaved RoPE and scaled by ``qk_scale``;
    v is divided by ``rho``.  Returns ``[B, T, H, Dh]`` tensors in ``qkv.dtype``.
    """
    _require_cuda(qkv, rho, cos, sin, qk_scale)
    _forward_only(qkv, rho, cos, sin, qk_scale)
    if qkv.dim() != 5 or qkv.shape[2] != 3:
        raise ValueError("qkv must have shape [B, T, 3, H, Dh]")
    bsz, seq_len, _, n_head, head_dim = qkv.shape
    if tuple(rho.shape) != (bsz, seq_len):
        raise ValueError("rho must have shape [batch, sequence]")
    if tuple(qk_scale.shape) != (n_head, head_dim):
        raise ValueError("qk_scale must have shape [n_head, head_dim]")
    half = (head_dim - head_dim % 2) // 2
    if cos.shape[-1] != half or cos.shape[0] < seq_len or sin.shape != cos.shape:
        raise ValueError("cos/sin must have shape [T, head_dim // 2]")
    qkv = qkv.contiguous()
    out = [torch.empty(bsz, seq_len, n_head, head_dim, device=qkv.device, dtype=qkv.dtype) for _ in range(3)]
    with torch.cuda.device(qkv.device):
        qkv_postprocess_into(qkv, _f32c(rho), _f32c(cos[:seq_len]), _f32c(sin[:seq_len]), _f32c(qk_scale), 1.0,
                             norm_eps, out[0], out[1], out[2], head_major=False)
    return out[0], out[1], out[2]


def attention_strides(q: Tensor, k: Tensor, v: Tensor, o: Tensor, head_major: bool) -> torch.Tensor:
    """Element strides (batch, token, head) of four ``[B,T,H,D]`` (or ``[B,H,T,D]``) tensors."""
    vals = []
    for t in (q, k, v, o):
        if t.stride(-1) != 1:
            raise ValueError("attention inputs need a contiguous head_dim axis")
        s = t.stride()
        vals += [s[0], s[2], s[1]] if head_major else [s[0], s[1], s[2]]
    return torch.tensor(vals, dtype=torch.int64)


def causal_attention_into(q: Tensor, k: Tensor, v: Tensor, o: Tensor, scale: float, strides: torch.Tensor,
                          bsz: int, seq_len: int, n_head: int, head_dim: int, impl: int = _lib.ATTN_AUTO) -> None:
    _lib.call("engpt_causal_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
              _lib.dtype_code(q.dtype), bsz, seq_len, n_head, head_dim, float(scale), strides.data_ptr(), impl,
              _lib.stream_handle(q.device))


def causal_sdpa(q: Tensor, k: Tensor, v: Tensor, *, scale: float, dropout_p: float, impl: str = "auto") -> Tensor:
    """Causal softmax attention on ``[B, T, H, D]`` inputs, returning ``[B, T, H, D]``.

    engpt/kernels.py:417-431 (``softmax(scale * q k^T + causal mask) v``).
    bf16 inputs with head_dim 64 or 128 run on the tcgen05 kernel; fp32 and
    other head dims run on the CUDA-core kernel.  ``impl`` ("auto",
    "tcgen05", "simt") forces a kernel.
    """
    _require_cuda(q, k, v)
    _forward_only(q, k, v)
    if dropout_p:
        raise NotImplementedError("engpt_b200 attention is inference-only (dropout_p must be 0)")
    if q.dim() != 4 or q.shape != k.shape or q.shape != v.shape:
        raise ValueError("q, k, v must share shape [B, T, H, D]")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise ValueError("q, k, v must share a dtype")
    bsz, seq_len, n_head, head_dim = q.shape
    q, k, v = (t if t.stride(-1) == 1 else t.contiguous() for t in (q, k, v))
    o = torch.empty(bsz, seq_len, n_head, head_dim, device=q.device, dtype=q.dtype)
    strides = attention_strides(q, k, v, o, head_major=False)
    code = {"auto": _lib.ATTN_AUTO, "tcgen05": _lib.ATTN_TCGEN05, "simt": _lib.ATTN_SIMT,
            "tcgen05_1tile": _lib.ATTN_TCGEN05_1TILE}[impl]
    with torch.cuda.device(q.device):
        causal_attention_into(q, k, v, o, scale, strides, bsz, seq_len, n_head, head_dim, code)
    return o


def carried_residual_into(y: Tensor, rho: Tensor, branch: Tensor, alpha: Tensor, alpha_mult: float,
                          alpha_abs: bool, branch_eps: float, residual_eps: float, max_radius: float,
                          y_out: Tensor, rho_out: Tensor, aux: Optional[Tensor], aux_mode: int) -> None:
    rows = rho.numel()
    d = y.shape[-1]
    _lib.call("engpt_carried_residual_gauge", y.data_ptr(), rho.data_ptr(), branch.data_ptr(),
              _lib.dtype_code(branch.dtype), alpha.data_ptr(), float(alpha_mult), 1 if alpha_abs else 0,
              float(branch_eps), float(residual_eps), float(max_radius), rows, d, y_out.data_ptr(),
              rho_out.data_ptr(), None if aux is None else aux.data_ptr(), aux_mode, _lib.stream_handle(y.device))


def carried_residual_gauge(y: Tensor, rho: Tensor, branch: Tensor, alpha: Tensor, branch_eps: float,
                           residual_eps: float, max_radius: float) -> Tuple[Tensor, Tensor]:
    """Carried nGPT residual with the exact gauge rescale, in one pass.

    engpt/kernels.py:277-324.  ``y`` ``[..., d]`` and ``rho`` ``[...]`` are
    carried in fp32 (as in the reference's autocast flow); ``branch`` may be
    bf16 or fp32; ``alpha`` is ``[d]`` (leading singleton dims allowed).
    """
    _require_cuda(y, rho, branch, alpha)
    _forward_only(y, rho, branch, alpha)
    if branch.shape != y.shape or tuple(rho.shape) != tuple(y.shape[:-1]):
        raise ValueError("y/branch must be [..., d] and rho [...]")
    d = y.shape[-1]
    if alpha.numel() != d:
        raise ValueError("alpha must have d elements")
    out_dtype = torch.promote_types(y.dtype, branch.dtype)
    yc = _f32c(y)
    bc = branch.contiguous() if branch.dtype in (torch.bfloat16, torch.float32) else branch.float().contiguous()
    y_out = torch.empty(y.shape, device=y.device, dtype=torch.float32)
    rho_out = torch.empty(rho.shape, device=y.device, dtype=torch.float32)
    with torch.cuda.device(y.device):
        carried_residual_into(yc, _f32c(rho), bc, _f32c(alpha.reshape(-1)), 1.0, False, branch_eps, residual_eps,
                              max_radius, y_out, rho_out, None, _lib.AUX_NONE)
    if out_dtype != torch.float32:
        return y_out.to(out_dtype), rho_out.to(out_dtype)
    return y_out, rho_out


def carried_residual(y: Tensor, rho: Tensor, branch: Tensor, alpha: Tensor, branch_eps: float,
                     residual_eps: float) -> Tuple[Tensor, Tensor]:
    """engpt/kernels.py:232-274: the residual without the gauge (``max_radius <= 0``)."""
    return carried_residual_gauge(y, rho, branch, alpha, branch_eps, residual_eps, 0.0)


def swiglu_into(ug: Tensor, s_u: Tensor, s_gate: Tensor, u_mult: float, gate_mult: float, out: Tensor) -> None:
    width = out.shape[-1]
    rows = out.numel() // width
    _lib.call("engpt_swiglu", ug.data_ptr(), _lib.dtype_code(ug.dtype), s_u.data_ptr(), s_gate.data_ptr(),
              float(u_mult), float(gate_mult), rows, width, out.data_ptr(), _lib.dtype_code(out.dtype),
              _lib.stream_handle(ug.device))


def carried_up_gate_swiglu(y: Tensor, rho: Tensor, weight: Tensor, s_u: Tensor, s_gate: Tensor, *, sqrt_d: float,
                           scale_u_by_sqrt_d: bool) -> Tensor:
    """MLP up/gate projection of ``Y/rho`` + SwiGLU -- engpt/kernels.py:182-206.

    Under bf16 autocast (the reference's GPU flow) with a width that is a
    multiple of 128: the tcgen05 GEMM with SwiGLU in its epilogue
    (``engpt_up_gate_swiglu``), so the ``[.., 2W]`` projection is never
    written; otherwise a cuBLAS GEMM (through torch, honouring autocast) and
    the SwiGLU kernel.  The result has the reference's dtype (bf16 GEMM output
    times fp32 scales: fp32).
    """
    _require_cuda(y, rho, weight, s_u, s_gate)
    _forward_only(y, rho, weight, s_u, s_gate)
    mlp_in = y / rho.unsqueeze(-1)
    d = mlp_in.shape[-1]
    width = weight.shape[0] // 2
    if (torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16
            and width % 128 == 0 and d % 8 == 0 and weight.shape[1] == d):
        x = mlp_in.reshape(-1, d).to(torch.bfloat16).contiguous()
        w = weight.to(torch.bfloat16).contiguous()
        hidden = torch.empty(x.shape[0], width, device=x.device, dtype=torch.bfloat16)
        su, sg = _f32c(s_u), _f32c(s_gate)
        with torch.cuda.device(y.device):
            _lib.call("engpt_up_gate_swiglu", x.data_ptr(), w.data_ptr(), su.data_ptr(), sg.data_ptr(),
                      float(sqrt_d if scale_u_by_sqrt_d else 1.0), float(sqrt_d), x.shape[0], d, width,
                      hidden.data_ptr(), _lib.stream_handle(y.device))
        out_dtype = torch.promote_types(torch.bfloat16, s_u.dtype)
        return hidden.view(*mlp_in.shape[:-1], width).to(out_dtype)
    ug = torch.nn.functional.linear(mlp_in, weight).contiguous()
    width = ug.shape[-1] // 2
    out = torch.empty(*ug.shape[:-1], width, device=ug.device, dtype=torch.promote_types(ug.dtype, s_u.dtype))
    with torch.cuda.device(y.device):
        swiglu_into(ug, _f32c(s_u), _f32c(s_gate), sqrt_d if scale_u_by_sqrt_d else 1.0, sqrt_d, out)
    return out


def scaled_logits_from_carried(y: Tensor, rho: Tensor, output_emb: Tensor, logit_scale: Tensor) -> Tensor:
    """``<Y, E_out[v]> s_z[v] / rho`` -- engpt/kernels.py:209-229 (cuBLAS GEMM on row-scaled weights)."""
    _require_cuda(y, rho, output_emb, logit_scale)
    _forward_only(y, rho, output_emb, logit_scale)
    h = y / rho.unsqueeze(-1)
    w = torch.empty(output_emb.shape, device=y.device,
                    dtype=torch.bfloat16 if torch.is_autocast_enabled("cuda") else torch.float32)
    emb32, scale32 = _f32c(output_emb), _f32c(logit_scale)
    with torch.cuda.device(y.device):
        _lib.call("engpt_scale_rows_cast", emb32.data_ptr(), scale32.data_ptr(), 1.0, output_emb.shape[0],
                  output_emb.shape[1], w.data_ptr(), _lib.dtype_code(w.dtype), _lib.stream_handle(y.device))
    return torch.nn.functional.linear(h.to(w.dtype), w)


# ------------------------------------------------------------ optimizer-side sphere operations
def _sphere_matrix(x: Tensor, what: str) -> None:
    if not x.is_cuda:
        raise RuntimeError("engpt_b200 ops run on CUDA tensors only (no CPU fallback)")
    if x.ndim != 2 or not x.is_contiguous():
        raise ValueError(f"{what}: needs a contiguous 2-D matrix, got shape {tuple(x.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise NotImplementedError(f"{what}: float32 and bfloat16 only, got {x.dtype}")


@torch.no_grad()
def normalize_rows_(x: Tensor, eps: float = 1e-12) -> Tensor:
    """In place: every row to unit L2 norm, ``x[r] /= max(|x[r]|, eps)`` -- engpt/kernels.py:98-105."""
    _sphere_matrix(x, "normalize_rows_")
    with torch.cuda.device(x.device):
        _lib.call("engpt_normalize_rows", x.data_ptr(), _lib.dtype_code(x.dtype), x.shape[0], x.shape[1],
                  float(eps), _lib.stream_handle(x.device))
    return x


def _column_scratch(x: Tensor) -> Tensor:
    n = int(_lib.load().engpt_column_scratch_floats(x.shape[0], x.shape[1]))
    return torch.empty(max(n, 1), device=x.device, dtype=torch.float32)


@torch.no_grad()
def normalize_columns_(x: Tensor, eps: float = 1e-12) -> Tensor:
    """In place: every column to unit L2 norm, ``x[:, c] /= max(|x[:, c]|, eps)`` -- engpt/kernels.py:108-116."""
    _sphere_matrix(x, "normalize_columns_")
    scratch = _column_scratch(x)
    with torch.cuda.device(x.device):
        _lib.call("engpt_normalize_columns", x.data_ptr(), _lib.dtype_code(x.dtype), x.shape[0], x.shape[1],
                  float(eps), scratch.data_ptr(), _lib.stream_handle(x.device))
    return x


def _check_pair(weight: Tensor, grad: Tensor, what: str) -> None:
    _sphere_matrix(weight, what)
    _sphere_matrix(grad, what)
    if weight.shape != grad.shape or weight.dtype != grad.dtype or weight.device != grad.device:
        raise ValueError(f"{what}: weight and grad must share shape, dtype and device")


@torch.no_grad()
def project_row_grad_(weight: Tensor, grad: Tensor) -> None:
    """In place: ``grad[r] -= (grad[r] . weight[r]) weight[r]`` (tangent space of unit rows) --
    engpt/kernels.py:119-125."""
    _check_pair(weight, grad, "project_row_grad_")
    with torch.cuda.device(grad.device):
        _lib.call("engpt_project_row_grad", weight.data_ptr(), grad.data_ptr(), _lib.dtype_code(grad.dtype),
                  grad.shape[0], grad.shape[1], _lib.stream_handle(grad.device))


@torch.no_grad()
def project_column_grad_(weight: Tensor, grad: Tensor) -> None:
    """In place: ``grad[:, c] -= (grad[:, c] . weight[:, c]) weight[:, c]`` (tangent space of unit columns) --
    engpt/kernels.py:128-136."""
    _check_pair(weight, grad, "project_column_grad_")
    scratch = _column_scratch(grad)
    with torch.cuda.device(grad.device):
        _lib.call("engpt_project_column_grad", weight.data_ptr(), grad.data_ptr(), _lib.dtype_code(grad.dtype),
                  grad.shape[0], grad.shape[1], scratch.data_ptr(), _lib.stream_handle(grad.device))


# ------------------------------------------------------------ paged key-value cache
# Argument checks and launches are in the compiled binding (csrc/bindings.cpp).
def advance_block_tables(lengths: Tensor, new_tokens: Tensor, block_table: Tensor, free_pages: Tensor,
                         free_count: Tensor, *, page_size: int, max_new: int, finished: Optional[Tensor] = None
                         ) -> Tuple[Tensor, Tensor]:
    """One step of the page allocator on the device; returns the new tokens' ``(slots, positions)``.

    ``lengths`` ``[B]`` (tokens of each request in the cache), ``block_table``
    ``[B, W]``, the stack ``free_pages`` ``[num_pages]`` and its size
    ``free_count`` ``[1]``, all int32, are updated in place.  Rows with
    ``finished`` (bool ``[B]``) set first give all their pages back and become
    empty; then every row takes the pages that ``new_tokens[b]`` more tokens
    need, rows in order.  ``slots`` and ``positions`` are int32 ``[B,
    max_new]``: a token's place in the cache (``page * page_size + offset``)
    and in its sequence; ``-1`` and 0 behind a row's last new token.  At most 8192
    rows.

    A row whose request cannot be met (more than ``max_new`` tokens, a table
    row too short, no pages left) is refused whole: its length stays, its
    slots are ``-1``, and ``engpt_b200._lib.raise_on_device_status`` reports it.
    """
    return _lib.native().advance_block_tables(lengths, new_tokens, block_table, free_pages, free_count, page_size,
                                              max_new, finished)


def qkv_append_from_carried(qkv: Tensor, rho: Tensor, cos: Tensor, sin: Tensor, qk_scale: Tensor, norm_eps: float,
                            positions: Tensor, slots: Tensor, k_pages: Tensor, v_pages: Tensor, *,
                            qk_mult: float = 1.0) -> Tensor:
    """``qkv_postprocess_from_carried`` at given positions, with k and v written to the paged cache.

    ``qkv`` ``[..., 3, H, Dh]`` holds raw projection rows of carried ``Y`` with
    radii ``rho`` ``[...]``; ``positions`` ``[...]`` selects each token's rotary
    row and ``slots`` ``[...]`` its place in ``k_pages`` / ``v_pages``
    ``[num_pages, H, page_size, Dh]`` (``-1``: k and v are not kept), both
    int32.  Slots other than ``-1`` must be distinct.  Returns q ``[..., H,
    Dh]``; the scale applied to q and k is ``qk_scale * qk_mult``.
    """
    return _lib.native().qkv_append(qkv, rho, cos, sin, qk_scale, norm_eps, positions, slots, k_pages, v_pages,
                                    qk_mult)


def write_kv_pages(k: Tensor, v: Tensor, slots: Tensor, k_pages: Tensor, v_pages: Tensor) -> None:
    """Copy finished k and v ``[..., H, Dh]`` into their cache slots (``slots`` ``[...]`` int32, ``-1``: none).

    k and v may be views into the packed ``[B, T, 3, H, Dh]`` projection.
    Slots other than ``-1`` must be distinct.
    """
    _lib.native().write_kv_pages(k, v, slots, k_pages, v_pages)


def paged_sdpa(q: Tensor, k_pages: Tensor, v_pages: Tensor, block_table: Tensor, lengths: Tensor, *,
               scale: float) -> Tensor:
    """Attention of one new token per request over its cached keys and values; returns ``[B, H, Dh]``.

    ``softmax(scale * q k^T) v`` over the first ``lengths[b]`` tokens of the
    pages in ``block_table[b]`` (int32, as ``advance_block_tables`` keeps them);
    query head ``h`` reads kv head ``h // (H // kv_heads)``.  A row of length 0
    gives zeros.  Whatever lies in the cache behind a row's length (stale or
    NaN) has no effect.  ``k_pages`` and ``v_pages`` are ``[num_pages, kv_heads,
    page_size, Dh]`` with any strides and a contiguous last axis, ``Dh`` at most
    256.  bf16 with ``Dh`` up to 128 and a multiple of 8, pages of a multiple of 8
    tokens and 16-byte aligned strides runs on the tensor cores.

    How the work is split follows from the width of ``block_table``, as the
    lengths are on the device: where they are known to be short, a table cut to
    them (``block_table[:, :n]``) is faster than a wide one.
    """
    return _lib.native().paged_sdpa(q, k_pages, v_pages, block_table, lengths, scale)


# ------------------------------------------------------------ the paged cache in 8 bits
# k_pages / v_pages: int8 or float8_e4m3fn [num_pages, kv_heads, page_size, Dh]; k_scales / v_scales: float32 [num_pages,
# kv_heads, blocks per page].  A block is page_size / blocks tokens of one page and kv head; a number is code * scale.
def write_kv_pages_q8(k: Tensor, v: Tensor, slots: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Tensor,
                      v_scales: Tensor) -> None:
    """Quantise finished k and v ``[..., H, Dh]`` (bf16 or fp32) into their cache slots (``-1``: none).

    The tokens that one call puts into a block are quantised together.  If one of
    them is the block's first token the block starts anew with the scale that they
    need, ``max(max |x|, 2^-100) / top`` (``top`` 127 for int8, 448 for e4m3);
    otherwise it keeps the larger one of that and its scale so far, and where
    that grows, the codes of its other tokens become ``round(code * (scale before
    / scale))``.  Codes are ``round(x / scale)``, with the quotient as a product
    of fp32 numbers: next to the middle between two codes either may be taken.
    An infinity or NaN makes the block's scale NaN until the block starts anew.

    Slots other than ``-1`` must be distinct, and those of one block stand side by
    side in ``slots`` (seen as one row) and follow one another, ``s, s + 1, s + 2``, as
    ``advance_block_tables`` gives them.  A token beside another one of its block, but
    not in the next slot, is left out with those that follow it, and
    ``engpt_b200._lib.raise_on_device_status`` reports it.  Where tokens of other blocks or
    ``-1`` stand between those of one block, its numbers are undefined.
    """
    _lib.native().write_kv_pages_q8(k, v, slots, k_pages, v_pages, k_scales, v_scales)


def qkv_append_from_carried_q8(qkv: Tensor, rho: Tensor, cos: Tensor, sin: Tensor, qk_scale: Tensor, norm_eps: float,
                               positions: Tensor, slots: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Tensor,
                               v_scales: Tensor, *, qk_mult: float = 1.0) -> Tensor:
    """``qkv_append_from_carried`` into a cache of 8 bits (the rules of ``write_kv_pages_q8``).

    k and v are quantised from their fp32 values, without a rounding to
    ``qkv``'s type in between.  Returns q ``[..., H, Dh]`` in ``qkv``'s type.
    """
    return _lib.native().qkv_append_q8(qkv, rho, cos, sin, qk_scale, norm_eps, positions, slots, k_pages, v_pages,
                                       k_scales, v_scales, qk_mult)


def read_kv_pages_q8(slots: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Tensor, v_scales: Tensor, *,
                     dtype: torch.dtype = torch.bfloat16) -> Tuple[Tensor, Tensor]:
    """The numbers ``code * scale`` of given cache slots (int32 ``[...]``; ``-1`` gives zeros).

    Returns k and v ``[..., H, Dh]`` in ``dtype`` (bfloat16 or float32).
    """
    return _lib.native().read_kv_pages_q8(slots, k_pages, v_pages, k_scales, v_scales, dtype)


def paged_sdpa_q8(q: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Tensor, v_scales: Tensor,
                  block_table: Tensor, lengths: Tensor, *, scale: float) -> Tensor:
    """``paged_sdpa`` over a cache of 8 bits: ``softmax(scale * q k^T) v`` with k and v the numbers that it stands for.

    q ``[B, H, Dh]`` and the result are bf16 or fp32.  Codes and scales behind a
    row's length have no effect, whatever they are.  The tensor cores are used for
    ``Dh`` up to 128 and a multiple of 16, pages and blocks of a multiple of 8
    tokens and 16-byte aligned strides.  There an element of q is good to 2^-15
    (fp32: 2^-23) of its row's largest one over int8 codes, and a weight of a
    value to 2^-11 (fp32: 2^-21), or 2^-39 of its head's largest.
    """
    return _lib.native().paged_sdpa_q8(q, k_pages, v_pages, k_scales, v_scales, block_table, lengths, scale)
