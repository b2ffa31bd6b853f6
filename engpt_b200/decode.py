"""Generation from an ``EfficientNGPT`` with a paged key-value cache.

The reference has no cache: its forwards are whole sequences.  Here a
``PagedKVCache`` holds the post-processed keys and values (unit vectors times
s_qk, V / rho) of up to ``max_batch`` requests in pages shared by all of
them, and a ``PagedDecoder`` runs the model over it:

* ``prefill(idx, rows)`` takes prompts in through the model's whole-sequence
  forward (tcgen05 GEMMs and attention) and writes every layer's k and v to
  the requests' pages (``kernels.write_kv_pages``);
* ``step(idx)`` adds one token to every request.  Per layer:

    qkv      = Y @ W_qkv^T                                     cuBLAS
    q        = post-process, k and v to their slots            kernels.qkv_append_from_carried
    attn     = attention over the request's pages              kernels.paged_sdpa
    Y, rho   = carried residual of attn @ W_o^T                engpt_carried_residual_gauge
    Y, rho   = carried residual of SwiGLU(..) @ W_down^T       cuBLAS, engpt_swiglu

The cache can be held in 8 bits (int8 or float8_e4m3fn codes with a scale for
each head and block of tokens): k and v are quantised as they are written and
the attention reads the codes (the ``_q8`` forms of the three operators).  A
prompt's own attention sees its k and v before that.

Pages are handed out and taken back on the GPU
(``kernels.advance_block_tables``), so a step makes no host synchronisation
and can be captured: ``enable_cuda_graphs()`` replays the whole step.
"""

from __future__ import annotations

import math
from typing import Callable, List, Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import _lib
from . import kernels as K
from .config import ModelConfig
from .models import plain_tensors

__all__ = ["PagedKVCache", "PagedDecoder"]

_CODES = (torch.int8, torch.float8_e4m3fn)


class PagedKVCache:
    """Page pools of all layers and the page allocator's state for ``max_batch`` requests.

    ``k_pages`` / ``v_pages`` ``[layers, num_pages, heads, page_size, Dh]``;
    ``lengths`` ``[max_batch]``, ``block_table`` ``[max_batch, pages per
    request]``, ``free_pages`` ``[num_pages]`` and ``free_count`` ``[1]`` are int32
    views of one buffer.  A page holds ``page_size`` tokens of one request in
    every layer.  A request has at most ``max_len`` tokens (default
    ``block_size``), rounded up to whole pages.

    With ``dtype`` int8 or float8_e4m3fn the pools hold codes, and ``k_scales`` /
    ``v_scales`` float32 ``[layers, num_pages, heads, page_size / scale_block]`` their
    scales, one for every ``scale_block`` tokens of a page (a divisor of
    ``page_size``; default 16, or 8, if it is one, else the page).
    """

    @plain_tensors
    def __init__(self, cfg: ModelConfig, max_batch: int, num_pages: int, *, page_size: int = 64,
                 max_len: Optional[int] = None, dtype: torch.dtype = torch.bfloat16,
                 scale_block: Optional[int] = None, device: Optional[torch.device] = None) -> None:
        if min(max_batch, num_pages, page_size) < 1:
            raise ValueError("max_batch, num_pages and page_size must be positive")
        if dtype not in (torch.bfloat16, torch.float32, *_CODES):
            raise NotImplementedError("a paged cache holds float32, bfloat16, int8 or float8_e4m3fn, got "
                                      f"{dtype}")
        if dtype in _CODES:
            if scale_block is None:
                scale_block = next((b for b in (16, 8) if page_size % b == 0), page_size)
            if scale_block < 1 or page_size % scale_block:
                raise ValueError(f"scale_block must divide page_size {page_size}, got {scale_block}")
        elif scale_block is not None:
            raise ValueError(f"a cache of {dtype} has no scales")
        device = torch.device("cuda") if device is None else torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("engpt_b200 ops run on CUDA tensors only (no CPU fallback)")
        self.max_batch, self.num_pages, self.page_size = max_batch, num_pages, page_size
        self.pages_per_request = -(-(cfg.block_size if max_len is None else max_len) // page_size)
        shape = (cfg.n_layer, num_pages, cfg.n_head, page_size, cfg.head_dim)
        self.k_pages = torch.empty(shape, dtype=dtype, device=device)
        self.v_pages = torch.empty(shape, dtype=dtype, device=device)
        self.scale_block = scale_block
        self.k_scales = self.v_scales = None
        if self.quantised:
            shape = shape[:3] + (page_size // scale_block,)
            self.k_scales = torch.zeros(shape, dtype=torch.float32, device=device)
            self.v_scales = torch.zeros(shape, dtype=torch.float32, device=device)
        state = torch.empty(max_batch + 1 + num_pages + max_batch * self.pages_per_request, dtype=torch.int32,
                            device=device)
        self.lengths, self.free_count, self.free_pages, table = state.split(
            [max_batch, 1, num_pages, max_batch * self.pages_per_request])
        self.block_table = table.view(max_batch, self.pages_per_request)
        self.reset()

    @property
    def capacity(self) -> int:
        """Tokens that one request can have."""
        return self.pages_per_request * self.page_size

    @property
    def quantised(self) -> bool:
        """Whether the pools hold 8-bit codes."""
        return self.k_pages.dtype in _CODES

    def layer(self, i: int) -> Tuple[Tensor, ...]:
        """Pools of layer ``i``: k and v pages, and their scales if they hold codes."""
        if not self.quantised:
            return self.k_pages[i], self.v_pages[i]
        return self.k_pages[i], self.v_pages[i], self.k_scales[i], self.v_scales[i]

    @torch.no_grad()
    def read(self, layer: int, row: int, n: int, *, dtype: Optional[torch.dtype] = None) -> Tuple[Tensor, Tensor]:
        """k and v ``[n, heads, Dh]`` of the first ``n`` tokens of request ``row`` in a layer, zeros behind its length.

        ``dtype`` is bfloat16 or float32 (default: the pools' own, bfloat16 for codes).
        """
        if not 0 <= row < self.max_batch or not 0 <= n <= self.capacity:
            raise ValueError(f"row must be in [0, {self.max_batch}) and n in [0, {self.capacity}], got {row} and {n}")
        pos = torch.arange(n, device=self.lengths.device)
        page = self.block_table[row].index_select(0, pos // self.page_size)
        there = pos < self.lengths[row]
        slots = torch.where(there, page * self.page_size + pos % self.page_size, -1).to(torch.int32)
        pools = self.layer(layer)
        if self.quantised:
            return K.read_kv_pages_q8(slots, *pools, dtype=torch.bfloat16 if dtype is None else dtype)
        at = slots.clamp(min=0).long()
        return tuple(p[at // self.page_size, :, at % self.page_size].masked_fill_(~there[:, None, None], 0.0).to(
            p.dtype if dtype is None else dtype) for p in pools)

    def reset(self) -> None:
        """Drop all requests: every page is free."""
        self.lengths.zero_()
        self.block_table.fill_(-1)
        self.free_pages.copy_(torch.arange(self.num_pages - 1, -1, -1, dtype=torch.int32))   # page 0 on top
        self.free_count.fill_(self.num_pages)

    def advance(self, new_tokens: Tensor, max_new: int, finished: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
        """``kernels.advance_block_tables`` on this cache."""
        return K.advance_block_tables(self.lengths, new_tokens, self.block_table, self.free_pages, self.free_count,
                                      page_size=self.page_size, max_new=max_new, finished=finished)


class _StepGraph:
    """A captured step: static inputs, the graph and its logits."""

    @plain_tensors
    def __init__(self, dec: "PagedDecoder") -> None:
        b, dev = dec.cache.max_batch, dec.device
        self.idx = torch.zeros(b, dtype=torch.int64, device=dev)
        self.new_tokens = torch.zeros(b, dtype=torch.int32, device=dev)
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            dec._step(self.idx, self.new_tokens)       # warm-up (no new tokens: the cache is left as it is)
        torch.cuda.current_stream(dev).wait_stream(side)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.logits = dec._step(self.idx, self.new_tokens)

    def replay(self, idx: Tensor, new_tokens: Tensor) -> Tensor:
        self.idx.copy_(idx, non_blocking=True)
        self.new_tokens.copy_(new_tokens, non_blocking=True)
        self.graph.replay()
        return self.logits


class PagedDecoder:
    """Generates from ``model`` for up to ``max_batch`` requests at a time (see the module's text).

    ``dtype`` is the compute type: bfloat16 (as the model under bf16 autocast)
    or float32.  Steps use the parameters that the decoder took when it was built
    or last refreshed (in bfloat16 its own copies of the linear weights, in both
    types its own scaled copy of the head): call ``refresh_weights()`` after the
    model's parameters have changed, in place or for other tensors.  ``cache_dtype``
    (default: ``dtype``) int8 or float8_e4m3fn holds the cache in 8 bits, with a
    scale for every ``scale_block`` tokens (``PagedKVCache``).  Requests are
    rows ``0 .. max_batch - 1``.  ``prefill`` uses the model's parameters and
    activation buffers, as its forward does: one stream at a time.
    """

    @plain_tensors
    def __init__(self, model, max_batch: int, num_pages: int, *, page_size: int = 64, max_len: Optional[int] = None,
                 dtype: torch.dtype = torch.bfloat16, cache_dtype: Optional[torch.dtype] = None,
                 scale_block: Optional[int] = None) -> None:
        p = model.token_emb.weight
        if not p.is_cuda:
            raise RuntimeError("engpt_b200 EfficientNGPT runs on CUDA only (no CPU fallback); call .cuda()")
        if p.dtype != torch.float32:
            raise NotImplementedError(f"engpt_b200 forward runs fp32 parameters (got {p.dtype})")
        if model.head_split is not None:
            raise NotImplementedError("a head-split model cannot decode from a paged cache")
        self.model, self.cfg, self.device, self.dtype = model, model.cfg, p.device, dtype
        if dtype not in (torch.bfloat16, torch.float32):
            raise NotImplementedError(f"engpt_b200 kernels support float32 and bfloat16, got {dtype}")
        if cache_dtype is not None and cache_dtype != dtype and cache_dtype not in _CODES:
            raise NotImplementedError(f"the cache holds the compute type {dtype}, int8 or float8_e4m3fn, got {cache_dtype}")
        self.cache = PagedKVCache(model.cfg, max_batch, num_pages, page_size=page_size, max_len=max_len,
                                  dtype=dtype if cache_dtype is None else cache_dtype, scale_block=scale_block,
                                  device=p.device)
        self.cos, self.sin = K.rotary_frequencies(self.cache.capacity, model.cfg.head_dim, device=p.device,
                                                  dtype=torch.float32, theta=model.cfg.rope_theta)
        self._graph: Optional[_StepGraph] = None
        self.cuda_graphs = False
        self._ones = torch.ones(max_batch, dtype=torch.int32, device=p.device)
        # what a step reads of each block, and the embedding: held here, so that neither an eager step nor a captured
        # one can read a tensor that the model has given up, and a step's parameters are all of one refresh
        self._w: List[dict] = [{} for _ in model.blocks]
        self._emb = torch.empty(0)
        self._w_head = torch.zeros(-(-model.cfg.vocab_size // 64) * 64, model.cfg.n_embd, device=self.device,
                                   dtype=dtype)
        self.refresh_weights()

    def _take(self, name: str, p: Tensor, *shape: int) -> Tensor:
        if p.device != self.device or p.dtype != torch.float32 or tuple(p.shape) != shape:
            raise ValueError(f"{name} must be float32 {list(shape)} on {self.device}, got {p.dtype} {list(p.shape)} on "
                             f"{p.device}")
        return p.detach().contiguous()

    @plain_tensors
    def refresh_weights(self) -> None:
        """Take the model's current parameters (in float32 all but the head are used in place).

        A captured step is captured again if a parameter that it reads in place
        has become another tensor.
        """
        m, cfg = self.model, self.cfg
        d, width = cfg.n_embd, cfg.mlp_width
        linear = {"qkv": (3 * d, d), "out_proj": (d, d), "up_gate": (2 * width, d), "down_proj": (d, width)}
        small = {"s_qk": (cfg.n_head, cfg.head_dim), "s_u": (width,), "s_gate": (width,), "alpha_attn_raw": (d,),
                 "alpha_mlp_raw": (d,)}
        # everything is looked at before anything is taken
        emb = self._take("token_emb.weight", m.token_emb.weight, cfg.vocab_size, d)
        out = self._take("output_emb", m.output_emb, cfg.vocab_size, d)
        s_z = self._take("s_z", m.s_z, cfg.vocab_size)
        taken = []
        for i, b in enumerate(m.blocks):
            taken.append({n: self._take(f"blocks.{i}.{n}.weight", getattr(b, n).weight, *s) for n, s in linear.items()})
            taken[i].update((n, self._take(f"blocks.{i}.{n}", getattr(b, n), *s)) for n, s in small.items())
        if self.dtype == torch.bfloat16:
            for old, new in zip(self._w, taken):
                for n in linear:
                    new[n] = old[n].copy_(new[n]) if old else new[n].to(self.dtype)
        if self._addresses(emb, taken) != self._addresses(self._emb, self._w):
            self._graph = None
        self._emb, self._w = emb, taken
        with torch.cuda.device(self.device):
            _lib.call("engpt_scale_rows_cast", out.data_ptr(), s_z.data_ptr(), float(m.logit_mult),
                      cfg.vocab_size, cfg.n_embd, self._w_head.data_ptr(), _lib.dtype_code(self.dtype),
                      _lib.stream_handle(self.device))

    @staticmethod
    def _addresses(emb: Tensor, blocks: List[dict]) -> List[int]:
        return [emb.data_ptr()] + [t.data_ptr() for b in blocks for t in b.values()]

    # ---------------------------------------------------------------- requests
    def _rows_mask(self, rows: Sequence[int]) -> Tuple[List[int], Tensor]:
        rows = [int(r) for r in rows]
        if len(set(rows)) != len(rows) or any(r < 0 or r >= self.cache.max_batch for r in rows):
            raise ValueError(f"rows must be distinct and in [0, {self.cache.max_batch}), got {rows}")
        mask = torch.zeros(self.cache.max_batch, dtype=torch.bool)
        mask[rows] = True
        return rows, mask.to(self.device, non_blocking=True)

    @torch.no_grad()
    def release(self, rows: Sequence[int]) -> None:
        """Give the pages of these requests back."""
        _, mask = self._rows_mask(rows)
        self.cache.advance(torch.zeros_like(self._ones), 0, mask)

    @torch.no_grad()
    def prefill(self, idx: Tensor, rows: Optional[Sequence[int]] = None,
                lengths: Optional[Sequence[int]] = None) -> Tensor:
        """Start requests in ``rows`` (default ``0 .. n-1``) with the prompts ``idx`` ``[n, T]``.

        ``lengths`` gives the prompts' lengths (1 to T, default T; what is behind
        them in ``idx`` is ignored but must be valid token ids).  Whatever the rows
        held before is released.  Returns the logits ``[n, V]`` after each prompt's
        last token.  A prompt that finds too few pages is refused
        (``advance_block_tables``): its row stays empty and its logits are zeros.
        """
        if idx.dim() != 2 or idx.shape[0] == 0 or idx.shape[1] == 0:
            raise ValueError("idx must have shape [requests, tokens]")
        n, seq_len = idx.shape
        if seq_len > min(self.cfg.block_size, self.cache.capacity):
            raise ValueError("sequence length exceeds block_size or the cache's max_len")
        rows, mask = self._rows_mask(range(n) if rows is None else rows)
        lens = [seq_len] * n if lengths is None else [int(x) for x in lengths]
        if len(rows) != n or len(lens) != n or any(x < 1 or x > seq_len for x in lens):
            raise ValueError("rows and lengths must have one entry per prompt, lengths in [1, T]")
        cache = self.cache
        new = torch.zeros(cache.max_batch, dtype=torch.int32)
        new[rows] = torch.tensor(lens, dtype=torch.int32)
        with torch.cuda.device(self.device):
            slots, _ = cache.advance(new.to(self.device, non_blocking=True), seq_len, mask)
            slots = slots.index_select(0, torch.tensor(rows).to(self.device, non_blocking=True))
            refused = slots[:, :1] < 0
            last = torch.tensor([b * seq_len + x - 1 for b, x in enumerate(lens)]).to(self.device, non_blocking=True)

            write = K.write_kv_pages_q8 if cache.quantised else K.write_kv_pages

            def keep(layer: int, k: Tensor, v: Tensor) -> None:
                write(k, v, slots, *cache.layer(layer))

            with torch.autocast("cuda", dtype=torch.bfloat16, enabled=self.dtype == torch.bfloat16):
                logits, _ = self.model._run(idx=idx, kv_callback=keep, head_rows=last)
        return logits.masked_fill_(refused, 0.0)

    # ---------------------------------------------------------------- one token
    @torch.no_grad()
    def step(self, idx: Tensor, active: Optional[Tensor] = None) -> Tensor:
        """Append token ``idx[b]`` to every request and return the logits ``[max_batch, V]`` that follow it.

        ``active`` (bool ``[max_batch]``) leaves the other rows' requests as they
        are; their logits are zeros.  A request that finds no page, has ``block_size``
        tokens already or fills the cache's capacity is refused
        (``advance_block_tables``): its token is not kept, its logits are zeros too.
        With CUDA graphs the returned logits are overwritten by the next step.
        """
        b = self.cache.max_batch
        if tuple(idx.shape) != (b,):
            raise ValueError(f"idx must have shape [{b}]")
        if active is not None and (active.dtype != torch.bool or tuple(active.shape) != (b,)):
            raise ValueError(f"active must be a bool tensor of shape [{b}]")
        new = self._ones if active is None else active.to(device=self.device, dtype=torch.int32, non_blocking=True)
        idx = idx.to(device=self.device, dtype=torch.int64, non_blocking=True)
        # (the compute type is the decoder's, whatever autocast region the caller is in)
        with torch.cuda.device(self.device), torch.autocast("cuda", enabled=False):
            if self.cuda_graphs:
                if self._graph is None:
                    self._graph = _StepGraph(self)
                return self._graph.replay(idx, new)
            return self._step(idx.contiguous(), new)

    def enable_cuda_graphs(self, enabled: bool = True) -> None:
        """Replay ``step`` from one captured CUDA graph (captured by the first step)."""
        self.cuda_graphs = enabled
        if not enabled:
            self._graph = None

    def _step(self, idx: Tensor, new_tokens: Tensor) -> Tensor:
        m, cfg, cache = self.model, self.cfg, self.cache
        b, d, heads, dim, width = cache.max_batch, cfg.n_embd, cfg.n_head, cfg.head_dim, cfg.mlp_width
        bf16 = self.dtype == torch.bfloat16
        st = _lib.stream_handle(self.device)
        y = torch.empty(b, d, device=self.device, dtype=torch.float32)
        rho = torch.empty(b, device=self.device, dtype=torch.float32)
        x = torch.empty(b, d, device=self.device, dtype=self.dtype) if bf16 else y
        h = x if bf16 else torch.empty_like(y)     # operand Y / rho of the MLP and the head
        hidden = torch.empty(b, width, device=self.device, dtype=self.dtype)
        if cache.capacity > cfg.block_size:
            # whole pages may leave room behind the block size: two tokens where one may be asked for are refused
            new_tokens = torch.where(cache.lengths < cfg.block_size, new_tokens, 2 * new_tokens)
        slots, positions = cache.advance(new_tokens, 1)
        slots, positions = slots.view(b), positions.view(b)
        _lib.call("engpt_embed_carried", idx.data_ptr(), self._emb.data_ptr(), b, d, cfg.vocab_size,
                  y.data_ptr(), rho.data_ptr(), x.data_ptr() if bf16 else None, st)
        scale, sqrt_d = K.ngpt_attention_scale(dim), math.sqrt(float(d))
        u_mult = sqrt_d if cfg.scale_mlp_u_by_sqrt_d else 1.0
        act, aux_h = _lib.dtype_code(self.dtype), _lib.AUX_BF16_H if bf16 else _lib.AUX_F32_H
        last = cfg.n_layer - 1
        append, attend = ((K.qkv_append_from_carried_q8, K.paged_sdpa_q8) if cache.quantised else
                          (K.qkv_append_from_carried, K.paged_sdpa))
        for i, (blk, w) in enumerate(zip(m.blocks, self._w)):
            qkv = torch.mm(x, w["qkv"].t()).view(b, 3, heads, dim)
            pools = cache.layer(i)
            q = append(qkv, rho, self.cos, self.sin, w["s_qk"], cfg.norm_eps, positions, slots, *pools,
                       qk_mult=blk.qk_mult)
            attn = attend(q, *pools, cache.block_table, cache.lengths, scale=scale)
            branch = torch.mm(attn.view(b, d), w["out_proj"].t())
            K.carried_residual_into(y, rho, branch, w["alpha_attn_raw"], blk.alpha_mult, True, cfg.norm_eps,
                                    cfg.norm_eps, cfg.carried_gauge_max, y, rho, h, aux_h)
            ug = torch.mm(h, w["up_gate"].t())
            _lib.call("engpt_swiglu", ug.data_ptr(), act, w["s_u"].data_ptr(), w["s_gate"].data_ptr(), float(u_mult),
                      float(sqrt_d), b, width, hidden.data_ptr(), act, st)
            branch = torch.mm(hidden, w["down_proj"].t())
            # what comes next reads Y (the next layer's QKV) or Y / rho (the head)
            aux = aux_h if i == last else (_lib.AUX_BF16_Y if bf16 else _lib.AUX_NONE)
            K.carried_residual_into(y, rho, branch, w["alpha_mlp_raw"], blk.alpha_mult, True, cfg.norm_eps,
                                    cfg.norm_eps, cfg.carried_gauge_max, y, rho,
                                    None if aux == _lib.AUX_NONE else h, aux)
        h.masked_fill_((slots < 0).unsqueeze(1), 0.0)    # refused rows (and inactive ones)
        return torch.mm(h, self._w_head.t())[:, :cfg.vocab_size]

    # ---------------------------------------------------------------- generation
    @torch.no_grad()
    def generate(self, idx: Tensor, max_new_tokens: int, *, lengths: Optional[Sequence[int]] = None,
                 pick: Optional[Callable[[Tensor], Tensor]] = None) -> Tensor:
        """``max_new_tokens`` tokens for each of the prompts ``idx`` ``[n, T]``, as ``[n, max_new_tokens]``.

        ``pick`` chooses the next tokens ``[n]`` from the logits ``[n, V]``
        (default: the largest).  The requests take rows ``0 .. n-1`` and are released
        at the end, also if ``pick`` raises.  Raises if a token id was out of range or the pages ran out.
        """
        n, b = idx.shape[0], self.cache.max_batch
        if n > b:
            raise ValueError(f"{n} prompts, but the decoder has {b} rows")
        if max_new_tokens < 1:
            raise ValueError("max_new_tokens must be positive")
        longest = max(lengths) if lengths is not None else idx.shape[1]
        if longest + max_new_tokens - 1 > min(self.cfg.block_size, self.cache.capacity):
            raise ValueError("sequence length exceeds block_size or the cache's max_len")
        pick = (lambda z: z.argmax(dim=-1)) if pick is None else pick
        active = torch.zeros(b, dtype=torch.bool, device=self.device)
        active[:n] = True
        logits = self.prefill(idx, lengths=lengths)
        out = torch.empty(n, max_new_tokens, dtype=torch.int64, device=self.device)
        tokens = torch.zeros(b, dtype=torch.int64, device=self.device)
        try:
            for t in range(max_new_tokens):
                out[:, t] = pick(logits)
                if t + 1 < max_new_tokens:
                    tokens[:n] = out[:, t]
                    logits = self.step(tokens, active)[:n]
        finally:
            self.release(range(n))
        with torch.cuda.device(self.device):
            _lib.raise_on_device_status()
        return out
