"""Workloads of the 8-bit paged key-value cache operators: what a serving step and a prompt do with such a cache.

Four operators, each with a plain form in elementary torch operations (``own`` false) and the call that a
program makes of ``engpt_b200.kernels`` (``own`` true):

``write``      write_kv_pages_q8: finished k and v rows of a prompt are quantised into their cache slots
``append``     qkv_append_from_carried_q8: nGPT post-process of raw QKV rows at given positions; q is returned,
               k and v are quantised into their cache slots
``read``       read_kv_pages_q8: the keys and values of given cache slots as numbers again
``attention``  paged_sdpa_q8: one new token of every request attends to its cached keys and values

The cache is ``[pages, kv heads, page size, head_dim]`` in int8 or float8 e4m3, with one fp32 scale for each head and
each block of ``block`` tokens of a page, ``[pages, kv heads, page size / block]``; a value is ``code * scale``.
``write`` and ``append`` quantise all tokens that one call puts into a block together:

    need  = max(largest |x| of them, 2^-100) / top        (top: 127 for int8, 448 for e4m3)
    scale = need                  if one of them is the block's first token: the block starts anew
            max(scale, need)      otherwise; where that raises it, the other codes of the block become
                                  round(code * (scale before / scale))
    code  = round(x / scale)

They change the cache, which is held in 8 bits: what they return of it is the values that it stands for, read back
with ``read``, and the scales.
"""

import math

import torch

own = False

_BF16, _F32 = "bf16", "f32"
_DTYPES = {_BF16: torch.bfloat16, _F32: torch.float32}
_ESIZE = {_BF16: 2, _F32: 4}
_INT8, _E4M3 = "int8", "e4m3"
_CODES = {_INT8: torch.int8, _E4M3: torch.float8_e4m3fn}
_TOP = {_INT8: 127.0, _E4M3: 448.0}
_LEAST = 2.0 ** -100


# ------------------------------------------------------------------ cases
def listed():
    return [
        # k and v of 16 prompts, out of the packed [B, T, 3, H, Dh] buffer that the forward leaves
        {"name": "write prompts 16x2048", "op": "write", "batch": 16, "tokens": 2048, "heads": 16, "dim": 64,
         "page": 64, "block": 16, "dtype": _BF16, "codes": _INT8},
        # fp32 mode, short prompts, small heads
        {"name": "write f32 5x33", "op": "write", "batch": 5, "tokens": 33, "heads": 2, "dim": 16, "page": 16,
         "block": 16, "dtype": _F32, "codes": _E4M3},
        # the new tokens of 32 decoding requests of the 16-head, head_dim 64 model
        {"name": "append step 32", "op": "append", "batch": 32, "tokens": 1, "heads": 16, "dim": 64, "page": 64,
         "block": 16, "max_len": 2048, "dtype": _BF16, "codes": _INT8},
        # fp32 mode, the 4-head model, a small odd batch of short prompts
        {"name": "append f32 3x129", "op": "append", "batch": 3, "tokens": 129, "heads": 4, "dim": 64, "page": 16,
         "block": 8, "max_len": 129, "dtype": _F32, "codes": _INT8},
        # prompts of odd length, the long-context model (16 heads of 128), one scale for a whole page
        {"name": "append prompts 4x2047", "op": "append", "batch": 4, "tokens": 2047, "heads": 16, "dim": 128,
         "page": 64, "block": 64, "max_len": 2047, "dtype": _BF16, "codes": _E4M3},
        # fp32 mode, five requests of different length, padded to the longest
        {"name": "read f32 5 to 1021", "op": "read", "batch": 5, "heads": 4, "dim": 64, "page": 16, "block": 16,
         "max_len": 1021, "dtype": _F32, "codes": _E4M3},
        # the caches of 16 requests handed on, the 16-head, head_dim 64 model
        {"name": "read 16 to 2048", "op": "read", "batch": 16, "heads": 16, "dim": 64, "page": 64, "block": 16,
         "max_len": 2048, "dtype": _BF16, "codes": _INT8},
        # a single chat with little context, the 4-head model: latency
        {"name": "attention 1 of 257", "op": "attention", "batch": 1, "heads": 4, "kv_heads": 4, "dim": 64,
         "page": 16, "block": 16, "max_len": 257, "ragged": False, "dtype": _BF16, "codes": _INT8},
        # fp32 mode, five requests of different length
        {"name": "attention f32 5 to 1021", "op": "attention", "batch": 5, "heads": 4, "kv_heads": 4, "dim": 64,
         "page": 16, "block": 8, "max_len": 1021, "ragged": True, "dtype": _F32, "codes": _INT8},
        # one long document, the long-context model: the work has to be split over the cache's length
        {"name": "attention 1 of 8192", "op": "attention", "batch": 1, "heads": 16, "kv_heads": 16, "dim": 128,
         "page": 64, "block": 16, "max_len": 8192, "ragged": False, "dtype": _BF16, "codes": _INT8},
        # query heads that share kv heads, some long contexts
        {"name": "attention 8 to 8192 grouped", "op": "attention", "batch": 8, "heads": 32, "kv_heads": 4,
         "dim": 128, "page": 64, "block": 64, "max_len": 8192, "ragged": True, "dtype": _BF16, "codes": _E4M3},
        # a full server of the 16-head, head_dim 64 model, requests of every length
        {"name": "attention 64 to 4096", "op": "attention", "batch": 64, "heads": 16, "kv_heads": 16, "dim": 64,
         "page": 64, "block": 16, "max_len": 4096, "ragged": True, "dtype": _BF16, "codes": _INT8},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "append", "read", "attention", "attention"])
    page = rng.choice([8, 16, 32, 64, 128])
    block = rng.choice([b for b in (8, 16, 16, page) if b <= page])
    dtype = rng.choice([_BF16, _BF16, _F32])
    codes = rng.choice([_INT8, _INT8, _E4M3])
    common = {"page": page, "block": block, "dtype": dtype, "codes": codes}
    if op != "attention":
        heads, dim = rng.choice([(2, 16), (4, 64), (12, 64), (16, 64), (16, 128), (5, 80)])
        common.update(heads=heads, dim=dim)
    if op == "append":
        batch = _log(rng, 1, 64)
        room = 8188 * 2048 // (2 if dtype == _F32 else 1)
        tokens = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, room // (batch * heads * dim)))
        return {"op": op, "batch": batch, "tokens": tokens, "max_len": tokens + _log(rng, 1, 2048), **common}
    if op in ("write", "read"):
        batch = _log(rng, 1, 16)
        room = 16 * 2048 * 1024 // (2 if dtype == _F32 else 1)
        most = max(1, room // (batch * heads * dim))
        if op == "read":
            return {"op": op, "batch": batch, "max_len": _log(rng, 1, min(32768, most)), **common}
        return {"op": op, "batch": batch, "tokens": _log(rng, 1, most), **common}
    dim = rng.choice([16, 64, 64, 64, 80, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([g for g in (1, 1, 1, 2, 4, 8) if kv_heads * g <= 32])
    batch = _log(rng, 1, 64)
    # K and V elements at most what the largest listed case has
    most = 64 * 2048 * 16 * 64 // (2 if dtype == _F32 else 1) // (batch * kv_heads * dim)
    return {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "max_len": _log(rng, 1, max(1, min(32768, most))), "ragged": rng.random() < 0.7, **common}


# ------------------------------------------------------------------ sizes that follow from a case
def _up(n, page):
    return -(-n // page)


def _spread(batch, most):
    """Lengths of a mixed batch: from `most` down to 0, in equal steps (a single request has `most`)."""
    if batch == 1:
        return [most]
    return [most - (most * b) // (batch - 1) for b in range(batch)]


def _lengths(case):
    ragged = case["op"] == "read" or case["ragged"]
    return _spread(case["batch"], case["max_len"]) if ragged else [case["max_len"]] * case["batch"]


def work(case):
    op, es, block = case["op"], _ESIZE[case["dtype"]], case["block"]
    if op == "attention":
        total = sum(_lengths(case))
        d = case["dim"]
        pages = sum(_up(n, case["page"]) for n in _lengths(case))
        blocks = sum(_up(n, block) for n in _lengths(case))
        return {"bytes": 2 * total * case["kv_heads"] * d + 8 * blocks * case["kv_heads"]
                + 2 * es * case["batch"] * case["heads"] * d + 4 * (pages + case["batch"]),
                "flops": 4 * total * case["heads"] * d}
    heads, dim = case["heads"], case["dim"]
    row = heads * dim
    if op == "read":
        # slots and codes in, numbers out (zeros where a request has no token)
        rows = case["batch"] * case["max_len"]
        live = sum(_lengths(case))
        return {"bytes": 4 * rows + 2 * live * row + 8 * sum(_up(n, block) for n in _lengths(case)) * heads
                + 2 * es * rows * row, "flops": 2 * live * row}
    rows = case["batch"] * case["tokens"]
    blocks = case["batch"] * _up(case["tokens"], block)
    # the cache: codes and scales out; then the pages that hold them in, their numbers (16 bits) and scales out
    kept = case["batch"] * _up(case["tokens"], case["page"]) * case["page"]
    cache = 2 * rows * row + 8 * blocks * heads + 2 * kept * row * (1 + 2) + 4 * kept + 8 * kept // block * heads
    if op == "write":
        return {"bytes": 2 * es * rows * row + 4 * rows + cache, "flops": 3 * 2 * rows * row}
    # append: 3 rows in, q out; rho, position, slot and one rotary row of each token; about 9 operations an element
    return {"bytes": 4 * es * rows * row + 12 * rows + 4 * dim * min(rows, case["max_len"]) + 4 * row + cache,
            "flops": 9 * 3 * rows * row + 3 * 2 * rows * row}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _order(n, gen):
    return torch.randperm(n, generator=gen, device="cuda")


def _unit_rows(shape, gen):
    """Rows on the sphere, as the model's post-processed q and k (effective s_qk about 1)."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x = x / x.norm(dim=-1, keepdim=True)
    s = 1.0 + 0.1 * torch.randn(shape[-1], generator=gen, device="cuda")
    return x * s


def prepare(case, seed):
    gen = _gen(seed)
    return {"write": _prepare_write, "append": _prepare_append, "read": _prepare_read,
            "attention": _prepare_attention}[case["op"]](case, gen)


def _cache(case, pool, heads, gen):
    """A pool in use: codes and scales of rows of this or of former requests, in one buffer (codes, then scales)."""
    page, dim, block = case["page"], case["dim"], case["block"]
    top, kind = _TOP[case["codes"]], _CODES[case["codes"]]
    shape = (pool, heads, page, dim)
    n, blocks = pool * heads * page * dim, pool * heads * (page // block)
    scales_at = -(-2 * n // 16) * 16
    state = torch.zeros(scales_at + 8 * blocks, dtype=torch.uint8, device="cuda")
    views = _cache_views(state, case, pool, heads)
    for i in range(2):
        # (values of a token differ in size from token to token)
        x = _unit_rows(shape, gen) if i == 0 else torch.randn(shape, generator=gen, device="cuda") * torch.exp(
            0.3 * torch.randn(shape[:3] + (1,), generator=gen, device="cuda"))
        x = x.view(pool, heads, page // block, block, dim)
        scale = x.abs().amax((-2, -1)) / top
        x = x / scale[..., None, None]
        views[i].copy_((x.round() if kind == torch.int8 else x).to(kind).view(shape))
        views[2 + i].copy_(scale)
    return state


def _cache_views(state, case, pool, heads):
    page, dim, block, kind = case["page"], case["dim"], case["block"], _CODES[case["codes"]]
    n, blocks = pool * heads * page * dim, pool * heads * (page // block)
    scales_at = -(-2 * n // 16) * 16
    codes = [state[i * n:(i + 1) * n].view(kind).view(pool, heads, page, dim) for i in range(2)]
    scales = [state[scales_at + 4 * i * blocks:scales_at + 4 * (i + 1) * blocks].view(torch.float32).view(
        pool, heads, page // block) for i in range(2)]
    return (*codes, *scales)


def _slots_of(first, tokens, page, gen, spare):
    """Pages in random order for requests that each write `tokens` tokens from position `first[b]` on."""
    batch = len(first)
    touched = [_up(f + tokens, page) - f // page for f in first]
    pool = batch * _up(tokens + page - 1, page) + spare      # (of the size that any first positions ask for)
    pages = _order(pool, gen)
    pos = torch.tensor(first, device="cuda")[:, None] + torch.arange(tokens, device="cuda")[None, :]
    start = torch.tensor([sum(touched[:b]) for b in range(batch)], device="cuda")[:, None]
    base = torch.tensor([f // page for f in first], device="cuda")[:, None]
    slots = pages[start + pos // page - base] * page + pos % page
    return slots.to(torch.int32), pos.to(torch.int32), pool


def _all_slots(pool, page):
    return torch.arange(pool * page, dtype=torch.int32, device="cuda")


def _prepare_write(case, gen):
    batch, tokens, heads, dim, page = (case[k] for k in ("batch", "tokens", "heads", "dim", "page"))
    slots, _, pool = _slots_of([0] * batch, tokens, page, gen, 1)
    # prompts of different length, padded to the longest: the last tokens of every other one have no slot
    for b in range(1, batch, 2):
        slots[b, tokens - tokens // 8:] = -1
    packed = torch.randn((batch, tokens, 3, heads, dim), generator=gen, device="cuda")
    packed *= torch.exp(0.3 * torch.randn((batch, tokens, 3, 1, 1), generator=gen, device="cuda"))
    packed = packed.to(_DTYPES[case["dtype"]])
    return {"op": "write", "case": case, "k": packed[:, :, 1], "v": packed[:, :, 2], "slots": slots, "pool": pool,
            "state": _cache(case, pool, heads, gen), "all": _all_slots(pool, page)}


def _prepare_append(case, gen):
    batch, tokens, heads, dim, page = (case[k] for k in ("batch", "tokens", "heads", "dim", "page"))
    dtype = _DTYPES[case["dtype"]]
    room = case["max_len"] - tokens
    first = torch.randint(0, room + 1, (batch,), generator=gen, device="cuda").tolist()
    slots, pos, pool = _slots_of(first, tokens, page, gen, 1)
    # the rows of a unit-norm projection of a carried state with radius rho
    rho = torch.exp(torch.randn((batch, tokens), generator=gen, device="cuda"))
    qkv = torch.randn((batch, tokens, 3, heads, dim), generator=gen, device="cuda") * rho[:, :, None, None, None]
    half = dim // 2
    inv = 10000.0 ** (-2.0 * torch.arange(half, dtype=torch.float64, device="cuda") / (2 * half))
    ang = torch.arange(case["max_len"], dtype=torch.float64, device="cuda")[:, None] * inv
    s_qk = 1.0 + 0.1 * torch.randn((heads, dim), generator=gen, device="cuda")
    initial = _cache(case, pool, heads, gen)
    return {"op": "append", "case": case, "qkv": qkv.to(dtype), "rho": rho, "cos": ang.cos().float(),
            "sin": ang.sin().float(), "s_qk": s_qk, "eps": 1e-6, "pos": pos, "slots": slots, "pool": pool,
            # a request that goes on finds its last block partly filled: each pass starts from that
            "initial": initial if room else None, "state": initial.clone(), "all": _all_slots(pool, page)}


def _tables(case, gen):
    """Lengths in random order and a block table of pages in random order."""
    batch, page = case["batch"], case["page"]
    lens = _lengths(case)
    lens = [lens[i] for i in _order(batch, gen).tolist()]
    width = _up(case["max_len"], page) + 1
    pool = sum(_up(n, page) for n in lens) + 1
    pages = _order(pool, gen).to(torch.int32)
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    have = (lengths + page - 1) // page
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    col = torch.arange(width, device="cuda")[None, :]
    held = col < have[:, None]
    table[held] = pages[((torch.cumsum(have, 0) - have)[:, None] + col)[held]]
    return lengths, table, pool


def _prepare_read(case, gen):
    lengths, table, pool = _tables(case, gen)
    page = case["page"]
    pos = torch.arange(case["max_len"], device="cuda")[None, :]
    slots = torch.where(pos < lengths[:, None], table[:, pos[0] // page] * page + pos % page, -1).to(torch.int32)
    return {"op": "read", "case": case, "slots": slots, "pool": pool,
            "state": _cache(case, pool, case["heads"], gen)}


def _prepare_attention(case, gen):
    lengths, table, pool = _tables(case, gen)
    q = _unit_rows((case["batch"], case["heads"], case["dim"]), gen).to(_DTYPES[case["dtype"]])
    return {"op": "attention", "case": case, "q": q, "table": table, "lengths": lengths, "pool": pool,
            "state": _cache(case, pool, case["kv_heads"], gen), "scale": math.sqrt(case["dim"])}


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _RUN_OWN[state["op"]](state)
    return _RUN_PLAIN[state["op"]](state)


def _views(st):
    case = st["case"]
    return _cache_views(st["state"], case, st["pool"], case["kv_heads"] if st["op"] == "attention" else case["heads"])


def _own_write(st):
    from engpt_b200 import kernels as K
    cache = _views(st)
    K.write_kv_pages_q8(st["k"], st["v"], st["slots"], *cache)
    return K.read_kv_pages_q8(st["all"], *cache, dtype=torch.bfloat16), cache[2], cache[3]


def _own_append(st):
    from engpt_b200 import kernels as K
    if st["initial"] is not None:
        st["state"].copy_(st["initial"])
    cache = _views(st)
    q = K.qkv_append_from_carried_q8(st["qkv"], st["rho"], st["cos"], st["sin"], st["s_qk"], st["eps"], st["pos"],
                                     st["slots"], *cache)
    return q, K.read_kv_pages_q8(st["all"], *cache, dtype=torch.bfloat16), cache[2], cache[3]


def _own_read(st):
    from engpt_b200 import kernels as K
    return K.read_kv_pages_q8(st["slots"], *_views(st), dtype=_DTYPES[st["case"]["dtype"]])


def _own_attention(st):
    from engpt_b200 import kernels as K
    return K.paged_sdpa_q8(st["q"], *_views(st), st["table"], st["lengths"], scale=st["scale"])


def _plain_codes(x, kind):
    """Numbers within the codes' range rounded to them, as fp32."""
    if kind == torch.int8:
        return x.round().clamp(-127.0, 127.0)
    return x.clamp(-448.0, 448.0).to(kind).float()


def _plain_store(x, slots, codes, scales):
    """Rows x [n, H, Dh] (fp32) into the pool, as the text above says."""
    pool, heads, page, dim = codes.shape
    per_page = scales.shape[2]
    block, kind = page // per_page, codes.dtype
    top = 127.0 if kind == torch.int8 else 448.0
    live = slots >= 0
    at, x = slots[live].long(), x[live]
    of = at // block                                                     # block in the pool, in order of its slots
    old = scales.permute(0, 2, 1).reshape(-1, heads)
    largest = torch.zeros_like(old).index_reduce_(0, of, x.abs().amax(-1), "amax")
    written = torch.zeros(old.shape[0], dtype=torch.bool, device=x.device)
    anew = written.clone()
    written[of] = True
    anew[of[at % block == 0]] = True
    need = largest.clamp(min=_LEAST) / top
    new = torch.where(anew[:, None], need, torch.where(written[:, None], torch.maximum(old, need), old))
    ratio = torch.where((written & ~anew)[:, None], old / new, 1.0)
    held = codes.permute(0, 2, 1, 3).reshape(-1, block, heads, dim).float()   # [blocks, tokens, H, Dh]
    held = _plain_codes(held * ratio[:, None, :, None], kind).reshape(-1, heads, dim)
    held[at] = _plain_codes(x * (torch.ones_like(new) / new)[of][:, :, None], kind)
    codes.copy_(held.view(pool, page, heads, dim).permute(0, 2, 1, 3).to(kind))
    scales.copy_(new.view(pool, per_page, heads).permute(0, 2, 1))


def _plain_values(codes, scales):
    """The pool's numbers [slots, H, Dh] in fp32."""
    pool, heads, page, dim = codes.shape
    x = codes.float().view(pool, heads, scales.shape[2], -1, dim) * scales[..., None, None]
    return x.view(pool, heads, page, dim).permute(0, 2, 1, 3).reshape(-1, heads, dim)


def _plain_pools(cache):
    return tuple(_plain_values(cache[i], cache[2 + i]).to(torch.bfloat16) for i in range(2)), cache[2], cache[3]


def _plain_write(st):
    cache = _views(st)
    slots = st["slots"].view(-1)
    _plain_store(st["k"].float().flatten(0, 1), slots, cache[0], cache[2])
    _plain_store(st["v"].float().flatten(0, 1), slots, cache[1], cache[3])
    return _plain_pools(cache)


def _plain_append(st):
    if st["initial"] is not None:
        st["state"].copy_(st["initial"])
    cache = _views(st)
    qkv = st["qkv"].float()
    pos, slots = st["pos"].long(), st["slots"].view(-1)
    rho = st["rho"][:, :, None, None]
    c, s = st["cos"][pos][:, :, None, :], st["sin"][pos][:, :, None, :]

    def rotate(x):
        norm = torch.maximum(x.pow(2).sum(-1, keepdim=True).sqrt(), rho * st["eps"])
        half = c.shape[-1]
        even, odd = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y = torch.stack((even * c - odd * s, even * s + odd * c), dim=-1).flatten(-2)
        return y / norm * st["s_qk"]

    _plain_store(rotate(qkv[:, :, 1]).flatten(0, 1), slots, cache[0], cache[2])
    _plain_store((qkv[:, :, 2] / rho).flatten(0, 1), slots, cache[1], cache[3])
    return rotate(qkv[:, :, 0]).to(st["qkv"].dtype), *_plain_pools(cache)


def _plain_read(st):
    cache = _views(st)
    slots = st["slots"]
    page, dtype = cache[0].shape[2], _DTYPES[st["case"]["dtype"]]
    there = (slots >= 0)[..., None, None]
    at = slots.clamp(min=0).long()
    in_block = at % page // (page // cache[2].shape[2])

    def values(codes, scales):
        x = codes.view(torch.uint8)[at // page, :, at % page].view(codes.dtype).float()
        return torch.where(there, x * scales[at // page, :, in_block][..., None], 0.0).to(dtype)

    return values(cache[0], cache[2]), values(cache[1], cache[3])


def _plain_attention(st):
    k_codes, v_codes, k_scales, v_scales = _views(st)
    q, table, lengths = st["q"].float(), st["table"].clamp(min=0).long(), st["lengths"]
    batch, heads, dim = q.shape
    _, kv_heads, page, _ = k_codes.shape

    def gather(codes, scales):
        x = codes.view(torch.uint8)[table].view(codes.dtype).float()
        x = x.view(*x.shape[:3], scales.shape[2], -1, dim) * scales[table][..., None, None]
        return x.view(batch, -1, kv_heads, page, dim).permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, -1, dim)

    k, v = gather(k_codes, k_scales), gather(v_codes, v_scales)
    there = torch.arange(k.shape[2], device=q.device)[None, :] < lengths[:, None]
    s = q.view(batch, kv_heads, heads // kv_heads, dim) @ k.transpose(-1, -2) * st["scale"]
    s = s.masked_fill(~there[:, None, None, :], float("-inf"))
    m = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(s - m)
    o = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.reshape(batch, heads, dim).to(st["q"].dtype)


_RUN_OWN = {"write": _own_write, "append": _own_append, "read": _own_read, "attention": _own_attention}
_RUN_PLAIN = {"write": _plain_write, "append": _plain_append, "read": _plain_read, "attention": _plain_attention}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"write": _exact_write, "append": _exact_append, "read": _exact_read,
            "attention": _exact_attention}[case["op"]](st)


def _exact_codes(x, kind):
    """64-bit numbers to the nearest code (even ones in the middle)."""
    if kind == torch.int8:
        return torch.round(x).clamp(-127, 127)
    # 3 bits behind the leading one, down to 2^-6, and steps of 2^-9 below that
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_store(x, slots, codes, scales):
    """Block by block (all at once, in the order of the slots): [blocks, block, H, Dh] of codes and of rows."""
    pool, heads, page, dim = codes.shape
    per_page, kind = scales.shape[2], codes.dtype
    block = page // per_page
    n = pool * per_page
    held = codes.double().transpose(1, 2).reshape(n, block, heads, dim)
    rows = torch.full(held.shape, float("nan"), dtype=torch.float64, device=held.device)
    keep = torch.nonzero(slots >= 0)[:, 0]
    rows.view(-1, heads, dim).index_copy_(0, slots[keep].long(), x[keep])
    fresh = ~torch.isnan(rows[:, :, :1, :1])                             # [blocks, block, 1, 1]: written by this call
    old = scales.double().transpose(1, 2).reshape(n, 1, heads, 1)
    largest = torch.where(fresh, rows, 0.0).abs().amax((1, 3), keepdim=True)
    need = largest.clamp(min=2.0 ** -100) / (127 if kind == torch.int8 else 448)
    first = fresh[:, :1]
    new = torch.where(first, need, torch.maximum(old, need))
    new = torch.where(fresh.any(1, keepdim=True), new, old)
    moved = _exact_codes(held * torch.where(first, 1.0, old / new), kind)
    out = torch.where(fresh, _exact_codes(rows / new, kind), moved)
    values = (out * new).reshape(pool * page, heads, dim)
    return values, new.reshape(pool, per_page, heads).transpose(1, 2)


def _exact_both(k, v, st, cache):
    slots = st["slots"].view(-1)
    k, ks = _exact_store(k.reshape(-1, *k.shape[2:]), slots, cache[0], cache[2])
    v, vs = _exact_store(v.reshape(-1, *v.shape[2:]), slots, cache[1], cache[3])
    return (k, v), ks, vs


def _exact_write(st):
    return _exact_both(st["k"].double(), st["v"].double(), st, _views(st))


def _exact_append(st):
    x, rho = st["qkv"].double(), st["rho"].double()[:, :, None, None]
    half = st["cos"].shape[1]
    turn = torch.complex(st["cos"].double(), st["sin"].double())[st["pos"].long()][:, :, None, :]
    out = []
    for part in (0, 1):
        row = x[:, :, part]
        den = torch.linalg.vector_norm(row, dim=-1, keepdim=True)
        den = torch.where(den > rho * st["eps"], den, rho * st["eps"])
        pair = torch.view_as_complex(row[..., :2 * half].reshape(*row.shape[:-1], half, 2).contiguous())
        row = torch.view_as_real(pair * turn).flatten(-2)
        out.append(row * st["s_qk"].double() / den)
    return out[0], *_exact_both(out[1], x[:, :, 2] / rho, st, _views(st))


def _exact_read(st):
    cache = _views(st)
    page = cache[0].shape[2]
    slots = st["slots"].view(-1)
    keep = torch.nonzero(slots >= 0)[:, 0]
    at = slots[keep].long()
    out = []
    for codes, scales in ((cache[0], cache[2]), (cache[1], cache[3])):
        wide = scales.double().repeat_interleave(page // scales.shape[2], dim=2)[..., None]   # a scale for each slot
        x = torch.zeros(slots.shape[0], codes.shape[1], codes.shape[3], dtype=torch.float64, device="cuda")
        for h in range(codes.shape[1]):
            flat = (codes[:, h].double() * wide[:, h]).reshape(-1, codes.shape[3])
            x[keep, h] = flat[at]
        out.append(x.view(*st["slots"].shape, codes.shape[1], codes.shape[3]))
    return tuple(out)


def _exact_attention(st):
    k_codes, v_codes, k_scales, v_scales = _views(st)
    q = st["q"].double()
    batch, heads, dim = q.shape
    kv_heads, page = k_codes.shape[1], k_codes.shape[2]
    block = page // k_scales.shape[2]
    out = torch.zeros_like(q)
    for b, n in enumerate(st["lengths"].tolist()):
        if n == 0:
            continue
        pages = st["table"][b, :_up(n, page)].long()
        for g in range(kv_heads):
            # (an index of a strided pool: codes are taken page by page as bytes)
            k = k_codes.view(torch.uint8)[pages, g].view(k_codes.dtype).double().reshape(-1, dim)[:n]
            v = v_codes.view(torch.uint8)[pages, g].view(v_codes.dtype).double().reshape(-1, dim)[:n]
            ks = k_scales[pages, g].double().reshape(-1).repeat_interleave(block)[:n]
            vs = v_scales[pages, g].double().reshape(-1).repeat_interleave(block)[:n]
            heads_of = slice(g * heads // kv_heads, (g + 1) * heads // kv_heads)
            p = torch.softmax((q[b, heads_of] @ k.T) * ks * st["scale"], dim=-1)
            out[b, heads_of] = (p * vs) @ v
    return out
