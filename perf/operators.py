"""Workloads of the paged key-value cache operators: what a serving step and a prompt do with the cache.

Four operators, each with a plain form in elementary torch operations (``own`` false) and the call that a
program makes of ``engpt_b200.kernels`` (``own`` true):

``tables``     advance_block_tables: finished requests give their pages back, every request gets the pages that
               its new tokens need, and the tokens' cache slots and positions are written
``append``     qkv_append_from_carried: nGPT post-process of raw QKV rows at given positions; q is returned,
               k and v go to their cache slots
``write``      write_kv_pages: finished k and v rows of a prompt go to their cache slots
``attention``  paged_sdpa: one new token of every request attends to its cached keys and values

The cache is ``[pages, kv heads, page size, head_dim]``; a request's block table row lists its pages and a
slot is ``page * page_size + offset``.
"""

import math

import torch

own = False

_BF16, _F32 = "bf16", "f32"
_DTYPES = {_BF16: torch.bfloat16, _F32: torch.float32}
_ESIZE = {_BF16: 2, _F32: 4}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding step of a busy server: 64 requests, two thousand tokens of context at most, one new token
        # each; every eighth request has finished and its row is taken by the next one
        {"name": "tables step 64", "op": "tables", "batch": 64, "page": 16, "max_len": 2048, "max_new": 1,
         "every": 8},
        # a thousand rows (odd), long contexts
        {"name": "tables step 999", "op": "tables", "batch": 999, "page": 16, "max_len": 8192, "max_new": 1,
         "every": 5},
        # 32 prompts of up to 2048 tokens are taken in at once
        {"name": "tables prompts 32x2048", "op": "tables", "batch": 32, "page": 64, "max_len": 0, "max_new": 2048,
         "every": 0},
        # the new tokens of 32 decoding requests of the 16-head, head_dim 64 model
        {"name": "append step 32", "op": "append", "batch": 32, "tokens": 1, "heads": 16, "dim": 64, "page": 16,
         "max_len": 2048, "dtype": _BF16},
        # fp32 mode, the 4-head model, a small odd batch of short prompts
        {"name": "append f32 3x129", "op": "append", "batch": 3, "tokens": 129, "heads": 4, "dim": 64, "page": 16,
         "max_len": 129, "dtype": _F32},
        # prompts of odd length, the long-context model (16 heads of 128)
        {"name": "append prompts 4x2047", "op": "append", "batch": 4, "tokens": 2047, "heads": 16, "dim": 128,
         "page": 64, "max_len": 2047, "dtype": _BF16},
        # k and v of 16 prompts, out of the packed [B, T, 3, H, Dh] buffer that the forward leaves
        {"name": "write prompts 16x2048", "op": "write", "batch": 16, "tokens": 2048, "heads": 16, "dim": 64,
         "page": 16, "dtype": _BF16},
        # fp32 mode, short prompts, small heads
        {"name": "write f32 5x33", "op": "write", "batch": 5, "tokens": 33, "heads": 2, "dim": 16, "page": 16,
         "dtype": _F32},
        # a single chat with little context, the 4-head model: latency
        {"name": "attention 1 of 257", "op": "attention", "batch": 1, "heads": 4, "kv_heads": 4, "dim": 64,
         "page": 16, "max_len": 257, "ragged": False, "dtype": _BF16},
        # fp32 mode, five requests of different length
        {"name": "attention f32 5 to 1021", "op": "attention", "batch": 5, "heads": 4, "kv_heads": 4, "dim": 64,
         "page": 16, "max_len": 1021, "ragged": True, "dtype": _F32},
        # one long document, the long-context model: the work has to be split over the cache's length
        {"name": "attention 1 of 8192", "op": "attention", "batch": 1, "heads": 16, "kv_heads": 16, "dim": 128,
         "page": 64, "max_len": 8192, "ragged": False, "dtype": _BF16},
        # a full server of the 16-head, head_dim 64 model, requests of every length
        {"name": "attention 64 to 4096", "op": "attention", "batch": 64, "heads": 16, "kv_heads": 16, "dim": 64,
         "page": 16, "max_len": 4096, "ragged": True, "dtype": _BF16},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tables", "append", "write", "attention", "attention"])
    page = rng.choice([8, 16, 32, 64, 128])
    dtype = rng.choice([_BF16, _BF16, _F32])
    if op == "tables":
        if rng.random() < 0.6:
            return {"op": op, "batch": _log(rng, 1, 999), "page": page, "max_len": _log(rng, 64, 8192),
                    "max_new": 1, "every": rng.choice([0, 3, 8])}
        batch = _log(rng, 1, 64)
        return {"op": op, "batch": batch, "page": page, "max_len": rng.choice([0, 1000]),
                "max_new": _log(rng, 2, min(2048, 65536 // batch)), "every": rng.choice([0, 4])}
    if op == "append":
        heads, dim = rng.choice([(2, 16), (4, 64), (12, 64), (16, 64), (16, 128), (5, 80)])
        batch = _log(rng, 1, 64)
        room = 8188 * 2048 // (2 if dtype == _F32 else 1)
        tokens = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, room // (batch * heads * dim)))
        return {"op": op, "batch": batch, "tokens": tokens, "heads": heads, "dim": dim, "page": page,
                "max_len": tokens + _log(rng, 1, 2048), "dtype": dtype}
    if op == "write":
        heads, dim = rng.choice([(2, 16), (4, 64), (12, 64), (16, 64), (16, 128), (5, 80)])
        batch = _log(rng, 1, 16)
        room = 16 * 2048 * 1024 // (2 if dtype == _F32 else 1)
        return {"op": op, "batch": batch, "tokens": _log(rng, 1, max(1, room // (batch * heads * dim))),
                "heads": heads, "dim": dim, "page": page, "dtype": dtype}
    dim = rng.choice([16, 64, 64, 64, 80, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([g for g in (1, 1, 1, 2, 4, 8) if kv_heads * g <= 32])
    batch = _log(rng, 1, 64)
    # K and V elements at most what the largest listed case has
    most = 64 * 2048 * 16 * 64 // (2 if dtype == _F32 else 1) // (batch * kv_heads * dim)
    return {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "max_len": _log(rng, 1, max(1, min(32768, most))), "ragged": rng.random() < 0.7, "dtype": dtype}


# ------------------------------------------------------------------ sizes that follow from a case
def _pages(n, page):
    return -(-n // page)


def _spread(batch, most):
    """Lengths of a mixed batch: from `most` down to 0, in equal steps (a single request has `most`)."""
    if batch == 1:
        return [most]
    return [most - (most * b) // (batch - 1) for b in range(batch)]


def _table_counts(case):
    """Per request: tokens in the cache before, finished or not, new tokens."""
    batch, every = case["batch"], case["every"]
    old = _spread(batch, case["max_len"])
    done = [bool(every) and b % every == every // 2 for b in range(batch)]
    if case["max_new"] == 1:
        new = [1] * batch
    else:
        new = [max(1, n) for n in _spread(batch, case["max_new"])]
    return old, done, new


def _lengths(case):
    return _spread(case["batch"], case["max_len"]) if case["ragged"] else [case["max_len"]] * case["batch"]


def work(case):
    op = case["op"]
    if op == "tables":
        old, done, new = _table_counts(case)
        page = case["page"]
        tokens = case["batch"] * case["max_new"]
        freed = sum(_pages(n, page) for n, d in zip(old, done) if d)
        taken = sum(_pages((0 if d else n) + t, page) - _pages(0 if d else n, page)
                    for n, d, t in zip(old, done, new))
        # lengths in and out, new token counts, finished marks; freed pages from the table to the free list, new
        # ones from the free list to the table; slots and positions out, and one table entry for each page that
        # new tokens fall into
        touched = sum(_pages((0 if d else n) + t, page) - (0 if d else n) // page for n, d, t in zip(old, done, new))
        return {"bytes": 4 * (4 * case["batch"] + 2 * freed + 2 * taken + 2 * tokens + touched + 2), "flops": 0}
    if op == "attention":
        total = sum(_lengths(case))
        es = _ESIZE[case["dtype"]]
        d = case["dim"]
        pages = sum(_pages(n, case["page"]) for n in _lengths(case))
        return {"bytes": 2 * es * total * case["kv_heads"] * d + 2 * es * case["batch"] * case["heads"] * d
                + 4 * (pages + case["batch"]),
                "flops": 4 * total * case["heads"] * d}
    rows = case["batch"] * case["tokens"]
    width = rows * case["heads"] * case["dim"] * _ESIZE[case["dtype"]]
    if op == "write":
        return {"bytes": 4 * width + 4 * rows, "flops": 0}
    # append: 3 rows in, 3 out; rho, position, slot and one rotary row of each token; about 9 operations an element
    return {"bytes": 6 * width + 12 * rows + 4 * case["dim"] * min(rows, case["max_len"])
            + 4 * case["heads"] * case["dim"],
            "flops": 9 * 3 * rows * case["heads"] * case["dim"]}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _order(n, gen):
    return torch.randperm(n, generator=gen, device="cuda")


def _unit_rows(shape, gen, dtype):
    """Rows on the sphere, as the model's post-processed q and k (effective s_qk about 1)."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x = x / x.norm(dim=-1, keepdim=True)
    s = 1.0 + 0.1 * torch.randn(shape[-1], generator=gen, device="cuda")
    return (x * s).to(dtype)


def prepare(case, seed):
    gen = _gen(seed)
    return {"tables": _prepare_tables, "append": _prepare_append, "write": _prepare_write,
            "attention": _prepare_attention}[case["op"]](case, gen)


def _prepare_tables(case, gen):
    batch, page = case["batch"], case["page"]
    old, done, new = _table_counts(case)
    perm = _order(batch, gen)
    old = torch.tensor(old, dtype=torch.int32, device="cuda")[perm]
    done = torch.tensor(done, device="cuda")[perm]
    new = torch.tensor(new, dtype=torch.int32, device="cuda")[perm]
    width = _pages(case["max_len"] + case["max_new"], page)
    have = (old + page - 1) // page
    n_have = int(have.sum())
    pool = n_have + _pages(int(new.sum()), page) + 2 * batch + 1
    pages = _order(pool, gen).to(torch.int32)
    # one buffer holds the allocator's state: lengths, the number of free pages, the free pages, the block table
    state = torch.empty(batch + 1 + pool + batch * width, dtype=torch.int32, device="cuda")
    lengths, count, free, table = _table_views(state, batch, pool, width)
    lengths.copy_(old)
    count.fill_(pool - n_have)
    free.fill_(-1)
    free[:pool - n_have] = pages[n_have:]
    table.fill_(-1)
    col = torch.arange(width, device="cuda")[None, :]
    held = col < have[:, None]
    start = torch.cumsum(have, 0) - have
    table[held] = pages[(start[:, None] + col)[held]]
    return {"op": "tables", "case": case, "initial": state, "state": state.clone(), "new": new,
            "done": done if case["every"] else None, "pool": pool, "width": width}


def _table_views(state, batch, pool, width):
    return (state[:batch], state[batch:batch + 1], state[batch + 1:batch + 1 + pool],
            state[batch + 1 + pool:].view(batch, width))


def _cache(pool, heads, page, dim, gen, dtype):
    """A pool in use: every page holds rows of this or of former requests."""
    return (_unit_rows((pool, heads, page, dim), gen, dtype),
            torch.randn((pool, heads, page, dim), generator=gen, device="cuda").to(dtype))


def _slots_of(first, tokens, page, gen, spare):
    """Pages in random order for requests that each write `tokens` tokens from position `first[b]` on."""
    batch = len(first)
    touched = [_pages(f + tokens, page) - f // page for f in first]
    pool = sum(touched) + spare
    pages = _order(pool, gen)
    pos = torch.tensor(first, device="cuda")[:, None] + torch.arange(tokens, device="cuda")[None, :]
    start = torch.tensor([sum(touched[:b]) for b in range(batch)], device="cuda")[:, None]
    base = torch.tensor([f // page for f in first], device="cuda")[:, None]
    slots = pages[start + pos // page - base] * page + pos % page
    return slots.to(torch.int32), pos.to(torch.int32), pool


def _prepare_append(case, gen):
    batch, tokens, heads, dim, page = (case[k] for k in ("batch", "tokens", "heads", "dim", "page"))
    dtype = _DTYPES[case["dtype"]]
    room = case["max_len"] - tokens
    first = torch.randint(0, room + 1, (batch,), generator=gen, device="cuda").tolist()
    slots, pos, pool = _slots_of(first, tokens, page, gen, 3)
    # the rows of a unit-norm projection of a carried state with radius rho
    rho = torch.exp(torch.randn((batch, tokens), generator=gen, device="cuda"))
    qkv = torch.randn((batch, tokens, 3, heads, dim), generator=gen, device="cuda") * (rho / math.sqrt(dim))[
        :, :, None, None, None]
    half = dim // 2
    inv = 10000.0 ** (-2.0 * torch.arange(half, dtype=torch.float64, device="cuda") / (2 * half))
    ang = torch.arange(case["max_len"], dtype=torch.float64, device="cuda")[:, None] * inv
    k_pages, v_pages = _cache(pool, heads, page, dim, gen, dtype)
    s_qk = 1.0 + 0.1 * torch.randn((heads, dim), generator=gen, device="cuda")
    return {"op": "append", "case": case, "qkv": qkv.to(dtype), "rho": rho, "cos": ang.cos().float(),
            "sin": ang.sin().float(), "s_qk": s_qk, "eps": 1e-6, "pos": pos, "slots": slots, "k_pages": k_pages,
            "v_pages": v_pages}


def _prepare_write(case, gen):
    batch, tokens, heads, dim, page = (case[k] for k in ("batch", "tokens", "heads", "dim", "page"))
    dtype = _DTYPES[case["dtype"]]
    slots, _, pool = _slots_of([0] * batch, tokens, page, gen, 3)
    # prompts of different length, padded to the longest: the last tokens of every other one have no slot
    for b in range(1, batch, 2):
        slots[b, tokens - tokens // 8:] = -1
    packed = torch.randn((batch, tokens, 3, heads, dim), generator=gen, device="cuda").to(dtype)
    k_pages, v_pages = _cache(pool, heads, page, dim, gen, dtype)
    return {"op": "write", "case": case, "k": packed[:, :, 1], "v": packed[:, :, 2], "slots": slots,
            "k_pages": k_pages, "v_pages": v_pages}


def _prepare_attention(case, gen):
    batch, heads, kv_heads, dim, page = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "page"))
    dtype = _DTYPES[case["dtype"]]
    lens = _lengths(case)
    lens = [lens[i] for i in _order(batch, gen).tolist()]
    width = _pages(case["max_len"], page) + 1
    pool = sum(_pages(n, page) for n in lens) + 3
    pages = _order(pool, gen).to(torch.int32)
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    have = (lengths + page - 1) // page
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    col = torch.arange(width, device="cuda")[None, :]
    held = col < have[:, None]
    table[held] = pages[((torch.cumsum(have, 0) - have)[:, None] + col)[held]]
    k_pages, v_pages = _cache(pool, kv_heads, page, dim, gen, dtype)
    q = _unit_rows((batch, heads, dim), gen, dtype)
    return {"op": "attention", "case": case, "q": q, "k_pages": k_pages, "v_pages": v_pages, "table": table,
            "lengths": lengths, "scale": math.sqrt(dim)}


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _RUN_OWN[state["op"]](state)
    return _RUN_PLAIN[state["op"]](state)


def _own_tables(st):
    from engpt_b200 import kernels as K
    case = st["case"]
    st["state"].copy_(st["initial"])
    lengths, count, free, table = _table_views(st["state"], case["batch"], st["pool"], st["width"])
    slots, pos = K.advance_block_tables(lengths, st["new"], table, free, count, page_size=case["page"],
                                        max_new=case["max_new"], finished=st["done"])
    return slots, pos, lengths, count, free, table


def _own_append(st):
    from engpt_b200 import kernels as K
    q = K.qkv_append_from_carried(st["qkv"], st["rho"], st["cos"], st["sin"], st["s_qk"], st["eps"], st["pos"],
                                  st["slots"], st["k_pages"], st["v_pages"])
    return q, st["k_pages"], st["v_pages"]


def _own_write(st):
    from engpt_b200 import kernels as K
    K.write_kv_pages(st["k"], st["v"], st["slots"], st["k_pages"], st["v_pages"])
    return st["k_pages"], st["v_pages"]


def _own_attention(st):
    from engpt_b200 import kernels as K
    return K.paged_sdpa(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lengths"], scale=st["scale"])


def _plain_tables(st):
    case = st["case"]
    page, max_new = case["page"], case["max_new"]
    st["state"].copy_(st["initial"])
    lengths, count, free, table = _table_views(st["state"], case["batch"], st["pool"], st["width"])
    width = st["width"]
    col = torch.arange(width, device=table.device)[None, :]
    # finished requests push their pages on the free list, request by request
    if st["done"] is not None:
        held = (lengths + page - 1) // page * st["done"]
        at = (count + torch.cumsum(held, 0) - held)[:, None] + col
        mine = col < held[:, None]
        free[at[mine]] = table[mine]
        count += held.sum()
        lengths.masked_fill_(st["done"], 0)
    # new tokens pop pages from the end of the free list, request by request
    have = (lengths + page - 1) // page
    need = (lengths + st["new"] + page - 1) // page - have
    before = torch.cumsum(need, 0) - need
    mine = (col >= have[:, None]) & (col < (have + need)[:, None])
    table[mine] = free[(count - 1 - (before[:, None] + col - have[:, None]))[mine]]
    count -= need.sum()
    # slots and positions of the new tokens
    i = torch.arange(max_new, device=table.device)[None, :]
    live = i < st["new"][:, None]
    pos = torch.where(live, lengths[:, None] + i, 0).to(torch.int32)
    entry = torch.gather(table, 1, (pos // page).long())
    slots = torch.where(live, entry * page + pos % page, -1).to(torch.int32)
    lengths += st["new"]
    return slots, pos, lengths, count, free, table


def _plain_append(st):
    qkv = st["qkv"].float()
    dtype = st["qkv"].dtype
    pos = st["pos"].long()
    rho = st["rho"][:, :, None, None]
    c, s = st["cos"][pos][:, :, None, :], st["sin"][pos][:, :, None, :]

    def rotate(x):
        norm = torch.maximum(x.pow(2).sum(-1, keepdim=True).sqrt(), rho * st["eps"])
        half = c.shape[-1]
        even, odd = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y = torch.stack((even * c - odd * s, even * s + odd * c), dim=-1).flatten(-2)
        return (y / norm * st["s_qk"]).to(dtype)

    q, k, v = rotate(qkv[:, :, 0]), rotate(qkv[:, :, 1]), (qkv[:, :, 2] / rho).to(dtype)
    _plain_store(k, v, st["slots"], st["k_pages"], st["v_pages"])
    return q, st["k_pages"], st["v_pages"]


def _plain_store(k, v, slots, k_pages, v_pages):
    page = k_pages.shape[2]
    live = slots >= 0
    at = slots[live].long()
    k_pages[at // page, :, at % page] = k[live]
    v_pages[at // page, :, at % page] = v[live]


def _plain_write(st):
    _plain_store(st["k"], st["v"], st["slots"], st["k_pages"], st["v_pages"])
    return st["k_pages"], st["v_pages"]


def _plain_attention(st):
    q, table, lengths = st["q"].float(), st["table"], st["lengths"]
    batch, heads, dim = q.shape
    _, kv_heads, page, _ = st["k_pages"].shape
    group = heads // kv_heads
    out = torch.empty_like(q)
    # a few requests at a time, so that the gathered keys and values stay within some GB
    step = max(1, (1 << 28) // (table.shape[1] * page * kv_heads * dim))
    for b in range(0, batch, step):
        rows = table[b:b + step].clamp(min=0).long()
        n = rows.shape[0]
        k = st["k_pages"][rows].float().permute(0, 2, 1, 3, 4).reshape(n, kv_heads, -1, dim)
        v = st["v_pages"][rows].float().permute(0, 2, 1, 3, 4).reshape(n, kv_heads, -1, dim)
        there = torch.arange(k.shape[2], device=q.device)[None, :] < lengths[b:b + step, None]
        s = q[b:b + step].view(n, kv_heads, group, dim) @ k.transpose(-1, -2) * st["scale"]
        s = s.masked_fill(~there[:, None, None, :], float("-inf"))
        m = s.amax(-1, keepdim=True).clamp(min=-1e30)
        p = torch.exp(s - m)
        v = v.masked_fill(~there[:, None, :, None], 0.0)
        o = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
        out[b:b + step] = o.reshape(n, heads, dim)
    return out.to(st["q"].dtype)


_RUN_OWN = {"tables": _own_tables, "append": _own_append, "write": _own_write, "attention": _own_attention}
_RUN_PLAIN = {"tables": _plain_tables, "append": _plain_append, "write": _plain_write,
              "attention": _plain_attention}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"tables": _exact_tables, "append": _exact_append, "write": _exact_write,
            "attention": _exact_attention}[case["op"]](st)


def _exact_tables(st):
    # whole numbers, request by request
    case = st["case"]
    page = case["page"]
    host = st["initial"].cpu()
    lengths, count, free, table = (x.tolist() for x in _table_views(host, case["batch"], st["pool"], st["width"]))
    stack = free[:count[0]]
    done = st["done"].tolist() if st["done"] is not None else [False] * case["batch"]
    for b, d in enumerate(done):
        if d:
            stack += table[b][:_pages(lengths[b], page)]
            lengths[b] = 0
    free = stack + free[len(stack):]
    slots, pos = [], []
    for b, n in enumerate(st["new"].tolist()):
        row_s, row_p = [-1] * case["max_new"], [0] * case["max_new"]
        for i in range(n):
            at = lengths[b]
            if at % page == 0:
                table[b][at // page] = stack.pop()
            row_s[i], row_p[i] = table[b][at // page] * page + at % page, at
            lengths[b] = at + 1
        slots.append(row_s)
        pos.append(row_p)
    return tuple(torch.tensor(x, dtype=torch.int32, device="cuda").view(shape) for x, shape in (
        (slots, (case["batch"], -1)), (pos, (case["batch"], -1)), (lengths, (-1,)), ([len(stack)], (-1,)),
        (free, (-1,)), (table, (case["batch"], -1))))


def _exact_store(k, v, st):
    page = st["k_pages"].shape[2]
    kp, vp = st["k_pages"].double(), st["v_pages"].double()
    slots = st["slots"].reshape(-1).long()
    keep = torch.nonzero(slots >= 0)[:, 0]
    slots = slots[keep]
    for h in range(kp.shape[1]):
        for pool, rows in ((kp, k), (vp, v)):
            flat = pool[:, h].reshape(-1, pool.shape[3]).clone()
            flat.index_copy_(0, slots, rows.reshape(-1, rows.shape[-2], rows.shape[-1])[keep, h])
            pool[:, h] = flat.view(-1, page, pool.shape[3])
    return kp, vp


def _exact_write(st):
    return _exact_store(st["k"].double(), st["v"].double(), st)


def _exact_append(st):
    x, rho = st["qkv"].double(), st["rho"].double()[:, :, None, None]
    half = st["cos"].shape[1]
    turn = torch.complex(st["cos"].double(), st["sin"].double())[st["pos"].long()][:, :, None, :]
    out = []
    for part in (0, 1):
        row = x[:, :, part]
        den = torch.linalg.vector_norm(row, dim=-1, keepdim=True).clamp(min=0)
        den = torch.where(den > rho * st["eps"], den, rho * st["eps"])
        pair = torch.view_as_complex(row[..., :2 * half].reshape(*row.shape[:-1], half, 2).contiguous())
        row = torch.view_as_real(pair * turn).flatten(-2)
        out.append(row * st["s_qk"].double() / den)
    kp, vp = _exact_store(out[1], x[:, :, 2] / rho, st)
    return out[0], kp, vp


def _exact_attention(st):
    q = st["q"].double()
    batch, heads, dim = q.shape
    kv_heads, page = st["k_pages"].shape[1], st["k_pages"].shape[2]
    out = torch.zeros_like(q)
    for b, n in enumerate(st["lengths"].tolist()):
        if n == 0:
            continue
        pages = st["table"][b, :_pages(n, page)].long()
        for g in range(kv_heads):
            k = st["k_pages"][pages, g].reshape(-1, dim)[:n].double()
            v = st["v_pages"][pages, g].reshape(-1, dim)[:n].double()
            for h in range(g * heads // kv_heads, (g + 1) * heads // kv_heads):
                out[b, h] = torch.softmax(k @ q[b, h] * st["scale"], dim=0) @ v
    return out
