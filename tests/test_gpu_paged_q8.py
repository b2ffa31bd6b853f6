"""The 8-bit paged key-value cache operators on B200, against plain 64-bit forms (tests/paged_q8_ref.py)."""

import math

import numpy as np
import pytest
import torch

from engpt_b200 import _lib, kernels as K
from tests import paged_q8_ref as Q, paged_ref as R

pytestmark = pytest.mark.gpu

ERR_ARG = 7
KINDS = ["int8", "e4m3"]
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(autouse=True)
def _clean(cuda):
    _lib.clear_device_status()
    with torch.no_grad():
        yield
    status = _lib.device_status()
    _lib.clear_device_status()
    assert status == 0, f"a kernel recorded a device-side failure: {status:#x}"


def expect_status(site):
    word = _lib.device_status()
    _lib.clear_device_status()
    assert word & 0xFF == ERR_ARG and word >> 8 == site, hex(word)


def state(cache):
    return [Q.raw(cache[0]), Q.raw(cache[1]), cache[2].cpu().clone(), cache[3].cpu().clone()]


def check_both(cache, before, k, v, slots, err_k=0.0, err_v=0.0, dead=()):
    slots = slots.reshape(-1).tolist()
    Q.check_store(cache[0], cache[2], before[0], before[2], k, slots, err_k, dead)
    Q.check_store(cache[1], cache[3], before[1], before[3], v, slots, err_v, dead)


def rows(n, heads, dim, dtype, seed):
    """k, v [n, heads, dim] as views into packed rows, tokens of different size."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, 3, heads, dim, generator=gen, device="cuda")
    x = (x * torch.exp(0.7 * torch.randn(n, 3, heads, 1, generator=gen, device="cuda"))).to(dtype)
    return x[:, 1], x[:, 2]


def f64(t):
    return t.cpu().double()


# ------------------------------------------------------------------ write
SIZES = [  # heads, dim, page, block
    (16, 64, 16, 16), (4, 64, 64, 16), (16, 128, 64, 64), (5, 80, 32, 8), (2, 16, 16, 4), (3, 33, 6, 3), (2, 8, 1, 1),
    (3, 64, 16, 1), (2, 256, 128, 128), (1, 24, 40, 20)]


@pytest.mark.parametrize("layout", ["head", "token", "both", "odd"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dim,page,block", SIZES)
def test_write_prompts(cuda, kind, dtype, layout, heads, dim, page, block):
    """Three requests: from the start of a page, from inside a block, and one that is padded."""
    tokens = 2 * page + block // 2 + 3
    first = [0, block // 2 + 1, page]
    pool = 3 * (tokens // page + 2)
    cache = Q.make_pools(pool, heads, page, dim, block, kind, layout)
    Q.fill_pools(cache, heads + dim)
    before = state(cache)
    slots = Q.prompt_slots(first, tokens, page, pool, dim, pad=(0, 0, min(5, tokens - 1)))
    k, v = rows(3 * tokens, heads, dim, dtype, page + dim)
    K.write_kv_pages_q8(k.unflatten(0, (3, tokens)), v.unflatten(0, (3, tokens)), slots.cuda(), *cache)
    check_both(cache, before, f64(k), f64(v), slots)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dim,page,block", SIZES)
def test_write_one_token_at_a_time(cuda, kind, dtype, heads, dim, page, block):
    """Requests that grow token by token: each write raises the scale of its block or leaves it."""
    bsz, steps = 5, 2 * block + 3
    first = [0, block - 1, block // 2, page - 1, 1 % block]
    pages = -(-(page + steps) // page)
    cache = Q.make_pools(bsz * pages, heads, page, dim, block, kind)
    Q.fill_pools(cache, dim)
    slots = Q.prompt_slots(first, steps, page, bsz * pages, page)
    k, v = rows(bsz * steps, heads, dim, dtype, dim)
    k, v = k.unflatten(0, (bsz, steps)), v.unflatten(0, (bsz, steps))
    for t in range(min(steps, 12)):
        before = state(cache)
        K.write_kv_pages_q8(k[:, t], v[:, t], slots[:, t].contiguous().cuda(), *cache)
        check_both(cache, before, f64(k[:, t]), f64(v[:, t]), slots[:, t])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 700, 9000])
def test_write_many_single_tokens(cuda, kind, dtype, n):
    """Decoding requests, each in a block of its own, up to thousands in one call."""
    heads, dim, page, block = 2, 64, 32, 16
    rng = np.random.default_rng(n)
    slots = torch.from_numpy((rng.permutation(n) * page + rng.integers(0, page, n)).astype(np.int32))
    cache = Q.make_pools(n, heads, page, dim, block, kind)
    Q.fill_pools(cache, n, -6.0, 1.0)
    before = state(cache)
    k, v = rows(n, heads, dim, dtype, n)
    K.write_kv_pages_q8(k, v, slots.cuda(), *cache)
    if n <= 700:
        check_both(cache, before, f64(k), f64(v), slots)
    else:                              # the same call on a part of the rows gives the same blocks
        part = torch.arange(5, n, 17)
        again = Q.make_pools(n, heads, page, dim, block, kind)
        for c, b in zip(again, before):
            Q.copy_codes(c, b) if c.dim() == 4 else c.copy_(b)
        K.write_kv_pages_q8(k[part.cuda()], v[part.cuda()], slots[part].cuda(), *again)
        pages = (slots[part] // page).long().cuda()
        for a, b in zip(cache, again):
            assert torch.equal(a[pages].view(torch.uint8), b[pages].view(torch.uint8))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 33])
def test_write_strided_and_bad_slots(cuda, kind, dim):
    heads, page, block, pool = 4, 16, 8, 5
    k = torch.randn(6, 2 * heads, dim, device=cuda)[:, ::2]
    v = torch.randn(heads, 6, dim, device=cuda).transpose(0, 1)
    cache = Q.make_pools(pool, heads, page, dim, block, kind)
    Q.fill_pools(cache, 1)
    before = state(cache)
    slots = torch.tensor([3, -1, 79, 80, -2, 2 ** 31 - 1], dtype=torch.int32)
    K.write_kv_pages_q8(k, v, slots.cuda(), *cache)
    expect_status(43)
    ok = torch.tensor([3, -1, 79, -1, -1, -1])
    check_both(cache, before, f64(k), f64(v), ok)
    before = state(cache)
    K.write_kv_pages_q8(k[:0], v[:0], slots[:0].cuda(), *cache)
    assert all(torch.equal(a, b) for a, b in zip(state(cache), before))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 33])
def test_write_extreme_numbers(cuda, kind, dim):
    """Zeros, the smallest and the largest numbers, and numbers of very different size in one block."""
    heads, page, block = 1, 16, 8
    cache = Q.make_pools(6, heads, page, dim, block, kind)
    x = torch.zeros(40, heads, dim, device=cuda)
    x[8:16] = torch.randn(8, heads, dim, device=cuda) * 1e-42
    x[16:24] = torch.randn(8, heads, dim, device=cuda).clamp(-3, 3) * 1e38
    x[24:32] = torch.randn(8, heads, dim, device=cuda) * torch.logspace(-30, 30, 8, device=cuda).view(8, 1, 1)
    x[32:40, :, 0] = 1e-30
    slots = torch.arange(40, dtype=torch.int32)
    before = state(cache)
    K.write_kv_pages_q8(x, -x, slots.cuda(), *cache)
    check_both(cache, before, f64(x), -f64(x), slots)
    assert (Q.values(cache[0], cache[2])[0, 0, :8] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 33])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_write_infinities_and_nan(cuda, kind, dim, bad):
    """A number that is none makes its block's scale NaN, of its head and pool alone, until the block starts anew."""
    heads, page, block = 2, 16, 8
    cache = Q.make_pools(2, heads, page, dim, block, kind)
    Q.fill_pools(cache, 2)
    k, v = torch.randn(16, heads, dim, device=cuda), torch.randn(16, heads, dim, device=cuda)
    k[3, 1, dim - 1] = bad
    slots = torch.arange(16, dtype=torch.int32, device=cuda)
    K.write_kv_pages_q8(k, v, slots, *cache)
    got_k, got_v = K.read_kv_pages_q8(slots, *cache, dtype=torch.float32)
    nan = got_k.isnan()
    assert nan[:8, 1].all() and not nan[:8, 0].any() and not nan[8:].any() and not got_v.isnan().any()
    k[5, 1] = 1.0
    K.write_kv_pages_q8(k[5:6], v[5:6], slots[5:6], *cache)        # inside the block: still NaN
    assert K.read_kv_pages_q8(slots[:8], *cache)[0][:, 1].isnan().all()
    K.write_kv_pages_q8(k[:3], v[:3], slots[:3], *cache)           # its first token: anew
    assert not K.read_kv_pages_q8(slots[:3], *cache)[0].isnan().any()


# ------------------------------------------------------------------ append
def append_inputs(n, heads, dim, dtype, seed, table=300):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rho = torch.exp(torch.randn(n, generator=gen, device="cuda"))
    qkv = (torch.randn(n, 3, heads, dim, generator=gen, device="cuda") * rho.view(-1, 1, 1, 1)).to(dtype)
    if n > 2:
        qkv[2, 0, 0] *= 1e-9             # the rho * eps guard
        qkv[1, 1, 0] = 0                 # a key of length 0
    cos, sin = K.rotary_frequencies(table, dim, device=torch.device("cuda", 0), dtype=torch.float32, theta=10000.0)
    scale = 1.0 + 0.1 * torch.randn(heads, dim, generator=gen, device="cuda")
    pos = torch.randint(0, table, (n,), generator=gen, device="cuda", dtype=torch.int32)
    return qkv, rho, cos, sin, scale, pos


def append_error(ref):
    """k and v before the quantisation are some ten fp32 operations, or the approximate reciprocals of the bf16 path (2 ulp
    each): 2^-18 of the row's largest value (the rotation's difference of two products can cancel)."""
    return 2.0 ** -18 * ref.abs().amax(-1, keepdim=True)


@pytest.mark.parametrize("layout", ["head", "token", "odd"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dim,page,block,bsz,tokens", [
    (16, 64, 64, 16, 6, 1), (4, 64, 16, 8, 3, 37), (16, 128, 64, 64, 2, 70), (5, 80, 8, 8, 2, 9), (3, 33, 5, 5, 2, 12),
    (2, 16, 16, 4, 3, 20), (12, 64, 16, 16, 2, 18), (2, 64, 16, 1, 2, 7), (2, 256, 16, 16, 2, 19)])
def test_append(cuda, layout, dtype, kind, heads, dim, page, block, bsz, tokens):
    pool = bsz * (tokens // page + 2) + 2
    qkv, rho, cos, sin, scale, pos = append_inputs(bsz * tokens, heads, dim, dtype, dim + tokens)
    cache = Q.make_pools(pool, heads, page, dim, block, kind, layout)
    Q.fill_pools(cache, dim)
    before = state(cache)
    slots = Q.prompt_slots([b * (block // 2) for b in range(bsz)], tokens, page, pool, dim, pad=(0, min(3, tokens - 1)))
    keep = qkv.clone()
    lead = (bsz, tokens)
    q = K.qkv_append_from_carried_q8(qkv.unflatten(0, lead), rho.view(lead), cos, sin, scale, 1e-6, pos.view(lead),
                                     slots.cuda(), *cache)
    assert torch.equal(qkv, keep)
    rq, rk, rv = R.postprocess(qkv, rho, cos, sin, scale, 1e-6, pos)
    check_both(cache, before, rk, rv, slots, append_error(rk), append_error(rv))
    assert q.shape == (*lead, heads, dim) and q.dtype == dtype
    got = q.flatten(0, 1).cpu().double()
    assert ((got - rq).abs() <= torch.finfo(dtype).eps / 2 * rq.abs() + append_error(rq)).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dim", [(4, 64), (3, 33)])
def test_append_bad_positions_and_slots(cuda, kind, heads, dim):
    """A token with a bad position is left out of its run; its q is zero."""
    qkv, rho, cos, sin, scale, _ = append_inputs(8, heads, dim, torch.float32, 1, table=50)
    cache = Q.make_pools(2, heads, 16, dim, 8, kind)
    Q.fill_pools(cache, 3)
    before = state(cache)
    qkv[1] *= 1e6                                                  # would set the scale if it counted
    pos = torch.tensor([3, 50, 49, 0, -1, 5, 6, 7], dtype=torch.int32, device=cuda)
    slots = torch.tensor([3, 4, 5, -1, 16, 24, 25, 26], dtype=torch.int32)
    q = K.qkv_append_from_carried_q8(qkv, rho, cos, sin, scale, 1e-6, pos, slots.cuda(), *cache)
    expect_status(42)
    assert (q[1] == 0).all() and (q[4] == 0).all() and (q[[0, 2, 3, 5]] != 0).any(-1).all()
    _, rk, rv = R.postprocess(qkv, rho, cos, sin, scale, 1e-6, pos.clamp(0, 49))
    check_both(cache, before, rk, rv, slots, append_error(rk), append_error(rv), dead=(1, 4))
    pos = torch.arange(8, dtype=torch.int32, device=cuda)
    slots = torch.tensor([32, -2, 2, -1, 2 ** 31 - 1, 8, 9, 10], dtype=torch.int32)
    before = state(cache)
    q = K.qkv_append_from_carried_q8(qkv, rho, cos, sin, scale, 1e-6, pos, slots.cuda(), *cache)
    expect_status(43)
    assert (q != 0).any(-1).all()
    _, rk, rv = R.postprocess(qkv, rho, cos, sin, scale, 1e-6, pos)
    check_both(cache, before, rk, rv, torch.tensor([-1, -1, 2, -1, -1, 8, 9, 10]), append_error(rk), append_error(rv))


# ------------------------------------------------------------------ read
@pytest.mark.parametrize("layout", ["head", "token", "both", "odd"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dim,page,block", SIZES)
def test_read(cuda, kind, dtype, layout, heads, dim, page, block):
    pool = 7
    cache = Q.make_pools(pool, heads, page, dim, block, kind, layout)
    Q.fill_pools(cache, dim)
    rng = np.random.default_rng(dim)
    slots = torch.from_numpy(rng.integers(-1, pool * page, (3, 11)).astype(np.int32))   # (reading may repeat slots)
    got = K.read_kv_pages_q8(slots.cuda(), *cache, dtype=dtype)
    for part in range(2):
        x = Q.values(cache[part], cache[2 + part])
        assert got[part].shape == (3, 11, heads, dim) and got[part].dtype == dtype
        for (b, t), s in np.ndenumerate(slots.numpy()):
            ref = x[s // page, :, s % page] if s >= 0 else torch.zeros(heads, dim, dtype=torch.float64)
            # one fp32 product, rounded once more to the type
            assert ((f64(got[part][b, t]) - ref).abs() <= ref.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -23)).all()


def test_read_bad_slots_and_none(cuda):
    cache = Q.make_pools(2, 2, 16, 64, 16, "int8")
    Q.fill_pools(cache, 1)
    slots = torch.tensor([0, 32, -2, 31], dtype=torch.int32, device=cuda)
    k, v = K.read_kv_pages_q8(slots, *cache)
    expect_status(43)
    assert (k[1:3] == 0).all() and (v[1:3] == 0).all() and (k[[0, 3]] != 0).any()
    k, v = K.read_kv_pages_q8(slots[:0], *cache)
    assert k.shape == (0, 2, 64) and v.shape == (0, 2, 64)


@pytest.mark.parametrize("kind,tol", [("int8", 0.5 / 127), ("e4m3", 2.0 ** -4)])
def test_write_then_read(cuda, kind, tol):
    """What comes back is within half a step of what went in: of the block's largest number (int8), of the number (e4m3,
    or 2^-10 of a 448th of the block's largest one)."""
    bsz, tokens, heads, dim, page, block = 3, 100, 4, 64, 32, 16
    k, v = rows(bsz * tokens, heads, dim, torch.bfloat16, 5)
    k, v = k.unflatten(0, (bsz, tokens)), v.unflatten(0, (bsz, tokens))
    cache = Q.make_pools(15, heads, page, dim, block, kind)
    slots = Q.prompt_slots([0] * bsz, tokens, page, 15, 2).cuda()
    K.write_kv_pages_q8(k, v, slots, *cache)
    for x, y in zip((k, v), K.read_kv_pages_q8(slots, *cache, dtype=torch.float32)):
        x, y = f64(x), f64(y)
        for t in range(0, tokens, block):
            part, back = x[:, t:t + block], y[:, t:t + block]
            amax = part.abs().amax((1, 3), keepdim=True)
            lim = tol * amax if kind == "int8" else torch.maximum(tol * part.abs(), 2.0 ** -10 / 448 * amax)
            assert ((part - back).abs() <= lim * (1 + 2.0 ** -14)).all()


# ------------------------------------------------------------------ attention
def attention_inputs(lengths, heads, kv_heads, dim, page, block, dtype, kind, layout="head", seed=0, spare_width=1,
                     width=None, spread=1.0, pool=None):
    """A cache whose codes and scales behind the lengths are NaN where the type has one."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    need = max([R.pages_of(max(n, 0), page) for n in lengths] + [0]) + spare_width
    width = width or need
    pool = pool or sum(R.pages_of(max(n, 0), page) for n in lengths) + 3
    table, _ = R.random_table(lengths, page, width, pool, rng)
    cache = Q.make_pools(pool, kv_heads, page, dim, block, kind, layout)
    Q.fill_pools(cache, seed, -5.5, -4.0)
    codes, scales = torch.ones(pool, page, dtype=torch.bool), torch.ones(pool, page // block, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for j in range(R.pages_of(max(n, 0), page)):
            t = min(page, n - j * page)
            codes[int(table[b, j]), :t] = False
            scales[int(table[b, j]), :R.pages_of(t, block)] = False
    for i in range(2):
        dead = codes[:, None, :, None].expand(cache[i].shape).cuda()
        cache[i].view(torch.uint8).masked_fill_(dead, 0x7f if kind == "e4m3" else 0x80)
        cache[2 + i].masked_fill_(scales[:, None].expand(cache[2].shape).cuda(), float("nan"))
    q = (spread * torch.randn(len(lengths), heads, dim, generator=gen, device="cuda")).to(dtype)
    return q, cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), 1.0 / math.sqrt(dim)


def attend(args):
    q, cache, table, lengths, scale = args
    return K.paged_sdpa_q8(q, *cache, table, lengths, scale=scale)


def check_attention(args, out=None):
    q, cache, table, lengths, scale = args
    out = attend(args) if out is None else out
    assert out.shape == q.shape and out.dtype == q.dtype
    ref, tol = Q.attention(q, cache, table, lengths, scale)
    err = (out.cpu().double() - ref).abs()
    assert (err <= tol).all(), f"max error {err.max().item()}, over its tolerance by {(err / tol).max().item()}"
    return out


LENGTHS = [0, 1, 7, 8, 9, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 300]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 16, 80, 33, 256, 24])
@pytest.mark.parametrize("page,block", [(16, 16), (64, 16), (8, 8), (24, 8), (24, 24), (6, 3), (1, 1), (64, 64)])
def test_attention_lengths(cuda, dtype, kind, dim, page, block):
    check_attention(attention_inputs(LENGTHS, 4, 4, dim, page, block, dtype, kind, seed=dim + page))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30, 3.0])
def test_attention_scales(cuda, dtype, kind, dim, scale):
    args = attention_inputs([0, 5, 64, 333], 3, 3, dim, 16, 16, dtype, kind, seed=dim)
    check_attention(args[:4] + (scale,))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (6, 2), (8, 1), (16, 2), (12, 1), (40, 2), (5, 5)])
@pytest.mark.parametrize("dim", [64, 128, 48])
def test_attention_head_groups(cuda, dtype, kind, heads, kv_heads, dim):
    check_attention(attention_inputs([70, 0, 513, 1], heads, kv_heads, dim, 16, 8, dtype, kind, seed=heads))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (16, 2)])
@pytest.mark.parametrize("dim", [16, 32, 48, 80, 96, 112])
@pytest.mark.parametrize("bsz,width_tokens", [(1, 100), (1, 3000), (9, 700), (60, 400)])
def test_attention_widths_of_any_number_of_pieces(cuda, dtype, kind, heads, kv_heads, dim, bsz, width_tokens):
    """Head dims of 1, 2, 3, 5, 6 and 7 pieces of 16 codes, in every form of a launch."""
    page = 24 if dim == 48 else 32
    rng = np.random.default_rng(bsz)
    lengths = [int(x) for x in rng.integers(0, width_tokens + 1, bsz)]
    lengths[-1] = width_tokens
    check_attention(attention_inputs(lengths, heads, kv_heads, dim, page, 8, dtype, kind, seed=dim))


@pytest.mark.parametrize("layout", ["token", "both", "odd"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (48, 16), (80, 64), (16, 16)])
def test_attention_cache_layouts(cuda, dtype, kind, layout, dim, page):
    check_attention(attention_inputs([90, 300, 33], 6, 3, dim, page, 16, dtype, kind, layout=layout, seed=dim))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads", [(16, 16), (16, 2)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bsz,width_tokens", [(1, 64), (1, 512), (1, 2048), (1, 8192), (3, 512), (3, 2048), (12, 1024),
                                              (20, 512), (40, 256)])
def test_attention_every_form_with_short_and_long_rows(cuda, dtype, heads, kv_heads, dim, bsz, width_tokens):
    """The table's width decides the form of a launch; the rows themselves may be of any length within it."""
    page = 64
    kind = KINDS[(bsz + dim // 64) % 2]
    rng = np.random.default_rng(bsz + width_tokens)
    lengths = [int(x) for x in rng.integers(0, 130, bsz)]
    lengths[-1] = width_tokens
    args = attention_inputs(lengths, heads, kv_heads, dim, page, 16, dtype, kind, seed=bsz, width=width_tokens // page)
    check_attention(args)
    args[3][-1] = 3          # the same form, nothing left of the long row
    check_attention(args)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bsz,n,heads,dim,page", [(1, 5000, 2, 64, 16), (1, 9001, 16, 128, 64), (2, 4097, 4, 64, 128),
                                                  (3, 2500, 3, 80, 16)])
def test_attention_long(cuda, dtype, kind, bsz, n, heads, dim, page):
    check_attention(attention_inputs([n] + [37] * (bsz - 1), heads, heads, dim, page, 8, dtype, kind, seed=n))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bsz", [200, 1500, 9000])
def test_attention_many_rows(cuda, kind, bsz):
    rng = np.random.default_rng(bsz)
    lengths = rng.integers(0, 90 if bsz < 9000 else 30, bsz).tolist()
    lengths[5] = 700 if bsz < 9000 else 40
    check_attention(attention_inputs(lengths, 4 if bsz < 9000 else 2, 2, 64, 16, 16, torch.bfloat16, kind, seed=bsz))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 80])
def test_attention_scales_of_very_different_size(cuda, dtype, kind, dim):
    """Scales of blocks between 1e-20 and 1e12 (values) and rising along the cache (keys), scores of some hundreds."""
    args = attention_inputs([400, 130, 64], 2, 2, dim, 16, 8, dtype, kind, seed=9, spread=20.0)
    _, cache, table, lengths, _ = args
    for b, n in enumerate(lengths.tolist()):
        for j in range(0, n, 8):
            pg, bl = int(table[b, j // 16]), j % 16 // 8
            cache[2][pg, :, bl] *= 0.02 + j / n
            cache[3][pg, :, bl] = 10.0 ** (12 - (j // 8 * 7) % 33)
    check_attention(args)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 48, 33])
def test_attention_q_of_any_size(cuda, dtype, dim):
    """Rows of q far outside the range of 16-bit numbers, of zeros, and with elements of very different size."""
    args = list(attention_inputs([100, 33, 90, 257, 12], 2, 2, dim, 16, 16, dtype, "int8", seed=4))
    q = args[0].float()
    q[0] *= 1e20
    q[1] *= 1e-25
    q[2] = 0
    q[3, 0] *= torch.logspace(-12, 0, dim, device=cuda)
    args[0] = q.to(dtype)
    args[1][2][int(args[2][0, 0])] *= 1e-20                        # (scores of row 0 stay finite)
    for j in range(7):
        args[1][2][int(args[2][0, j])] = 1e-21
    check_attention(tuple(args))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 48, 33])
def test_attention_ignores_what_lies_behind_a_length(cuda, dtype, kind, dim):
    """Codes and scales behind a length, and table entries behind its pages, change no bit."""
    args = attention_inputs([5, 64, 0, 77], 2, 2, dim, 16, 8, dtype, kind, seed=3, spare_width=4)
    out = check_attention(args)
    q, cache, table, lens, scale = args
    for fill, byte in ((float("inf"), 0x7f), (0.0, 0xff), (3.0e38, 0)):
        other = [c.clone() for c in cache]
        for i in range(2):
            u = other[i].view(torch.uint8)
            u.copy_(torch.where(u == (0x7f if kind == "e4m3" else 0x80), torch.full_like(u, byte), u))
            other[2 + i] = torch.where(cache[2 + i].isnan(), torch.full_like(cache[2 + i], fill), cache[2 + i])
        t2 = torch.where(table < 0, torch.full_like(table, 2 ** 31 - 1 if fill else cache[0].shape[0]), table)
        assert torch.equal(out, attend((q, other, t2, lens, scale)))


@pytest.mark.parametrize("dim", [64, 33])
def test_attention_of_a_block_without_numbers(cuda, dim):
    """A NaN scale in use shows in its row and heads, and nowhere else."""
    q, cache, table, lens, scale = attention_inputs([50, 40], 4, 2, dim, 16, 8, torch.bfloat16, "int8", seed=3)
    clean = attend((q, cache, table, lens, scale))
    cache[2][int(table[0, 1]), 1, 1] = float("nan")
    cache[3][int(table[1, 0]), 0, 0] = float("nan")
    out = attend((q, cache, table, lens, scale))
    nan = out.isnan()
    assert nan[0, 2:].all() and nan[1, :2].all()
    assert torch.equal(out[0, :2], clean[0, :2]) and torch.equal(out[1, 2:], clean[1, 2:])


@pytest.mark.parametrize("dim", [64, 33])
def test_attention_bad_pages_and_lengths(cuda, dim):
    """A page outside the pool counts as absent, a length beyond the table is cut; both are recorded."""
    q, cache, table, lens, scale = attention_inputs([40, 20], 2, 2, dim, 16, 8, torch.bfloat16, "int8", spare_width=0)
    ref = check_attention((q, cache, table, lens, scale))
    for bad in (-1, cache[0].shape[0], 2 ** 31 - 1, -2 ** 31):
        t2 = table.clone()
        t2[1, 1] = bad
        out = attend((q, cache, t2, lens, scale))
        expect_status(44)
        short = lens.clone()
        short[1] = 16
        want, tol = Q.attention(q, cache, table, short, scale)
        assert ((out.cpu().double() - want).abs() <= tol).all()
    lens2 = lens.clone()
    lens2[0] = 2 ** 31 - 1
    out = attend((q, cache, table, lens2, scale))
    expect_status(44)
    assert torch.equal(out[1], ref[1])
    lens2[0] = -5
    out = attend((q, cache, table, lens2, scale))
    assert (out[0] == 0).all() and torch.equal(out[1], ref[1])


def test_attention_zero_sizes(cuda):
    q, cache, table, lens, scale = attention_inputs([3], 2, 2, 64, 16, 16, torch.bfloat16, "int8")
    assert attend((q[:0], cache, table[:0], lens[:0], scale)).shape == (0, 2, 64)
    empty = [c[:0] for c in cache]
    out = attend((q, empty, table[:, :0], torch.zeros_like(lens), scale))
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_strided_q(cuda, dtype):
    args = attention_inputs([90, 300, 33], 6, 3, 64, 16, 16, dtype, "int8", seed=1)
    packed = torch.zeros(3, 3, 6, 64, dtype=dtype, device=cuda)
    packed[:, 0] = args[0]
    out = attend((packed[:, 0],) + args[1:])
    assert torch.equal(out, check_attention(args))
    odd = torch.zeros(3, 6, 65, dtype=dtype, device=cuda)[..., 1:]
    odd.copy_(args[0])
    check_attention((odd,) + args[1:], attend((odd,) + args[1:]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 80, 33])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attention_of_a_query_that_is_no_number(cuda, dtype, kind, dim, bad):
    """Its own result is NaN; the other heads of its row and kv head, and the other rows, are untouched."""
    args = attention_inputs([50, 400], 8, 2, dim, 16, 8, dtype, kind, seed=3)
    clean = check_attention(args)
    q = args[0].clone()
    q[1, 2, 5] = bad
    out = attend((q,) + args[1:])
    assert out[1, 2].isnan().all()
    keep = torch.ones(2, 8, dtype=torch.bool, device=cuda)
    keep[1, 2] = False
    assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [128, 80, 112])
def test_attention_most_rows_that_the_list_takes(cuda, dtype, dim):
    """8192 rows with eight query heads on a kv head: the most shared memory that a launch asks for."""
    rng = np.random.default_rng(2)
    lengths = rng.integers(0, 20, 8192).tolist()
    lengths[4000] = 130
    check_attention(attention_inputs(lengths, 8, 1, dim, 16, 16, dtype, "int8", seed=1))


def test_attention_far_into_a_large_pool(cuda):
    """Codes more than 2^31 bytes behind the pool's start, scales of strides that are not their shape's."""
    page, heads, dim, pool = 64, 8, 128, 36000                        # 2.36e9 codes each
    if torch.cuda.mem_get_info()[0] < 12e9:
        pytest.skip("needs 12 GB")
    k = torch.zeros(pool, heads, page, dim, dtype=torch.int8, device=cuda)
    v = torch.zeros_like(k)
    ks, vs = (torch.zeros(heads, 4, pool, device=cuda).permute(2, 0, 1) for _ in range(2))
    n = 200
    pages = torch.tensor([pool - 1, 3, pool - 2, 17], dtype=torch.int32)
    slots = torch.tensor([int(pages[p // page]) * page + p % page for p in range(n)], dtype=torch.int32, device=cuda)
    kr, vr = rows(n, heads, dim, torch.bfloat16, 5)
    K.write_kv_pages_q8(kr, vr, slots, k, v, ks, vs)
    back = K.read_kv_pages_q8(slots, k, v, ks, vs, dtype=torch.float32)
    small = [x[pages.long().to(cuda)].contiguous() for x in (k, v, ks, vs)]
    near = torch.tensor([(p // page) * page + p % page for p in range(n)], dtype=torch.int32, device=cuda)
    for a, b in zip(back, K.read_kv_pages_q8(near, *small, dtype=torch.float32)):
        assert torch.equal(a, b) and (a != 0).any()
    q = torch.randn(1, 16, dim, device=cuda).bfloat16()
    lens = torch.tensor([n], dtype=torch.int32, device=cuda)
    out = K.paged_sdpa_q8(q, k, v, ks, vs, pages[None].to(cuda), lens, scale=0.1)
    check_attention((q, small, torch.arange(4, dtype=torch.int32, device=cuda)[None], lens, 0.1), out)


@pytest.mark.parametrize("kind", KINDS)
def test_calls_on_two_streams_and_in_graphs(cuda, kind):
    """Calls at the same time on two streams, and replays of one captured graph of all four operators, give what they give
    alone."""
    heads, dim, page, block, n = 4, 64, 16, 16, 60
    sets = []
    for seed in range(2):
        qkv, rho, cos, sin, scale, pos = append_inputs(n, heads, dim, torch.bfloat16, seed)
        cache = Q.make_pools(n, heads, page, dim, block, kind)
        Q.fill_pools(cache, seed)
        slots = Q.prompt_slots([3] * 4, n // 4, page, n, seed).flatten().to(cuda)
        k, v = rows(n, heads, dim, torch.bfloat16, seed)
        table = (slots.view(4, -1)[:, [0, -1]] // page).contiguous()
        lens = torch.tensor([18] * 4, dtype=torch.int32, device=cuda)
        sets.append((qkv, rho, cos, sin, scale, pos, cache, [c.clone() for c in cache], slots, k, v, table, lens))

    def run(s):
        qkv, rho, cos, sin, scale, pos, cache, first, slots, k, v, table, lens = s
        for c, f in zip(cache, first):
            c.copy_(f)
        K.write_kv_pages_q8(k, v, slots, *cache)
        q = K.qkv_append_from_carried_q8(qkv, rho, cos, sin, scale, 1e-6, pos, slots, *cache)
        o = K.paged_sdpa_q8(q[:4].contiguous(), *cache, table, lens, scale=0.125)
        return (q, o, *K.read_kv_pages_q8(slots, *cache))

    want = [[x.clone() for x in run(s)] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
    with torch.cuda.stream(streams[0]):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[0]):
            out = run(sets[0])
        for _ in range(3):
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want[0]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("tokens", [1, 64, 2048])
def test_numbers_that_are_none_in_bf16(cuda, kind, block, bad, tokens):
    """One bad element of a bf16 row, in the write and in the append, whatever form the call takes: its head's block of its
    pool is NaN (of k and q's row where it is in k or q), every other number is one."""
    heads, dim, page, pool = 8, 128, 64, tokens // 64 + 2
    slots = torch.arange(tokens, dtype=torch.int32, device=cuda)
    at, h = tokens * 2 // 3, 5
    blk = slice(at // block * block, min(tokens, at // block * block + block))
    k, v = (torch.randn(tokens, heads, dim, device=cuda).bfloat16() for _ in range(2))
    v[at, h, 77] = bad
    cache = Q.make_pools(pool, heads, page, dim, block, kind)
    K.write_kv_pages_q8(k, v, slots, *cache)
    got_k, got_v = K.read_kv_pages_q8(slots, *cache)
    nan = torch.zeros(tokens, heads, dim, dtype=torch.bool, device=cuda)
    nan[blk, h] = True
    assert torch.equal(got_v.isnan(), nan) and got_k.isfinite().all()

    qkv, rho, cos, sin, scale, pos = append_inputs(tokens, heads, dim, torch.bfloat16, 3)
    qkv[at, 1, h, 3] = bad
    cache = Q.make_pools(pool, heads, page, dim, block, kind)
    q = K.qkv_append_from_carried_q8(qkv, rho, cos, sin, scale, 1e-6, pos, slots, *cache)
    got_k, got_v = K.read_kv_pages_q8(slots, *cache)
    assert torch.equal(got_k.isnan(), nan) and got_v.isfinite().all() and q.isfinite().all()
