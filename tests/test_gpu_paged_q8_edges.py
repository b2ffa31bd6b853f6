"""Corners of the 8-bit paged cache operators on B200: numbers of extreme size, tokens that are left out, scales that are
zero or far apart."""

import pytest
import torch

from engpt_b200 import _lib, kernels as K
from tests import paged_q8_blocks as B, paged_q8_ref as Q, paged_ref as R
from tests.test_gpu_paged_q8 import (DTYPES, KINDS, append_error, append_inputs, attend, attention_inputs,
                                     expect_status, rows)
from tests.test_gpu_paged_q8_large import check_both, sizes, state

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean(cuda):
    _lib.clear_device_status()
    with torch.no_grad():
        yield
    status = _lib.device_status()
    _lib.clear_device_status()
    assert status == 0, f"a kernel recorded a device-side failure: {status:#x}"


# Calls of a token per warp (n None: a few tokens), in windows of blocks, and of the kernel for any head_dim.
CALLS = [(64, 8, None), (64, 16, "large"), (128, 64, "large"), (33, 8, None)]


def tokens_of(n, heads):
    return 64 if n is None else sizes(heads, True, 1) // 64 * 64 + 64


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,block,n", CALLS)
def test_append_zeros_with_small_radii(cuda, dtype, kind, dim, block, n):
    """A v row of zeros is zeros whatever its rho (V / rho), in a block of such rows and beside others."""
    heads, page = 16, 64
    n = tokens_of(n, heads)
    qkv, rho, cos, sin, scale, pos = append_inputs(n, heads, dim, dtype, 7)
    radii = torch.tensor([1e-3, 1e-5, 1.6e-6, 1e-6, 4e-7, 1e-8, 1e-12, 1e-20, 1e-30, 1.0], device=cuda)
    zero = torch.arange(n, device=cuda) // block % 3 < 2          # two blocks of three
    zero |= torch.arange(n, device=cuda) % 5 == 1
    rho = torch.where(zero, radii[torch.arange(n, device=cuda) % 10], rho)
    qkv[zero] = 0
    slots = torch.arange(n, dtype=torch.int32, device=cuda)
    cache = Q.make_pools(n // page, heads, page, dim, block, kind)
    Q.fill_pools(cache, 1)
    before = state(cache)
    q = K.qkv_append_from_carried_q8(qkv, rho, cos, sin, scale, 1e-6, pos, slots, *cache)
    for x in (q, *K.read_kv_pages_q8(slots, *cache, dtype=torch.float32)):
        assert (x[zero] == 0).all() and x.isfinite().all()
    for c in cache[:2]:
        assert (c.transpose(1, 2).flatten(0, 1)[zero].float() == 0).all()              # (codes of 0, with either sign)
    _, rk, rv = B.postprocess(qkv, rho, cos, sin, scale, 1e-6, pos)
    check_both(cache, before, rk, rv, slots, append_error(rk), append_error(rv))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,block,n", CALLS)
def test_append_values_below_the_least_scale(cuda, dtype, kind, dim, block, n):
    """V / rho around and below 2^-100, where a block's scale has its least value, of V near the end of fp32's range."""
    heads, page = 16, 64
    n = tokens_of(n, heads)
    qkv, rho, cos, sin, scale, pos = append_inputs(n, heads, dim, dtype, 8)
    at = torch.arange(n, device=cuda)
    size = torch.tensor([1e-37, 1e-36, 1e-37, 1e-34, 1.0], device=cuda)[at // block % 5]
    rho = torch.tensor([1e-7, 1e-7, 1e-5, 1e-3, 1e-7], device=cuda)[at // block % 5]
    qkv[:, 2] = (torch.randn(n, heads, dim, device=cuda) * size[:, None, None]).to(dtype)
    qkv[:, :2] = torch.randn(n, 2, heads, dim, device=cuda).to(dtype)
    slots = torch.arange(n, dtype=torch.int32, device=cuda)
    cache = Q.make_pools(n // page, heads, page, dim, block, kind)
    Q.fill_pools(cache, 1)
    before = state(cache)
    K.qkv_append_from_carried_q8(qkv, rho, cos, sin, scale, 1e-6, pos, slots, *cache)
    _, rk, rv = B.postprocess(qkv, rho, cos, sin, scale, 1e-6, pos)
    check_both(cache, before, rk, rv, slots, append_error(rk), append_error(rv))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,block,n", CALLS)
@pytest.mark.parametrize("radius", [0.0, float("nan"), float("inf"), 1e-38, -1.0])
def test_append_radii_of_tokens_that_are_left_out(cuda, dtype, kind, dim, block, n, radius):
    """A token with a bad position has no part in its block's scales, whatever its rho and its numbers."""
    heads, page = 16, 64
    n = tokens_of(n, heads)
    qkv, rho, cos, sin, scale, pos = append_inputs(n, heads, dim, dtype, 9, table=50)
    at = torch.arange(n, device=cuda)
    dead = (at % 7 == 3) | ((at + 3) // block % 5 == 4)           # in runs of others, and whole runs
    pos = torch.where(dead, torch.where(at % 2 == 0, 50, -1), pos).to(torch.int32)
    rho = torch.where(dead, radius, rho)
    qkv[dead & (at % 3 == 0)] = float("nan")
    slots = torch.arange(3, n + 3, dtype=torch.int32, device=cuda)
    cache = Q.make_pools(n // page + 1, heads, page, dim, block, kind)
    Q.fill_pools(cache, 2)
    before = state(cache)
    q = K.qkv_append_from_carried_q8(qkv, rho, cos, sin, scale, 1e-6, pos, slots, *cache)
    expect_status(42)
    assert (q[dead] == 0).all() and q.isfinite().all()
    _, rk, rv = B.postprocess(qkv, rho, cos, sin, scale, 1e-6, pos.clamp(0, 49))
    rk[dead], rv[dead] = 0.0, 0.0
    check_both(cache, before, rk, rv, slots, append_error(rk), append_error(rv), dead)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("dim,block,n", CALLS)
@pytest.mark.parametrize("step", ["gap", "down", "twice"])
def test_slots_that_do_not_follow_one_another(cuda, dtype, kind, append, dim, block, n, step):
    """A token beside another one of its block, but not in the next slot, is recorded and left out with those behind it; the
    tokens before it, and the other blocks, are written as if it were not there."""
    heads, page = 16, 64
    n = tokens_of(n, heads)
    slots = torch.arange(n, dtype=torch.int32, device=cuda)
    given, kept = slots.clone(), slots.clone()
    for b in range(1, n // block, 3):
        at = b * block + 3
        if step == "gap":                                          # .., 2, 4, 5, ..
            given[at:at + block - 4] += 1
            given[b * block + block - 1] = -1
        elif step == "down":                                       # .., 2, 1 (the rest -1)
            given[at] = at - 2
            given[at + 1:(b + 1) * block] = -1
        else:                                                      # .., 2, 2, 3, ..
            given[at:(b + 1) * block] -= 1
        kept[at:(b + 1) * block] = -1
    cache = Q.make_pools(n // page, heads, page, dim, block, kind)
    Q.fill_pools(cache, 4)
    before = state(cache)
    if append:
        qkv, rho, cos, sin, scale, pos = append_inputs(n, heads, dim, dtype, 5)
        q = K.qkv_append_from_carried_q8(qkv, rho, cos, sin, scale, 1e-6, pos, given, *cache)
        rq, rk, rv = B.postprocess(qkv, rho, cos, sin, scale, 1e-6, pos)
        assert ((q.double() - rq).abs() <= torch.finfo(dtype).eps / 2 * rq.abs() + append_error(rq)).all()
        err = append_error(rk), append_error(rv)
    else:
        k, v = rows(n, heads, dim, dtype, 5)
        K.write_kv_pages_q8(k, v, given, *cache)
        rk, rv, err = k.double(), v.double(), (0.0, 0.0)
    expect_status(43)
    check_both(cache, before, rk, rv, kept, *err)


# ------------------------------------------------------------------ attention
def weighted(args):
    """The 64-bit result, and the tolerance of check_weighted."""
    q, cache, table, lengths, scale = args
    k, v = Q.values(cache[0], cache[2]), Q.values(cache[1], cache[3])
    step = cache[3].cpu().double().abs().repeat_interleave(cache[1].shape[2] // cache[3].shape[2], dim=2)[..., None]
    off = Q.query_error(q, cache[0].dtype)
    qd, table = q.cpu().double(), table.cpu()
    heads, dim = q.shape[1:]
    group = heads // k.shape[1]
    out, tol = torch.zeros_like(qd), torch.zeros_like(qd)
    top = Q.TOP[cache[0].dtype]
    for b, n in enumerate(lengths.tolist()):
        if n <= 0:
            continue
        rows, vals, steps = (R.gather_rows(x, table[b], n) for x in (k, v, step))
        for h in range(heads):
            kh, vh, sh = rows[:, h // group], vals[:, h // group], steps[:, h // group, 0]
            p = torch.softmax(kh @ qd[b, h] * scale, dim=0)
            out[b, h] = p @ vh
            score = ((dim + 8) * 2.0 ** -24 * (kh.abs() @ qd[b, h].abs()).max() + (kh.abs() @ off[b, h]).max()) * abs(scale)
            weight = 1.45 * score + 2.0 ** -20 + 2 * n * 2.0 ** -24
            spread = p @ vh.abs()
            small = n * 2.0 ** -39 * (p * sh).max() * top
            tol[b, h] = (torch.finfo(q.dtype).eps / 2 * out[b, h].abs() + weight * (spread + out[b, h].abs()) +
                         (2.0 ** -21 if q.dtype == torch.float32 else 2.0 ** -11) * spread + small + 1e-37)
    return out, tol


def check_weighted(args, out=None):
    """Against the 64-bit result, with a tolerance that follows the values with their weights.

    As paged_q8_ref.attention_tolerance, but what the values' weights are off by is taken on sum p |v|, not on the largest
    value of the row: a relative error of a weight (of the scores, the exponentials and the sums) moves numerator and
    denominator by as much of sum p |v| and of the result.  A weight p vs (vs: the value's scale) is one fp16 number, half a
    step 2^-11 (fp32 results: two, 2^-21), or half of 2^-24 where it is below fp16's normal numbers: the head's largest
    p vs is at least 2^14 there, so that is 2^-39 of it, times a code, for each of n keys.
    """
    out = attend(args) if out is None else out
    ref, tol = weighted(args)
    err = (out.cpu().double() - ref).abs()
    assert (err <= tol).all(), f"max error {err.max().item()}, over its tolerance by {(err / tol).max().item()}"
    return out


FORMS = [([400, 130, 64, 7], 2, 2, 16), ([300] * 150, 2, 2, 32), ([3000], 8, 1, 64), ([333, 64, 65], 12, 2, 24)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 80, 33])
@pytest.mark.parametrize("lengths,heads,kv_heads,page", FORMS)
@pytest.mark.parametrize("ratio", [2.0 ** 20, 2.0 ** 33, 2.0 ** 90])
def test_attention_large_values_without_weight(cuda, dtype, kind, dim, lengths, heads, kv_heads, page, ratio):
    """Keys that get next to no weight have values of far larger scale than the others: these keep their bits."""
    args = attention_inputs(lengths, heads, kv_heads, dim, page, 8, dtype, kind, seed=dim)
    q, cache, table, lens, _ = args
    scale = 1.0
    q.copy_(0.05 * torch.randn(q.shape, device=cuda))
    for b, n in enumerate(lengths):
        for j in range(0, n, 8):
            if j // 8 % 5 != 2 or j // 8 in (0, (n - 1) // 8):
                continue
            pg, bl = int(table[b, j // page]), j % page // 8
            cache[3][pg, :, bl] *= ratio
            # the key is against the first kv head's queries: a score of some -150 for all of its group
            cache[2][pg, :, bl] = 1.0
            cache[0].view(torch.uint8)[pg, :, bl * 8:bl * 8 + 8] = 0
            cache[0].view(torch.uint8)[pg, :, bl * 8:bl * 8 + 8, 0] = 0x85 if kind == "int8" else 0xf6   # -123, -224
    q[..., 0] = 1.25 if kind == "int8" else 0.7
    check_weighted((q, cache, table, lens, scale))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 80, 33])
@pytest.mark.parametrize("lengths,heads,kv_heads,page", FORMS)
def test_attention_scales_far_apart(cuda, dtype, kind, dim, lengths, heads, kv_heads, page):
    """Values of very different scale beside each other, with weights that are as far apart."""
    args = attention_inputs(lengths, heads, kv_heads, dim, page, 8, dtype, kind, seed=dim + 1, spread=20.0)
    cache = args[1]
    gen = torch.Generator(device="cuda").manual_seed(3)
    e = torch.rand(cache[3].shape, generator=gen, device="cuda") * 60 - 30
    cache[3].copy_(torch.where(cache[3].isnan(), cache[3], torch.exp2(e.round())))
    check_weighted(args)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 80, 33])
@pytest.mark.parametrize("lengths,heads,kv_heads,page", FORMS)
@pytest.mark.parametrize("least", [0.0, 1e-43, 2.0 ** -121, 2.0 ** -115])
def test_attention_scales_of_nearly_nothing(cuda, dtype, kind, dim, lengths, heads, kv_heads, page, least):
    """Value scales of 0 (a block that was never written, a foreign cache), or too small to be one of the quantising write,
    first in a row, everywhere, or everywhere but at its end."""
    args = attention_inputs(lengths, heads, kv_heads, dim, page, 8, dtype, kind, seed=dim)
    q, cache, table, lens, scale = args
    for b, n in enumerate(lengths):
        pages = table[b, :R.pages_of(n, page)].long()
        last = pages[-1:] if b % 2 else pages[:0]
        keep = cache[3][last].clone()
        cache[3][pages] = torch.where(cache[3][pages].isnan(), cache[3][pages], least)
        cache[3][last] = keep
    out = check_weighted(args)
    if least == 0.0:
        assert (out[::2] == 0).all()
    for i in range(0, len(lengths), 2):
        cache[2][table[i, 0]] = 0.0                                # scores of 0 too
    check_weighted(args)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 80, 33])
def test_attention_whole_tiles_of_bad_pages(cuda, dtype, kind, dim):
    """The pages of a row's first tiles are outside the pool: they count as absent."""
    page = 64
    q, cache, table, lens, scale = attention_inputs([500, 300, 190], 4, 2, dim, page, 8, dtype, kind, seed=2)
    bad = table.clone()
    bad[:, :2] = torch.tensor([-1, cache[0].shape[0]], dtype=torch.int32, device=cuda)
    out = attend((q, cache, bad, lens, scale))
    expect_status(44)
    check_weighted((q, cache, table[:, 2:].contiguous(), lens - 2 * page, scale), out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 48, 128])
@pytest.mark.parametrize("top", [1.6e38, 1.72e38, 2.5e38, 3.38e38])
def test_attention_of_the_largest_queries(cuda, dtype, kind, dim, top):
    """Elements of q up to the end of the range, over keys so small that the scores are ordinary ones."""
    args = attention_inputs([100, 300, 1], 4, 2, dim, 16, 16, dtype, kind, seed=6)
    q, cache, table, lens, _ = args
    q.copy_(torch.randn(q.shape, device=cuda).clamp(-3, 3) / 3 * top)
    q[0, :, 3], q[1, :, 5] = top, -top
    cache[2].mul_(1e-36)
    check_weighted((q, cache, table, lens, 0.05))
    check_weighted((q, cache, table, lens, -0.05))
