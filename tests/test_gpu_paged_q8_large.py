"""The quantising write and append of calls that are large enough for their forms that take a block's tokens together
(the smaller ones of test_gpu_paged_q8.py take a token per warp), against the definition in 64 bits."""

import pytest
import torch

from engpt_b200 import _lib, kernels as K
from tests import paged_q8_blocks as B, paged_q8_ref as Q
from tests.test_gpu_paged_q8 import DTYPES, KINDS, append_error, append_inputs, rows

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean(cuda):
    _lib.clear_device_status()
    with torch.no_grad():
        yield
    status = _lib.device_status()
    _lib.clear_device_status()
    assert status == 0, f"a kernel recorded a device-side failure: {status:#x}"


def state(cache):
    return [c.view(torch.uint8).clone() if c.dim() == 4 else c.clone() for c in cache]


def check_both(cache, before, k, v, slots, err_k=0.0, err_v=0.0, dead=None):
    B.check_store(cache[0], cache[2], before[0], before[2], k, slots, err_k, dead)
    B.check_store(cache[1], cache[3], before[1], before[3], v, slots, err_v, dead)


def held(dim, dtype):
    """Tokens that a warp of the form holds at once: 32 lanes of 8 elements, times 4 (bf16) or 2 (fp32)."""
    lanes = next(n for n in (2, 4, 8, 16, 32) if 8 * n >= dim)
    return 32 // lanes * (4 if dtype == torch.bfloat16 else 2)


def sizes(heads, append, bsz=5):
    """Tokens of each of bsz requests, so that a call has more (token, head) rows than the one-token form takes: 256 per
    SM of q and of k and v (append), 64 per SM (write)."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    least = sms * (128 if append else 64) // heads + 1
    return -(-least // bsz) + 11


def layout_of(dim, dtype, blocks):
    """(block, page): a run fits a warp's registers in one load, in two, needs a team of warps, or more than it holds."""
    block = {"one": 1, "two": 2, "team": 4, "long": 16, "odd": 3}[blocks] * held(dim, dtype)
    if blocks == "odd":
        block -= 1
    return block, block * (1 if block >= 64 else 2)


FORMS = ["one", "two", "team", "long", "odd"]
DIMS = [(32, 16), (24, 32), (16, 64), (5, 80), (16, 128), (8, 256)]    # heads, head_dim


def requests(heads, dim, dtype, blocks, append):
    """Requests that begin at a page, inside blocks, at a block's last slot; some are padded, so that no window of tokens
    is one of the cache's blocks."""
    block, page = layout_of(dim, dtype, blocks)
    tokens = sizes(heads, append)
    first = [0, block // 2 + 1, block - 1, page - 1, block // 3]
    pool = 5 * ((tokens + page) // page + 2)
    slots = Q.prompt_slots(first, tokens, page, pool, dim + block, pad=(0, 3, tokens // 2, 0, min(block + 1, tokens - 1)))
    return block, page, pool, tokens, slots.cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dim", DIMS)
@pytest.mark.parametrize("blocks", FORMS)
def test_write_prompts(cuda, kind, dtype, heads, dim, blocks):
    block, page, pool, tokens, slots = requests(heads, dim, dtype, blocks, False)
    cache = Q.make_pools(pool, heads, page, dim, block, kind, "token" if dim == 64 else "head")
    Q.fill_pools(cache, dim, -6.0, 0.0)
    before = state(cache)
    k, v = rows(5 * tokens, heads, dim, dtype, dim)
    K.write_kv_pages_q8(k.unflatten(0, (5, tokens)), v.unflatten(0, (5, tokens)), slots, *cache)
    check_both(cache, before, k.double(), v.double(), slots.flatten())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dim", DIMS)
@pytest.mark.parametrize("blocks", FORMS)
def test_append_prompts(cuda, kind, dtype, heads, dim, blocks):
    block, page, pool, tokens, slots = requests(heads, dim, dtype, blocks, True)
    cache = Q.make_pools(pool, heads, page, dim, block, kind, "token" if dim == 64 else "head")
    Q.fill_pools(cache, dim, -6.0, 0.0)
    before = state(cache)
    lead = (5, tokens)
    qkv, rho, cos, sin, scale, pos = append_inputs(5 * tokens, heads, dim, dtype, dim)
    keep = qkv.clone()
    q = K.qkv_append_from_carried_q8(qkv.unflatten(0, lead), rho.view(lead), cos, sin, scale, 1e-6, pos.view(lead), slots,
                                     *cache)
    assert torch.equal(qkv, keep)
    rq, rk, rv = B.postprocess(qkv, rho, cos, sin, scale, 1e-6, pos)
    check_both(cache, before, rk, rv, slots.flatten(), append_error(rk), append_error(rv))
    assert ((q.flatten(0, 1).double() - rq).abs() <= torch.finfo(dtype).eps / 2 * rq.abs() + append_error(rq)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("block", [16, 64])
def test_append_a_token_each(cuda, kind, dtype, block):
    """Thousands of requests that add one token: windows of tokens that are as many runs."""
    heads, dim, page = 16, 64, 64
    n = sizes(heads, True, 1) + 300
    qkv, rho, cos, sin, scale, pos = append_inputs(n, heads, dim, dtype, block)
    gen = torch.Generator().manual_seed(n)
    slots = (torch.randperm(n, generator=gen) * page + torch.randint(0, page, (n,), generator=gen)).to(torch.int32).cuda()
    slots[::13] = -1
    cache = Q.make_pools(n, heads, page, dim, block, kind)
    Q.fill_pools(cache, n, -6.0, 0.0)
    before = state(cache)
    q = K.qkv_append_from_carried_q8(qkv, rho, cos, sin, scale, 1e-6, pos, slots, *cache)
    rq, rk, rv = B.postprocess(qkv, rho, cos, sin, scale, 1e-6, pos)
    check_both(cache, before, rk, rv, slots, append_error(rk), append_error(rv))
    assert ((q.double() - rq).abs() <= torch.finfo(dtype).eps / 2 * rq.abs() + append_error(rq)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("blocks", ["one", "two", "team", "long"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_numbers_that_are_none(cuda, kind, dtype, blocks, bad):
    """One bad element of a row: its head's block of its pool is NaN (of k and q's row where it is in k or q), every other
    number is one."""
    heads, dim = 16, 128
    block, page = layout_of(dim, dtype, blocks)
    tokens = sizes(heads, True, 1)
    slots = torch.arange(tokens, dtype=torch.int32, device=cuda)
    at, h = tokens * 2 // 3, 5
    nan = torch.zeros(tokens, heads, dim, dtype=torch.bool, device=cuda)
    nan[at // block * block:at // block * block + block, h] = True
    k, v = (torch.randn(tokens, heads, dim, device=cuda).to(dtype) for _ in range(2))
    v[at, h, 77] = bad
    cache = Q.make_pools(tokens // page + 1, heads, page, dim, block, kind)
    K.write_kv_pages_q8(k, v, slots, *cache)
    got_k, got_v = K.read_kv_pages_q8(slots, *cache, dtype=torch.float32)
    assert torch.equal(got_v.isnan(), nan) and got_k.isfinite().all()

    for part in range(3):
        qkv, rho, cos, sin, scale, pos = append_inputs(tokens, heads, dim, dtype, 3)
        qkv[at, part, h, 3] = bad
        q = K.qkv_append_from_carried_q8(qkv, rho, cos, sin, scale, 1e-6, pos, slots, *cache)
        got_k, got_v = K.read_kv_pages_q8(slots, *cache, dtype=torch.float32)
        if part == 0:
            assert q[at, h].isnan().any() and q.isnan().any(-1).sum() == 1
        else:
            assert q.isfinite().all()
        for i, got in ((1, got_k), (2, got_v)):
            assert torch.equal(got.isnan(), nan) if part == i else got.isfinite().all()
