"""Corners of the 8-bit paged cache operators on B200: numbers of extreme size, tokens that are left out, scales that are
zero or far apart."""

import pytest
import torch

from engpt_b200 import _lib, kernels as K
from tests import paged_q8_blocks as B, paged_q8_ref as Q
from tests.test_gpu_paged_q8 import DTYPES, KINDS, append_error, append_inputs, expect_status
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
