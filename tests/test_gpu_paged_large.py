"""Paged key-value cache operators on B200 at the sizes that reach their large-launch code, and with inputs in which every
key counts."""

import numpy as np
import pytest
import torch

from engpt_b200 import kernels as K
from tests import paged_ref as R
from tests.test_gpu_paged import (_clean, append_inputs, append_tolerance, attention_inputs, check_attention,  # noqa: F401
                                  make_pools, random_slots)

pytestmark = pytest.mark.gpu


def split_slots(n, pool, page, seed):
    """Distinct random slots, every seventh token (and the last) without one."""
    slots = random_slots(n, pool, page, seed)
    slots[::7] = -1
    slots[-1] = -1
    return slots


def store(pages, rows, slots):
    """What the pool is to hold: plain torch indexing."""
    page, live = pages.shape[2], slots >= 0
    at = slots[live].long()
    want = pages.clone()
    want[at // page, :, at % page] = rows[live]
    return want


# ------------------------------------------------------------------ append
# walking CTAs begin at 2368 tokens of 16 heads of 64 and 1184 of 16 of 128 (148 SMs, 2048 threads each); with several
# tokens side by side at 148 * 2048 / 128 groups of 128 / lanes tokens: 2 heads of 16 have 4 lanes, 3 of 48 (padded to 8
# lanes a row) 24, 5 of 80 80
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("n,heads,dim,page", [(2369, 16, 64, 16), (5003, 16, 64, 64), (2501, 16, 128, 16),
                                              (5003, 16, 128, 24), (4001, 12, 64, 16), (80001, 2, 16, 16),
                                              (16007, 3, 48, 8), (6007, 5, 80, 16), (2500, 7, 256, 16)])
def test_append_large(cuda, dtype, layout, n, heads, dim, page):
    rows = 3000
    pool = n // page + 3
    qkv, rho, cos, sin, scale, pos = append_inputs(n, heads, dim, dtype, n, rows=rows)
    kp, vp = make_pools(pool, heads, page, dim, dtype, layout)
    slots = split_slots(n, pool, page, n)
    before = kp.clone()
    q = K.qkv_append_from_carried(qkv, rho, cos, sin, scale, 1e-6, pos, slots, kp, vp)
    # each token's own rotary row makes the whole-sequence operator do the same
    at = pos.long()
    q2, k2, v2 = K.qkv_postprocess_from_carried(qkv[None], rho[None], cos[at], sin[at], scale, 1e-6)
    wk, wv = store(before, k2[0], slots), store(before, v2[0], slots)
    if dim in (16, 64, 128) and 3 * heads * dim // 8 <= 768 and 3 * heads * dim // 8 % 32 == 0:
        assert torch.equal(q, q2[0]) and torch.equal(kp, wk) and torch.equal(vp, wv)
    else:       # that operator's kernel for any size divides where this one multiplies by the reciprocal
        for got, want in ((q, q2[0]), (kp, wk), (vp, wv)):
            want = want.double()
            assert ((got.double() - want).abs() <= 2 * append_tolerance(dtype, want)).all()


def test_append_large_at_given_values(cuda):
    """The same size against 64-bit arithmetic."""
    n, heads, dim, page = 5003, 16, 64, 16
    for dtype in (torch.float32, torch.bfloat16):
        qkv, rho, cos, sin, scale, pos = append_inputs(n, heads, dim, dtype, 1)
        kp, vp = make_pools(n // page + 3, heads, page, dim, dtype)
        slots = split_slots(n, n // page + 3, page, 2)
        q = K.qkv_append_from_carried(qkv, rho, cos, sin, scale, 1e-6, pos, slots, kp, vp)
        rq, rk, rv = R.postprocess(qkv, rho, cos, sin, scale, 1e-6, pos)
        live = slots.cpu() >= 0
        at = slots.cpu()[live].long()
        for got, ref in ((q.cpu(), rq), (kp.cpu()[at // page, :, at % page], rk[live]),
                         (vp.cpu()[at // page, :, at % page], rv[live])):
            assert ((got.double() - ref).abs() <= append_tolerance(dtype, ref)).all()


# ------------------------------------------------------------------ write
# a thread's second piece carries data above 148 * 8 * 256 = 303104 pieces, and it comes back for a third above twice that
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["head", "token", "both", "odd"])
@pytest.mark.parametrize("n,heads,dim,page", [(2501, 16, 64, 16), (5999, 16, 64, 64), (20011, 16, 64, 16),
                                              (9001, 5, 80, 24), (30011, 3, 33, 7)])
def test_write_large(cuda, dtype, layout, n, heads, dim, page):
    pool = n // page + 3
    gen = torch.Generator(device="cuda").manual_seed(n)
    packed = torch.randn(n, 3, heads, dim, generator=gen, device="cuda").to(dtype)
    kp, vp = make_pools(pool, heads, page, dim, dtype, layout)
    before = kp.clone()
    slots = split_slots(n, pool, page, n)
    K.write_kv_pages(packed[:, 1], packed[:, 2], slots, kp, vp)
    assert torch.equal(kp, store(before, packed[:, 1], slots))
    assert torch.equal(vp, store(before, packed[:, 2], slots))


# ------------------------------------------------------------------ attention in which every key counts
def counting_inputs(lengths, heads, kv_heads, dim, page, dtype, levels, width=None, seed=0):
    """Values that are unit vectors, eight keys in turn on one axis, so that the output along an axis is the weight of its
    keys alone (no cancellation): a key left out, or counted twice, changes its axis by its share of it.  The scores are a
    level of -3 to 0 per eight keys, rising along the cache, or all 0 (`levels` false: all weights are 1)."""
    rng = np.random.default_rng(seed)
    bsz, most = len(lengths), max(lengths)
    pool = sum(R.pages_of(n, page) for n in lengths) + 1
    table, _ = R.random_table(lengths, page, width or max(1, R.pages_of(most, page)), pool, rng)
    table = table.cuda()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kp, vp = (torch.full((pool, kv_heads, page, dim), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    q = torch.zeros(bsz, heads, dim, dtype=dtype, device="cuda")
    q[:, :, 0] = torch.randint(1, 4, (bsz, heads), generator=gen, device="cuda").to(dtype) / 4
    level = torch.zeros(bsz, kv_heads, most, dtype=dtype, device="cuda")
    if levels:
        steps = torch.randint(-8, 1, (bsz, kv_heads, -(-most // 8)), generator=gen, device="cuda") / 8
        level = (steps.repeat_interleave(8, 2)[:, :, :most] + 3.0 * torch.arange(most, device="cuda") / most).to(dtype)
    axis = (torch.arange(most, device="cuda") // 8) % dim
    out = torch.zeros(bsz, heads, dim, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        j = torch.arange(n, device="cuda")
        pages, off = table[b, j // page].long(), j % page
        k, v = (torch.zeros(n, kv_heads, dim, dtype=dtype, device="cuda") for _ in range(2))
        k[:, :, 0] = level[b, :, :n].t()
        v[j, :, axis[:n]] = 1.0
        kp[pages, :, off], vp[pages, :, off] = k, v
        s = q[b, :, 0].double()[:, None] * level[b, :, :n].double().repeat_interleave(heads // kv_heads, 0)
        out[b].index_add_(1, axis[:n], torch.softmax(s, -1))
    return (q, kp, vp, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), 1.0 if levels else 0.0), out


def counting_tolerance(dtype, levels):
    """Relative, as nothing cancels.  One rounding of the result and 2^-22 for the division.  With scores (up to 3.3 in
    base-2 units): four roundings of such a number move a weight by 4 * 3.3 ln 2 * 2^-24 = 9.2 * 2^-24, the exponential by
    2 units more, 4 * 2^-24; a rise of the running maximum and a join multiply by another such exponential, 14.2 * 2^-24
    with the product's rounding, at most 512 of them on any key's way (4096 keys of a row in 16 lane groups, and the joins);
    4096 additions of 2^-24.  Sum and divisor both carry this.  In bf16 the weights have 16 bits: 2^-17 each, twice."""
    tol = torch.finfo(dtype).eps / 2 + 2.0 ** -22
    if levels:
        tol += 2 * (512 * 14.2 + 4096 + 13.2) * 2.0 ** -24
        if dtype == torch.bfloat16:
            tol += 2 * 2.0 ** -17
    return tol


COUNTING = [
    # lengths, heads, kv heads, dim, page, table width in pages (None: the longest row)
    ([257], 4, 4, 64, 16, None), ([257], 4, 4, 64, 16, 512), ([5000], 2, 2, 64, 16, None),
    ([8192], 16, 16, 64, 64, None), ([8192], 16, 16, 128, 64, None), ([9001], 16, 16, 128, 64, None),
    ([8190], 32, 4, 128, 64, None), ([8192], 12, 1, 64, 16, None), ([4097, 37], 4, 4, 64, 128, None),
    ([2500, 37, 37], 3, 3, 80, 16, None), ([512] * 20, 4, 4, 64, 64, None), ([1024, 0, 5, 700] * 3, 16, 2, 64, 16, None),
    ([4096 - 65 * b for b in range(64)], 16, 16, 64, 16, None), ([2 * b + 1 for b in range(256)], 16, 16, 64, 16, None),
    ([b % 129 for b in range(256)], 16, 16, 64, 16, None), ([2048] * 4 + [31] * 29, 8, 2, 128, 32, None),
    ([1021, 700, 300, 64, 1], 4, 4, 33, 16, None), ([6001], 2, 1, 256, 16, None),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("levels", [False, True])
@pytest.mark.parametrize("case", COUNTING, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[1]}on{c[2]}-{c[3]}-{c[4]}-{c[5]}")
def test_attention_counts_every_key(cuda, dtype, levels, case):
    lengths, heads, kv_heads, dim, page, width = case
    args, want = counting_inputs(lengths, heads, kv_heads, dim, page, dtype, levels, width, seed=max(lengths))
    got = K.paged_sdpa(*args[:5], scale=args[5]).double()
    tol = counting_tolerance(dtype, levels)
    err = (got - want).abs()
    assert (err <= tol * want).all(), f"max relative error {(err / want.clamp(min=1e-30)).max().item()}, allowed {tol}"


def test_the_counting_inputs_show_a_lost_or_doubled_tile(cuda):
    """The mistake is made in the expected values: without 8 keys, or with a tile of 32 or 64 keys twice, each differs by
    more than the tolerance."""
    for dtype in (torch.float32, torch.bfloat16):
        for levels in (False, True):
            (q, kp, vp, table, lens, scale), want = counting_inputs([8190], 2, 1, 64, 16, dtype, levels)
            row = table[0].long()
            k, v = (x[row, 0].reshape(-1, 64)[:8190].double() for x in (kp, vp))
            w = torch.exp(scale * (k @ q[0].double().t()) - 3.0).t()
            for a, n, times in ((0, 8, 0.0), (4096, 8, 0.0), (8184, 6, 0.0), (4096, 64, 2.0), (64, 32, 2.0), (0, 64, 0.0)):
                x = w.clone()
                x[:, a:a + n] *= times
                wrong = (x @ v) / x.sum(-1, keepdim=True)
                assert ((wrong - want[0]).abs() > counting_tolerance(dtype, levels) * want[0]).any()
            assert torch.allclose((w @ v) / w.sum(-1, keepdim=True), want[0], rtol=1e-9, atol=0)


# ------------------------------------------------------------------ offsets
@pytest.mark.parametrize("dtype,page", [(torch.bfloat16, 128), (torch.bfloat16, 100), (torch.float32, 128)])
@pytest.mark.parametrize("heads,dim", [(16, 128), (15, 100)])
def test_far_into_a_pool(cuda, dtype, page, heads, dim):
    """Elements whose index passes 2^32: append (both kernels), write and attention (both kinds), against a small pool."""
    pool = 2 ** 32 // (2 * heads * page * dim) + 40
    kv = torch.empty(pool, 2, heads, page, dim, dtype=dtype, device=cuda)
    kp, vp = kv[:, 0], kv[:, 1]
    ids = torch.tensor([pool - 1, pool // 2 + 1, 0, pool - 7], device=cuda)
    assert (pool - 7) * kp.stride(0) > 2 ** 32
    kv[ids] = 0.0
    near = torch.zeros(4, 2, heads, page, dim, dtype=dtype, device=cuda)
    n = 4 * page - 3
    qkv, rho, cos, sin, scale, pos = append_inputs(n, heads, dim, dtype, 3, rows=600)
    at = torch.arange(n, device=cuda)
    slots = (ids[at // page] * page + at % page).int()
    q = K.qkv_append_from_carried(qkv, rho, cos, sin, scale, 1e-6, pos, slots, kp, vp)
    assert torch.equal(q, K.qkv_append_from_carried(qkv, rho, cos, sin, scale, 1e-6, pos, at.int(), near[:, 0],
                                                    near[:, 1]))
    assert torch.equal(kv[ids], near) and (near != 0).any()
    K.write_kv_pages(qkv[:100, 1], qkv[:100, 2], slots[7:107], kp, vp)
    K.write_kv_pages(qkv[:100, 1], qkv[:100, 2], at[7:107].int(), near[:, 0], near[:, 1])
    assert torch.equal(kv[ids], near)
    lens = torch.tensor([n], dtype=torch.int32, device=cuda)
    far = K.paged_sdpa(q[:1], kp, vp, ids.int()[None], lens, scale=0.1)
    assert torch.equal(far, K.paged_sdpa(q[:1], near[:, 0], near[:, 1], torch.arange(4, device=cuda).int()[None], lens,
                                         scale=0.1))


# ------------------------------------------------------------------ long chains of early starts
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bsz,width", [(2, 6), (3, 200), (300, 6)])
def test_long_eager_chains(cuda, dtype, bsz, width):
    """Calls back to back without a graph, each on the results of the one before: kernels that start ahead of their
    predecessors' end must still see all of them.  The same chain with a synchronisation after every call is the
    expected value, bit for bit."""
    heads, dim, page, layers, steps = 4, 64, 16, 12, 8
    qkv, rho, cos, sin, scale, _ = append_inputs(bsz * layers, heads, dim, dtype, bsz)
    qkv, rho = qkv.view(layers, bsz, 3, heads, dim), rho.view(layers, bsz)

    def chain(wait):
        i32 = dict(dtype=torch.int32, device=cuda)
        table, lengths = torch.full((bsz, width), -1, **i32), torch.zeros(bsz, **i32)
        free, count, ones = torch.arange(bsz * 6, **i32), torch.tensor([bsz * 6], **i32), torch.ones(bsz, **i32)
        pools = [make_pools(bsz * 6, heads, page, dim, dtype, fill=float("nan")) for _ in range(layers)]
        outs = []
        for _ in range(steps):
            slots, pos = K.advance_block_tables(lengths, ones, table, free, count, page_size=page, max_new=1)
            wait()
            slots, pos, o = slots.view(bsz), pos.view(bsz), None
            for i, (kp, vp) in enumerate(pools):
                x = qkv[i]
                if i % 3 == 1:       # on the attention's result, through a kernel of torch
                    x = x * (1.0 + o[:, None])
                q = K.qkv_append_from_carried(x, rho[i], cos, sin, scale, 1e-6, pos, slots, kp, vp)
                wait()
                if i % 3 == 2:       # the last values once more, from the attention's result as it is
                    K.write_kv_pages(q, o, slots, kp, vp)
                    wait()
                o = K.paged_sdpa(q, kp, vp, table, lengths, scale=4.0)
                wait()
                outs.append(o)
        return outs + [t for p in pools for t in p]

    want = chain(torch.cuda.synchronize)
    for _ in range(3):
        got = chain(lambda: None)
        assert all(torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0)) for a, b in zip(got, want))
