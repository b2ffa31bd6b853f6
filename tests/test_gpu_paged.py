"""Paged key-value cache operators on B200, against plain 64-bit forms (tests/paged_ref.py)."""

import math

import numpy as np
import pytest
import torch

from engpt_b200 import _lib, kernels as K
from tests import paged_ref as R

pytestmark = pytest.mark.gpu

ERR_ARG = 7


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


# ------------------------------------------------------------------ block tables
class Tables:
    def __init__(self, lengths, page, width, pool, seed=0, stride=None):
        rng = np.random.default_rng(seed)
        self.page, self.width, self.pool = page, width, pool
        table, left = R.random_table(lengths, page, width, pool, rng)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        buf = torch.full((len(lengths), stride or width), -7, dtype=torch.int32, device="cuda")
        self.buf = buf
        self.table = buf[:, :width]
        self.table.copy_(table)
        self.free = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
        self.free[:len(left)] = torch.tensor(left, dtype=torch.int32)
        self.count = torch.tensor([len(left)], dtype=torch.int32, device="cuda")

    def step_and_compare(self, new, max_new, finished=None):
        ref = R.advance(self.lengths.tolist(), new, self.table.tolist(), self.free.tolist(), int(self.count),
                        self.page, max_new, finished)
        fin = None if finished is None else torch.tensor(finished, dtype=torch.bool, device="cuda")
        slots, pos = K.advance_block_tables(self.lengths, torch.tensor(new, dtype=torch.int32, device="cuda"),
                                            self.table, self.free, self.count, page_size=self.page, max_new=max_new,
                                            finished=fin)
        n = ref[5]
        assert slots.tolist() == ref[0]
        assert pos.tolist() == ref[1]
        assert self.lengths.tolist() == ref[2]
        assert self.table.tolist() == ref[3]
        assert int(self.count) == n
        assert self.free.tolist()[:n] == ref[4][:n]
        if self.buf.shape[1] > self.width:
            assert (self.buf[:, self.width:] == -7).all()      # behind the table's rows: left as it was
        return slots, pos


@pytest.mark.parametrize("bsz,page", [(1, 1), (3, 16), (31, 7), (64, 16), (257, 8), (1025, 16), (3000, 64)])
def test_tables_many_steps(cuda, bsz, page):
    rng = np.random.default_rng(bsz)
    width = 6
    lengths = rng.integers(0, 3 * page + 1, bsz).tolist()
    lengths[0] = 0
    t = Tables(lengths, page, width, bsz * width + 5, seed=bsz, stride=width + 3)
    t.step_and_compare(rng.integers(0, 2 * page + 1, bsz).tolist(), 2 * page)
    for step in range(4):
        fin = (rng.random(bsz) < 0.3).tolist() if step % 2 else None
        # a row that would overrun its table row is asked for nothing
        new = [1 if n < width * page else 0 for n in t.lengths.tolist()]
        t.step_and_compare(new, 1, fin)


def test_tables_prompts_longer_than_a_block(cuda):
    t = Tables([0, 5, 0, 64, 130], 64, 40, 220)
    t.step_and_compare([2048, 2000, 1, 0, 1777], 2048, [False, False, False, True, False])


def test_tables_all_rows_finish_and_start_again(cuda):
    t = Tables([100, 33, 1, 0], 16, 8, 12)
    t.step_and_compare([0, 0, 0, 0], 1, [True] * 4)
    assert int(t.count) == 12 and sorted(t.free.tolist()) == list(range(12))
    t.step_and_compare([1, 17, 100, 5], 128)


@pytest.mark.parametrize("left", [0, 1])
def test_tables_refuse_rows_on_the_device(cuda, left):
    t = Tables([16, 30, 8, 4], 16, 4, 5 + left)    # 1 + 2 + 1 + 1 pages are in use
    t.step_and_compare([0, 1, 1, 1], 1)
    assert int(t.count) == left
    t.step_and_compare([1, 2, 1, 1], 2)            # row 0 takes the last page, row 1 (now 31 tokens) needs another
    expect_status(41)
    t.step_and_compare([3, 0, -1, 1], 2)           # more than max_new, and a negative count
    expect_status(40)
    assert t.lengths.tolist() == [16 + left, 31, 10, 7]
    wide = Tables([16, 5], 16, 1, 8)
    wide.step_and_compare([1, 1], 1)               # the first row's table is full
    expect_status(40)


def test_tables_zero_sizes(cuda):
    i32 = dict(dtype=torch.int32, device=cuda)
    s, p = K.advance_block_tables(torch.zeros(0, **i32), torch.zeros(0, **i32), torch.zeros(0, 3, **i32),
                                  torch.zeros(4, **i32), torch.tensor([4], **i32), page_size=16, max_new=5)
    assert s.shape == (0, 5) and p.shape == (0, 5)
    t = Tables([3, 4], 16, 2, 4)
    t.step_and_compare([0, 0], 0, [True, False])


# ------------------------------------------------------------------ append and write
def make_pools(pool, heads, page, dim, dtype, layout="head", fill=7.5):
    """Page pools [P, H, ps, Dh] in one of the layouts a user may hold, filled with a mark."""
    if layout == "head":
        k, v = (torch.full((pool, heads, page, dim), fill, dtype=dtype, device="cuda") for _ in range(2))
    elif layout == "token":          # stored [P, ps, H, Dh]
        k, v = (torch.full((pool, page, heads, dim), fill, dtype=dtype, device="cuda").transpose(1, 2)
                for _ in range(2))
    elif layout == "both":           # k and v of a page side by side
        kv = torch.full((pool, 2, heads, page, dim), fill, dtype=dtype, device="cuda")
        k, v = kv[:, 0], kv[:, 1]
    else:                            # "odd": rows one element longer than head_dim, the pools not 16-byte aligned
        k, v = (torch.full((pool, heads, page, dim + 1), fill, dtype=dtype, device="cuda")[..., 1:]
                for _ in range(2))
    return k, v


def random_slots(n, pool, page, seed, skip=()):
    rng = np.random.default_rng(seed)
    slots = rng.permutation(pool * page)[:n].astype(np.int32)
    for i in skip:
        slots[i] = -1
    return torch.from_numpy(slots).cuda()


def check_store(pages, before, rows, slots, exact):
    """Rows are in their slots (`exact`: bit for bit, else compared by the caller); the rest is untouched."""
    page = pages.shape[2]
    got = []
    want = before.clone()
    for i, s in enumerate(slots.reshape(-1).tolist()):
        if s >= 0:
            got.append(pages[s // page, :, s % page])
            want[s // page, :, s % page] = got[-1]
            if exact:
                assert torch.equal(got[-1], rows[i])
    assert torch.equal(pages, want)
    return torch.stack(got) if got else None


@pytest.mark.parametrize("layout", ["head", "token", "both", "odd"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,dim,page", [(16, 64, 16), (3, 48, 7), (2, 33, 1), (16, 128, 64)])
def test_write_pages(cuda, layout, dtype, heads, dim, page):
    n, pool = 41, 41 // page + 4
    gen = torch.Generator(device="cuda").manual_seed(heads + dim)
    packed = torch.randn(1, n, 3, heads, dim, generator=gen, device="cuda").to(dtype)
    k, v = packed[:, :, 1], packed[:, :, 2]
    kp, vp = make_pools(pool, heads, page, dim, dtype, layout)
    before = kp.clone()
    slots = random_slots(n, pool, page, 3, skip=(0, 17, 40)).view(1, n)
    K.write_kv_pages(k, v, slots, kp, vp)
    check_store(kp, before, k[0], slots, True)
    check_store(vp, before, v[0], slots, True)


def test_write_pages_strided_and_bad_slots(cuda):
    heads, dim, page, pool = 4, 64, 16, 5
    k = torch.randn(6, 2 * heads, dim, device=cuda)[:, ::2]
    v = torch.randn(heads, 6, dim, device=cuda).transpose(0, 1)
    kp, vp = make_pools(pool, heads, page, dim, torch.float32)
    before = kp.clone()
    slots = torch.tensor([3, -1, 79, 80, -2, 2 ** 31 - 1], dtype=torch.int32, device=cuda)
    K.write_kv_pages(k, v, slots, kp, vp)
    expect_status(43)
    ok = torch.tensor([3, -1, 79, -1, -1, -1])
    check_store(kp, before, k, ok, True)
    check_store(vp, before, v, ok, True)
    K.write_kv_pages(k[:0], v[:0], slots[:0], kp, vp)
    check_store(kp, before, k, ok, True)


def append_inputs(n, heads, dim, dtype, seed, rows=300):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rho = torch.exp(torch.randn(n, generator=gen, device="cuda"))
    qkv = (torch.randn(n, 3, heads, dim, generator=gen, device="cuda") * rho.view(-1, 1, 1, 1)).to(dtype)
    if n > 2:
        qkv[2, 0, 0] *= 1e-9             # the rho * eps guard
    cos, sin = K.rotary_frequencies(rows, dim, device=torch.device("cuda", 0), dtype=torch.float32, theta=10000.0)
    scale = 1.0 + 0.1 * torch.randn(heads, dim, generator=gen, device="cuda")
    pos = torch.randint(0, rows, (n,), generator=gen, device="cuda", dtype=torch.int32)
    return qkv, rho, cos, sin, scale, pos


def append_tolerance(dtype, ref):
    """A result is x * c / norm * s: an fp32 sum of dim squares and some ten fp32 operations, or the approximate
    reciprocals of the bf16 path (2 ulp each), then one rounding: half a step and 2^-18 of the row's largest value
    (the rotation's difference of two products can cancel)."""
    return torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -18 * ref.abs().amax(-1, keepdim=True)


@pytest.mark.parametrize("layout", ["head", "token", "odd"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,dim,page,n", [(16, 64, 16, 1), (4, 64, 16, 37), (16, 128, 64, 70), (5, 80, 8, 9),
                                              (3, 33, 5, 12), (2, 16, 16, 33), (12, 64, 16, 18)])
def test_append(cuda, layout, dtype, heads, dim, page, n):
    pool = n // page + 5
    qkv, rho, cos, sin, scale, pos = append_inputs(n, heads, dim, dtype, dim + n)
    kp, vp = make_pools(pool, heads, page, dim, dtype, layout)
    before = kp.clone()
    slots = random_slots(n, pool, page, n, skip=(3,) if n > 3 else ())
    keep = qkv.clone()
    q = K.qkv_append_from_carried(qkv, rho, cos, sin, scale, 1e-6, pos, slots, kp, vp)
    assert torch.equal(qkv, keep)
    rq, rk, rv = R.postprocess(qkv, rho, cos, sin, scale, 1e-6, pos)
    live = slots.cpu() >= 0
    gk = check_store(kp, before, None, slots, False).cpu().double()
    gv = check_store(vp, before, None, slots, False).cpu().double()
    for got, ref in ((q.cpu().double(), rq), (gk, rk[live]), (gv, rv[live])):
        assert ((got - ref).abs() <= append_tolerance(dtype, ref)).all()


def test_append_matches_the_whole_sequence_op(cuda):
    """At positions 0 .. T-1 the results are those of qkv_postprocess_from_carried, bit for bit."""
    bsz, seq, heads, dim, page = 2, 45, 16, 64, 16
    for dtype in (torch.float32, torch.bfloat16):
        qkv, rho, cos, sin, scale, _ = append_inputs(bsz * seq, heads, dim, dtype, 5)
        qkv, rho = qkv.view(bsz, seq, 3, heads, dim), rho.view(bsz, seq)
        pos = torch.arange(seq, dtype=torch.int32, device=cuda).repeat(bsz, 1)
        kp, vp = make_pools(8, heads, page, dim, dtype)
        slots = random_slots(bsz * seq, 8, page, 1).view(bsz, seq)
        q = K.qkv_append_from_carried(qkv, rho, cos, sin, scale, 1e-6, pos, slots, kp, vp)
        q2, k2, v2 = K.qkv_postprocess_from_carried(qkv, rho, cos, sin, scale, 1e-6)
        assert torch.equal(q, q2)
        check_store(kp, torch.full_like(kp, 7.5), k2.view(-1, heads, dim), slots, True)
        check_store(vp, torch.full_like(vp, 7.5), v2.view(-1, heads, dim), slots, True)


@pytest.mark.parametrize("heads,dim", [(4, 64), (3, 33)])
def test_append_bad_positions_and_slots(cuda, heads, dim):
    qkv, rho, cos, sin, scale, pos = append_inputs(5, heads, dim, torch.float32, 1, rows=50)
    kp, vp = make_pools(2, heads, 16, dim, torch.float32)
    before = kp.clone()
    pos = torch.tensor([50, -1, 49, 0, 7], dtype=torch.int32, device=cuda)
    slots = torch.tensor([0, 1, 2, -1, 3], dtype=torch.int32, device=cuda)
    q = K.qkv_append_from_carried(qkv, rho, cos, sin, scale, 1e-6, pos, slots, kp, vp)
    expect_status(42)
    assert (q[:2] == 0).all() and (q[2:] != 0).any(-1).all()
    check_store(kp, before, None, torch.tensor([-1, -1, 2, -1, 3]), False)
    slots = torch.tensor([32, -2, 2, -1, 3], dtype=torch.int32, device=cuda)
    pos = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device=cuda)
    q2 = K.qkv_append_from_carried(qkv, rho, cos, sin, scale, 1e-6, pos, slots, kp, vp)
    expect_status(43)
    assert (q2 != 0).any(-1).all()
    check_store(vp, before, None, torch.tensor([-1, -1, 2, -1, 3]), False)


# ------------------------------------------------------------------ attention
def attention_inputs(lengths, heads, kv_heads, dim, page, dtype, layout="head", seed=0, spare_width=1, pool=None,
                     spread=1.0):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    width = max([R.pages_of(max(n, 0), page) for n in lengths] + [0]) + spare_width
    pool = pool or sum(R.pages_of(max(n, 0), page) for n in lengths) + 3
    table, _ = R.random_table(lengths, page, width, pool, rng)
    kp, vp = make_pools(pool, kv_heads, page, dim, dtype, layout, fill=float("nan"))
    # only the tokens of a request have values: everything behind a length is NaN
    for b, n in enumerate(lengths):
        for p in range(n):
            pg = int(table[b, p // page])
            kp[pg, :, p % page] = torch.randn(kv_heads, dim, generator=gen, device="cuda").to(dtype)
            vp[pg, :, p % page] = torch.randn(kv_heads, dim, generator=gen, device="cuda").to(dtype)
    q = (spread * torch.randn(len(lengths), heads, dim, generator=gen, device="cuda")).to(dtype)
    return (q, kp, vp, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"),
            1.0 / math.sqrt(dim))


def check_attention(args, out=None):
    q, kp, vp, table, lengths, scale = args
    if out is None:
        out = K.paged_sdpa(q, kp, vp, table, lengths, scale=scale)
    ref, vmax, smax = R.attention(q, kp, vp, table, lengths, scale)
    n = max(1, int(lengths.max()) if lengths.numel() else 1)
    tol = R.attention_tolerance(q.dtype, ref, vmax, smax, q.shape[2], n)
    err = (out.cpu().double() - ref).abs()
    assert (err <= tol).all(), f"max error {err.max().item()}, over its tolerance by {(err / tol).max().item()}"
    return out


LENGTHS = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 300]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 16, 80, 33, 256])
@pytest.mark.parametrize("page", [16, 64, 8, 24, 1])
def test_attention_lengths(cuda, dtype, dim, page):
    check_attention(attention_inputs(LENGTHS, 4, 4, dim, page, dtype, seed=dim + page))


@pytest.mark.parametrize("dim,page", [(8, 8), (24, 16), (40, 64), (96, 8), (104, 40), (120, 128), (136, 16), (7, 16)])
def test_attention_other_head_dims_bf16(cuda, dim, page):
    """Head dims that are padded in shared memory, and the ones next to them that are not."""
    check_attention(attention_inputs([0, 1, 100, 257, 33], 4, 2, dim, page, torch.bfloat16, seed=dim))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30, 3.0])
def test_attention_scales(cuda, dtype, dim, scale):
    args = attention_inputs([0, 5, 64, 333], 3, 3, dim, 16, dtype, seed=dim)
    check_attention(args[:5] + (scale,))


def test_attention_more_rows_than_the_list_takes(cuda):
    """9000 rows: beyond the tensor-core kernels' prefix sums."""
    bsz, page, heads, dim = 9000, 16, 2, 64
    rng = np.random.default_rng(1)
    lengths = rng.integers(0, 40, bsz).tolist()
    pool = sum(R.pages_of(n, page) for n in lengths)
    table, _ = R.random_table(lengths, page, 3, pool, rng)
    gen = torch.Generator(device="cuda").manual_seed(bsz)
    kp, vp = (torch.randn(pool, heads, page, dim, generator=gen, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(bsz, heads, dim, generator=gen, device="cuda").bfloat16()
    check_attention((q, kp, vp, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device=cuda), 0.125))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads", [(16, 16), (16, 2)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bsz,width_tokens", [(1, 64), (1, 512), (1, 2048), (1, 8192), (3, 512), (3, 2048), (12, 1024),
                                              (20, 512), (40, 256)])
def test_attention_every_form_with_short_and_long_rows(cuda, dtype, heads, kv_heads, dim, bsz, width_tokens):
    """The table's width decides the form (clusters of 1 to 8 CTAs, the list); the rows themselves may be of any length
    within it, the last one as long as the table allows."""
    page = 64
    rng = np.random.default_rng(bsz + width_tokens)
    lengths = [int(x) for x in rng.integers(0, 130, bsz)]
    lengths[-1] = width_tokens
    pool = sum(R.pages_of(n, page) for n in lengths) + 1
    table, _ = R.random_table(lengths, page, width_tokens // page, pool, rng)
    gen = torch.Generator(device="cuda").manual_seed(bsz)
    kp, vp = (torch.randn(pool, kv_heads, page, dim, generator=gen, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn(bsz, heads, dim, generator=gen, device="cuda").to(dtype)
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    check_attention((q, kp, vp, table.cuda(), lens, 0.125))
    lens[-1] = 3          # the same form, nothing left of the long row
    check_attention((q, kp, vp, table.cuda(), lens, 0.125))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (6, 2), (8, 1), (16, 2), (12, 1), (40, 2), (5, 5)])
@pytest.mark.parametrize("dim", [64, 128, 48])
def test_attention_head_groups(cuda, dtype, heads, kv_heads, dim):
    check_attention(attention_inputs([70, 0, 513, 1], heads, kv_heads, dim, 16, dtype, seed=heads))


@pytest.mark.parametrize("layout", ["token", "both", "odd"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (48, 16)])
def test_attention_cache_layouts(cuda, dtype, layout, dim, page):
    check_attention(attention_inputs([90, 300, 33], 6, 3, dim, page, dtype, layout=layout, seed=dim))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bsz,n,heads,dim,page", [(1, 5000, 2, 64, 16), (1, 9001, 16, 128, 64), (2, 4097, 4, 64, 128),
                                                  (3, 2500, 3, 80, 16)])
def test_attention_long(cuda, dtype, bsz, n, heads, dim, page):
    """One long request split over many CTAs, next to short ones."""
    lengths = [n] + [37] * (bsz - 1)
    q, kp, vp, table, lens, scale = attention_inputs([1] * bsz, heads, heads, dim, page, dtype, seed=n)
    gen = torch.Generator(device="cuda").manual_seed(n)
    pool = sum(R.pages_of(x, page) for x in lengths) + 2
    table, _ = R.random_table(lengths, page, R.pages_of(n, page) + 2, pool, np.random.default_rng(n))
    kp, vp = (torch.randn(pool, heads, page, dim, generator=gen, device="cuda").to(dtype) for _ in range(2))
    check_attention((q, kp, vp, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device=cuda), scale))


@pytest.mark.parametrize("bsz", [200, 1500])
def test_attention_many_rows(cuda, bsz):
    rng = np.random.default_rng(bsz)
    lengths = rng.integers(0, 90, bsz).tolist()
    lengths[5] = 700
    page, heads, dim = 16, 4, 64
    pool = sum(R.pages_of(n, page) for n in lengths) + 1
    table, _ = R.random_table(lengths, page, 44, pool, rng)
    gen = torch.Generator(device="cuda").manual_seed(bsz)
    kp, vp = (torch.randn(pool, heads, page, dim, generator=gen, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(bsz, heads, dim, generator=gen, device="cuda").bfloat16()
    check_attention((q, kp, vp, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device=cuda), 0.125))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 80])
def test_attention_rising_and_large_scores(cuda, dtype, dim):
    """The running maximum rises along the cache, and scores reach some hundreds."""
    args = list(attention_inputs([400, 130], 2, 2, dim, 16, dtype, seed=9, spread=20.0))
    for b, n in enumerate((400, 130)):
        for p in range(n):
            args[1][int(args[3][b, p // 16]), :, p % 16] *= 0.02 + p / n
    check_attention(tuple(args))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 48])
def test_attention_ignores_what_lies_behind_a_length(cuda, dtype, dim):
    """Stale, infinite and NaN rows behind a length, and table entries behind its pages, change no bit."""
    args = attention_inputs([5, 64, 0, 77], 2, 2, dim, 16, dtype, seed=3, spare_width=4)
    out = check_attention(args)
    q, kp, vp, table, lens, scale = args
    for fill in (float("inf"), -float("inf"), 3.0e38, 0.0):
        k2, v2 = (torch.where(x.isnan(), torch.full_like(x, fill), x) for x in (kp, vp))
        t2 = torch.where(table < 0, torch.full_like(table, 2 ** 31 - 1 if fill else kp.shape[0]), table)
        assert torch.equal(out, K.paged_sdpa(q, k2, v2, t2, lens, scale=scale))
    assert (out[2] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 48])
def test_attention_records_bad_pages_and_lengths(cuda, dtype, dim):
    q, kp, vp, table, lens, scale = attention_inputs([40, 40, 40], 2, 2, dim, 16, dtype, seed=4, spare_width=0)
    t2, l2 = table.clone(), lens.clone()
    t2[0, 1] = kp.shape[0]            # outside the pool: the middle 16 tokens count as absent
    out = K.paged_sdpa(q, kp, vp, t2, l2, scale=scale)
    expect_status(44)
    same = K.paged_sdpa(q, kp, vp, table, lens, scale=scale)
    assert torch.equal(out[1:], same[1:])
    # the same keys as a request of 24 tokens on the first and the last page, the first one filled up
    one = torch.tensor([[int(table[0, 0]), int(table[0, 2])]], dtype=torch.int32, device=cuda)
    ref, vmax, smax = R.attention(q[:1], kp, vp, one, torch.tensor([24]), scale)
    assert ((out[:1].cpu().double() - ref).abs()
            <= R.attention_tolerance(dtype, ref, vmax, smax, dim, 24)).all()
    t2 = table.clone()
    t2[2] = -5                        # no page at all: zeros
    out = K.paged_sdpa(q, kp, vp, t2, lens, scale=scale)
    expect_status(44)
    assert (out[2] == 0).all() and torch.equal(out[:2], same[:2])
    l2[1] = -3                        # negative: an empty row, not an error
    out = K.paged_sdpa(q, kp, vp, table, l2, scale=scale)
    assert (out[1] == 0).all()
    l2[1] = 1000                      # longer than its table row: cut there
    kp.nan_to_num_(0.25)
    vp.nan_to_num_(0.25)
    out = K.paged_sdpa(q, kp, vp, table, l2, scale=scale)
    expect_status(44)
    full = torch.tensor([40, 48, 40], dtype=torch.int32, device=cuda)
    assert torch.equal(out, K.paged_sdpa(q, kp, vp, table, full, scale=scale))


def test_attention_nan_in_a_key_stays_in_its_row(cuda):
    for dtype, dim in ((torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 48)):
        q, kp, vp, table, lens, scale = attention_inputs([300, 300], 2, 2, dim, 16, dtype, seed=6)
        good = K.paged_sdpa(q, kp, vp, table, lens, scale=scale)
        kp[int(table[0, 3]), 1, 5] = float("nan")
        out = K.paged_sdpa(q, kp, vp, table, lens, scale=scale)
        assert out[0, 1].isnan().all()
        assert torch.equal(out[0, 0], good[0, 0]) and torch.equal(out[1], good[1])


def test_attention_strided_queries_and_tables(cuda):
    q, kp, vp, table, lens, scale = attention_inputs([100, 7, 260], 4, 4, 64, 16, torch.bfloat16, seed=8)
    want = check_attention((q, kp, vp, table, lens, scale))
    packed = torch.zeros(3, 3, 4, 64, dtype=torch.bfloat16, device=cuda)
    packed[:, 1] = q
    wide = torch.full((3, table.shape[1] + 5), 9, dtype=torch.int32, device=cuda)
    wide[:, :table.shape[1]] = table
    assert torch.equal(want, K.paged_sdpa(packed[:, 1], kp, vp, wide[:, :table.shape[1]], lens, scale=scale))
    assert torch.equal(want, K.paged_sdpa(q.transpose(1, 2).contiguous().transpose(1, 2), kp, vp, table, lens,
                                          scale=scale))
    odd = torch.zeros(3, 4 * 64 + 1, dtype=torch.bfloat16, device=cuda)[:, 1:].view(3, 4, 64)
    odd.copy_(q)
    check_attention((odd, kp, vp, table, lens, scale))


def test_attention_offsets_beyond_32_bits(cuda):
    """Pages whose element offset passes 2^32 in a pool of 2.5 G elements (5 GB each, keys and values shared)."""
    page, heads, dim = 128, 16, 128
    pool = 10000                                    # 262144 elements a page
    kv = torch.zeros(pool, heads, page, dim, dtype=torch.bfloat16, device=cuda)
    ids = [9999, 8192, 0, 8193]
    gen = torch.Generator(device="cuda").manual_seed(1)
    for i in ids:
        kv[i] = torch.randn(heads, page, dim, generator=gen, device="cuda").bfloat16()
    small = kv[torch.tensor(ids, device=cuda)].clone()
    q = torch.randn(1, heads, dim, generator=gen, device="cuda").bfloat16()
    lens = torch.tensor([500], dtype=torch.int32, device=cuda)
    far = K.paged_sdpa(q, kv, kv, torch.tensor([ids], dtype=torch.int32, device=cuda), lens, scale=0.1)
    near = K.paged_sdpa(q, small, small, torch.tensor([[0, 1, 2, 3]], dtype=torch.int32, device=cuda), lens, scale=0.1)
    assert torch.equal(far, near)
    rows = torch.randn(3, heads, dim, generator=gen, device="cuda").bfloat16()
    slots = torch.tensor([9998 * page + 5, 8192 * page, 9999 * page + 127], dtype=torch.int32, device=cuda)
    K.write_kv_pages(rows, rows, slots, kv, kv)
    assert torch.equal(kv[9998, :, 5], rows[0]) and torch.equal(kv[8192, :, 0], rows[1])
    assert torch.equal(kv[9999, :, 127], rows[2])


def test_attention_zero_rows_and_empty_pool(cuda):
    kp = torch.zeros(0, 2, 16, 64, dtype=torch.bfloat16, device=cuda)
    q = torch.randn(3, 2, 64, device=cuda).bfloat16()
    lens = torch.zeros(3, dtype=torch.int32, device=cuda)
    assert (K.paged_sdpa(q, kp, kp, torch.zeros(3, 0, dtype=torch.int32, device=cuda), lens, scale=1.0) == 0).all()
    assert (K.paged_sdpa(q, kp, kp, torch.zeros(3, 4, dtype=torch.int32, device=cuda), lens, scale=1.0) == 0).all()
    assert K.paged_sdpa(q[:0], kp, kp, torch.zeros(0, 4, dtype=torch.int32, device=cuda), lens[:0],
                        scale=1.0).shape == (0, 2, 64)


# ------------------------------------------------------------------ streams, graphs, repeatability
def test_results_repeat_bit_for_bit(cuda):
    args = attention_inputs([1000, 3, 517], 8, 2, 128, 16, torch.bfloat16, seed=11)
    q, kp, vp, table, lens, scale = args
    want = check_attention(args)
    for _ in range(5):
        assert torch.equal(want, K.paged_sdpa(q, kp, vp, table, lens, scale=scale))


def test_two_streams_and_two_graphs_at_once(cuda):
    """Calls that overlap share no scratch: on two streams, and in two captured graphs replayed side by side."""
    sets = [attention_inputs([1500, 40, 700], 4, 4, 64, 16, torch.bfloat16, seed=s) for s in (21, 22)]
    want = [check_attention(s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                got[i].append(K.paged_sdpa(*s[:5], scale=s[5]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(want[i], g) for g in got[i])
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(K.paged_sdpa(*s[:5], scale=s[5]))
        graphs.append(g)
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(want[i], outs[i])


def test_generation_step_in_a_graph_grows_the_cache(cuda):
    """advance -> append -> attention as one captured step, replayed: each replay adds a token to every row."""
    bsz, heads, dim, page, width, steps = 3, 4, 64, 16, 5, 40
    dtype = torch.bfloat16
    t = Tables([0] * bsz, page, width, bsz * width)
    kp, vp = make_pools(bsz * width, heads, page, dim, dtype, fill=float("nan"))
    qkv, rho, cos, sin, scale, _ = append_inputs(bsz * steps, heads, dim, dtype, 2)
    qkv, rho = qkv.view(steps, bsz, 3, heads, dim), rho.view(steps, bsz)
    step_qkv, step_rho = qkv[0].clone(), rho[0].clone()
    ones = torch.ones(bsz, dtype=torch.int32, device=cuda)
    fin = torch.zeros(bsz, dtype=torch.bool, device=cuda)
    K.advance_block_tables(t.lengths, 0 * ones, t.table, t.free, t.count, page_size=page, max_new=1, finished=fin)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots, pos = K.advance_block_tables(t.lengths, ones, t.table, t.free, t.count, page_size=page, max_new=1,
                                            finished=fin)
        q = K.qkv_append_from_carried(step_qkv, step_rho, cos, sin, scale, 1e-6, pos.view(bsz), slots.view(bsz), kp,
                                      vp)
        o = K.paged_sdpa(q, kp, vp, t.table, t.lengths, scale=8.0)
    outs = []
    for s in range(steps):
        step_qkv.copy_(qkv[s])
        step_rho.copy_(rho[s])
        graph.replay()
        outs.append(o.clone())
    assert t.lengths.tolist() == [steps] * bsz
    q, k, v = K.qkv_postprocess_from_carried(qkv.transpose(0, 1).contiguous(), rho.transpose(0, 1).contiguous(), cos,
                                             sin, scale, 1e-6)
    want = K.causal_sdpa(q.float(), k.float(), v.float(), scale=8.0, dropout_p=0.0)
    got = torch.stack(outs, 1).float()
    # the same bf16 q, k, v; the whole-sequence op in fp32: one bf16 rounding apart, and some fp32 noise
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4 * v.float().abs().max()).all()


def test_registered_operators_are_the_same_calls(cuda):
    ops = torch.ops.engpt_b200
    runs = []
    for f in (K, ops):
        t = Tables([5, 0, 40], 16, 4, 12, seed=1)
        kp, vp = make_pools(12, 4, 16, 64, torch.bfloat16, fill=0.5)
        new = torch.tensor([1, 3, 2], dtype=torch.int32, device=cuda)
        slots, pos = f.advance_block_tables(t.lengths, new, t.table, t.free, t.count, page_size=16, max_new=3,
                                            finished=torch.tensor([False, False, True], device=cuda))
        qkv, rho, cos, sin, scale, _ = append_inputs(9, 4, 64, torch.bfloat16, 4)
        q = f.qkv_append_from_carried(qkv.view(3, 3, 3, 4, 64), rho.view(3, 3), cos, sin, scale, 1e-6, pos, slots, kp,
                                      vp, qk_mult=0.5)
        f.write_kv_pages(qkv[:2, 1], qkv[:2, 2], torch.tensor([2, 1], dtype=torch.int32, device=cuda), kp, vp)
        o = f.paged_sdpa(q[:, 0].contiguous(), kp, vp, t.table, t.lengths, scale=0.3)
        runs.append((slots, pos, t.lengths, t.table, t.free, t.count, kp, vp, q, o))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
