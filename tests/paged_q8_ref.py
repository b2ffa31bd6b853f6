"""Plain 64-bit forms of the 8-bit paged cache operators, for the tests."""

import numpy as np
import torch

from tests import paged_ref as R

CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
LEAST = 2.0 ** -100


def make_pools(pool, heads, page, dim, block, kind, layout="head", device="cuda"):
    """k and v codes [P, H, ps, Dh] (bytes of 0x55) and scales [P, H, ps / block] in one of the layouts a user may hold."""
    code, nb = CODES[kind], page // block
    def full(*shape):
        return torch.full(shape, 0x55, dtype=torch.uint8, device=device).view(code)

    def ones(*shape):
        return torch.full(shape, 0.5, device=device)

    if layout == "head":
        c, s = [full(pool, heads, page, dim) for _ in range(2)], [ones(pool, heads, nb) for _ in range(2)]
    elif layout == "token":          # stored [P, ps, H, Dh], and the scales [P, blocks, H]
        c = [full(pool, page, heads, dim).transpose(1, 2) for _ in range(2)]
        s = [ones(pool, nb, heads).transpose(1, 2) for _ in range(2)]
    elif layout == "both":           # k and v of a page side by side
        kv, kvs = full(pool, 2, heads, page, dim), ones(pool, 2, heads, nb)
        c, s = [kv[:, 0], kv[:, 1]], [kvs[:, 0], kvs[:, 1]]
    else:                            # "odd": rows one code longer than head_dim, one code off any alignment
        c = [full(pool, heads, page, dim + 1)[..., 1:] for _ in range(2)]
        s = [ones(pool, heads, nb + 1)[..., 1:] for _ in range(2)]
    return c[0], c[1], s[0], s[1]


def fill_pools(cache, seed, low=-3.0, high=0.0):
    """A cache in use: random codes (none of them NaN), scales log-uniform in e^low .. e^high."""
    gen = torch.Generator().manual_seed(seed)
    for c, s in ((cache[0], cache[2]), (cache[1], cache[3])):
        if c.dtype == torch.int8:
            x = torch.randint(-127, 128, c.shape, generator=gen, dtype=torch.int8)
        else:
            x = torch.randint(0, 127, c.shape, generator=gen, dtype=torch.uint8)
            x = (x + 128 * torch.randint(0, 2, c.shape, generator=gen, dtype=torch.uint8)).view(torch.float8_e4m3fn)
        copy_codes(c, x)
        s.copy_(torch.exp(low + (high - low) * torch.rand(s.shape, generator=gen)))


def copy_codes(dst, src):
    dst.view(torch.uint8).copy_(src.view(torch.uint8))


def raw(codes):
    """The codes' bytes, on the CPU."""
    return codes.view(torch.uint8).cpu().clone()


def decode(codes):
    return codes.cpu().float().double()


def values(codes, scales):
    """The numbers that a pool stands for, float64 on the CPU."""
    nb = scales.shape[2]
    return decode(codes) * scales.cpu().double().repeat_interleave(codes.shape[2] // nb, dim=2)[..., None]


def half_step(y, kind):
    """Half a step of the code grid around y (in codes): what rounding to a code may be off by."""
    if kind == torch.int8:
        return torch.full_like(y, 0.5)
    # steps of 2^(e-3) for |y| in [2^e, 2^(e+1)), at least 2^-9; at a power of two the rounding from below counts
    _, e = torch.frexp(y.abs().clamp(min=2.0 ** -6))
    return torch.ldexp(torch.ones_like(y), e - 1 - 3) / 2


def runs_of(slots, block):
    """(first token, number of tokens) of the runs of one block that a call's slots make."""
    out, i = [], 0
    while i < len(slots):
        if slots[i] < 0:
            i += 1
            continue
        n = 1
        while i + n < len(slots) and slots[i + n] == slots[i] + n and slots[i + n] % block:
            n += 1
        out.append((i, n))
        i += n
    return out


def check_store(codes, scales, before, scales_before, x, slots, err=0.0, dead=()):
    """Checks a pool after a writing call against the definition, in 64 bits.

    before, scales_before: bytes and scales before; x [n, H, Dh] float64, each
    number off by at most err (of its row, broadcastable); slots: list; dead: tokens that were to be left out.

    The scale is max |x| / top rounded to fp32 (half a step 2^-24; x off by
    err).  A code is the product of x and the reciprocal of the scale, two fp32
    roundings (2^-23 relative, at most `top` of them in codes: 2^-22 * top
    covers them), rounded once to the grid.  A raised block's other codes: the
    ratio of the scales and its product with the code, the same.
    """
    kind, page = codes.dtype, codes.shape[2]
    block = page // scales.shape[2]
    top = TOP[kind]
    got, now, old = decode(codes), scales.cpu().double(), scales_before.cpu().double()
    was = before.view(kind).float().double()
    want = before.clone()
    untouched = torch.ones(now.shape, dtype=torch.bool)
    err = torch.as_tensor(err, dtype=torch.float64).expand(x.shape[0], x.shape[1], 1) if not torch.is_tensor(err) else err
    slack = top * 2.0 ** -22
    for i, n in runs_of(slots, block):
        live = [j for j in range(i, i + n) if j not in dead]
        if not live:
            continue
        pg, off = slots[i] // page, slots[i] % page
        bl, o = off // block, off % block
        xs, es = x[live], err[live]
        amax, emax = xs.abs().amax((0, 2)), es.amax((0, 2))
        need = amax.clamp(min=LEAST) / top
        s0, s1 = old[pg, :, bl], now[pg, :, bl]
        want_s = need if o == 0 else torch.maximum(s0, need)
        tol = want_s * 2.0 ** -23 + emax / top
        assert ((s1 - want_s).abs() <= tol).all(), (s1, want_s)
        if o > 0:
            keep = need + tol < s0
            assert (s1[keep] == s0[keep]).all()
        untouched[pg, :, bl] = False
        for j in live:
            sl = slots[j] % page
            y = x[j] / s1[:, None]
            assert ((got[pg, :, sl] - y).abs() <= half_step(y, kind) * (1 + 2.0 ** -18) + slack + err[j] / s1[:, None]).all()
            want[pg, :, sl] = codes[pg, :, sl].view(torch.uint8).cpu()
        for sl in range(bl * block, (bl + 1) * block):
            if off <= sl < off + n:
                continue
            if o > 0:
                raised = s1 > s0
                y = was[pg, :, sl] * (s0 / s1)[:, None]
                bad = (got[pg, :, sl] - y).abs() > half_step(y, kind) * (1 + 2.0 ** -18) + slack
                assert not (bad & raised[:, None]).any()
                want[pg, raised, sl] = codes[pg, :, sl].view(torch.uint8).cpu()[raised]
    assert torch.equal(raw(codes), want)                         # everything else, bit for bit
    assert torch.equal(now[untouched], old[untouched])


def query_error(q, kind):
    """How far the kernels' form of each element of q may be from it.

    For int8 codes a row is rounded to whole multiples of 2^-22 (fp32) or 2^-14
    (bf16) of a power of two that its largest element is about at least (0.992):
    half a step is 2^-23 or 2^-15 of the largest.  A bf16 element of at least 2^-6
    of it is exact (8 bits from there down are multiples of 2^-14).  For e4m3
    codes it is two fp16 parts of 11 bits each (fp32: 2^-22, and 2^-35 of the
    largest for what is too small for them) or one (bf16: its 8 bits fit, but
    for what lies below 2^-24 of the largest).
    """
    x = q.cpu().double().abs()
    most = x.amax(-1, keepdim=True)
    if kind == torch.int8:
        if q.dtype == torch.float32:
            return (1.01 * 2.0 ** -23 * most).expand(x.shape)
        return torch.where(x < 2.0 ** -6 * most, torch.minimum(x, 1.01 * 2.0 ** -15 * most), torch.zeros_like(x))
    if q.dtype == torch.float32:
        return 2.0 ** -22 * x + 2.0 ** -35 * most
    return torch.where(x < 2.0 ** -16 * most, torch.minimum(x, 2.0 ** -24 * most), torch.zeros_like(x))


def attention_tolerance(q, ref, vmax, smax, dmax, scale, n):
    """How far paged_sdpa_q8 may be from the 64-bit result on the cache's numbers.

    As paged_ref.attention_tolerance (fp32 dot products of dim terms,
    exponentials, sums over n terms, one rounding of the result), with the
    products with the scales (up to 8 roundings of 2^-24 on scores and
    weights) and the rounding of q (dmax: the largest sum of |k_i| times what q_i
    may be off by).  The weights of the values are fp16 numbers: for an fp32
    result two of them, 2^-21; for a bf16 result one, half a step 2^-11, in
    the sum over the values alone (the weights' own sum is of fp32 numbers), so
    the weighted mean moves by at most 2^-11 vmax.
    """
    dim = q.shape[2]
    score = (dim + 8) * 2.0 ** -24 * smax + dmax * abs(scale)
    weight = 1.45 * score + 2.0 ** -20 + 2 * n * 2.0 ** -24
    rounded = 0.0 if q.dtype == torch.float32 else 2.0 ** -11
    return torch.finfo(q.dtype).eps / 2 * ref.abs() + (2 * weight + rounded) * vmax + 1e-30


def attention(q, cache, table, lengths, scale):
    """The 64-bit result and its tolerance."""
    k, v = values(cache[0], cache[2]), values(cache[1], cache[3])
    ref, vmax, smax = R.attention(q, k, v, table, lengths, scale)
    off = query_error(q, cache[0].dtype)
    dmax = torch.zeros_like(vmax)
    group = q.shape[1] // k.shape[1]
    for b, n in enumerate(int(x) for x in lengths.cpu()):
        if n > 0:
            rows = R.gather_rows(k, table.cpu()[b], n).abs().repeat_interleave(group, dim=1)
            dmax[b, :, 0] = torch.einsum("nhd,hd->nh", rows, off[b]).amax(0)
    n = max(1, int(lengths.max()) if lengths.numel() else 1)
    return ref, attention_tolerance(q, ref, vmax, smax, dmax, scale, n)


def prompt_slots(first, tokens, page, pool, seed, pad=()):
    """Slots [B, T] of requests that each write `tokens` tokens from position first[b], in random pages; pad[b] of a row's
    last tokens have none."""
    perm = np.random.default_rng(seed).permutation(pool).tolist()
    rows = []
    for b, f in enumerate(first):
        pages = {}
        row = []
        for p in range(f, f + tokens):
            if p // page not in pages:
                pages[p // page] = perm.pop()
            row.append(pages[p // page] * page + p % page)
        if b < len(pad) and pad[b]:
            row[tokens - pad[b]:] = [-1] * pad[b]
        rows.append(row)
    return torch.tensor(rows, dtype=torch.int32)
