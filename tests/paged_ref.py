"""Plain 64-bit (and whole-number) forms of the paged key-value cache operators, for the tests."""

import numpy as np
import torch


def pages_of(n, page):
    return -(-n // page)


def advance(lengths, new, table, free, count, page, max_new, finished=None):
    """advance_block_tables on python lists; returns (slots, positions, lengths, table, free, count)."""
    bsz, width = len(lengths), len(table[0]) if table else 0
    lengths, table, free = list(lengths), [list(r) for r in table], list(free)
    if finished is not None:
        for b in range(bsz):
            if finished[b]:
                for j in range(pages_of(lengths[b], page)):
                    free[count] = table[b][j]
                    count += 1
                lengths[b] = 0
    slots = [[-1] * max_new for _ in range(bsz)]
    pos = [[0] * max_new for _ in range(bsz)]
    short = False
    for b in range(bsz):
        if new[b] < 0 or new[b] > max_new or lengths[b] + new[b] > width * page:
            continue
        have = pages_of(lengths[b], page)
        need = pages_of(lengths[b] + new[b], page) - have
        if need and (short or need > count):
            short = True          # the rows behind a row that found too few pages get none either
            continue
        for j in range(need):
            count -= 1
            table[b][have + j] = free[count]
        for i in range(new[b]):
            p = lengths[b] + i
            slots[b][i], pos[b][i] = table[b][p // page] * page + p % page, p
        lengths[b] += new[b]
    return slots, pos, lengths, table, free, count


def gather_rows(pages, table_row, n):
    """The first n rows [n, H, Dh] of a request, as float64."""
    ps = pages.shape[2]
    ids = torch.as_tensor([int(x) for x in table_row[:pages_of(n, ps)]], dtype=torch.long)
    return pages[ids].permute(0, 2, 1, 3).reshape(-1, pages.shape[1], pages.shape[3])[:n].double()


def attention(q, k_pages, v_pages, table, lengths, scale):
    """paged_sdpa in float64 on the CPU, and for each (row, head) the largest |v| and the largest sum |q_i k_i|."""
    q, k_pages, v_pages, table = (x.cpu() for x in (q, k_pages, v_pages, table))
    bsz, heads, dim = q.shape
    group = heads // k_pages.shape[1]
    out = torch.zeros(bsz, heads, dim, dtype=torch.float64)
    vmax = torch.zeros(bsz, heads, 1, dtype=torch.float64)
    smax = torch.zeros(bsz, heads, 1, dtype=torch.float64)
    for b, n in enumerate(int(x) for x in lengths.cpu()):
        if n <= 0:
            continue
        k, v = gather_rows(k_pages, table[b], n), gather_rows(v_pages, table[b], n)
        for h in range(heads):
            kh, vh, qh = k[:, h // group], v[:, h // group], q[b, h].double()
            p = torch.softmax(kh @ qh * scale, dim=0)
            out[b, h] = p @ vh
            vmax[b, h] = vh.abs().max()
            smax[b, h] = (kh.abs() @ qh.abs()).max() * abs(scale)
    return out, vmax, smax


def attention_tolerance(dtype, ref, vmax, smax, dim, n):
    """How far paged_sdpa may be from the 64-bit result.

    One rounding of the result to its type (half a step); every score is an
    fp32 dot product of dim terms, times the scale, in base-2 units
    (log2 e = 1.4427): relative error of e^s below (dim + 4) * 2^-24 * 1.45 *
    smax + 2^-21 (the exponential and the running-maximum rescales); sums
    over n terms: n * 2^-24 each for l and o; a weighted mean of values up to
    vmax moves by at most twice the weights' relative error.  With bf16 inputs
    the weights are held as two bf16 parts: 2^-16 more.
    """
    weight = (dim + 4) * 2.0 ** -24 * 1.45 * smax + 2.0 ** -21 + 2 * n * 2.0 ** -24
    if dtype == torch.bfloat16:
        weight = weight + 2.0 ** -16
    return torch.finfo(dtype).eps / 2 * ref.abs() + 2 * weight * vmax + 1e-30


def postprocess(qkv, rho, cos, sin, qk_scale, eps, pos):
    """qkv_postprocess in float64 at given positions: [n, 3, H, Dh] -> q, k, v [n, H, Dh]."""
    x, rho = qkv.cpu().double(), rho.cpu().double().view(-1, 1, 1)
    half = cos.shape[1]
    c, s = (t.cpu().double()[pos.cpu().long()][:, None, :] for t in (cos, sin))
    out = []
    for part in range(2):
        r = x[:, part]
        den = torch.maximum(r.pow(2).sum(-1, keepdim=True).sqrt(), rho * eps)
        y = r.clone()
        y[..., 0:2 * half:2] = r[..., 0:2 * half:2] * c - r[..., 1:2 * half:2] * s
        y[..., 1:2 * half:2] = r[..., 0:2 * half:2] * s + r[..., 1:2 * half:2] * c
        out.append(y / den * qk_scale.cpu().double())
    return out[0], out[1], x[:, 2] / rho


def random_table(lengths, page, width, pool, rng):
    """A block table (unused entries -1) with the requests' pages in random order, and the pages left over."""
    perm = rng.permutation(pool).tolist()
    table = np.full((len(lengths), width), -1, dtype=np.int32)
    for b, n in enumerate(lengths):
        for j in range(pages_of(max(n, 0), page)):
            table[b, j] = perm.pop()
    return torch.from_numpy(table), perm
