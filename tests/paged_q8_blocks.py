"""The quantising write's definition for whole calls at once (64 bits, block by block in parallel, on any device), for the
tests of large calls.  tests/paged_q8_ref.py says the same token by token."""

import torch

from tests import paged_q8_ref as Q


def blocks(t, per_page):
    """[P, H, page, ...] as [P * per_page, block, H, ...]."""
    t = t.transpose(1, 2)
    return t.reshape(t.shape[0] * per_page, t.shape[1] // per_page, *t.shape[2:])


def postprocess(qkv, rho, cos, sin, qk_scale, eps, pos):
    """qkv_postprocess in float64 at given positions: [n, 3, H, Dh] -> q, k, v [n, H, Dh]."""
    x, rho = qkv.double(), rho.double()[:, None, None]
    half = cos.shape[1]
    c, s = (t.double()[pos.long()][:, None, :] for t in (cos, sin))
    out = []
    for part in range(2):
        r = x[:, part]
        norm = torch.maximum((r * r).sum(-1, keepdim=True).sqrt(), rho * eps)
        even, odd = r[..., 0:2 * half:2], r[..., 1:2 * half:2]
        y = r.clone()
        y[..., 0:2 * half:2] = even * c - odd * s
        y[..., 1:2 * half:2] = even * s + odd * c
        out.append(y / norm * qk_scale.double())
    return out[0], out[1], x[:, 2] / rho


def check_store(codes, scales, was, old, x, slots, err=0.0, dead=None):
    """paged_q8_ref.check_store, with its tolerances, for any number of tokens.

    was: bytes before, [P, H, page, Dh]; old: scales before; x [n, H, Dh] float64, each number off by at most err [n, H, 1];
    slots [n]; dead [n] bool: tokens that have a slot and were to be left out.  Those of one block stand side by side.
    """
    per_page, kind = scales.shape[2], codes.dtype
    block, heads, dim = codes.shape[2] // per_page, codes.shape[1], codes.shape[3]
    top = Q.TOP[kind]
    slots = slots.to(x.device).long()
    dead = torch.zeros_like(slots, dtype=torch.bool) if dead is None else dead.to(x.device)
    err = torch.as_tensor(err, dtype=torch.float64, device=x.device).expand(x.shape[0], heads, 1)
    bytes_now, bytes_was = blocks(codes.view(torch.uint8), per_page), blocks(was, per_page)
    n = bytes_now.shape[0]
    got, held = blocks(codes, per_page).float().double(), bytes_was.view(kind).float().double()
    now, before = (blocks(s, per_page)[:, 0].double() for s in (scales, old))          # [blocks, H]

    live = (slots >= 0) & ~dead
    rows, errs = (torch.zeros(n * block, heads, w, dtype=torch.float64, device=x.device) for w in (dim, 1))
    rows[slots[live]], errs[slots[live]] = x[live], err[live]
    rows, errs = rows.view(n, block, heads, dim), errs.view(n, block, heads, 1)
    fresh, given = (torch.zeros(n * block, dtype=torch.bool, device=x.device) for _ in range(2))
    fresh[slots[live]] = True
    given[slots[slots >= 0]] = True
    fresh, given = fresh.view(n, block), given.view(n, block)
    touched = fresh.any(1)
    anew = touched & given[:, 0]

    need = rows.abs().amax((1, 3)).clamp(min=Q.LEAST) / top
    want = torch.where(anew[:, None], need, torch.maximum(before, need))
    tol = want * 2.0 ** -23 + errs.amax((1, 3)) / top
    assert ((now - want).abs() <= tol)[touched].all()
    kept = (touched & ~anew)[:, None] & (need + tol < before)
    assert (now == before)[kept | ~touched[:, None]].all()

    slack = top * 2.0 ** -22
    y = rows / now[:, None, :, None]
    lim = Q.half_step(y, kind) * (1 + 2.0 ** -18) + slack + errs / now[:, None, :, None]
    assert ((got - y).abs() <= lim)[fresh].all()

    raised = ((now > before) & (touched & ~anew)[:, None])[:, None, :] & ~given[:, :, None]   # [blocks, block, H]
    y = held * (before / now)[:, None, :, None]
    assert ((got - y).abs() <= Q.half_step(y, kind) * (1 + 2.0 ** -18) + slack)[raised].all()
    assert (bytes_now == bytes_was)[~(raised | fresh[:, :, None])].all()               # everything else, bit for bit
