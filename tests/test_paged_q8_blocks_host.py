"""The check of whole calls (tests/paged_q8_blocks.py) against the one that goes token by token (no GPU)."""

import pytest
import torch

from tests import paged_q8_blocks as B, paged_q8_ref as Q


def stored(kind, dead=()):
    """A small cache before and after a write that follows the definition, in plain Python."""
    cache = Q.make_pools(4, 2, 8, 6, 4, kind, device="cpu")
    Q.fill_pools(cache, 0)
    codes, scales = cache[0], cache[2]
    was, old = Q.raw(codes), scales.clone()
    slots = [9, 10, -1, 16, 17, 18, 19, 20, 6, 7, 24]
    x = (torch.randn(11, 2, 6, generator=torch.Generator().manual_seed(1)) * 2).double()
    x[4] *= 1e-3
    x[8:10] = 0

    def encode(y):
        if kind == "int8":
            return y.round().to(torch.int8).view(torch.uint8)
        return y.float().clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)

    out = codes.view(torch.uint8)
    for i, n in Q.runs_of(slots, 4):
        pg, off = slots[i] // 8, slots[i] % 8
        bl, o = off // 4, off % 4
        live = [j for j in range(i, i + n) if j not in dead]
        if not live:
            continue
        need = (x[live].abs().amax((0, 2)).clamp(min=Q.LEAST) / Q.TOP[codes.dtype]).float()
        new = need if o == 0 else torch.maximum(old[pg, :, bl], need)
        for sl in range(bl * 4, bl * 4 + 4):
            j = i + sl - off
            if j in live:
                out[pg, :, sl] = encode(x[j] / new.double()[:, None])
            elif o > 0 and not i <= j < i + n:
                r = encode(was[pg, :, sl].view(codes.dtype).float().double() * (old[pg, :, bl] / new).double()[:, None])
                out[pg, :, sl] = torch.where((new > old[pg, :, bl])[:, None], r, was[pg, :, sl])
        scales[pg, :, bl] = new
    return codes, scales, was, old, x, slots


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dead", [(), (1, 4)])
def test_both_checks_take_what_is_right(kind, dead):
    codes, scales, was, old, x, slots = stored(kind, dead)
    Q.check_store(codes, scales, was, old, x, slots, 0.0, dead)
    B.check_store(codes, scales, was, old, x, torch.tensor(slots), 0.0, torch.tensor([j in dead for j in range(11)]))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_both_checks_find_what_is_wrong(kind):
    codes, scales, was, old, x, slots = stored(kind)

    def refused(c, s):
        for check, at in ((Q.check_store, slots), (B.check_store, torch.tensor(slots))):
            with pytest.raises(AssertionError):
                check(c, s, was, old, x, at)

    # a written code, one beside it in a raised block, one of a block that starts anew, untouched ones
    for pg, sl in ((1, 1), (1, 2), (1, 0), (2, 1), (2, 5), (0, 7), (0, 5), (3, 1), (3, 4), (0, 0)):
        wrong = codes.clone()
        u = wrong.view(torch.uint8)
        u[pg, 1, sl, 2] = 0x7f if int(u[pg, 1, sl, 2]) < 0x40 else 0
        refused(wrong, scales)
    for pg, bl in ((2, 0), (1, 0), (0, 0), (3, 0)):
        for by in (1.001, float("nan")):
            wrong = scales.clone()
            wrong[pg, 0, bl] *= by
            refused(codes, wrong)
