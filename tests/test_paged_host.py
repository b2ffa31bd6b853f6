"""Refusals of the paged key-value cache operators (no GPU): argument checks in Python and at the C boundary."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from engpt_b200 import _lib, kernels as K


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def cuda_fakes():
    return FakeTensorMode()


def test_ops_refuse_cpu_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    kp = torch.zeros(4, 2, 16, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.advance_block_tables(i, i, torch.zeros(2, 3, dtype=torch.int32), i, i[:1], page_size=16, max_new=1)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.paged_sdpa(torch.zeros(2, 2, 64), kp, kp, torch.zeros(2, 3, dtype=torch.int32), i, scale=1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.write_kv_pages(torch.zeros(2, 2, 64), torch.zeros(2, 2, 64), i, kp, kp)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.qkv_append_from_carried(torch.zeros(2, 3, 2, 64), torch.ones(2), torch.zeros(4, 32), torch.zeros(4, 32),
                                  torch.ones(2, 64), 1e-6, i, i, kp, kp)


def test_paged_sdpa_argument_checks():
    with cuda_fakes():
        kp = torch.empty(8, 2, 16, 64, device="cuda", dtype=torch.bfloat16)
        q = torch.empty(3, 4, 64, device="cuda", dtype=torch.bfloat16)
        table = torch.empty(3, 5, device="cuda", dtype=torch.int32)
        lens = torch.empty(3, device="cuda", dtype=torch.int32)
        bad = [
            (q.float(), kp, kp, table, lens),                       # dtype of q
            (q[:, :3], kp, kp, table, lens),                        # 3 query heads on 2 kv heads
            (q[..., :32], kp, kp, table, lens),                     # head_dim
            (q, kp, kp[:4], table, lens),                           # pools differ
            (q, kp[0], kp[0], table, lens),                         # no pools
            (q, kp.transpose(2, 3), kp.transpose(2, 3), table, lens),
            (q, kp, kp, table.long(), lens),
            (q, kp, kp, table[:2], lens),
            (q, kp, kp, table.t().contiguous().t(), lens),
            (q, kp, kp, table, lens.long()),
            (q, kp, kp, table, lens[:2]),
            (q[:, 0], kp, kp, table, lens),
        ]
        for args in bad:
            with pytest.raises(ValueError):
                K.paged_sdpa(*args, scale=1.0)
        with pytest.raises(NotImplementedError, match="forward-only"):
            K.paged_sdpa(q.requires_grad_(True), kp, kp, table, lens, scale=1.0)


def test_append_write_and_table_argument_checks():
    with cuda_fakes():
        c = dict(device="cuda")
        kp = torch.empty(8, 2, 16, 64, dtype=torch.bfloat16, **c)
        i = torch.empty(3, dtype=torch.int32, **c)
        qkv = torch.empty(3, 3, 2, 64, dtype=torch.bfloat16, **c)
        rho, cs, s = torch.empty(3, **c), torch.empty(9, 32, **c), torch.empty(2, 64, **c)
        good = [qkv, rho, cs, cs, s, 1e-6, i, i, kp, kp]
        for at, wrong in ((0, qkv.float()), (0, qkv[:, :2]), (1, rho[:2]), (2, cs[:, :31]), (3, cs[:8]), (4, s[:1]),
                          (6, i.long()), (7, i[:2]), (7, i[::2]), (9, kp[:, :1])):
            args = list(good)
            args[at] = wrong
            with pytest.raises(ValueError):
                K.qkv_append_from_carried(*args)
        k = torch.empty(3, 2, 64, dtype=torch.bfloat16, **c)
        for args in ((k, k[:2], i, kp, kp), (k.float(), k.float(), i, kp, kp), (k, k, i[:2], kp, kp),
                     (k[:, :1], k[:, :1], i, kp, kp), (k, k, i.long(), kp, kp)):
            with pytest.raises(ValueError):
                K.write_kv_pages(*args)
        table = torch.empty(3, 5, dtype=torch.int32, **c)
        free, one = torch.empty(9, dtype=torch.int32, **c), torch.empty(1, dtype=torch.int32, **c)
        ok = [i, i, table, free, one]
        for at, wrong in ((0, i.long()), (1, i[:2]), (2, table[:2]), (2, table.long()), (3, table), (4, i),
                          (0, torch.empty(6, dtype=torch.int32, **c)[::2])):
            args = list(ok)
            args[at] = wrong
            with pytest.raises(ValueError):
                K.advance_block_tables(*args, page_size=16, max_new=1)
        for kw in (dict(page_size=0, max_new=1), dict(page_size=16, max_new=-1),
                   dict(page_size=16, max_new=1, finished=i), dict(page_size=16, max_new=1, finished=i[:2].bool())):
            with pytest.raises(ValueError):
                K.advance_block_tables(*ok, **kw)


def test_c_entry_points_check_before_any_launch():
    lib = _lib.load()
    p = 1 << 20           # a pointer that no check may follow
    adv = lib.engpt_advance_block_tables
    assert adv(p, p, None, 4, p, 3, 5, p, 9, p, 16, 1, p, p, None) == 1          # stride below the width
    assert adv(p, p, None, 4, p, 5, 5, p, 9, p, 0, 1, p, p, None) == 1
    assert adv(p, p, None, 4, p, 5, 5, p, 2 ** 28, p, 16, 1, p, p, None) == 1    # 2^32 slots
    assert adv(p, p, None, 9000, p, 5, 5, p, 9, p, 16, 1, p, p, None) == 6
    assert adv(p, None, None, 4, p, 5, 5, p, 9, p, 16, 1, p, p, None) == 7
    assert adv(p, p, None, 0, p, 5, 5, p, 9, p, 16, 1, p, p, None) == 0
    six, four, two = i64(1, 1, 1, 1, 1, 1), i64(1, 1, 1, 1), i64(1, 1)
    w = lib.engpt_write_kv_pages
    assert w(p, p, four, 5, 3, 2, 64, p, p, p, six, 4, 16, None) == 2
    assert w(p, p, four, 1, 3, 0, 64, p, p, p, six, 4, 16, None) == 1
    assert w(p, None, four, 1, 3, 2, 64, p, p, p, six, 4, 16, None) == 7
    assert w(p, p, four, 1, 3, 2, 64, p, p, p, six, 2 ** 28, 16, None) == 1
    assert w(p, p, four, 1, 0, 2, 64, p, p, p, six, 4, 16, None) == 0
    ap = lib.engpt_qkv_append
    assert ap(p, 1, p, p, p, 9, 33, p, 1.0, 0.0, 3, 2, 64, p, p, p, p, p, six, 4, 16, None) == 1
    assert ap(p, 3, p, p, p, 9, 32, p, 1.0, 0.0, 3, 2, 64, p, p, p, p, p, six, 4, 16, None) == 2
    assert ap(p, 1, p, None, p, 9, 32, p, 1.0, 0.0, 3, 2, 64, p, p, p, p, p, six, 4, 16, None) == 7
    assert ap(p, 1, p, p, p, 9, 32, p, 1.0, 0.0, 0, 2, 64, p, p, p, p, p, six, 4, 16, None) == 0
    at = lib.engpt_paged_attention
    assert at(p, two, p, p, six, 1, 2, 3, 2, 64, 4, 16, p, 5, 5, p, 1.0, p, p, None) == 1    # 3 heads on 2
    assert at(p, two, p, p, six, 1, 2, 4, 2, 257, 4, 16, p, 5, 5, p, 1.0, p, p, None) == 6
    assert at(p, two, p, p, six, 7, 2, 4, 2, 64, 4, 16, p, 5, 5, p, 1.0, p, p, None) == 2
    assert at(p, two, p, p, six, 1, 2, 4, 2, 64, 4, 16, None, 5, 5, p, 1.0, p, p, None) == 7
    assert at(p, two, p, p, six, 1, 2, 4, 2, 64, 4, 16, p, 4, 5, p, 1.0, p, p, None) == 1
    assert at(p, two, p, p, six, 1, 0, 4, 2, 64, 4, 16, p, 5, 5, p, 1.0, p, p, None) == 0
    assert b"paged_attention" in lib.engpt_last_error() or lib.engpt_last_error() == b""


def test_cache_and_decoder_refuse_the_cpu():
    from engpt_b200 import EfficientNGPT, ModelConfig, PagedKVCache
    from tests.helpers import SMALL
    cfg = ModelConfig(**SMALL)
    with pytest.raises(RuntimeError, match="CUDA"):
        PagedKVCache(cfg, 2, 4, device="cpu")
    with pytest.raises(ValueError):
        PagedKVCache(cfg, 2, 0)
    with pytest.raises(NotImplementedError):
        PagedKVCache(cfg, 2, 4, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        EfficientNGPT(cfg).decoder(2, 4)


def test_torch_ops_of_the_cache():
    """Registered operators: schemas with the changed arguments, fake shapes, no CPU kernel."""
    ops = torch.ops.engpt_b200
    s = str(ops.advance_block_tables.default._schema)
    assert "Tensor(a0!) lengths" in s and "Tensor(a2!) block_table" in s and "Tensor? finished" in s, s
    assert "k_pages" in str(ops.write_kv_pages.default._schema) and "!" in str(ops.write_kv_pages.default._schema)
    assert "!" not in str(ops.paged_sdpa.default._schema)
    with cuda_fakes():
        c = dict(device="cuda")
        i = torch.empty(3, dtype=torch.int32, **c)
        table, free = torch.empty(3, 5, dtype=torch.int32, **c), torch.empty(9, dtype=torch.int32, **c)
        slots, pos = ops.advance_block_tables(i, i.clone(), table, free, i[:1].clone(), page_size=16, max_new=7)
        assert slots.shape == pos.shape == (3, 7) and slots.dtype == torch.int32
        kp = torch.empty(8, 2, 16, 64, dtype=torch.bfloat16, **c)
        q = ops.qkv_append_from_carried(torch.empty(3, 1, 3, 2, 64, dtype=torch.bfloat16, **c),
                                        torch.empty(3, 1, **c), torch.empty(9, 32, **c), torch.empty(9, 32, **c),
                                        torch.empty(2, 64, **c), 1e-6, i.view(3, 1), i.view(3, 1).clone(), kp,
                                        kp.clone())
        assert q.shape == (3, 1, 2, 64) and q.dtype == torch.bfloat16
        o = ops.paged_sdpa(torch.empty(3, 4, 64, dtype=torch.bfloat16, **c), kp, kp, table, i, scale=1.0)
        assert o.shape == (3, 4, 64)
    x = torch.zeros(4, 2, 16, 64)
    with pytest.raises(NotImplementedError):
        ops.paged_sdpa(torch.zeros(1, 2, 64), x, x, torch.zeros(1, 2, dtype=torch.int32),
                       torch.zeros(1, dtype=torch.int32), scale=1.0)
