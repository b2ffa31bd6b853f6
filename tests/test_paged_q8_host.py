"""Refusals of the 8-bit paged cache operators and their registered forms (no GPU)."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from engpt_b200 import _lib, kernels as K
from tests import paged_q8_ref as Q


def fakes():
    c = dict(device="cuda")
    kp, vp = (torch.empty(8, 2, 16, 64, dtype=torch.int8, **c) for _ in range(2))
    ks, vs = (torch.empty(8, 2, 2, **c) for _ in range(2))
    i = torch.empty(3, dtype=torch.int32, **c)
    return i, kp, vp, ks, vs


def calls(i, cache, rows=torch.float32):
    c = dict(device="cuda")
    k = torch.empty(3, 2, 64, dtype=rows, **c)
    qkv, rho, cs, s = torch.empty(3, 3, 2, 64, dtype=rows, **c), torch.empty(3, **c), torch.empty(9, 32, **c), torch.empty(
        2, 64, **c)
    table = torch.empty(3, 4, dtype=torch.int32, **c)
    return (lambda: K.write_kv_pages_q8(k, k, i, *cache),
            lambda: K.qkv_append_from_carried_q8(qkv, rho, cs, cs, s, 1e-6, i, i, *cache),
            lambda: K.read_kv_pages_q8(i, *cache),
            lambda: K.paged_sdpa_q8(k, *cache, table, i, scale=1.0))


def test_refuses_other_caches():
    with FakeTensorMode():
        i, kp, vp, ks, vs = fakes()
        e = torch.empty
        c = dict(device="cuda")
        bad = [((kp.view(torch.uint8), vp.view(torch.uint8), ks, vs), NotImplementedError, "int8 or float8"),
               ((kp, vp.view(torch.float8_e4m3fn), ks, vs), ValueError, "share"),
               ((kp, vp[:7], ks, vs), ValueError, "share"),
               ((kp[0], vp[0], ks, vs), ValueError, "share"),
               ((kp.transpose(2, 3), vp.transpose(2, 3), ks, vs), ValueError, "contiguous head_dim"),
               ((kp, vp, ks, vs.double()), ValueError, "float32"),
               ((kp, vp, ks[:, :1], vs[:, :1]), ValueError, "float32"),
               ((kp, vp, ks[:, :, :0], vs[:, :, :0]), ValueError, "float32"),
               ((kp, vp, e(8, 2, 3, **c), e(8, 2, 3, **c)), ValueError, "multiple"),
               ((kp, vp, ks.cpu(), vs), RuntimeError, "CUDA")]
        for cache, err, text in bad:
            for call in calls(i, cache):
                with pytest.raises(err, match=text):
                    call()


def test_refuses_other_arguments():
    with FakeTensorMode():
        i, *cache = fakes()
        c = dict(device="cuda")
        for call in calls(i.long(), cache):
            with pytest.raises(ValueError, match="int32"):
                call()
        for n in (0, 1, 3):
            with pytest.raises(ValueError, match="int32"):
                calls(i[:2], cache)[n]()
            with pytest.raises(NotImplementedError, match="float32 and bfloat16"):
                calls(i, cache, torch.float16)[n]()
        k = torch.empty(3, 2, 64, **c)
        with pytest.raises(ValueError, match="heads and head_dim"):
            K.write_kv_pages_q8(k[..., :32], k[..., :32], i, *cache)
        with pytest.raises(ValueError, match="share a dtype"):
            K.write_kv_pages_q8(k, k.bfloat16(), i, *cache)
        with pytest.raises(ValueError, match="multiple of the cache's heads"):
            K.paged_sdpa_q8(torch.empty(3, 3, 64, **c), *cache, torch.empty(3, 4, dtype=torch.int32, **c), i, scale=1.0)
        with pytest.raises(NotImplementedError, match="float32 and bfloat16"):
            K.read_kv_pages_q8(i, *cache, dtype=torch.float16)
        with pytest.raises(TypeError):
            K.read_kv_pages_q8(i, *cache, dtype="bf16")


def test_forward_only():
    with FakeTensorMode():
        i, *cache = fakes()
        cache[3].requires_grad_(True)
        for call in calls(i, cache):
            with pytest.raises(NotImplementedError, match="forward-only"):
                call()
        with torch.no_grad(), pytest.raises(ValueError):       # (past that check, to the next one)
            calls(i.long(), cache)[0]()


def test_forward_only_in_every_tensor():
    """(float8 pools can ask for a gradient too)"""
    with FakeTensorMode():
        i, kp, vp, ks, vs = fakes()
        cache = [kp.view(torch.float8_e4m3fn), vp.view(torch.float8_e4m3fn), ks, vs]
        for t in cache:
            t.requires_grad_(True)
            for call in calls(i, cache):
                with pytest.raises(NotImplementedError, match="forward-only"):
                    call()
            t.requires_grad_(False)


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_c_abi_refusals():
    lib = _lib.load()
    p, six, four, two = ctypes.c_void_p(4096), i64(*[16] * 6), i64(1, 1, 1, 1), i64(1, 1)
    w = lib.engpt_write_kv_pages_q8

    def write(k=p, dtype=1, n=3, heads=2, dim=64, kp=p, ks=p, strides=six, code=0, pages=4, page=16, block=16):
        return w(k, p, four, dtype, n, heads, dim, p, kp, p, ks, p, strides, six, code, pages, page, block, None)

    def append(dtype=1, n=3, dim=64, half=32, cos=p, ks=p, code=0, page=16, block=16, rows=9):
        return lib.engpt_qkv_append_q8(p, dtype, p, cos, p, rows, half, p, 1.0, 0.0, n, 2, dim, p, p, p, p, p, ks, p, six,
                                       six, code, 4, page, block, None)

    def read(n=3, out=p, dtype=1, kp=p, code=0, page=16, block=16):
        return lib.engpt_read_kv_pages_q8(p, n, kp, p, p, p, six, six, code, 2, 64, 4, page, block, out, p, dtype, None)

    def attend(dtype=1, code=0, bsz=2, heads=4, kv=2, dim=64, pages=4, page=16, block=16, table=p, stride=5, width=5,
               ks=p, work=p):
        return lib.engpt_paged_attention_q8(p, two, p, p, ks, p, six, six, dtype, code, bsz, heads, kv, dim, pages, page,
                                            block, table, stride, width, p, 1.0, p, work, None)

    for f in (write, append, read, attend):
        assert f(dtype=5) == 2 and f(code=2) == 2 and f(code=-1) == 2
        assert f(block=0) == 1 and f(block=5) == 1 and f(block=32) == 1 and f(page=0, block=1) == 1
    assert write(n=0) == append(n=0) == read(n=0) == attend(bsz=0) == 0
    assert write(n=-1) == append(n=-1) == read(n=-1) == attend(bsz=-1) == 1
    assert write(k=None) == write(kp=None) == write(ks=None) == write(strides=None) == 7
    assert append(cos=None) == append(ks=None) == read(out=None) == read(kp=None) == attend(ks=None) == 7
    assert write(pages=2 ** 28) == attend(pages=2 ** 28) == 1
    assert write(heads=0) == write(dim=0) == append(half=33) == append(rows=-1) == 1
    assert attend(heads=3) == 1 and attend(dim=257) == 6 and attend(table=None) == 7 and attend(stride=4) == 1
    assert attend(bsz=65536) == 1
    assert attend(width=2 ** 27, stride=2 ** 27) == 1              # 2^31 keys in a row
    assert b"paged_attention_q8" in lib.engpt_last_error()
    assert lib.engpt_paged_attention_q8_floats(1, 0, 4, 2, 64, 5, 16, 16) == 0


def test_torch_ops():
    """Registered operators: schemas with the changed arguments, fake shapes, no CPU kernel."""
    ops = torch.ops.engpt_b200
    for name in ("write_kv_pages_q8", "qkv_append_from_carried_q8"):
        s = str(getattr(ops, name).default._schema)
        assert all(f"!) {t}" in s for t in ("k_pages", "v_pages", "k_scales", "v_scales")), s
    for name in ("read_kv_pages_q8", "paged_sdpa_q8"):
        assert "!" not in str(getattr(ops, name).default._schema)
    with FakeTensorMode(allow_non_fake_inputs=True):
        i, *cache = fakes()
        c = dict(device="cuda")
        q = ops.qkv_append_from_carried_q8(torch.empty(3, 1, 3, 2, 64, dtype=torch.bfloat16, **c),
                                           torch.empty(3, 1, **c), torch.empty(9, 32, **c), torch.empty(9, 32, **c),
                                           torch.empty(2, 64, **c), 1e-6, i.view(3, 1), i.view(3, 1).clone(), *cache)
        assert q.shape == (3, 1, 2, 64) and q.dtype == torch.bfloat16
        k, v = ops.read_kv_pages_q8(i.view(1, 3), *cache, dtype=torch.float32)
        assert k.shape == v.shape == (1, 3, 2, 64) and k.dtype == torch.float32
        o = ops.paged_sdpa_q8(torch.empty(3, 4, 64, dtype=torch.bfloat16, **c), *cache,
                              torch.empty(3, 5, dtype=torch.int32, **c), i, scale=1.0)
        assert o.shape == (3, 4, 64) and o.dtype == torch.bfloat16
    cpu = Q.make_pools(4, 2, 16, 64, 16, "int8", device="cpu")
    with pytest.raises(NotImplementedError):
        ops.read_kv_pages_q8(torch.zeros(3, dtype=torch.int32), *cpu)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.read_kv_pages_q8(torch.zeros(3, dtype=torch.int32), *cpu)


def test_the_reference_store_finds_a_wrong_code():
    """The tests' own check, on a cache that is right and on ones that are not."""
    cache = Q.make_pools(3, 2, 8, 6, 4, "int8", device="cpu")
    Q.fill_pools(cache, 0)
    before, scales = Q.raw(cache[0]), cache[2].clone()
    slots = [9, 10, -1, 16, 17, 18, 19, 20]
    x = torch.randn(8, 2, 6, dtype=torch.float64).float().double()
    for i, n in Q.runs_of(slots, 4):
        pg, off = slots[i] // 8, slots[i] % 8
        bl, o = off // 4, off % 4
        need = (x[i:i + n].abs().amax((0, 2)) / 127).float()
        new = need if o == 0 else torch.maximum(scales[pg, :, bl], need)
        for sl in range(bl * 4, bl * 4 + 4):
            if off <= sl < off + n:
                cache[0][pg, :, sl] = (x[i + sl - off] / new.double()[:, None]).round().to(torch.int8)
            elif o > 0:
                old = cache[0][pg, :, sl].double() * (scales[pg, :, bl] / new).double()[:, None]
                cache[0][pg, :, sl] = old.round().to(torch.int8)
        cache[2][pg, :, bl] = new
    Q.check_store(cache[0], cache[2], before, scales, x, slots)
    for pg, sl in ((1, 1), (1, 2), (1, 0), (2, 3), (0, 5)):
        wrong = cache[0].clone()
        wrong[pg, 1, sl, 2] += 2 if wrong[pg, 1, sl, 2] < 100 else -2
        with pytest.raises(AssertionError):
            Q.check_store(wrong, cache[2], before, scales, x, slots)
    wrong = cache[2].clone()
    wrong[2, 0, 0] *= 1.001
    with pytest.raises(AssertionError):
        Q.check_store(cache[0], wrong, before, scales, x, slots)


def test_cache_and_decoder_refusals():
    from engpt_b200 import EfficientNGPT, ModelConfig, PagedKVCache
    from tests.helpers import SMALL
    cfg = ModelConfig(**SMALL)
    for block in (0, -1, 5, 128):
        with pytest.raises(ValueError, match="scale_block"):
            PagedKVCache(cfg, 2, 4, page_size=64, dtype=torch.int8, scale_block=block)
    with pytest.raises(ValueError, match="no scales"):
        PagedKVCache(cfg, 2, 4, scale_block=16)
    with pytest.raises(NotImplementedError, match="int8 or float8"):
        PagedKVCache(cfg, 2, 4, dtype=torch.float8_e5m2)
    with pytest.raises(RuntimeError, match="CUDA"):
        PagedKVCache(cfg, 2, 4, dtype=torch.int8, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        EfficientNGPT(cfg).decoder(2, 4, cache_dtype=torch.int8)
