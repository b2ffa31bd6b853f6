"""Generation with the paged cache in 8 bits on B200."""

import numpy as np
import pytest
import torch

from engpt_b200 import PagedKVCache, ModelConfig, _lib, kernels as K
from tests import paged_q8_ref as Q, paged_ref as R
from tests.test_gpu_decode import CFGS, forward_logits, model_on, row_err, tokens

pytestmark = pytest.mark.gpu

KINDS = [torch.int8, torch.float8_e4m3fn]


@pytest.fixture(autouse=True)
def _clean(cuda):
    _lib.clear_device_status()
    with torch.no_grad():
        yield
    status = _lib.device_status()
    _lib.clear_device_status()
    assert status == 0, f"a kernel recorded a device-side failure: {status:#x}"


# The cache's rounding is what differs from the whole-sequence forward.  Rows of k have length about 1; with a block's
# largest element of some 3.5 root mean squares, int8 steps of 1/127 of it are off by 0.29 * 3.5 / 127 = 0.8 % of a
# root mean square (e4m3: 2^-4 / sqrt(12) * 1.2 = 2.2 %, a relative error).  A score 8 q.k (16, 128 wide) then is off
# by up to 0.022 * 8 = 0.18 in the sum of 64 random errors' length / sqrt(64), 0.022, so are the weights, and the
# values by 2.2 %: some 3 % of an attention branch, which enters the state with alpha = 0.05 or so per layer and is
# normalised: 0.2 % a layer, and up to 3 layers.  The bound is the engines' own tolerance for represented states.
TOL = 2e-2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("name", list(CFGS))
@pytest.mark.parametrize("page_size,scale_block", [(8, None), (16, 16), (64, None), (64, 64)])
def test_prefill_and_steps_are_near_the_forward(cuda, name, kind, dtype, page_size, scale_block):
    cfg = CFGS[name]
    model = model_on(cuda, name)
    lens, steps = [1, 33, 64, 50], 40
    idx = tokens(cfg, (4, 64 + steps), 1)
    full = forward_logits(model, idx, dtype)
    dec = model.decoder(4, 4 * (160 // page_size), page_size=page_size, dtype=dtype, cache_dtype=kind,
                        scale_block=scale_block)
    assert dec.cache.quantised and dec.cache.k_pages.dtype == kind
    logits = dec.prefill(idx[:, :64], lengths=lens).float()
    for b, n in enumerate(lens):                          # a prompt's own logits do not come from the cache
        assert row_err(logits[b:b + 1], full[b, n - 1:n]) < (1e-5 if dtype == torch.float32 else TOL)
    for s in range(steps):
        nxt = torch.stack([idx[b, n + s] for b, n in enumerate(lens)])
        logits = dec.step(nxt).float()
        for b, n in enumerate(lens):
            assert row_err(logits[b:b + 1], full[b, n + s:n + s + 1]) < TOL, (b, s)
    assert dec.cache.lengths.tolist() == [n + steps for n in lens]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("name", ["dh64", "dh128", "small"])
def test_every_call_of_a_generation(cuda, monkeypatch, name, kind, dtype):
    """What the decoder asks of the three operators, call by call, against their 64-bit forms."""
    model = model_on(cuda, name)
    idx = tokens(CFGS[name], (3, 30), 1)
    calls = {"write": 0, "append": 0, "attend": 0}
    write, append, attend = K.write_kv_pages_q8, K.qkv_append_from_carried_q8, K.paged_sdpa_q8

    def stored(cache, before, k, v, slots, err):
        for p, x in ((0, k), (1, v)):
            Q.check_store(cache[p], cache[2 + p], before[p], before[2 + p], x, slots,
                          err * x.abs().amax(-1, keepdim=True) if err else 0.0)

    def spy_write(k, v, slots, *cache):
        before = [Q.raw(cache[0]), Q.raw(cache[1]), cache[2].cpu().clone(), cache[3].cpu().clone()]
        write(k, v, slots, *cache)
        stored(cache, before, *(x.reshape(-1, *x.shape[-2:]).cpu().double() for x in (k, v)),
               slots.reshape(-1).tolist(), 0.0)
        calls["write"] += 1

    def spy_append(qkv, rho, cos, sin, s_qk, eps, pos, slots, *cache, qk_mult):
        before = [Q.raw(cache[0]), Q.raw(cache[1]), cache[2].cpu().clone(), cache[3].cpu().clone()]
        q = append(qkv, rho, cos, sin, s_qk, eps, pos, slots, *cache, qk_mult=qk_mult)
        rq, rk, rv = R.postprocess(qkv, rho, cos, sin, s_qk.double() * qk_mult, eps, pos)
        # (2^-18 of a row's largest value: tests/test_gpu_paged_q8.py; the product with qk_mult rounds once more)
        stored(cache, before, rk, rv, slots.tolist(), 2.0 ** -18)
        lim = torch.finfo(qkv.dtype).eps / 2 * rq.abs() + 2.0 ** -18 * rq.abs().amax(-1, keepdim=True)
        assert ((q.cpu().double() - rq).abs() <= lim).all()
        calls["append"] += 1
        return q

    def spy_attend(q, kp, vp, ks, vs, table, lengths, *, scale):
        o = attend(q, kp, vp, ks, vs, table, lengths, scale=scale)
        ref, tol = Q.attention(q, (kp, vp, ks, vs), table, lengths, scale)
        assert ((o.cpu().double() - ref).abs() <= tol).all()
        calls["attend"] += 1
        return o

    monkeypatch.setattr(K, "write_kv_pages_q8", spy_write)
    monkeypatch.setattr(K, "qkv_append_from_carried_q8", spy_append)
    monkeypatch.setattr(K, "paged_sdpa_q8", spy_attend)
    dec = model.decoder(4, 40, page_size=16, dtype=dtype, cache_dtype=kind, scale_block=8)
    dec.generate(idx, 12, lengths=[30, 3, 17])
    layers = CFGS[name]["n_layer"]
    assert calls == {"write": layers, "append": 11 * layers, "attend": 11 * layers}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_graphed_steps_equal_eager_steps(cuda, kind, dtype):
    cfg = CFGS["dh64"]
    model = model_on(cuda, "dh64")
    idx = tokens(cfg, (3, 60), 2)
    runs = []
    for graphs in (False, True):
        dec = model.decoder(3, 30, page_size=16, dtype=dtype, cache_dtype=kind)
        dec.enable_cuda_graphs(graphs)
        dec.prefill(idx[:, :20], lengths=[20, 7, 13])
        out = [dec.step(idx[:, 20 + s], torch.tensor([True, s % 3 != 1, True])).clone() for s in range(30)]
        dec.release([1])
        dec.prefill(idx[1:2, :9], rows=[1])               # the freed pages again, in a block that starts anew
        out += [dec.step(idx[:, 50 + s]).clone() for s in range(5)]
        runs.append((torch.stack(out), dec.cache.lengths.tolist(),
                     [dec.cache.read(i, 1, 14) for i in range(cfg["n_layer"])]))
    assert runs[0][1] == runs[1][1] == [55, 14, 48]
    on = torch.tensor([[True, s % 3 != 1, True] for s in range(30)] + [[True] * 3] * 5, device=cuda)
    assert torch.equal(runs[0][0][on], runs[1][0][on])
    for a, b in zip(runs[0][2], runs[1][2]):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("kind,rel", [(torch.int8, 0.0), (torch.float8_e4m3fn, 2.0 ** -4)])
def test_reading_a_request_back(cuda, kind, rel):
    """A prompt's k and v in the 8-bit cache are those of a full one, within half a step."""
    cfg = CFGS["dh64"]
    model = model_on(cuda, "dh64")
    idx = tokens(cfg, (2, 50), 2)
    full = model.decoder(2, 16, page_size=16, dtype=torch.float32)
    small = model.decoder(2, 16, page_size=16, dtype=torch.float32, cache_dtype=kind, scale_block=16)
    for dec in (full, small):
        dec.prefill(idx, lengths=[50, 37])
    for layer in range(cfg["n_layer"]):
        for row, n in ((0, 50), (1, 37)):
            want, got = full.cache.read(layer, row, 60), small.cache.read(layer, row, 60, dtype=torch.float32)
            for x, y in zip(want, got):
                assert x.dtype == y.dtype == torch.float32 and x.shape == y.shape == (60, cfg["n_head"], 64)
                assert (x[n:] == 0).all() and (y[n:] == 0).all() and (x[:n] != 0).any(-1).all()
                for t in range(0, n, 16):
                    a, b = x[t:min(t + 16, n)].double(), y[t:min(t + 16, n)].double()
                    amax = a.abs().amax((0, 2), keepdim=True)
                    lim = 0.5 / 127 * amax if kind == torch.int8 else torch.maximum(rel * a.abs(), 2.0 ** -10 / 448 * amax)
                    assert ((a - b).abs() <= lim * (1 + 2.0 ** -14)).all()
    assert small.cache.read(0, 0, 0)[0].shape == (0, cfg["n_head"], 64)
    with pytest.raises(ValueError):
        small.cache.read(0, 2, 5)


def test_sizes_and_defaults(cuda):
    cfg = ModelConfig(**CFGS["dh64"])
    for page, block in ((64, 16), (8, 8), (24, 8), (20, 20)):
        c = PagedKVCache(cfg, 2, 4, page_size=page, dtype=torch.int8)
        assert c.scale_block == block and c.k_scales.shape == (3, 4, 4, page // block) and len(c.layer(0)) == 4
    assert PagedKVCache(cfg, 2, 4).k_scales is None
    model = model_on(cuda, "dh64")
    assert model.decoder(2, 4).cache.k_pages.dtype == torch.bfloat16
    with pytest.raises(NotImplementedError):
        model.decoder(2, 4, cache_dtype=torch.float32)         # another compute type's cache
    with pytest.raises(NotImplementedError):
        model.decoder(2, 4, dtype=torch.int8)


def test_two_streams_and_graphs_at_once(cuda):
    """Two decoders on streams of their own, one of them graphed, give what they give alone."""
    cfg = CFGS["dh64"]
    model = model_on(cuda, "dh64")
    idx = tokens(cfg, (2, 60), 4)
    nxt = idx.cuda()

    def run(dec, out):
        for s in range(40):
            out.append(dec.step(nxt[:, 20 + s]).clone())

    decs, alone = [], []
    for i in range(2):
        for keep in (alone, decs):
            dec = model.decoder(2, 20, page_size=16, cache_dtype=KINDS[i])
            dec.enable_cuda_graphs(i == 1)
            dec.prefill(idx[:, :20])
            dec.step(nxt[:, 20], torch.zeros(2, dtype=torch.bool))     # (captures)
            keep.append(dec)
    torch.cuda.synchronize()
    want = [[], []]
    for i in range(2):
        run(alone[i], want[i])
    torch.cuda.synchronize()
    got, streams = [[], []], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in range(40):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(decs[i].step(nxt[:, 20 + s]).clone())
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(torch.stack(want[i]), torch.stack(got[i]))
