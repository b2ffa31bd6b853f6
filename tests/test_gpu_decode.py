"""Generation with the paged cache on B200: prefill and steps against whole-sequence forwards of the same model."""

import numpy as np
import pytest
import torch

from engpt_b200 import PagedDecoder, _lib
from oracle import ngpt_oracle as O
from tests.helpers import SMALL, seeded_model, state_numpy

pytestmark = pytest.mark.gpu

# head_dim 64 and 128 (bf16 tensor-core path) and 16 (the reference's small equivalence model)
CFGS = {
    "dh64": dict(vocab_size=301, block_size=160, n_layer=3, n_head=4, n_embd=256, mlp_ratio=4.0, dropout=0.0),
    "dh128": dict(vocab_size=301, block_size=160, n_layer=2, n_head=2, n_embd=256, mlp_ratio=4.0, dropout=0.0),
    "small": dict(SMALL, block_size=160),
}


@pytest.fixture(autouse=True)
def _clean(cuda):
    _lib.clear_device_status()
    with torch.no_grad():
        yield
    status = _lib.device_status()
    _lib.clear_device_status()
    assert status == 0, f"a kernel recorded a device-side failure: {status:#x}"


def model_on(cuda, name, seed=0):
    return seeded_model(CFGS[name], seed).to(cuda).requires_grad_(False)


def tokens(cfg, shape, seed):
    return torch.randint(0, cfg["vocab_size"], shape, generator=torch.Generator().manual_seed(seed))


def forward_logits(model, idx, dtype):
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=dtype == torch.bfloat16):
        return model(idx.cuda())[0].float()


# fp32: the two paths differ in the order of fp32 sums only.  bf16: the target's tolerance for represented states
# between engines, 2e-2 of the row norm
TOL = {torch.float32: 1e-5, torch.bfloat16: 2e-2}


def row_err(a, b):
    return ((a - b).norm(dim=-1) / b.norm(dim=-1)).max().item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", list(CFGS))
@pytest.mark.parametrize("page_size", [8, 16, 64])
def test_prefill_and_steps_match_the_forward(cuda, name, dtype, page_size):
    cfg = CFGS[name]
    model = model_on(cuda, name)
    lens, steps = [1, 33, 64, 50], 40
    idx = tokens(cfg, (4, 64 + steps), 1)
    full = forward_logits(model, idx, dtype)
    dec = model.decoder(4, 4 * (160 // page_size), page_size=page_size, dtype=dtype)
    logits = dec.prefill(idx[:, :64], lengths=lens).float()
    for b, n in enumerate(lens):
        assert row_err(logits[b:b + 1], full[b, n - 1:n]) < TOL[dtype]
    for s in range(steps):
        nxt = torch.stack([idx[b, n + s] for b, n in enumerate(lens)])
        logits = dec.step(nxt).float()
        for b, n in enumerate(lens):
            assert row_err(logits[b:b + 1], full[b, n + s:n + s + 1]) < TOL[dtype], (b, s)
    assert dec.cache.lengths.tolist() == [n + steps for n in lens]


def test_steps_match_the_oracle(cuda):
    """fp32 decoding from an empty cache, token by token, against the independent numpy forward."""
    cfg = CFGS["small"]
    model = seeded_model(cfg, 3)
    w = state_numpy(model)
    model = model.to(cuda).requires_grad_(False)
    idx = tokens(cfg, (2, 30), 5)
    ref, _, _ = O.efficient_ngpt_forward(O.OracleConfig(**cfg), w, idx.numpy(), None)
    dec = model.decoder(2, 8, page_size=8, dtype=torch.float32)
    for t in range(30):
        logits = dec.step(idx[:, t]).cpu().numpy()
        err = np.abs(logits - ref[:, t]).max() / np.abs(ref).max()
        assert err < 1e-5, (t, err)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_graphed_steps_equal_eager_steps(cuda, dtype):
    cfg = CFGS["dh64"]
    model = model_on(cuda, "dh64")
    idx = tokens(cfg, (3, 60), 2)
    runs = []
    for graphs in (False, True):
        dec = model.decoder(3, 30, page_size=16, dtype=dtype)
        dec.enable_cuda_graphs(graphs)
        dec.prefill(idx[:, :20], lengths=[20, 7, 13])
        out = [dec.step(idx[:, 20 + s], torch.tensor([True, s % 3 != 1, True])).clone() for s in range(30)]
        runs.append((torch.stack(out), dec.cache.lengths.tolist()))
    assert runs[0][1] == runs[1][1] == [50, 27, 43]
    on = torch.tensor([[True, s % 3 != 1, True] for s in range(30)], device=cuda)
    assert torch.equal(runs[0][0][on], runs[1][0][on])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("outer", [torch.bfloat16, torch.float16])
def test_an_outer_autocast_region_changes_nothing(cuda, dtype, outer):
    cfg = CFGS["dh64"]
    model = model_on(cuda, "dh64")
    idx = tokens(cfg, (2, 12), 3)
    logits = []
    for enabled in (False, True):
        dec = model.decoder(2, 4, page_size=16, dtype=dtype)
        with torch.autocast("cuda", dtype=outer, enabled=enabled):
            logits.append([dec.prefill(idx[:, :10]), dec.step(idx[:, 10]), dec.step(idx[:, 11])])
    assert all(torch.equal(a, b) for a, b in zip(*logits))


def test_requests_come_and_go(cuda):
    """Rows are released and refilled while others decode; every request sees only its own tokens."""
    cfg = CFGS["dh64"]
    dtype = torch.float32
    model = model_on(cuda, "dh64")
    dec = model.decoder(3, 18, page_size=16, dtype=dtype)
    seqs = {r: tokens(cfg, (1, 90), 10 + r) for r in range(5)}
    full = {r: forward_logits(model, s, dtype)[0] for r, s in seqs.items()}
    where, at = {0: 0, 1: 1}, {0: 40, 1: 3}               # request -> row, tokens so far
    dec.prefill(torch.cat([seqs[0][:, :40], seqs[1][:, :40]]), rows=[0, 1], lengths=[40, 3])

    def step(requests):
        nxt, active = torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.bool)
        for r in requests:
            nxt[where[r]], active[where[r]] = seqs[r][0, at[r]], True
        logits = dec.step(nxt, active)
        for r in requests:
            assert row_err(logits[where[r]][None], full[r][at[r]][None]) < TOL[dtype], r
            at[r] += 1

    for _ in range(9):
        step([0, 1])
    where[2], at[2] = 2, 17
    got = dec.prefill(seqs[2][:, :17], rows=[2])
    assert row_err(got, full[2][16][None]) < TOL[dtype]
    for _ in range(8):
        step([0, 2])
    dec.release([where.pop(1)])
    where[3], at[3] = 1, 60
    dec.prefill(seqs[3][:, :60], rows=[1])
    for _ in range(10):
        step([0, 2, 3])
    # row 0's request ends; a new one takes the row without a release in between
    where.pop(0)
    where[4], at[4] = 0, 50
    dec.prefill(seqs[4][:, :50], rows=[0])
    for _ in range(12):
        step([2, 3, 4])
    used = sum(-(-at[r] // 16) for r in where)
    assert int(dec.cache.free_count) == 18 - used
    dec.release([0, 1, 2])
    assert int(dec.cache.free_count) == 18
    assert sorted(dec.cache.free_pages.tolist()) == list(range(18))


def test_generate_equals_repeated_forwards(cuda):
    cfg = CFGS["dh64"]
    model = model_on(cuda, "dh64")
    idx = tokens(cfg, (2, 12), 4)
    lens = [12, 9]
    dec = model.decoder(3, 9, page_size=16, dtype=torch.float32)
    got = dec.generate(idx, 20, lengths=lens).cpu()
    for b, n in enumerate(lens):
        seq = idx[b:b + 1, :n]
        for t in range(20):
            nxt = int(forward_logits(model, seq, torch.float32)[0, -1].argmax())
            assert nxt == int(got[b, t]), (b, t)
            seq = torch.cat([seq, torch.tensor([[nxt]])], 1)
    assert int(dec.cache.free_count) == 9


def test_pool_runs_out(cuda):
    """A step that finds no page refuses the row, reports it, and serves the others."""
    cfg = CFGS["dh64"]
    model = model_on(cuda, "dh64")
    dec = model.decoder(2, 3, page_size=16, dtype=torch.float32)
    idx = tokens(cfg, (2, 60), 6)
    full = forward_logits(model, idx, torch.float32)
    dec.prefill(idx[:, :31], lengths=[20, 16])            # two pages and one: none left, row 1's is full
    logits = dec.step(torch.stack([idx[0, 20], idx[1, 16]]))
    assert dec.cache.lengths.tolist() == [21, 16]
    assert row_err(logits[:1], full[0, 20][None]) < 1e-5
    with pytest.raises(_lib.EngptError, match="site 41"):
        _lib.raise_on_device_status()
    dec.release([0])
    logits = dec.step(torch.stack([idx[0, 0], idx[1, 16]]))
    assert row_err(logits[1:], full[1, 16][None]) < 1e-5


def test_weights_are_taken_again(cuda):
    cfg = CFGS["dh64"]
    model = model_on(cuda, "dh64")
    other = model_on(cuda, "dh64", seed=7)
    idx = tokens(cfg, (1, 10), 8)
    for dtype in (torch.bfloat16, torch.float32):
        dec = model.decoder(1, 4, dtype=dtype)
        dec.enable_cuda_graphs()
        dec.step(idx[:, 0])
        model.load_state_dict(other.state_dict())
        dec.refresh_weights()
        dec.cache.reset()
        want = forward_logits(other, idx[:, :1], dtype)[:, 0]
        assert row_err(dec.step(idx[:, 0]).float(), want) < TOL[dtype]
        model.load_state_dict(seeded_model(cfg, 0).state_dict())


def test_decoder_refusals(cuda):
    cfg = CFGS["dh64"]
    model = model_on(cuda, "dh64")
    dec = model.decoder(2, 8, page_size=16, max_len=64, dtype=torch.float32)
    assert dec.cache.capacity == 64
    idx = tokens(cfg, (2, 65), 9)
    for bad in (lambda: dec.prefill(idx), lambda: dec.prefill(idx[:, :8], rows=[0, 0]),
                lambda: dec.prefill(idx[:, :8], rows=[0, 2]), lambda: dec.prefill(idx[:, :8], lengths=[0, 3]),
                lambda: dec.prefill(idx[:, :8], lengths=[9, 3]), lambda: dec.prefill(idx[:, :8], rows=[1]),
                lambda: dec.prefill(idx[0, :8]), lambda: dec.step(idx[:1, 0]),
                lambda: dec.step(idx[:, 0], torch.ones(2)), lambda: dec.release([5]),
                lambda: dec.generate(idx[:, :60], 6), lambda: dec.generate(idx[:, :6], 0),
                lambda: dec.generate(idx[:1].repeat(3, 1), 1), lambda: model.decoder(0, 4)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        model.decoder(1, 4, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        PagedDecoder(seeded_model(cfg), 1, 4)
