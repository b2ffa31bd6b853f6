"""Generation with the paged cache on B200, at its edges: replaced parameters, refused rows, the model's block size."""

import pytest
import torch

from engpt_b200 import _lib
from tests.helpers import seeded_model
from tests.test_gpu_decode import CFGS, TOL, _clean, forward_logits, model_on, row_err, tokens  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("how", ["load", "data"])
def test_replaced_parameters_are_taken(cuda, dtype, graphs, how):
    """Parameters that have become other tensors: the next refresh takes all of them, the step before it the old ones."""
    model, other = model_on(cuda, "dh64"), model_on(cuda, "dh64", seed=7)
    idx = tokens(CFGS["dh64"], (1, 12), 8)
    before, after = (forward_logits(m, idx[:, :1], dtype)[:, 0] for m in (model, other))
    assert row_err(before, after) > 0.5
    dec = model.decoder(1, 4, dtype=dtype)
    dec.enable_cuda_graphs(graphs)
    dec.step(idx[:, 0])
    state = {k: v.clone() for k, v in other.state_dict().items()}
    if how == "load":
        model.load_state_dict(state, assign=True)
    else:
        for k, p in model.named_parameters():
            p.data = state[k]
    assert row_err(forward_logits(model, idx[:, :1], dtype)[:, 0], after) < TOL[dtype]
    dec.cache.reset()
    assert row_err(dec.step(idx[:, 0]).float(), before) < TOL[dtype]
    dec.refresh_weights()
    dec.cache.reset()
    assert row_err(dec.step(idx[:, 0]).float(), after) < TOL[dtype]
    # and a whole generation of the new model: prompt and steps
    full = forward_logits(model, idx, dtype)
    dec.prefill(idx[:, :9])
    for t in range(9, 12):
        assert row_err(dec.step(idx[:, t]).float(), full[:, t]) < TOL[dtype]


def test_refresh_refuses_other_types_and_shapes(cuda):
    """A refused refresh leaves the decoder as it was."""
    idx = tokens(CFGS["dh64"], (1, 3), 8)
    for dtype in (torch.float32, torch.bfloat16):
        model = model_on(cuda, "dh64")
        dec = model.decoder(1, 4, dtype=dtype)
        want = dec.step(idx[:, 0])
        name, p = "blocks.1.s_u", model.blocks[1].s_u
        for bad in (p.data.bfloat16(), p.data.cpu(), p.data[:-1]):
            keep, p.data = p.data, bad
            with pytest.raises(ValueError, match=name):
                dec.refresh_weights()
            p.data = keep
        model.bfloat16()
        with pytest.raises(ValueError, match="token_emb"):
            dec.refresh_weights()
        dec.cache.reset()
        assert torch.equal(dec.step(idx[:, 0]), want)
        model.load_state_dict(seeded_model(CFGS["dh64"], 0).state_dict(), assign=True)
        model.cuda()
        dec.refresh_weights()
        dec.cache.reset()
        assert torch.equal(dec.step(idx[:, 0]), want)


@pytest.mark.parametrize("graphs", [False, True])
def test_steps_stop_at_the_block_size(cuda, graphs):
    """A cache of whole pages has room behind the model's block size; a step there is refused as a forward is."""
    model = seeded_model(dict(CFGS["dh64"], block_size=20), 0).to(cuda).requires_grad_(False)
    idx = tokens(CFGS["dh64"], (3, 21), 3)
    full = forward_logits(model, idx[:, :20], torch.float32)
    dec = model.decoder(3, 6, page_size=16, dtype=torch.float32)
    assert dec.cache.capacity == 32
    dec.enable_cuda_graphs(graphs)
    dec.prefill(idx[:, :19], lengths=[19, 10, 19])
    on = torch.tensor([True, True, False])
    logits = dec.step(torch.stack([idx[0, 19], idx[1, 10], idx[2, 19]]), on)
    assert row_err(logits[:1], full[0, 19][None]) < TOL[torch.float32]
    assert row_err(logits[1:2], full[1, 10][None]) < TOL[torch.float32]
    _lib.raise_on_device_status()
    logits = dec.step(torch.stack([idx[0, 20], idx[1, 11], idx[2, 19]]), on)
    assert dec.cache.lengths.tolist() == [20, 12, 19]
    assert row_err(logits[1:2], full[1, 11][None]) < TOL[torch.float32]
    with pytest.raises(_lib.EngptError, match="site 40"):
        _lib.raise_on_device_status()
    dec.step(torch.stack([idx[0, 20], idx[1, 12], idx[2, 19]]), torch.tensor([False, True, True]))
    assert dec.cache.lengths.tolist() == [20, 13, 20]      # a full row that is not asked to grow is no error


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_refused_rows_have_zero_logits(cuda, dtype):
    """A prompt or a step that finds no pages: the row's cache is as the refusal left it, its logits are zeros, and the
    other rows are served."""
    model = model_on(cuda, "dh64")
    idx = tokens(CFGS["dh64"], (3, 40), 6)
    full = forward_logits(model, idx, dtype)
    dec = model.decoder(3, 4, page_size=16, dtype=dtype)
    logits = dec.prefill(idx[:, :30], lengths=[16, 30, 20]).float()      # one page, two, and two where one is left
    assert dec.cache.lengths.tolist() == [16, 30, 0] and int(dec.cache.free_count) == 1
    assert row_err(logits[:1], full[0, 15][None]) < TOL[dtype] and row_err(logits[1:2], full[1, 29][None]) < TOL[dtype]
    assert (logits[2] == 0).all()
    with pytest.raises(_lib.EngptError, match="site 41"):
        _lib.raise_on_device_status()
    dec.step(torch.tensor([0, 0, 0]), torch.tensor([True, False, False]))     # row 0 takes the last page
    _lib.raise_on_device_status()
    dec.release([0])
    dec.prefill(idx[:1, :32], rows=[0])
    logits = dec.step(torch.stack([idx[0, 32], idx[1, 30], idx[2, 0]])).float()
    assert dec.cache.lengths.tolist() == [32, 31, 0]
    assert (logits[0] == 0).all() and (logits[2] == 0).all()
    assert row_err(logits[1:2], full[1, 30][None]) < TOL[dtype]
    with pytest.raises(_lib.EngptError, match="site 41"):
        _lib.raise_on_device_status()


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_inside_and_outside_inference_mode(cuda, dtype, graphs):
    """What is made in a call under inference_mode (the decoder, its captured step, the model's workspace) serves calls
    outside of it, and the other way round."""
    idx = tokens(CFGS["dh64"], (2, 12), 5)
    runs = []
    for modes in ((False,) * 5, (True, False) * 3, (False, True) * 3):
        with torch.inference_mode(modes[0]), torch.no_grad():
            model = model_on(cuda, "dh64")
            model.enable_cuda_graphs(graphs)
            dec = model.decoder(2, 8, page_size=16, dtype=dtype)
            dec.enable_cuda_graphs(graphs)
        out = []
        for i, inside in enumerate(modes[1:5]):
            with torch.inference_mode(inside), torch.no_grad():
                dec.refresh_weights()
                dec.cache.reset()
                out.append(dec.prefill(idx[:, :9]).clone())
                out.append(dec.step(idx[:, 9]).clone())
                out.append(dec.generate(idx[:, :9], 3).clone())
                out.append(forward_logits(model, idx, dtype).clone())
                if dtype == torch.bfloat16:     # with targets: the fused head's scratch is kept too
                    with torch.autocast("cuda", dtype=torch.bfloat16):
                        out.append(model(idx.cuda(), idx.cuda())[1].clone())
        runs.append(out)
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_generate_releases_its_rows_when_pick_raises(cuda):
    model = model_on(cuda, "dh64")
    idx = tokens(CFGS["dh64"], (2, 20), 5)
    dec = model.decoder(3, 9, page_size=16, dtype=torch.float32)
    dec.prefill(idx[:1], rows=[2])
    for at in (1, 3):
        seen = []

        def pick(z):
            seen.append(z)
            if len(seen) == at:
                raise KeyError("stop")
            return z.argmax(-1)

        with pytest.raises(KeyError):
            dec.generate(idx, 8, pick=pick)
        assert dec.cache.lengths.tolist() == [0, 0, 20] and int(dec.cache.free_count) == 7
    with pytest.raises(ValueError):
        dec.generate(idx, 8, lengths=[21, 3])
    assert dec.cache.lengths.tolist() == [0, 0, 20]
