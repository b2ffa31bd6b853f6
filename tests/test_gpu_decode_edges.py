"""Generation with the paged cache on B200, at its edges: replaced parameters, refused rows, the model's block size."""

import pytest
import torch

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
