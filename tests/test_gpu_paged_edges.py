"""Paged key-value cache operators on B200, at their edges: what the tests of ordinary calls do not reach."""

import ctypes

import pytest
import torch

from engpt_b200 import _lib, kernels as K
from tests.test_gpu_paged import _clean, attention_inputs, check_attention  # noqa: F401

pytestmark = pytest.mark.gpu


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def attention_call(args, out, stream=None):
    """engpt_paged_attention on the tensors of `attention_inputs` with the result at `out`: the call's argument list and
    what has to live as long as it runs."""
    q, kp, vp, table, lens, scale = args
    (bsz, heads, dim), (pool, kv_heads, page, _) = q.shape, kp.shape
    code, width = _lib.dtype_code(q.dtype), table.shape[1]
    floats = _lib.load().engpt_paged_attention_floats(code, bsz, heads, kv_heads, dim, width, page)
    work = torch.empty(max(floats, 1), device=q.device)
    strides, pages = i64(*q.stride()[:2]), i64(*kp.stride()[:3], *vp.stride()[:3])
    stream = stream or torch.cuda.current_stream()
    return (q.data_ptr(), strides, kp.data_ptr(), vp.data_ptr(), pages, code, bsz, heads, kv_heads, dim, pool, page,
            table.data_ptr(), table.stride(0), width, lens.data_ptr(), scale, out.data_ptr(), work.data_ptr(),
            stream.cuda_stream), (args, work, stream)


# ------------------------------------------------------------------ the C boundary
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 48])
@pytest.mark.parametrize("lengths", [[40, 0, 300], [0, 17, 64, 1] * 40])
@pytest.mark.parametrize("shift", [0, 1, 2, 4, 8])
def test_output_of_any_alignment(cuda, dtype, dim, lengths, shift):
    """`o` may start at any element of a larger buffer (rows without keys among those written)."""
    args = attention_inputs(lengths, 4, 4, dim, 16, dtype, seed=dim)
    n = args[0].numel()
    buf = torch.full((n + 32,), 7.5, dtype=dtype, device=cuda)
    out = buf[8 + shift:8 + shift + n].view(args[0].shape)
    call, keep = attention_call(args, out)
    assert _lib.load().engpt_paged_attention(*call) == 0
    torch.cuda.synchronize()
    check_attention(args, out)
    assert (buf[:8 + shift] == 7.5).all() and (buf[8 + shift + n:] == 7.5).all()
