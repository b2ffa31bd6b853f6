"""Paged key-value cache operators on B200, at their edges: what the tests of ordinary calls do not reach."""

import ctypes
import threading

import numpy as np
import pytest
import torch

from engpt_b200 import _lib, kernels as K
from tests import paged_ref as R
from tests.test_gpu_paged import _clean, append_inputs, attention_inputs, check_attention, make_pools  # noqa: F401

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


# ------------------------------------------------------------------ infinite values
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (2, 2, 128), (8, 1, 64), (2, 2, 48), (4, 1, 80)])
@pytest.mark.parametrize("lengths", [[1, 33, 300], [1] * 5 + [17, 0, 64] * 30, [2500]])
def test_infinite_values_in_use(cuda, dtype, heads, kv_heads, dim, lengths):
    """An infinite element of a value makes that element of its heads' output infinite and no other; two of opposite
    signs make it NaN.  The weights here are all far above the smallest normal number."""
    q, kp, vp, table, lens, scale = attention_inputs(lengths, heads, kv_heads, dim, 16, dtype, seed=dim)
    b = max(range(len(lengths)), key=lambda i: lengths[i])
    n, inf = lengths[b], float("inf")
    marks = [(0, 3, inf), (n - 1, 5, -inf), (n // 2, 5, -inf), (n // 3, dim - 1, inf), (n // 2, dim - 1, -inf)]
    for key, e, x in marks:
        vp[int(table[b, key // 16]), 0, key % 16, e] = x
    if lengths[0] == 1:
        vp[int(table[0, 0]), 0, 0, 7] = inf
    out = K.paged_sdpa(q, kp, vp, table, lens, scale=scale).cpu().double()
    group = heads // kv_heads
    want = torch.zeros_like(out)
    want[b, :group, 3], want[b, :group, 5], want[b, :group, dim - 1] = inf, -inf, float("nan")
    if lengths[0] == 1:
        want[0, :group, 7] = inf
    marked = want != 0
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out[marked].nan_to_num(0.0), want[marked].nan_to_num(0.0))
    ref, vmax, smax = R.attention(q, kp, vp.nan_to_num(nan=0.0, posinf=0.0, neginf=0.0), table, lens, scale)
    tol = R.attention_tolerance(dtype, ref, vmax, smax, dim, max(lengths))
    assert ((out - ref).abs() <= tol)[~marked].all()


# ------------------------------------------------------------------ calls from several host threads
def run_threads(calls, times):
    """Each call `times` times in a thread of its own, all at once, through the C boundary (which holds no lock): the
    status codes of each."""
    codes, gate = [set() for _ in calls], threading.Barrier(len(calls))

    def work(i):
        torch.cuda.synchronize()
        gate.wait()
        for _ in range(times):
            codes[i].add(calls[i]())

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return codes


def test_attention_from_several_threads(cuda):
    """Calls whose kernels need different amounts of shared memory."""
    lib, calls, outs = _lib.load(), [], []
    for seed, (bsz, heads) in enumerate([(8000, 2), (300, 2), (300, 16)]):
        rng = np.random.default_rng(seed)
        lengths = rng.integers(0, 20, bsz).tolist()
        lengths[3] = 700
        pool = sum(R.pages_of(n, 16) for n in lengths)
        table, _ = R.random_table(lengths, 16, 44, pool, rng)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        kp, vp = (torch.randn(pool, 2, 16, 64, generator=gen, device="cuda").bfloat16() for _ in range(2))
        q = torch.randn(bsz, heads, 64, generator=gen, device="cuda").bfloat16()
        args = (q, kp, vp, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device=cuda), 0.125)
        out = torch.empty_like(q)
        call, keep = attention_call(args, out, torch.cuda.Stream())
        calls.append(lambda c=call: lib.engpt_paged_attention(*c))
        outs.append((K.paged_sdpa(*args[:5], scale=args[5]), out, keep))
    torch.cuda.synchronize()
    assert run_threads(calls, 500) == [{0}] * 3
    assert all(torch.equal(want, out) for want, out, _ in outs)


def test_tables_from_several_threads(cuda):
    lib, calls, keep = _lib.load(), [], []
    i32 = dict(dtype=torch.int32, device=cuda)
    for bsz in (8192, 2500, 4000):
        t = dict(lengths=torch.zeros(bsz, **i32), new=torch.zeros(bsz, **i32), table=torch.zeros(bsz, 2, **i32),
                 free=torch.arange(bsz, **i32), count=torch.tensor([bsz], **i32), slots=torch.empty(bsz, **i32),
                 pos=torch.empty(bsz, **i32))
        p, stream = {k: v.data_ptr() for k, v in t.items()}, torch.cuda.Stream()
        call = (p["lengths"], p["new"], None, bsz, p["table"], 2, 2, p["free"], bsz, p["count"], 16, 1, p["slots"],
                p["pos"], stream.cuda_stream)
        calls.append(lambda c=call: lib.engpt_advance_block_tables(*c))
        keep.append((t, stream))
    torch.cuda.synchronize()
    assert run_threads(calls, 1000) == [{0}] * 3
    assert all(int(t["count"]) == len(t["free"]) and (t["slots"] == -1).all() for t, _ in keep)


def test_whole_sequence_attention_from_several_threads(cuda):
    """The CUDA-core kernel at head dims of one instantiation that need different amounts of shared memory."""
    lib, calls, outs = _lib.load(), [], []
    for dim in (136, 200, 256):
        gen = torch.Generator(device="cuda").manual_seed(dim)
        q, k, v = (torch.randn(1, 40, 2, dim, generator=gen, device="cuda") for _ in range(3))
        want, out, stream = K.causal_sdpa(q, k, v, scale=0.1, dropout_p=0.0), torch.empty_like(q), torch.cuda.Stream()
        strides = K.attention_strides(q, k, v, out, head_major=False)
        call = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _lib.F32, 1, 40, 2, dim, 0.1, strides.data_ptr(),
                _lib.ATTN_SIMT, stream.cuda_stream)
        calls.append(lambda c=call: lib.engpt_causal_attention(*c))
        outs.append((want, out, (q, k, v, strides, stream)))
    torch.cuda.synchronize()
    assert run_threads(calls, 500) == [{0}] * 3
    assert all(torch.equal(want, out) for want, out, _ in outs)


@pytest.mark.parametrize("bsz", [2, 300])
def test_attention_as_the_first_cuda_call_of_a_thread(cuda, bsz):
    """A thread that has made no CUDA call has no context of its own yet: both forms on the tensor cores."""
    lib = _lib.load()
    args = attention_inputs([70] + [1] * (bsz - 1), 2, 2, 64, 16, torch.bfloat16)
    out = torch.empty_like(args[0])
    call, keep = attention_call(args, out)
    torch.cuda.synchronize()
    codes = []
    t = threading.Thread(target=lambda: codes.append(lib.engpt_paged_attention(*call)))
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert codes == [0]
    check_attention(args, out)


def test_other_tensor_map_kernels_as_the_first_cuda_call_of_a_thread(cuda):
    lib = _lib.load()
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(1, 256, 2, 64, generator=gen, device="cuda").bfloat16() for _ in range(3))
    want, out = K.causal_sdpa(q, k, v, scale=0.125, dropout_p=0.0, impl="tcgen05"), torch.empty_like(q)
    strides = K.attention_strides(q, k, v, out, head_major=False)
    w, x = (torch.randn(n, 256, generator=gen, device="cuda").bfloat16() for n in (512, 300))
    y, stream = torch.empty(300, 512, device=cuda, dtype=torch.bfloat16), torch.cuda.current_stream().cuda_stream
    calls = [lambda: lib.engpt_causal_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 1, 1, 256, 2, 64,
                                                0.125, strides.data_ptr(), _lib.ATTN_TCGEN05, stream),
             lambda: lib.engpt_gemm_bf16(x.data_ptr(), 256, w.data_ptr(), 256, y.data_ptr(), 512, 300, 512, 256, stream)]
    torch.cuda.synchronize()
    codes = []
    for call in calls:
        t = threading.Thread(target=lambda: codes.append(call()))
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert codes == [0, 0]
    assert torch.equal(out, want)
    ref = x.double() @ w.double().t()      # 256 products of fp32 sums, one rounding
    assert ((y.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -16 * (x.abs().double() @ w.abs().double().t())).all()


# ------------------------------------------------------------------ in-place writes and autograd
def test_writes_are_counted(cuda):
    """The tensors that a call changes in place get a new version, views of them too; inference tensors have none."""
    def state():
        i32 = dict(dtype=torch.int32, device=cuda)
        kp, vp = make_pools(2, 2, 4, 64, torch.bfloat16)
        return dict(lengths=torch.zeros(1, **i32), table=torch.zeros(1, 2, **i32), free=torch.tensor([1, 0], **i32),
                    count=torch.tensor([2], **i32), kp=kp, vp=vp, new=torch.ones(1, **i32))

    def calls(t):
        qkv, rho, cos, sin, scale, pos = append_inputs(1, 2, 64, torch.bfloat16, 1)
        slots, _ = K.advance_block_tables(t["lengths"], t["new"], t["table"], t["free"], t["count"], page_size=4,
                                          max_new=1)
        yield ("lengths", "table", "free", "count")
        K.qkv_append_from_carried(qkv, rho, cos, sin, scale, 1e-6, pos, slots.view(1), t["kp"], t["vp"])
        yield ("kp", "vp")
        K.write_kv_pages(qkv[:, 1], qkv[:, 2], slots.view(1), t["kp"], t["vp"])
        yield ("kp", "vp")
        K.paged_sdpa(qkv[:, 0], t["kp"], t["vp"], t["table"], t["lengths"], scale=1.0)
        yield ()

    t = state()
    before = {k: v._version for k, v in t.items()}
    for changed in calls(t):
        now = {k: v._version for k, v in t.items()}
        assert {k for k in now if now[k] > before[k]} == set(changed)
        before = now
    with torch.enable_grad():
        x = torch.ones(64, device=cuda, dtype=torch.bfloat16, requires_grad=True)
        y = (x * t["kp"]).sum()
    K.write_kv_pages(t["kp"][:1, :, 0], t["kp"][:1, :, 0], t["new"], t["kp"], t["vp"])
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    with torch.inference_mode():
        t = state()
    assert len(list(calls(t))) == 4
