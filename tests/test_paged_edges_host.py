"""Refusals of the paged key-value cache operators (no GPU) next to those of tests/test_paged_host.py."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from engpt_b200 import kernels as K


def test_writes_are_forward_only():
    """Tensors that need a gradient are refused by every operator that reads or writes them, not only where q is made."""
    with FakeTensorMode():
        c = dict(device="cuda")
        i = torch.empty(3, dtype=torch.int32, **c)
        kp, vp, k, v = (torch.empty(*s, **c) for s in ((8, 2, 16, 64), (8, 2, 16, 64), (3, 2, 64), (3, 2, 64)))
        qkv, rho, cs, s = (torch.empty(*x, **c) for x in ((3, 3, 2, 64), (3,), (9, 32), (2, 64)))

        def write():
            K.write_kv_pages(k, v, i, kp, vp)

        def append():
            K.qkv_append_from_carried(qkv, rho, cs, cs, s, 1e-6, i, i, kp, vp)

        for call, tensors in ((write, (k, v, kp, vp)), (append, (qkv, rho, s, kp, vp))):
            for t in tensors:
                t.requires_grad_(True)
                with pytest.raises(NotImplementedError, match="forward-only"):
                    call()
                t.requires_grad_(False)
