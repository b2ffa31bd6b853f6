"""Refusals of the paged key-value cache operators (no GPU) next to those of tests/test_paged_host.py."""

import os
import subprocess
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from engpt_b200 import build as B, kernels as K


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


def test_the_library_builds_without_torch():
    """Callers of the C ABI alone have no torch: the build then leaves the Python binding out."""
    assert os.path.exists(B.LIB)
    code = ("import sys, runpy; sys.modules['torch'] = None\n"
            "import importlib.util as u; find = u.find_spec\n"
            "u.find_spec = lambda name, *a: None if name == 'torch' else find(name, *a)\n"
            f"ns = runpy.run_path({B.__file__!r})\n"
            "print(ns['build']())")
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert res.returncode == 0 and res.stdout.strip() == B.LIB, res.stderr
