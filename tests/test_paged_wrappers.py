"""CPU: what the paged wrappers pass on (workspace sizes, numbers) and keep between calls."""
from __future__ import annotations

import ctypes as C
import os

import pytest
import torch

from tests.paged_inputs import cache

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "scope_amd", "libscope_amd.so")
needs_lib = pytest.mark.skipif(not os.path.exists(LIB), reason="libscope_amd.so not built")


class Reached(Exception):
    """A call passed the wrapper's checks: (name, arguments)."""


@pytest.fixture()
def on_cpu(monkeypatch):
    """The wrappers up to the library call, which is raised instead of made."""
    from scope_amd import ops

    def reached(dev, name, *args):
        raise Reached(name, args)

    monkeypatch.setattr(ops, "_gpu", lambda who, *ts: torch.device("cpu"))
    monkeypatch.setattr(ops, "_launch", reached)
    return ops


@needs_lib
def test_a_workspace_size_is_the_librarys_own(on_cpu, monkeypatch):
    """A size that a stand-in for the library once answered is not used again."""
    from scope_amd import _lib

    ops = on_cpu
    c = cache([40, 5], Hq=4, Hkv=2, D=64, bs=16)
    MP = c["table"].shape[1]
    num, idx = torch.ones(2, 2, dtype=torch.int32), torch.zeros(2, 2, 3, dtype=torch.int32)
    real, sizes = torch.empty, []

    def empty(*a, **kw):
        if kw.get("dtype") == torch.uint8:
            sizes.append(a[0])
        return real(*a, **kw)

    def call():
        with pytest.raises(Reached):
            ops.paged_decode_attn(c["q"], c["k_pages"], c["v_pages"], c["table"], c["lens"], scale=0.1, kv_num=num, kv_idx=idx,
                                  mass=torch.zeros(2, 2, MP))

    with monkeypatch.context() as m:
        m.setattr(ops, "query", lambda *a: 16)
        call()
    with monkeypatch.context() as m:
        m.setattr(torch, "empty", empty)
        call()
    p = _lib.PagedCache(2, 2, 64, 16, MP)
    assert sizes == [_lib.load().scope_paged_attn_workspace_bytes(C.byref(p), 4, 3, 1)] and sizes[0] > 16
