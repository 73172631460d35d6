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


@needs_lib
def test_more_logits_than_a_launch_holds_are_refused():
    """2^32 work-items or more: the stated refusal, before the launch (the pointers are never followed)."""
    from scope_amd import _lib

    lib, one = _lib.load(), C.c_void_p(16)
    # (512 threads of 8 words, and 1024 with rows in eights where the history is long)
    for B, V, T in ((65535, 2 ** 19 + 1, 5), (65535, 2 ** 31 - 1, 5), (32768, 2 ** 20, 5), (65529, 524289, 20000), (32761, 2 ** 20, 20000)):
        p = _lib.PenaltyParams(B=B, type=2, V=V, T=T, repetition=1.0, temperature=1.0)
        rc = lib.scope_logit_penalties(C.byref(p), one, one, one, *[None] * 8, one, None)
        assert rc == -1 and "more than one launch holds" in lib.scope_last_error().decode(), lib.scope_last_error()


@pytest.mark.parametrize("x,want", [(2 ** 63 - 1, 2 ** 31 - 1), (2 ** 40, 2 ** 31 - 1), (-2 ** 40, -2 ** 31), (2 ** 31, 2 ** 31 - 1), (10 ** 30, 2 ** 31 - 1),
                                    (2 ** 31 - 1, 2 ** 31 - 1), (-2 ** 31, -2 ** 31), (7, 7), (-1, -1), (True, 1)])
def test_numbers_past_32_bits_stay_on_their_side(on_cpu, x, want):
    """A number counts as a tensor of it does."""
    ops = on_cpu
    dev = torch.device("cpu")
    assert ops._ints("x", "x", x, 3, dev).tolist() == [want] * 3
    if -2 ** 63 <= x < 2 ** 63 and not isinstance(x, bool):
        assert ops._ints("x", "x", torch.tensor([x] * 3), 3, dev).tolist() == [want] * 3


def test_calls_with_numbers_past_32_bits_are_made(on_cpu):
    ops = on_cpu
    table, mass, lens = torch.zeros((2, 5), dtype=torch.int32), torch.zeros((2, 1, 5)), torch.tensor([80, 3])
    with pytest.raises(Reached):
        ops.paged_evict(table, mass, lens, 2 ** 63 - 1, bs=16)
    z, t = torch.zeros(2, 70), torch.zeros(2, 9, dtype=torch.int64)
    for kw in (dict(n_prompt=2 ** 63 - 1), dict(first=2 ** 40), dict(first=-2 ** 40)):
        with pytest.raises(Reached):
            ops.logit_penalties(z, t, 2 ** 40, **kw)


def test_sizes_past_a_c_int_are_refused(on_cpu):
    """Not the page size or the table of their low 32 bits (the expanded tensors hold no memory)."""
    ops = on_cpu
    table, mass, lens = torch.zeros((2, 5), dtype=torch.int32), torch.zeros((2, 1, 5)), torch.tensor([80, 3])
    for bs in (2 ** 32 + 16, 2 ** 31, 0, -16, 2 ** 32):
        with pytest.raises(RuntimeError, match="paged_evict: bs="):
            ops.paged_evict(table, mass, lens, 1, bs=bs)
    c = cache([20, 5], Hq=4, Hkv=2, D=64, bs=16)
    args = [c[k] for k in ("q", "k_pages", "v_pages", "table", "lens")]
    idx = torch.zeros(1, dtype=torch.int32).expand(2, 2, 2 ** 32 + 3)
    with pytest.raises(RuntimeError, match="kv_idx"):
        ops.paged_decode_attn(*args, scale=0.1, kv_num=torch.ones(2, 2, dtype=torch.int32), kv_idx=idx)


def test_penalties_that_fp32_does_not_hold_are_refused(on_cpu):
    """1e-50 and 1e50 are 0 and infinity to the kernel: a quotient by 0, a product of infinity and 0."""
    ops = on_cpu
    z, t = torch.zeros(2, 70), torch.zeros(2, 9, dtype=torch.int64)
    for name in ("repetition", "temperature", "presence", "frequency"):
        for x in (1e50, -1e50) + ((1e-50, 0.0, -1.0) if name in ("repetition", "temperature") else (float("nan"),)):
            with pytest.raises(ValueError, match="logit_penalties"):
                ops.logit_penalties(z, t, 3, **{name: x})
        with pytest.raises(Reached):
            ops.logit_penalties(z, t, 3, **{name: 2.0 ** -126})
        with pytest.raises(Reached):
            ops.logit_penalties(z, t, 3, **{name: 3.4e38})


def test_a_gradient_that_reaches_the_results_raises(on_cpu, monkeypatch):
    """Not a silent zero; without gradients, or with none asked for, nothing is recorded."""
    ops = on_cpu
    monkeypatch.setattr(ops, "_launch", lambda *a: None)
    monkeypatch.setattr(ops, "query", lambda *a: 16)
    c = cache([20, 5], Hq=4, Hkv=2, D=64, bs=16)
    rest = [c[k] for k in ("k_pages", "v_pages", "table", "lens")]
    q, mass = c["q"].clone().requires_grad_(), torch.zeros(2, 2, c["table"].shape[1])
    out, lse = ops.paged_decode_attn(q, *rest, scale=0.1, mass=mass)
    for y in (out, lse):
        with pytest.raises(RuntimeError, match="paged_decode_attn is not differentiable"):
            y.float().sum().backward()
    z, t = torch.zeros(2, 70, requires_grad=True), torch.zeros(2, 9, dtype=torch.int64)
    bias = torch.zeros(70, requires_grad=True)
    for got in (ops.logit_penalties(z, t, 3, bias=bias.detach()), ops.logit_penalties(z.detach(), t, 3, bias=bias)):
        assert got.shape == z.shape
        with pytest.raises(RuntimeError, match="logit_penalties is not differentiable"):
            got.sum().backward()
    with torch.no_grad():
        quiet = [*ops.paged_decode_attn(q, *rest, scale=0.1), ops.logit_penalties(z, t, 3, bias=bias)]
    quiet += [*ops.paged_decode_attn(q.detach(), *rest, scale=0.1), ops.logit_penalties(z.detach(), t, 3)]
    assert not any(y.requires_grad for y in quiet)
    assert ops.logit_penalties(z.detach(), t, 3, out=z.detach()).requires_grad is False
    with pytest.raises(RuntimeError, match="kv_num and kv_idx"):
        ops.paged_decode_attn(q, *rest, scale=0.1, kv_num=torch.ones(2, 2, dtype=torch.int32))


@pytest.mark.parametrize("name", ["repetition", "presence", "frequency", "temperature"])
def test_a_gradient_that_reaches_a_penaltys_rows_raises(on_cpu, monkeypatch, name):
    """Penalties of one number a row, asked for a gradient."""
    ops = on_cpu
    monkeypatch.setattr(ops, "_launch", lambda *a: None)
    z, t = torch.zeros(2, 70), torch.zeros(2, 9, dtype=torch.int64)
    x = torch.ones(2, requires_grad=True)
    with pytest.raises(RuntimeError, match="logit_penalties is not differentiable"):
        ops.logit_penalties(z, t, 3, **{name: x}).sum().backward()
    assert ops.logit_penalties(z, t, 3, **{name: x}, out=z).requires_grad is False
    assert ops.logit_penalties(z, t, 3, **{name: x.detach()}).requires_grad is False
