"""Penalties, biases and grammar bits on logits, on the GPU against the oracle in
64 bits.  The kernel takes five fp32 steps in a row and rounds the result once to
the logits' type: each step is off by half a step of fp32 of its own result (six
roundings of at most 2^-24 of the largest value on the way), the last by half a
step of the type."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import paged as OP

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from scope_amd import ops

    return ops


def check(ops, logits, tokens, lens, **kw):
    to = lambda x: x.to(DEV) if isinstance(x, torch.Tensor) else x  # noqa: E731
    got = ops.logit_penalties(logits.to(DEV), to(tokens), to(lens), **{k: to(v) for k, v in kw.items()})
    assert got.shape == logits.shape and got.dtype == logits.dtype
    z2 = logits if logits.dim() == 2 else logits[None]
    want = OP.penalties(z2, tokens, lens, **kw).reshape(logits.shape)
    got = got.double().cpu()
    open_ = torch.isfinite(want)
    assert torch.equal(got[~open_], want[~open_])
    # the largest value on the way: |z| r + f c + p + |bias|, over the temperature
    big = lambda x: float(x.abs().max()) if isinstance(x, torch.Tensor) else abs(float(x))  # noqa: E731
    T = tokens.shape[-1]
    r, t = kw.get("repetition", 1.0), kw.get("temperature", 1.0)
    small_t = float(t.min()) if isinstance(t, torch.Tensor) else t
    finite = logits.float()[torch.isfinite(logits.float())]
    way = (big(finite) * max(1.0, big(r), 1 / (float(r.min()) if isinstance(r, torch.Tensor) else r)) + big(kw.get("frequency", 0.0)) * T
           + big(kw.get("presence", 0.0)) + (big(kw["bias"]) if kw.get("bias") is not None else 0.0))
    bound = 6 * 2.0 ** -24 * way / min(1.0, small_t)
    if logits.dtype != torch.float32:
        bound = bound + torch.finfo(logits.dtype).eps / 2 * want[open_].abs() + 2.0 ** -25
    assert open_.sum() == 0 or ((got - want).abs()[open_] - bound).max() <= 0
    return got


def full(B, V, T, seed):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, T + 1, (B,), generator=g)
    lens[0] = T
    tokens = (torch.rand((B, T), generator=g) ** 3 * V).long()
    return dict(tokens=tokens, lens=lens, first=(lens * torch.rand(B, generator=g) * 0.5).long(),
                n_prompt=(lens * torch.rand(B, generator=g)).long(), repetition=1 + 0.5 * torch.rand(B, generator=g),
                presence=torch.randn(B, generator=g), frequency=torch.rand(B, generator=g),
                temperature=0.5 + torch.rand(B, generator=g), bias=torch.randn((B, V), generator=g),
                mask=torch.randint(-2 ** 31, 2 ** 31, (B, -(-V // 32)), generator=g).to(torch.int32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,V,T", [(1, 1, 1), (1, 33, 5), (2, 300, 40), (3, 4096, 100), (2, 4097, 2000), (2, 9001, 77), (3, 12295, 1500),
                                   (1, 8193, 16384), (9, 8200, 16385), (17, 130, 20001)])
def test_everything_at_once(ops, dtype, B, V, T):
    print(f"penalties {dtype} B={B} V={V} T={T}", flush=True)
    logits = (torch.randn((B, V), generator=torch.Generator().manual_seed(V)) * 5).to(dtype)
    check(ops, logits, **full(B, V, T, V + T))


@pytest.mark.parametrize("name,value", [("repetition", 1.3), ("repetition", 0.7), ("presence", 0.6), ("frequency", 0.25),
                                        ("temperature", 0.8), ("first", 3), ("n_prompt", 9)])
def test_one_at_a_time(ops, name, value):
    g = torch.Generator().manual_seed(2)
    logits, tokens = torch.randn((2, 500), generator=g), torch.randint(0, 500, (2, 60), generator=g)
    kw = {name: value}
    if name in ("first", "n_prompt"):
        kw["frequency"] = 0.5
    check(ops, logits, tokens, torch.tensor([60, 25]), **kw)


@pytest.mark.parametrize("T", [16384, 40000])
@pytest.mark.parametrize("token", [torch.int32, torch.int64])
def test_token_types_and_edges_of_the_history(ops, T, token):
    """Histories that start and end at every place of a 16-byte load, and of one to nine tokens."""
    g = torch.Generator().manual_seed(T)
    tokens = torch.randint(0, 300, (9, T), generator=g).to(token)
    logits = torch.randn((9, 300), generator=g)
    for first in (0, 1, 2, 3):
        for n in (1, 2, 3, 4, 5, 8, 9, 4096, 8193):
            lens = torch.full((9,), first + n) + torch.arange(9) % 2
            check(ops, logits, tokens, lens, first=first, n_prompt=first + n // 2, frequency=0.25, repetition=1.5, presence=0.5)


def test_nothing_asked_is_the_logits(ops):
    logits = torch.randn((3, 777), generator=torch.Generator().manual_seed(1)).to(DEV)
    tokens = torch.zeros((3, 4), dtype=torch.int64, device=DEV)
    assert torch.equal(ops.logit_penalties(logits, tokens, 4), logits)
    # and without any history
    none = torch.zeros((3, 0), dtype=torch.int64, device=DEV)
    assert torch.equal(ops.logit_penalties(logits, none, 0, repetition=2.0, frequency=1.0), logits)


def test_tokens_outside_the_vocabulary_and_lengths_outside_the_history(ops):
    g = torch.Generator().manual_seed(3)
    logits = torch.randn((4, 100), generator=g)
    tokens = torch.randint(0, 100, (4, 30), generator=g)
    tokens[:, ::5] = torch.tensor([-1, 100, 2 ** 40, -2 ** 62, 2 ** 31 + 5, 4096]).repeat(4, 1)
    check(ops, logits, tokens, torch.tensor([30, 2 ** 40, -3, 17]), repetition=1.5, frequency=0.5)
    check(ops, logits, tokens.clamp(-2 ** 31, 2 ** 31 - 1).int(), torch.tensor([30, 1000, -3, 17], dtype=torch.int32),
          repetition=1.5, frequency=0.5, first=torch.tensor([-5, 29, 0, 40]), n_prompt=torch.tensor([-1, 500, 0, 3]))


def test_nothing_counts_from_the_largest_position_on(ops):
    g = torch.Generator().manual_seed(4)
    logits, tokens = torch.randn((2, 100), generator=g).to(DEV), torch.randint(0, 100, (2, 30), generator=g).to(DEV)
    got = ops.logit_penalties(logits, tokens, 30, n_prompt=torch.tensor([2 ** 63 - 1, 2 ** 32], device=DEV), frequency=1.0, presence=1.0)
    assert torch.equal(got, logits)


def test_infinite_logits_and_rows_without_a_word(ops):
    """-inf and the type's lowest value stay, NaN stays, a mask of zeros leaves -inf everywhere."""
    logits = torch.tensor([[0.0, -math.inf, math.inf, math.nan, -0.0, 1.0, torch.finfo(torch.float32).min, 5.0]])
    tokens = torch.arange(8)[None]
    got = ops.logit_penalties(logits.to(DEV), tokens.to(DEV), 8, repetition=2.0, presence=0.5)
    want = torch.tensor([[-0.5, -math.inf, math.inf, math.nan, -0.5, 0.0, -math.inf, 2.0]])
    assert torch.equal(got.cpu().nan_to_num(nan=7.0, posinf=math.inf, neginf=-math.inf),
                       want.nan_to_num(nan=7.0, posinf=math.inf, neginf=-math.inf))
    got = ops.logit_penalties(logits.to(DEV), tokens.to(DEV), 8, mask=torch.zeros(1, dtype=torch.int32, device=DEV))
    assert bool((got == -math.inf).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_strides_alignment_and_in_place(ops, dtype, off):
    """Rows inside wider ones at odd offsets (the decoder's padded logits), shared histories, in place."""
    g = torch.Generator().manual_seed(4)
    wide = torch.randn((3, 1300), generator=g).to(dtype)
    tokens = torch.randint(0, 1201, (64,), generator=g)
    bias, mask = torch.randn(1201, generator=g), torch.randint(-2 ** 31, 2 ** 31, (38,), generator=g).int()
    view = lambda w: w[:, off:off + 1201]  # noqa: E731
    kw = dict(repetition=1.4, presence=0.3, bias=bias, mask=mask)
    want = check(ops, view(wide).contiguous(), tokens, torch.tensor([64, 10, 0]), **kw)
    d = wide.to(DEV)
    kwd = {k: (x.to(DEV) if isinstance(x, torch.Tensor) else x) for k, x in kw.items()}
    lens = torch.tensor([64, 10, 0], device=DEV)
    got = ops.logit_penalties(view(d), tokens.to(DEV), lens, **kwd)
    assert torch.equal(got.double().cpu(), want)
    ret = ops.logit_penalties(view(d), tokens.to(DEV), lens, out=view(d), **kwd)
    assert ret.data_ptr() == view(d).data_ptr() and torch.equal(view(d).double().cpu(), want)
    assert torch.equal(d[:, :off].cpu(), wide[:, :off]) and torch.equal(d[:, off + 1201:].cpu(), wide[:, off + 1201:])
    # bias rows inside wider ones
    wb = torch.zeros((3, 1300), device=DEV)
    view(wb).copy_(bias.to(DEV).expand(3, 1201))
    got = ops.logit_penalties(view(wide.to(DEV)), tokens.to(DEV), lens, **{**kwd, "bias": view(wb)})
    assert torch.equal(got.double().cpu(), want)


def test_long_history_of_one_word(ops):
    """Counts in the ten thousands, all on one counter; two rows share a history."""
    logits = torch.randn((2, 50), generator=torch.Generator().manual_seed(5))
    tokens = torch.full((70001,), 7)
    tokens[::1000] = 8
    check(ops, logits, tokens, torch.tensor([70001, 999]), frequency=0.001, repetition=1.1)


def test_captured_and_replayed(ops):
    V = 5000
    g = torch.Generator().manual_seed(6)
    logits = torch.randn(V, generator=g).to(DEV)
    tokens, t = torch.zeros(300, dtype=torch.int64, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    ops.logit_penalties(logits, tokens, t, repetition=1.2, frequency=0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.logit_penalties(logits, tokens, t, repetition=1.2, frequency=0.1)
    for i in range(0, 300, 13):
        tokens[i:i + 13] = torch.randint(0, V, (min(13, 300 - i),), generator=g).to(DEV)
        logits.copy_(torch.randn(V, generator=g))
        t.fill_(min(i + 13, 300))
        graph.replay()
        assert torch.equal(out, ops.logit_penalties(logits, tokens, min(i + 13, 300), repetition=1.2, frequency=0.1)), f"replay {i}"
