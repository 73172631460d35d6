"""Paged calls captured into graphs and replayed, among eager calls and in turn with
another graph: every replay against the eager call on the same state."""
from __future__ import annotations

import threading

import pytest
import torch

from tests.paged_inputs import cache, tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from scope_amd import ops

    return ops


def captured(call):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    return graph, out


def test_evictions(ops):
    """Weights, lengths and the table change between replays; the budget is a number."""
    g = torch.Generator().manual_seed(1)
    B, Hkv, MP, bs = 5, 3, 1300, 16
    table, mass = torch.arange(B * MP, dtype=torch.int32, device=DEV).reshape(B, MP), torch.zeros((B, Hkv, MP), device=DEV)
    lens, out = torch.zeros(B, dtype=torch.int32, device=DEV), torch.empty((B, MP), dtype=torch.int32, device=DEV)
    graph, got = captured(lambda: ops.paged_evict(table, mass, lens, 300, bs=bs, window=3, n_global=1, out=out))
    for i in range(6):
        mass.copy_(torch.randint(0, 40, (B, Hkv, MP), generator=g).float())
        lens.copy_(torch.randint(0, MP * bs + 9, (B,), generator=g))
        table.copy_(torch.randint(-MP, 4 * MP, (B, MP), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        want = ops.paged_evict(table, mass, lens, 300, bs=bs, window=3, n_global=1)
        assert all(torch.equal(x, y) for x, y in zip(got, want)), f"replay {i}"


@pytest.mark.parametrize("dtype,fp8", [("fp16", False), ("bf16", True)])
def test_two_graphs_in_turn(ops, dtype, fp8):
    """Attention over all pages with weights, and over lists, each in a graph of its own."""
    c = cache([3000, 70, 900], Hq=8, Hkv=2, D=128, bs=32, dtype=dtype, fp8=fp8, seed=3)
    d = {k: (x.to(DEV) if isinstance(x, torch.Tensor) else x) for k, x in c.items()}
    args, kw = [d[k] for k in ("q", "k_pages", "v_pages", "table", "lens")], dict(scale=0.12, k_scale=d["k_scale"], v_scale=d["v_scale"])
    MP = c["table"].shape[1]
    g = torch.Generator().manual_seed(2)
    mass = torch.zeros((3, 2, MP), device=DEV)
    kv_idx = torch.stack([torch.randperm(MP, generator=g)[:40] for _ in range(6)]).reshape(3, 2, 40).int().to(DEV)
    kv_num = torch.tensor([[40, 3], [40, 40], [17, 0]], dtype=torch.int32, device=DEV)
    first = torch.zeros(3, dtype=torch.int32, device=DEV)
    full, a = captured(lambda: ops.paged_decode_attn(*args, mass=mass, first=first, **kw))
    lists, b = captured(lambda: ops.paged_decode_attn(*args, kv_num=kv_num, kv_idx=kv_idx, **kw))
    for i in range(8):
        d["q"].copy_(torch.randn(d["q"].shape, generator=g).to(d["q"].dtype))
        d["lens"].copy_(torch.randint(0, 3100, (3,), generator=g))
        first.copy_(torch.randint(0, 200, (3,), generator=g))
        before = mass.clone()
        for graph in ((full, lists), (lists, full))[i % 2]:
            graph.replay()
        wa = ops.paged_decode_attn(*args, mass=before, first=first, **kw)
        wb = ops.paged_decode_attn(*args, kv_num=kv_num, kv_idx=kv_idx, **kw)
        for got, want in ((a, wa), (b, wb)):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), f"replay {i}"
        assert torch.equal(mass, before), f"replay {i}"


def test_ragged_appends(ops):
    B, Hkv, D, bs, MP, N = 4, 2, 64, 16, 12, 90
    g = torch.Generator().manual_seed(4)
    table, P = tables([MP * bs] * B, bs, MP, seed=4)
    rows = torch.zeros((N, 2 * Hkv, D), dtype=torch.float16, device=DEV)
    cu, lens, table = torch.zeros(B + 1, dtype=torch.int32, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV), table.to(DEV)
    scale = torch.tensor([0.01, 0.02], device=DEV)
    pages = [torch.zeros((P, Hkv, bs, D), device=DEV).to(torch.float8_e4m3fn) for _ in range(4)]

    def call(kp, vp):
        ops.paged_append(rows[:, :Hkv], rows[:, Hkv:], kp, vp, table, lens, cu=cu, k_scale=scale, v_scale=scale)

    graph, _ = captured(lambda: call(*pages[:2]))
    for p in pages:
        p.view(torch.uint8).zero_()
    for i in range(6):
        rows.copy_(torch.randn(rows.shape, generator=g))
        cu[1:].copy_(torch.randint(0, N + 1, (B,), generator=g).sort().values)
        lens.copy_(torch.randint(0, MP * bs, (B,), generator=g))
        graph.replay()
        call(*pages[2:])
        for x, y in zip(pages[:2], pages[2:]):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), f"replay {i}"


def test_two_threads_at_once(ops):
    """Two threads, each on a stream of its own, over the same pages."""
    c = cache([2000, 500], Hq=8, Hkv=2, D=64, bs=64, dtype="fp16", seed=5)
    d = {k: x.to(DEV) for k, x in c.items() if isinstance(x, torch.Tensor)}
    args = [d[k] for k in ("q", "k_pages", "v_pages", "table", "lens")]
    want = ops.paged_decode_attn(*args, scale=0.12)
    logits, tokens = torch.randn((2, 5000), device=DEV), torch.randint(0, 5000, (2, 900), device=DEV)
    wz = ops.logit_penalties(logits, tokens, 700, repetition=1.3, frequency=0.2)
    torch.cuda.synchronize()
    got, failed = [], []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    got.append((*ops.paged_decode_attn(*args, scale=0.12), ops.logit_penalties(logits, tokens, 700, repetition=1.3, frequency=0.2)))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for out, lse, z in got:
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and torch.equal(z, wz)
