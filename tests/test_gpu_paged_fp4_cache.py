"""The 4-bit paged cache in use: PagedKVCache over a run of prompts, steps, evictions,
reads and sequences that end, against the oracle on rows kept aside; calls captured
into graphs, on other streams and from two threads."""
from __future__ import annotations

import threading

import pytest
import torch

from oracle import paged as OP
from tests.paged_fp4_inputs import E8M0, FP4, bounds4, cache4
from tests.paged_inputs import TYPES, assert_within
from tests.test_gpu_paged_captured import captured

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from scope_amd import ops

    return ops


@pytest.mark.parametrize("rows_t", [torch.bfloat16, torch.float16])
def test_cache_in_use(rows_t):
    from scope_amd import PagedKVCache

    B, Hq, Hkv, D, bs = 3, 4, 2, 64, 16
    g = torch.Generator().manual_seed(7)
    c = PagedKVCache(pages=24, sequences=B, max_len=160, kv_heads=Hkv, head_dim=D, page_size=bs, dtype=FP4)
    assert c.k_pages.shape == (24, Hkv, bs, D // 2) and c.v_scale.shape == (24, Hkv, bs, D // 32) and c.k_scale.dtype == E8M0
    held = [[] for _ in range(B)]  # every row ever appended, by sequence

    def append(rows):
        n = sum(rows) if rows is not None else B
        k, v = (torch.randn((n, Hkv, D), generator=g).to(rows_t) for _ in range(2))
        c.append(k.to(DEV), v.to(DEV), rows)
        at = 0
        for b, m in enumerate(rows or [1] * B):
            held[b] += [(k[at + i], v[at + i]) for i in range(m)]
            at += m

    def values(b, which):  # what the rows of sequence b stand for, zeros where their page is gone
        x = torch.stack([r[which] for r in held[b]])
        x = OP.e2m1_values(*OP.quantise(x)).to(rows_t)
        gone = c.table[b].cpu()[torch.arange(len(held[b])) // bs] < 0
        x[gone] = 0
        return x

    def check():
        q = torch.randn((B, Hq, D), generator=g).to(rows_t)
        before = c.mass.cpu()
        out, lse = c.attend(q.to(DEV), scale=0.12)
        assert [c.length(b) for b in range(B)] == [len(h) for h in held] == c.lens.tolist()
        # the oracle's pages hold the same rows in places of their own, where the cache still has a page
        table = c.table.cpu()
        pages = torch.full(table.shape, -1, dtype=torch.int32)
        pages[table >= 0] = torch.arange(int((table >= 0).sum()), dtype=torch.int32)
        kp, vp = (torch.zeros((max(1, int(pages.max()) + 1), Hkv, bs, D), dtype=rows_t) for _ in range(2))
        for b in range(B):
            if held[b]:
                cu = torch.tensor([0, len(held[b])])
                kp = OP.append(values(b, 0), kp, pages[b:b + 1], torch.zeros(1), cu)
                vp = OP.append(values(b, 1), vp, pages[b:b + 1], torch.zeros(1), cu)
        r = OP.decode_attn(q, kp, vp, pages, torch.tensor([len(h) for h in held]), scale=0.12)
        b_out, b_lse, b_w = bounds4(rows_t, D, r)
        assert_within("lse", lse, r["lse"], b_lse)
        assert_within("out", out, r["out"], b_out)
        want = before.double() + r["weights"]
        assert_within("mass", c.mass, want, b_w + 2.0 ** -24 * want.abs())
        # and the rows themselves
        got = c.read(dtype=rows_t)
        for x, which in zip(got, (0, 1)):
            parts = [values(b, which) for b in range(B) if held[b]]
            assert torch.equal(x.cpu(), torch.cat(parts) if parts else x.cpu()[:0])

    append([50, 0, 17])
    check()
    append([0, 33, 0])
    for step in range(12):
        append(None)
        check()
    k, v = c.read([5, 0, 20], [40, 3, 0], dtype=rows_t)
    assert torch.equal(k.cpu(), torch.cat((values(0, 0)[40:45], values(2, 0)[:20]))) and torch.equal(v.cpu(), torch.cat((values(0, 1)[40:45], values(2, 1)[:20])))
    freed = c.evict(2, window=1, n_global=1)
    assert freed == sum(max(0, -(-len(h) // bs) - 2) for h in held) and freed > 0
    for step in range(5):
        append(None)
        check()
    c.release(1)
    held[1] = []
    append([0, 40, 0])  # another takes its place, in pages that others left
    check()
    for rows, first in (([1, 0, 0], [len(held[0]), 0, 0]), ([0, 0, -1], None), ([1, 1], None), ([0, 0, 0], [0, -1, 0])):
        with pytest.raises(ValueError, match="PagedKVCache: rows"):
            c.read(rows, first)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
def test_rows_of_the_other_caches_are_read(dtype):
    """16-bit pages give the rows back bit for bit, e4m3 pages their rounded ones."""
    from scope_amd import PagedKVCache

    g = torch.Generator().manual_seed(3)
    fp8 = dtype == torch.float8_e4m3fn
    scale = torch.tensor([0.02, 0.01], device=DEV) if fp8 else None
    t = torch.bfloat16 if fp8 else dtype
    c = PagedKVCache(pages=12, sequences=2, max_len=100, kv_heads=2, head_dim=64, page_size=16, dtype=dtype, k_scale=scale, v_scale=scale)
    k, v = (torch.randn((90, 2, 64), generator=g).to(t).to(DEV) for _ in range(2))
    c.append(k, v, [60, 30])
    got = c.read()
    want = ((x.float() / scale[:, None]).clamp(-448, 448).to(dtype).float() * scale[:, None] if fp8 else x for x in (k, v))
    for x, y in zip(got, want):
        assert x.dtype == t and torch.equal(x, y.to(t))
    if not fp8:
        with pytest.raises(RuntimeError, match="pages of their type"):
            c.read(dtype=torch.float16 if dtype == torch.bfloat16 else torch.bfloat16)


def test_what_a_4_bit_cache_refuses(monkeypatch):
    from scope_amd import PagedKVCache

    kw = dict(pages=4, sequences=1, max_len=64, kv_heads=1, head_dim=64, page_size=16, dtype=FP4)
    with pytest.raises(ValueError, match="scales themselves"):
        PagedKVCache(**kw, k_scale=torch.ones(1, device=DEV))
    with pytest.raises(ValueError, match="multiple of 32"):
        PagedKVCache(**dict(kw, head_dim=72))
    c = PagedKVCache(**kw)
    x = torch.zeros((1, 1, 64), dtype=torch.bfloat16, device=DEV)
    c.append(x, x)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="on the host"):
            c.read()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_a_captured_step(ops, dtype):
    """One graph that writes a row a sequence, attends and reads the rows back: replayed while the inputs, lengths and
    the table change, with eager work between the replays; every replay as the eager calls on the same state."""
    B, Hq, Hkv, D, bs = 3, 8, 2, 128, 32
    g = torch.Generator().manual_seed(2)
    c = {k: x.to(DEV) for k, x in cache4([900, 70, 333], Hq=Hq, Hkv=Hkv, D=D, bs=bs, dtype=dtype, MP=40, seed=3).items()}
    t = TYPES[dtype]
    table = torch.arange(B * 40, dtype=torch.int32, device=DEV).reshape(B, 40)
    P = B * 40
    pool = {n: torch.randint(0, 256, (P, Hkv, bs, D // 2), generator=g, dtype=torch.uint8).to(DEV) for n in ("k", "v")}
    scales = {n: torch.randint(120, 128, (P, Hkv, bs, D // 32), generator=g, dtype=torch.uint8).to(DEV) for n in ("k", "v")}
    lens, held = torch.zeros(B, dtype=torch.int32, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)
    q, k, v = torch.zeros((B, Hq, D), dtype=t, device=DEV), torch.zeros((B, Hkv, D), dtype=t, device=DEV), torch.zeros((B, Hkv, D), dtype=t, device=DEV)
    mass = torch.zeros((B, Hkv, 40), device=DEV)

    def step(p, s, m):
        kw = dict(k_scale=s["k"].view(E8M0), v_scale=s["v"].view(E8M0))
        kp, vp = p["k"].view(FP4), p["v"].view(FP4)
        ops.paged_append(k, v, kp, vp, table, held, **kw)
        out, lse = ops.paged_decode_attn(q, kp, vp, table, lens, scale=0.12, mass=m, **kw)
        return out, lse, *ops.paged_read(kp, vp, table, lens, rows=B, first=held, dtype=t, **kw)

    graph, got = captured(lambda: step(pool, scales, mass))
    for i in range(5):
        held.copy_(torch.randint(0, 40 * bs - 1, (B,), generator=g))
        lens.copy_(held + 1)
        table.copy_(torch.randperm(P, generator=g).reshape(B, 40))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g))
        before = {n: x.clone() for n, x in pool.items()}, {n: x.clone() for n, x in scales.items()}, mass.clone()
        graph.replay()
        torch.cuda.synchronize()
        want = step(*before)
        assert all(torch.equal(x, y) for x, y in zip(got, want)), f"replay {i}"
        assert torch.equal(mass, before[2]) and all(torch.equal(pool[n], before[0][n]) and torch.equal(scales[n], before[1][n]) for n in pool)


def test_two_graphs_in_turn(ops):
    """Attention over all pages with weights, and over lists, each in a graph of its own, in turn."""
    d = {k: x.to(DEV) for k, x in cache4([3000, 70, 900], Hq=8, Hkv=2, D=128, bs=32, seed=3).items()}
    MP = d["table"].shape[1]
    g = torch.Generator().manual_seed(2)
    mass = torch.zeros((3, 2, MP), device=DEV)
    kv_idx = torch.stack([torch.randperm(MP, generator=g)[:7] for _ in range(6)]).reshape(3, 2, 7).int().to(DEV)
    kv_num = torch.tensor([[7, 3], [1, 0], [5, 7]], dtype=torch.int32, device=DEV)
    args, kw = [d[k] for k in ("q", "k_pages", "v_pages", "table", "lens")], dict(scale=0.12, k_scale=d["k_scale"], v_scale=d["v_scale"])
    ga, a = captured(lambda: ops.paged_decode_attn(*args, mass=mass, **kw))
    gb, b = captured(lambda: ops.paged_decode_attn(*args, kv_num=kv_num, kv_idx=kv_idx, **kw))
    for i in range(4):
        d["q"].copy_(torch.randn(d["q"].shape, generator=g))
        m = mass.clone()
        wa, wb = ops.paged_decode_attn(*args, mass=m, **kw), ops.paged_decode_attn(*args, kv_num=kv_num, kv_idx=kv_idx, **kw)
        (ga, gb)[i % 2].replay()
        (gb, ga)[i % 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((*a, *b), (*wa, *wb))) and torch.equal(mass, m), f"replay {i}"


def test_another_stream(ops):
    """Inputs made on one stream, used on another that waits for it."""
    c = cache4([700, 33], Hq=8, Hkv=2, D=64, bs=16, seed=5)
    d = {k: x.to(DEV) for k, x in c.items()}
    args, kw = [d[k] for k in ("q", "k_pages", "v_pages", "table", "lens")], dict(k_scale=d["k_scale"], v_scale=d["v_scale"])
    want = ops.paged_decode_attn(*args, scale=0.12, **kw) + ops.paged_read(*args[1:], rows=2, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.paged_decode_attn(*args, scale=0.12, **kw) + ops.paged_read(*args[1:], rows=2, **kw)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_two_threads(ops):
    """Calls of two threads on streams of their own, each on its own cache."""
    caches = [{k: x.to(DEV) for k, x in cache4([400, 77], Hq=4, Hkv=2, D=64, bs=16, seed=s).items()} for s in (1, 2)]

    def call(d):
        kw = dict(k_scale=d["k_scale"], v_scale=d["v_scale"])
        args = [d[k] for k in ("q", "k_pages", "v_pages", "table", "lens")]
        return ops.paged_decode_attn(*args, scale=0.12, **kw) + ops.paged_read(*args[1:], rows=2, first=d["lens"] - 1, **kw)

    want = [call(d) for d in caches]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got = call(caches[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(x, y) for x, y in zip(got, want[i])):
                    wrong.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not wrong
