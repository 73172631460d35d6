"""The paged cache in 4 bits on the GPU against the oracle: rows quantised as they are
written (codes and scales bit for bit), rows read back out of pages of every type
(equal), and the attention of one new token a sequence (bounds derived in
tests/paged_fp4_inputs.py)."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import paged as OP
from tests.paged_fp4_inputs import E8M0, FP4, bounds4, cache4, check4, pages
from tests.paged_inputs import TYPES, assert_within, cache, check_attn, tables
from tests.test_paged_fp4 import groups

pytestmark = pytest.mark.gpu
DEV = "cuda"
TENSORS = ("q", "k_pages", "v_pages", "table", "lens")


@pytest.fixture(scope="module")
def ops():
    from scope_amd import ops

    return ops


def on_gpu(c):
    return {k: (x.to(DEV) if isinstance(x, torch.Tensor) else x) for k, x in c.items()}


def raw(x):
    return x.view(torch.uint8).cpu()


def attend(ops, d, **kw):
    return ops.paged_decode_attn(*(d[k] for k in TENSORS), scale=0.12, k_scale=d["k_scale"], v_scale=d["v_scale"], **kw)


# ---- append -------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,bs,Hkv", [(64, 16, 1), (64, 64, 3), (128, 128, 8), (256, 32, 3)])
def test_append(ops, dtype, D, bs, Hkv):
    """Ragged prompts, an empty one, rows of no sequence, rows past the table and of absent pages; the rest stays."""
    print(f"append fp4 {dtype} D={D} bs={bs} Hkv={Hkv}", flush=True)
    g = torch.Generator().manual_seed(D)
    held, cu = [0, 5, 2 * bs - 1, 3, 7 * bs - 3], [2, 40, 40, 41 + 2 * bs, 44 + 2 * bs, 60 + 2 * bs]
    MP, N = 7, cu[-1] + 9
    table, P = tables([MP * bs] * 5, bs, MP, seed=bs)
    table[3, 0], table[0, 1] = -1, P
    kv = (torch.randn((N, 2 * Hkv, D), generator=g) * torch.exp(2 * torch.randn((N, 2 * Hkv, D), generator=g))).to(TYPES[dtype])
    k, v = kv[:, :Hkv], kv[:, Hkv:]
    (kp, ks), (vp, vs) = (pages(g, P, Hkv, bs, D) for _ in range(2))
    held, cu = torch.tensor(held, dtype=torch.int32), torch.tensor(cu, dtype=torch.int32)
    dk, dks, dv, dvs, kvd = (x.to(DEV) for x in (kp, ks, vp, vs, kv))
    ops.paged_append(kvd[:, :Hkv], kvd[:, Hkv:], dk, dv, table.to(DEV), held.to(DEV), cu=cu.to(DEV), k_scale=dks, v_scale=dvs)
    for got, gs, before, bscale, x in ((dk, dks, kp, ks, k), (dv, dvs, vp, vs, v)):
        want, ws = OP.append_e2m1(x, before, bscale, table, held, cu)
        assert torch.equal(raw(gs), raw(ws)) and torch.equal(raw(got), raw(want))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_append_rounds_as_the_definition(ops, dtype):
    """Ties, carries of the scale, the type's ends, zeros of both signs, infinities and NaN."""
    x = groups(dtype)
    x = torch.cat((x, x[:len(x) % 2]))  # (two groups a row)
    x = x.reshape(-1, 1, 64)
    N = x.shape[0]
    kp, vp = (torch.zeros((2, 1, 256, 32), dtype=torch.uint8, device=DEV).view(FP4) for _ in range(2))
    ks, vs = (torch.zeros((2, 1, 256, 2), dtype=torch.uint8, device=DEV).view(E8M0) for _ in range(2))
    ops.paged_append(x.to(DEV), (-x).to(DEV), kp, vp, torch.ones((1, 1), dtype=torch.int32, device=DEV), torch.tensor([0], device=DEV),
                     cu=torch.tensor([0, N], device=DEV), k_scale=ks, v_scale=vs)
    for got, s, y in ((kp, ks, x), (vp, vs, -x)):
        q, e = OP.quantise(y)
        assert torch.equal(raw(s)[1, 0, :N], e[:, 0]) and torch.equal(raw(got)[1, 0, :N], q[:, 0])
        assert not raw(got)[0].any() and not raw(got)[1, 0, N:].any() and not raw(s)[1, 0, N:].any()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_append_of_every_16_bit_value(ops, dtype):
    """Each value as the largest of a group and among others."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    x = bits.view(TYPES[dtype]).reshape(-1, 1, 1).expand(-1, 1, 128).clone()
    g = torch.Generator().manual_seed(3)
    x[:, :, 1:] = (x[:, :, :1].double() * torch.rand((65536, 1, 127), generator=g, dtype=torch.float64) * 0.999).to(TYPES[dtype])
    table = torch.arange(256, dtype=torch.int32, device=DEV)[None]
    kp, vp = (torch.zeros((256, 1, 256, 64), dtype=torch.uint8, device=DEV).view(FP4) for _ in range(2))
    ks, vs = (torch.zeros((256, 1, 256, 4), dtype=torch.uint8, device=DEV).view(E8M0) for _ in range(2))
    ops.paged_append(x.to(DEV), x.flip(-1).to(DEV), kp, vp, table, torch.tensor([0], device=DEV), cu=torch.tensor([0, 65536], device=DEV),
                     k_scale=ks, v_scale=vs)
    for got, s, y in ((kp, ks, x), (vp, vs, x.flip(-1))):
        q, e = OP.quantise(y)
        assert torch.equal(raw(s).reshape(e.shape), e) and torch.equal(raw(got).reshape(q.shape), q)


def test_append_one_row_each(ops):
    """A decode step: fewer rows than sequences, int64 lengths, token-major pages and scales of other strides."""
    B, Hkv, D, bs = 6, 2, 64, 16
    g = torch.Generator().manual_seed(3)
    held = torch.tensor([0, 15, 16, 31, 100, 5])
    table, P = tables([112] * B, bs, 7, seed=1)
    x = torch.randn((5, Hkv, D), generator=g).to(torch.bfloat16)
    kp, ks = pages(g, P, Hkv, bs, D)
    vp, vs = pages(g, P, Hkv, bs, D)
    dk = kp.view(torch.uint8).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3).to(DEV).view(FP4)
    dks = ks.view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).to(DEV).view(E8M0)
    dv, dvs = vp.to(DEV), vs.to(DEV)
    ops.paged_append(x.to(DEV), (-x).to(DEV), dk, dv, table.to(DEV), held.to(DEV), k_scale=dks, v_scale=dvs)
    cu = torch.arange(B + 1).clamp(max=5)
    for got, s, y, p0, s0 in ((dk, dks, x, kp, ks), (dv, dvs, -x, vp, vs)):
        want, ws = OP.append_e2m1(y, p0, s0, table, held, cu)
        assert torch.equal(raw(got), raw(want)) and torch.equal(raw(s), raw(ws))


# ---- read ---------------------------------------------------------------------------
KINDS = [("bf16", "16"), ("fp16", "16"), ("bf16", "fp8"), ("fp16", "fp8"), ("bf16", "fp4"), ("fp16", "fp4")]


def pool(kind, dtype, g, P, Hkv, bs, D):
    """(pages, scale, the numbers that they stand for in dtype)."""
    t = TYPES[dtype]
    if kind == "fp4":
        p, s = pages(g, P, Hkv, bs, D)
        return p, s, OP.e2m1_values(p, s).to(t)
    x = torch.randn((P, Hkv, bs, D), generator=g)
    if kind == "fp8":
        s = 0.004 + 0.02 * torch.rand(Hkv, generator=g)
        p = (x / s[:, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        return p, s, (p.float() * s[:, None, None]).to(t)
    return x.to(t), None, x.to(t)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("D,bs,Hkv", [(64, 16, 1), (64, 32, 3), (128, 128, 8), (256, 64, 2)])
def test_read(ops, dtype, kind, D, bs, Hkv):
    """Ragged ranges, an empty one, rows of no sequence, before zero, behind the length, past the table and of absent pages."""
    print(f"read {kind} as {dtype} D={D} bs={bs} Hkv={Hkv}", flush=True)
    g = torch.Generator().manual_seed(D + Hkv)
    MP = 5
    table, P = tables([MP * bs] * 5, bs, MP, seed=bs)
    table[1, 1], table[2, 0] = -1, P
    lens = torch.tensor([3 * bs + 1, 5 * bs, 2 * bs, 9 * bs, 0], dtype=torch.int32)
    first = torch.tensor([bs - 1, 0, -4, 4 * bs - 2, 0], dtype=torch.int32)
    cu = torch.tensor([1, 1 + bs, 40 + 3 * bs, 40 + 3 * bs, 80 + 4 * bs, 82 + 4 * bs], dtype=torch.int32)
    rows = int(cu[-1]) + 7
    (kp, ks, kx), (vp, vs, vx) = (pool(kind, dtype, g, P, Hkv, bs, D) for _ in range(2))
    dev = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    for f in (first, None):
        k, v = ops.paged_read(dev(kp), dev(vp), dev(table), dev(lens), rows=rows, cu=dev(cu), first=dev(f), k_scale=dev(ks),
                              v_scale=dev(vs), dtype=TYPES[dtype])
        for got, x in ((k, kx), (v, vx)):
            assert got.dtype == TYPES[dtype] and torch.equal(got.cpu(), OP.read(x, table, lens, rows, cu, f))
    # one row a sequence, by default in the pages' type or bfloat16
    k, v = ops.paged_read(dev(kp), dev(vp), dev(table), dev(lens), rows=4, first=dev(first.long()), k_scale=dev(ks), v_scale=dev(vs),
                          dtype=None if dtype == "bf16" or kind == "16" else TYPES[dtype])
    assert torch.equal(k.cpu(), OP.read(kx, table, lens, 4, None, first)) and torch.equal(v.cpu(), OP.read(vx, table, lens, 4, None, first))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_read_of_every_byte_and_scale(ops, dtype):
    """All codes under all scales, the ends of fp32 and NaN among them: rounded once to the rows' type."""
    codes = torch.arange(256, dtype=torch.uint8).reshape(1, 1, 8, 32).expand(256, 1, 8, 32)  # 8 rows of 64
    kp = torch.cat((codes, codes.flip(2)), 2).contiguous()
    ks = torch.arange(256, dtype=torch.uint8).reshape(256, 1, 1, 1).expand(256, 1, 16, 2).contiguous()
    table = torch.arange(256, dtype=torch.int32)[None]
    k, v = ops.paged_read(kp.to(DEV).view(FP4), kp.to(DEV).view(FP4), table.to(DEV), torch.tensor([4096], device=DEV), rows=4096,
                          cu=torch.tensor([0, 4096], device=DEV), k_scale=ks.to(DEV).view(E8M0), v_scale=ks.to(DEV).view(E8M0), dtype=TYPES[dtype])
    want = OP.e2m1_values(kp, ks).reshape(4096, 1, 64).to(TYPES[dtype])
    for x in (k, v):
        assert torch.equal(torch.isnan(x.cpu()), torch.isnan(want)) and torch.equal(x.cpu().nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_read_is_infinite_where_the_type_does_not_hold_the_value(ops, dtype):
    """All codes under all scales, infinities as such: from 2^128 on in bf16 (scales 253 and 254), past 65504 in fp16."""
    codes = torch.arange(16, dtype=torch.uint8).repeat_interleave(2).reshape(1, 1, 1, 32).expand(256, 1, 16, 32) * 17  # (both features)
    ks = torch.arange(256, dtype=torch.uint8).reshape(256, 1, 1, 1).expand(256, 1, 16, 2).contiguous()
    table = torch.arange(256, dtype=torch.int32, device=DEV)[None]
    p, s = codes.contiguous().to(DEV).view(FP4), ks.to(DEV).view(E8M0)
    got, _ = ops.paged_read(p, p, table, torch.tensor([4096], device=DEV), rows=4096, cu=torch.tensor([0, 4096], device=DEV), k_scale=s,
                            v_scale=s, dtype=TYPES[dtype])
    want = OP.e2m1_values(codes, ks).reshape(4096, 1, 64).to(TYPES[dtype])
    nan, got = torch.isnan(want), got.cpu()
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], want[~nan])
    assert bool(torch.isinf(got).any()) and bool(torch.isinf(got[:253 * 16]).any()) == (dtype == "fp16")


def test_read_from_one_number_on(ops):
    c = cache([40, 3, 25], Hq=2, Hkv=1, D=64, bs=16, seed=2)
    d = on_gpu(c)
    for first in (0, 2, 24, -5, 10 ** 12):
        k, _ = ops.paged_read(*(d[k] for k in TENSORS[1:]), rows=3, first=first)
        assert torch.equal(k.cpu(), OP.read(c["k_pages"], c["table"], c["lens"], 3, None, [first] * 3))


def test_rows_past_the_largest_grid_of_two_a_wavefront(ops):
    """2^27 + 3 rows (one row's memory, expanded) written, of which a few blocks have a page; and their ends read."""
    N, bs, held = 2 ** 27 + 3, 256, 5
    MP = -(-(N + held) // bs)
    print(f"append of {N} rows", flush=True)
    table = torch.full((1, MP), -1, dtype=torch.int32, device=DEV)
    blocks = [0, 1, MP // 3, MP - 2, MP - 1]
    table[0, torch.tensor(blocks, device=DEV)] = torch.arange(len(blocks), dtype=torch.int32, device=DEV)
    row = torch.randn((1, 1, 64), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    kp, vp = (torch.zeros((len(blocks) + 1, 1, bs, 32), dtype=torch.uint8, device=DEV).view(FP4) for _ in range(2))
    ks, vs = (torch.zeros((len(blocks) + 1, 1, bs, 2), dtype=torch.uint8, device=DEV).view(E8M0) for _ in range(2))
    ops.paged_append(row.to(DEV).expand(N, 1, 64), -row.to(DEV).expand(N, 1, 64), kp, vp, table, torch.tensor([held], device=DEV),
                     cu=torch.tensor([0, N], dtype=torch.int32, device=DEV), k_scale=ks, v_scale=vs)
    pos = torch.tensor(blocks)[:, None] * bs + torch.arange(bs)
    written = (pos >= held) & (pos < N + held)
    for got, s, x in ((kp, ks, row), (vp, vs, -row)):
        q, e = OP.quantise(x[0])
        for t, want in ((raw(got), q), (raw(s), e)):
            assert torch.equal(t[:-1, 0][written], want.expand(int(written.sum()), -1)) and not t[:-1, 0][~written].any() and not t[-1].any()
    lens = torch.tensor([N + held], device=DEV)
    k, v = ops.paged_read(kp, vp, table, lens, rows=bs, cu=torch.tensor([0, bs], device=DEV), first=N + held - bs + 3, k_scale=ks, v_scale=vs)
    want = OP.e2m1_values(*OP.quantise(row[0])).to(torch.bfloat16).to(DEV)
    assert torch.equal(k[:bs - 3, 0], want.expand(bs - 3, -1)) and torch.equal(v[:bs - 3, 0], -want.expand(bs - 3, -1)) and not k[bs - 3:].any()


def test_read_of_more_than_2_31_values(ops):
    """One page under every block of a long sequence: the last rows of outputs past 2^31 elements."""
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB of device memory")
    bs, Hkv, D, rows = 256, 8, 128, 2 ** 21 + 77
    c = on_gpu(cache4([bs], Hq=8, Hkv=Hkv, D=D, bs=bs, seed=4))
    table = c["table"][:, :1].expand(1, -(-rows // bs)).contiguous()
    kw = dict(k_scale=c["k_scale"], v_scale=c["v_scale"])
    k, v = ops.paged_read(c["k_pages"], c["v_pages"], table, torch.tensor([rows], device=DEV), rows=rows,
                          cu=torch.tensor([0, rows], device=DEV), **kw)
    wk, wv = ops.paged_read(c["k_pages"], c["v_pages"], table[:, :1], torch.tensor([bs], device=DEV), rows=bs,
                            cu=torch.tensor([0, bs], device=DEV), **kw)
    for got, want in ((k, wk), (v, wv)):
        assert torch.equal(got[-77:], want[:77]) and torch.equal(got[-77 - bs:-77], want) and torch.equal(got[:bs], want)


def test_read_without_rows(ops):
    c = on_gpu(cache4([20], Hq=2, Hkv=1, D=64, bs=16))
    for cu in (None, torch.zeros(2, dtype=torch.int32, device=DEV)):
        k, v = ops.paged_read(*(c[k] for k in TENSORS[1:]), rows=0, cu=cu, k_scale=c["k_scale"], v_scale=c["v_scale"])
        assert k.shape == v.shape == (0, 1, 64)


def test_what_is_written_is_read(ops):
    """The rows' own values where the grid holds them; a second writing changes nothing."""
    g = torch.Generator().manual_seed(5)
    x = torch.tensor(OP.E2M1 + [-f for f in OP.E2M1])[torch.randint(0, 16, (300, 2, 128), generator=g)]
    x[:, :, ::32] = 6.0
    x = (x.reshape(300, 2, 4, 32) * 2.0 ** torch.randint(-9, 9, (300, 2, 4, 1), generator=g)).reshape(300, 2, 128).to(torch.bfloat16).to(DEV)
    c = on_gpu(cache4([300], Hq=2, Hkv=2, D=128, bs=64, seed=6))
    cu, zero = torch.tensor([0, 300], device=DEV), torch.tensor([0], device=DEV)
    kw = dict(k_scale=c["k_scale"], v_scale=c["v_scale"])
    for _ in range(2):
        ops.paged_append(x, x.flip(0), c["k_pages"], c["v_pages"], c["table"], zero, cu=cu, **kw)
        k, v = ops.paged_read(*(c[k] for k in TENSORS[1:]), rows=300, cu=cu, **kw)
        assert torch.equal(k, x) and torch.equal(v, x.flip(0))


# ---- attention --------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
def test_attn_types_and_sizes(ops, dtype, D, bs):
    """Ragged lengths from zero on, pages that end inside a tile, grouped heads."""
    print(f"paged attn fp4 {dtype} D={D} bs={bs}", flush=True)
    lens = [0, 1, 17, bs, bs + 1, 5 * bs - 1, 300]
    c = cache4(lens, Hq=6, Hkv=2, D=D, bs=bs, dtype=dtype, seed=D + bs)
    mass = torch.rand((len(lens), 2, c["table"].shape[1]), generator=torch.Generator().manual_seed(1))
    out, lse = check4(ops, c, DEV, scale=0.12, mass=mass)
    assert torch.all(out[0] == 0) and torch.all(lse[0] == -math.inf)


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (8, 8), (7, 1), (16, 1), (17, 1), (40, 2), (24, 8), (64, 4)])
def test_attn_head_groups(ops, Hq, Hkv, D):
    print(f"paged attn fp4 heads {Hq}/{Hkv} D={D}", flush=True)
    c = cache4([33, 700], Hq=Hq, Hkv=Hkv, D=D, bs=32, seed=Hq)
    check4(ops, c, DEV, scale=0.12, mass=torch.zeros((2, Hkv, c["table"].shape[1])))


@pytest.mark.parametrize("B,hi", [(1, 9000), (3, 5000), (70, 400), (200, 130)])
def test_attn_ragged_batches(ops, B, hi):
    """Long sequences beside short and empty ones: the split over the length and its join."""
    print(f"paged attn fp4 B={B} hi={hi}", flush=True)
    g = torch.Generator().manual_seed(B)
    lens = [hi] + [int(hi ** float(torch.rand(1, generator=g))) - 1 for _ in range(B - 1)]
    c = cache4(lens, Hq=2, Hkv=1, D=128, bs=16, seed=B)
    check4(ops, c, DEV, scale=0.12, mass=torch.zeros((B, 1, c["table"].shape[1])))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("bs", [16, 128])
@pytest.mark.parametrize("first", [[0, 5, 400, 900, 127], [-3, 2 ** 30, 16, 512, 1]])
def test_attn_first_position(ops, dtype, bs, first):
    """Windows that start inside a page, at its edge, behind the last key, and before zero."""
    c = cache4([600, 600, 401, 900, 128], Hq=4, Hkv=2, D=128, bs=bs, dtype=dtype, seed=bs)
    check4(ops, c, DEV, scale=0.12, first=torch.tensor(first, dtype=torch.int32), mass=torch.zeros((5, 2, c["table"].shape[1])))


@pytest.mark.parametrize("bs", [16, 32, 128])
def test_attn_absent_pages(ops, bs):
    """Table entries below zero and past the pool are blocks without a page; a sequence without any sees nothing."""
    c = cache4([10 * bs - 3, 10 * bs, 7 * bs + 1], Hq=4, Hkv=2, D=64, bs=bs, seed=3)
    table = c["table"].clone()
    table[0, 1], table[0, 2], table[0, 9], table[1, 0], table[1, 5] = -1, -2 ** 31, -1, c["k_pages"].shape[0], 2 ** 31 - 1
    table[2] = -1
    out, lse = check4(ops, c, DEV, scale=0.12, table=table, mass=torch.zeros((3, 2, table.shape[1])))
    assert torch.all(out[2] == 0) and torch.all(lse[2] == -math.inf)


def test_attn_lengths_outside_the_table(ops):
    c = cache4([64, 64, 64], Hq=2, Hkv=1, D=64, bs=16, MP=4, seed=5)
    c["lens"] = torch.tensor([65, 2 ** 31 - 1, -7], dtype=torch.int32)
    check4(ops, c, DEV, scale=0.12, mass=torch.zeros((3, 1, 4)))


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64), ("bf16", 256)])
@pytest.mark.parametrize("bs,maxkv", [(16, 5), (16, 64), (64, 9), (128, 9), (256, 3)])
def test_attn_lists(ops, dtype, D, bs, maxkv):
    """Per-head block lists: several lengths, none, entries outside the table and behind the last key."""
    print(f"paged attn fp4 lists bs={bs} maxkv={maxkv} D={D}", flush=True)
    lens = [bs * 70 - 5, bs * 12, 1]
    c = cache4(lens, Hq=6, Hkv=3, D=D, bs=bs, dtype=dtype, seed=maxkv)
    MP = c["table"].shape[1]
    g = torch.Generator().manual_seed(maxkv)
    kv_idx = torch.stack([torch.stack([torch.randperm(MP, generator=g)[:maxkv] for _ in range(3)]) for _ in lens]).int()
    kv_num = torch.randint(0, maxkv + 1, (3, 3), generator=g).int()
    kv_num[0, 0], kv_num[0, 1], kv_num[1, 2], kv_num[1, 1] = maxkv, 0, maxkv + 9, -4
    kv_idx[2, :, 0], kv_num[2] = 0, 1
    kv_idx[1, 2, 1], kv_idx[1, 2, 3 % maxkv] = -1, MP
    check4(ops, c, DEV, scale=0.12, kv_num=kv_num, kv_idx=kv_idx, mass=torch.zeros((3, 3, MP)))
    check4(ops, c, DEV, scale=0.12, kv_num=kv_num, kv_idx=kv_idx, first=torch.tensor([bs * 3 + 1, 5, 0], dtype=torch.int32))


def test_attn_a_block_listed_twice_counts_twice(ops):
    c = cache4([200], Hq=2, Hkv=1, D=64, bs=32, seed=2)
    kv_idx = torch.tensor([[[3, 0, 3, 6, 3]]], dtype=torch.int32)
    check4(ops, c, DEV, scale=0.12, kv_num=torch.tensor([[5]], dtype=torch.int32), kv_idx=kv_idx)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_attn_strides(ops, D):
    """Token-major pages, pages among others' memory, scales of other strides, q from a projection's rows."""
    c = cache4([200, 77], Hq=8, Hkv=2, D=D, bs=32, seed=9)

    def strided(d):
        d = dict(d)
        d["k_pages"] = d["k_pages"].view(torch.uint8).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3).view(FP4)
        big = torch.full((2 * d["v_pages"].shape[0], 3, 32, D), 0x77, dtype=torch.uint8, device=DEV)
        big[::2, 1:, :, D // 2:] = d["v_pages"].view(torch.uint8)
        d["v_pages"] = big[::2, 1:, :, D // 2:].view(FP4)
        wide = torch.full((2 * d["v_pages"].shape[0], 5, 32, D // 32), 255, dtype=torch.uint8, device=DEV)
        wide[1::2, 1:4:2] = d["k_scale"].view(torch.uint8)
        d["k_scale"] = wide[1::2, 1:4:2].view(E8M0)
        d["v_scale"] = d["v_scale"].view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).view(E8M0)
        rows = torch.full((2, 24, D), math.nan, dtype=d["q"].dtype, device=DEV)
        rows[:, 8:16] = d["q"]
        d["q"] = rows[:, 8:16]
        return d

    check4(ops, c, DEV, scale=0.12, strided=strided, mass=torch.zeros((2, 2, c["table"].shape[1])))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,bs", [(64, 16), (64, 128), (128, 16), (128, 128), (256, 16), (256, 64)])
def test_attn_rows_behind_the_last_key_do_not_count(ops, dtype, D, bs):
    """Codes of the largest size under NaN scales in rows that are masked: behind the length, before the first position,
    in pages of no block; the same bits come out."""
    c = cache4([bs + 3, 3 * bs - 1], Hq=4, Hkv=2, D=D, bs=bs, dtype=dtype, seed=11)
    first = torch.tensor([2, bs + 5], dtype=torch.int32)
    want = attend(ops, on_gpu(c), first=first.to(DEV))
    bad = {k: (x.view(torch.uint8).clone() if k.endswith(("pages", "scale")) else x) for k, x in c.items()}
    live = torch.zeros(c["k_pages"].shape[0], bs, dtype=torch.bool)
    for b, n in enumerate(c["lens"].tolist()):
        for j in range(int(first[b]), n):
            live[c["table"][b, j // bs], j % bs] = True
    for name in ("k_pages", "v_pages", "k_scale", "v_scale"):
        bad[name].transpose(1, 2)[~live] = 255 if name.endswith("scale") else 0x77
        bad[name] = bad[name].view(c[name].dtype)
    mass = torch.zeros((2, 2, c["table"].shape[1]))
    out, lse = check4(ops, bad, DEV, scale=0.12, first=first, mass=mass)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_attn_nan_in_seen_rows(ops, D):
    """A group of K without a number: its head's queries have none; of V: those 32 features."""
    c = cache4([500], Hq=4, Hkv=2, D=D, bs=64, seed=13)
    page, G = int(c["table"][0, 3]), 32
    for name in ("k_scale", "v_scale"):
        bad = dict(c, **{name: c[name].view(torch.uint8).clone().view(E8M0)})
        bad[name].view(torch.uint8)[page, 0, 5, 1] = 255
        out, lse = attend(ops, on_gpu(bad))
        nan = torch.isnan(out[0].float())
        assert not nan[2:].any() and bool(torch.isfinite(lse[0, 2:]).all())
        if name == "k_scale":
            assert bool(nan[:2].all()) and bool(torch.isnan(lse[0, :2]).all())
        else:
            assert bool(nan[:2, G:2 * G].all()) and int(nan.sum()) == 2 * G and bool(torch.isfinite(lse).all())


@pytest.mark.parametrize("G,D", [(2, 64), (8, 128), (9, 64), (4, 256)])
@pytest.mark.parametrize("name", ["v_scale", "k_scale"])
def test_attn_of_the_largest_scales(ops, G, D, name):
    """One group of one seen row under scales up to NaN: no other feature (of K: no other key head) gets another bit; of
    V its own are right while 2^8 times the sum of the row's |v| is below 2^128, and not finite from 2^128 on."""
    c = cache4([300], Hq=2 * G, Hkv=2, D=D, bs=64, seed=23)
    page, group = int(c["table"][0, 3]), slice(32, 64)
    c[name.replace("scale", "pages")].view(torch.uint8)[page, 0, 5, 16:32] = 0x77  # (6 in every feature of the group)
    d = on_gpu(c)
    want, wl = attend(ops, d)
    apart = torch.ones(want.shape, dtype=torch.bool, device=DEV)
    apart[0, :G, group if name == "v_scale" else slice(None)] = False
    for byte in (200, 230, 240, 244, 246, 248, 250, 251, 252, 253, 254, 255):
        c[name].view(torch.uint8)[page, 0, 5, 1] = byte
        d[name] = c[name].to(DEV)
        out, lse = attend(ops, d)
        assert torch.equal(out[apart], want[apart]), byte
        if name == "k_scale":
            assert torch.equal(lse[0, G:], wl[0, G:]), byte
            continue
        assert torch.equal(lse, wl), byte
        if byte <= 244:  # (2^8 · 6 · 2^117 and little more)
            assert bool(torch.isfinite(out.float()).all()), byte
            r = OP.decode_attn(c["q"], OP.e2m1_values(c["k_pages"], c["k_scale"]), OP.e2m1_values(c["v_pages"], c["v_scale"]), c["table"],
                               c["lens"], scale=0.12)
            assert_within("out", out, r["out"], bounds4(c["q"].dtype, D, r)[0])
        elif byte > 252:
            assert not bool(torch.isfinite(out[0, :G, group].float()).any()), byte


@pytest.mark.parametrize("D", [64, 128, 256])
def test_attn_of_large_values_in_16_bits(ops, D):
    """bf16 pages whose values of V are up to 2^108: 2^8 times their sum over 700 rows is below 2^128."""
    c = cache([700, 33], Hq=4, Hkv=2, D=D, bs=32, seed=24)
    c["v_pages"] = c["v_pages"] * 2.0 ** 106
    seen = c["v_pages"].double().abs().amax() * 700 * 2 ** 8
    assert seen < 2.0 ** 128
    check_attn(ops, c, DEV, scale=0.12)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attn_extreme_scores(ops, dtype):
    """Scores of several hundred (one key takes all), none, of the other sign; keys whose scores rise all along the cache."""
    c = cache4([500], Hq=2, Hkv=2, D=128, bs=64, dtype=dtype, seed=13, amplitude=8.0)
    mass = torch.zeros((1, 2, c["table"].shape[1]))
    for scale in (0.12, -0.12, 0.0):
        check4(ops, c, DEV, scale=scale, mass=mass)
    c = cache4([4000], Hq=4, Hkv=1, D=64, bs=16, dtype=dtype, seed=15)
    kp, ks = c["k_pages"].view(torch.uint8), c["k_scale"].view(torch.uint8)
    for i in range(250):
        at = int(c["table"][0, i])
        kp[at, 0], ks[at, 0] = OP.quantise((c["q"][0, 0].float() * (0.02 * i)).to(TYPES[dtype]).expand(16, 64))
    check4(ops, c, DEV, scale=0.12, mass=torch.zeros((1, 1, c["table"].shape[1])))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attn_of_every_code_and_of_small_and_large_scales(ops, dtype):
    """Codes and scales drawn evenly, scales over sixty powers of two in one row; q of the type's small values."""
    g = torch.Generator().manual_seed(8)
    c = cache4([333, 60], Hq=6, Hkv=2, D=128, bs=32, dtype=dtype, seed=4)
    for n in ("k_pages", "v_pages"):
        c[n] = torch.randint(0, 256, c[n].shape, generator=g, dtype=torch.uint8).view(FP4)
    c["k_scale"] = torch.randint(127 - 50, 127 - 1, c["k_scale"].shape, generator=g, dtype=torch.uint8).view(E8M0)
    c["v_scale"] = torch.randint(127 - 50, 127 + 6, c["v_scale"].shape, generator=g, dtype=torch.uint8).view(E8M0)
    check4(ops, c, DEV, scale=0.12, mass=torch.zeros((2, 2, c["table"].shape[1])))
    c["q"][:, ::2] *= 2.0 ** -12 if dtype == "fp16" else 2.0 ** -60
    check4(ops, c, DEV, scale=0.12)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attn_of_scales_at_the_ends(ops, dtype):
    """Scales of V over 240 powers of two (what fp16 holds), of K down to the smallest ones."""
    g = torch.Generator().manual_seed(9)
    c = cache4([200, 61], Hq=6, Hkv=2, D=64, bs=32, dtype=dtype, seed=4)
    of = lambda x, n: torch.tensor(x, dtype=torch.uint8)[torch.randint(0, len(x), c[n].shape, generator=g)].view(E8M0)  # noqa: E731
    c["v_scale"] = of([8, 60, 127, 200, 245] if dtype == "bf16" else [100, 110, 127, 135], "v_scale")
    c["k_scale"] = of([0, 1, 2, 30, 100, 128], "k_scale")
    check4(ops, c, DEV, scale=0.12)


@pytest.mark.parametrize("B,Hq,Hkv", [(3000, 2, 1), (9, 300, 150)])
def test_attn_of_many_sequences_and_of_many_heads(ops, B, Hq, Hkv):
    """More sequences than are looked through at once, more columns than workgroups fit: as the attention over the
    same cache in 16 bits, each rounded once."""
    print(f"paged attn fp4 B={B} heads {Hq}/{Hkv}", flush=True)
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 70, (B,), generator=g).tolist()
    c = on_gpu(cache4(lens, Hq=Hq, Hkv=Hkv, D=64, bs=16, seed=B))
    out, lse = attend(ops, c)
    rows = sum(lens)
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0)
    k, v = ops.paged_read(*(c[k] for k in TENSORS[1:]), rows=rows, cu=cu, k_scale=c["k_scale"], v_scale=c["v_scale"])
    kp, vp = (torch.zeros((c["k_pages"].shape[0], Hkv, 16, 64), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    ops.paged_append(k, v, kp, vp, c["table"], torch.zeros(B, dtype=torch.int32, device=DEV), cu=cu)
    want, wl = ops.paged_decode_attn(c["q"], kp, vp, c["table"], c["lens"], scale=0.12)
    none = torch.tensor(lens, device=DEV) == 0
    assert bool((out[none] == 0).all()) and bool((lse[none] == -math.inf).all())
    # each result is rounded to bf16; before that a score, |scale|·Σ|q k| below 8, is off by 2^-14 at most, a probability
    # by 2^-13 of it and an output by that of Σp|v|, below 8 too
    assert bool(((out.float() - want.float()).abs() <= 2 * 2.0 ** -8 * want.float().abs() + 2 * 2.0 ** -10).all())
    assert (lse - wl)[~none].abs().max() <= 2 * 2.0 ** -13


def test_attn_is_that_over_the_values(ops):
    """The same cache widened to 16-bit pages by paged_read and paged_append: one result, each rounded once."""
    c = on_gpu(cache4([1100, 37], Hq=8, Hkv=2, D=128, bs=32, seed=21))
    out, lse = attend(ops, c)
    cu = torch.tensor([0, 1100, 1137], device=DEV)
    k, v = ops.paged_read(*(c[k] for k in TENSORS[1:]), rows=1137, cu=cu, k_scale=c["k_scale"], v_scale=c["v_scale"])
    kp, vp = (torch.zeros((c["k_pages"].shape[0], 2, 32, 128), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    ops.paged_append(k, v, kp, vp, c["table"], torch.zeros(2, dtype=torch.int32, device=DEV), cu=cu)
    want, wl = ops.paged_decode_attn(c["q"], kp, vp, c["table"], c["lens"], scale=0.12)
    assert bool(((out.float() - want.float()).abs() <= 2 * 2.0 ** -8 * want.float().abs() + 2.0 ** -16).all())
    assert (lse - wl).abs().max() <= 2.0 ** -15


@pytest.mark.parametrize("D,G", [(64, 3), (128, 12), (256, 16)])
def test_attn_of_an_evicted_cache(ops, D, G):
    """Most blocks without a page, long runs of them among those that have one: more than a wavefront looks up at once."""
    bs = 16
    c = cache4([9000, 20, 5000], Hq=G, Hkv=1, D=D, bs=bs, seed=18)
    table = c["table"].clone()
    g = torch.Generator().manual_seed(1)
    table[torch.rand(table.shape, generator=g) < 0.6] = -1
    table[0, 20:520] = -1
    check4(ops, c, DEV, scale=0.12, table=table, mass=torch.zeros((3, 1, table.shape[1])))


def test_attn_shared_pages(ops):
    c = cache4([300, 300], Hq=2, Hkv=1, D=64, bs=32, seed=17)
    table = c["table"].clone()
    table[1, :5] = table[0, :5]
    check4(ops, c, DEV, scale=0.12, table=table)


def test_attn_same_bits_every_time(ops):
    c = on_gpu(cache4([5000, 30, 900], Hq=8, Hkv=2, D=128, bs=32, seed=21))
    m1, m2 = (torch.zeros((3, 2, c["table"].shape[1]), device=DEV) for _ in range(2))
    a, b = attend(ops, c, mass=m1), attend(ops, c, mass=m2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(m1, m2)


def test_offsets_past_32_bits(ops):
    """A pool of more than 2^32 bytes: rows written, read and attended to at its far end."""
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB of device memory")
    bs, D, Hkv = 256, 128, 8
    P = 2 ** 32 // (bs * D // 2 * Hkv) + 40
    pool4 = torch.empty((P, Hkv, bs, D // 2), dtype=torch.uint8, device=DEV)
    # (the scales lie that far apart too)
    far = torch.empty((P, 16 * Hkv, bs, D // 32), dtype=torch.uint8, device=DEV)
    c = cache4([600, 1], Hq=8, Hkv=Hkv, D=D, bs=bs, seed=19)
    n = c["k_pages"].shape[0]
    at = torch.linspace(0, P - 1, n).long()
    d = on_gpu(c)
    pool4[at.to(DEV)] = d["k_pages"].view(torch.uint8)
    far[at.to(DEV), 15 * Hkv:] = d["k_scale"].view(torch.uint8)
    pool4, far = pool4.view(FP4), far[:, 15 * Hkv:].view(E8M0)
    assert far.stride(0) * (P - 1) > 2 ** 32
    table = torch.where(c["table"] >= 0, at[c["table"].clamp(min=0).long()], -1).int().to(DEV)
    out, lse = ops.paged_decode_attn(d["q"], pool4, pool4, table, d["lens"], scale=0.12, k_scale=far, v_scale=far)
    want, wl = ops.paged_decode_attn(d["q"], d["k_pages"], d["k_pages"], d["table"], d["lens"], scale=0.12, k_scale=d["k_scale"],
                                     v_scale=d["k_scale"])
    assert torch.equal(out, want) and torch.equal(lse, wl)
    cu = torch.tensor([0, 600, 601], device=DEV)
    k, v = ops.paged_read(pool4, pool4, table, d["lens"], rows=601, cu=cu, k_scale=far, v_scale=far)
    wk, _ = ops.paged_read(d["k_pages"], d["k_pages"], d["table"], d["lens"], rows=601, cu=cu, k_scale=d["k_scale"], v_scale=d["k_scale"])
    assert torch.equal(k, wk) and torch.equal(v, wk)
    rows = torch.randn((2, Hkv, D), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    ops.paged_append(rows.to(DEV), rows.to(DEV), pool4, pool4, table, d["lens"], k_scale=far, v_scale=far)
    q, s = OP.quantise(rows)
    for b in range(2):
        page, slot = int(table[b, int(c["lens"][b]) // bs]), int(c["lens"][b]) % bs
        assert torch.equal(raw(pool4[page, :, slot]), q[b]) and torch.equal(raw(far[page, :, slot]), s[b])
