"""The paged cache on the GPU against the oracle in 64 bits: rows appended, the
attention of one new token a sequence, the pages that leave, and a run of them
together.  Bounds are derived in tests/paged_inputs.py (attn_bounds); written
rows, page tables and ids are equal bit for bit."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import paged as OP
from tests.paged_inputs import TYPES, assert_within, cache, check_attn, tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from scope_amd import ops

    return ops


# ---- attention --------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
def test_attn_types_and_sizes(ops, dtype, fp8, D, bs):
    """Ragged lengths from zero on, pages that end inside a tile, grouped heads."""
    print(f"paged attn {dtype} fp8={fp8} D={D} bs={bs}", flush=True)
    lens = [0, 1, 17, bs, bs + 1, 5 * bs - 1, 300]
    c = cache(lens, Hq=6, Hkv=2, D=D, bs=bs, dtype=dtype, fp8=fp8, seed=D + bs)
    mass = torch.rand((len(lens), 2, c["table"].shape[1]), generator=torch.Generator().manual_seed(1))
    out, lse = check_attn(ops, c, DEV, scale=0.12, mass=mass)
    assert torch.all(out[0] == 0) and torch.all(lse[0] == -math.inf)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (8, 8), (7, 1), (16, 1), (17, 1), (40, 2), (24, 8), (64, 4)])
def test_attn_head_groups(ops, Hq, Hkv):
    print(f"paged attn heads {Hq}/{Hkv}", flush=True)
    c = cache([33, 700], Hq=Hq, Hkv=Hkv, D=64, bs=32, seed=Hq)
    check_attn(ops, c, DEV, scale=0.12, mass=torch.zeros((2, Hkv, c["table"].shape[1])))


@pytest.mark.parametrize("G", [15, 16, 17, 33])
@pytest.mark.parametrize("fp8", [False, True])
def test_attn_wide_groups_of_wide_heads(ops, G, fp8):
    """D = 256 with a full group of sixteen columns and more: the largest share of LDS."""
    print(f"paged attn D=256 G={G} fp8={fp8}", flush=True)
    c = cache([900, 65], Hq=G, Hkv=1, D=256, bs=64, fp8=fp8, seed=G)
    check_attn(ops, c, DEV, scale=0.06, mass=torch.zeros((2, 1, c["table"].shape[1])))


def test_strides_of_dimensions_of_one(ops):
    """One sequence, one key head and one page as odd views: their strides are never taken."""
    c = cache([13], Hq=2, Hkv=1, D=64, bs=16, MP=1, seed=4)
    odd = lambda x: x.contiguous().as_strided(x.shape, (5,) + x.stride()[1:])  # noqa: E731

    def strided(d):
        d = dict(d, q=odd(d["q"]))
        page = int(d["table"][0, 0])
        for n in ("k_pages", "v_pages"):
            one = d[n][page:page + 1].contiguous()
            d[n] = one.as_strided(one.shape, (3, 7, 64, 1))
        return d

    d = strided({k: (x.to(DEV) if isinstance(x, torch.Tensor) else x) for k, x in c.items()})
    zero = torch.zeros((1, 1), dtype=torch.int32, device=DEV)
    out, lse = ops.paged_decode_attn(d["q"], d["k_pages"], d["v_pages"], zero, d["lens"], scale=0.12)
    want, wl = check_attn(ops, c, DEV, scale=0.12)
    assert torch.equal(out, want) and torch.equal(lse, wl)
    row = torch.randn((1, 1, 64), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    ops.paged_append(row.as_strided((1, 1, 64), (3, 5, 1)), row, d["k_pages"], d["v_pages"], zero, d["lens"])
    assert torch.equal(d["k_pages"][0, 0, 13], row[0, 0]) and torch.equal(d["v_pages"][0, 0, 13], row[0, 0])


@pytest.mark.parametrize("B,hi", [(1, 9000), (3, 5000), (70, 400), (200, 130)])
def test_attn_ragged_batches(ops, B, hi):
    """Long sequences beside short and empty ones: the split over the length and its join."""
    print(f"paged attn B={B} hi={hi}", flush=True)
    g = torch.Generator().manual_seed(B)
    lens = [hi] + [int(hi ** float(torch.rand(1, generator=g))) - 1 for _ in range(B - 1)]
    c = cache(lens, Hq=2, Hkv=1, D=128, bs=16, seed=B)
    check_attn(ops, c, DEV, scale=0.12, mass=torch.zeros((B, 1, c["table"].shape[1])))


@pytest.mark.parametrize("bs", [16, 128])
@pytest.mark.parametrize("first", [[0, 5, 400, 900, 127], [-3, 2 ** 30, 16, 512, 1]])
def test_attn_first_position(ops, bs, first):
    """Windows that start inside a page, at its edge, behind the last key, and before zero."""
    c = cache([600, 600, 401, 900, 128], Hq=4, Hkv=2, D=128, bs=bs, seed=bs)
    check_attn(ops, c, DEV, scale=0.12, first=torch.tensor(first, dtype=torch.int32),
               mass=torch.zeros((5, 2, c["table"].shape[1])))


@pytest.mark.parametrize("bs", [16, 32, 128])
def test_attn_absent_pages(ops, bs):
    """Table entries below zero and past the pool are blocks without a page; a sequence without any sees nothing."""
    c = cache([10 * bs - 3, 10 * bs, 7 * bs + 1], Hq=4, Hkv=2, D=64, bs=bs, seed=3)
    table = c["table"].clone()
    table[0, 1], table[0, 2], table[0, 9], table[1, 0], table[1, 5] = -1, -2 ** 31, -1, c["k_pages"].shape[0], 2 ** 31 - 1
    table[2] = -1
    out, lse = check_attn(ops, c, DEV, scale=0.12, table=table, mass=torch.zeros((3, 2, table.shape[1])))
    assert torch.all(out[2] == 0) and torch.all(lse[2] == -math.inf)


def test_attn_lengths_outside_the_table(ops):
    """A length past the table's positions is cut to them, a negative one is zero."""
    c = cache([64, 64, 64], Hq=2, Hkv=1, D=64, bs=16, MP=4, seed=5)
    c["lens"] = torch.tensor([65, 2 ** 31 - 1, -7], dtype=torch.int32)
    check_attn(ops, c, DEV, scale=0.12, mass=torch.zeros((3, 1, 4)))


@pytest.mark.parametrize("bs,maxkv", [(16, 5), (16, 64), (64, 9), (128, 9), (256, 3)])
def test_attn_lists(ops, bs, maxkv):
    """Per-head block lists: several lengths, none, entries outside the table and behind the last key."""
    print(f"paged attn lists bs={bs} maxkv={maxkv}", flush=True)
    lens = [bs * 70 - 5, bs * 12, 1]
    c = cache(lens, Hq=6, Hkv=3, D=128, bs=bs, seed=maxkv)
    MP = c["table"].shape[1]
    g = torch.Generator().manual_seed(maxkv)
    kv_idx = torch.stack([torch.stack([torch.randperm(MP, generator=g)[:maxkv] for _ in range(3)]) for _ in lens]).int()
    kv_num = torch.randint(0, maxkv + 1, (3, 3), generator=g).int()
    kv_num[0, 0], kv_num[0, 1], kv_num[1, 2], kv_num[1, 1] = maxkv, 0, maxkv + 9, -4
    kv_idx[2, :, 0], kv_num[2] = 0, 1
    kv_idx[1, 2, 1], kv_idx[1, 2, 3 % maxkv] = -1, MP
    check_attn(ops, c, DEV, scale=0.12, kv_num=kv_num, kv_idx=kv_idx, mass=torch.zeros((3, 3, MP)))
    check_attn(ops, c, DEV, scale=0.12, kv_num=kv_num, kv_idx=kv_idx, first=torch.tensor([bs * 3 + 1, 5, 0], dtype=torch.int32))


def test_attn_a_block_listed_twice_counts_twice(ops):
    c = cache([200], Hq=2, Hkv=1, D=64, bs=32, seed=2)
    kv_idx = torch.tensor([[[3, 0, 3, 6, 3]]], dtype=torch.int32)
    check_attn(ops, c, DEV, scale=0.12, kv_num=torch.tensor([[5]], dtype=torch.int32), kv_idx=kv_idx)


def test_no_sequences_and_no_rows(ops):
    """Nothing to append is nothing done; a batch of none is refused, lists or not."""
    c = cache([20], Hq=2, Hkv=1, D=64, bs=16)
    d = {k: x.to(DEV) for k, x in c.items() if isinstance(x, torch.Tensor)}
    before = d["k_pages"].clone()
    none = torch.empty((0, 1, 64), dtype=torch.bfloat16, device=DEV)
    ops.paged_append(none, none, d["k_pages"], d["v_pages"], d["table"], d["lens"], cu=torch.zeros(2, dtype=torch.int32, device=DEV))
    ops.paged_append(none, none, d["k_pages"], d["v_pages"], d["table"], d["lens"])
    assert torch.equal(d["k_pages"], before)
    i32 = dict(dtype=torch.int32, device=DEV)
    for kw in ({}, dict(kv_num=torch.empty((0, 1), **i32), kv_idx=torch.empty((0, 1, 3), **i32))):
        with pytest.raises(RuntimeError, match="bad sizes"):
            ops.paged_decode_attn(d["q"][:0], d["k_pages"], d["v_pages"], d["table"][:0], d["lens"][:0], scale=0.1, **kw)


def test_attn_equals_the_contiguous_decode_attention(ops):
    """One sequence whose pages lie in order, over the pointer mask's lists: the framework's contiguous call."""
    H, bs, T = 8, 128, 1152
    c = cache([T], Hq=H, Hkv=H, D=128, bs=bs, seed=8)
    kv_idx = torch.tensor([0, 2, 3, 7, 8], dtype=torch.int32).repeat(H, 1)
    kv_num = torch.tensor([5, 4, 3, 2, 1, 5, 5, 5], dtype=torch.int32)
    n = T // bs
    k, v = (x[c["table"][0, :n].long()].transpose(0, 1).reshape(H, T, 128).to(DEV) for x in (c["k_pages"], c["v_pages"]))
    want, wl = ops.decode_attn(c["q"][0].to(DEV), k, v, kv_num.to(DEV), kv_idx.to(DEV), torch.zeros(T, dtype=torch.int32, device=DEV),
                               T - 1, bs=bs, scale=0.12)
    out, lse = check_attn(ops, c, DEV, scale=0.12, kv_num=kv_num[None], kv_idx=kv_idx[None])
    # both round one result to bf16: half a step each of values below 1
    assert (out[0].float() - want.float()).abs().max() <= 2 * 2.0 ** -8
    assert (lse[0] - wl).abs().max() <= 2.0 ** -15


def test_attn_strides(ops):
    """Token-major pages, q from a projection's rows, pages among others' memory."""
    c = cache([200, 77], Hq=8, Hkv=2, D=64, bs=32, seed=9)

    def strided(d):
        d = dict(d)
        d["k_pages"] = d["k_pages"].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        big = torch.full((2 * d["v_pages"].shape[0], 3, 32, 128), math.nan, dtype=d["v_pages"].dtype, device=DEV)
        big[::2, 1:, :, 64:] = d["v_pages"]
        d["v_pages"] = big[::2, 1:, :, 64:]
        rows = torch.full((2, 24, 64), math.nan, dtype=d["q"].dtype, device=DEV)
        rows[:, 8:16] = d["q"]
        d["q"] = rows[:, 8:16]
        return d

    check_attn(ops, c, DEV, scale=0.12, strided=strided, mass=torch.zeros((2, 2, c["table"].shape[1])))


@pytest.mark.parametrize("bs", [16, 128])
@pytest.mark.parametrize("fp8", [False, True])
def test_attn_rows_behind_the_last_key_do_not_count(ops, bs, fp8):
    """NaN and infinities in rows that are masked: behind the length, before the first position, in pages of no block."""
    c = cache([bs + 3, 3 * bs - 1], Hq=4, Hkv=2, D=128, bs=bs, fp8=fp8, seed=11)
    first = torch.tensor([2, bs + 5], dtype=torch.int32)
    want = ops.paged_decode_attn(*(c[k].to(DEV) for k in ("q", "k_pages", "v_pages", "table", "lens")), scale=0.12,
                                 first=first.to(DEV), **{n: c[n].to(DEV) for n in ("k_scale", "v_scale") if fp8})
    bad = {k: (x.clone() if isinstance(x, torch.Tensor) else x) for k, x in c.items()}
    live = torch.zeros(c["k_pages"].shape[0], bs, dtype=torch.bool)
    for b, n in enumerate(c["lens"].tolist()):
        for j in range(int(first[b]), n):
            live[c["table"][b, j // bs], j % bs] = True
    for name, poison in (("k_pages", math.nan), ("v_pages", math.nan if fp8 else math.inf)):
        x = bad[name].float()
        x.transpose(1, 2)[~live] = poison
        bad[name] = x.to(bad[name].dtype)
    mass = torch.zeros((2, 2, c["table"].shape[1]))
    out, lse = check_attn(ops, bad, DEV, scale=0.12, first=first, mass=mass)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_attn_extreme_scores(ops):
    """Scores of several hundred (one key takes all), an infinite key, NaN among the seen keys."""
    c = cache([500], Hq=2, Hkv=2, D=128, bs=64, seed=13, amplitude=8.0)
    check_attn(ops, c, DEV, scale=0.12, mass=torch.zeros((1, 2, c["table"].shape[1])))
    check_attn(ops, c, DEV, scale=-0.12)
    check_attn(ops, c, DEV, scale=0.0)
    page = int(c["table"][0, 3])
    c["k_pages"][page, 0, 5, 7] = math.nan
    out, lse = ops.paged_decode_attn(*(c[k].to(DEV) for k in ("q", "k_pages", "v_pages", "table", "lens")), scale=0.12)
    assert bool(torch.isnan(out[0, 0].float()).all()) and bool(torch.isnan(lse[0, 0]))
    assert bool(torch.isfinite(out[0, 1].float()).all())


def test_attn_rising_scores(ops):
    """Keys whose scores rise all along the cache: the running maximum moves in every tile."""
    c = cache([4000], Hq=4, Hkv=1, D=64, bs=16, seed=15)
    q = c["q"].float()
    for i in range(250):
        c["k_pages"][int(c["table"][0, i]), 0] = (q[0, 0] * (0.02 * i)).to(torch.bfloat16)
    check_attn(ops, c, DEV, scale=0.12, mass=torch.zeros((1, 1, c["table"].shape[1])))


def test_attn_shared_pages(ops):
    """Two sequences with one prefix's pages."""
    c = cache([300, 300], Hq=2, Hkv=1, D=64, bs=32, seed=17)
    table = c["table"].clone()
    table[1, :5] = table[0, :5]
    check_attn(ops, c, DEV, scale=0.12, table=table)


def test_attn_offsets_past_32_bits(ops):
    """A pool whose pages lie more than 2^32 elements apart."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    bs, D, Hkv = 256, 128, 8
    P = (2 ** 32 // (bs * D * Hkv)) + 40
    pool = torch.empty((P, Hkv, bs, D), dtype=torch.bfloat16, device=DEV)
    c = cache([600, 1], Hq=8, Hkv=Hkv, D=D, bs=bs, seed=19)
    n = c["k_pages"].shape[0]
    at = torch.linspace(0, P - 1, n).long()
    pool[at.to(DEV)] = c["k_pages"].to(DEV)
    d = {k: x.to(DEV) for k, x in c.items() if isinstance(x, torch.Tensor)}
    table = torch.where(c["table"] >= 0, at[c["table"].clamp(min=0).long()], -1).int().to(DEV)
    out, lse = ops.paged_decode_attn(d["q"], pool, pool, table, d["lens"], scale=0.12)
    want, wl = ops.paged_decode_attn(d["q"], d["k_pages"], d["k_pages"], d["table"], d["lens"], scale=0.12)
    assert torch.equal(out, want) and torch.equal(lse, wl)
    # and rows written there
    rows = torch.randn((2, Hkv, D), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)
    ops.paged_append(rows, rows, pool, pool, table, d["lens"])
    for b in range(2):
        assert torch.equal(pool[table[b, int(c["lens"][b]) // bs].long(), :, int(c["lens"][b]) % bs], rows[b])


def test_attn_same_bits_every_time(ops):
    c = cache([5000, 30, 900], Hq=8, Hkv=2, D=128, bs=32, seed=21)
    d = {k: x.to(DEV) for k, x in c.items() if isinstance(x, torch.Tensor)}
    m1, m2 = (torch.zeros((3, 2, c["table"].shape[1]), device=DEV) for _ in range(2))
    a = ops.paged_decode_attn(*(d[k] for k in ("q", "k_pages", "v_pages", "table", "lens")), scale=0.12, mass=m1)
    b = ops.paged_decode_attn(*(d[k] for k in ("q", "k_pages", "v_pages", "table", "lens")), scale=0.12, mass=m2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(m1, m2)


# ---- append -------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,fp8", [("bf16", False), ("fp16", False), ("bf16", True), ("fp16", True)])
@pytest.mark.parametrize("D,bs,Hkv", [(64, 16, 1), (128, 128, 8), (256, 32, 3)])
def test_append(ops, dtype, fp8, D, bs, Hkv):
    """Ragged prompts, an empty one, rows of no sequence, rows past the table and of absent pages."""
    print(f"append {dtype} fp8={fp8} D={D} bs={bs}", flush=True)
    g = torch.Generator().manual_seed(D)
    held, cu = [0, 5, 2 * bs - 1, 3, 7 * bs - 3], [2, 40, 40, 41 + 2 * bs, 44 + 2 * bs, 60 + 2 * bs]
    MP, N = 7, cu[-1] + 9
    table, P = tables([MP * bs] * 5, bs, MP, seed=bs)
    table[3, 0], table[0, 1] = -1, P
    kv = (torch.randn((N, 2 * Hkv, D), generator=g) * 3).to(TYPES[dtype])
    k, v = kv[:, :Hkv], kv[:, Hkv:]
    ks = vs = None
    if fp8:
        ks, vs = 0.004 + 0.02 * torch.rand(Hkv, generator=g), 0.004 + 0.02 * torch.rand(Hkv, generator=g)
        kp, vp = ((torch.randn((P, Hkv, bs, D), generator=g) * 50).to(torch.float8_e4m3fn) for _ in range(2))
    else:
        kp, vp = (torch.randn((P, Hkv, bs, D), generator=g).to(TYPES[dtype]) for _ in range(2))
    held, cu = torch.tensor(held, dtype=torch.int32), torch.tensor(cu, dtype=torch.int32)
    dk, dv, kvd = kp.to(DEV), vp.to(DEV), kv.to(DEV)
    ops.paged_append(kvd[:, :Hkv], kvd[:, Hkv:], dk, dv, table.to(DEV), held.to(DEV), cu=cu.to(DEV),
                     k_scale=ks.to(DEV) if fp8 else None, v_scale=vs.to(DEV) if fp8 else None)
    for got, before, x, s in ((dk, kp, k, ks), (dv, vp, v, vs)):
        want = OP.append(x, before, table, held, cu, s)
        assert torch.equal(got.cpu().view(torch.uint8), want.view(torch.uint8))


def test_append_one_row_each(ops):
    """A decode step: fewer rows than sequences, int64 lengths, pages in token-major order."""
    B, Hkv, D, bs = 6, 2, 64, 16
    g = torch.Generator().manual_seed(3)
    held = torch.tensor([0, 15, 16, 31, 100, 5])
    table, P = tables([112] * B, bs, 7, seed=1)
    x = torch.randn((5, Hkv, D), generator=g).to(torch.bfloat16)
    kp = torch.randn((P, bs, Hkv, D), generator=g).to(torch.bfloat16).permute(0, 2, 1, 3)
    vp = torch.randn((P, Hkv, bs, D), generator=g).to(torch.bfloat16)
    dk, dv = kp.to(DEV), vp.to(DEV)
    ops.paged_append(x.to(DEV), (-x).to(DEV), dk, dv, table.to(DEV), held.to(DEV))
    cu = torch.arange(B + 1).clamp(max=5)
    assert torch.equal(dk.cpu(), OP.append(x, kp, table, held, cu)) and torch.equal(dv.cpu(), OP.append(-x, vp, table, held, cu))


def test_append_e4m3_rounding(ops):
    """Ties, values past the largest, infinities, NaN, zeros of both signs, values below the smallest: as torch rounds."""
    x = torch.tensor([0.0, -0.0, 448.0, 464.0, 465.0, 1e30, -1e30, math.inf, -math.inf, math.nan, 1.0625, 1.1875, 17.0, 19.0,
                      2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, 2.0 ** -11, -2.0 ** -10 * 1.01, 240.0, 255.0, 0.3])
    x = torch.cat([x, torch.randn(64 - len(x), generator=torch.Generator().manual_seed(0)) * 100]).to(torch.bfloat16)
    kp = torch.zeros((1, 1, 16, 64), dtype=torch.float8_e4m3fn, device=DEV)
    vp = torch.zeros_like(kp)
    s = torch.tensor([0.7], device=DEV)
    ops.paged_append(x.to(DEV).reshape(1, 1, 64), x.to(DEV).reshape(1, 1, 64), kp, vp, torch.zeros((1, 1), dtype=torch.int32, device=DEV),
                     torch.tensor([3], device=DEV), k_scale=s)
    want_k = (x.float() / 0.7).clamp(-448, 448).to(torch.float8_e4m3fn)
    want_v = x.float().clamp(-448, 448).to(torch.float8_e4m3fn)
    for got, want in ((kp, want_k), (vp, want_v)):
        got = got[0, 0, 3].cpu().float()
        nan = torch.isnan(want.float())
        assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], want.float()[~nan])
        assert torch.equal(torch.signbit(got[~nan]), torch.signbit(want.float()[~nan]))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_append_e4m3_of_every_value(ops, dtype):
    """All 65536 values of the type over scales of every kind, the ones that take a plain division among
    them, as torch divides, cuts and rounds."""
    t = TYPES[dtype]
    x = torch.arange(-2 ** 15, 2 ** 15).to(torch.int16).view(t).reshape(1024, 1, 64).to(DEV)
    table, zero = torch.arange(64, dtype=torch.int32, device=DEV)[None], torch.zeros(1, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 1024], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(0)
    scales = [1.0, 0.0, -1.0, math.inf, math.nan, 1e-30, 1e30, 2.0 ** -60, 2.0 ** 61, 2.0 ** -140, 2 - 2.0 ** -23, 0.1, 1 / 3, 448.0]
    scales += torch.exp(torch.randn(12, generator=g) * 4).tolist()
    kp, vp = (torch.zeros((64, 1, 16, 64), dtype=torch.float8_e4m3fn, device=DEV) for _ in range(2))
    for s in scales:
        s = torch.tensor([s], device=DEV)
        ops.paged_append(x, x, kp, vp, table, zero, cu=cu, k_scale=s)
        want = (x.float() / s).clamp(-448, 448).to(torch.float8_e4m3fn).reshape(64, 16, 64)
        got = kp[:, 0].view(torch.uint8)
        nan = torch.isnan(want.float())
        assert torch.equal(torch.isnan(kp[:, 0].float()), nan), f"scale {s.item()}"
        assert torch.equal(got[~nan], want.view(torch.uint8)[~nan]), f"scale {s.item()}"


# ---- eviction -------------------------------------------------------------------------
@pytest.mark.parametrize("B,Hkv,MP", [(1, 1, 1), (3, 8, 7), (5, 2, 64), (4, 3, 1027), (2, 8, 4099), (1, 1, 20000), (2, 1, 65536)])
@pytest.mark.parametrize("window,n_global", [(1, 0), (4, 2)])
def test_evict(ops, B, Hkv, MP, window, n_global):
    print(f"evict B={B} Hkv={Hkv} MP={MP}", flush=True)
    bs = 16
    g = torch.Generator().manual_seed(MP + window)
    lens = torch.randint(0, MP * bs + 40, (B,), generator=g)
    lens[0] = MP * bs
    table = torch.randint(-MP // 4, 4 * MP, (B, MP), generator=g).int()
    # equal sums among them, zeros of both signs, NaN and infinity
    mass = torch.randint(0, 5, (B, Hkv, MP), generator=g).float() * 0.25
    mass[:, 0, ::7] = -0.0
    mass[:, 0, 3::11] = torch.rand(mass[:, 0, 3::11].shape, generator=g)
    if MP > 8:
        mass[0, 0, 5], mass[0, 0, 6], mass[0, 0, 7] = math.nan, math.inf, -1.5
    for budget in (0, 1, MP // 3, MP // 2 + 1, MP, -5):
        want = OP.evict(table, mass, lens, torch.full((B,), budget), bs=bs, window=window, n_global=n_global)
        got = ops.paged_evict(table.to(DEV), mass.to(DEV), lens.to(DEV), budget, bs=bs, window=window, n_global=n_global)
        for name, x, y in zip(("table", "freed", "n_freed"), got, want):
            assert torch.equal(x.cpu(), y), f"{name} at budget {budget}"


def test_evict_in_place_and_by_budgets(ops):
    g = torch.Generator().manual_seed(1)
    table = torch.arange(4 * 90, dtype=torch.int32).reshape(4, 90)
    mass = torch.rand((4, 2, 90), generator=g)
    lens, budget = torch.tensor([90 * 32, 50 * 32 + 1, 3, 0]), torch.tensor([10, 40, 0, 5])
    want = OP.evict(table, mass, lens, budget, bs=32, window=2, n_global=1)
    d = table.to(DEV)
    out, freed, n = ops.paged_evict(d, mass.to(DEV), lens.to(DEV), budget.to(DEV), bs=32, window=2, n_global=1, out=d)
    assert out is d and torch.equal(d.cpu(), want[0]) and torch.equal(freed.cpu(), want[1]) and torch.equal(n.cpu(), want[2])


def test_integers_past_32_bits(ops):
    """int64 budgets, lengths, first positions and list entries that no int32 holds: as the number says."""
    none = 2 ** 63 - 1
    table = torch.arange(2 * 40, dtype=torch.int32, device=DEV).reshape(2, 40)
    out, _, n = ops.paged_evict(table, torch.rand((2, 1, 40), device=DEV), torch.tensor([2 ** 33, 640], device=DEV),
                                torch.tensor([none, 2 ** 32 + 30], device=DEV), bs=16)
    assert torch.equal(out, table) and n.tolist() == [0, 0]
    for kw in (dict(window=2 ** 32 + 1), dict(n_global=2 ** 32)):
        out, _, n = ops.paged_evict(table, torch.rand((2, 1, 40), device=DEV), torch.tensor([640, 640], device=DEV), 1, bs=16, **kw)
        assert torch.equal(out, table) and n.tolist() == [0, 0]
    c = {k: x.to(DEV) if torch.is_tensor(x) else x for k, x in cache([200, 90], Hq=2, Hkv=1, D=64, bs=32, seed=21).items()}
    args = [c[k] for k in ("q", "k_pages", "v_pages", "table")]
    want = ops.paged_decode_attn(*args, c["lens"], scale=0.1)
    for first, seen in ((2 ** 32, False), (-2 ** 32 - 1, True)):
        got, lse = ops.paged_decode_attn(*args, c["lens"], scale=0.1, first=torch.tensor([first, 0], device=DEV))
        assert torch.equal(got[1], want[0][1])
        assert torch.equal(got[0], want[0][0]) if seen else bool((got[0] == 0).all()) and bool((lse[0] == -math.inf).all())
    idx = torch.tensor([1, 2 ** 32, 0], device=DEV).repeat(2, 1, 1)
    got = ops.paged_decode_attn(*args, c["lens"], scale=0.1, kv_num=torch.full((2, 1), 2 ** 40, device=DEV), kv_idx=idx)
    ref = ops.paged_decode_attn(*args, c["lens"], scale=0.1, kv_num=torch.full((2, 1), 3, device=DEV),
                                kv_idx=torch.tensor([1, -1, 0], device=DEV).repeat(2, 1, 1))
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


# ---- together ---------------------------------------------------------------------------
@pytest.mark.parametrize("fp8", [False, True])
def test_prompts_steps_and_evictions_together(ops, fp8):
    """Prompts appended, then steps (append, attend with the mass, now and then evict), all
    against the oracle on the same state."""
    B, Hq, Hkv, D, bs, MP, P = 3, 4, 2, 64, 16, 12, 40
    g = torch.Generator().manual_seed(4)
    t = torch.float8_e4m3fn if fp8 else torch.bfloat16
    ks = torch.tensor([0.01, 0.02]) if fp8 else None
    sc = dict(k_scale=ks, v_scale=ks)
    scd = {n: (x.to(DEV) if x is not None else None) for n, x in sc.items()}
    kp = torch.zeros((P, Hkv, bs, D)).to(t)
    dk, dv = kp.to(DEV), kp.to(DEV)
    kp, vp = kp.clone(), kp.clone()
    table = torch.randperm(P, generator=g)[:B * MP].reshape(B, MP).int()
    dt = table.to(DEV)
    lens = torch.zeros(B, dtype=torch.int32)
    mass = torch.zeros((B, Hkv, MP))
    dm = mass.to(DEV)
    for step in range(12):
        n = [70, 1, 33] if step == 0 else [1, 1, 1]
        cu = torch.tensor([0, n[0], n[0] + n[1], sum(n)], dtype=torch.int32)
        k, v = (torch.randn((sum(n), Hkv, D), generator=g).to(torch.bfloat16) for _ in range(2))
        dl = lens.to(DEV)
        ops.paged_append(k.to(DEV), v.to(DEV), dk, dv, dt, dl, cu=None if step else cu.to(DEV), **scd)
        kp, vp = OP.append(k, kp, table, lens, cu, ks), OP.append(v, vp, table, lens, cu, ks)
        assert torch.equal(dk.cpu().view(torch.uint8), kp.view(torch.uint8)) and torch.equal(dv.cpu().view(torch.uint8), vp.view(torch.uint8))
        lens = lens + torch.tensor(n, dtype=torch.int32)
        q = torch.randn((B, Hq, D), generator=g).to(torch.bfloat16)
        c = dict(q=q, k_pages=kp, v_pages=vp, table=table, lens=lens, **sc)
        check_attn(ops, c, DEV, scale=0.12, mass=dm.cpu())
        ops.paged_decode_attn(q.to(DEV), dk, dv, dt, lens.to(DEV), scale=0.12, mass=dm, **scd)
        if step % 4 == 3:
            want = OP.evict(table, dm.cpu(), lens, torch.full((B,), 3), bs=bs, window=1, n_global=1)
            got = ops.paged_evict(dt, dm, lens.to(DEV), 3, bs=bs, window=1, n_global=1, out=dt)
            assert all(torch.equal(x.cpu(), y) for x, y in zip(got, want))
            table = want[0]


def test_captured_and_replayed(ops):
    """A step captured once and replayed while lengths, table and rows change in place, with eager calls between."""
    c = cache([500, 40], Hq=8, Hkv=2, D=128, bs=32, MP=20, seed=23)
    d = {k: x.to(DEV) for k, x in c.items() if isinstance(x, torch.Tensor)}
    table2, _ = tables([640, 640], 32, 20, seed=5, spare=0)
    P = 40
    dk, dv = (torch.zeros((P, 2, 32, 128), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    rows = torch.zeros((2, 2, 128), dtype=torch.bfloat16, device=DEV)
    table, lens = table2.to(DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    mass = torch.zeros((2, 2, 20), device=DEV)
    q = d["q"]

    def step(mass):
        ops.paged_append(rows, rows, dk, dv, table, lens)
        lens.add_(1)
        out, lse = ops.paged_decode_attn(q, dk, dv, table, lens, scale=0.12, mass=mass)
        return out, lse

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(mass.clone())
    torch.cuda.current_stream().wait_stream(side)
    lens.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step(mass)
    lens.zero_()
    g = torch.Generator().manual_seed(6)
    for i in range(70):
        if i % 9 == 4:
            lens.add_(64)  # a prompt's worth of rows is there already
        rows.copy_(torch.randn((2, 2, 128), generator=g).to(torch.bfloat16))
        before = mass.clone()
        graph.replay()
        want, wl = ops.paged_decode_attn(q, dk, dv, table, lens, scale=0.12, mass=before)
        assert torch.equal(out, want) and torch.equal(lse, wl) and torch.equal(mass, before), f"replay {i}"
        if i % 20 == 19:
            torch.cuda.synchronize()
            ops.paged_evict(table, mass, lens, 12, bs=32, window=2, out=table)


def test_two_streams_at_once(ops):
    """Calls on two streams share nothing but what they are given."""
    c = cache([3000, 100], Hq=8, Hkv=2, D=128, bs=64, seed=25)
    d = {k: x.to(DEV) for k, x in c.items() if isinstance(x, torch.Tensor)}
    args = [d[k] for k in ("q", "k_pages", "v_pages", "table", "lens")]
    want = ops.paged_decode_attn(*args, scale=0.12)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_decode_attn(*args, scale=0.12))
    torch.cuda.synchronize()
    for one in got[0] + got[1]:
        assert torch.equal(one[0], want[0]) and torch.equal(one[1], want[1])
