"""Inputs of the paged-cache tests, seeded and made on the CPU."""
from __future__ import annotations

import torch

from oracle import paged as OP

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def tables(lens, bs, MP, seed, spare=3):
    """(table [B, MP], P): the pages each length needs, shuffled; the rest -1."""
    g = torch.Generator().manual_seed(seed)
    need = [min(-(-max(n, 0) // bs), MP) for n in lens]
    P = sum(need) + spare
    ids = torch.randperm(P, generator=g).tolist()
    table = torch.full((len(lens), MP), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(ids[:n], dtype=torch.int32)
        ids = ids[n:]
    return table, P


def cache(lens, *, Hq, Hkv, D, bs, dtype="bf16", fp8=False, MP=None, seed=0, amplitude=1.0):
    """q, pages, table, lens and scales of a filled cache."""
    g = torch.Generator().manual_seed(seed)
    MP = MP or max(1, -(-max(max(lens), 1) // bs) + 1)
    table, P = tables(lens, bs, MP, seed)
    t = TYPES[dtype]
    q = (torch.randn((len(lens), Hq, D), generator=g) * amplitude).to(t)
    k = torch.randn((P, Hkv, bs, D), generator=g) * amplitude
    v = torch.randn((P, Hkv, bs, D), generator=g)
    ks = vs = None
    if fp8:
        ks, vs = 0.004 + 0.02 * torch.rand(Hkv, generator=g), 0.004 + 0.02 * torch.rand(Hkv, generator=g)
        k, v = ((x / s[:, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn) for x, s in ((k, ks), (v, vs)))
    else:
        k, v = k.to(t), v.to(t)
    return dict(q=q, k_pages=k, v_pages=v, table=table, lens=torch.tensor(lens, dtype=torch.int32), k_scale=ks, v_scale=vs)


def attn_bounds(dtype: torch.dtype, D: int, r: dict):
    """Bounds of (out, lse, weights), element by element, against fp64 (r: the oracle's).

    u: half a step of the 16-bit type.  The result is rounded to it (u·|out|).
    The kernel takes each probability into its product with V as a sum of two
    such values (u²·Σp|v|; in fp16 one below the normal range is off by up to
    2^-25 relative to a maximum of at least 1: 2^-25·Σ|v|, and so may be the
    result).  Scores are fp32 sums of D exact products, one scaling and one
    difference: off by at most δ = ((D + 2)·2^-24 + 3·2^-23)·max scale·Σ|q_d k_d|
    (+ 2^-22 for the exponential's and logarithm's own error), so that p is off
    by 2δ relative.  Sums of positive terms are formed as a few hundred partial
    sums of at most a few hundred terms, half a step of fp32 each: 2^-16.  A
    probability below 2^-126 has no normal fp32 number and may be 0: a weight
    sums at most bs·G <= 2^16 of them, so it is off by up to 2^-110."""
    u = torch.finfo(dtype).eps / 2
    delta = ((D + 2) * 2.0 ** -24 + 3 * 2.0 ** -23) * r["size"] + 2.0 ** -22
    rel = 2 * delta + 2.0 ** -16
    low = 2.0 ** -25 * (1 + r["total"]) if dtype == torch.float16 else 0.0
    b_out = u * r["out"].abs() + (u * u + rel)[..., None] * r["spread"] + low
    b_lse = delta + 2.0 ** -16 + 2.0 ** -23 * r["lse"].abs().nan_to_num(posinf=0.0)
    b_w = (rel.max() + 2.0 ** -23) * r["weights"] + 2.0 ** -110
    return b_out, b_lse, b_w


def assert_within(name, got, ref, bound):
    got = got.double().cpu()
    assert got.shape == ref.shape, name
    finite = torch.isfinite(ref)
    assert torch.equal(got[~finite], ref[~finite]), f"{name}: infinite values differ"
    assert bool(torch.isfinite(got[finite]).all()), f"{name}: not finite"
    err = (got - ref).abs()[finite]
    over = err - bound.expand_as(ref)[finite]
    assert err.numel() == 0 or over.max() <= 0, f"{name}: {err.max().item():.3e} off, {over.max().item():.3e} over its bound"


def check_attn(ops, c, dev, *, scale, first=None, kv_num=None, kv_idx=None, mass=None, table=None, strided=None):
    """One call against the oracle; returns (out, lse)."""
    table = c["table"] if table is None else table
    d = {k: (x.to(dev) if isinstance(x, torch.Tensor) else x) for k, x in c.items()}
    if strided:
        d = strided(d)
    kw = dict(scale=scale, k_scale=d["k_scale"], v_scale=d["v_scale"],
              **{k: x.to(dev) for k, x in dict(first=first, kv_num=kv_num, kv_idx=kv_idx).items() if x is not None})
    acc = None if mass is None else mass.to(dev)
    out, lse = ops.paged_decode_attn(d["q"], d["k_pages"], d["v_pages"], table.to(dev), d["lens"], mass=acc, **kw)
    r = OP.decode_attn(c["q"], c["k_pages"], c["v_pages"], table, c["lens"], scale=scale, first=first,
                       kv_num=kv_num, kv_idx=kv_idx, k_scale=c["k_scale"], v_scale=c["v_scale"])
    b_out, b_lse, b_w = attn_bounds(c["q"].dtype, c["q"].shape[-1], r)
    assert out.dtype == c["q"].dtype
    assert_within("lse", lse, r["lse"], b_lse)
    assert_within("out", out, r["out"], b_out)
    if mass is not None:
        want = mass.double() + r["weights"]
        assert_within("mass", acc, want, b_w + 2.0 ** -24 * want.abs())
    return out, lse
