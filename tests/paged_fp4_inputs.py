"""Inputs of the 4-bit paged-cache tests, seeded and made on the CPU, and their bounds."""
from __future__ import annotations

import torch

from oracle import paged as OP
from tests.paged_inputs import TYPES, assert_within, tables

FP4, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def pages(g, P, Hkv, bs, D, dtype="bf16", amplitude=1.0):
    """(pages, scales) of quantised normal rows whose features differ in size."""
    x = torch.randn((P, Hkv, bs, D), generator=g) * amplitude * torch.exp(0.7 * torch.randn((Hkv, 1, D), generator=g))
    q, s = OP.quantise(x.to(TYPES[dtype]))
    return q.view(FP4), s.view(E8M0)


def cache4(lens, *, Hq, Hkv, D, bs, dtype="bf16", MP=None, seed=0, amplitude=1.0):
    """q, pages, scales, table and lens of a filled cache."""
    g = torch.Generator().manual_seed(seed)
    MP = MP or max(1, -(-max(max(lens), 1) // bs) + 1)
    table, P = tables(lens, bs, MP, seed)
    q = (torch.randn((len(lens), Hq, D), generator=g) * amplitude).to(TYPES[dtype])
    k, ks = pages(g, P, Hkv, bs, D, dtype, amplitude)
    v, vs = pages(g, P, Hkv, bs, D, dtype)
    return dict(q=q, k_pages=k, v_pages=v, table=table, lens=torch.tensor(lens, dtype=torch.int32), k_scale=ks, v_scale=vs)


def bounds4(dtype: torch.dtype, D: int, r: dict):
    """Bounds of (out, lse, weights), element by element, against fp64 (r: the oracle's).

    u: half a step of the 16-bit type, to which the result is rounded (u·|out|, and
    for fp16 half of its smallest step, 2^-25).  Products of q and K in parts that
    bf16 holds are exact in fp32 (a q in fp16 is two of them); a score is an fp32
    sum of at most 2 D products, one scaling and one difference, off by at most δ =
    ((2 D + 2)·2^-24 + 3·2^-23)·max scale·Σ|q_d k_d| (+ 2^-22 for the exponential's
    and logarithm's own error), so that p is off by 2δ relative.  A probability
    enters the product with V as three bf16 values, off by 2^-23 of it at most.
    Sums of positive terms are formed as a few hundred partial sums of at most a few
    hundred terms, half a step of fp32 each: 2^-16.  A probability below 2^-126 may
    be 0: a weight sums at most bs·G <= 2^16 of them, so it is off by up to 2^-110."""
    u = torch.finfo(dtype).eps / 2
    delta = ((2 * D + 2) * 2.0 ** -24 + 3 * 2.0 ** -23) * r["size"] + 2.0 ** -22
    rel = 2 * delta + 2.0 ** -16
    b_out = u * r["out"].abs() + (2.0 ** -23 + rel)[..., None] * r["spread"] + 2.0 ** -110 * r["total"]
    if dtype == torch.float16:
        b_out = b_out + 2.0 ** -25
    b_lse = delta + 2.0 ** -16 + 2.0 ** -23 * r["lse"].abs().nan_to_num(posinf=0.0)
    b_w = (rel.max() + 2.0 ** -23) * r["weights"] + 2.0 ** -110
    return b_out, b_lse, b_w


def check4(ops, c, dev, *, scale, first=None, kv_num=None, kv_idx=None, mass=None, table=None, strided=None):
    """One call against the oracle; returns (out, lse)."""
    table = c["table"] if table is None else table
    d = {k: x.to(dev) for k, x in c.items()}
    if strided:
        d = strided(d)
    kw = {k: x.to(dev) for k, x in dict(first=first, kv_num=kv_num, kv_idx=kv_idx).items() if x is not None}
    acc = None if mass is None else mass.to(dev)
    out, lse = ops.paged_decode_attn(d["q"], d["k_pages"], d["v_pages"], table.to(dev), d["lens"], scale=scale, mass=acc,
                                     k_scale=d["k_scale"], v_scale=d["v_scale"], **kw)
    r = OP.decode_attn(c["q"], OP.e2m1_values(c["k_pages"], c["k_scale"]), OP.e2m1_values(c["v_pages"], c["v_scale"]), table,
                       c["lens"], scale=scale, first=first, kv_num=kv_num, kv_idx=kv_idx)
    b_out, b_lse, b_w = bounds4(c["q"].dtype, c["q"].shape[-1], r)
    assert out.dtype == c["q"].dtype
    assert_within("lse", lse, r["lse"], b_lse)
    assert_within("out", out, r["out"], b_out)
    if mass is not None:
        want = mass.double() + r["weights"]
        assert_within("mass", acc, want, b_w + 2.0 ** -24 * want.abs())
    return out, lse
