"""The attention over 4-bit pages where a wavefront works on many tiles: the next one's loads
under way, maxima that move, runs of blocks without a page, more tiles than are looked up
at once.  Against the oracle within the bounds of tests/paged_fp4_inputs.py, and the same
bits in every copy of a key head."""
from __future__ import annotations

import pytest
import torch

from oracle import paged as OP
from tests.paged_fp4_inputs import bounds4
from tests.paged_fp4_tiles import DISTINCT, FORMS, KINDS, make, repeated
from tests.paged_inputs import assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 0.12


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D,G,bs,dtype", FORMS)
def test_many_tiles(kind, D, G, bs, dtype):
    from scope_amd import ops

    print(f"4-bit attention, many tiles: {kind} D={D} G={G} bs={bs} {dtype}", flush=True)
    c = make(kind, D, G, bs, dtype)
    d = {k: (x.to(DEV) if isinstance(x, torch.Tensor) else x) for k, x in c.items()}
    n = KINDS[kind]["Hkv"]
    d = repeated(d, n)
    kw = dict(scale=SCALE, first=d["first"], kv_num=d["kv_num"], kv_idx=d["kv_idx"], k_scale=d["k_scale"], v_scale=d["v_scale"])
    args = [d[k] for k in ("q", "k_pages", "v_pages", "table", "lens")]
    out, lse = ops.paged_decode_attn(*args, mass=d["mass"], **kw)
    plain = ops.paged_decode_attn(*args, **kw)
    assert torch.equal(out, plain[0]) and torch.equal(lse, plain[1])
    B = len(c["lens"])
    per_head = [x.reshape(B, n // DISTINCT, -1) for x in (out, lse, d["mass"])]
    for x in per_head:
        assert torch.equal(x, x[:, :1].expand_as(x))
    r = OP.decode_attn(c["q"], OP.e2m1_values(c["k_pages"], c["k_scale"]), OP.e2m1_values(c["v_pages"], c["v_scale"]), c["table"], c["lens"],
                       scale=SCALE, first=c["first"], kv_num=c["kv_num"], kv_idx=c["kv_idx"])
    b_out, b_lse, b_w = bounds4(c["q"].dtype, D, r)
    # a wavefront's outputs are one sum over its tiles: a tile adds two times three products of sixteen terms beside
    # zeros to it, each addition half a step of fp32 off at most (the sum of weights is one of T + 16 additions)
    b_out = b_out + 96 * KINDS[kind]["most"] * 2.0 ** -24 * r["spread"]
    got = [x[:, 0] for x in per_head]
    assert_within("lse", got[1].reshape(r["lse"].shape), r["lse"], b_lse)
    assert_within("out", got[0].reshape(r["out"].shape), r["out"], b_out)
    want = c["mass"].double() + r["weights"]
    assert_within("mass", got[2].reshape(want.shape), want, b_w + 2.0 ** -24 * want.abs())
