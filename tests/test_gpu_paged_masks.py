"""The paged attention's masks, splits and running maxima in both 16-bit types and
e4m3 pages, on the GPU against the oracle in 64 bits.

The bound is tests/paged_inputs.py's but for what a probability loses on its way
into the product with V: 2^-23 of it in bf16 and 2^-21 in fp16, where all keys of
a row together lose 2^-34 of the largest |v| more (tests/test_gpu_paged_weights.py
derives it) and the result's own smallest half step is 2^-25."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import paged as OP
from tests.paged_inputs import assert_within, attn_bounds, cache

pytestmark = pytest.mark.gpu
DEV = "cuda"
KINDS = [("bf16", False), ("fp16", False), ("bf16", True), ("fp16", True)]


@pytest.fixture(scope="module")
def ops():
    from scope_amd import ops

    return ops


def check(ops, c, *, scale, mass=True, **kw):
    dev = lambda x: x.to(DEV) if isinstance(x, torch.Tensor) else x  # noqa: E731
    B, Hq, D = c["q"].shape
    acc = torch.zeros((B, c["k_pages"].shape[1], c["table"].shape[1]), device=DEV) if mass else None
    out, lse = ops.paged_decode_attn(*(dev(c[k]) for k in ("q", "k_pages", "v_pages", "table", "lens")), scale=scale, mass=acc,
                                     k_scale=dev(c["k_scale"]), v_scale=dev(c["v_scale"]), **{k: dev(x) for k, x in kw.items()})
    r = OP.decode_attn(c["q"], c["k_pages"], c["v_pages"], c["table"], c["lens"], scale=scale, k_scale=c["k_scale"], v_scale=c["v_scale"],
                       **kw)
    t = c["q"].dtype
    _, b_lse, b_w = attn_bounds(t, D, r)
    delta = ((D + 2) * 2.0 ** -24 + 3 * 2.0 ** -23) * r["size"] + 2.0 ** -22
    rel = 2 * delta + 2.0 ** -16 + (2.0 ** -21 if t == torch.float16 else 2.0 ** -23)
    b_out = torch.finfo(t).eps / 2 * r["out"].abs() + rel[..., None] * r["spread"]
    if t == torch.float16:
        b_out = b_out + 2.0 ** -25 + 2.0 ** -34 * OP.values(c["v_pages"], c["v_scale"]).abs().nan_to_num(posinf=0.0).max()
    assert_within("lse", lse, r["lse"], b_lse)
    assert_within("out", out, r["out"], b_out)
    if mass:
        assert_within("mass", acc, r["weights"], b_w + 2.0 ** -24 * r["weights"])
    return out, lse


@pytest.mark.parametrize("dtype,fp8", KINDS)
@pytest.mark.parametrize("B,hi,bs", [(1, 9000, 16), (3, 5000, 128), (70, 400, 16)])
def test_ragged_batches(ops, dtype, fp8, B, hi, bs):
    print(f"masks ragged {dtype} fp8={fp8} B={B} hi={hi} bs={bs}", flush=True)
    g = torch.Generator().manual_seed(B)
    lens = [hi] + [int(hi ** float(torch.rand(1, generator=g))) - 1 for _ in range(B - 1)]
    check(ops, cache(lens, Hq=2, Hkv=1, D=128, bs=bs, dtype=dtype, fp8=fp8, seed=B), scale=0.12)


@pytest.mark.parametrize("dtype,fp8", KINDS)
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("bs", [16, 64])
def test_lists_windows_and_absent_pages(ops, dtype, fp8, D, bs):
    """Listed tiles that the window hides as a whole between seen ones, and blocks without a page."""
    print(f"masks lists {dtype} fp8={fp8} D={D} bs={bs}", flush=True)
    n = 30
    c = cache([bs * n - 3, bs * 11], Hq=6, Hkv=2, D=D, bs=bs, dtype=dtype, fp8=fp8, seed=D + bs)
    MP = c["table"].shape[1]
    g = torch.Generator().manual_seed(bs)
    kv_idx = torch.stack([torch.stack([torch.randperm(MP, generator=g)[:20] for _ in range(2)]) for _ in range(2)]).int()
    kv_num = torch.tensor([[20, 13], [20, 0]], dtype=torch.int32)
    first = torch.tensor([bs * 14 + 5, 3], dtype=torch.int32)
    c["table"][0, 20], c["table"][1, 2] = -1, c["k_pages"].shape[0]
    check(ops, c, scale=0.12, kv_num=kv_num, kv_idx=kv_idx, first=first)
    check(ops, c, scale=0.12, first=first)
    # a window behind the last key of one of them
    check(ops, c, scale=0.12, first=torch.tensor([bs * n, bs * 11 - 1], dtype=torch.int32))


@pytest.mark.parametrize("dtype,fp8", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("shape", ["rising", "falling", "waves"])
def test_scores_that_move(ops, dtype, fp8, D, shape):
    """Scores that climb, sink or swing by some hundreds along the cache, another height every tile: the largest of
    a tile lies far below and far above those before it."""
    print(f"masks moving {dtype} fp8={fp8} D={D} {shape}", flush=True)
    bs, n = 32, 130
    c = cache([bs * n - 7], Hq=4, Hkv=2, D=D, bs=bs, dtype=dtype, fp8=fp8, seed=D)
    at = torch.arange(n)
    level = {"rising": at / n, "falling": 1 - at / n, "waves": torch.sin(at * 0.9)}[shape] * 200
    c["q"][:, :, 0] = torch.tensor([1.0, -1.0, 0.5, 1.0]).to(c["q"].dtype)
    for i in range(n):
        k = c["k_pages"][int(c["table"][0, i])].float()
        k[:, :, 0] = level[i] if not fp8 else (level[i] / c["k_scale"][:, None]).clamp(-448, 448)
        c["k_pages"][int(c["table"][0, i])] = k.to(c["k_pages"].dtype)
    check(ops, c, scale=1.0 if not fp8 else 20.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_infinite_and_nan_keys(ops, dtype):
    """A key whose score is -inf takes no weight, one of +inf or NaN makes its heads NaN and no others."""
    c = cache([900, 200], Hq=4, Hkv=2, D=64, bs=32, dtype=dtype, seed=6)
    page = int(c["table"][0, 11])
    dev = lambda: [c[k].to(DEV) for k in ("q", "k_pages", "v_pages", "table", "lens")]  # noqa: E731
    c["q"][0, :2, 7] = -1.0
    c["k_pages"][page, 0, 5, 7] = 3e4
    want, wl = ops.paged_decode_attn(*dev(), scale=0.5)  # (its weight is 0)
    c["k_pages"][page, 0, 5, 7] = math.inf
    out, lse = ops.paged_decode_attn(*dev(), scale=0.5)
    assert torch.equal(out, want) and torch.equal(lse, wl)
    for bad in (-math.inf, math.nan):
        c["k_pages"][page, 0, 5, 7] = bad
        out, lse = ops.paged_decode_attn(*dev(), scale=0.5)
        assert bool(torch.isnan(out[0, :2].float()).all()) and bool((torch.isnan(lse[0, :2]) | torch.isposinf(lse[0, :2])).all())
        assert torch.equal(out[0, 2:], want[0, 2:]) and torch.equal(out[1], want[1]) and torch.equal(lse[1], wl[1])


@pytest.mark.parametrize("bs", [16, 128])
@pytest.mark.parametrize("dtype,fp8", [("fp16", False), ("fp16", True)])
def test_rows_that_are_not_seen_do_not_count(ops, dtype, fp8, bs):
    """NaN and infinities behind the length, before the first position and in pages of no block: the same bits."""
    c = cache([bs + 3, 3 * bs - 1], Hq=4, Hkv=2, D=128, bs=bs, dtype=dtype, fp8=fp8, seed=11)
    first = torch.tensor([2, bs + 5], dtype=torch.int32)
    want, wl = check(ops, c, scale=0.12, first=first)
    live = torch.zeros(c["k_pages"].shape[0], bs, dtype=torch.bool)
    for b, n in enumerate(c["lens"].tolist()):
        for j in range(int(first[b]), n):
            live[c["table"][b, j // bs], j % bs] = True
    d = dict(c)
    for name, poison in (("k_pages", math.nan), ("v_pages", math.nan if fp8 else math.inf)):
        x = c[name].float()
        x.transpose(1, 2)[~live] = poison
        d[name] = x.to(c[name].dtype)
    dev = lambda x: x.to(DEV) if isinstance(x, torch.Tensor) else x  # noqa: E731
    out, lse = ops.paged_decode_attn(*(dev(d[k]) for k in ("q", "k_pages", "v_pages", "table", "lens")), scale=0.12, first=first.to(DEV),
                                     k_scale=dev(d["k_scale"]), v_scale=dev(d["v_scale"]))
    assert torch.equal(out, want) and torch.equal(lse, wl)
