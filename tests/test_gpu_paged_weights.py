"""Small weights, cancelling weights and infinite values in the paged decode
attention, on the GPU against closed forms in 64 bits.

The kernel takes a probability into its product with V as a sum of 16-bit parts:
three in bf16, off by at most 2^-23 of it; two in fp16, off by at most 2^-21 of
it, or by 2^-39 of the largest among the 32 keys of its tile where that is more
(half of fp16's smallest step, the largest scaled to 2^14 or more).  The tiles'
largest sum to no more than all probabilities do, so fp16 loses at most
32·2^-39 = 2^-34 of the largest |v| of the output, however long the cache is."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def ops():
    from scope_amd import ops

    return ops


def paged(x, bs, seed):
    """Rows [B, T, Hkv, D] as pages in shuffled places: (pages, table)."""
    B, T, Hkv, D = x.shape
    MP = -(-T // bs)
    rows = torch.zeros((B, MP * bs, Hkv, D), dtype=torch.float32, device=DEV)
    rows[:, :T] = x
    place = torch.randperm(B * MP, generator=torch.Generator().manual_seed(seed)).to(DEV)
    pages = torch.zeros((B * MP, Hkv, bs, D), dtype=torch.float32, device=DEV)
    pages[place] = rows.reshape(B * MP, bs, Hkv, D).transpose(1, 2)
    return pages, place.reshape(B, MP).to(torch.int32)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype,fp8", [("fp16", False), ("fp16", True), ("bf16", False), ("bf16", True)])
@pytest.mark.parametrize("D,bs,T", [(64, 128, 131072), (128, 16, 40001), (256, 64, 32768)])
@pytest.mark.parametrize("sink", ["first", "inside", "last"])
def test_small_weights_add_up(ops, dtype, fp8, D, bs, T, sink):
    """One key that takes nearly all of the weight and has no value, the others 0 to 24 nats below it
    (one gap a query head) with values about 1: the output is what the many small weights sum to."""
    print(f"small weights {dtype} fp8={fp8} D={D} bs={bs} T={T} sink={sink}", flush=True)
    t = TYPES[dtype]
    gaps = torch.tensor([0.0, 5.0, 12.0, 16.5, 17.0, 17.375, 18.0, 20.0, 21.0, 22.0, 23.0, 24.0], device=DEV)
    at = {"first": 0, "inside": T // 2 + 7, "last": T - 1}[sink]
    q = torch.zeros((1, len(gaps), D), device=DEV)
    q[0, :, 3] = gaps
    k = torch.zeros((1, T, 1, D), device=DEV)
    k[0, at, 0, 3] = 1.0
    g = torch.Generator(device=DEV).manual_seed(T)
    page_t = torch.float8_e4m3fn if fp8 else t
    v = (0.5 + torch.rand((1, T, 1, D), generator=g, device=DEV)).to(page_t).float()
    v[0, at] = 0.0
    kp, table = paged(k, bs, 1)
    vp, _ = paged(v, bs, 1)
    out, lse = ops.paged_decode_attn(q.to(t), kp.to(page_t), vp.to(page_t), table, torch.tensor([T], device=DEV), scale=1.0)
    # relative to the sink: its own weight 1, each other's e^-gap
    small, total = torch.exp(-gaps.double()), v[0, :, 0].double().sum(0)
    whole = 1 + (T - 1) * small
    want = (small / whole)[:, None] * total
    assert ((lse[0].double() - (gaps.double() + torch.log(whole))).abs() <= 2.0 ** -16 + 2.0 ** -22 * gaps).all()
    # (the result's rounding: half a step of it, or of the smallest number; scores up to 24 in log2 units of 35, three
    # roundings of 2^-24 each, and the exponential's: 35·3·2^-24 + 2^-22 of a weight; sums of partial sums 2^-16)
    rel = 2.0 ** -21 + 105 * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -16
    bound = (half_step(t) + rel) * want
    if dtype == "fp16":
        bound = bound + 2.0 ** -25 + 2.0 ** -34 * 1.5  # (|v| <= 1.5)
    over = (out[0].double() - want).abs() - bound
    assert over.max() <= 0, f"gap {gaps[int(over.amax(1).argmax())].item()}: {over.max().item():.3e} over its bound"


@pytest.mark.parametrize("dtype,fp8", [("fp16", False), ("fp16", True), ("bf16", False), ("bf16", True)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_weights_that_cancel(ops, dtype, fp8, D):
    """Two keys whose weighted values cancel but for the rounding of one of them: what is left shows
    a weight's error."""
    t, B, H = TYPES[dtype], 32, 4
    page_t = torch.float8_e4m3fn if fp8 else t
    g = torch.Generator(device=DEV).manual_seed(D)
    gap = (0.01 + 0.09 * torch.rand((B, H), generator=g, device=DEV)).to(t)
    q = torch.zeros((B, H, D), dtype=t, device=DEV)
    q[:, :, 0] = gap
    w = torch.exp(-gap.double())
    a = (0.5 + torch.rand((B, H, D), generator=g, device=DEV)).to(page_t).double()
    k, v = (torch.zeros((B, 2, H, D), device=DEV) for _ in range(2))
    k[:, 0, :, 0] = 1.0
    v[:, 0] = a.float()
    v[:, 1] = -(a / w[..., None]).float().to(page_t).float()
    kp, table = paged(k, 16, 2)
    vp, _ = paged(v, 16, 2)
    out, _ = ops.paged_decode_attn(q, kp.to(page_t), vp.to(page_t), table, torch.full((B,), 2, device=DEV), scale=1.0)
    b = v[:, 1].double()
    want = (a + w[..., None] * b) / (1 + w[..., None])
    spread = (a.abs() + w[..., None] * b.abs()) / (1 + w[..., None])
    # parts 2^-21 (fp16) or 2^-23; the exponential 2^-22 and its argument, a difference of numbers up to 0.15, 2^-25;
    # a few fp32 additions and the division, 2^-21 in all
    bound = half_step(t) * want.abs() + 2.0 ** -20 * spread + (2.0 ** -25 if dtype == "fp16" else 0.0)
    over = (out.double() - want).abs() - bound
    assert over.max() <= 0, f"{over.max().item():.3e} over its bound, {(over > 0).double().mean().item():.3f} of the outputs"


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,bs", [(64, 16), (128, 128), (256, 32)])
def test_infinite_values_stay_infinite(ops, dtype, D, bs):
    """Infinities of either sign in seen rows whose weight is at least 2^-15 of the largest: their feature is that
    infinity, all others are as without them."""
    t, B, H, T = TYPES[dtype], 3, 4, 300
    g = torch.Generator(device=DEV).manual_seed(D)
    q = torch.randn((B, H, D), generator=g, device=DEV).clamp_(-2, 2).to(t)
    k = torch.randn((B, T, 2, D), generator=g, device=DEV).clamp_(-2, 2)
    scale = 5.0 / (4 * D)  # scores within 5 either way
    v = torch.randn((B, T, 2, D), generator=g, device=DEV)
    bad = v.clone()
    signs = torch.zeros((B, 2, D), device=DEV)
    for b in range(B):
        for h in range(2):
            for f, sign in ((1 + b, 1.0), (D - 1 - h, -1.0), (D // 2 + b + 3 * h, 1.0)):
                bad[b, (37 * b + 101 * h + 11 * f) % T, h, f] = sign * math.inf
                signs[b, h, f] = sign
    kp, table = paged(k, bs, 3)
    lens = torch.full((B,), T, device=DEV)
    out, lse = (ops.paged_decode_attn(q, kp.to(t), paged(x, bs, 3)[0].to(t), table, lens, scale=scale) for x in (v, bad))
    signs = signs.repeat_interleave(2, dim=1)
    clean, got = out[0], lse[0]
    assert torch.equal(out[1], lse[1])  # (the sums do not see V)
    assert torch.equal(got[signs != 0].float(), signs[signs != 0] * math.inf)
    assert torch.equal(got[signs == 0], clean[signs == 0])
