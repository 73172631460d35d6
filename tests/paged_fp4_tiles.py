"""Cases of the 4-bit attention whose wavefronts work on many tiles each, seeded and made
on the CPU.

The device has room for a few workgroups more than key heads here, so that the plan
gives every sequence one piece (or two) whatever its length: HEADS key heads, which
repeat DISTINCT different ones.  The oracle goes over those; the others have to give
the same bits."""
from __future__ import annotations

import torch

from oracle import paged as OP
from tests.paged_fp4_inputs import E8M0, FP4, pages
from tests.paged_inputs import TYPES

DISTINCT = 3

# (D, query heads a key head, page size, type): both ways of loading ahead, groups of up to 8 and of 9 to 16
# heads, two groups, pages of 16 and others
FORMS = [(64, 1, 16, "bf16"), (64, 2, 64, "fp16"), (64, 12, 32, "bf16"), (64, 9, 16, "fp16"), (128, 2, 16, "bf16"), (128, 8, 128, "bf16"),
         (128, 12, 16, "fp16"), (128, 20, 64, "bf16"), (256, 1, 64, "bf16"), (256, 3, 16, "fp16"), (256, 12, 32, "bf16"), (256, 9, 16, "fp16")]

# every number of tiles up to five for each wavefront, full and cut, and one piece past the 256 tiles that a
# workgroup's wavefronts look up at once
RAGGED = [32 * n - 7 * (n % 3) for n in range(1, 21)] + [9000]
KINDS = {
    "ragged": dict(Hkv=1536, lens=RAGGED, most=71),
    "windows": dict(Hkv=1536, lens=[4000, 1500, 700, 9300], first=[2531, 3, 690, 37], most=73),
    "rising": dict(Hkv=1536, lens=[4111, 9000], rise=0.08, most=71),
    "falling": dict(Hkv=1536, lens=[1111, 3000], rise=-0.08, most=24),
    "absent": dict(Hkv=1536, lens=[20000, 9999], runs=[(150, 12500), (3000, 9500)], some=0.3, most=157),
    "lists": dict(Hkv=1536, lens=[13001, 9600], listed=9600, most=75),
    "split": dict(Hkv=768, lens=[9000], most=36, pieces=2),
    "split_batch": dict(Hkv=768, lens=[9000, 700, 8000], most=36, pieces=2),
}


def heads(x, n):
    """Dimension 1 repeated to n."""
    return x[:, torch.arange(n, device=x.device) % x.shape[1]]


def make(kind, D, G, bs, dtype):
    """The case's tensors over the DISTINCT key heads."""
    k, g = KINDS[kind], torch.Generator().manual_seed(D + G + bs)
    lens = k["lens"]
    B, MP = len(lens), max(-(-n // bs) for n in lens) + 1
    need = [-(-n // bs) for n in lens]
    table = torch.full((B, MP), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = 0
        if "runs" in k:
            lo, hi = k["runs"][b]
            gone = torch.rand(n, generator=g) < k["some"]
            gone[lo // bs:hi // bs] = True
            gone[n - 1] = False
            table[b, :n][gone] = -1
    P = int((table == 0).sum())
    table[table == 0] = torch.randperm(P, generator=g).int()
    q = torch.randn((B, DISTINCT * G, D), generator=g).to(TYPES[dtype])
    (kp, ks), (vp, vs) = (pages(g, P, DISTINCT, bs, D, dtype) for _ in range(2))
    if "rise" in k:  # the first query of the first head: keys along it, longer from tile to tile (or shorter)
        for b, n in enumerate(need):
            pos = torch.arange(n * bs).reshape(n, bs)
            f = (pos if k["rise"] > 0 else pos[-1, -1] - pos) // 32 * abs(k["rise"]) / D * 64
            c, s = OP.quantise((q[b, 0].float() * f[..., None]).to(TYPES[dtype]))
            kp.view(torch.uint8)[table[b, :n].long(), 0], ks.view(torch.uint8)[table[b, :n].long(), 0] = c, s
    c = dict(q=q, k_pages=kp, v_pages=vp, k_scale=ks, v_scale=vs, table=table, lens=torch.tensor(lens, dtype=torch.int32),
             first=None, kv_num=None, kv_idx=None, mass=torch.rand((B, DISTINCT, MP), generator=g))
    if "first" in k:
        c["first"] = torch.tensor(k["first"], dtype=torch.int32)
    if "listed" in k:
        L = -(-k["listed"] // bs)  # (blocks behind the length among them, and none)
        c["kv_idx"] = torch.stack([torch.stack([torch.randperm(MP, generator=g)[:L] for _ in range(DISTINCT)]) for _ in lens]).int()
        c["kv_idx"] = torch.cat((c["kv_idx"], torch.full((B, DISTINCT, L - c["kv_idx"].shape[2]), -1, dtype=torch.int32)), 2)
        c["kv_idx"][0, 1, 5], c["kv_idx"][1, 0, 1] = MP, -1
        c["kv_num"] = torch.tensor([[L, L * 5 // 9, 1], [L + 3, 0, L - 1]], dtype=torch.int32)
    return c


def repeated(c, n):
    """The case over n key heads that repeat its own."""
    r = {k: x for k, x in c.items()}
    for k in ("k_pages", "v_pages", "k_scale", "v_scale"):
        r[k] = heads(c[k].view(torch.uint8), n).view(FP4 if k.endswith("pages") else E8M0)
    B, Hq, D = c["q"].shape
    G = Hq // DISTINCT
    r["q"] = heads(c["q"].reshape(B, DISTINCT, G, D), n).reshape(B, n * G, D)
    for k in ("mass", "kv_num", "kv_idx"):
        r[k] = None if c[k] is None else heads(c[k], n).contiguous()
    return r
