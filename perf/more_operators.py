"""The paged key-value cache in 4 bits: rows quantised as they are written, rows read
back, and the attention of one new token a sequence over such pages.

A row's features go in groups of 32 to e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives), two a byte, the lower nibble first, with a power of two as each group's
scale (e8m0).

``listed()`` names the cases, ``draw(rng)`` gives others of the same ranges,
``prepare`` makes a case's inputs on the GPU and ``run`` is one pass: the plain
form in elementary torch operations, or with ``own`` the framework's calls.
``work`` is what a pass cannot do without and ``exact`` the outputs in 64 bits.

Kinds:

* ``attend``  attention of one new token a sequence over 4-bit pages, all of them or
              per-head lists (the pointer mask's form), from a first position on; with
              the pages' weights added to a running mass.
* ``write``   new rows into 4-bit pages, one a sequence (a decode step) or ragged
              prompts, and the same rows read back as the values that are held.
* ``read``    ranges of rows of a batch out of pages of any type (4 bits, e4m3, 16
              bits), one after the other, as a dense attention takes them.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3_MAX = 448.0
GROUP = 32
# the largest power of two of a scale: six times it is finite in the rows' type
TOP = {torch.bfloat16: 125, torch.float16: 13}
LEAST = -125


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    return [
        # one decoder layer of one sequence: blocks of 128, the pointer mask's lists of nine blocks a head
        dict(name="attend_lists", kind="attend", B=1, Hq=8, Hkv=8, D=128, bs=128, lo=33000, hi=33000, lists=9, window=0,
             mass=False, type="bf16"),
        # a serving batch of ragged lengths, from one token to 16k, small pages, grouped heads
        dict(name="attend_ragged", kind="attend", B=32, Hq=32, Hkv=8, D=128, bs=16, lo=1, hi=16384, lists=0, window=0,
             mass=False, type="bf16"),
        # one long document, every page attended to and its weight accumulated
        dict(name="attend_128k_mass", kind="attend", B=1, Hq=8, Hkv=8, D=128, bs=128, lo=130995, hi=130995, lists=0,
             window=0, mass=True, type="bf16"),
        # narrow heads in half precision behind a window of positions, weights accumulated
        dict(name="attend_window_d64", kind="attend", B=48, Hq=12, Hkv=6, D=64, bs=32, lo=900, hi=20001, lists=0,
             window=4096, mass=True, type="fp16"),
        # wide heads, a batch of middling lengths
        dict(name="attend_d256", kind="attend", B=16, Hq=16, Hkv=4, D=256, bs=64, lo=700, hi=32768, lists=0, window=0,
             mass=False, type="bf16"),
        # the largest: eight query heads a key head, long sequences
        dict(name="attend_many", kind="attend", B=24, Hq=64, Hkv=8, D=128, bs=64, lo=9001, hi=65536, lists=0, window=0,
             mass=False, type="bf16"),
        # a decode step's rows
        dict(name="write_step", kind="write", N=64, B=64, Hkv=8, D=128, bs=128, held=8191, type="bf16"),
        # a chunk of three prompts, narrow heads in half precision
        dict(name="write_chunk_d64", kind="write", N=4099, B=3, Hkv=6, D=64, bs=32, held=5000, type="fp16"),
        # whole prompts, small pages
        dict(name="write_prompts", kind="write", N=65539, B=5, Hkv=8, D=128, bs=16, held=700, type="bf16"),
        # one long document out of 4-bit pages
        dict(name="read_document", kind="read", B=1, Hkv=8, D=128, bs=128, hi=131072, share=1.0, pages="fp4", type="bf16"),
        # the last half of each of a batch's sequences, 8-bit pages
        dict(name="read_batch_fp8", kind="read", B=32, Hkv=8, D=128, bs=16, hi=8192, share=0.5, pages="fp8", type="bf16"),
        # a few short sequences to be moved elsewhere, 16-bit pages
        dict(name="read_few", kind="read", B=7, Hkv=6, D=64, bs=64, hi=600, share=1.0, pages="16", type="fp16"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "write", "write", "read"])
    Hkv = rng.choice([1, 2, 4, 6, 8])
    D = rng.choice([64, 128, 128, 256])
    bs = rng.choice([16, 32, 64, 128, 256])
    type_ = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "attend":
        G = rng.choice([1, 1, 2, 3, 4, 7, 8, 16])
        B = _log(rng, 1, 96)
        # at most 0.8 G values in K
        hi = _log(rng, 64, max(64, min(131072, 800000000 // (B * Hkv * D))))
        lists = rng.choice([0, 0, _log(rng, 1, 40)])
        return dict(kind="attend", B=B, Hq=Hkv * G, Hkv=Hkv, D=D, bs=bs, lo=rng.choice([1, hi, max(1, hi // 2)]), hi=hi,
                    lists=lists, window=rng.choice([0, 0, _log(rng, 1, hi)]), mass=rng.random() < 0.5, type=type_)
    if kind == "write":
        step = rng.random() < 0.4
        B = _log(rng, 1, 256) if step else _log(rng, 1, 32)
        N = B if step else _log(rng, B, max(B, 70000000 // (Hkv * D)))
        return dict(kind="write", N=N, B=B, Hkv=Hkv, D=D, bs=bs, held=_log(rng, 1, 4096) - 1, type=type_)
    B = _log(rng, 1, 64)
    return dict(kind="read", B=B, Hkv=Hkv, D=D, bs=bs, hi=_log(rng, 1, min(131072, 100000000 // (B * Hkv * D))),
                share=rng.choice([1.0, 0.5, 0.1]), pages=rng.choice(["fp4", "fp4", "fp8", "16"]), type=type_)


def _lengths(lo, hi, n, rng):
    """Lengths between lo and hi, over their logarithm; the first is hi."""
    return [hi] + [_log(rng, lo, hi) for _ in range(n - 1)]


# --------------------------------------------------------------------------
# the 4-bit values
# --------------------------------------------------------------------------
def _quantise(x):
    """(bytes [..., D / 2], scale bytes [..., D / 32]) of 16-bit rows [..., D]."""
    f = x.float().reshape(*x.shape[:-1], -1, GROUP)
    m, e = torch.frexp(f.abs().amax(dim=-1))
    # the group's largest value is at most 6 of the scale, or 7 rounded to it
    e = torch.where(m >= 0.875, e - 2, e - 3).clamp_(LEAST, TOP[x.dtype])
    y = torch.ldexp(f, -e[..., None])
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp_(max=6)
    # 0 .. 2 in halves, then 3, 4, 6
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code | (torch.signbit(y).to(torch.uint8) << 3)
    code = code.reshape(*x.shape[:-1], -1, 2)
    return code[..., 0] | (code[..., 1] << 4), (e + 127).to(torch.uint8)


def _values(code, scale):
    """The fp32 numbers [..., D] that bytes and scale bytes stand for."""
    one = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float32, device=code.device)
    i = torch.arange(256, device=code.device)
    two = torch.stack((one[i % 16], one[i // 16]), dim=-1)
    x = two[code.int()].reshape(*scale.shape, GROUP)
    return (x * scale.view(torch.float8_e8m0fnu).float()[..., None]).reshape(*code.shape[:-1], -1)


def _take(pages, scale, page, head):
    """The listed pages of each key head [..., bs, D], fp32."""
    return _values(pages.view(torch.uint8)[page, head], scale.view(torch.uint8)[page, head])


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _rows(g, *shape, dtype):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _pool(g, P, Hkv, bs, D, pages, dtype):
    """Pages (and scales) whose rows have the spread of normed keys and values."""
    x = torch.randn((P, Hkv, bs, D), generator=g, device=DEV, dtype=torch.float32)
    if pages == "fp4":
        # some features are larger than others throughout, as those of keys are
        x *= torch.exp(0.5 * torch.randn((Hkv, 1, D), generator=g, device=DEV))
        code = torch.empty((P, Hkv, bs, D // 2), dtype=torch.uint8, device=DEV)
        scale = torch.empty((P, Hkv, bs, D // GROUP), dtype=torch.uint8, device=DEV)
        for at in range(0, P, 1 + 100000000 // (Hkv * bs * D)):  # a few at a time
            part = slice(at, at + 1 + 100000000 // (Hkv * bs * D))
            code[part], scale[part] = _quantise(x[part].to(dtype))
        return code.view(torch.float4_e2m1fn_x2), scale.view(torch.float8_e8m0fnu)
    if pages == "fp8":
        # a few heads are scaled so that some values saturate
        scale = 0.004 + 0.02 * torch.rand(Hkv, generator=g, device=DEV)
        return (x / scale[:, None, None]).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale
    return x.to(dtype), None


def _tables(g, B, MP, need, P):
    """A table whose first need[b] entries are pages of a shuffled pool, the rest none."""
    need = torch.tensor(need, device=DEV)
    held = torch.arange(MP, device=DEV)[None] < need[:, None]
    table = torch.full((B, MP), -1, dtype=torch.int32, device=DEV)
    table[held] = torch.randperm(P, generator=g, device=DEV)[:int(need.sum())].to(torch.int32)
    return table


def prepare(case, seed):
    rng = random.Random(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"attend": _prepare_attend, "write": _prepare_write, "read": _prepare_read}[case["kind"]](case, rng, g)


def _prepare_attend(case, rng, g):
    B, Hq, Hkv, D, bs, t = case["B"], case["Hq"], case["Hkv"], case["D"], case["bs"], TYPES[case["type"]]
    lens = _lengths(case["lo"], case["hi"], B, rng)
    MP = -(-max(lens) // bs) + 2
    need = [-(-n // bs) for n in lens]
    table = _tables(g, B, MP, need, sum(need))
    k_pages, ks = _pool(g, sum(need), Hkv, bs, D, "fp4", t)
    v_pages, vs = _pool(g, sum(need), Hkv, bs, D, "fp4", t)
    st = dict(case=case, q=_rows(g, B, Hq, D, dtype=t), k_pages=k_pages, v_pages=v_pages, k_scale=ks, v_scale=vs, table=table,
              lens=torch.tensor(lens, dtype=torch.int32, device=DEV), scale=0.12 if D == 128 else D ** -0.5, first=None,
              kv_num=None, kv_idx=None, mass=None)
    if case["window"]:
        st["first"] = (st["lens"] - case["window"]).clamp_(min=0)
    if case["lists"]:
        # the last blocks and others before them, distinct, in ascending order; lists of several lengths
        L = min(case["lists"], MP)
        nb = -(-st["lens"].long() // bs)
        key = torch.rand((B, Hkv, MP), generator=g, device=DEV)
        i = torch.arange(MP, device=DEV)
        key = torch.where(i >= nb[:, None, None] - max(1, L // 2), key + 1, key)
        key = torch.where(i < nb[:, None, None], key, key - 2)
        pick = key.topk(L, dim=-1).indices
        num = torch.minimum(nb[:, None].expand(B, Hkv), L - torch.randint(0, 1 + L // 4, (B, Hkv), generator=g, device=DEV))
        # the chosen ones first: sort those in use, the others behind them
        use = torch.arange(L, device=DEV) < num[..., None]
        st["kv_idx"] = torch.where(use, pick, MP).sort(dim=-1).values.clamp_(max=MP - 1).to(torch.int32)
        st["kv_num"] = num.to(torch.int32)
    if case["mass"]:
        st["mass"] = torch.rand((B, Hkv, MP), generator=g, device=DEV)
    return st


def _prepare_write(case, rng, g):
    N, B, Hkv, D, bs, t = case["N"], case["B"], case["Hkv"], case["D"], case["bs"], TYPES[case["type"]]
    if N == B:
        cu, rows = None, [1] * B
    else:
        cuts = [0] + sorted(rng.randint(0, N) for _ in range(B - 1)) + [N]
        rows = [b - a for a, b in zip(cuts, cuts[1:])]
        cu = torch.tensor(cuts, dtype=torch.int32, device=DEV)
    held = [rng.randint(0, case["held"]) for _ in range(B)]
    need = [-(-(h + r) // bs) for h, r in zip(held, rows)]
    # pages wholly before the new rows belong to the cache too, but are not touched: one for each sequence is kept here
    first = torch.tensor([max(0, h // bs - 1) for h in held], device=DEV)
    i = torch.arange(max(need) + 1, device=DEV)
    live = (i[None] >= first[:, None]) & (i[None] < torch.tensor(need, device=DEV)[:, None])
    # a pool that holds them whatever the lengths: a sequence's rows, and up to three pages that they share with others
    P = N // bs + 3 * B
    table = torch.full(live.shape, -1, dtype=torch.int32, device=DEV)
    table[live] = torch.randperm(P, generator=g, device=DEV)[:int(live.sum())].to(torch.int32)
    k_pages, ks = _pool(g, P, Hkv, bs, D, "fp4", t)
    v_pages, vs = _pool(g, P, Hkv, bs, D, "fp4", t)
    # k and v as slices of one projection's rows; some features are larger than others throughout
    kv = torch.randn((N, 2 * Hkv, D), generator=g, device=DEV)
    kv = (kv * torch.exp(0.5 * torch.randn((2 * Hkv, D), generator=g, device=DEV))).to(t)
    held = torch.tensor(held, dtype=torch.int32, device=DEV)
    return dict(case=case, k=kv[:, :Hkv], v=kv[:, Hkv:], k_pages=k_pages, v_pages=v_pages, table=table, cu=cu, k_scale=ks,
                v_scale=vs, held=held, lens=held + torch.tensor(rows, dtype=torch.int32, device=DEV))


def _prepare_read(case, rng, g):
    B, Hkv, D, bs, t = case["B"], case["Hkv"], case["D"], case["bs"], TYPES[case["type"]]
    # the same lengths in another order: the outputs are as long as their sum
    lens = _lengths(1, case["hi"], B, random.Random(0))
    rng.shuffle(lens)
    first = [n - max(1, int(case["share"] * n)) for n in lens]
    need = [-(-n // bs) for n in lens]
    table = _tables(g, B, max(need) + 1, need, sum(need))
    k_pages, ks = _pool(g, sum(need), Hkv, bs, D, case["pages"], t)
    v_pages, vs = _pool(g, sum(need), Hkv, bs, D, case["pages"], t)
    cuts = [0]
    for a, n in zip(first, lens):
        cuts.append(cuts[-1] + n - a)
    return dict(case=case, k_pages=k_pages, v_pages=v_pages, table=table, k_scale=ks, v_scale=vs, rows=cuts[-1], type=t,
                lens=torch.tensor(lens, dtype=torch.int32, device=DEV), first=torch.tensor(first, dtype=torch.int32, device=DEV),
                cu=torch.tensor(cuts, dtype=torch.int32, device=DEV))


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(state):
    return {"attend": _attend, "write": _write, "read": _read}[state["case"]["kind"]](state)


def _attend(s):
    if own:
        from scope_amd import ops

        out, lse = ops.paged_decode_attn(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], scale=s["scale"],
                                         first=s["first"], kv_num=s["kv_num"], kv_idx=s["kv_idx"], mass=s["mass"],
                                         k_scale=s["k_scale"], v_scale=s["v_scale"])
    else:
        q, kp, vp, table, lens = s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"]
        B, Hq, D = q.shape
        _, Hkv, bs, _ = kp.shape
        MP = table.shape[1]
        G = Hq // Hkv
        if s["kv_idx"] is None:
            lb = torch.arange(MP, device=q.device).expand(B, Hkv, MP)
            use = torch.ones_like(lb, dtype=torch.bool)
        else:
            lb = s["kv_idx"].long()
            use = torch.arange(lb.shape[-1], device=q.device) < s["kv_num"][..., None]
        E = lb.shape[-1]
        page = table.long()[:, None].expand(B, Hkv, MP).gather(2, lb)
        pos = lb[..., None] * bs + torch.arange(bs, device=q.device)
        low = torch.zeros_like(lens) if s["first"] is None else s["first"]
        see = (use & (page >= 0))[..., None] & (pos >= low[:, None, None, None]) & (pos < lens[:, None, None, None])
        see = see.reshape(B, Hkv, 1, E * bs)
        head = torch.arange(Hkv, device=q.device)[None, :, None]
        k = _take(kp, s["k_scale"], page.clamp(min=0), head).reshape(B, Hkv, E * bs, D)
        z = torch.matmul(q.float().reshape(B, Hkv, G, D), k.transpose(2, 3)) * s["scale"]
        del k
        z = torch.where(see, z, -math.inf)
        top = z.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
        p = torch.exp(z - top)
        total = p.sum(dim=-1, keepdim=True)
        p = p / torch.where(total > 0, total, 1.0)
        v = _take(vp, s["v_scale"], page.clamp(min=0), head).reshape(B, Hkv, E * bs, D)
        out = torch.matmul(p, v).reshape(B, Hq, D).to(q.dtype)
        lse = torch.where(total > 0, top + torch.log(total), -math.inf).reshape(B, Hq)
        if s["mass"] is not None:
            s["mass"].scatter_add_(2, lb, torch.where(use, p.reshape(B, Hkv, G, E, bs).sum(dim=(2, 4)), 0.0))
    return {"out": out, "lse": lse} if s["mass"] is None else {"out": out, "lse": lse, "mass": s["mass"]}


def _places(table, bs, cu, start, N):
    """(page, slot) of N rows from the positions `start` of their sequences on."""
    row = torch.arange(N, device=table.device)
    if cu is None:
        b, pos = row, start.long()
    else:
        b = torch.searchsorted(cu.long(), row, right=True) - 1
        pos = start.long()[b] + row - cu.long()[b]
    return table.long()[b, pos // bs], pos % bs


def _write(s):
    k, v, kp, vp, table, bs, N = s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["k_pages"].shape[2], s["k"].shape[0]
    if own:
        from scope_amd import ops

        ops.paged_append(k, v, kp, vp, table, s["held"], cu=s["cu"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        k, v = ops.paged_read(kp, vp, table, s["lens"], rows=N, cu=s["cu"], first=s["held"], k_scale=s["k_scale"],
                              v_scale=s["v_scale"], dtype=k.dtype)
        return {"k": k, "v": v}
    page, slot = _places(table, bs, s["cu"], s["held"], N)
    for x, pages, scale in ((k, kp, s["k_scale"]), (v, vp, s["v_scale"])):
        pages.view(torch.uint8)[page, :, slot], scale.view(torch.uint8)[page, :, slot] = _quantise(x)
    return {"k": _read_back(kp, s["k_scale"], page, slot, k.dtype), "v": _read_back(vp, s["v_scale"], page, slot, v.dtype)}


def _read_back(pages, scale, page, slot, dtype):
    """Rows [N, Hkv, D] out of their pages."""
    if pages.dtype == torch.float4_e2m1fn_x2:
        return _values(pages.view(torch.uint8)[page, :, slot], scale.view(torch.uint8)[page, :, slot]).to(dtype)
    if pages.dtype == torch.float8_e4m3fn:
        return (pages.view(torch.uint8)[page, :, slot].view(pages.dtype).float() * scale[:, None]).to(dtype)
    return pages[page, :, slot]


def _read(s):
    if own:
        from scope_amd import ops

        k, v = ops.paged_read(s["k_pages"], s["v_pages"], s["table"], s["lens"], rows=s["rows"], cu=s["cu"], first=s["first"],
                              k_scale=s["k_scale"], v_scale=s["v_scale"], dtype=s["type"])
        return {"k": k, "v": v}
    page, slot = _places(s["table"], s["k_pages"].shape[2], s["cu"], s["first"], s["rows"])
    return {"k": _read_back(s["k_pages"], s["k_scale"], page, slot, s["type"]),
            "v": _read_back(s["v_pages"], s["v_scale"], page, slot, s["type"])}


# --------------------------------------------------------------------------
# what a pass cannot do without, and its outputs in 64 bits
# --------------------------------------------------------------------------
def work(case):
    D, Hkv = case["D"], case["Hkv"]
    held = D / 2 + D / GROUP  # bytes of a row
    if case["kind"] == "attend":
        # the inputs of one seed stand for the others: the lengths are spread alike
        Hq, bs = case["Hq"], case["bs"]
        lens = _lengths(case["lo"], case["hi"], case["B"], random.Random(0))
        keys = 0
        for n in lens:
            seen = min(n, case["window"]) if case["window"] else n
            keys += min(seen, case["lists"] * bs) if case["lists"] else seen
        extra = 8 * case["B"] * Hkv * -(-max(lens) // bs) if case["mass"] else 0
        return {"bytes": 2 * keys * Hkv * held + 4 * case["B"] * Hq * D + extra, "flops": 4 * keys * Hq * D}
    if case["kind"] == "write":
        # the rows, the pages that they become and the values that these stand for
        return {"bytes": 2 * case["N"] * Hkv * (4 * D + held), "flops": 0}
    lens = _lengths(1, case["hi"], case["B"], random.Random(0))
    rows = sum(max(1, int(case["share"] * n)) for n in lens)
    return {"bytes": 2 * rows * Hkv * (2 * D + {"fp4": held, "fp8": D, "16": 2 * D}[case["pages"]]), "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "write": _exact_write, "read": _exact_read}[case["kind"]](s)


def _exact_values(pages, scale):
    """The numbers that pages [..., D / 2] with their scales, or whole rows, stand for."""
    b = pages.view(torch.uint8).long()
    nibbles = torch.stack((b & 15, b >> 4), dim=-1).flatten(-2)
    exponent, mantissa = (nibbles >> 1) & 3, (nibbles & 1).double()
    x = torch.where(exponent == 0, 0.5 * mantissa, (1 + 0.5 * mantissa) * 2.0 ** (exponent.double() - 1))
    x = torch.where(nibbles >= 8, -x, x)
    return x * (2.0 ** (scale.view(torch.uint8).double() - 127)).repeat_interleave(GROUP, dim=-1)


def _exact_attend(s):
    q = s["q"].double()
    B, Hq, D = q.shape
    Hkv, bs = s["k_pages"].shape[1:3]
    G = Hq // Hkv
    out = torch.zeros((B, Hq, D), dtype=torch.float64, device=DEV)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device=DEV)
    mass = None if s["mass"] is None else s["mass"].double()
    for b in range(B):
        n = int(s["lens"][b])
        low = 0 if s["first"] is None else int(s["first"][b])
        for h in range(Hkv):
            blocks = range(low // bs, -(-n // bs)) if s["kv_idx"] is None else s["kv_idx"][b, h, :int(s["kv_num"][b, h])].tolist()
            blocks = torch.tensor([i for i in blocks if i * bs < n and (i + 1) * bs > low], dtype=torch.long, device=DEV)
            if not len(blocks):
                continue
            pages = s["table"][b].long()[blocks]
            k, v = (_exact_values(x.view(torch.uint8)[pages, h], c.view(torch.uint8)[pages, h]).reshape(-1, D)
                    for x, c in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])))
            j = (blocks[:, None] * bs + torch.arange(bs, device=DEV)).reshape(-1)
            z = (q[b, h * G:(h + 1) * G] @ k.T) * s["scale"]
            z[:, (j < low) | (j >= n)] = -math.inf
            w = torch.softmax(z, dim=-1)
            out[b, h * G:(h + 1) * G] = w @ v
            lse[b, h * G:(h + 1) * G] = torch.logsumexp(z, dim=-1)
            if mass is not None:
                mass[b, h].index_add_(0, blocks, w.reshape(G, len(blocks), bs).sum(dim=(0, 2)))
    return {"out": out, "lse": lse} if mass is None else {"out": out, "lse": lse, "mass": mass}


def _exact_write(s):
    """Each value's nearest in the group's grid, by its distance to the borders between them."""
    grid = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    outs = {}
    for name in ("k", "v"):
        x = s[name].double()
        y = x.reshape(*x.shape[:2], -1, GROUP)
        a = y.abs().amax(dim=-1, keepdim=True)
        low = torch.floor(torch.log2(torch.where(a > 0, a, 1.0)))
        low = torch.where(2.0 ** low > a, low - 1, torch.where(2.0 ** (low + 1) <= a, low + 1, low))
        e = torch.where(a >= 1.75 * 2.0 ** low, low - 1, low - 2)
        e = torch.where(a > 0, e, float(LEAST)).clamp(LEAST, TOP[s[name].dtype])
        y = y / 2.0 ** e
        r = torch.zeros_like(y)
        for i in range(7):
            border = (grid[i] + grid[i + 1]) / 2
            # on a border the even one of the two codes
            past = (y.abs() >= border) if i % 2 else (y.abs() > border)
            r = torch.where(past, float(grid[i + 1]), r)
        outs[name] = (r * torch.sign(y) * 2.0 ** e).reshape(x.shape)
    return outs


def _exact_read(s):
    bs = s["k_pages"].shape[2]
    outs = {}
    for name, pages, scale in (("k", s["k_pages"], s["k_scale"]), ("v", s["v_pages"], s["v_scale"])):
        parts = []
        for b in range(s["table"].shape[0]):
            i = torch.arange(int(s["first"][b]), int(s["lens"][b]), device=DEV)
            page = s["table"][b].long()[i // bs]
            if pages.dtype == torch.float4_e2m1fn_x2:
                x = _exact_values(pages.view(torch.uint8)[page, :, i % bs], scale.view(torch.uint8)[page, :, i % bs])
            elif pages.dtype == torch.float8_e4m3fn:
                x = pages.view(torch.uint8)[page, :, i % bs].view(pages.dtype).double() * scale.double()[:, None]
            else:
                x = pages[page, :, i % bs].double()
            parts.append(x)
        outs[name] = torch.cat(parts)
    return outs
