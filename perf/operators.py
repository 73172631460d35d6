"""The serving operators: a paged key-value cache (filling it, attending to it with
one new token a sequence, keeping it within a budget) and the penalties, biases
and grammar bits on a step's logits.

``listed()`` names the cases, ``draw(rng)`` gives others of the same ranges,
``prepare`` makes a case's inputs on the GPU and ``run`` is one pass: the plain
form in elementary torch operations, or with ``own`` the framework's calls.
``work`` is what a pass cannot do without and ``exact`` the outputs in 64 bits.

Kinds:

* ``append``    rows of new tokens into the pages: one a sequence (a decode step)
                or ragged prompts.  Pages of the rows' type or in e4m3.
* ``attend``    attention of one new token a sequence over its pages, all of them
                or per-head lists (the pointer mask's form), from a first
                position on; with the pages' weights added to a running mass.
* ``evict``     the pages of least accumulated weight leave, down to a budget.
* ``penalise``  repetition, presence and frequency penalties, temperature, a
                dense bias and grammar bits on the logits.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3_MAX = 448.0


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    return [
        # one decoder layer of one sequence: blocks of 128, the pointer mask's lists of nine blocks a head
        dict(name="attend_lists", kind="attend", B=1, Hq=8, Hkv=8, D=128, bs=128, lo=33000, hi=33000, lists=9, window=0,
             mass=False, type="bf16", fp8=False),
        # a serving batch of ragged lengths, from one token to 16k, small pages, grouped heads
        dict(name="attend_ragged", kind="attend", B=32, Hq=32, Hkv=8, D=128, bs=16, lo=1, hi=16384, lists=0, window=0,
             mass=False, type="bf16", fp8=False),
        # one long document, every page attended to and its weight accumulated
        dict(name="attend_128k_mass", kind="attend", B=1, Hq=8, Hkv=8, D=128, bs=128, lo=130995, hi=130995, lists=0,
             window=0, mass=True, type="bf16", fp8=False),
        # narrow heads in half precision behind a window of positions, weights accumulated
        dict(name="attend_window_d64", kind="attend", B=48, Hq=12, Hkv=6, D=64, bs=32, lo=900, hi=20001, lists=0,
             window=4096, mass=True, type="fp16", fp8=False),
        # the largest: 8-bit pages, eight query heads a key head
        dict(name="attend_fp8", kind="attend", B=24, Hq=64, Hkv=8, D=128, bs=64, lo=9001, hi=65536, lists=0, window=0,
             mass=False, type="bf16", fp8=True),
        # the write of a decode step
        dict(name="append_step", kind="append", N=64, B=64, Hkv=8, D=128, bs=128, held=8191, type="bf16", fp8=False),
        # ragged prompts into 8-bit pages
        dict(name="append_prompts", kind="append", N=65539, B=5, Hkv=8, D=128, bs=16, held=700, type="bf16", fp8=True),
        # one sequence of 128k tokens down to a quarter of its blocks
        dict(name="evict_one", kind="evict", B=1, Hkv=8, MP=1027, bs=128, keep=256, window=4, n_global=1),
        # a batch with small pages
        dict(name="evict_batch", kind="evict", B=64, Hkv=8, MP=8192, bs=16, keep=3001, window=8, n_global=2),
        # the token loop of one sequence: the repetition penalty over a prompt of nine blocks
        dict(name="penalise_one", kind="penalise", B=1, V=50257, T=131456, lo=1152, hi=1152, type="fp32", full=False),
        # a batch with everything on, half-precision logits
        dict(name="penalise_batch", kind="penalise", B=128, V=50304, T=8192, lo=1, hi=8192, type="bf16", full=True),
        # long histories over a larger vocabulary of odd size
        dict(name="penalise_long", kind="penalise", B=16, V=100003, T=131072, lo=60000, hi=131072, type="fp32", full=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "evict", "penalise"])
    if kind == "attend":
        Hkv = rng.choice([1, 2, 4, 6, 8])
        G = rng.choice([1, 1, 2, 3, 4, 7, 8, 16])
        D = rng.choice([64, 128, 128, 256])
        bs = rng.choice([16, 32, 64, 128, 256])
        B = _log(rng, 1, 96)
        fp8 = rng.random() < 0.35
        # at most half a gigabyte of K and V rows
        hi = _log(rng, 64, max(64, min(131072, int(5e8 / (B * Hkv * D * (2 if fp8 else 4))))))
        lists = rng.choice([0, 0, _log(rng, 1, 40)])
        return dict(kind="attend", B=B, Hq=Hkv * G, Hkv=Hkv, D=D, bs=bs, lo=rng.choice([1, hi, max(1, hi // 2)]), hi=hi,
                    lists=lists, window=rng.choice([0, 0, _log(rng, 1, hi)]), mass=rng.random() < 0.5,
                    type=rng.choice(["bf16", "fp16"]), fp8=fp8)
    if kind == "append":
        step = rng.random() < 0.4
        B = _log(rng, 1, 256) if step else _log(rng, 1, 32)
        Hkv, D = rng.choice([1, 2, 4, 6, 8]), rng.choice([64, 128, 256])
        N = B if step else _log(rng, B, max(B, 70000000 // (Hkv * D)))
        return dict(kind="append", N=N, B=B, Hkv=Hkv, D=D, bs=rng.choice([16, 32, 64, 128, 256]), held=_log(rng, 1, 4096) - 1,
                    type=rng.choice(["bf16", "fp16"]), fp8=rng.random() < 0.4)
    if kind == "evict":
        B = _log(rng, 1, 96)
        MP = _log(rng, 4, max(4, 500000 // B))
        return dict(kind="evict", B=B, Hkv=rng.choice([1, 2, 4, 6, 8]), MP=min(MP, 16384), bs=rng.choice([16, 32, 64, 128, 256]),
                    keep=_log(rng, 1, min(MP, 16384)), window=rng.randint(1, 8), n_global=rng.randint(0, 4))
    B = _log(rng, 1, 128)
    V = _log(rng, 300, 160000)
    T = _log(rng, 1, max(1, min(131072, 2000000 // B)))
    return dict(kind="penalise", B=B, V=V, T=T, lo=rng.choice([0, T, T // 2]), hi=T, type=rng.choice(["fp32", "bf16", "fp16"]),
                full=rng.random() < 0.6)


def _lengths(case, n, rng):
    """Lengths between lo and hi, over their logarithm; the first is hi."""
    lo, hi = case["lo"], case["hi"]
    out = [hi] + [_log(rng, lo, hi) if lo >= 1 else rng.randint(lo, hi) for _ in range(n - 1)]
    return out


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _rows(g, *shape, dtype):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _pool(g, P, Hkv, bs, D, case):
    """Pages whose rows have the spread of normed keys and values."""
    if not case["fp8"]:
        t = TYPES[case["type"]]
        return torch.randn((P, Hkv, bs, D), generator=g, device=DEV, dtype=torch.float32).to(t), None
    # a few heads are scaled so that some values saturate
    scale = 0.004 + 0.02 * torch.rand(Hkv, generator=g, device=DEV)
    x = torch.randn((P, Hkv, bs, D), generator=g, device=DEV, dtype=torch.float32) / scale[:, None, None]
    return x.clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _tables(g, B, MP, need):
    """A table whose first need[b] entries are pages of a shuffled pool, the rest none; and the pool's size."""
    need = torch.tensor(need, device=DEV)
    held = torch.arange(MP, device=DEV)[None] < need[:, None]
    P = max(1, int(need.sum()))
    table = torch.full((B, MP), -1, dtype=torch.int32, device=DEV)
    table[held] = torch.randperm(P, generator=g, device=DEV).to(torch.int32)
    return table, P


def prepare(case, seed):
    import random

    rng = random.Random(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"attend": _prepare_attend, "append": _prepare_append, "evict": _prepare_evict,
            "penalise": _prepare_penalise}[case["kind"]](case, rng, g)


def _prepare_attend(case, rng, g):
    B, Hq, Hkv, D, bs = case["B"], case["Hq"], case["Hkv"], case["D"], case["bs"]
    lens = _lengths(case, B, rng)
    MP = -(-max(lens) // bs) + 2
    table, P = _tables(g, B, MP, [-(-n // bs) for n in lens])
    k_pages, ks = _pool(g, P, Hkv, bs, D, case)
    v_pages, vs = _pool(g, P, Hkv, bs, D, case)
    st = dict(case=case, q=_rows(g, B, Hq, D, dtype=TYPES[case["type"]]), k_pages=k_pages, v_pages=v_pages, k_scale=ks,
              v_scale=vs, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
              scale=0.12 if D == 128 else D ** -0.5, first=None, kv_num=None, kv_idx=None, mass=None)
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


def _prepare_append(case, rng, g):
    N, B, Hkv, D, bs = case["N"], case["B"], case["Hkv"], case["D"], case["bs"]
    if N == B:
        cu, rows = None, [1] * B
    else:
        cuts = [0] + sorted(rng.randint(0, N) for _ in range(B - 1)) + [N]
        rows = [b - a for a, b in zip(cuts, cuts[1:])]
        cu = torch.tensor(cuts, dtype=torch.int32, device=DEV)
    held = [rng.randint(0, case["held"]) if case["held"] else 0 for _ in range(B)]
    need = [-(-(h + r) // bs) for h, r in zip(held, rows)]
    # pages wholly behind the new rows belong to the cache too, but are not touched: one for each sequence is kept here
    table, _ = _tables(g, B, max(need) + 1, need)
    first = torch.tensor([max(0, h // bs - 1) for h in held], device=DEV)
    i = torch.arange(table.shape[1], device=DEV)
    live = (i[None] >= first[:, None]) & (table >= 0)
    # a pool that holds them whatever the lengths: a sequence's rows, and up to three pages that they share with others
    P = N // bs + 3 * B
    table = torch.where(live, 0, -1).to(torch.int32)
    table[live] = torch.randperm(P, generator=g, device=DEV)[:int(live.sum())].to(torch.int32)
    t = TYPES[case["type"]]
    k_pages, ks = _pool(g, P, Hkv, bs, D, case)
    v_pages, vs = _pool(g, P, Hkv, bs, D, case)
    # k and v as slices of one projection's rows
    kv = _rows(g, N, 2 * Hkv, D, dtype=t)
    return dict(case=case, k=kv[:, :Hkv], v=kv[:, Hkv:], k_pages=k_pages, v_pages=v_pages, table=table, cu=cu, k_scale=ks,
                v_scale=vs, lens=torch.tensor(held, dtype=torch.int32, device=DEV))


def _prepare_evict(case, rng, g):
    B, Hkv, MP, bs = case["B"], case["Hkv"], case["MP"], case["bs"]
    lens = [MP * bs - rng.randint(0, bs - 1) if b == 0 else rng.randint(0, MP * bs) for b in range(B)]
    table, _ = _tables(g, B, MP, [-(-n // bs) for n in lens])
    # some pages went in earlier passes
    table = torch.where(torch.rand((B, MP), generator=g, device=DEV) < 0.1, -1, table)
    # weights fall off steeply: few pages hold most of them, some have none yet
    mass = torch.randn((B, Hkv, MP), generator=g, device=DEV).mul_(2.0).exp_()
    mass = mass * (torch.rand((B, 1, MP), generator=g, device=DEV) < 0.95)
    budget = torch.tensor([max(0, case["keep"] - rng.randint(0, case["keep"] // 2)) for _ in range(B)], dtype=torch.int32,
                          device=DEV)
    return dict(case=case, table=table, mass=mass, lens=torch.tensor(lens, dtype=torch.int32, device=DEV), budget=budget)


def _prepare_penalise(case, rng, g):
    B, V, T = case["B"], case["V"], case["T"]
    lens = _lengths(case, B, rng)
    # tokens of a text: low ones often, high ones seldom
    u = torch.rand((B, T), generator=g, device=DEV, dtype=torch.float64)
    tokens = (torch.exp(u * math.log(V + 1.0)) - 1).long().clamp_(0, V - 1)
    st = dict(case=case, logits=(torch.randn((B, V), generator=g, device=DEV) * 4).to(TYPES[case["type"]]), tokens=tokens,
              lens=torch.tensor(lens, dtype=torch.int32, device=DEV), first=None, n_prompt=None, repetition=1.3, presence=0.0,
              frequency=0.0, temperature=1.0, bias=None, mask=None)
    if case["full"]:
        st["first"] = torch.tensor([rng.randint(0, n // 4) for n in lens], dtype=torch.int32, device=DEV)
        st["n_prompt"] = torch.tensor([rng.randint(0, n) for n in lens], dtype=torch.int32, device=DEV)
        for name, a, b in (("repetition", 1.0, 1.5), ("presence", -0.5, 1.0), ("frequency", 0.0, 0.4), ("temperature", 0.5, 1.5)):
            st[name] = a + (b - a) * torch.rand(B, generator=g, device=DEV)
        st["bias"] = torch.randn(V, generator=g, device=DEV) * (torch.rand(V, generator=g, device=DEV) < 0.02)
        # a grammar that leaves half of the words open
        words = torch.randint(-2 ** 31, 2 ** 31, (B, -(-V // 32)), generator=g, device=DEV, dtype=torch.int64)
        st["mask"] = words.to(torch.int32)
    return st


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(state):
    return {"attend": _attend, "append": _append, "evict": _evict, "penalise": _penalise}[state["case"]["kind"]](state)


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
        k = _take(kp, page.clamp(min=0), head).float().reshape(B, Hkv, E * bs, D)
        if s["k_scale"] is not None:
            k = k * s["k_scale"][:, None, None]
        z = torch.matmul(q.float().reshape(B, Hkv, G, D), k.transpose(2, 3)) * s["scale"]
        z = torch.where(see, z, -math.inf)
        top = z.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
        p = torch.exp(z - top)
        total = p.sum(dim=-1, keepdim=True)
        p = p / torch.where(total > 0, total, 1.0)
        v = _take(vp, page.clamp(min=0), head).float().reshape(B, Hkv, E * bs, D)
        if s["v_scale"] is not None:
            v = v * s["v_scale"][:, None, None]
        out = torch.matmul(p, v).reshape(B, Hq, D).to(q.dtype)
        lse = torch.where(total > 0, top + torch.log(total), -math.inf).reshape(B, Hq)
        if s["mass"] is not None:
            s["mass"].scatter_add_(2, lb, torch.where(use, p.reshape(B, Hkv, G, E, bs).sum(dim=(2, 4)), 0.0))
    return {"out": out, "lse": lse} if s["mass"] is None else {"out": out, "lse": lse, "mass": s["mass"]}


def _take(pages, page, head):
    """The listed pages of each key head [B, Hkv, E, bs, D]."""
    if pages.dtype == torch.float8_e4m3fn:
        return pages.view(torch.uint8)[page, head].view(torch.float8_e4m3fn)
    return pages[page, head]


def _append(s):
    if own:
        from scope_amd import ops

        ops.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], cu=s["cu"], k_scale=s["k_scale"],
                         v_scale=s["v_scale"])
    else:
        kp, vp, table = s["k_pages"], s["v_pages"], s["table"]
        N, bs = s["k"].shape[0], kp.shape[2]
        row = torch.arange(N, device=table.device)
        if s["cu"] is None:
            b, pos = row, s["lens"].long()
        else:
            b = torch.searchsorted(s["cu"].long(), row, right=True) - 1
            pos = s["lens"].long()[b] + row - s["cu"].long()[b]
        page = table.long()[b, pos // bs]
        for pages, x, scale in ((kp, s["k"], s["k_scale"]), (vp, s["v"], s["v_scale"])):
            if scale is None:
                pages[page, :, pos % bs] = x
            else:
                x = (x.float() / scale[:, None]).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
                pages.view(torch.uint8)[page, :, pos % bs] = x.view(torch.uint8)
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _evict(s):
    c = s["case"]
    if own:
        from scope_amd import ops

        table, freed, n = ops.paged_evict(s["table"], s["mass"], s["lens"], s["budget"], bs=c["bs"], window=c["window"],
                                          n_global=c["n_global"])
    else:
        MP = s["table"].shape[1]
        i = torch.arange(MP, device=s["table"].device)
        nb = ((s["lens"].long().clamp(max=MP * c["bs"]) + c["bs"] - 1) // c["bs"])[:, None]
        held = (s["table"] >= 0) & (i < nb)
        may = held & (i >= c["n_global"]) & (i < nb - c["window"])
        # summed in 64 bits, so that the order of the heads changes nothing next to a border
        score = torch.where(may, s["mass"].double().sum(dim=1).float(), math.inf)
        order = score.sort(dim=1, stable=True).indices
        rank = torch.empty_like(order).scatter_(1, order, i.expand_as(order))
        go = may & (rank < (held.sum(dim=1) - s["budget"])[:, None])
        table = torch.where(go, -1, s["table"])
        n = go.sum(dim=1).to(torch.int32)
        place = torch.where(go, go.cumsum(dim=1) - 1, MP)
        freed = torch.full((go.shape[0], MP + 1), -1, dtype=torch.int32, device=table.device)
        freed = freed.scatter_(1, place, torch.where(go, s["table"], -1))[:, :MP].contiguous()
    return {"table": table, "freed": freed, "n": n}


def _penalise(s):
    if own:
        from scope_amd import ops

        return ops.logit_penalties(s["logits"], s["tokens"], s["lens"], first=s["first"], n_prompt=s["n_prompt"],
                                   repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                                   temperature=s["temperature"], bias=s["bias"], mask=s["mask"])
    z = s["logits"].float()
    B, V = z.shape
    at = torch.arange(s["tokens"].shape[1], device=z.device)
    live = at < s["lens"][:, None]
    if s["first"] is not None:
        live = live & (at >= s["first"][:, None])
    new = live if s["n_prompt"] is None else live & (at >= s["n_prompt"][:, None])
    seen = torch.zeros((B, V), dtype=torch.int32, device=z.device).scatter_add_(1, s["tokens"], live.int()) > 0
    count = torch.zeros((B, V), dtype=torch.int32, device=z.device).scatter_add_(1, s["tokens"], new.int()).float()
    r, f, p, t = ((x[:, None] if isinstance(x, torch.Tensor) else x)
                  for x in (s["repetition"], s["frequency"], s["presence"], s["temperature"]))
    z = torch.where(seen, torch.where(z > 0, z / r, z * r), z)
    z = z - f * count
    z = z - p * (count > 0)
    if s["bias"] is not None:
        z = z + s["bias"]
    z = z / t
    if s["mask"] is not None:
        word = torch.arange(V, device=z.device)
        z = torch.where((s["mask"][:, word // 32] >> (word % 32).to(torch.int32)) & 1 != 0, z, -math.inf)
    return z.to(s["logits"].dtype)


# --------------------------------------------------------------------------
# what a pass cannot do without, and its outputs in 64 bits
# --------------------------------------------------------------------------
def work(case):
    import random

    if case["kind"] == "attend":
        # the inputs of one seed stand for the others: the lengths are spread alike
        D, Hq, Hkv, bs = case["D"], case["Hq"], case["Hkv"], case["bs"]
        size = 1 if case["fp8"] else 2
        lens = _lengths(case, case["B"], random.Random(0))
        keys = 0
        for n in lens:
            seen = min(n, case["window"]) if case["window"] else n
            keys += min(seen, case["lists"] * bs) if case["lists"] else seen
        extra = 8 * case["B"] * Hkv * -(-max(lens) // bs) if case["mass"] else 0
        return {"bytes": 2 * keys * Hkv * D * size + 4 * case["B"] * Hq * D + extra, "flops": 4 * keys * Hq * D}
    if case["kind"] == "append":
        return {"bytes": 2 * case["N"] * case["Hkv"] * case["D"] * (3 if case["fp8"] else 4), "flops": 0}
    if case["kind"] == "evict":
        pages = case["MP"] * (1 + (case["B"] - 1) / 2)
        return {"bytes": 4 * pages * case["Hkv"] + 12 * case["B"] * case["MP"], "flops": pages * case["Hkv"]}
    size = TYPES[case["type"]].itemsize
    lens = _lengths(case, case["B"], random.Random(0))
    shared = (case["B"] * case["V"] / 8 + 4 * case["V"]) if case["full"] else 0
    return {"bytes": 2 * size * case["B"] * case["V"] + 8 * sum(lens) + shared, "flops": 8 * case["B"] * case["V"]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "evict": lambda s: None, "penalise": _exact_penalise}[case["kind"]](s)


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
            k, v = ((x.view(torch.uint8)[pages, h].view(x.dtype) if x.dtype == torch.float8_e4m3fn else x[pages, h])
                    .double().reshape(-1, D) * (1.0 if c is None else c[h].double())
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


def _exact_append(s):
    bs = s["k_pages"].shape[2]
    outs = {}
    for name, x, scale in (("k_pages", s["k"], s["k_scale"]), ("v_pages", s["v"], s["v_scale"])):
        x = x.double()
        if scale is not None:
            x = (x / scale.double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        pages = s[name].double()
        for b in range(s["table"].shape[0]):
            r0, r1 = (b, b + 1) if s["cu"] is None else (int(s["cu"][b]), int(s["cu"][b + 1]))
            pos = torch.arange(r1 - r0, device=DEV) + s["lens"][b].long()
            pages[s["table"][b].long()[pos // bs], :, pos % bs] = x[r0:r1]
        outs[name] = pages
    return outs


def _exact_penalise(s):
    B, V = s["logits"].shape
    z = s["logits"].double().clone()
    of = lambda x, b: float(x[b]) if isinstance(x, torch.Tensor) else x  # noqa: E731
    for b in range(B):
        lo = 0 if s["first"] is None else int(s["first"][b])
        hi = int(s["lens"][b])
        cut = max(lo, 0 if s["n_prompt"] is None else int(s["n_prompt"][b]))
        every = torch.unique(s["tokens"][b, lo:hi])
        r = of(s["repetition"], b)
        z[b, every] = torch.where(z[b, every] > 0, z[b, every] / r, z[b, every] * r)
        late, times = torch.unique(s["tokens"][b, cut:hi], return_counts=True)
        z[b, late] -= of(s["frequency"], b) * times.double() + of(s["presence"], b)
        if s["bias"] is not None:
            z[b] += s["bias"].double()
        z[b] /= of(s["temperature"], b)
        if s["mask"] is not None:
            bits = (s["mask"][b][:, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
            z[b, bits.reshape(-1)[:V] == 0] = -math.inf
    return z
