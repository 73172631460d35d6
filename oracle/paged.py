"""The paged cache and the logit penalties of a decode loop, in plain torch and
64 bits, one sequence and one head at a time.  The reference has no decode path:
these are the definitions that the kernels are held to."""
from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0


def values(pages: torch.Tensor, scale: torch.Tensor | None) -> torch.Tensor:
    """The numbers that pages [P, Hkv, bs, D] stand for, fp64."""
    x = pages if pages.dtype == torch.float64 else pages.float().double()
    return x if scale is None else x * scale.double()[:, None, None]


# ---- 4 bits: groups of 32 features as e2m1 codes with one e8m0 scale ----------------
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
GROUP = 32
SCALE_MIN, SCALE_MAX = -125, {torch.bfloat16: 125, torch.float16: 13}  # powers of two that are written


def quantise_group(x) -> tuple[list[int], int]:
    """(codes, scale byte) of one group's 16-bit values, by the definition: Python's
    exact floats, each code the nearest grid value, the even code of two."""
    top = SCALE_MAX[x.dtype]
    v = [float(f) for f in x.double()]
    if not all(math.isfinite(f) for f in v):
        return [0] * len(v), 255
    a = max(abs(f) for f in v)
    e = SCALE_MIN
    if a > 0:
        low = math.frexp(a)[1] - 1
        e = low - 1 if a >= 1.75 * 2.0 ** low else low - 2
    e = min(max(e, SCALE_MIN), top)
    codes = []
    for f in v:
        y = abs(f) / 2.0 ** e
        best = min(range(8), key=lambda c: (abs(E2M1[c] - y), c % 2))
        codes.append(best + (8 if math.copysign(1.0, f) < 0 else 0))
    return codes, e + 127


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(bytes [..., D / 2], scale bytes [..., D / 32]) of 16-bit rows [..., D]: the even
    feature in the low nibble.  The definition of quantise_group, over tensors in fp64."""
    y = x.double().reshape(*x.shape[:-1], -1, GROUP)
    bad = ~torch.isfinite(y).all(-1)
    y = torch.where(bad[..., None], 0.0, y)
    a = y.abs().amax(-1)
    m, e = torch.frexp(a)
    e = torch.where(a > 0, e - 3 + (m >= 0.875).int(), SCALE_MIN).clamp(SCALE_MIN, SCALE_MAX[x.dtype])
    z = torch.ldexp(y, -e[..., None])
    grid = torch.tensor(E2M1, dtype=torch.float64)
    edges = (grid[1:] + grid[:-1]) / 2
    code = torch.bucketize(z.abs().contiguous(), edges)  # (on an edge the lower code)
    on = (code < 7) & (z.abs() == edges[code.clamp(max=6)])
    code = code + (on & (code % 2 == 1)).long() + 8 * torch.signbit(z).long()
    code = torch.where(bad[..., None], 0, code).reshape(*x.shape[:-1], -1, 2)
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), torch.where(bad, 255, e + 127).to(torch.uint8)


def e2m1_values(pages: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """The numbers that 4-bit pages [..., D / 2] with scales [..., D / 32] stand for, fp64."""
    b, s = pages.view(torch.uint8).long(), scale.view(torch.uint8).double()
    code = torch.stack((b % 16, b // 16), -1).flatten(-2)
    x = torch.tensor(E2M1 + [-f for f in E2M1], dtype=torch.float64)[code]
    return x * torch.where(s == 255, math.nan, 2.0 ** (s - 127)).repeat_interleave(GROUP, -1)


def append_e2m1(x, pages, scale, table, lens, cu=None):
    """(pages, scales) after the rows x were quantised into them."""
    q, s = quantise(x)
    return tuple(append(r, t.view(torch.uint8), table, lens, cu).view(t.dtype) for r, t in ((q, pages), (s, scale)))


def read(vals: torch.Tensor, table, lens, rows, cu=None, first=None) -> torch.Tensor:
    """Rows [rows, Hkv, D] out of pages of values [P, Hkv, bs, D], one at a time."""
    P, Hkv, bs, D = vals.shape
    B, MP = table.shape
    out = torch.zeros((rows, Hkv, D), dtype=vals.dtype)
    for b in range(B):
        r0, r1 = (b, b + 1) if cu is None else (int(cu[b]), int(cu[b + 1]))
        for i in range(max(r0, 0), min(r1, rows)):
            pos = (0 if first is None else int(first[b])) + i - r0
            if 0 <= pos < min(int(lens[b]), MP * bs) and 0 <= int(table[b, pos // bs]) < P:
                out[i] = vals[int(table[b, pos // bs]), :, pos % bs]
    return out


def append(x, pages, table, lens, cu=None, scale=None) -> torch.Tensor:
    """Pages after the rows x [N, Hkv, D] were written, by sequence and row."""
    P, _, bs, _ = pages.shape
    B, MP = table.shape
    out = pages.clone()
    raw = out.view(torch.uint8) if out.dtype == torch.float8_e4m3fn else out
    for b in range(B):
        r0, r1 = (b, b + 1) if cu is None else (int(cu[b]), int(cu[b + 1]))
        for i in range(max(r0, 0), min(r1, x.shape[0])):
            pos = int(lens[b]) + i - r0
            if not 0 <= pos < MP * bs:
                continue
            page = int(table[b, pos // bs])
            if not 0 <= page < P:
                continue
            row = x[i]
            if out.dtype == torch.float8_e4m3fn:
                s = torch.ones(x.shape[1]) if scale is None else scale
                row = (row.float() / s[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
            raw[page, :, pos % bs] = row
    return out


def seen_positions(table_row, length, first, P, bs, blocks=None) -> list[tuple[int, int, int]]:
    """(position, block, page) of every key that a new token sees, in list order."""
    MP = table_row.numel()
    end = min(max(int(length), 0), MP * bs)
    got = []
    for i in (range(MP) if blocks is None else blocks):
        if not 0 <= i < MP or not 0 <= int(table_row[i]) < P:
            continue
        got += [(j, i, int(table_row[i])) for j in range(i * bs, (i + 1) * bs) if max(int(first), 0) <= j < end]
    return got


def decode_attn(q, k_pages, v_pages, table, lens, *, scale, first=None, kv_num=None, kv_idx=None, k_scale=None,
                v_scale=None):
    """dict of out [B, Hq, D], lse [B, Hq] and weights [B, Hkv, MP], and of what
    error bounds are made of: spread = Σ p|v| and total = Σ|v| [B, Hq, D], size =
    max over the seen keys of |scale|·Σ|q_d k_d| [B, Hq]; all fp64."""
    q = q.double()
    B, Hq, D = q.shape
    P, Hkv, bs, _ = k_pages.shape
    MP = table.shape[1]
    G = Hq // Hkv
    k, v = values(k_pages, k_scale), values(v_pages, v_scale)
    out = torch.zeros((B, Hq, D), dtype=torch.float64)
    spread, total = torch.zeros((B, Hq, D), dtype=torch.float64), torch.zeros((B, Hq, D), dtype=torch.float64)
    size = torch.zeros((B, Hq), dtype=torch.float64)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64)
    weights = torch.zeros((B, Hkv, MP), dtype=torch.float64)
    for b in range(B):
        for hk in range(Hkv):
            blocks = None
            if kv_idx is not None:
                n = min(max(int(kv_num[b, hk]), 0), kv_idx.shape[-1])
                blocks = kv_idx[b, hk, :n].tolist()
            got = seen_positions(table[b], lens[b], 0 if first is None else first[b], P, bs, blocks)
            if not got:
                continue
            j, blk, page = (torch.tensor(x) for x in zip(*got))
            kk, vv = k[page, hk, j % bs], v[page, hk, j % bs]
            for h in range(hk * G, (hk + 1) * G):
                s = scale * (kk @ q[b, h])
                p = torch.softmax(s, 0)
                out[b, h], lse[b, h], spread[b, h] = p @ vv, torch.logsumexp(s, 0), p @ vv.abs()
                total[b, h] = vv.abs().sum(0)
                size[b, h] = abs(scale) * (kk.abs() @ q[b, h].abs()).max()
                weights[b, hk].index_add_(0, blk, p)
    return dict(out=out, lse=lse, weights=weights, spread=spread, total=total, size=size)


def evict(table, mass, lens, budget, *, bs, window=1, n_global=0):
    """(table, freed, n_freed), by sorting each sequence's pages."""
    B, MP = table.shape
    new, freed, num = table.clone(), torch.full_like(table, -1), torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        n = min(max((int(lens[b]) + bs - 1) // bs, 0), MP)
        held = [i for i in range(n) if int(table[b, i]) >= 0]
        may = [i for i in held if n_global <= i < n - window]
        score = mass[b].double().sum(0).float()
        may.sort(key=lambda i: (math.isnan(score[i]), 0.0 if math.isnan(score[i]) else float(score[i]), i))
        go = sorted(may[:max(0, len(held) - max(int(budget[b]), 0))])
        for at, i in enumerate(go):
            freed[b, at] = table[b, i]
            new[b, i] = -1
        num[b] = len(go)
    return new, freed, num


def penalties(logits, tokens, lens, *, first=None, n_prompt=None, repetition=1.0, presence=0.0, frequency=0.0,
              temperature=1.0, bias=None, mask=None):
    """Logits [B, V] after the penalties, fp64, by word and sequence."""
    B, V = logits.shape
    z = logits.double().clone()

    def of(x, b, default=0):
        return default if x is None else x[b].item() if isinstance(x, torch.Tensor) and x.dim() else x

    for b in range(B):
        row = tokens if tokens.dim() == 1 else tokens[b]
        lo, hi = max(int(of(first, b)), 0), min(int(of(lens, b)), row.numel())
        cut, r, f = int(of(n_prompt, b)), float(of(repetition, b)), float(of(frequency, b))
        seen, count = set(), {}
        for j in range(lo, max(lo, hi)):
            t = int(row[j])
            if 0 <= t < V:
                seen.add(t)
                if j >= cut:
                    count[t] = count.get(t, 0) + 1
        for t in seen:
            z[b, t] = z[b, t] / r if z[b, t] > 0 else z[b, t] * r
        for t, c in count.items():
            z[b, t] -= f * c + float(of(presence, b))
        if bias is not None:
            z[b] += (bias if bias.dim() == 1 else bias[b]).double()
        z[b] /= float(of(temperature, b))
        if mask is not None:
            words = mask if mask.dim() == 1 else mask[b]
            for v in range(V):
                if not (int(words[v // 32]) >> (v % 32)) & 1:
                    z[b, v] = -math.inf
    return z
