"""PagedKVCache in use (prompts, steps, weights, evictions, a sequence that ends and
one that takes its place, pointer lists over the pages) against the oracle on rows
kept aside, and the decoder's token loop with penalties against its own logits."""
from __future__ import annotations

import pytest
import torch

from oracle import paged as OP
from tests.paged_inputs import assert_within, attn_bounds

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
def test_cache_in_use(dtype):
    from scope_amd import PagedKVCache

    B, Hq, Hkv, D, bs = 3, 4, 2, 64, 16
    g = torch.Generator().manual_seed(7)
    fp8 = dtype == torch.float8_e4m3fn
    scale = torch.tensor([0.02, 0.01]) if fp8 else None
    dev_scale = scale.to(DEV) if fp8 else None
    rows_t = torch.bfloat16 if fp8 else dtype
    c = PagedKVCache(pages=24, sequences=B, max_len=160, kv_heads=Hkv, head_dim=D, page_size=bs, dtype=dtype,
                     k_scale=dev_scale, v_scale=dev_scale)
    held = [[] for _ in range(B)]  # every row ever appended, by sequence

    def append(rows):
        n = sum(rows) if rows is not None else B
        k, v = (torch.randn((n, Hkv, D), generator=g).to(rows_t) for _ in range(2))
        c.append(k.to(DEV), v.to(DEV), rows)
        at = 0
        for b, m in enumerate(rows or [1] * B):
            held[b] += [(k[at + i], v[at + i]) for i in range(m)]
            at += m

    def check():
        q = torch.randn((B, Hq, D), generator=g).to(rows_t)
        before = c.mass.cpu()
        out, lse = c.attend(q.to(DEV), scale=0.12)
        assert [c.length(b) for b in range(B)] == [len(h) for h in held] == c.lens.tolist()
        # the oracle's pages hold the same rows in places of their own, where the cache still has a page
        table = c.table.cpu()
        pages = torch.full(table.shape, -1, dtype=torch.int32)
        pages[table >= 0] = torch.arange(int((table >= 0).sum()), dtype=torch.int32)
        kp, vp = (torch.zeros((max(1, int(pages.max()) + 1), Hkv, bs, D)).to(dtype) for _ in range(2))
        for b in range(B):
            if held[b]:
                k, v = (torch.stack(x) for x in zip(*held[b]))
                cu = torch.tensor([0, len(held[b])])
                kp = OP.append(k, kp, pages[b:b + 1], torch.zeros(1), cu, scale)
                vp = OP.append(v, vp, pages[b:b + 1], torch.zeros(1), cu, scale)
        r = OP.decode_attn(q, kp, vp, pages, torch.tensor([len(h) for h in held]), scale=0.12, k_scale=scale, v_scale=scale)
        b_out, b_lse, b_w = attn_bounds(rows_t, D, r)
        assert_within("lse", lse, r["lse"], b_lse)
        assert_within("out", out, r["out"], b_out)
        want = before.double() + r["weights"]
        assert_within("mass", c.mass, want, b_w + 2.0 ** -24 * want.abs())

    append([50, 0, 17])
    check()
    append([0, 33, 0])
    for step in range(20):
        append(None)
        check()
    assert c.free_pages == 24 - sum(-(-len(h) // bs) for h in held)
    freed = c.evict(3, window=1, n_global=1)
    assert freed == sum(max(0, -(-len(h) // bs) - 3) for h in held) and freed > 0
    assert all(int((row >= 0).sum()) <= 3 for row in c.table.cpu())
    for step in range(15):
        append(None)
        check()
    c.release(1)
    held[1] = []
    append([0, 40, 0])  # another takes its place, in pages that others left
    check()
    with pytest.raises(RuntimeError, match="positions of 160"):
        c.append(torch.zeros((160, Hkv, D), dtype=rows_t, device=DEV), torch.zeros((160, Hkv, D), dtype=rows_t, device=DEV), [160, 0, 0])


def test_calls_that_a_replay_would_not_repeat_are_refused(monkeypatch):
    from scope_amd import PagedKVCache

    c = PagedKVCache(pages=4, sequences=1, max_len=64, kv_heads=1, head_dim=64, page_size=16)
    x = torch.zeros((1, 1, 64), dtype=torch.bfloat16, device=DEV)
    c.append(x, x)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        for call in (lambda: c.append(x, x), lambda: c.append(x, x, [1]), lambda: c.reserve([3]), lambda: c.evict(1), lambda: c.release(0)):
            with pytest.raises(RuntimeError, match="on the host"):
                call()
    assert c.length(0) == 1 and c.free_pages == 3 and c.lens.tolist() == [1]


def test_pointer_lists_over_pages():
    """The pointer selection's lists of each sequence's newest block, attended to over shuffled pages; a page
    that eviction took is not seen though its block is listed."""
    from scope_amd import ops

    H, D, bs, nb, B = 4, 128, 128, 24, 2
    g = torch.Generator().manual_seed(9)
    P = B * nb
    table = torch.randperm(P, generator=g).reshape(B, nb).int()
    kp, vp = (torch.randn((P, H, bs, D), generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn((B, H, D), generator=g).to(torch.bfloat16)
    lens = torch.tensor([nb * bs - 5, nb * bs], dtype=torch.int32)
    nums, idxs = [], []
    for b in range(B):
        kbar = kp[table[b].long()].float().mean(2).transpose(0, 1).contiguous().to(DEV)  # [H, nb, D]
        qbar = torch.zeros((H, nb, D), device=DEV)
        qbar[:, -1] = q[b].float().to(DEV)
        docs = torch.zeros(nb * bs, dtype=torch.int32, device=DEV)
        ds_ptr, ds_local, _ = ops.doc_starts(docs, bs)
        kv_num, kv_idx, _ = ops.pointer_select(ds_ptr, ds_local, bs=bs, NB=nb, H=H, window=2, n_global=1, budget=4, qbar=qbar,
                                               kbar=kbar)
        nums.append(kv_num[:, -1])
        idxs.append(kv_idx[:, -1])
    kv_num, kv_idx = torch.stack(nums), torch.stack(idxs).contiguous()
    for gone in (False, True):
        if gone:
            table[0, 0], table[1, int(kv_idx[1, 0, 1])] = -1, -1
        mass = torch.zeros((B, H, nb), device=DEV)
        out, lse = ops.paged_decode_attn(q.to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV), lens.to(DEV), scale=0.12, kv_num=kv_num,
                                         kv_idx=kv_idx, mass=mass)
        r = OP.decode_attn(q, kp, vp, table, lens, scale=0.12, kv_num=kv_num.cpu(), kv_idx=kv_idx.cpu())
        b_out, b_lse, b_w = attn_bounds(torch.bfloat16, D, r)
        assert_within("lse", lse, r["lse"], b_lse)
        assert_within("out", out, r["out"], b_out)
        assert_within("mass", mass, r["weights"], b_w)


@pytest.mark.parametrize("use_graph", [False, True])
def test_generate_with_penalties(use_graph):
    """Each token is the argmax of the penalised logits of a decoder stepped by hand over the same tokens."""
    from scope_amd.decode import DecoderConfig, ScopeDecoder

    cfg = DecoderConfig(vocab_size=1000, num_layers=6, num_heads=2, model_dim=256, no_attn_layer=3)
    g = torch.Generator().manual_seed(3)
    prompt = torch.randint(0, 1000, (256,), generator=g)
    n = 20
    bias = torch.zeros(1000, device=DEV)
    bias[5] = -3.0
    mask = torch.full((32,), -1, dtype=torch.int32, device=DEV)
    mask[3] = 0  # words 96 .. 127
    kw = dict(repetition=1.2, presence=0.5, frequency=0.25, temperature=0.9, bias=bias, mask=mask)
    m = ScopeDecoder(cfg, max_len=512, seed=1, use_graph=use_graph)
    first = int(m.prefill(prompt.to(DEV))[:1000].argmax())
    got = m.generate(n, first, penalties=kw).tolist()
    m = ScopeDecoder(cfg, max_len=512, seed=1, use_graph=use_graph)
    m.prefill(prompt.to(DEV))
    fed, tokens = [first], prompt.tolist()
    for s in range(n):
        z = m.step(fed[-1])[:1000].cpu()[None]
        tokens.append(fed[-1])
        want = OP.penalties(z, torch.tensor(tokens), torch.tensor([len(tokens)]), n_prompt=torch.tensor([256]),
                            **{k: (x.cpu() if isinstance(x, torch.Tensor) else x) for k, x in kw.items()})[0]
        # (fp32 against fp64: the chosen word is within their difference of the best)
        assert want[got[s]] >= want.max() - 1e-4, f"step {s}"
        assert not 96 <= got[s] < 128
        fed.append(got[s])
    # without penalties the loop repeats sooner: the words are not the same
    m.prefill(prompt.to(DEV))
    assert m.generate(n, first).tolist() != got
