"""Numbers past 32 bits as budgets, lengths and positions, on the GPU: as tensors of them."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_numbers_as_tensors_of_them():
    from scope_amd import PagedKVCache, ops

    g = torch.Generator().manual_seed(1)
    table = torch.arange(2 * 40, dtype=torch.int32, device=DEV).reshape(2, 40)
    mass, lens = torch.rand((2, 1, 40), generator=g).to(DEV), torch.tensor([640, 300], device=DEV)
    for budget in (2 ** 63 - 1, 2 ** 32 + 1, -2 ** 40, 5):
        a = ops.paged_evict(table, mass, lens, budget, bs=16)
        b = ops.paged_evict(table, mass, lens, torch.full((2,), budget, device=DEV), bs=16)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    logits, tokens = torch.randn((2, 100), generator=g).to(DEV), torch.randint(0, 100, (2, 30), generator=g).to(DEV)
    for kw in (dict(n_prompt=2 ** 63 - 1), dict(first=2 ** 32), dict(first=-2 ** 32 - 1, n_prompt=-2 ** 40)):
        a = ops.logit_penalties(logits, tokens, 2 ** 40, frequency=1.0, repetition=1.5, **kw)
        b = ops.logit_penalties(logits, tokens, torch.full((2,), 2 ** 40, device=DEV), frequency=1.0, repetition=1.5,
                                **{k: torch.full((2,), x, device=DEV) for k, x in kw.items()})
        assert torch.equal(a, b)
    c = PagedKVCache(pages=4, sequences=1, max_len=64, kv_heads=1, head_dim=64, page_size=16)
    x = torch.zeros((40, 1, 64), dtype=torch.bfloat16, device=DEV)
    c.append(x, x, [40])
    assert c.evict(2 ** 40) == 0 and c.free_pages == 1
