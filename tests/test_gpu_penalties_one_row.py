"""One row of logits over a long token buffer, on the GPU against the oracle in 64
bits: histories that hold little of it, all of it, and everything on."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_penalties import check, full

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from scope_amd import ops

    return ops


@pytest.mark.parametrize("token", [torch.int32, torch.int64])
@pytest.mark.parametrize("held", [0, 1, 1152, 16385, 40001])
def test_one_row_over_a_long_buffer(ops, token, held):
    print(f"penalties one row, {held} held, {token}", flush=True)
    kw = full(1, 9001, 40001, held)
    kw.update(tokens=kw["tokens"].to(token), lens=torch.tensor([held]), first=torch.tensor([held // 7]), n_prompt=torch.tensor([held // 2 + 1]))
    check(ops, torch.randn((1, 9001), generator=torch.Generator().manual_seed(held)) * 5, **kw)
