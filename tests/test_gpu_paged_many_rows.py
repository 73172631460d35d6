"""More appended rows than one row or two a wavefront leave a grid for, on the GPU."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_rows_past_the_largest_grid_of_two_a_wavefront():
    """2^27 + 3 rows (one row's memory, expanded), of which a few blocks have a page."""
    from scope_amd import ops

    N, bs, held = 2 ** 27 + 3, 256, 5
    MP = -(-(N + held) // bs)
    print(f"append of {N} rows", flush=True)
    table = torch.full((1, MP), -1, dtype=torch.int32, device=DEV)
    blocks = [0, 1, MP // 3, MP - 2, MP - 1]
    table[0, torch.tensor(blocks, device=DEV)] = torch.arange(len(blocks), dtype=torch.int32, device=DEV)
    row = torch.randn((1, 1, 64), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    kp, vp = (torch.zeros((len(blocks) + 1, 1, bs, 64), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    ops.paged_append(row.expand(N, 1, 64), (-row).expand(N, 1, 64), kp, vp, table, torch.tensor([held], device=DEV),
                     cu=torch.tensor([0, N], dtype=torch.int32, device=DEV))
    pos = torch.tensor(blocks)[:, None] * bs + torch.arange(bs)
    written = ((pos >= held) & (pos < N + held)).to(DEV)
    for pages, x in ((kp, row[0, 0]), (vp, -row[0, 0])):
        got = pages[:len(blocks), 0]
        assert torch.equal(got[written], x.expand(int(written.sum()), 64)) and not got[~written].any()
        assert not pages[len(blocks)].any()
