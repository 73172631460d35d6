"""A paged key-value cache for decoding several sequences, over the operators of
``scope_amd.ops``: the pool of pages, the page table and the lengths of one
attention layer.

    cache = PagedKVCache(pages=4096, sequences=8, max_len=131072, kv_heads=8, head_dim=128)
    cache.append(k, v, rows=[1000, 17, 0, 0, 0, 0, 0, 0])    # prompts, ragged
    cache.append(k, v)                                       # one row a sequence
    out, lse = cache.attend(q, scale=0.12)                   # weights accumulate
    k, v = cache.read()                                      # every row that is held, for a dense attention
    cache.evict(512, window=4, n_global=1)                   # back to 512 pages a sequence
    cache.release(3)                                         # a sequence ends

The reference has no decode path and no cache.  Pages are taken from the pool
when a sequence grows into them, on the host, whose copy of the lengths needs no
reading back; ``evict`` reads the table back to know what it freed.  ``attend``
never waits for the GPU.  ``append`` waits where it takes pages and wherever it is
given ``rows``: the new table entries and the counts are copied from pageable host
memory; a step (no ``rows``) within the pages taken does not.  A cache is used on one
stream at a time: a page goes from one sequence to another in stream order.
``attend`` may be captured into a graph; the calls that also change the host's
copy, or go by it (``read``), which a replay would not, raise there.
"""
from __future__ import annotations

import torch

from . import ops


class PagedKVCache:
    """Keys and values of one attention layer in pages of ``page_size`` positions.

    ``pages`` the pool holds, for ``sequences`` sequences of up to ``max_len``
    positions each.  ``dtype``: bfloat16 or float16, or float8_e4m3fn with
    ``k_scale`` / ``v_scale`` [kv_heads] fp32 (value = stored · scale; None: 1),
    or float4_e2m1fn_x2, whose scales (a power of two for 32 features) are formed
    as rows are written: 68 bytes for a row of 128 features.

    k_pages, v_pages [pages, kv_heads, page_size, head_dim] (4 bits: head_dim / 2,
    with k_scale, v_scale [pages, kv_heads, page_size, head_dim / 32]
    float8_e8m0fnu), table [sequences, max pages] int32 (-1: no page), lens
    [sequences] int32 and mass [sequences, kv_heads, max pages] fp32 live on the
    device and may be handed to ``ops.paged_*`` directly; they keep their addresses."""

    def __init__(self, *, pages: int, sequences: int, max_len: int, kv_heads: int, head_dim: int, page_size: int = 128,
                 dtype: torch.dtype = torch.bfloat16, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None, device="cuda"):
        if pages < 1 or sequences < 1 or max_len < 1:
            raise ValueError(f"PagedKVCache: pages={pages}, sequences={sequences} and max_len={max_len} must be at least 1")
        self.page_size, self.max_len = page_size, max_len
        width = -(-max_len // page_size)
        if dtype == torch.float4_e2m1fn_x2:
            if k_scale is not None or v_scale is not None:
                raise ValueError("PagedKVCache: 4-bit pages form their scales themselves")
            if head_dim % 32:
                raise ValueError(f"PagedKVCache: 4-bit pages need a head dim that is a multiple of 32, got {head_dim}")
            k_scale, v_scale = (torch.zeros((pages, kv_heads, page_size, head_dim // 32), dtype=torch.uint8,
                                            device=device).view(torch.float8_e8m0fnu) for _ in range(2))
            self.k_pages, self.v_pages = (torch.zeros((pages, kv_heads, page_size, head_dim // 2), dtype=torch.uint8,
                                                      device=device).view(dtype) for _ in range(2))
        else:
            self.k_pages, self.v_pages = (torch.zeros((pages, kv_heads, page_size, head_dim), dtype=dtype, device=device)
                                          for _ in range(2))
        self.k_scale, self.v_scale = k_scale, v_scale
        self.table = torch.full((sequences, width), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(sequences, dtype=torch.int32, device=device)
        self.mass = torch.zeros((sequences, kv_heads, width), dtype=torch.float32, device=device)
        self._free = list(range(pages - 1, -1, -1))  # taken from the end: the lowest first
        self._len = [0] * sequences
        self._pages: list[dict[int, int]] = [{} for _ in range(sequences)]  # block -> page

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, sequence: int) -> int:
        return self._len[sequence]

    def _on_host(self, what: str, does: str = "changes lengths or pages on the host, which a replayed graph would not") -> None:
        if self.table.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"PagedKVCache: {what} {does}; capture the operators of scope_amd.ops instead")

    def reserve(self, rows) -> None:
        """Takes the pages that rows[b] more positions of each sequence b need;
        raises before it takes any if the pool or a sequence's table is too short."""
        self._on_host("reserve")
        if len(rows) != len(self._len) or any(n < 0 for n in rows):
            raise ValueError(f"PagedKVCache: rows must be {len(self._len)} numbers of at least 0, got {list(rows)}")
        want = []
        for b, n in enumerate(rows):
            end = self._len[b] + n
            if n and end > self.max_len:
                raise RuntimeError(f"PagedKVCache: sequence {b} would hold {end} positions of {self.max_len}")
            # (a block that eviction emptied gets no page again: it never holds the newest position)
            want += [(b, i) for i in range(self._len[b] // self.page_size, -(-end // self.page_size))
                     if n and i not in self._pages[b]]
        if len(want) > len(self._free):
            raise RuntimeError(f"PagedKVCache: {len(want)} pages needed, {len(self._free)} free: evict or release first")
        if not want:
            return
        taken = [(b, i, self._free.pop()) for b, i in want]
        for b, i, page in taken:
            self._pages[b][i] = page
        at = torch.tensor(taken, dtype=torch.int64).to(self.table.device)
        self.table[at[:, 0], at[:, 1]] = at[:, 2].to(torch.int32)

    def append(self, k: torch.Tensor, v: torch.Tensor, rows=None) -> None:
        """Appends k, v [N, kv_heads, head_dim]: rows[b] of them, in order, to each
        sequence b (their sum is N), or without ``rows`` one to every sequence."""
        self._on_host("append")
        B = len(self._len)
        one_each = rows is None
        rows = [1] * B if one_each else [int(n) for n in rows]
        if k.shape[0] != sum(rows):
            raise ValueError(f"PagedKVCache: {k.shape[0]} rows given, {sum(rows)} announced")
        self.reserve(rows)
        if one_each:
            ops.paged_append(k, v, self.k_pages, self.v_pages, self.table, self.lens, k_scale=self.k_scale, v_scale=self.v_scale)
            self.lens.add_(1)
        else:
            n = torch.tensor([rows], dtype=torch.int32).to(self.lens.device)[0]
            cu = torch.cat((n.new_zeros(1), n.cumsum(0, dtype=torch.int32)))
            ops.paged_append(k, v, self.k_pages, self.v_pages, self.table, self.lens, cu=cu, k_scale=self.k_scale,
                             v_scale=self.v_scale)
            self.lens.add_(n)
        self._len = [a + b for a, b in zip(self._len, rows)]

    def attend(self, q: torch.Tensor, *, scale: float, first: torch.Tensor | None = None,
               kv_num: torch.Tensor | None = None, kv_idx: torch.Tensor | None = None, accumulate: bool = True):
        """``ops.paged_decode_attn`` of q [sequences, heads, head_dim] over the cache
        -> (out, lse); with ``accumulate`` the blocks' weights are added to ``mass``."""
        return ops.paged_decode_attn(q, self.k_pages, self.v_pages, self.table, self.lens, scale=scale, first=first,
                                     kv_num=kv_num, kv_idx=kv_idx, mass=self.mass if accumulate else None,
                                     k_scale=self.k_scale, v_scale=self.v_scale)

    def read(self, rows=None, first=None, *, dtype: torch.dtype | None = None):
        """The rows of the ``rows[b]`` positions from first[b] on of each sequence b, one
        sequence after the other -> k, v [sum(rows), kv_heads, head_dim] of ``dtype``
        (``ops.paged_read``; 16-bit pages in their own).  ``first`` may be one number
        for all, None is 0; ``rows`` of None is what each sequence holds from there on;
        positions whose page was evicted are zeros.  The numbers are the host's: nothing
        waits for the GPU but their copy from pageable memory."""
        self._on_host("read", "goes by the lengths on the host, which a replayed graph would not see change")
        B = len(self._len)
        first = 0 if first is None else first.tolist() if isinstance(first, torch.Tensor) else first
        first = [int(n) for n in first] if hasattr(first, "__iter__") else [int(first)] * B
        rows = [max(0, n - f) for n, f in zip(self._len, first)] if rows is None else [int(n) for n in rows]
        if len(first) != B or len(rows) != B or any(f < 0 or n < 0 or (n and f + n > held) for f, n, held in zip(first, rows, self._len)):
            raise ValueError(f"PagedKVCache: rows {rows} from {first} on are not held ({self._len})")
        # (where no row is read, first may be any number)
        at, n = torch.tensor([[f if n else 0 for f, n in zip(first, rows)], rows], dtype=torch.int32).to(self.lens.device)
        cu = torch.cat((n.new_zeros(1), n.cumsum(0, dtype=torch.int32)))
        return ops.paged_read(self.k_pages, self.v_pages, self.table, self.lens, rows=sum(rows), cu=cu, first=at,
                              k_scale=self.k_scale, v_scale=self.v_scale, dtype=dtype)

    def evict(self, budget, *, window: int = 1, n_global: int = 0) -> int:
        """Brings every sequence back to ``budget`` pages (a number or int [sequences])
        by ``ops.paged_evict`` on the accumulated weights; returns how many pages
        went back to the pool.  Waits for the GPU."""
        self._on_host("evict")
        ops.paged_evict(self.table, self.mass, self.lens, budget, bs=self.page_size, window=window, n_global=n_global,
                        out=self.table)
        count = 0
        for held, row in zip(self._pages, self.table.tolist()):
            for i in [i for i in held if row[i] < 0]:
                self._free.append(held.pop(i))
                count += 1
        return count

    def release(self, sequence: int) -> None:
        """Ends a sequence: its pages go back to the pool, its length and weights to 0."""
        self._on_host("release")
        held = self._pages[sequence]
        self._free += [held[i] for i in sorted(held, reverse=True)]
        held.clear()
        self._len[sequence] = 0
        self.table[sequence].fill_(-1)
        self.lens[sequence].zero_()
        self.mass[sequence].zero_()
