"""Writes and reads of one long prompt over the 4-bit cache: the walk through its table, past 64 and 256 columns, and where it
ends."""

import numpy as np
import pytest
import torch

from femtovllm import fp4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first,tokens", [(0, 1024), (0, 1025), (5, 4090), (0, 4096), (0, 4097), (37, 16500)])
def test_one_prompt(ops, gpu, first, tokens):
    """As many sequences of a page each; a column that ends the walk, or a table that does, leaves what is behind it."""
    g = torch.Generator().manual_seed(tokens)
    k, v = (torch.randn((tokens, 1, 32), generator=g).to(torch.bfloat16).to(gpu) for _ in range(2))
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=gpu)
    cols = -(-(first + tokens) // 16)
    table = torch.randperm(cols + 7, generator=g)[:cols].to(torch.int32)
    start = torch.randint(0, 100, (cols + 7, 1, fp4.page_bytes(32)), generator=g, dtype=torch.uint8).to(gpu)
    pos = np.arange(first, first + tokens)
    ends = [16 * c for c in range(first // 16 + 1, cols)]
    cu_pages = i32([0] + [e - first for e in ends] + [tokens])
    # page by page: each sequence's first token is at its own position of a table of its own
    want = start.clone()
    rows = torch.stack([torch.where(torch.arange(cols) == c, table, table) for c in range(first // 16, cols)]).to(gpu)
    ops.kv_cache_write_fp4(k, v, want, i32(pos), rows, cu_pages, 16)
    got = start.clone()
    cu = i32([0, tokens])
    ops.kv_cache_write_fp4(k, v, got, i32(pos), table[None].to(gpu), cu, tokens)
    assert torch.equal(got, want) and not torch.equal(got, start)
    whole = ops.kv_cache_read_fp4(got, 32, torch.bfloat16, i32(pos), table[None].to(gpu), cu, tokens)
    for c in sorted({c for c in (first // 16, 63, 64, 65, 255, 256, 257, 511, 512, 700, cols - 1) if first // 16 <= c < cols}):
        seen = max(0, 16 * c - first)
        for how in ("hole", "outside", "short"):
            t = table.clone()
            if how == "short":
                t = t[:c]
            else:
                t[c] = -1 if how == "hole" else cols + 7
            pool = start.clone()
            ops.kv_cache_write_fp4(k, v, pool, i32(pos), t[None].to(gpu), cu, tokens)
            kept = table[:c].long().to(gpu)
            left = torch.ones(cols + 7, dtype=torch.bool, device=gpu)
            left[kept] = False
            assert torch.equal(pool[kept], want[kept]) and torch.equal(pool[left], start[left]), (c, how)
            for x, y in zip(ops.kv_cache_read_fp4(want, 32, torch.bfloat16, i32(pos), t[None].to(gpu), cu, tokens), whole):
                assert torch.equal(x[:seen], y[:seen]) and not x[seen:].any(), (c, how)
