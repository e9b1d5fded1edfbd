"""The operators as a serving loop uses them, one after the other on one cache.

A chunk's keys are rotated into the pages and attend under the window, then tokens are decoded one at a time, then
many sequences go on from that text as their common prefix.  Each operator is checked against the 64-bit oracle on what
the ones before it left in the pools, within its own bounds (test_rope_gpu.py, helpers.assert_close); the pools
themselves against the oracle's rotation.
"""

import numpy as np
import pytest
import torch

import oracle.added as added
from femtovllm.rope import scaled_rope_tables
from helpers import assert_close, np32, np64
from test_rope_gpu import check_rotated

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
H, KVH, D, PAGE = 8, 2, 128, 16


class Cache:
    def __init__(self, blocks, dtype, device):
        self.k = torch.full((blocks, KVH, PAGE, D), float("nan"), dtype=dtype, device=device)
        self.v = torch.full_like(self.k, float("nan"))


def draw(gen, tokens, heads, dtype):
    return torch.randn((tokens, heads, D), generator=gen).to(dtype)


def i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_chunk_then_tokens_then_common_prefix(ops, gpu, dtype, interleaved):
    window, sinks = 150, 4
    gen = torch.Generator().manual_seed(int(interleaved))
    tables = scaled_rope_tables(2048, 64, base=10000.0)
    cos, sin = (t.to(gpu) for t in tables)
    cos64, sin64 = (t.numpy() for t in tables)
    cache = Cache(120, dtype, gpu)
    order = np.random.default_rng(1).permutation(120)
    table = [order[:40].tolist(), order[40:60].tolist()]
    pages = i32([t + [-1] * (40 - len(t)) for t in table], gpu)

    def write(counts, starts):
        """Rotates a step's rows into the cache -> (q as (H, T, D), positions, cu_seqlens)."""
        n = sum(counts)
        q, k, v = draw(gen, n, H, dtype), draw(gen, n, KVH, dtype), draw(gen, n, KVH, dtype)
        pos = np.concatenate([np.arange(s, s + c) for s, c in zip(starts, counts)])
        cu = np.concatenate([[0], np.cumsum(counts)])
        got = ops.rope_cache_write(q.to(gpu), k.to(gpu), v.to(gpu), cos, sin, i32(pos, gpu), cache.k, cache.v, pages,
                                   cu_seqlens=i32(cu, gpu), max_q_len=max(counts), interleaved=interleaved)
        check_rotated(got, q, cos64, sin64, pos, interleaved, "q")
        for b in range(2):
            t = slice(cu[b], cu[b + 1])
            blocks = [table[b][p // PAGE] for p in pos[t]]
            rows = [p % PAGE for p in pos[t]]
            check_rotated(cache.k[blocks, :, rows], k[t], cos64, sin64, pos[t], interleaved, "k")
            assert torch.equal(cache.v[blocks, :, rows].cpu(), v[t])
        return got.transpose(0, 1), i32(pos, gpu), i32(cu, gpu)

    # chunks of two prompts, the second call behind the first
    done = [0, 0]
    for counts in ([333, 20], [64, 200]):
        q, pos, cu = write(counts, done)
        done = [a + c for a, c in zip(done, counts)]
        out = ops.paged_attention_gemm_window(q, cache.k, cache.v, cu, max(counts), pages, i32(done, gpu), pos, window, sinks)
        want = added.window_prefill(np64(q), np32(cache.k), np32(cache.v), cu.tolist(), pages.cpu().numpy(), done,
                                    pos.cpu().numpy(), window, sinks)
        assert_close(out, want, dtype, f"chunks {counts}")
    # one token each
    for _ in range(3):
        q, pos, cu = write([1, 1], done)
        done = [a + 1 for a in done]
        out = ops.paged_attention_gemv_window(q, cache.k, cache.v, pages, i32(done, gpu), max(done), window, sinks)
        want = added.window_decode(np64(q), np32(cache.k), np32(cache.v), pages.cpu().numpy(), done, window, sinks)
        assert_close(out, want, dtype, "token")
    # five sequences go on from the first 24 pages of the first one, each with pages of its own
    own = [[-1] * 24 + order[60 + 4 * b : 64 + 4 * b].tolist() for b in range(5)]
    many, lens = i32(own, gpu), [24 * PAGE + b + 1 for b in range(5)]
    for b in range(5):  # the tails' tokens, one call a sequence
        c = lens[b] - 24 * PAGE
        q, k, v = draw(gen, c, H, dtype), draw(gen, c, KVH, dtype), draw(gen, c, KVH, dtype)
        whole = torch.cat([pages[:1, :24], many[b : b + 1, 24:]], dim=1)
        ops.rope_cache_write(q.to(gpu), k.to(gpu), v.to(gpu), cos, sin, i32(range(24 * PAGE, lens[b]), gpu), cache.k, cache.v,
                             whole, cu_seqlens=i32([0, c], gpu), max_q_len=c, interleaved=interleaved)
    q = draw(gen, 5, H, dtype).to(gpu).transpose(0, 1)
    out = ops.paged_attention_gemv_shared_prefix(q, cache.k, cache.v, pages[0, :24].contiguous(), many, i32(lens, gpu), max(lens))
    want = added.shared_prefix_decode(np64(q), np32(cache.k), np32(cache.v), table[0][:24], np.array(own), lens)
    assert_close(out, want, dtype, "common prefix")
    # the same keys through whole tables and a window past every context: two operators, one result
    whole = torch.cat([pages[:1, :24].expand(5, -1), many[:, 24:]], dim=1).contiguous()
    same = ops.paged_attention_gemv_window(q, cache.k, cache.v, whole, i32(lens, gpu), max(lens), 10000, 0)
    assert_close(same, want, dtype, "whole tables")


def test_captured_step_replayed_token_by_token(ops, gpu):
    """A graph of (rotate and write, attend) replayed with moving positions and new inputs: each replay equals the
    eager step on a copy of the cache."""
    tables = [t.to(gpu) for t in scaled_rope_tables(1024, 128)]
    gen = torch.Generator().manual_seed(3)
    caches = [Cache(100, BF16, gpu) for _ in range(2)]
    for c in caches:
        c.k.zero_()
        c.v.zero_()
    pages = torch.arange(90, dtype=torch.int32, device=gpu).view(3, 30)
    fixed = [t.to(gpu) for t in (draw(gen, 3, H, BF16), draw(gen, 3, KVH, BF16), draw(gen, 3, KVH, BF16))]
    pos = i32([400, 14, 0], gpu)
    lens = pos + 1

    def step(c, q, k, v, pos, lens):
        q = ops.rope_cache_write(q, k, v, *tables, pos, c.k, c.v, pages)
        return ops.paged_attention_gemv_window(q.transpose(0, 1), c.k, c.v, pages, lens, 480, 385, 2)

    step(caches[0], *fixed, pos, lens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(caches[0], *fixed, pos, lens)
    caches[1].k.copy_(caches[0].k)
    caches[1].v.copy_(caches[0].v)
    for _ in range(5):
        for t in fixed:
            t.copy_(draw(gen, *t.shape[:2], BF16))
        g.replay()
        want = step(caches[1], *(t.clone() for t in fixed), pos.clone(), lens.clone())
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)
        pos += 1
        lens += 1
