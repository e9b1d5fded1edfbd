"""Batches on a 4-bit cache for the tests: pools filled by the oracle's format, tables, lengths."""

import numpy as np
import torch

import oracle.fp4 as of
from femtovllm import fp4


def quantized(x):
    """(codes (..., 32 N) uint8, scale bytes (..., N) uint8) of rows x (..., D), on whole arrays."""
    n = of.blocks(x.shape[-1])
    y = np.zeros((*x.shape[:-1], 32 * n))
    y[..., : x.shape[-1]] = x
    y = y.reshape(*x.shape[:-1], n, 32)
    top = np.abs(y).max(-1)
    f, e = np.frexp(top)
    e = np.clip(np.where(top > 0, e - 3 + (f > 0.875), -119), -119, 125)
    a = np.abs(y) / 2.0 ** e[..., None].astype(float)
    code = ((a > 0.25).astype(np.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
            + 8 * np.signbit(y)).astype(np.uint8)
    return code.reshape(*x.shape[:-1], 32 * n), (e + 127).astype(np.uint8)


def pool_of(K, V):
    """Pool of rows K, V (num_blocks, n_kv_heads, 16, D) float64, finite."""
    D = K.shape[-1]
    n = of.blocks(D)
    P = 256 * n
    pool = np.zeros((*K.shape[:2], of.page_bytes(D)), dtype=np.uint8)
    (ck, sk), (cv, sv) = quantized(K), quantized(V)
    i, r, b = np.arange(16 * n), np.arange(16)[:, None], np.arange(n)
    pair = lambda c: c[..., 0::2] | (c[..., 1::2] << 4)
    pool[..., 256 * (i // 16) + 16 * r + i % 16] = pair(ck)
    pool[..., P + 64 * n * (r // 4) + 16 * (i // 4) + 4 * (r % 4) + i % 4] = pair(cv)
    pool[..., 2 * P + 4 * r + b] = sk
    pool[..., 2 * P + 64 + 16 * (r // 4) + 4 * b + r % 4] = sv
    return pool


def poison(pool, blk, rows, dim):
    """Rows of a page become NaN (scale bytes 255, codes of all ones)."""
    n = of.blocks(dim)
    P = 256 * n
    for r in rows:
        for b in range(4):
            pool[blk, :, 2 * P + 4 * r + b] = 255
            pool[blk, :, 2 * P + 64 + 16 * (r // 4) + 4 * b + r % 4] = 255


class Batch:
    """chunks: (cached, new) tokens of each sequence; every block that no sequence holds and every row behind a sequence's
    last token is NaN."""

    def __init__(self, chunks, n_heads, n_kv_heads, dim, dtype, seed, decode=False, scale=1.0, extra=3):
        rng = np.random.default_rng(seed)
        self.chunks, self.dim, self.dtype = chunks, dim, dtype
        lens = [p + n for p, n in chunks]
        pages = [-(-n // 16) for n in lens]
        num_blocks = sum(pages) + extra
        order = rng.permutation(num_blocks).tolist()
        K, V = (rng.standard_normal((num_blocks, n_kv_heads, 16, dim)) * np.exp(0.4 * rng.standard_normal((num_blocks, n_kv_heads, 16, 1)))
                for _ in range(2))
        self.pool = pool_of(K * scale, V)
        self.tables = np.full((len(chunks), max(max(pages), 1)), -1, dtype=np.int32)
        for b, m in enumerate(pages):
            self.tables[b, :m] = [order.pop() for _ in range(m)]
            if lens[b] % 16:
                poison(self.pool, self.tables[b, m - 1], range(lens[b] % 16, 16), dim)
        for blk in order:
            poison(self.pool, blk, range(16), dim)
        self.kv_lens = np.array(lens, dtype=np.int32)
        self.cu = np.cumsum([0] + [n for _, n in chunks]).astype(np.int32)
        self.pos = np.concatenate([np.arange(p, p + n) for p, n in chunks] + [np.zeros(0)]).astype(np.int32)
        tokens = len(chunks) if decode else int(self.cu[-1])
        g = torch.Generator().manual_seed(seed)
        self.q = torch.randn((n_heads, tokens, dim), generator=g).to(dtype)

    def on(self, device):
        t = lambda x: torch.tensor(x, device=device)
        return t(self.pool), t(self.tables), t(self.kv_lens), t(self.cu), t(self.pos), self.q.to(device)


def page_bytes(dim):
    return fp4.page_bytes(dim)
