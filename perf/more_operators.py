"""Measured cases of the operators of ``femtovllm.ops`` on a KV cache held in 4 bits.

Each case is a dict of plain values.  ``kind`` names the entry point:

* ``write``    ``ops.kv_cache_write_fp4``: the new K and V rows of a step, rounded to 4 bits, into the paged cache;
* ``rope``     ``ops.rope_cache_write_fp4``: the norms and rotation of q and k (``norm`` says whether there are norms)
  and the same write;
* ``decode``   ``ops.paged_attention_gemv_fp4``: one query token per sequence over that cache;
* ``prefill``  ``ops.paged_attention_gemm_fp4``: chunks of new tokens after cached prefixes, causal, with or without
  decode rows in the same call.

The two writes also read their tokens back (``ops.kv_cache_read_fp4``, which thereby is measured with them): what the
cache holds in 4 bits comes back as the values it stands for.

The cache: ``kv_pool`` (num_blocks, n_kv_heads, page_bytes) uint8, a page being 16 tokens of K and V of one head.  Dims
are in blocks of 32 (the last may be half full, zeros behind it), N = ceil(dim / 32) of them.  Each (token, block) has
one scale 2^(byte - 127) and 32 signed values of {0, 0.5, 1, 1.5, 2, 3, 4, 6} times it, 4 bits each: bit 3 the sign,
bits 0-2 the index in that list.  With R the token's row in the page and P = 256 N,

* K, block b, dims 32 b + 2 i (low half of the byte) and + 1 (high): byte 256 b + 16 R + i;
* V, dims 8 c + 2 i and + 1: byte P + (R // 4) * 64 N + 16 c + 4 (R % 4) + i;
* K's scale of block b: byte 2 P + 4 R + b; V's: byte 2 P + 64 + 16 (R // 4) + 4 b + R % 4;
* page_bytes = 2 P + 128.

The scale is the smallest power of two for which the block's largest magnitude is at most 7 of it (so that none is more
than half a step off), from 2^-119 to 2^125; values round to the nearest of the list, ties to the even index, magnitudes
past 6 to 6; a block that holds an infinity or a NaN has the scale byte 255 and zeros, and stands for NaN.

A paged batch is ``chunks`` (text, "cached+new ..."), or ``seqs`` chunks (``new_min..new_max`` tokens after
``prefix_min..prefix_max`` cached ones), followed by ``rows`` decode rows (contexts ``ctx_min..ctx_max``) and
``pad`` empty slots (no keys, a table of -1); lengths are drawn from ``lens`` so that a case's work does not
depend on the seed.  Blocks are placed by a random permutation of a pool 1.1 times the used blocks.
"""

import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "nano-vllm-practice_amd")

PAGE = 16
BLOCK = 32
EPS = 1e-6
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _case(kind, dtype, heads, kv_heads, dim=128, **kw):
    c = {"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim}
    c.update(kw)
    return c


def listed():
    return [
        # A decode step of the serving batch writes one token of each sequence: the smallest call.
        _case("write", "bf16", 16, 8, name="write_decode_64", rows=64, ctx_min=16, ctx_max=1000, lens=31),
        # The chunked prefill of the benchmark, 8 chunks of 512 tokens, in float16 on heads of 64 dims.
        _case("write", "f16", 32, 8, dim=64, name="write_8x512", seqs=8, new_min=512, new_max=512, prefix_min=0,
              prefix_max=2048, lens=1003),
        # A decode step of the framework's own model: norms, rotation and write of 64 tokens.
        _case("rope", "bf16", 16, 8, name="rope_decode_64", norm=True, rotary=128, interleaved=False, rows=64, ctx_min=16,
              ctx_max=1000, lens=32),
        # The benchmark's 4096 tokens on the 32/8 head shape, a model without norms.
        _case("rope", "bf16", 32, 8, name="rope_8x512", norm=False, rotary=128, interleaved=False, seqs=8, new_min=512,
              new_max=512, prefix_min=0, prefix_max=2048, lens=1003),
        # One user's long chat: the step is launches and latency.
        _case("decode", "bf16", 16, 8, name="decode_one_user", rows=1, ctx_min=5000, ctx_max=5000, lens=1),
        # The serving batch with contexts up to 16k, very uneven; three slots of the batch are empty.
        _case("decode", "bf16", 16, 8, name="decode_64", rows=61, pad=3, ctx_min=256, ctx_max=16384, lens=1002),
        # Long conversations on the 32/8 head shape in float16.
        _case("decode", "f16", 32, 8, name="decode_f16_long", rows=16, ctx_min=8192, ctx_max=32768, lens=3),
        # A full server: what 4 bits are for, four times the sequences that 16 bits would hold.
        _case("decode", "bf16", 32, 8, name="decode_256", rows=256, ctx_min=1024, ctx_max=8192, lens=4),
        # A first prompt of one user in float16, of odd length.
        _case("prefill", "f16", 16, 8, name="prefill_prompt", chunks="0+777", lens=0),
        # Chunked prefill of the benchmark: 8 chunks of 512 after prefixes of up to 2048.
        _case("prefill", "bf16", 16, 8, name="prefill_8x512", seqs=8, new_min=512, new_max=512, prefix_min=0,
              prefix_max=2048, lens=1003),
        # The last chunk of a 32k prompt on the 32/8 head shape: the largest call.
        _case("prefill", "bf16", 32, 8, name="prefill_long", chunks="30720+2048", lens=0),
        # Unified batch: one prefill chunk beside 127 decode rows.
        _case("prefill", "bf16", 32, 8, name="mixed_128", chunks="4096+1024", rows=127, ctx_min=512, ctx_max=8192,
              lens=1005),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# No drawn case costs more than the largest listed ones.
MAX_FLOPS, MAX_BYTES, MAX_POOL = 1.05e12, 1.2e9, 2.0e9


def draw(rng):
    while True:
        kind = rng.choice(["write", "rope", "decode", "decode", "prefill", "prefill"])
        dtype = rng.choice(["bf16", "bf16", "f16"])
        heads, kv_heads = rng.choice([(16, 8), (16, 8), (32, 8), (32, 8), (4, 1), (2, 1), (64, 8), (16, 16), (6, 2), (20, 1)])
        dim = rng.choice([128, 128, 128, 64, 80, 112])
        lens = rng.randrange(1 << 30)
        rows = dict(rows=_log(rng, 1, 256), ctx_max=_log(rng, 1, 32768))
        rows["ctx_min"] = max(1, int(rows["ctx_max"] * rng.uniform(0.03, 1.0)))
        pre = dict(seqs=_log(rng, 1, 16), new_max=_log(rng, 2, 2048), prefix_max=rng.choice([0, _log(rng, 16, 30720)]))
        pre["new_min"] = max(1, int(pre["new_max"] * rng.uniform(0.1, 1.0)))
        pre["prefix_min"] = int(pre["prefix_max"] * rng.uniform(0.0, 1.0))
        if kind == "decode":
            c = _case(kind, dtype, heads, kv_heads, dim, lens=lens, pad=rng.choice([0, 0, rng.randint(1, 9)]), **rows)
        elif kind == "prefill":
            c = _case(kind, dtype, heads, kv_heads, dim, lens=lens, **pre)
            if rng.random() < 0.4:
                c.update(rows)
        else:
            c = _case(kind, dtype, heads, kv_heads, dim, lens=lens)
            if kind == "rope":
                c.update(norm=rng.random() < 0.5, interleaved=rng.random() < 0.4,
                         rotary=rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)]))
            c.update(pre if rng.random() < 0.5 else dict(rows, ctx_max=min(rows["ctx_max"], 2048), ctx_min=1))
        w = work(c)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES and _pool_bytes(c) <= MAX_POOL:
            return c


# ---- the batch ------------------------------------------------------------


def _chunks(case):
    """(cached, new) tokens of every sequence: the chunks, the decode rows, the empty slots."""
    r = random.Random(case["lens"])
    out = []
    if case.get("chunks"):
        out += [tuple(int(x) for x in part.split("+")) for part in case["chunks"].split()]
    for _ in range(case.get("seqs", 0)):
        out.append((r.randint(case["prefix_min"], case["prefix_max"]), r.randint(case["new_min"], case["new_max"])))
    for _ in range(case.get("rows", 0)):
        out.append((r.randint(case["ctx_min"], case["ctx_max"]) - 1, 1))
    return out + [(0, 0)] * case.get("pad", 0)


def _pages(n):
    return -(-n // PAGE)


def _blocks(dim):
    return -(-dim // BLOCK)


def _page_bytes(dim):
    return 2 * 256 * _blocks(dim) + 128


def _pool_bytes(case):
    return 1.1 * sum(_pages(p + n) for p, n in _chunks(case)) * case["kv_heads"] * _page_bytes(case["dim"])


def _randn(shape, gen, dtype):
    return torch.randn(shape, generator=gen, dtype=dtype, device=gen.device)


def _rows(shape, gen, dtype):
    """K or V rows (..., heads, dim): magnitudes differ from token to token, and some channels of each head are larger."""
    x = _randn(shape, gen, torch.float32)
    x = x * (0.3 * _randn((*shape[:-1], 1), gen, torch.float32)).exp()
    return (x * (0.5 * _randn(shape[-2:], gen, torch.float32)).exp()).to(dtype)


def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt, H, KVH, D = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    chunks = _chunks(case)
    kv = [p + n for p, n in chunks]
    num_blocks = max(1, math.ceil(1.1 * sum(_pages(n) for n in kv)))
    perm = torch.randperm(num_blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    cursor, tables = 0, []
    for n in kv:
        tables.append(perm[cursor : cursor + _pages(n)])
        cursor += _pages(n)
    width = max(len(t) for t in tables)

    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    st = {"case": case, "chunks": chunks}
    st["tables"] = i32([t + [-1] * (width - len(t)) for t in tables]).reshape(len(tables), width)
    st["kv_lens"], st["max_kv_len"] = i32(kv), max(kv)
    st["positions"] = torch.cat([torch.arange(p, p + n, dtype=torch.int32) for p, n in chunks]).to(dev)
    cu = [0]
    for _, n in chunks:
        cu.append(cu[-1] + n)
    st["cu_seqlens"], st["max_q_len"] = i32(cu), max(n for _, n in chunks)
    # Decode calls have a query row for every slot of the batch, the empty ones too.
    tokens = len(chunks) if case["kind"] == "decode" else cu[-1]
    pool = torch.randint(0, 256, (num_blocks, KVH, _page_bytes(D)), generator=gen, dtype=torch.uint8, device=dev)
    st["kv_pool"] = pool
    if case["kind"] in ("decode", "prefill"):
        # Cached rows, written a slice of the pool at a time; what is behind a sequence's last row stays as it was.
        for a in range(0, num_blocks, 4096):
            n = min(num_blocks - a, 4096)
            k, v = (_rows((n * PAGE, KVH, D), gen, dt) for _ in range(2))
            at = torch.arange(n * PAGE, device=dev)
            _store(pool, a + at // PAGE, at % PAGE, k.float(), v.float())
        _spoil(st, pool)
        q = _randn((tokens, H, D), gen, dt)
        st["q"] = q.transpose(0, 1)  # the projection's (tokens, heads, dim), as a decoder layer hands it over
        return st
    st["k"], st["v"] = _rows((tokens, KVH, D), gen, dt), _rows((tokens, KVH, D), gen, dt)
    if case["kind"] == "rope":
        st["q"] = _rows((tokens, H, D), gen, dt)
        half = case["rotary"] // 2
        inv = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
        angle = torch.arange(max(kv), dtype=torch.float64, device=dev)[:, None] * inv[None, :]
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
        if case["norm"]:
            st["q_w"], st["k_w"] = ((1 + 0.2 * _randn((D,), gen, torch.float32)).to(dt) for _ in range(2))
    return st


def _spoil(st, pool):
    """Rows of each sequence's last page that hold no token of it: scales of 255, which stand for NaN."""
    last = st["kv_lens"].long() - 1
    has = last >= 0
    block = st["tables"][has].long().gather(1, (last[has] // PAGE)[:, None])[:, 0]
    row = torch.arange(PAGE, device=pool.device)
    n, r = torch.nonzero(row[None, :] > (last[has] % PAGE)[:, None], as_tuple=True)
    scales = pool.size(2) - 128
    for b in range(4):
        pool[block[n], :, scales + 4 * r + b] = 255
        pool[block[n], :, scales + 64 + 16 * (r // 4) + 4 * b + r % 4] = 255


# ---- one pass ---------------------------------------------------------------


def run(st):
    kind = st["case"]["kind"]
    if own:
        return _own(st, kind)
    if kind == "write":
        return _plain_write(st, st["k"].float(), st["v"].float())
    if kind == "rope":
        return _plain_rope(st)
    return _plain_attention(st)


def _own(st, kind):
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    from femtovllm import ops

    c, pool, tables = st["case"], st["kv_pool"], st["tables"]
    if kind == "decode":
        return ops.paged_attention_gemv_fp4(st["q"], pool, tables, st["kv_lens"], st["max_kv_len"])
    if kind == "prefill":
        return ops.paged_attention_gemm_fp4(st["q"], pool, st["cu_seqlens"], st["max_q_len"], tables, st["kv_lens"],
                                            st["positions"])
    cu = None if st["max_q_len"] == 1 else st["cu_seqlens"]
    out = {"kv_pool": pool}
    if kind == "write":
        ops.kv_cache_write_fp4(st["k"], st["v"], pool, st["positions"], tables, cu_seqlens=cu, max_q_len=st["max_q_len"])
    else:
        out["q"] = ops.rope_cache_write_fp4(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["positions"], pool, tables,
                                            cu_seqlens=cu, max_q_len=st["max_q_len"], interleaved=c["interleaved"],
                                            q_norm_weight=st.get("q_w"), k_norm_weight=st.get("k_w"), eps=EPS)
    out["k"], out["v"] = ops.kv_cache_read_fp4(pool, c["dim"], DTYPES[c["dtype"]], st["positions"], tables, cu_seqlens=cu,
                                               max_q_len=st["max_q_len"])
    return out


_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _power(e):
    """2^e, float32, of whole numbers of [-126, 127]."""
    return ((e.int().clamp(-126, 127) + 127) << 23).view(torch.float32)


def _quantize(x):
    """(codes (..., N, 32) uint8, scale bytes (..., N) uint8) of rows x (..., dim), float32."""
    n = _blocks(x.size(-1))
    x = torch.nn.functional.pad(x, (0, n * BLOCK - x.size(-1))).unflatten(-1, (n, BLOCK))
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    f, e = torch.frexp(torch.where(bad, torch.ones_like(top), top))  # top = f 2^e, f in [0.5, 1)
    e = torch.where(top == 0, torch.full_like(e, -1000), e - 3 + (f > 0.875))  # 7 = 0.875 * 2^3
    e = e.clamp(-119, 125)
    y = x * _power(-e)[..., None]
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
            + 8 * torch.signbit(x).to(torch.uint8))
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    return code, torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


def _store(pool, block, row, k, v):
    """Rows k and v (T, heads, dim), float32, to (block, row) of the pool."""
    (ck, sk), (cv, sv) = _quantize(k), _quantize(v)
    T, KVH, n = sk.shape
    dev = pool.device
    at, h = block[:, None, None], torch.arange(KVH, device=dev)[None, :, None]
    r = row[:, None, None]
    b = torch.arange(n, device=dev)
    pair = lambda c: c[..., 0::2] | (c[..., 1::2] << 4)  # noqa: E731
    i = torch.arange(16 * n, device=dev)
    pool[at, h, 256 * (i // 16) + 16 * r + i % 16] = pair(ck).reshape(T, KVH, 16 * n)
    pool[at, h, 256 * n + 64 * n * (r // 4) + 16 * (i // 4) + 4 * (r % 4) + i % 4] = pair(cv).reshape(T, KVH, 16 * n)
    pool[at, h, 512 * n + 4 * r + b] = sk
    pool[at, h, 512 * n + 64 + 16 * (r // 4) + 4 * b + r % 4] = sv


def _load(pool, dim):
    """K and V (..., 16, dim) float32 of pages (..., page_bytes)."""
    n, lead = _blocks(dim), pool.shape[:-1]
    table = torch.tensor(_LEVELS + tuple(-x for x in _LEVELS), dtype=torch.float32, device=pool.device)

    def values(codes, scales):  # (..., 16, N, 16) bytes, (..., 16, N) bytes
        x = table[torch.stack((codes & 15, codes >> 4), -1).int()].flatten(-2)
        s = torch.where(scales == 255, torch.full((), math.nan, device=pool.device), _power(scales.int() - 127))
        return (x * s[..., None]).flatten(-2)[..., :dim]

    kc = pool[..., : 256 * n].reshape(*lead, n, 16, 16).transpose(-3, -2)
    vc = pool[..., 256 * n : 512 * n].reshape(*lead, 4, 4 * n, 4, 4).transpose(-3, -2).reshape(*lead, 16, n, 16)
    ks = pool[..., 512 * n : 512 * n + 64].reshape(*lead, 16, 4)[..., :n]
    vs = pool[..., 512 * n + 64 :].reshape(*lead, 4, 4, 4).transpose(-2, -1).reshape(*lead, 16, 4)[..., :n]
    return values(kc, ks), values(vc, vs)


def _slots(st):
    """Block and row of every token's cache entry."""
    lens = st["cu_seqlens"].diff().long()
    seq = torch.repeat_interleave(torch.arange(lens.numel(), device=lens.device), lens)
    pos = st["positions"].long()
    return st["tables"][seq, pos // PAGE].long(), pos % PAGE


def _plain_write(st, k, v):
    pool, dim = st["kv_pool"], st["case"]["dim"]
    block, row = _slots(st)
    _store(pool, block, row, k, v)
    out = {"kv_pool": pool, "k": torch.empty_like(st["k"]), "v": torch.empty_like(st["v"])}
    for a in range(0, row.numel(), 4096):  # (a page of every token at a time)
        kk, vv = _load(pool[block[a : a + 4096]], dim)
        at = row[a : a + 4096, None, None, None].expand(-1, kk.size(1), 1, dim)
        out["k"][a : a + 4096], out["v"][a : a + 4096] = kk.gather(2, at)[:, :, 0], vv.gather(2, at)[:, :, 0]
    return out


def _plain_rope(st):
    """The norms in 64 bits, rounded to 32, and the rotation in 32 bits (each product and each sum rounded): a value that
    is next to a border of the 4-bit list must not fall on either side of it by the order of a sum."""
    c = st["case"]
    R = c["rotary"]
    pos = st["positions"].long()
    cos, sin = st["cos"][pos][:, None, :], st["sin"][pos][:, None, :]

    def rotate(x, w):
        y = x.float()
        if w is not None:
            d = x.double()
            d = d * (1 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)) * w.double()
            y = d.float()
        y, z = y.clone(), y
        if c["interleaved"]:
            a, b = z[..., 0:R:2], z[..., 1:R:2]
            y[..., 0:R:2], y[..., 1:R:2] = a * cos - b * sin, b * cos + a * sin
        else:
            a, b = z[..., : R // 2], z[..., R // 2 : R]
            y[..., : R // 2], y[..., R // 2 : R] = a * cos - b * sin, b * cos + a * sin
        return y

    out = _plain_write(st, rotate(st["k"], st.get("k_w")), st["v"].float())
    return {"q": rotate(st["q"], st.get("q_w")).to(st["q"].dtype), **out}


def _plain_attention(st):
    """Decode rows 16 sequences at a time, chunks one by one."""
    c, q, tables = st["case"], st["q"], st["tables"]
    H, KVH, D = c["heads"], c["kv_heads"], c["dim"]
    rep = H // KVH
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    single = [b for b, (_, n) in enumerate(st["chunks"]) if n <= 1]
    first = [0]
    for _, n in st["chunks"]:
        first.append(first[-1] + (1 if c["kind"] == "decode" else n))

    def weighted(x, k, v, seen):  # (B, KVH, M, D), (B, KVH, L, D) twice, (B, 1, M or 1, L)
        s = torch.matmul(x, k.transpose(-2, -1).contiguous()) / math.sqrt(D)
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        w = torch.exp(s - s.amax(-1, keepdim=True))
        return torch.matmul(w, v) / w.sum(-1, keepdim=True)

    def cached(rows, pages):
        blocks = tables[rows, :pages].long()
        k, v = _load(st["kv_pool"][blocks.clamp(min=0)], D)
        k, v = (t.transpose(1, 2).flatten(2, 3) for t in (k, v))  # (B, KVH, 16 pages, D)
        j = torch.arange(PAGE * pages, device=q.device)
        there = (j[None, :] < st["kv_lens"][rows][:, None])[:, None, :, None]
        return torch.where(there, k, torch.zeros_like(k)), torch.where(there, v, torch.zeros_like(v)), j

    for a in range(0, len(single), 16):
        seqs = single[a : a + 16]
        pages = max(_pages(sum(st["chunks"][b])) for b in seqs)
        if pages == 0:  # empty slots: zeros
            continue
        rows = torch.tensor(seqs, device=q.device)
        k, v, j = cached(rows, pages)
        at = torch.tensor([first[b] for b in seqs], device=q.device)
        x = q[:, at].float().transpose(0, 1).reshape(len(seqs), KVH, rep, D)
        seen = (j[None, :] < st["kv_lens"][rows][:, None])[:, None, None, :]
        o = weighted(x, k, v, seen).reshape(len(seqs), H, D).transpose(0, 1)
        empty = (st["kv_lens"][rows] == 0)[None, :, None]
        out[:, at] = torch.where(empty, torch.zeros_like(o), o).to(q.dtype)
    for b, (p, n) in enumerate(st["chunks"]):
        if n <= 1:
            continue
        t = slice(first[b], first[b] + n)
        k, v, j = cached(torch.tensor([b], device=q.device), _pages(p + n))
        pos = st["positions"][t].long().repeat(rep)[:, None]
        x = q[:, t].float().reshape(1, KVH, rep * n, D)
        out[:, t] = weighted(x, k, v, (j[None, :] <= pos)[None, None]).reshape(H, n, D).to(q.dtype)
    return out


# ---- work and 64-bit results ------------------------------------------------


def work(case):
    """Attention: the codes and scales of every key once per KV head, q in and out once, the tables and lengths;
    4 * dim flops per visible (query, key) pair and query head.  Writes: q, k and v rows in, the rotated q out, the
    codes and scales out, and for the tokens read back the same codes and scales in and the values out."""
    H, KVH, D = case["heads"], case["kv_heads"], case["dim"]
    chunks = _chunks(case)
    tokens = sum(n for _, n in chunks)
    row = 2 * (D // 2 + _blocks(D))  # K and V of one token and head
    if case["kind"] in ("write", "rope"):
        total = tokens * KVH * (2 * 4 * D + 2 * row)
        if case["kind"] == "rope":
            total += tokens * (4 * D * H + 4 * case["rotary"])
        return {"bytes": total, "flops": 0}
    keys = sum(p + n for p, n in chunks)
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in chunks)
    return {"bytes": row * KVH * keys + 4 * D * H * tokens + 4 * _pages(keys) + 8 * len(chunks), "flops": 4 * D * H * pairs}


def _exact_values(data, scale):
    """Values of bytes (..., m) under one scale byte each (...): sign, two bits of exponent, one of mantissa."""
    code = torch.stack((data % 16, data // 16), -1).flatten(-2).long()
    e, m = (code // 2) % 4, (code % 2).double()
    x = torch.where(e == 0, m / 2, (1 + m / 2) * torch.pow(2.0, (e - 1).double()))
    x = torch.where(code >= 8, -x, x) * torch.pow(torch.full((), 2.0, dtype=torch.float64, device=data.device),
                                                  scale.double() - 127)[..., None]
    return torch.where((scale == 255)[..., None], torch.full_like(x, math.nan), x)


def _exact_rows(pool, blocks, head, length, dim):
    """K and V (length, dim) in 64 bits of one head of one sequence."""
    n, page = _blocks(dim), pool[blocks, head]
    pos = torch.arange(length, device=pool.device)
    p, r = pos // PAGE, pos % PAGE
    k, v = [], []
    for b in range(n):
        i = torch.arange(16, device=pool.device)
        data = page[p[:, None], 256 * b + 16 * r[:, None] + i]
        k.append(_exact_values(data, page[p, 512 * n + 4 * r + b]))
        data = page[p[:, None], 256 * n + (r // 4 * 64 * n)[:, None] + 16 * (4 * b + i // 4) + 4 * (r % 4)[:, None] + i % 4]
        v.append(_exact_values(data, page[p, 512 * n + 64 + 16 * (r // 4) + 4 * b + r % 4]))
    return torch.cat(k, -1)[:, :dim], torch.cat(v, -1)[:, :dim]


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] in ("write", "rope"):
        return _exact_write(case, st)
    q = st["q"].double()
    D, rep = case["dim"], case["heads"] // case["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lens, cu = st["kv_lens"].tolist(), st["cu_seqlens"].tolist()
    for b, L in enumerate(lens):
        if L == 0:
            continue
        lo, hi = (cu[b], cu[b + 1]) if case["kind"] == "prefill" else (b, b + 1)
        blocks = st["tables"][b, : _pages(L)].long()
        j = torch.arange(L, device=q.device)
        for g in range(case["kv_heads"]):
            k, v = _exact_rows(st["kv_pool"], blocks, g, L, D)
            k = k.t().contiguous()
            for a in range(lo, hi, 1024):
                z = min(hi, a + 1024)
                pos = (torch.arange(a, z, device=q.device) - hi + L).repeat(rep)
                x = q[g * rep : (g + 1) * rep, a:z].reshape(-1, D)
                logits = torch.mm(x, k).mul_(1.0 / math.sqrt(D)).masked_fill_(j[None, :] > pos[:, None], -math.inf)
                out[g * rep : (g + 1) * rep, a:z] = torch.mm(torch.softmax(logits, dim=-1), v).reshape(rep, z - a, D)
    return out


def _exact_nearest(x):
    """The values that rows x (..., dim) in 64 bits are held as."""
    dim = x.size(-1)
    x = torch.nn.functional.pad(x, (0, _blocks(dim) * BLOCK - dim)).unflatten(-1, (-1, BLOCK))
    top = x.abs().amax(-1, keepdim=True)
    step = torch.pow(2.0, torch.ceil(torch.log2(top / 7)).clamp(min=-119))
    step = torch.where(top > 7 * step, 2 * step, torch.where((top <= 3.5 * step) & (step > 2.0 ** -119), step / 2, step))
    step = step.clamp(max=2.0**125)
    level = torch.tensor([0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0], dtype=torch.float64, device=x.device)  # even indices first
    near = level[((x / step).abs()[..., None] - level).abs().argmin(-1)]
    return (near * step * torch.sign(x)).flatten(-2)[..., :dim]


def _exact_write(case, st):
    """The rotation as a complex product, token by token's own table row."""
    k, q = st["k"].double(), st["q"].double() if "q" in st else None
    if case["kind"] == "rope":
        R, pos = case["rotary"], st["positions"].long()
        turn = torch.complex(st["cos"].double(), st["sin"].double())[pos][:, None, :]

        def rotated(x, w):
            if w is not None:
                x = x / (x.square().sum(-1, keepdim=True) / x.size(-1) + EPS).sqrt() * w.double()
            head = x[..., :R]
            if case["interleaved"]:
                z = torch.view_as_complex(head.reshape(*head.shape[:-1], R // 2, 2).contiguous()) * turn
                head = torch.view_as_real(z).reshape(head.shape)
            else:
                z = torch.complex(head[..., : R // 2].contiguous(), head[..., R // 2 :].contiguous()) * turn
                head = torch.cat((z.real, z.imag), dim=-1)
            return torch.cat((head, x[..., R:]), dim=-1)

        k, q = rotated(k, st.get("k_w")), rotated(q, st.get("q_w"))
    held = [torch.cat([_exact_nearest(x[a : a + 256]) for a in range(0, x.size(0), 256)]) for x in (k, st["v"].double())]
    out = {"kv_pool": None, "k": held[0], "v": held[1]}
    return out if q is None else {"q": q, **out}
