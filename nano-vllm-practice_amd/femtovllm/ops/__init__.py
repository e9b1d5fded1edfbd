"""Attention operators with the reference's call signatures.

``paged_attention_gemv`` and ``paged_attention_gemm`` keep the signatures,
defaults, constants and error behaviour of femtovllm/ops/__init__.py:21-156
of the reference, so the engine, scheduler, prefix tree and block tables
drive them unchanged.  Both run hand-written HIP kernels for gfx950
(``libfemto_attn.so`` through :mod:`femtovllm._C`); importing this module
raises ``ImportError`` when that library is missing (ops/__init__.py:6-16).

``impl`` is kept for signature compatibility: ``ImplCustomKernel.CUDA`` and,
for the prefill op, ``ImplCustomKernel.TRITON`` (the reference's default)
both select the HIP kernels; anything else raises ``NotImplementedError``
as in the reference (ops/__init__.py:106-107, 155-156).

``kv_cache_write`` and ``qk_norm_rope_cache_write`` have no operator
counterpart in the reference: the first replaces the per-sequence slicing
loops that write the new K/V into the paged pools before the attention ops
(femtovllm/models/qwen/qwen3.py:240-264 for decode, 322-366 for prefill),
taking the same metadata; the second also fuses the q/k RMSNorm and the
rotary embedding that precede those loops (qwen3.py:230-238, 312-320).

``paged_attention_gemv_window`` and ``paged_attention_gemm_window`` are the
two attention operators under a sliding window whose first tokens may stay
visible; the reference has no windowed attention.
``paged_attention_gemv_shared_prefix`` is decode for a batch on a common
prefix, which the reference reads once per sequence.  ``rope_cache_write`` is
the prologue of layers without q/k norms, for every rotary layout.

The operators whose names end in ``_fp4`` work on a KV cache held in 4 bits
(:mod:`femtovllm.fp4`): the write of new tokens, the prologue with norms and
rotation, a read of tokens, and both attention operators.  The reference's
cache is 16 bits wide.

One deliberate difference: ``q`` arrives as ``q.transpose(0, 1)`` of a
``(tokens, n_heads, head_dim)`` tensor (femtovllm/models/qwen/qwen3.py:270,
372).  The reference copies it with ``.contiguous()``; the HIP kernels take
the head and token strides directly, so no copy is made as long as the
head dimension is contiguous.
"""

import torch

import femtovllm
from femtovllm.protocol import ImplCustomKernel

try:
    from femtovllm import _C as _hip_backend
except ImportError as e:
    raise ImportError(
        "Failed to load the femtovllm HIP backend (libfemto_attn.so).\n"
        "Build it for gfx950 with:\n"
        "    python nano-vllm-practice_amd/build.py"
    ) from e

MAX_KV_LEN_NON_SPLIT = _hip_backend.kMaxKVLenNonSplit

KV_LEN_PER_PAGE = _hip_backend.kKVLenPerPage
# The kernels are built for this exact head dim (register tiling), as in the
# reference (femtovllm/ops/__init__.py:24-26).
DIM_HEAD = _hip_backend.kDimHead


def _ensure_valid_tensor(t: torch.Tensor, name: str) -> torch.Tensor:
    """Require a GPU tensor (ValueError otherwise, ops/__init__.py:36-39).

    Strided views are passed through; only a tensor whose innermost
    dimension is not contiguous is copied.
    """
    if not t.is_cuda:
        raise ValueError(f"Argument '{name}' must be a CUDA tensor. Got device={t.device}")
    if t.stride(-1) != 1:
        return t.contiguous()
    return t


def paged_attention_gemv(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    kv_page_tables: torch.Tensor,
    kv_lens: torch.Tensor,
    max_kv_len: int,
    #####
    impl: ImplCustomKernel = None,
):
    """Decode attention over the paged KV cache.

    q (n_heads, num_seqs, head_dim); pools (num_blocks, n_kv_heads, 16,
    head_dim); kv_page_tables (num_seqs, max_pages) int32, -1 padded;
    kv_lens (num_seqs,) int32.  Returns (n_heads, num_seqs, head_dim).
    ``max_kv_len`` above ``MAX_KV_LEN_NON_SPLIT`` raises ``RuntimeError`` as in
    the reference unless ``femtovllm._DEV.split_kv_decode`` is set.
    """
    q = _ensure_valid_tensor(q, "q")

    impl = femtovllm._DEV.impl_custom_gemv if (impl is None) else impl

    if impl == ImplCustomKernel.CUDA:
        return _hip_backend._paged_attention_gemv(
            q,
            k_pool,
            v_pool,
            kv_page_tables,
            kv_lens,
            max_kv_len,
            require_contiguous_q=False,
            # getattr: a reference checkout's DevFlags has no such field
            max_kv_len_limit=None if getattr(femtovllm._DEV, "split_kv_decode", False) else MAX_KV_LEN_NON_SPLIT,
        )
    else:
        raise NotImplementedError()


def paged_attention_gemm(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    cu_seqlens: torch.Tensor,
    max_q_len: int,
    Q_TILE_SIZE: int,
    cu_q_tiles: torch.Tensor,
    q_tile_to_seq_idx: torch.Tensor,
    kv_page_tables: torch.Tensor,
    kv_lens: torch.Tensor,
    positions: torch.Tensor,
    #####
    impl: ImplCustomKernel = None,
):
    """Chunked / varlen / causal prefill over the paged KV cache.

    q (n_heads, num_tokens, head_dim) with sequences delimited by
    cu_seqlens; token t sees key j iff j < kv_lens[seq] and
    j <= positions[t].  ``Q_TILE_SIZE``, ``cu_q_tiles`` and
    ``q_tile_to_seq_idx`` describe the reference Triton kernel's launch grid;
    the HIP kernel derives its own tiles from ``cu_seqlens`` and ignores them.
    Returns (n_heads, num_tokens, head_dim).
    """
    q = _ensure_valid_tensor(q, "q")

    impl = femtovllm._DEV.impl_custom_gemm if (impl is None) else impl

    if impl == ImplCustomKernel.CUDA or impl == ImplCustomKernel.TRITON:
        return _hip_backend._paged_attention_gemm(
            q,
            k_pool,
            v_pool,
            cu_seqlens,
            max_q_len,
            kv_page_tables,
            kv_lens,
            positions,
            require_contiguous_q=False,
        )
    else:
        raise NotImplementedError()


def paged_attention_gemv_window(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    kv_page_tables: torch.Tensor,
    kv_lens: torch.Tensor,
    max_kv_len: int,
    window: int,
    sinks: int = 0,
):
    """:func:`paged_attention_gemv` under a sliding window with sinks.

    Sequence b's query, at position ``kv_lens[b] - 1``, sees key j iff
    ``j < kv_lens[b]`` and (``j >= kv_lens[b] - window`` or ``j < sinks``).
    ``window >= 1`` counts the query's own key; one larger than the contexts
    sees all keys.  Blocks that hold no visible key are not read, so their
    table entries may be -1 or handed to another sequence.  Contexts may be of
    any length (no ``MAX_KV_LEN_NON_SPLIT`` here); an empty one gives zeros.
    """
    return _hip_backend._paged_attention_gemv_window(_ensure_valid_tensor(q, "q"), k_pool, v_pool, kv_page_tables,
                                                     kv_lens, max_kv_len, window, sinks)


def paged_attention_gemm_window(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    cu_seqlens: torch.Tensor,
    max_q_len: int,
    kv_page_tables: torch.Tensor,
    kv_lens: torch.Tensor,
    positions: torch.Tensor,
    window: int,
    sinks: int = 0,
):
    """:func:`paged_attention_gemm` under a sliding window with sinks.

    Token t of sequence b sees key j iff ``j < kv_lens[b]``, ``j <=
    positions[t]`` and (``j > positions[t] - window`` or ``j < sinks``).  A
    token that sees no key gives NaN, as in ``paged_attention_gemm``.  Blocks
    that no token of the call sees are not read.  V has to be finite in keys
    that some token of a sequence sees: one that is not may also reach tokens
    up to 128 away that do not see it.
    """
    return _hip_backend._paged_attention_gemm_window(_ensure_valid_tensor(q, "q"), k_pool, v_pool, cu_seqlens,
                                                     max_q_len, kv_page_tables, kv_lens, positions, window, sinks)


def paged_attention_gemv_shared_prefix(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    prefix_pages: torch.Tensor,
    kv_page_tables: torch.Tensor,
    kv_lens: torch.Tensor,
    max_kv_len: int,
):
    """:func:`paged_attention_gemv` for a batch whose sequences share their first blocks.

    ``prefix_pages`` (P,) int32: the blocks of the common prefix, full ones (a
    node of the prefix tree; ``kv_page_tables[0, :P]`` where that row holds
    them).  Key j of sequence b is in block ``prefix_pages[j // 16]`` for
    ``j < 16 P`` and in ``kv_page_tables[b, j // 16]`` after that; the tables'
    first P columns are not read.  ``kv_lens`` counts the prefix too and may
    end inside it.  The prefix is read once for the whole batch, and the call
    costs its tails beside that.  bf16 or f16, head_dim a multiple of 16;
    contexts of any length; an empty one gives zeros.  V of the prefix has to be
    finite: a value that is not may also reach sequences that end before it.
    """
    return _hip_backend._paged_attention_gemv_shared_prefix(_ensure_valid_tensor(q, "q"), k_pool, v_pool, prefix_pages,
                                                            kv_page_tables, kv_lens, max_kv_len)


def kv_cache_write(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache_pool: torch.Tensor,
    v_cache_pool: torch.Tensor,
    positions: torch.Tensor,
    kv_page_tables: torch.Tensor,
    cu_seqlens: torch.Tensor = None,
    max_q_len: int = 1,
):
    """Write the new K/V rows into the paged pools (in place, bit-exact).

    k, v (num_tokens, n_kv_heads, head_dim), as produced by the projections
    (femtovllm/models/qwen/qwen3.py:231-238); pools (num_blocks, n_kv_heads,
    16, head_dim).  Prefill: sequence b owns tokens cu_seqlens[b] ..
    cu_seqlens[b+1] and writes them at positions[cu_seqlens[b]] + 0, 1, ...
    (qwen3.py:322-366); decode (``cu_seqlens=None``, as in the decode
    metadata of femtovllm/engine/model_runner.py:316-330): token b at
    positions[b] (qwen3.py:240-264).  max_q_len is the metadata's
    ``max_q_len``.  Position p goes to block kv_page_tables[b][p // 16], row
    p % 16; as in the reference loops, a sequence's writes stop at the first
    table entry that is -1 (and at block ids outside the pool).
    """
    for name, t in (("k", k), ("v", v)):
        if not t.is_cuda:
            raise ValueError(f"Argument '{name}' must be a CUDA tensor. Got device={t.device}")
    k = k if k.stride(-1) == 1 else k.contiguous()
    v = v if v.stride(-1) == 1 else v.contiguous()
    _hip_backend._kv_cache_write(k, v, k_cache_pool, v_cache_pool, positions, kv_page_tables, cu_seqlens, max_q_len)


def qk_norm_rope_cache_write(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    q_norm_weight: torch.Tensor,
    k_norm_weight: torch.Tensor,
    eps: float,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor,
    k_cache_pool: torch.Tensor,
    v_cache_pool: torch.Tensor,
    kv_page_tables: torch.Tensor,
    cu_seqlens: torch.Tensor = None,
    max_q_len: int = 1,
    out: torch.Tensor = None,
):
    """The attention layer's prologue in one kernel; returns the rotated q.

    q (num_tokens, n_heads, 128), k and v (num_tokens, n_kv_heads, 128) as
    produced by the projections; ``q_norm_weight`` / ``k_norm_weight`` and
    ``eps`` of the layer's ``q_norm`` / ``k_norm`` RMSNorms; ``cos`` / ``sin``
    the rotary tables of ``QwenRotaryEmbedding`` (float32, (max_seqlen,
    128)); ``positions`` each token's position.  Computes
    ``rotary_embd(q_norm(q))`` (returned, in ``out`` if given, which may be
    ``q``) and ``rotary_embd(k_norm(k))``, and writes that k and v into the
    pools exactly as :func:`kv_cache_write` (qwen3.py:230-264, 312-366).
    Each output element is rounded once from fp32.
    """
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not t.is_cuda:
            raise ValueError(f"Argument '{name}' must be a CUDA tensor. Got device={t.device}")
    return _hip_backend._qk_norm_rope_cache_write(q, k, v, q_norm_weight, k_norm_weight, eps, cos, sin, positions,
                                                   k_cache_pool, v_cache_pool, kv_page_tables, cu_seqlens,
                                                   max_q_len, out)


def rope_cache_write(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor,
    k_cache_pool: torch.Tensor,
    v_cache_pool: torch.Tensor,
    kv_page_tables: torch.Tensor,
    cu_seqlens: torch.Tensor = None,
    max_q_len: int = 1,
    interleaved: bool = False,
    out: torch.Tensor = None,
):
    """The prologue of layers without q/k norms in one kernel; returns the rotated q.

    q (num_tokens, n_heads, head_dim), k and v (num_tokens, n_kv_heads,
    head_dim), head_dim at most 128; ``cos`` / ``sin`` float32 tables
    (max_seqlen, rotary_dim / 2), e.g. of ``femtovllm.rope.scaled_rope_tables``;
    ``positions`` each token's position.  Rotates the first ``rotary_dim`` dims
    of each q and k head, as pairs (i, i + rotary_dim / 2) or, ``interleaved``,
    (2 i, 2 i + 1): (a, b) -> (a cos - b sin, b cos + a sin); the other dims
    pass through.  The rotated q goes to ``out`` (new; if given, ``q`` itself
    or no element of ``q``; none of ``k`` and ``v`` either way), the rotated k and
    v into the pools exactly as :func:`kv_cache_write`.  Each output element is
    rounded once from fp32; a position outside the tables gives NaN in the rotated
    dims.
    """
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not t.is_cuda:
            raise ValueError(f"Argument '{name}' must be a CUDA tensor. Got device={t.device}")
    return _hip_backend._rope_cache_write(q, k, v, cos, sin, positions, k_cache_pool, v_cache_pool, kv_page_tables,
                                          cu_seqlens, max_q_len, interleaved, out)


def kv_cache_write_fp4(
    k: torch.Tensor,
    v: torch.Tensor,
    kv_pool: torch.Tensor,
    positions: torch.Tensor,
    kv_page_tables: torch.Tensor,
    cu_seqlens: torch.Tensor = None,
    max_q_len: int = 1,
):
    """:func:`kv_cache_write` into a cache held in 4 bits (in place).

    ``kv_pool`` is a pool of :func:`femtovllm.fp4.new_pool`; k and v (bf16 or
    f16, head_dim a multiple of 16 up to 128), ``positions``, the tables and
    ``cu_seqlens`` are those of :func:`kv_cache_write`.  Each 32 dims of a row are
    rounded to the nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} times their scale, the
    smallest power of two of which no magnitude is more than 7 (from 2^-119 to 2^125);
    32 dims that hold an infinity or a NaN become NaN.  ``max_q_len`` decides nothing
    here: sequences of any length are written whole.  Tokens of one call want
    places of their own: two at one place leave a mix of both there.
    """
    for name, t in (("k", k), ("v", v)):
        if not t.is_cuda:
            raise ValueError(f"Argument '{name}' must be a CUDA tensor. Got device={t.device}")
    k = k if k.stride(-1) == 1 else k.contiguous()
    v = v if v.stride(-1) == 1 else v.contiguous()
    _hip_backend._kv_cache_write_fp4(k, v, kv_pool, positions, kv_page_tables, cu_seqlens, max_q_len)


def kv_cache_read_fp4(
    kv_pool: torch.Tensor,
    head_dim: int,
    dtype: torch.dtype,
    positions: torch.Tensor,
    kv_page_tables: torch.Tensor,
    cu_seqlens: torch.Tensor = None,
    max_q_len: int = 1,
):
    """(k, v), each (num_tokens, n_kv_heads, head_dim) of ``dtype`` (bf16 or f16), of tokens in a 4-bit cache.

    The tokens are those that :func:`kv_cache_write_fp4` would write with the
    same arguments, e.g. a whole prefix that moves to 16-bit pools; zeros where
    that would have stopped, and for tokens that are in no sequence (before
    ``cu_seqlens[0]``, from ``cu_seqlens[-1]`` on).  bf16 holds every value exactly;
    f16 rounds, and values past its range are infinities, 65536 among them, which
    the cache holds for f16 values past 57344.
    """
    if not kv_pool.is_cuda:
        raise ValueError(f"Argument 'kv_pool' must be a CUDA tensor. Got device={kv_pool.device}")
    return _hip_backend._kv_cache_read_fp4(kv_pool, head_dim, dtype, positions, kv_page_tables, cu_seqlens, max_q_len)


def rope_cache_write_fp4(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor,
    kv_pool: torch.Tensor,
    kv_page_tables: torch.Tensor,
    cu_seqlens: torch.Tensor = None,
    max_q_len: int = 1,
    interleaved: bool = False,
    q_norm_weight: torch.Tensor = None,
    k_norm_weight: torch.Tensor = None,
    eps: float = 1e-6,
    out: torch.Tensor = None,
):
    """The attention layer's prologue over a 4-bit cache in one kernel; returns the rotated q.

    :func:`rope_cache_write` (same layouts, tables, positions and rules for
    ``out``) with k and v rounded to 4 bits as :func:`kv_cache_write_fp4` does.
    With ``q_norm_weight`` and ``k_norm_weight`` ((head_dim,) of q's dtype, both or
    neither) and ``eps``, q and k first pass the layer's RMSNorms, as in
    :func:`qk_norm_rope_cache_write`.  bf16 or f16.  k is rounded once, from
    float32.  Rows of ``out`` of tokens in no sequence are left as they were (a
    new ``out`` holds nothing of meaning there).
    """
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not t.is_cuda:
            raise ValueError(f"Argument '{name}' must be a CUDA tensor. Got device={t.device}")
    return _hip_backend._rope_cache_write_fp4(q, k, v, cos, sin, positions, kv_pool, kv_page_tables, cu_seqlens,
                                              max_q_len, interleaved, q_norm_weight, k_norm_weight, eps, out)


def paged_attention_gemv_fp4(
    q: torch.Tensor,
    kv_pool: torch.Tensor,
    kv_page_tables: torch.Tensor,
    kv_lens: torch.Tensor,
    max_kv_len: int,
):
    """:func:`paged_attention_gemv` over a KV cache held in 4 bits.

    q (n_heads, num_seqs, head_dim) bf16 or f16, head_dim a multiple of 16 up to
    128; ``kv_pool`` (num_blocks, n_kv_heads, page bytes) as written by
    :func:`kv_cache_write_fp4`.  Contexts of any length; an empty one gives zeros.
    Keys and values are what the cache stands for (f16: V from 131072 on, twice its
    range, is an infinity); rows behind a context may hold anything.
    """
    return _hip_backend._paged_attention_gemv_fp4(_ensure_valid_tensor(q, "q"), kv_pool, kv_page_tables, kv_lens, max_kv_len)


def paged_attention_gemm_fp4(
    q: torch.Tensor,
    kv_pool: torch.Tensor,
    cu_seqlens: torch.Tensor,
    max_q_len: int,
    kv_page_tables: torch.Tensor,
    kv_lens: torch.Tensor,
    positions: torch.Tensor,
):
    """:func:`paged_attention_gemm` over a KV cache held in 4 bits.

    Token t of sequence b sees key j iff ``j < kv_lens[b]`` and ``j <=
    positions[t]``; a token that sees no key gives NaN.  Types, dims and the
    pool as :func:`paged_attention_gemv_fp4`; chunks and single tokens may share a
    call.  V that is NaN reaches the tokens that see its key and no other; V that is an
    infinity to f16 (from 131072 on) also reaches, as NaN, those of its query tile
    (up to 128 tokens of the chunk) that do not.
    """
    return _hip_backend._paged_attention_gemm_fp4(_ensure_valid_tensor(q, "q"), kv_pool, cu_seqlens, max_q_len,
                                                  kv_page_tables, kv_lens, positions)
