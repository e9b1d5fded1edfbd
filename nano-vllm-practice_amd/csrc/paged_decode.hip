// Paged decode attention (one query token per sequence) for gfx950.
//
// Semantics follow PagedAttentionGemvKernel
// (csrc/paged_attention/paged_attention_gemv.cu:16-221 of the reference):
// out[h, b] = softmax(q[h, b] . K_b^T / sqrt(D)) . V_b over kv_lens[b] keys,
// key j of sequence b at k_pool[tables[b][j / 16], h / n_rep, j % 16].
//
// Design (memory-bound GEMV):
//  * waves are independent workers: per group of NREP query heads sharing a
//    KV head, the pages of all sequences are concatenated and cut into equal
//    slices, one per wave (one wave per SIMD); every K/V byte is loaded once
//    and used by all NREP query heads (the reference loads it n_rep times);
//  * inside a wave, DPP row r (16 lanes) owns page rows r, r+4, r+8, r+12 and
//    lane c of the row owns 8 head dims, so each K/V page is 4 coalesced
//    16-byte loads per lane (bf16/f16; f32 uses 8), issued with the
//    non-temporal hint (each byte is read once per call), and the q.k
//    reduction stays inside a DPP row;
//  * block ids are fetched 64 at a time (one per lane) and broadcast with
//    readlane, and a page's loads go out two pages ahead of its math, so
//    the table never adds a dependent load per page;
//  * every lane keeps an online-softmax state (max, sum, 8 accumulators) per
//    query head over the keys it saw; states merge across the four DPP rows
//    with permlane swaps, each sequence segment of a slice leaves one partial
//    state in the workspace, and a small merge kernel on the same stream
//    combines them (no cross-workgroup fences or atomics, which on gfx950
//    would write back and invalidate the XCD's L2);
//  * rows past kv_len are never read (loads are clamped to the last visible
//    row and their scores masked) and block ids outside the pool are never
//    dereferenced (their page reads as zeros), so NaN in unused pool memory
//    cannot leak.  The repeated row has weight 0: where it holds an infinity
//    of V, that output is NaN and not infinite.
#include "decode_kernels.h"

namespace femto {

// One wave per SIMD (4 per CU), each with a page of K and V in flight behind
// those it computes.  HBM read throughput peaks there: more resident waves queue
// more requests and lose bandwidth (on the 545 MB Qwen3-0.6B-shaped batch, 16
// waves per CU ran at 4.85 TB/s and 4 per CU at 5.2 TB/s with ordinary loads;
// 8 per CU with non-temporal loads was 2 % slower than 4, and 6 or 8 per CU
// 3-12 % slower with the dot2 page math).  Sets a.waves_per_group and returns
// the workgroups of 4 waves that cover the workers (0 on a device error).
int decode_worker_blocks(DecodeArgs& a) {
    int cus = 0;
    if (device_cu_count(cus) != hipSuccess) return 0;
    const int total_waves = cus * 4;
    a.waves_per_group = total_waves / a.grid_heads > 0 ? total_waves / a.grid_heads : 1;
    return (a.waves_per_group * a.grid_heads + 3) / 4;
}

hipError_t launch_paged_decode_merge(int dtype, const DecodeArgs& a, int num_seqs, hipStream_t st) {
    return launch_merge_dtype<kAllPages>(dtype, a, num_seqs, st);
}

hipError_t launch_paged_decode(int dtype, const DecodeArgs& a, int nrep_tile, int num_seqs, bool single,
                               hipStream_t st) {
    return launch_decode_dtype<kAllPages>(dtype, a, nrep_tile, num_seqs, single, st);
}

}  // namespace femto
