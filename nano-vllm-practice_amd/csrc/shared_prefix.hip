// Decode attention of a batch whose sequences share their first pages.
//
// Formula: out[h, b] = sum_j w_j v_j / sum_j w_j, w_j = exp(q[h, b] . k_j / sqrt(D)),
// over the prefix's keys j < min(kv_lens[b], 16 P) and the sequence's own from
// page P on.  The two sums have the same shape, so each is formed by the unit
// that it suits, relative to its own maximum, and a merge launch joins them:
//  * prefix: every K/V byte serves all sequences, so it is a matrix product of
//    the batch's query rows with the prefix, on the MFMA tiles of
//    attention_tiles.h, read from HBM once and not once per sequence.  It has
//    few query tiles (one per 32-128 sequences and KV head), so its keys are
//    cut into pieces, one workgroup each;
//  * tails: bound by their bytes, on the MFMA workers of mfma_decode.h, in
//    the same launch, one workgroup per CU beside the tiles.
// 256 sequences on 16384 keys, tails of up to 1024, 32/8 heads: 132-135 us, bound by
// both, the tails' 509 MB (92 us alone) and the tiles, 64 in series (104 alone);
// 64 on 4096, tails of up to 512, f16 16/8 heads 27.5 us; 8 on 1024 11.7 us, two
// launches and their round trips.
#include "attention_tiles.h"
#include "decode_merge.h"
#include "prefix_plan.h"

namespace femto {

static_assert(kPrefixTile == kKvTile, "the prefix is cut between key tiles");

SharedPrefixPlan plan_shared_prefix(int num_seqs, int n_heads, int n_kv_heads, int prefix_pages, int max_kv_len,
                                    int dtype, int cus) {
    SharedPrefixPlan p{};
    const int n_rep = n_heads / n_kv_heads, G = prefill_group(n_rep), BT = 32 * (4 / G);
    const int tail = (int)std::max<int64_t>(1, (int64_t)max_kv_len - (int64_t)prefix_pages * kPage);
    p.tail = plan_paged_decode(n_heads, n_kv_heads, tail, dtype);
    const PrefixPieces c = prefix_pieces(num_seqs, n_heads, n_kv_heads, G, BT, prefix_pages * kPage, tail, cus);
    p.pieces = c.pieces;
    p.piece_keys = c.piece_keys;
    p.longest = c.longest;
    return p;
}

hipError_t launch_shared_prefix(int dtype, PrefillArgs a, hipStream_t st) {
    if (a.num_seqs <= 0) return hipSuccess;
    const int G = prefill_group(a.n_rep), BT = 32 * (4 / G);
    a.head_groups = a.n_rep / G;
    a.tiles_per_group = (a.num_seqs + BT - 1) / BT;
    a.total_work = a.tiles_per_group * a.n_kv_heads * a.head_groups * a.dec.prefix_pieces;
    set_mfma_heads(a.dec);
    a.decode_blocks = decode_worker_blocks(a.dec);
    if (a.decode_blocks <= 0) return hipErrorInvalidDevice;
    a.decode_blocks = (a.decode_blocks + 7) / 8 * 8;
    hipError_t e = launch_dtype<true, kTailPages>(dtype, G, a, st);
    if (e != hipSuccess) return e;
    return launch_merge_rows(dtype, a.dec, a.num_seqs, st);
}

}  // namespace femto
