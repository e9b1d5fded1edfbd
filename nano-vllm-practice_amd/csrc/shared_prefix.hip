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
// 256 sequences on 16384 keys, tails of up to 1024, 32/8 heads: 132 us, bound by
// both, the tails' 509 MB (92 us alone) and the tiles, 64 in series (104 alone);
// 64 on 4096, tails of up to 512, f16 16/8 heads 27.5 us; 8 on 1024 11.9 us, two
// launches and their round trips.
#include <cmath>

#include "attention_tiles.h"
#include "decode_merge.h"

namespace femto {

SharedPrefixPlan plan_shared_prefix(int num_seqs, int n_heads, int n_kv_heads, int prefix_pages, int max_kv_len,
                                    int dtype, int cus) {
    SharedPrefixPlan p{};
    const int n_rep = n_heads / n_kv_heads, G = prefill_group(n_rep), BT = 32 * (4 / G);
    const int tail = (int)std::max<int64_t>(1, (int64_t)max_kv_len - (int64_t)prefix_pages * kPage);
    p.tail = plan_paged_decode(n_heads, n_kv_heads, tail, dtype);
    if (prefix_pages <= 0) return p;
    // Pieces of the prefix: more of them shorten the tiles' chains (1.2 us per
    // tile of 64 keys where a CU has one), but each writes and merges 520
    // bytes per query row.  With T key tiles and R query rows the best of 2 .. 64
    // pieces was near 2 sqrt(T) / (1 + R / 24 / 128) over 160 shapes (3-256
    // sequences, prefixes of 256-16384 keys, five head shapes): 16384 keys, 16
    // sequences on 16/8 heads 28 us with 32, 31 with 16, 45 with 8; 256 on 64/8
    // heads 195 us with 4, 231 with 16; 4096 keys, 8 on 16/8 heads 15.2 with 16,
    // 16.6 with 12, 18.9 with 8.  Beyond one workgroup per CU beside the workers
    // (U row tiles, one workgroup each per piece) they only queue (4096 keys,
    // 256 sequences on 16/8 heads with tails of up to 512: 65 us with 4, 71 with
    // 8, 79 with 16).
    const int tiles = (prefix_pages * kPage + kKvTile - 1) / kKvTile;
    const double units = (double)(n_heads / G) * ((num_seqs + BT - 1) / BT), rows = (double)num_seqs * n_heads;
    const double best = std::min(2.0 * std::sqrt((double)tiles) / (1.0 + rows / (24.0 * 128)), std::max(4.0, cus / units));
    const int per = std::max({1, (tiles + 63) / 64, (int)(tiles / best + 0.5)});
    p.pieces = (tiles + per - 1) / per;
    p.piece_keys = per * kKvTile;
    // Long pieces beside short tails: their waves issue before the workers' on
    // the same SIMD.  32/8 heads, prefix of 16384 keys, tails of up to 1024, us
    // without and with: 256 sequences 141 and 135, 128 sequences 85 and 79, 64
    // 51.7 and 50.9; where the tails take as long, or pieces are short, it costs:
    // 8192 keys 115 and 118; 1024 keys, 64 sequences on 16/8 heads, tails of up to 64 17.1 and 18.9.
    p.longest = per >= 16 && prefix_pages * (int64_t)kPage >= 16 * (int64_t)tail;
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
