// Prefill under a sliding window with sinks: the tile kernel of
// attention_tiles.h with its window rule.
//
// Formula: out[h, t] = sum_j w_j v_j / sum_j w_j, w_j = exp(q[h, t] . k_j / sqrt(D)),
// over the keys j < kv_len, j <= p with j > p - window or j < sinks, p the
// token's position.  The tiles between the sinks and the window are left out,
// so long chunks are bound by the tile loop as without a window: 2048 tokens
// at position 30720, window 4096, 32/8 heads 138 us, 998 TFLOP/s, 5.3 VALU
// instructions per MFMA.  Short windows pay for the tiles that cross the
// window's start: 8 x 512 tokens, window 1024, 16/8 heads 48.6 us, 674 TFLOP/s, five of
// a query tile's 18 key tiles masked.  A chunk of 1024 beside 127 rows, window 1024,
// 32/8 heads: 100 us, 5.5 TB/s (one launch, see window_row in mfma_decode.h).
#include "attention_tiles.h"

namespace femto {

hipError_t launch_window_tiles(int dtype, int G, const PrefillArgs& a, hipStream_t st) {
    return launch_dtype<true, kWindowPages>(dtype, G, a, st);
}

}  // namespace femto
