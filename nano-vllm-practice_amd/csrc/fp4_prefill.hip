// Prefill over a KV cache held in 4 bits: the tile kernel of attention_tiles.h
// with its 4-bit rule.
//
// Formula: out[h, t] = sum_j w_j v_j / sum_j w_j, w_j = exp(q[h, t] . k_j / sqrt(D)),
// over the keys j < kv_len, j <= p, p the token's position; k and v are the
// values that the cache stands for.
#include "attention_tiles.h"

namespace femto {

hipError_t launch_fp4_tiles(int dtype, int G, const PrefillArgs& a, hipStream_t st) {
    return launch_dtype<true, kFp4Pages>(dtype, G, a, st);
}

}  // namespace femto
