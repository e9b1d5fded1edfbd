// Prefill over a KV cache held in 4 bits: the tile kernel of attention_tiles.h
// with its 4-bit rule.
//
// Formula: out[h, t] = sum_j w_j v_j / sum_j w_j, w_j = exp(q[h, t] . k_j / sqrt(D)),
// over the keys j < kv_len, j <= p, p the token's position; k and v are the
// values that the cache stands for.
//
// Measured (bf16 of 128 dims, us): 2048 tokens behind 30720, 32/8 heads, 858-890
// (1.20-1.24 PFLOP/s; the kernel over a 16-bit cache 960), bound by issue: 6.2 VALU
// instructions per MFMA, the matrix units busy 48 %, and by the clock (inputs of
// zeros -22 %); 8 x 512 tokens, 16/8, 72, bound by the longest query tile's 40 key
// tiles in series; 1024 behind 4096 beside 127 rows, 32/8, 165-168, memory (646 MB)
// and tiles on the same CUs; f16, a prompt of 777, 16/8, 20.2, latency.  With a large
// channel of q in every wave (fp4_query_large) 2048 behind 30720 take 989.  Heads of
// fewer dims take as long, the absent ones' products being made with zeros: of 64
// the long chunk 832, 8 x 512 76 where 128 takes 79.
#include "attention_tiles.h"

namespace femto {

hipError_t launch_fp4_tiles(int dtype, int G, const PrefillArgs& a, hipStream_t st) {
    return launch_dtype<true, kFp4Pages>(dtype, G, a, st);
}

}  // namespace femto
