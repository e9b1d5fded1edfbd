// Decode under a sliding window with sinks: the kernels of paged_decode.hip
// over the pages that the query sees.
//
// Sequence b's query stands at position kv_lens[b] - 1 and sees key j iff
// j < kv_lens[b] and (j >= kv_lens[b] - window or j < sinks).  The pages
// before the window that hold no sink are left out of the page list
// (PageList in decode_worker.h), so the slices of the split workers are equal
// in pages read, whatever the contexts: a call costs min(context, window +
// sinks) per sequence.  Only the last page, the sinks' last and the window's
// first mask rows.
#include "decode_kernels.h"

namespace femto {

hipError_t launch_window_decode_merge(int dtype, const DecodeArgs& a, int num_seqs, hipStream_t st) {
    return launch_merge_dtype<kWindowPages>(dtype, a, num_seqs, st);
}

hipError_t launch_window_decode(int dtype, const DecodeArgs& a, int nrep_tile, int num_seqs, bool single,
                                hipStream_t st) {
    return launch_decode_dtype<kWindowPages>(dtype, a, nrep_tile, num_seqs, single, st);
}

}  // namespace femto
