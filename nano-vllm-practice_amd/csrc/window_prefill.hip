// Prefill under a sliding window with sinks: the tile kernel of
// attention_tiles.h with its window rule.
#include "attention_tiles.h"

namespace femto {

hipError_t launch_window_tiles(int dtype, int G, const PrefillArgs& a, hipStream_t st) {
    return launch_dtype<true, kWindowPages>(dtype, G, a, st);
}

}  // namespace femto
