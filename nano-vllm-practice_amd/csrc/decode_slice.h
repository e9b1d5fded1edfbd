// A split decode worker's share of the pages (host and device code, no HIP header).
#pragma once

#include <cstdint>

#ifdef __HIP__
#define FEMTO_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define FEMTO_HOST_DEVICE inline
#endif

namespace femto {

// Pages [begin, end) of the wi-th slice of C pages of `total`; false: none.  C
// follows the caller's max_kv_len, which may be far above the real lengths, so
// wi * C does not fit 32 bits (1023 * 4194304 for a max_kv_len of 2^31 - 1).
FEMTO_HOST_DEVICE bool slice_pages(int wi, int C, int total, int& begin, int& end) {
    const int64_t x = (int64_t)wi * C;
    if (x >= total) return false;
    begin = (int)x;
    end = total - begin <= C ? total : begin + C;
    return true;
}

}  // namespace femto
