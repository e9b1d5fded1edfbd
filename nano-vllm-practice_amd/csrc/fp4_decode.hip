// Decode over a KV cache held in 4 bits: the kernel of fp4_decode.h and its
// launches.
#include "fp4_decode.h"

namespace femto {

constexpr int kFp4Stages = 3;  // pairs of pages in registers, one of them computed

template <typename E, bool FULL, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2))) void fp4_decode_kernel(DecodeArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[W * kFp4WaveLds];
    __shared__ float s_ml[W][kMfmaHeads][2];
    __shared__ int s_old;
    fp4_row<E, FULL, W, kFp4Stages>(a, blockIdx.x, lds, s_ml, &s_old);
}

template <typename E, bool FULL>
static hipError_t launch_rows(const DecodeArgs& a, int num_seqs, hipStream_t st) {
    const int64_t grid = (int64_t)num_seqs * a.grid_heads * a.parts;
    if (grid > 0x7fffffff) return hipErrorInvalidValue;
    if (a.single_waves == 8) hipLaunchKernelGGL((fp4_decode_kernel<E, FULL, 8>), dim3((unsigned)grid), dim3(512), 0, st, a);
    else hipLaunchKernelGGL((fp4_decode_kernel<E, FULL, 4>), dim3((unsigned)grid), dim3(256), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_fp4_decode(int dtype, DecodeArgs a, int num_seqs, hipStream_t st) {
    if (num_seqs <= 0 || a.n_heads <= 0) return hipSuccess;
    if (a.head_dim <= 0 || a.head_dim > kDimHead || a.head_dim % 16) return hipErrorInvalidValue;
    set_mfma_heads(a);
    const bool full = a.head_dim == kDimHead;
    switch (dtype) {
        case kDtypeBF16: return full ? launch_rows<BF16, true>(a, num_seqs, st) : launch_rows<BF16, false>(a, num_seqs, st);
        case kDtypeF16: return full ? launch_rows<F16, true>(a, num_seqs, st) : launch_rows<F16, false>(a, num_seqs, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace femto
