// Decode over a KV cache held in 4 bits: the kernel of fp4_decode.h and its
// launches.
//
// Measured (bf16 of 128 dims; a call of many, us): bound by memory, 61 sequences of
// 256-16384 keys, 16/8 heads, 90.0 (556 MB at 6.2 TB/s: split kernel 84, merge 4.5),
// 256 of 1024-8192, 32/8, 199.9 (1.22 GB at 6.1 TB/s); f16, 16 of 8192-32768, 32/8,
// 65.1 (5.7 TB/s).  The matrix units are busy 15 % of that.  One sequence of 5000
// keys 9.6, bound by latency: table, pages, states to memory, count, states back.
// Of fewer dims the lanes of absent blocks load block 0 again: the 61 and the 256
// sequences of 64 dims 71 and 147 (3.9 and 4.1 TB/s), of 80 77 and 162.
#include <algorithm>

#include "fp4_decode.h"

namespace femto {

// Pairs of pages in registers, one of them computed (three: 2 % slower).
constexpr int kFp4Stages = 2;
// Split workers: waves per CU (6: 4 % slower, 4 18 %, 10 or more 3-8 %).
constexpr int kFp4SplitWaves = 8;

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

template <typename E, bool FULL>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void fp4_split_kernel(DecodeArgs a) {
    fp4_waves<E, FULL, kFp4Stages>(a, blockIdx.x);
}

template <typename E, bool FULL>
static hipError_t launch_split(int dtype, DecodeArgs a, int num_seqs, hipStream_t st) {
    int cus = 0;
    hipError_t e = device_cu_count(cus);
    if (e != hipSuccess) return e;
    a.waves_per_group = std::max(1, cus * kFp4SplitWaves / a.grid_heads);
    const int grid = (a.waves_per_group * a.grid_heads + 3) / 4;
    hipLaunchKernelGGL((fp4_split_kernel<E, FULL>), dim3(grid), dim3(256), 0, st, a);
    e = hipGetLastError();
    return e == hipSuccess ? launch_paged_decode_merge(dtype, a, num_seqs, st) : e;
}

hipError_t launch_fp4_split(int dtype, DecodeArgs a, int num_seqs, hipStream_t st) {
    if (num_seqs <= 0 || a.n_heads <= 0) return hipSuccess;
    if (a.head_dim <= 0 || a.head_dim > kDimHead || a.head_dim % 16) return hipErrorInvalidValue;
    set_mfma_heads(a);
    const bool full = a.head_dim == kDimHead;
    switch (dtype) {
        case kDtypeBF16: return full ? launch_split<BF16, true>(dtype, a, num_seqs, st) : launch_split<BF16, false>(dtype, a, num_seqs, st);
        case kDtypeF16: return full ? launch_split<F16, true>(dtype, a, num_seqs, st) : launch_split<F16, false>(dtype, a, num_seqs, st);
        default: return hipErrorInvalidValue;
    }
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
