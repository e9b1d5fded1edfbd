// Decode under a sliding window with sinks.
//
// Sequence b's query stands at position kv_lens[b] - 1 and sees key j iff
// j < kv_lens[b] and (j >= kv_lens[b] - window or j < sinks).  The pages
// before the window that hold no sink are left out of the page list
// (PageList in decode_worker.h): a call costs min(context, window + sinks) per
// sequence, and only the last page, the sinks' last and the window's first mask
// rows.  The window also bounds what sequences differ by, so 16-bit types run
// as whole rows (window_row in mfma_decode.h), a workgroup per (sequence, KV
// head group), or a few of them where there would be fewer than CUs.  f32 runs
// on the kernels of paged_decode.hip.
//
// Bound by the bytes of K and V where the batch fills the chip: 61 sequences,
// window 2048, 16/8 heads (491 MB) 77 us, 6.4 TB/s; 16 sequences, window 4096, f16
// 32/8 heads (269 MB) 45.6 us, 5.9 TB/s, one workgroup per CU.  One sequence of 1028
// keys: 8.5 us, the launch and the round trips table, pages, states, count, states.
#include "decode_kernels.h"
#include "mfma_decode.h"

namespace femto {

// Two pages of LDS per wave, one on its way (three or four: 1-4 % slower: more
// requests in flight than HBM takes).
constexpr int kStages = 2;

template <typename E, bool FULL, int W>
__global__ __launch_bounds__(64 * W) void window_decode_kernel(DecodeArgs a) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[W * kWorkerLds<kStages>];
    __shared__ float s_ml[W][kMfmaHeads][2];
    __shared__ int s_old;
    window_row<E, FULL, W, kStages>(a, blockIdx.x, lds, s_ml, &s_old);
}

template <typename E, bool FULL>
static hipError_t launch_rows(DecodeArgs a, int num_seqs, hipStream_t st) {
    set_mfma_heads(a);
    const int64_t grid = (int64_t)num_seqs * a.grid_heads * a.parts;
    if (grid > 0x7fffffff) return hipErrorInvalidValue;
    if (a.single_waves == 8) hipLaunchKernelGGL((window_decode_kernel<E, FULL, 8>), dim3((unsigned)grid), dim3(512), 0, st, a);
    else hipLaunchKernelGGL((window_decode_kernel<E, FULL, 4>), dim3((unsigned)grid), dim3(256), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_window_decode(int dtype, const DecodeArgs& a, int nrep_tile, int num_seqs, bool single,
                                hipStream_t st) {
    if (num_seqs <= 0 || a.n_heads <= 0) return hipSuccess;
    if (single && a.cu_seqlens) return hipErrorInvalidValue;  // decode calls only
    if (a.head_dim <= 0 || a.head_dim > kDimHead) return hipErrorInvalidValue;
    const bool full = a.head_dim == kDimHead;
    switch (dtype) {
        case kDtypeBF16: return full ? launch_rows<BF16, true>(a, num_seqs, st) : launch_rows<BF16, false>(a, num_seqs, st);
        case kDtypeF16: return full ? launch_rows<F16, true>(a, num_seqs, st) : launch_rows<F16, false>(a, num_seqs, st);
        case kDtypeF32: return full ? launch_e<F32, true, kWindowPages>(a, nrep_tile, num_seqs, single, st)
                                    : launch_e<F32, false, kWindowPages>(a, nrep_tile, num_seqs, single, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace femto
