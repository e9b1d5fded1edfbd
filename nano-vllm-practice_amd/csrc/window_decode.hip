// Decode under a sliding window with sinks.
//
// Sequence b's query stands at position kv_lens[b] - 1 and sees key j iff
// j < kv_lens[b] and (j >= kv_lens[b] - window or j < sinks).  The pages
// before the window that hold no sink are left out of the page list
// (PageList in decode_worker.h), so the slices of the split workers are equal
// in pages read, whatever the contexts: a call costs min(context, window +
// sinks) per sequence.  Only the last page, the sinks' last and the window's
// first mask rows.  16-bit types run on the MFMA workers of mfma_decode.h, f32
// on those of paged_decode.hip.
#include "decode_kernels.h"
#include "decode_merge.h"
#include "mfma_decode.h"

namespace femto {

// Two pages of LDS per wave, one on its way (three or four: 1-4 % slower, as are
// eight waves per CU: more requests in flight than HBM takes).
constexpr int kStages = 2;

template <typename E, bool FULL>
__global__ __launch_bounds__(256) void window_decode_kernel(DecodeArgs a) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * kWorkerLds<kStages>];
    mfma_waves<E, FULL, kWindowPages, kStages>(a, blockIdx.x, lds);
}

// One workgroup of W waves per (sequence, KV head group), wave w taking the w-th
// of W contiguous shares of the pages; the waves fold their states through LDS
// (each over its own, done, pages), so no workspace and no merge launch are
// needed.  The window bounds the sequences' work, so that workgroups of whole
// sequences are balanced wherever there is one for every CU (window_plan in
// femto_attn_api.hip).
template <typename E, bool FULL, int W>
__global__ __launch_bounds__(64 * W) void window_decode_single_kernel(DecodeArgs a) {
    constexpr int kWaveLds = kWorkerLds<kStages>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[W * kWaveLds];
    __shared__ float s_ml[W][kMfmaHeads][2];
    static_assert(kWaveLds >= kMfmaHeads * kDimHead * 4, "a wave's outputs");
    const int b = blockIdx.x, grp = blockIdx.y;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kvh = grp / a.head_groups, hg = grp - kvh * a.head_groups;
    const int h0 = kvh * a.n_rep + hg * a.heads_per_wave;
    const int nh = min(a.heads_per_wave, a.n_rep - hg * a.heads_per_wave);
    int row, kv_len, start;
    decode_row_of<kWindowPages>(a, b, row, kv_len, start);
    const int npg = pages_seen<kWindowPages>(a, kv_len, start);
    const int per = (npg + W - 1) / W;
    const int lp0 = min(npg, wave * per), n = min(npg, lp0 + per) - lp0;
    uint8_t* own = lds + wave * kWaveLds;
    HeadState s;
    if (n > 0) mfma_segment<E, FULL, kWindowPages, kStages>(a, b, kv_len, start, lp0, n, row, h0, nh, (int64_t)kvh * a.pool_stride_head, own, s);
    else s.clear();
    if (c < nh) {
        float* acc = reinterpret_cast<float*>(own) + c * kDimHead + 4 * g;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4*>(acc + 16 * dt) = s.o[dt];
        if (g == 0) {
            s_ml[wave][c][0] = s.m;
            s_ml[wave][c][1] = s.l;
        }
    }
    __syncthreads();
    char* out = reinterpret_cast<char*>(a.out);
    for (int i = threadIdx.x; i < nh * kDimHead; i += 64 * W) {
        const int r = i / kDimHead, d = i - r * kDimHead;
        if (!FULL && d >= a.head_dim) continue;
        const int64_t o = (int64_t)(h0 + r) * a.out_stride_head + (int64_t)row * a.out_stride_seq + d;
        if (npg == 0) {  // empty context
            store_elem<E>(out, o, 0.0f);
            continue;
        }
        float M = kEmptyMax;
#pragma unroll
        for (int w = 0; w < W; ++w) M = fmaxf(M, s_ml[w][r][0]);
        float L = 0.0f, O = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = fast_exp2(s_ml[w][r][0] - M);
            L = fmaf(s_ml[w][r][1], f, L);
            O = fmaf(reinterpret_cast<const float*>(lds + w * kWaveLds)[r * kDimHead + d], f, O);
        }
        store_elem<E>(out, o, O / L);
    }
}

hipError_t launch_window_decode_merge(int dtype, const DecodeArgs& a, int num_seqs, hipStream_t st) {
    return launch_merge_rows<kWindowPages>(dtype, a, num_seqs, st);
}

template <typename E, bool FULL>
static hipError_t launch_mfma(int dtype, DecodeArgs a, int num_seqs, bool single, hipStream_t st) {
    set_mfma_heads(a);
    if (single) {
        const dim3 grid(num_seqs, a.grid_heads);
        if (a.single_waves == 8) hipLaunchKernelGGL((window_decode_single_kernel<E, FULL, 8>), grid, dim3(512), 0, st, a);
        else hipLaunchKernelGGL((window_decode_single_kernel<E, FULL, 4>), grid, dim3(256), 0, st, a);
        return hipGetLastError();
    }
    const int grid = decode_worker_blocks(a);
    if (grid <= 0) return hipErrorInvalidDevice;
    hipLaunchKernelGGL((window_decode_kernel<E, FULL>), dim3(grid), dim3(256), 0, st, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? launch_window_decode_merge(dtype, a, num_seqs, st) : e;
}

hipError_t launch_window_decode(int dtype, const DecodeArgs& a, int nrep_tile, int num_seqs, bool single,
                                hipStream_t st) {
    if (num_seqs <= 0 || a.n_heads <= 0) return hipSuccess;
    if (single && a.cu_seqlens) return hipErrorInvalidValue;  // decode calls only
    if (a.head_dim <= 0 || a.head_dim > kDimHead) return hipErrorInvalidValue;
    const bool full = a.head_dim == kDimHead;
    switch (dtype) {
        case kDtypeBF16: return full ? launch_mfma<BF16, true>(dtype, a, num_seqs, single, st)
                                     : launch_mfma<BF16, false>(dtype, a, num_seqs, single, st);
        case kDtypeF16: return full ? launch_mfma<F16, true>(dtype, a, num_seqs, single, st)
                                    : launch_mfma<F16, false>(dtype, a, num_seqs, single, st);
        case kDtypeF32: return full ? launch_e<F32, true, kWindowPages>(a, nrep_tile, num_seqs, single, st)
                                    : launch_e<F32, false, kWindowPages>(a, nrep_tile, num_seqs, single, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace femto
