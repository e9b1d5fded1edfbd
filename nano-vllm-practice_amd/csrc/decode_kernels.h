// Decode kernels (paged_decode.hip says how they work) and their launches, by
// page rule: paged_decode.hip instantiates the plain rule, window_decode.hip
// the window's.
#pragma once

#include "decode_worker.h"

namespace femto {

template <typename E, int NREP, bool FULL, int RULE>
__global__ __launch_bounds__(256) void paged_decode_kernel(DecodeArgs a) {
    decode_waves<E, NREP, FULL, false, RULE>(a, blockIdx.x);
}

// One-launch decode for calls of short contexts: one workgroup of W waves per
// (sequence, KV head group), wave w taking the w-th of W contiguous shares
// of the sequence's pages; the waves fold their states through LDS and
// write the normalised rows, so no workspace and no merge launch are needed.
// Decode calls only (query row b, kv_lens[b] keys).  W = 8 lets each wave walk
// half as many pages, whose chain of loads and math sets the length of a call
// of one workgroup per CU; with more workgroups than CUs it takes more rounds
// (64 sequences of up to 512 keys on 16/8 heads 18.6 us with four waves, 21.6
// with eight).  decode_route picks.
template <typename E, int NREP, bool FULL, int W, int RULE>
__global__ __launch_bounds__(64 * W) void paged_decode_single_kernel(DecodeArgs a) {
    __shared__ float s_ml[W][NREP][2];
    __shared__ float s_acc[W][NREP][kDimHead];
    const int b = blockIdx.x, grp = blockIdx.y;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int c = lane & 15, rg = lane >> 4;
    const int kvh = grp / a.head_groups;
    const int h0 = kvh * a.n_rep + (grp - kvh * a.head_groups) * NREP;
    const int kv_len = a.kv_lens[b];
    const int start = RULE == kWindowPages ? max(0, max(kv_len, 0) - a.window) : 0;
    const int npg = pages_seen<RULE>(a, kv_len, start);
    const int per = (npg + W - 1) / W;
    const int lp0 = min(npg, wave * per), lp1 = min(npg, lp0 + per);
    float m[NREP], l[NREP], acc[NREP][8];
    if (lp1 > lp0) {
        decode_segment<E, NREP, FULL, RULE>(a, b, kv_len, start, lp0, lp1 - lp0, b, h0,
                                            (int64_t)kvh * a.pool_stride_head, m, l, acc);
    } else {
#pragma unroll
        for (int r = 0; r < NREP; ++r) {
            m[r] = kEmptyMax;
            l[r] = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[r][e] = 0.0f;
        }
    }
    if (rg == 0) {
#pragma unroll
        for (int r = 0; r < NREP; ++r) {
#pragma unroll
            for (int e = 0; e < 8; ++e) s_acc[wave][r][RowSlice<E>::dim(c, e)] = acc[r][e];
            if (c == 0) {
                s_ml[wave][r][0] = m[r];
                s_ml[wave][r][1] = l[r];
            }
        }
    }
    __syncthreads();
    char* out = reinterpret_cast<char*>(a.out);
    for (int i = threadIdx.x; i < NREP * kDimHead; i += 64 * W) {
        const int r = i / kDimHead, d = i - r * kDimHead;
        if (!FULL && d >= a.head_dim) continue;
        const int64_t o = (int64_t)(h0 + r) * a.out_stride_head + (int64_t)b * a.out_stride_seq + d;
        if (npg == 0) {  // empty context: the reference stores its zero accumulator
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
            O = fmaf(s_acc[w][r][d], f, O);
        }
        store_elem<E>(out, o, O / L);
    }
}

// Final softmax merge: one workgroup per (sequence, query head), one thread
// per head dim.  Runs after the split kernel on the same stream.
template <typename E, int RULE>
__global__ __launch_bounds__(128) void paged_decode_merge_kernel(DecodeArgs a) {
    __shared__ float s_w[128];  // slot maxima
    __shared__ float s_lv[128];  // slot sums
    const int h = blockIdx.x;
    const int b = blockIdx.y;
    const int t = threadIdx.x;
    char* out = reinterpret_cast<char*>(a.out);
    int row, kvl, start;
    if (!decode_row_of<RULE>(a, b, row, kvl, start)) return;  // a prefill row (whole workgroup)
    const int64_t o = (int64_t)h * a.out_stride_head + (int64_t)row * a.out_stride_seq + t;
    const int64_t sl0 = ((int64_t)b * a.n_heads + h) * a.max_slots;
    const float* src = a.part_acc + sl0 * kDimHead + t;
    // Every load that does not depend on another is issued first: kv_len,
    // the slot count, (m, l) of every slot this (sequence, head) may own and
    // the accumulators of its first kSpec slots (a sequence usually spans a
    // few slices).  Entries past the count are stale and are masked below.
    constexpr int kSpec = 4;
    const int count_ld = a.seq_slots[b];
    const float m_ld = t < a.max_slots ? a.part_ml[(sl0 + t) * 2] : kEmptyMax;
    const float l_ld = t < a.max_slots ? a.part_ml[(sl0 + t) * 2 + 1] : 0.0f;
    float v[kSpec];
#pragma unroll
    for (int i = 0; i < kSpec; ++i) v[i] = i < a.max_slots ? src[(int64_t)i * kDimHead] : 0.0f;
    if (pages_seen<RULE>(a, kvl, start) == 0) {
        // Empty context.  Decode call: the reference's P.V loop never runs
        // and its zero accumulator is stored (paged_attention_gemv.cu:203-218).
        // Decode row of a prefill call: 0 / 0, NaN, as the prefill kernels
        // give for a row with no visible key.
        if (t < a.head_dim) store_elem<E>(out, o, a.cu_seqlens ? __builtin_nanf("") : 0.0f);
        return;
    }
    const int count = count_ld;
    // Thread i < count publishes slot i's (m, l); after one barrier every
    // thread folds the count slots itself (a sequence spans a few slices,
    // at most max_slots <= 128), so no further reduction round is needed.
    if (t < count) {
        s_w[t] = m_ld;
        s_lv[t] = l_ld;
    }
    __syncthreads();
    float M = kEmptyMax;
    for (int i = 0; i < count; ++i) M = fmaxf(M, s_w[i]);
    float L = 0.0f, O = 0.0f;
#pragma unroll
    for (int i = 0; i < kSpec; ++i) {
        const float wi = i < count ? fast_exp2(s_w[i < count ? i : 0] - M) : 0.0f;
        L = fmaf(i < count ? s_lv[i] : 0.0f, wi, L);
        O = fmaf(i < count ? v[i] : 0.0f, wi, O);
    }
    for (int i = kSpec; i < count; ++i) {
        const float wi = fast_exp2(s_w[i] - M);
        L = fmaf(s_lv[i], wi, L);
        O = fmaf(src[(int64_t)i * kDimHead], wi, O);
    }
    if (t < a.head_dim) store_elem<E>(out, o, O / L);
}

template <typename E, int RULE>
static hipError_t launch_merge_t(const DecodeArgs& a, int num_seqs, hipStream_t st) {
    hipLaunchKernelGGL((paged_decode_merge_kernel<E, RULE>), dim3(a.n_heads, num_seqs), dim3(kDimHead), 0, st, a);
    return hipGetLastError();
}

template <int RULE>
static hipError_t launch_merge_dtype(int dtype, const DecodeArgs& a, int num_seqs, hipStream_t st) {
    switch (dtype) {
        case kDtypeF32: return launch_merge_t<F32, RULE>(a, num_seqs, st);
        case kDtypeF16: return launch_merge_t<F16, RULE>(a, num_seqs, st);
        case kDtypeBF16: return launch_merge_t<BF16, RULE>(a, num_seqs, st);
        default: return hipErrorInvalidValue;
    }
}

template <typename E, int NREP, bool FULL, int RULE>
static hipError_t launch_t(DecodeArgs a, int num_seqs, bool single, hipStream_t st) {
    if (single) {
        const dim3 grid(num_seqs, a.grid_heads);
        if constexpr (NREP == 1 || (NREP <= 4 && !std::is_same<E, F32>::value)) {
            if (a.single_waves == 8) {
                hipLaunchKernelGGL((paged_decode_single_kernel<E, NREP, FULL, 8, RULE>), grid, dim3(512), 0, st, a);
                return hipGetLastError();
            }
        }
        if (a.single_waves != 4) return hipErrorInvalidValue;
        hipLaunchKernelGGL((paged_decode_single_kernel<E, NREP, FULL, 4, RULE>), grid, dim3(256), 0, st, a);
        return hipGetLastError();
    }
    const int grid = decode_worker_blocks(a);
    if (grid <= 0) return hipErrorInvalidDevice;
    hipLaunchKernelGGL((paged_decode_kernel<E, NREP, FULL, RULE>), dim3(grid), dim3(256), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return launch_merge_t<E, RULE>(a, num_seqs, st);
}

template <typename E, bool FULL, int RULE>
static hipError_t launch_e(const DecodeArgs& a, int nrep_tile, int num_seqs, bool single, hipStream_t st) {
    switch (nrep_tile) {
        case 1: return launch_t<E, 1, FULL, RULE>(a, num_seqs, single, st);
        case 2: return launch_t<E, 2, FULL, RULE>(a, num_seqs, single, st);
        case 4: return launch_t<E, 4, FULL, RULE>(a, num_seqs, single, st);
        case 8:
            if constexpr (!std::is_same<E, F32>::value) return launch_t<E, 8, FULL, RULE>(a, num_seqs, single, st);
            return hipErrorInvalidValue;  // f32 plans stop at 4 heads per wave
        default: return hipErrorInvalidValue;
    }
}

template <int RULE>
static hipError_t launch_decode_dtype(int dtype, const DecodeArgs& a, int nrep_tile, int num_seqs, bool single,
                                      hipStream_t st) {
    if (num_seqs <= 0 || a.grid_heads <= 0) return hipSuccess;
    if (single && a.cu_seqlens) return hipErrorInvalidValue;  // decode calls only
    if (a.head_dim <= 0 || a.head_dim > kDimHead) return hipErrorInvalidValue;
    const bool full = a.head_dim == kDimHead;
    switch (dtype) {
        case kDtypeF32: return full ? launch_e<F32, true, RULE>(a, nrep_tile, num_seqs, single, st)
                                    : launch_e<F32, false, RULE>(a, nrep_tile, num_seqs, single, st);
        case kDtypeF16: return full ? launch_e<F16, true, RULE>(a, nrep_tile, num_seqs, single, st)
                                    : launch_e<F16, false, RULE>(a, nrep_tile, num_seqs, single, st);
        case kDtypeBF16: return full ? launch_e<BF16, true, RULE>(a, nrep_tile, num_seqs, single, st)
                                     : launch_e<BF16, false, RULE>(a, nrep_tile, num_seqs, single, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace femto
