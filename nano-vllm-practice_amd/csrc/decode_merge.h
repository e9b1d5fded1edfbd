// Merge launch of a shared-prefix call's partial softmax states
// (shared_prefix.hip).
#pragma once

#include "decode_worker.h"

namespace femto {

// One wave per (sequence, query head), lane t holding dims 2t and 2t + 1: the
// workers' slots, then the pieces of the prefix that hold keys of the sequence.  Lane i keeps slot i's maximum and sum, so the weights of 64
// slots at a time cost one exponential and two wave reductions; the slots'
// outputs are loaded kMergeAhead at a time, before their weights are known.
// Slots are added in order: the result does not depend on which wave wrote last.
constexpr int kMergeRows = 4;    // waves per workgroup
constexpr int kMergeAhead = 16;  // slots in flight (12: 64 sequences on 4096 keys 2.6 % slower, 256 on 16384 0.5 %)

template <typename E>
__global__ __launch_bounds__(64 * kMergeRows) void merge_rows_kernel(DecodeArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t i = (int64_t)blockIdx.x * kMergeRows + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (i >= (int64_t)a.num_seqs * a.n_heads) return;  // no barriers below
    const int b = (int)(i / a.n_heads), h = (int)(i - (int64_t)b * a.n_heads);
    const int worker_slots = a.seq_slots[b];  // stale where no worker met the sequence
    const int kv_len = a.kv_lens[b];
    const int workers = pages_seen<kTailPages>(a, kv_len, 0) > 0 ? worker_slots : 0;
    const int prefix_keys = min(kv_len, a.first_page * kPage);
    const int count = workers + (prefix_keys > 0 ? (prefix_keys + a.prefix_piece_keys - 1) / a.prefix_piece_keys : 0);
    char* out = reinterpret_cast<char*>(a.out);
    const int64_t o = (int64_t)h * a.out_stride_head + (int64_t)b * a.out_stride_seq + 2 * lane;
    auto store = [&](float x, float y) __attribute__((always_inline)) {
        if (2 * lane < a.head_dim) {
            store_elem<E>(out, o, x);
            store_elem<E>(out, o + 1, y);
        }
    };
    if (count == 0) return store(0.0f, 0.0f);  // no key
    const int64_t sl0 = i * slot_stride<kTailPages>(a);
    auto slot = [&](int k) __attribute__((always_inline)) {
        return sl0 + (k < workers ? k : a.max_slots + (k - workers));
    };
    float M = kEmptyMax, L = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int base = 0; base < count; base += kWave) {
        const int n = min(kWave, count - base);
        float2 v[kMergeAhead];
        auto load = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < kMergeAhead; ++u)  // past the end: the last slot again, left out below
                v[u] = *reinterpret_cast<const float2*>(a.part_acc + slot(base + min(k0 + u, n - 1)) * kDimHead + 2 * lane);
        };
        load(0);
        float2 ml = make_float2(kEmptyMax, 0.0f);
        if (lane < n) ml = *reinterpret_cast<const float2*>(a.part_ml + slot(base + lane) * 2);
        const float Mn = fmaxf(M, wave_max_f32(ml.x));
        const float keep = fast_exp2(M - Mn);
        const float w = lane < n ? fast_exp2(ml.x - Mn) : 0.0f;
        L = fmaf(L, keep, wave_sum_f32(ml.y * w));
        o0 *= keep;
        o1 *= keep;
        M = Mn;
        for (int k0 = 0; k0 < n; k0 += kMergeAhead) {
            if (k0) load(k0);
#pragma unroll
            for (int u = 0; u < kMergeAhead; ++u) {
                if (k0 + u >= n) break;  // wave-uniform
                const float wu = lane_f32(w, k0 + u);
                o0 = fmaf(v[u].x, wu, o0);
                o1 = fmaf(v[u].y, wu, o1);
            }
        }
    }
    store(o0 / L, o1 / L);
}

static hipError_t launch_merge_rows(int dtype, const DecodeArgs& a, int num_seqs, hipStream_t st) {
    const dim3 grid((unsigned)(((int64_t)num_seqs * a.n_heads + kMergeRows - 1) / kMergeRows)), block(64 * kMergeRows);
    switch (dtype) {
        case kDtypeBF16: hipLaunchKernelGGL(merge_rows_kernel<BF16>, grid, block, 0, st, a); break;
        case kDtypeF16: hipLaunchKernelGGL(merge_rows_kernel<F16>, grid, block, 0, st, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace femto
