// Decode attention of a batch whose sequences share their first pages.
//
// Formula: out[h, b] = sum_j w_j v_j / sum_j w_j, w_j = exp(q[h, b] . k_j / sqrt(D)),
// over the prefix's keys j < min(kv_lens[b], 16 P) and the sequence's own from
// page P on.  The two sums have the same shape, so each is formed by the unit
// that it suits, relative to its own maximum, and a merge launch joins them:
//  * prefix: every K/V byte serves all sequences, so it is a matrix product of
//    the batch's query rows with the prefix, on the MFMA tiles of
//    attention_tiles.h, read from HBM once and not once per sequence.  It has
//    few query tiles (one per 32-128 sequences and KV head), so its keys are
//    cut into pieces, one workgroup each;
//  * tails: bound by their bytes, on the decode workers of decode_worker.h, in
//    the same launch, one workgroup per CU beside the tiles.
#include "attention_tiles.h"

namespace femto {

// One workgroup per (query head, sequence), one thread per head dim: the
// tail's slots, then the pieces of the prefix that hold keys of the sequence.
template <typename E>
__global__ __launch_bounds__(kDimHead) void shared_prefix_merge_kernel(DecodeArgs a) {
    __shared__ float s_m[kDimHead], s_l[kDimHead];
    const int h = blockIdx.x, b = blockIdx.y, t = threadIdx.x;
    const int kv_len = a.kv_lens[b];
    char* out = reinterpret_cast<char*>(a.out);
    const int64_t o = (int64_t)h * a.out_stride_head + (int64_t)b * a.out_stride_seq + t;
    if (kv_len <= 0) {  // an empty slot: zeros, as in a plain decode call
        if (t < a.head_dim) store_elem<E>(out, o, 0.0f);
        return;
    }
    const int tail = pages_seen<kTailPages>(a, kv_len, 0) > 0 ? a.seq_slots[b] : 0;
    const int prefix_keys = min(kv_len, a.first_page * kPage);
    const int count = tail + (prefix_keys > 0 ? (prefix_keys + a.prefix_piece_keys - 1) / a.prefix_piece_keys : 0);
    const int64_t sl0 = ((int64_t)b * a.n_heads + h) * slot_stride<kTailPages>(a);
    auto slot = [&](int i) { return sl0 + (i < tail ? i : a.max_slots + (i - tail)); };
    if (t < count) {
        s_m[t] = a.part_ml[slot(t) * 2];
        s_l[t] = a.part_ml[slot(t) * 2 + 1];
    }
    __syncthreads();
    float M = kEmptyMax;
    for (int i = 0; i < count; ++i) M = fmaxf(M, s_m[i]);
    float L = 0.0f, O = 0.0f;
    for (int i = 0; i < count; ++i) {
        const float w = fast_exp2(s_m[i] - M);
        L = fmaf(s_l[i], w, L);
        if (t < a.head_dim) O = fmaf(a.part_acc[slot(i) * kDimHead + t], w, O);
    }
    if (t < a.head_dim) store_elem<E>(out, o, O / L);
}

SharedPrefixPlan plan_shared_prefix(int num_seqs, int n_heads, int n_kv_heads, int prefix_pages, int max_kv_len,
                                    int dtype, int cus) {
    SharedPrefixPlan p{};
    const int n_rep = n_heads / n_kv_heads, G = prefill_group(n_rep), BT = 32 * (4 / G);
    const int tail = (int)std::max<int64_t>(1, (int64_t)max_kv_len - (int64_t)prefix_pages * kPage);
    p.tail = plan_paged_decode(n_heads, n_kv_heads, tail, dtype);
    p.tail.nrep_tile = G;
    if (prefix_pages <= 0) return p;
    const int tiles = (prefix_pages * kPage + kKvTile - 1) / kKvTile;
    const int64_t units = (int64_t)(n_heads / G) * ((num_seqs + BT - 1) / BT);
    const int pieces = (int)std::max<int64_t>(1, std::min<int64_t>({(int64_t)tiles, 2 * cus / units, 64}));
    const int per = (tiles + pieces - 1) / pieces;
    p.pieces = (tiles + per - 1) / per;
    p.piece_keys = per * kKvTile;
    return p;
}

hipError_t launch_shared_prefix(int dtype, PrefillArgs a, hipStream_t st) {
    if (a.num_seqs <= 0) return hipSuccess;
    const int G = prefill_group(a.n_rep), BT = 32 * (4 / G);
    a.head_groups = a.n_rep / G;
    a.tiles_per_group = (a.num_seqs + BT - 1) / BT;
    a.total_work = a.tiles_per_group * a.n_kv_heads * a.head_groups * a.dec.prefix_pieces;
    a.decode_blocks = decode_worker_blocks(a.dec);
    if (a.decode_blocks <= 0) return hipErrorInvalidDevice;
    a.decode_blocks = (a.decode_blocks + 7) / 8 * 8;
    hipError_t e = launch_dtype<true, kTailPages>(dtype, G, a, st);
    if (e != hipSuccess) return e;
    const dim3 grid(a.n_heads, a.num_seqs);
    switch (dtype) {
        case kDtypeBF16: hipLaunchKernelGGL(shared_prefix_merge_kernel<BF16>, grid, dim3(kDimHead), 0, st, a.dec); break;
        case kDtypeF16: hipLaunchKernelGGL(shared_prefix_merge_kernel<F16>, grid, dim3(kDimHead), 0, st, a.dec); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace femto
