// Rotary positions of q and k, with the KV-cache write of the rotated k and of
// v, for heads without norms.
//
// Formula: the first R of a head's D dims are R / 2 pairs (a, b); the token's
// position p selects row p of the caller's fp32 tables, and
//     a' = a cos[p][i] - b sin[p][i],   b' = b cos[p][i] + a sin[p][i]
// for pair i: dims (i, i + R / 2) in the half layout, (2i, 2i + 1) interleaved.
// Dims from R on pass through.  Scalings for long contexts live in the tables.
// In fp32, one rounding per output.  A position outside the tables gives NaN in
// the rotated dims.  The cache write follows kv_cache_write.hip: sequence b's
// tokens go to positions[q_begin] + 0, 1, ..., up to the first table column
// that is -1, past the table or outside the pool.
//
// Work: one wave per token, no barriers and no LDS.  A head row is cut into
// items of two 16-byte chunks, one lane each: in the half layout the two
// chunks that hold both ends of the same pairs, else neighbours.  So every
// pair is inside a lane, and lane i's table fragment (the 2 x 8 floats of pairs
// 8i .. 8i + 7; 2 x 4 for f32) is loaded once and serves all H + KVH rows of
// the token.  The wave's rows move in batches of kRowBatch loads per lane in
// flight; the placement's table columns are looked up by the whole wave while
// the first batch is on its way.  Half layouts whose R / 2 is no whole number of
// chunks (R = 24 in 16-bit types) take each row's partner elements one by one
// from memory, which the wave has read before it stores the row (the output may
// be q itself).
//
// Bound by its bytes: 8 x 512 tokens of 32/8 bf16 heads (103 MB) take 20.5 us a
// call, 5.02 TB/s, a plain copy's rate.  Stores are non-temporal: the launch
// does not end with dirty lines to write back (24.5 us with ordinary ones;
// non-temporal loads besides 21.8).  Followed by the attention that reads q
// and the pages the two take as long either way.  64 tokens: 5.6 us, the launch
// and three dependent round trips.  Where an item's two chunks are neighbours a
// store writes every other 16 bytes of a line, and the L2 passes some on by halves
// (79 MB written to HBM for 50): the same tokens interleaved 31.6 us, with R = 32
// 29.4, with R = 24 (and partners one by one) 35.9.  1024 tokens beside
// 127 of one token each: 30.6 us, 7.8 without them, for workgroups without a token.
#include "common.h"
#include "launch.h"

namespace femto {

constexpr int kRopeTokens = 4;  // waves per workgroup
constexpr int kRowBatch = 6;    // rows per lane in flight

enum RopePairs { kInterleaved, kHalfChunks, kHalfAny };

template <typename E>
struct Chunk;  // 16 bytes as floats
template <>
struct Chunk<BF16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(u32x4 w, float* f) { unpack8(BF16{}, w, *reinterpret_cast<float(*)[8]>(f)); }
    static __device__ __forceinline__ u32x4 put(const float* f) { return pack8(BF16{}, *reinterpret_cast<const float(*)[8]>(f)); }
    static __device__ __forceinline__ float elem(const char* p) { return (float)*reinterpret_cast<const __bf16*>(p); }
};
template <>
struct Chunk<F16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(u32x4 w, float* f) { unpack8(F16{}, w, *reinterpret_cast<float(*)[8]>(f)); }
    static __device__ __forceinline__ u32x4 put(const float* f) { return pack8(F16{}, *reinterpret_cast<const float(*)[8]>(f)); }
    static __device__ __forceinline__ float elem(const char* p) { return (float)*reinterpret_cast<const _Float16*>(p); }
};
template <>
struct Chunk<F32> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(u32x4 w, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
    }
    static __device__ __forceinline__ u32x4 put(const float* f) {
        return u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    }
    static __device__ __forceinline__ float elem(const char* p) { return *reinterpret_cast<const float*>(p); }
};

template <typename E, int PAIRS>
__global__ __launch_bounds__(64 * kRopeTokens) void rope_cache_write_kernel(RopeArgs a) {
    constexpr int EB = E::kBytes, N = Chunk<E>::N;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.y;
    int q_begin, q_end;
    if (a.cw.cu_seqlens) {
        q_begin = a.cw.cu_seqlens[b];
        q_end = a.cw.cu_seqlens[b + 1];
    } else {  // decode: one token per sequence
        q_begin = b;
        q_end = b + 1;
    }
    const int R = a.rotary_dim, half = R / 2;
    const int chunks = a.cw.row_chunks;
    const int i = lane & (a.row_lanes - 1);         // item of the row
    const int row0 = lane >> a.row_shift;           // first row of the lane
    const int rows_per_pass = 64 >> a.row_shift;
    // The item's chunks: both ends of pairs N i .. N i + N - 1, then (dims past
    // R) neighbours; c1 == chunks: none.
    int c0, c1;
    if (PAIRS == kHalfChunks && i < half / N) {
        c0 = i;
        c1 = i + half / N;
    } else {
        c0 = 2 * i;
        c1 = 2 * i + 1;
    }
    const bool has0 = i < a.row_lanes && c0 < chunks, has1 = has0 && c1 < chunks;
    const int H = a.n_heads, KVH = a.cw.n_kv_heads, rows = H + 2 * KVH;
    const int32_t* table = a.cw.tables + (int64_t)b * a.cw.table_stride;

    // max_q_len only sizes the grid: longer sequences take more rounds.
    for (int t = q_begin + (int)blockIdx.x * kRopeTokens + wave; t < q_end; t += (int)gridDim.x * kRopeTokens) {
        const char* src[3] = {static_cast<const char*>(a.q) + (int64_t)t * a.q_stride_token * EB,
                              static_cast<const char*>(a.cw.k) + (int64_t)t * a.cw.k_stride_token * EB,
                              static_cast<const char*>(a.cw.v) + (int64_t)t * a.cw.v_stride_token * EB};
        auto row_ptr = [&](int r) __attribute__((always_inline)) {
            const int s = r < H ? 0 : r < H + KVH ? 1 : 2;
            const int64_t hs = s == 0 ? a.q_stride_head : s == 1 ? a.cw.k_stride_head : a.cw.v_stride_head;
            const char* base = s == 0 ? src[0] : s == 1 ? src[1] : src[2];
            return base + (int64_t)(s == 0 ? r : s == 1 ? r - H : r - H - KVH) * hs * EB;
        };
        u32x4 w0[kRowBatch], w1[kRowBatch];
        auto load = [&](int base) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < kRowBatch; ++u) {
                const int r = base + u * rows_per_pass + row0;
                if (r < rows) {
                    const char* p = row_ptr(r);
                    if (has0) w0[u] = ld16(p + c0 * 16);
                    if (has1) w1[u] = ld16(p + c1 * 16);
                }
            }
        };
        load(0);

        // Placement: block of the token's cache row, -1 where the walk ends before it.
        const int p0 = a.cw.positions[q_begin];
        const int pc = p0 + (t - q_begin);
        const int col = pc / kPage;
        int blk = -1;
        if (p0 >= 0 && pc >= 0) {  // (pc wraps past 2^31: not written)
            uint64_t ends = 0;
            for (int c = p0 / kPage; c <= col; c += 64) {
                const int id = c + lane <= col && c + lane < a.cw.num_pages_per_seq ? table[c + lane] : -1;
                ends |= __ballot(c + lane <= col && (id < 0 || (int64_t)id >= a.cw.num_blocks));
                if (c + 64 > col) blk = __builtin_amdgcn_readlane(id, col - c);
            }
            if (ends) blk = -1;
        }
        const int64_t slot = (int64_t)blk * a.cw.pool_stride_block + (int64_t)(pc % kPage) * a.cw.pool_stride_row;

        // The lane's table fragment.
        constexpr int F = PAIRS == kHalfAny ? 2 * N : N;
        float cs[F], sn[F];
        const int pos = a.cw.positions[t];
        const bool in_tables = pos >= 0 && pos < a.rope_rows;
        const float* ct = a.cos + (int64_t)(in_tables ? pos : 0) * a.rope_stride;
        const float* st = a.sin + (int64_t)(in_tables ? pos : 0) * a.rope_stride;
        if (PAIRS != kHalfAny && a.table_vectors && N * i + N <= half) {
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                *reinterpret_cast<u32x4*>(cs + e) = ld16(ct + N * i + e);
                *reinterpret_cast<u32x4*>(sn + e) = ld16(st + N * i + e);
            }
        } else {
#pragma unroll
            for (int e = 0; e < F; ++e) {
                // kHalfAny: element e of the item's 2 N dims; else pair N i + e
                int j = F * i + e;
                if (PAIRS == kHalfAny && j >= half) j -= half;
                const bool in = PAIRS == kHalfAny ? F * i + e < R : j < half;
                cs[e] = in ? ct[j] : 1.0f;
                sn[e] = in ? st[j] : 0.0f;
            }
        }
        if (!in_tables) {
#pragma unroll
            for (int e = 0; e < F; ++e) cs[e] = sn[e] = __builtin_nanf("");
        }

        for (int base = 0; base < rows; base += kRowBatch * rows_per_pass) {
            if (base) load(base);
#pragma unroll
            for (int u = 0; u < kRowBatch; ++u) {
                const int r = base + u * rows_per_pass + row0;
                if (r >= rows || !has0) continue;
                if (r < H + KVH) {
                    float x[2 * N];
                    Chunk<E>::get(w0[u], x);
                    if (has1) Chunk<E>::get(w1[u], x + N);
                    if constexpr (PAIRS == kHalfChunks) {
                        if (N * i < half) {
#pragma unroll
                            for (int e = 0; e < N; ++e) {
                                const float p = x[e], q = x[N + e];
                                x[e] = fmaf(p, cs[e], -(q * sn[e]));
                                x[N + e] = fmaf(q, cs[e], p * sn[e]);
                            }
                        }
                    } else if constexpr (PAIRS == kInterleaved) {
#pragma unroll
                        for (int e = 0; e < N; ++e) {
                            const float p = x[2 * e], q = x[2 * e + 1];
                            const bool in = N * i + e < half;
                            x[2 * e] = in ? fmaf(p, cs[e], -(q * sn[e])) : p;
                            x[2 * e + 1] = in ? fmaf(q, cs[e], p * sn[e]) : q;
                        }
                    } else {
                        const char* p = row_ptr(r);
#pragma unroll
                        for (int e = 0; e < 2 * N; ++e) {
                            const int d = 2 * N * i + e;
                            if (d >= R) continue;
                            const float y = Chunk<E>::elem(p + (d < half ? d + half : d - half) * EB);
                            x[e] = d < half ? fmaf(x[e], cs[e], -(y * sn[e])) : fmaf(x[e], cs[e], y * sn[e]);
                        }
                    }
                    w0[u] = Chunk<E>::put(x);
                    if (has1) w1[u] = Chunk<E>::put(x + N);
                }
                char* dst;
                if (r < H) {
                    dst = static_cast<char*>(a.q_out) + ((int64_t)t * a.q_out_stride_token + (int64_t)r * a.q_out_stride_head) * EB;
                } else {
                    if (blk < 0) continue;
                    const int h = r < H + KVH ? r - H : r - H - KVH;
                    dst = static_cast<char*>(r < H + KVH ? a.cw.k_pool : a.cw.v_pool) + (slot + (int64_t)h * a.cw.pool_stride_head) * EB;
                }
                st16_nt(dst + c0 * 16, w0[u]);
                if (has1) st16_nt(dst + c1 * 16, w1[u]);
            }
        }
    }
}

template <typename E>
static hipError_t launch_rope_t(const RopeArgs& a, dim3 grid, hipStream_t st) {
    const dim3 block(64 * kRopeTokens);
    if (a.interleaved) {
        hipLaunchKernelGGL((rope_cache_write_kernel<E, kInterleaved>), grid, block, 0, st, a);
    } else if (a.rotary_dim / 2 % Chunk<E>::N == 0) {
        hipLaunchKernelGGL((rope_cache_write_kernel<E, kHalfChunks>), grid, block, 0, st, a);
    } else {
        hipLaunchKernelGGL((rope_cache_write_kernel<E, kHalfAny>), grid, block, 0, st, a);
    }
    return hipGetLastError();
}

hipError_t launch_rope_cache_write(int dtype, RopeArgs a, int max_q_len, hipStream_t st) {
    if (a.cw.num_seqs <= 0 || max_q_len <= 0) return hipSuccess;
    const int items = (a.cw.row_chunks + 1) / 2;
    a.row_shift = 0;
    while ((1 << a.row_shift) < items) ++a.row_shift;
    a.row_lanes = 1 << a.row_shift;
    if (a.row_lanes > 64) return hipErrorInvalidValue;
    a.table_vectors = a.rope_stride % 4 == 0 && (uintptr_t)a.cos % 16 == 0 && (uintptr_t)a.sin % 16 == 0;
    const dim3 grid((max_q_len + kRopeTokens - 1) / kRopeTokens, a.cw.num_seqs);
    switch (dtype) {
        case kDtypeBF16: return launch_rope_t<BF16>(a, grid, st);
        case kDtypeF16: return launch_rope_t<F16>(a, grid, st);
        case kDtypeF32: return launch_rope_t<F32>(a, grid, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace femto
