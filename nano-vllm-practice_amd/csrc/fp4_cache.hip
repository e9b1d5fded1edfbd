// Writes to a KV cache held in 4 bits (layout and rounding: fp4.h), and reads
// of its tokens.
//
// Placement is kv_cache_write.hip's: sequence b's tokens go to positions
// positions[q_begin] + 0, 1, ..., until the first table column that is -1, past the
// table or outside the pool.  A read gives zeros where a write would have
// stopped, and for tokens of no sequence.
//
// The prologue also norms (optional) and rotates q and k on the way:
//   y = x w / sqrt(mean(x^2) + eps), per head;
//   (a, b) -> (a cos - b sin, b cos + a sin) for pairs as rope_cache_write.hip.
// A value next to a border of the 4-bit list falls on one side by its last
// bit.  So that what is cached does not hang on the order of a sum or on
// contraction, the norm is formed in 64 bits and rounded to 32, and each product
// and sum of the rotation is rounded by itself; k rounds to 4 bits from there, q
// to its type.
//
// Work: one wave per token, or two or four where there are few, four head rows at a
// time, 16 lanes of 8 dims each; a block of 32 dims is a quad of lanes, and its
// largest magnitude two DPP steps.  Rows move in batches of loads; the placement is
// looked up by the whole wave while the first batch is on its way.  The other ends
// of half-split pairs come from their lane (ds_bpermute; loading and norming them
// twice: 22.6 us for 20.0 below), and the 1 / rms of a batch's 16 rows is one
// division and root, a row per lane of each quad.
//
// The grid is by tokens and a wave looks its sequence up, beside its first loads: a
// grid of sequences by their longest has 32768 workgroups for 1024 new tokens
// beside 127 rows, 383 of them with a token.  Each token walks its sequence's new
// columns up to its own, 64 at a time, which a very long prompt in one call
// pays for: 32768 tokens written in 47 us and read in 41, as 64 sequences in 40 and
// 31; 131072 in 343 and 279, as 256 sequences in 158 and 113.  (256 columns a round:
// 289 and 222, but 8 x 512 tokens 11.4 us a call for 10.9.)
//
// Measured (bf16, 32 / 8 heads of 128): prologue of 8 x 512 tokens 20.0 us, 4.4 TB/s,
// bound by memory; with norms 29.3: 176 registers leave two waves per SIMD, so the
// 4096 waves run in two rounds, in each of which the VALU is busy 60 % and a wave
// waits 44 % of its time for loads that nothing else is there to hide.  Of 64 decode
// tokens 5.0 and 5.7, bound by latency (placement, table, batch); of 1024 beside 127
// rows 10.2.  Write of 8 x 512
// tokens (16.8 MB read, 4.5 written) 6.5-7, read 4-5; of 64 tokens 3.6 and 3.4, the
// launch and three dependent round trips, which the larger calls pay as well: all
// their waves are resident at once.
#include <type_traits>

#include "fp4.h"
#include "launch.h"

namespace femto {

constexpr int kFp4Waves = 4;  // per workgroup
constexpr int kFp4Batch = 4;   // passes of four rows whose loads are in flight

enum Fp4Pairs { kFp4NoPairs, kFp4Interleaved, kFp4HalfChunks, kFp4HalfAny };

// Block of the cache row that the token i after position p0 has, -1 where the
// walk ends before it (whole wave, uniform).
__device__ __forceinline__ int fp4_block_of(const Fp4CacheArgs& a, const int32_t* table, int p0, int i) {
    const int lane = threadIdx.x & 63;
    const int pc = (int)((uint32_t)p0 + (uint32_t)i);
    if (p0 < 0 || pc < 0) return -1;  // (wraps past 2^31: not in the cache)
    const int col = pc / kPage;
    int blk = -1;
    uint64_t ends = 0;
    for (int c = p0 / kPage; c <= col; c += 64) {
        const int id = c + lane <= col && c + lane < a.num_pages_per_seq ? table[c + lane] : -1;
        ends |= __ballot(c + lane <= col && (id < 0 || (int64_t)id >= a.num_blocks));
        if (c + 64 > col) blk = __builtin_amdgcn_readlane(id, col - c);
    }
    return ends ? -1 : blk;
}

// Sequence b that token t belongs to and its first token (whole wave, t uniform);
// false: none.  64 bounds at a time; a sequence without tokens is passed over.
__device__ __forceinline__ bool fp4_sequence_of(const Fp4CacheArgs& a, int t, int& b, int& q_begin) {
    b = q_begin = t;
    if (!a.cu_seqlens) return t < a.num_seqs;
    const int lane = threadIdx.x & 63;
    int first = 0, count = a.num_seqs + 1, step;
    do {  // the last bound that is not past t
        step = (count + 63) / 64;
        const bool in = lane * step < count;
        const int bound = in ? a.cu_seqlens[first + lane * step] : 0;
        const uint64_t up = __ballot(in && bound <= t);
        if (!up) return false;
        const int i = 63 - __builtin_clzll(up);
        q_begin = __builtin_amdgcn_readlane(bound, i);
        first += i * step;
        count = min(step, count - i * step);
    } while (step > 1);
    b = first;
    return b < a.num_seqs && q_begin >= 0;
}

template <typename E>
__device__ __forceinline__ float elem_at(const char* p);
template <>
__device__ __forceinline__ float elem_at<BF16>(const char* p) { return (float)*reinterpret_cast<const __bf16*>(p); }
template <>
__device__ __forceinline__ float elem_at<F16>(const char* p) { return (float)*reinterpret_cast<const _Float16*>(p); }

template <int kCtrl>
__device__ __forceinline__ double dpp_f64(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = dpp_i32<kCtrl>((int)(uint32_t)b), hi = dpp_i32<kCtrl>((int)(uint32_t)(b >> 32));
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double row16_sum_f64(double x) {
    x += dpp_f64<0x128>(x);  // row_ror:8
    x += dpp_f64<0x124>(x);  // row_ror:4
    x += dpp_f64<0x4E>(x);   // quad_perm [2,3,0,1]
    x += dpp_f64<0xB1>(x);   // quad_perm [1,0,3,2]
    return x;
}
// That of lane u of the quad (u a constant once unrolled).
__device__ __forceinline__ double quad_f64(double x, int u) {
    return u == 0 ? dpp_f64<0x00>(x) : u == 1 ? dpp_f64<0x55>(x) : u == 2 ? dpp_f64<0xAA>(x) : dpp_f64<0xFF>(x);
}

template <typename E, int PAIRS, bool NORM>
__global__ __launch_bounds__(64 * kFp4Waves) void fp4_cache_write_kernel(Fp4CacheArgs a) {
#pragma clang fp contract(off)
    constexpr bool ROPE = PAIRS != kFp4NoPairs;
    const int lane = threadIdx.x & 63, c = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int first = wave & ((1 << a.split_shift) - 1);
    const int t = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * (kFp4Waves >> a.split_shift)) + (wave >> a.split_shift));
    if ((uint32_t)t >= (uint32_t)a.num_tokens) return;
    const int D = a.head_dim, N = fp4_blocks(D), R = a.rotary_dim, half = R / 2;
    const int H = ROPE ? a.n_heads : 0, KVH = a.n_kv_heads, rows = H + 2 * KVH;
    const bool has = 8 * c < D;        // dims of the row
    const bool held = 8 * c < 32 * N;  // and those that pad its last block
    const bool turned = ROPE && 8 * c < R;
    // The lane that has the other ends of this one's pairs.
    const int other = 4 * ((lane & 48) | (turned ? (8 * c < half ? c + half / 8 : c - half / 8) : c));

    const char* src[3] = {ROPE ? static_cast<const char*>(a.q) + (int64_t)t * a.q_stride_token * 2 : nullptr,
                          static_cast<const char*>(a.k) + (int64_t)t * a.k_stride_token * 2,
                          static_cast<const char*>(a.v) + (int64_t)t * a.v_stride_token * 2};
    auto row_ptr = [&](int r) __attribute__((always_inline)) {
        const int s = r < H ? 0 : r < H + KVH ? 1 : 2;
        const int64_t hs = s == 0 ? a.q_stride_head : s == 1 ? a.k_stride_head : a.v_stride_head;
        const char* base = s == 0 ? src[0] : s == 1 ? src[1] : src[2];
        return base + (int64_t)(s == 0 ? r : s == 1 ? r - H : r - H - KVH) * hs * 2;
    };
    u32x4 w[kFp4Batch];
    auto load = [&](int base) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kFp4Batch; ++u) {
            const int r = base + 4 * u + (lane >> 4);
            w[u] = u32x4{0, 0, 0, 0};
            if (r < rows && has) w[u] = ld16(row_ptr(r) + 16 * c);
        }
    };
    const int begin = 4 * kFp4Batch * first;
    load(begin);

    int b, q_begin;
    if (!fp4_sequence_of(a, t, b, q_begin)) return;
    const int32_t* table = a.tables + (int64_t)b * a.table_stride;
    const int p0 = a.positions[q_begin];
    const int blk = fp4_block_of(a, table, p0, t - q_begin);
    const int row = (int)((uint32_t)p0 + (uint32_t)(t - q_begin)) & (kPage - 1);

    // The lane's table fragment and weights; sn: -sin at a pair's first end.
    float cs[8], sn[8];
    float wq[8], wk[8];
    if constexpr (ROPE) {
        const int pos = a.positions[t];
        const bool in_tables = pos >= 0 && pos < a.rope_rows;
        const float* ct = a.cos + (int64_t)(in_tables ? pos : 0) * a.rope_stride;
        const float* st = a.sin + (int64_t)(in_tables ? pos : 0) * a.rope_stride;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = 8 * c + e;
            const int j = PAIRS == kFp4Interleaved ? d / 2 : d < half ? d : d - half;
            const bool in = d < R;
            const bool lead = PAIRS == kFp4Interleaved ? (e & 1) == 0 : d < half;
            cs[e] = in ? ct[j] : 1.0f;
            sn[e] = in ? st[j] : 0.0f;
            if (lead) sn[e] = -sn[e];
            if (!in_tables) cs[e] = sn[e] = __builtin_nanf("");
        }
        if constexpr (NORM) {
            auto weights = [&](const void* p, float (&f)[8]) __attribute__((always_inline)) {
                u32x4 g{0, 0, 0, 0};
                if (has) g = ld16(static_cast<const char*>(p) + 16 * c);
                unpack8(E{}, g, f);
            };
            weights(a.q_weight, wq);
            weights(a.k_weight, wk);
        }
    }

    for (int base = begin; base < rows; base += 4 * kFp4Batch << a.split_shift) {
        if (base != begin) load(base);
        // 1 / rms of the batch's rows, pass u's by lane u of each quad.
        double inv = 1.0;
        if constexpr (NORM) {
            double mine = 1.0;
#pragma unroll
            for (int u = 0; u < kFp4Batch; ++u) {
                float x[8];
                unpack8(E{}, w[u], x);
                double s = 0.0;  // (squares are exact)
#pragma unroll
                for (int e = 0; e < 8; ++e) s = __builtin_fma((double)x[e], (double)x[e], s);
                s = row16_sum_f64(s);
                if ((lane & 3) == u) mine = s;
            }
            inv = 1.0 / sqrt(mine / (double)D + (double)a.eps);
        }
#pragma unroll
        for (int u = 0; u < kFp4Batch; ++u) {
            const int r = base + 4 * u + (lane >> 4);
            float x[8];
            unpack8(E{}, w[u], x);
            if constexpr (ROPE) {
                if (r < H + KVH) {
                    double by = 1.0;
                    if constexpr (NORM) by = quad_f64(inv, u);
                    auto normed = [&](float v, float g) __attribute__((always_inline)) {
                        return NORM ? (float)((double)v * by * (double)g) : v;
                    };
                    if constexpr (NORM) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = normed(x[e], r < H ? wq[e] : wk[e]);
                    }
                    float y[8];  // the other ends
                    if constexpr (PAIRS == kFp4HalfAny) {
                        const char* p = row_ptr(r);
                        const char* g = static_cast<const char*>(r < H ? a.q_weight : a.k_weight);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int d = 8 * c + e, o = d < half ? d + half : d - half;
                            y[e] = d < R ? normed(elem_at<E>(p + 2 * o), NORM ? elem_at<E>(g + 2 * o) : 1.0f) : 0.0f;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            y[e] = PAIRS == kFp4Interleaved
                                       ? x[e ^ 1]
                                       : __int_as_float(__builtin_amdgcn_ds_bpermute(other, __float_as_int(x[e])));
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float z = x[e] * cs[e], o = y[e] * sn[e];
                        if (PAIRS == kFp4HalfChunks ? turned : 8 * c + e < R) x[e] = z + o;
                    }
                }
            }
            if (ROPE && r < H) {
                if (has)
                    st16_nt(static_cast<char*>(a.q_out) + ((int64_t)t * a.q_out_stride_token + (int64_t)r * a.q_out_stride_head) * 2 + 16 * c,
                            pack8(E{}, x));
                continue;
            }
            // The block's largest magnitude: this lane's and its quad's.
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
            top = max(top, (uint32_t)dpp_i32<0xB1>((int)top));
            top = max(top, (uint32_t)dpp_i32<0x4E>((int)top));
            if (r >= rows || blk < 0 || !held) continue;
            const int byte = fp4_scale_byte(top);
            const uint32_t word = byte == kFp4NanScale ? 0u : fp4_pack8(x, fp4_scale(byte));
            const bool is_k = r < H + KVH;
            const int h = is_k ? r - H : r - H - KVH;
            uint8_t* page = a.pool + ((int64_t)blk * KVH + h) * fp4_page_bytes(D);
            *reinterpret_cast<uint32_t*>(page + (is_k ? fp4_k_at(row, c) : fp4_v_at(N, row, c))) = word;
            if ((c & 3) == 0) page[is_k ? fp4_k_scale_at(N, row, c >> 2) : fp4_v_scale_at(N, row, c >> 2)] = (uint8_t)byte;
        }
    }
}

// Rows of the tokens at positions[q_begin] + 0, 1, .. of each sequence, as E.
template <typename E>
__global__ __launch_bounds__(64 * kFp4Waves) void fp4_cache_read_kernel(Fp4CacheArgs a) {
    const int lane = threadIdx.x & 63, c = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = (int)(blockIdx.x * kFp4Waves) + wave;
    const int D = a.head_dim, N = fp4_blocks(D), KVH = a.n_kv_heads;
    if ((uint32_t)t >= (uint32_t)a.num_tokens) return;
    int b, q_begin, blk = -1, row = 0;  // (a token of no sequence: zeros)
    if (fp4_sequence_of(a, t, b, q_begin)) {
        const int p0 = a.positions[q_begin];
        blk = fp4_block_of(a, a.tables + (int64_t)b * a.table_stride, p0, t - q_begin);
        row = (int)((uint32_t)p0 + (uint32_t)(t - q_begin)) & (kPage - 1);
    }
    for (int base = 0; base < 2 * KVH; base += 4 * kFp4Batch) {
        uint32_t word[kFp4Batch];
        int byte[kFp4Batch];
#pragma unroll
        for (int u = 0; u < kFp4Batch; ++u) {
            const int r = base + 4 * u + (lane >> 4);
            word[u] = 0;
            byte[u] = kFp4MinScale;
            if (r < 2 * KVH && blk >= 0 && 8 * c < D) {
                const bool is_k = r < KVH;
                const uint8_t* page = a.pool + ((int64_t)blk * KVH + (is_k ? r : r - KVH)) * fp4_page_bytes(D);
                word[u] = *reinterpret_cast<const uint32_t*>(page + (is_k ? fp4_k_at(row, c) : fp4_v_at(N, row, c)));
                byte[u] = page[is_k ? fp4_k_scale_at(N, row, c >> 2) : fp4_v_scale_at(N, row, c >> 2)];
            }
        }
#pragma unroll
        for (int u = 0; u < kFp4Batch; ++u) {
            const int r = base + 4 * u + (lane >> 4);
            if (r >= 2 * KVH || 8 * c >= D) continue;
            const bool is_k = r < KVH;
            char* out = static_cast<char*>(is_k ? a.k_out : a.v_out) +
                        ((int64_t)t * KVH + (is_k ? r : r - KVH)) * D * 2 + 16 * c;
            st16_nt(out, fp4_unpack8(E{}, word[u], fp4_scale(byte[u])));
        }
    }
}

template <typename E, int PAIRS>
static void launch_write(const Fp4CacheArgs& a, dim3 grid, hipStream_t st) {
    const dim3 block(64 * kFp4Waves);
    if constexpr (PAIRS != kFp4NoPairs) {
        if (a.q_weight) {
            hipLaunchKernelGGL((fp4_cache_write_kernel<E, PAIRS, true>), grid, block, 0, st, a);
            return;
        }
    }
    hipLaunchKernelGGL((fp4_cache_write_kernel<E, PAIRS, false>), grid, block, 0, st, a);
}

template <typename E>
static hipError_t launch_cache(Fp4CacheOp op, const Fp4CacheArgs& a, dim3 grid, hipStream_t st) {
    if (op == kFp4Read) hipLaunchKernelGGL(fp4_cache_read_kernel<E>, grid, dim3(64 * kFp4Waves), 0, st, a);
    else if (op == kFp4Write) launch_write<E, kFp4NoPairs>(a, grid, st);
    else if (a.interleaved) launch_write<E, kFp4Interleaved>(a, grid, st);
    else if (a.rotary_dim % 16 == 0) launch_write<E, kFp4HalfChunks>(a, grid, st);
    else launch_write<E, kFp4HalfAny>(a, grid, st);
    return hipGetLastError();
}

hipError_t launch_fp4_cache(int dtype, Fp4CacheOp op, Fp4CacheArgs a, hipStream_t st) {
    if (a.num_seqs <= 0 || a.num_tokens <= 0) return hipSuccess;
    a.split_shift = 0;
    // A token's batches over several waves, while there are at most two tokens per
    // CU.  bf16, 32/8 heads of 128 with norms, us by one, two and four waves a token:
    // 64 tokens 9.6, 7.8, 6.0; 512 11.3, 9.3, 8.3; 1024 11.8, 11.1, 14.2; 16/2 heads (two
    // batches) 64 tokens 6.7, 5.4, 5.9, 512 8.0, 6.4, 7.5.
    if (op == kFp4Prologue) {
        int cus = 0;
        const hipError_t e = device_cu_count(cus);
        if (e != hipSuccess) return e;
        const int batches = (a.n_heads + 2 * a.n_kv_heads - 1) / (4 * kFp4Batch) + 1;
        if (a.num_tokens <= 2 * cus) a.split_shift = batches > 2 ? 2 : batches - 1;
    }
    const dim3 grid((((int64_t)a.num_tokens << a.split_shift) - 1) / kFp4Waves + 1);
    switch (dtype) {
        case kDtypeBF16: return launch_cache<BF16>(op, a, grid, st);
        case kDtypeF16: return launch_cache<F16>(op, a, grid, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace femto
