// Decode over a KV cache held in 4 bits (layout: fp4.h): one query token per
// sequence, for decode calls (fp4_decode.hip) and the decode rows of a prefill
// call.
//
// Formula: out[h] = sum_j w_j v_j / sum_j w_j, w_j = exp(q[h] . k_j / sqrt(D)), over
// the keys j < kv_len, as paged_decode.hip; k and v are the values that the cache
// stands for.
//
// As in mfma_decode.h up to 16 query heads of a KV head are the columns of two
// matrix products, here over two pages (32 keys) at a time:
//   S^T (16 keys x 16 heads) = K . Q^T, v_mfma_scale_f32_16x16x128, K straight from
//     memory: the lane of key r and block b holds 32 4-bit dims and their scale,
//     which is the operand that the instruction takes.
//   O^T (128 dims x 16 heads) += V^T . P^T, 8 x v_mfma_f32_16x16x32.
// The first product reads K without converting it.  Its other operand may have
// 6 bits at the same rate (8 bits halve it): q is split into four terms of 6 bits,
// each with a scale for 32 dims, which leave out at most 2^-18 of the largest of
// those dims (fp4_query): nothing of a bf16 dim down to 2^-11 of it, of an f16 one
// to 2^-8; products are exact and sums 32-bit.  (Three terms, 2^-14, leave a dim of 1
// beside one of 512 off by 1.6e-2.  The fourth: 61 sequences to 16k 89.9 us either
// way, one of 5000 keys 9.4 and 9.6.)
// V is wanted by dims, its values convert to 16 bits two dims at a time
// (v_cvt_scalef32_pk, exact in bf16; f16: halves of them, fp4_value_scale), and a
// permute per two values pairs keys: a 16-byte load holds 8 dims of four keys, so
// no V passes through LDS.  Row 4 g + i of the O^T tile dt is dim 8 (4 g + i) + dt.
// P rounds to q's type, and the row sum adds the rounded P.
#pragma once

#include "fp4.h"
#include "lds_copy.h"
#include "mfma_decode.h"

namespace femto {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));
typedef float f32x32 __attribute__((ext_vector_type(32)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr int kFp4Terms = 4;
constexpr int kFormatFp6 = 2, kFormatFp4 = 4;  // operand formats of the scaled matrix instructions

// 32 dims of a query as `TERMS` terms of 6 bits (a sign, 0 to 7.5); byte i of
// `scales` is the scale byte of term i.
template <int TERMS>
struct Fp4Query {
    u32x6 term[TERMS];
    uint32_t scales;
};

// Dims 32 b .. of a row of 16-bit values; dims from D on, and rows that are not there: zeros.
struct Fp4QueryWords {
    u32x4 w[4];
};
__device__ __forceinline__ Fp4QueryWords fp4_query_words(const char* row, int b, int D, bool valid) {
    Fp4QueryWords q;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = 32 * b + 8 * i;
        q.w[i] = valid && d < D ? ld16(row + 2 * d) : u32x4{0, 0, 0, 0};
    }
    return q;
}
// The largest magnitude's bits.
__device__ __forceinline__ uint32_t fp4_query_top(const Fp4QueryWords& q) {
    u16x2 top = {0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, q.w[i >> 2][i & 3] & 0x7fff7fffu));
    return max(top[0], top[1]);
}

// The terms of x = (dims) scale.  With the first term's scale s no |x / s| is past
// 7.75, so it leaves at most s / 4; of the second's scale, s / 16, that is at most
// 4, and at most an eighth of it is left; of the third's, s / 512, again at most 4
// and an eighth: 2^-12 s; and of the fourth's, s / 2^14, 2^-17 s, where the largest
// magnitude is above 3.875 s.  (Of dims below 2 s each leaves half as much.)  A
// block with an infinity or a NaN has NaN scales: its scores are NaN.
template <typename E, int TERMS>
__device__ __forceinline__ Fp4Query<TERMS> fp4_query(const Fp4QueryWords& words, float scale) {
    f32x16 even, odd;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float f[8];
        unpack8(E{}, words.w[i], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            even[4 * i + e] = f[2 * e] * scale;
            odd[4 * i + e] = f[2 * e + 1] * scale;
        }
    }
    float f[8];
    unpack8(E{}, u32x4{fp4_query_top(words), 0, 0, 0}, f);
    const uint32_t top = __float_as_uint(f[0] * scale) & 0x7fffffffu;  // (rounding keeps the order)
    const int byte = top >= 0x7f800000u ? kFp4NanScale : max(15, (int)((top + 0x7ffffu) >> 23) - 2);
    constexpr int kDown[kFp4Terms] = {0, 4, 9, 14};
    Fp4Query<TERMS> q;
    q.scales = 0;
#pragma unroll
    for (int t = 0; t < TERMS; ++t) {
        const int b = byte == kFp4NanScale ? byte : byte - kDown[t];
        const float s = fp4_scale(byte == kFp4NanScale ? 127 : b);
        q.scales |= (uint32_t)b << (8 * t);
        // These conversions write their first registers before they have read their
        // last (with the result over registers 2 to 7 of a source: wrong values), and
        // the compiler takes a source that ends here for free: it is kept.
        auto w = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, s);
        asm("" : "+v"(w) : "v"(even), "v"(odd), "v"(s));
        q.term[t] = __builtin_bit_cast(u32x6, w);
        if (t + 1 < TERMS) {
            f32x32 back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(w, s);
            asm("" : "+v"(back) : "v"(w), "v"(s));
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                even[i] -= back[2 * i];
                odd[i] -= back[2 * i + 1];
            }
        }
    }
    return q;
}

// Whether three terms do not do for the block.  They leave up to 2^-15 of the
// largest magnitude of small dims, more than half a step of their own in bf16 below
// 1/256 of it, in f16 below 1/32.  Five such dims of a block make it so in bf16, 12 of
// 32 or 6 of 16 in f16 (where fewer are small, the steps of the others count for
// more).  Of normal values that is one block of 32 in 200 000, in f16 one in a
// million.  Zeros among them, which any term holds, are not told apart, but for
// dims from D on.
template <typename E>
__device__ __forceinline__ bool fp4_query_large(const Fp4QueryWords& q, int b, int D) {
    const int below = std::is_same<E, F16>::value ? 5 << 10 : 8 << 7;
    const uint32_t limit = (uint32_t)max((int)fp4_query_top(q) - below, 0) * 0x10001u;
    int others = 0;  // (bit 15 of a half stays where the subtraction does not borrow it: the magnitude is no smaller)
#pragma unroll
    for (int i = 0; i < 16; ++i) others += __builtin_popcount(((q.w[i >> 2][i & 3] | 0x80008000u) - limit) & 0x80008000u);
    const int absent = max(32 * b + 32 - max(D, 32 * b), 0);  // zeros, small where the limit is not 0
    const int enough = std::is_same<E, F16>::value ? 3 * (32 - absent) / 8 : 5;
    return limit > 0 && 32 - others - absent >= enough;
}

__device__ __forceinline__ i32x8 fp4_operand(u32x4 w) {
    return i32x8{(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
}
__device__ __forceinline__ i32x8 fp4_operand(u32x6 w) {
    return i32x8{(int)w[0], (int)w[1], (int)w[2], (int)w[3], (int)w[4], (int)w[5], 0, 0};
}
// c + K . (term T of q) over 128 dims: K's 16 keys x 4 blocks with the scale in byte 0 of ks.
template <int T>
__device__ __forceinline__ f32x4 fp4_scores16(u32x4 k, uint32_t ks, const Fp4Query<kFp4Terms>& q, f32x4 c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(k), fp4_operand(q.term[T]), c, kFormatFp4, kFormatFp6,
                                                            0, (int)ks, T, (int)q.scales);
}

// A page in registers: the lane of key (or dims) c = lane % 16 and block (or four
// keys) g = lane / 16.
struct Fp4Page {
    u32x4 k, v;       // dims 32 g .. of key c; dims 8 c .. of keys 4 g ..
    uint32_t ks, vs;  // scale of k; of v's four keys, a byte each
};

// Heads h0 .. h0 + nh - 1 of sequence b over pages [lp0, lp0 + n) of its kv_len
// keys.  FULL: head_dim 128.  Else lanes of dims past the row's blocks read block
// 0 (q is zero there, and those output dims are not stored).
template <typename E, bool FULL, int STAGES>
__device__ __forceinline__ void fp4_segment(const DecodeArgs& a, int b, int kv_len, int lp0, int n, int qrow, int h0, int nh,
                                            int kvh, HeadState& s) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int D = FULL ? kDimHead : a.head_dim, N = fp4_blocks(D);
    s.clear();
    const Fp4QueryWords qw = fp4_query_words(static_cast<const char*>(a.q) + ((int64_t)(h0 + c) * a.q_stride_head + (int64_t)qrow * a.q_stride_seq) * 2,
                                             g, D, c < nh);
    const int kb = FULL || g < N ? g : 0, vc = FULL || c < 4 * N ? c : 0;
    const uint32_t k_at = 256 * kb + 16 * c, v_at = 256 * N + 64 * N * g + 16 * vc;
    const uint32_t ks_at = 512 * N + 4 * c, vs_at = 512 * N + 64 + 16 * g + 4 * (vc >> 2);
    const GlobalBytes pool = as_global(a.k_pool) + (int64_t)kvh * a.pool_stride_head;
    uint64_t zero = (uint64_t)(uintptr_t)g_zero_page;
    asm volatile("" : "+s"(zero));  // (else its address is loaded, and waited for, for every page)
    const uint32_t blocks = (uint32_t)min(a.num_blocks, (int64_t)0x7fffffff);
    const int32_t* table = a.tables + (int64_t)b * a.table_stride;
    int tbl = -1;
    // Every page's loads go out, whether it is there or not (past the segment and
    // for a block outside the pool those of a page of zeros): the waits
    // count them.
    auto issue = [&](int i, Fp4Page& p) __attribute__((always_inline)) {
        if ((i & 63) == 0) {
            const int pg = lp0 + i + lane;
            tbl = i + lane < n && pg < a.num_pages_per_seq ? table[pg] : -1;
            asm volatile("" : "+v"(tbl));  // waited for here, once per 64 pages
        }
        const int blk = __builtin_amdgcn_readlane(tbl, i & 63);
        // (an id below 0 is past the pool, too)
        const GlobalBytes page = (uint32_t)blk < blocks ? pool + (int64_t)blk * a.pool_stride_block : (GlobalBytes)(uintptr_t)zero;
        // Codes are read once (non-temporal: 61 sequences up to 16k 106 -> 92 us);
        // the scales share a line, of which each load takes half.
        p.k = load_global_nt<u32x4>(page + k_at);
        p.v = load_global_nt<u32x4>(page + v_at);
        p.ks = load_global<uint32_t>(page + ks_at);
        p.vs = load_global<uint32_t>(page + vs_at);
    };
    const float scale = a.scale_log2;
    Fp4Query<kFp4Terms> q;
    auto consume = [&](int i, Fp4Page (&p)[2]) __attribute__((always_inline)) {
        float sc[8];
        {
            // The smallest term first; the two pages' products take turns.
            const uint32_t ks[2] = {p[0].ks >> (8 * kb), p[1].ks >> (8 * kb)};
            f32x4 x[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int h = 0; h < 2; ++h) x[h] = fp4_scores16<3>(p[h].k, ks[h], q, x[h]);
#pragma unroll
            for (int h = 0; h < 2; ++h) x[h] = fp4_scores16<2>(p[h].k, ks[h], q, x[h]);
#pragma unroll
            for (int h = 0; h < 2; ++h) x[h] = fp4_scores16<1>(p[h].k, ks[h], q, x[h]);
#pragma unroll
            for (int h = 0; h < 2; ++h) x[h] = fp4_scores16<0>(p[h].k, ks[h], q, x[h]);
#pragma unroll
            for (int j = 0; j < 8; ++j) sc[j] = x[j >> 2][j & 3];
        }
        // Keys past the segment or the context: no weight, and V of zeros (0
        // times a NaN would not be 0).
        const int key0 = (lp0 + i) * kPage, end = min(kv_len, (lp0 + n) * kPage);
        if (key0 + 2 * kPage > end) {  // wave-uniform
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const int h = x >> 2, j = x & 3;
                const bool seen = key0 + kPage * h + 4 * g + j < end;
                sc[x] = seen ? sc[x] : -INFINITY;
                p[h].v[j] = seen ? p[h].v[j] : 0;
                p[h].vs = seen ? p[h].vs : p[h].vs & ~(0xffu << (8 * j));
            }
        }
        float mx = fmaxf(sc[0], sc[1]);
#pragma unroll
        for (int x = 2; x < 8; ++x) mx = fmaxf(mx, sc[x]);
        mx *= scale;
        if (__ballot(mx > s.m + kLazyMax)) {
            const float mn = fmaxf(s.m, head_max(mx));
            const float al = fast_exp2(s.m - mn);
            s.l *= al;
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) s.o[dt] *= al;
            s.m = mn;
        }
        u32x4 pw;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            pw[x] = pack2(E{}, fast_exp2(fmaf(sc[2 * x], scale, -s.m)), fast_exp2(fmaf(sc[2 * x + 1], scale, -s.m)));
            s.l = sum2(E{}, pw[x], s.l);
        }
        float vsc[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t w = p[h].vs;
            vsc[4 * h] = fp4_value_scale<E>(__uint_as_float((w << 23) & 0x7f800000u));
            vsc[4 * h + 1] = fp4_value_scale<E>(__uint_as_float((w << 15) & 0x7f800000u));
            vsc[4 * h + 2] = fp4_value_scale<E>(__uint_as_float((w << 7) & 0x7f800000u));
            vsc[4 * h + 3] = fp4_value_scale<E>(__uint_as_float((w >> 1) & 0x7f800000u));
        }
        auto dims = [&](auto pair) __attribute__((always_inline)) {  // 2 pair and 2 pair + 1 of the lane's 8
            constexpr int I = decltype(pair)::value;
            uint32_t w[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) w[x] = fp4_pair<I>(E{}, p[x >> 2].v[x & 3], vsc[x]);
            u32x4 lo, hi;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                lo[x] = __builtin_amdgcn_perm(w[2 * x + 1], w[2 * x], 0x05040100u);
                hi[x] = __builtin_amdgcn_perm(w[2 * x + 1], w[2 * x], 0x07060302u);
            }
            s.o[2 * I] = mfma16x16x32(E{}, lo, pw, s.o[2 * I]);
            s.o[2 * I + 1] = mfma16x16x32(E{}, hi, pw, s.o[2 * I + 1]);
        };
        dims(std::integral_constant<int, 0>{});
        dims(std::integral_constant<int, 1>{});
        dims(std::integral_constant<int, 2>{});
        dims(std::integral_constant<int, 3>{});
    };

    // STAGES - 1 pairs of pages are on their way during a pair's math.
    Fp4Page p[STAGES][2];
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
        issue(2 * i, p[i][0]);
        issue(2 * i + 1, p[i][1]);
    }
    __builtin_amdgcn_sched_barrier(0);
    q = fp4_query<E, kFp4Terms>(qw, 1.0f);  // (while they are on their way)
    for (int i0 = 0; i0 < n; i0 += 2 * STAGES) {
#pragma unroll
        for (int x = 0; x < STAGES; ++x) {
            const int i = i0 + 2 * x;
            if (i >= n) break;
            const int next = i + 2 * (STAGES - 1);
            issue(next, p[(x + STAGES - 1) % STAGES][0]);
            issue(next + 1, p[(x + STAGES - 1) % STAGES][1]);
            consume(i, p[x]);
        }
    }
    s.l = fp4_row_sum<E>(head_sum(s.l));
}

// The lane's share of head c's outputs: dims 32 g + 8 i + dt, o[dt][i].
__device__ __forceinline__ void fp4_put_outputs(float* row, int g, const HeadState& s) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        *reinterpret_cast<f32x4*>(row + 32 * g + 8 * i) = f32x4{s.o[0][i], s.o[1][i], s.o[2][i], s.o[3][i]};
        *reinterpret_cast<f32x4*>(row + 32 * g + 8 * i + 4) = f32x4{s.o[4][i], s.o[5][i], s.o[6][i], s.o[7][i]};
    }
}

// Workgroup `block` of W waves takes part (block % a.parts) of the pages of one
// sequence for one KV head group's query heads, wave w the w-th of W contiguous
// shares of it; finish_row (mfma_decode.h) folds the waves' states and writes the
// row.  lds: W * kFp4WaveLds bytes, s_ml: [W][kMfmaHeads][2].
constexpr int kFp4WaveLds = kMfmaHeads * kDimHead * 4;
template <typename E, bool FULL, int W, int STAGES>
__device__ __forceinline__ void fp4_row(const DecodeArgs& a, int block, uint8_t* lds, float (*s_ml)[kMfmaHeads][2], int* s_old) {
    const int P = a.parts;
    const int part = block % P, bg = block / P;
    const int b = bg / a.grid_heads, grp = bg - b * a.grid_heads;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kvh = grp / a.head_groups, hg = grp - kvh * a.head_groups;
    const int h0 = kvh * a.n_rep + hg * a.heads_per_wave;
    const int nh = min(a.heads_per_wave, a.n_rep - hg * a.heads_per_wave);
    int row, kv_len, start;
    if (b >= a.num_seqs || !decode_row_of<kAllPages>(a, b, row, kv_len, start)) return;  // a chunk's tiles
    const int npg = pages_of(kv_len);
    const int per_part = (npg + P - 1) / P;
    const int first = part * per_part, mine = min(npg - first, per_part);
    const int parts = npg > 0 ? (npg + per_part - 1) / per_part : 1;  // with pages
    if (part >= parts) return;
    const int per = (mine + W - 1) / W;
    const int lp0 = min(mine, wave * per), n = min(mine, lp0 + per) - lp0;
    HeadState s;
    if (n > 0) fp4_segment<E, FULL, STAGES>(a, b, kv_len, first + lp0, n, row, h0, nh, kvh, s);
    else s.clear();
    if (c < nh) {
        fp4_put_outputs(reinterpret_cast<float*>(lds + wave * kFp4WaveLds) + c * kDimHead, g, s);
        if (g == 0) {
            s_ml[wave][c][0] = s.m;
            s_ml[wave][c][1] = s.l;
        }
    }
    __syncthreads();
    finish_row<E, FULL, W, kFp4WaveLds>(a, b, bg, h0, nh, row, npg, part, parts, lds, s_ml, s_old);
}

// Split workers, as decode_waves (decode_worker.h): wave of workgroup `block`
// walks its equal slice of the pages of all sequences and leaves a partial state
// per sequence segment and query head for the merge launch.
template <typename E, bool FULL, int STAGES>
__device__ __forceinline__ void fp4_waves(const DecodeArgs& a, int block) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int gw = block * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = gw / a.waves_per_group;
    const int wi = gw - grp * a.waves_per_group;
    if (grp >= a.grid_heads) return;  // waves are independent: no barriers below
    const int kvh = grp / a.head_groups, hg = grp - kvh * a.head_groups;
    const int h0 = kvh * a.n_rep + hg * a.heads_per_wave;
    const int nh = min(a.heads_per_wave, a.n_rep - hg * a.heads_per_wave);
    walk_slice<kAllPages>(a, wi, [&](int b, int kv_len, int, int lp0, int n, int qrow, int slot, int, bool last)
                                __attribute__((always_inline)) {
        HeadState s;
        fp4_segment<E, FULL, STAGES>(a, b, kv_len, lp0, n, qrow, h0, nh, kvh, s);
        if (c < nh) {
            const int64_t sl = ((int64_t)b * a.n_heads + h0 + c) * a.max_slots + slot;
            fp4_put_outputs(a.part_acc + sl * kDimHead, g, s);
            if (g == 0) *reinterpret_cast<float2*>(a.part_ml + sl * 2) = make_float2(s.m, s.l);
        }
        if (lane == 0 && grp == 0 && last) a.seq_slots[b] = slot + 1;  // last segment: slot count
    });
}

}  // namespace femto
