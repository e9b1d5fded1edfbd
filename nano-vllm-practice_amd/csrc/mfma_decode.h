// Decode on MFMA, for the calls that read a part of each context: window
// decode (window_decode.hip) and the decode rows of a windowed prefill call
// (attention_tiles.h) as whole rows, window_row; the tails of a shared-prefix
// call (attention_tiles.h) as slices, mfma_waves.
//
// Same work as decode_worker.h: one query token per sequence, slices of pages
// per wave, bound by the bytes of K and V.  There a lane forms four scores per
// page and query head by dot products and DPP sums, ~400 VALU instructions a
// page at four heads per wave, and beside MFMA tiles on the same SIMD (mixed
// batches, shared prefixes) the two contend for the VALU.  Here a page is two
// matrix products with up to 16 query heads of a KV head as columns, whatever
// their number:
//   S^T (16 keys x 16 heads) = K . Q^T, 4 x v_mfma_f32_16x16x32;
//   O^T (128 dims x 16 heads) += V^T . P^T, 8 x v_mfma_f32_16x16x16.
// K and V come from HBM straight into the wave's own LDS (global_load_lds, 1 KB
// of consecutive bytes per instruction; K loaded into the operand's registers,
// 64 bytes of 16 rows per instruction, ran as fast alone but slowed tiles on
// the same CU: 1024 new tokens beside 127 rows 122 -> 147 us), K read back as
// the A operand (ds_read_b128), V transposed (ds_read_b64_tr_b16).  The scores
// leave lane l with keys 4 (l / 16) .. + 3 for head l % 16, which is the B
// operand that P^T needs: P never moves.  Softmax as there: a running maximum
// per head that moves by jumps of kLazyMax, 32-bit sums; P rounds to the
// storage type for the product (and the row sum adds the rounded P).
#pragma once

#include "decode_worker.h"
#include "lds_copy.h"

namespace femto {

constexpr int kMfmaHeads = 16;                    // query heads per wave
constexpr int kPageLds = 2 * kPage * kDimHead * 2;  // K and V of a page in LDS
// Pages in LDS per wave: one computed, the others on their way.
constexpr int kStagesTiles = 2;  // beside tiles (the launch's 64 KB of LDS)
template <int STAGES>
constexpr int kWorkerLds = STAGES * kPageLds;

__device__ __forceinline__ f32x4 mfma16x16x32(BF16, u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16x16x32(F16, u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 mfma16x16x16(BF16, u32x2 a, u32x2 b, f32x4 c) {
    typedef short v4s __attribute__((ext_vector_type(4)));
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(v4s, a), __builtin_bit_cast(v4s, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16x16x16(F16, u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
}

// State of the wave's heads: lane l keeps head l % 16; m (log2 units) and the
// reduced l are the same in its four lanes, o[dt] holds dims 16 dt + 4 (l / 16) ..
struct HeadState {
    float m, l;
    f32x4 o[8];
    __device__ __forceinline__ void clear() {
        m = kEmptyMax;
        l = 0.0f;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
};

// x over the four lanes of a head.
__device__ __forceinline__ float head_sum(float x) {
    float a, b;
    pair16(x, a, b);
    pair32(a + b, a, b);
    return a + b;
}
__device__ __forceinline__ float head_max(float x) {
    float a, b;
    pair16(x, a, b);
    pair32(fmaxf(a, b), a, b);
    return fmaxf(a, b);
}

// Heads h0 .. h0 + nh - 1 of sequence b over pages [lp0, lp0 + n) of its list;
// lds: the wave's kWorkerLds<STAGES> bytes.
template <typename E, bool FULL, int RULE, int STAGES>
__device__ __forceinline__ void mfma_segment(const DecodeArgs& a, int b, int kv_len, int start, int lp0, int n, int qrow,
                                             int h0, int nh, int64_t head_off, uint8_t* lds, HeadState& s) {
    constexpr int EB = 2;
    const int lane = threadIdx.x & 63;
    const int c = lane & 15, g = lane >> 4;
    const int D = FULL ? kDimHead : a.head_dim;
    s.clear();

    u32x4 q[4];  // B operand of the scores: head c, dims 32 kk + 8 g ..
    {
        const char* qr = reinterpret_cast<const char*>(a.q) +
                         ((int64_t)(h0 + c) * a.q_stride_head + (int64_t)qrow * a.q_stride_seq) * EB;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            const int d = 32 * kk + 8 * g;
            q[kk] = c < nh && (FULL || d < D) ? ld16(qr + d * EB) : u32x4{0, 0, 0, 0};
        }
    }
    // Copy j of a page: lane 16 g + c fetches the chunk of row 4 j + g that
    // lives at chunk position c (swizzled by row, see swz_k and swz_v).  Chunks
    // past head_dim read chunk 0 (Q is zero there, and those output dims are
    // not stored).  koff, voff: byte offsets inside a page; kch, vch: in a row.
    const int rs = (int)a.pool_stride_row * EB;
    const int nchunks = FULL ? 16 : D / 8;
    uint32_t koff[4], voff[4];
    int kch[4], vch[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int row = 4 * j + g, ck = c ^ swz_k(row), cv = c ^ swz_v(row);
        kch[j] = 16 * (FULL || ck < nchunks ? ck : 0);
        vch[j] = 16 * (FULL || cv < nchunks ? cv : 0);
        koff[j] = (uint32_t)(row * rs + kch[j]);
        voff[j] = (uint32_t)(row * rs + vch[j]);
    }
    const char* zero = reinterpret_cast<const char*>(g_zero_page);
    const uint32_t lds_base = lds_addr(lds);

    const PageList<RULE> pages(a, kv_len, start);
    const int32_t* table = a.tables + (int64_t)b * a.table_stride;
    int tbl = -1;
    auto fetch_table = [&](int i0) __attribute__((always_inline)) {
        const int pg = pages.page(lp0 + i0 + lane);
        tbl = (i0 + lane < n && pg < a.num_pages_per_seq) ? table[pg] : -1;
        // Waited for here, once per 64 pages: as a pending load it would make
        // every issue wait out the copies before it.
        asm volatile("" : "+v"(tbl));
    };
    auto seen = [&](int key) __attribute__((always_inline)) {
        bool ok = key < kv_len;
        if constexpr (RULE == kWindowPages) ok &= key >= start || key < a.sinks;
        return ok;
    };
    // Whether a page has rows that the query does not see (wave-uniform).
    auto ragged_page = [&](int pg) __attribute__((always_inline)) {
        bool r = pg * kPage + kPage > kv_len;
        if constexpr (RULE == kWindowPages) r |= pg * kPage < start && pg * kPage + kPage > a.sinks;
        return r;
    };
    // Eight copies of page i: K, then V.  A block id outside the pool reads
    // as zeros, and so do V's rows that the query does not see (their weights
    // are 0, and 0 times a NaN or an infinity would not be).
    auto issue = [&](int i, int stage) __attribute__((always_inline)) {
        if ((i & 63) == 0) fetch_table(i);
        const int blk = __builtin_amdgcn_readlane(tbl, i & 63);
        const bool ok = blk >= 0 && (int64_t)blk < a.num_blocks;
        const int64_t page_off = ((int64_t)blk * a.pool_stride_block + head_off) * EB;
        const char* kp = reinterpret_cast<const char*>(a.k_pool) + page_off;
        const char* vp = reinterpret_cast<const char*>(a.v_pool) + page_off;
        const uint32_t dst = lds_base + stage * kPageLds;
        const int pg = pages.page(lp0 + i);
        if (ok && !ragged_page(pg)) {
            lds_dma_rows(kp, koff, dst);
            lds_dma_rows(vp, voff, dst + kPageLds / 2);
        } else {
            uint64_t ka[4], va[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool vis = ok && seen(pg * kPage + 4 * j + g);
                ka[j] = ok ? (uint64_t)(uintptr_t)kp + koff[j] : (uint64_t)(uintptr_t)zero + kch[j];
                va[j] = vis ? (uint64_t)(uintptr_t)vp + voff[j] : (uint64_t)(uintptr_t)zero + vch[j];
            }
            lds_dma_rows(ka, dst);
            lds_dma_rows(va, dst + kPageLds / 2);
        }
    };
    // Transposed reads: in each group of 16 lanes, lane i supplies key base +
    // i / 4, dims 4 (i % 4) .. of a block of 16; lane j then holds dim j of the
    // four keys base ..; group g reads keys 4 g ...
    const int v_key = 4 * g + (c >> 2), v_dim = 4 * (c & 3);
    const float scale = a.scale_log2;
    auto consume = [&](int i, int stage) __attribute__((always_inline)) {
        const uint8_t* ks = lds + stage * kPageLds;
        const uint8_t* vs = ks + kPageLds / 2;
        f32x4 sc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
            sc = mfma16x16x32(E{}, *reinterpret_cast<const u32x4*>(ks + c * 256 + (((4 * kk + g) ^ swz_k(c)) << 4)), q[kk], sc);
        const int pg = pages.page(lp0 + i);
        if (ragged_page(pg)) {
#pragma unroll
            for (int x = 0; x < 4; ++x) sc[x] = seen(pg * kPage + 4 * g + x) ? sc[x] : -INFINITY;
        }
        const float mx = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])) * scale;
        if (__ballot(mx > s.m + kLazyMax)) {
            const float mn = fmaxf(s.m, head_max(mx));
            const float al = fast_exp2(s.m - mn);
            s.l *= al;
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) s.o[dt] *= al;
            s.m = mn;
        }
        u32x2 pw;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            pw[x] = pack2(E{}, fast_exp2(fmaf(sc[2 * x], scale, -s.m)), fast_exp2(fmaf(sc[2 * x + 1], scale, -s.m)));
            s.l = sum2(E{}, pw[x], s.l);
        }
        // Every block of 16 dims, also those past head_dim (not stored): with an
        // exit after the last one the compiler left out the wait between a
        // block's MFMA and the copy of its result at the exit's target, and
        // four-wave calls of 64 dims lost a page in dims 50, 51, 54, 55, ..  (61
        // sequences, window 2048: 64 dims 44.3 us either way, 112 69.7 and 68.4,
        // 16 30.3 and 31.0.)
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            const int dim = 16 * dt + v_dim;
            const int off = v_key * 256 + ((((dim >> 3) ^ swz_v(v_key)) << 4) | ((dim & 4) << 1));
            const u32x2 vt = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vs + off)));
            s.o[dt] = mfma16x16x16(E{}, vt, pw, s.o[dt]);
        }
    };

    // STAGES - 1 pages are on their way during a page's math: the wait counts
    // their copies, 8 each.
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
        if (i < n) issue(i, i);
    for (int i0 = 0; i0 < n; i0 += STAGES) {
#pragma unroll
        for (int x = 0; x < STAGES; ++x) {
            if (i0 + x >= n) break;
            if (i0 + x + STAGES - 1 < n) {
                issue(i0 + x + STAGES - 1, (x + STAGES - 1) % STAGES);
                asm volatile("s_waitcnt vmcnt(%0)" : : "n"(8 * (STAGES - 1)) : "memory");
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            consume(i0 + x, x);
        }
    }
    s.l = head_sum(s.l);
}

// Partial slot `sl` <- the lane's share of the state (m and l from lanes 0 .. nh - 1).
__device__ __forceinline__ void store_partial(const DecodeArgs& a, int64_t sl, int g, const HeadState& s) {
    float* dst = a.part_acc + sl * kDimHead + 4 * g;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4*>(dst + 16 * dt) = s.o[dt];
    if (g == 0) *reinterpret_cast<float2*>(a.part_ml + sl * 2) = make_float2(s.m, s.l);
}

// Window rows: workgroup `block` of W waves takes part (block % a.parts) of the
// pages that one KV head group's query heads of one sequence see; wave w the
// w-th of W contiguous shares of it.  The waves fold their states through LDS
// (each over its own, done, pages).  A sequence in one part is written at once.
// Else the part's state goes to its slot with system-scope stores (written
// through to memory) and the workgroup counts itself in; the one that comes
// last reads all slots (system-scope loads, in part order: the result does not
// depend on who was last), writes the rows and leaves the counter zero.
// lds: W * kWorkerLds<STAGES> bytes, s_ml: [W][kMfmaHeads][2].
template <typename E, bool FULL, int W, int STAGES>
__device__ __forceinline__ void window_row(const DecodeArgs& a, int block, uint8_t* lds, float (*s_ml)[kMfmaHeads][2],
                                           int* s_old) {
    constexpr int kWaveLds = kWorkerLds<STAGES>;
    static_assert(kWaveLds >= kMfmaHeads * kDimHead * 4, "a wave's outputs");
    const int P = a.parts;
    const int part = block % P, bg = block / P;
    const int b = bg / a.grid_heads, grp = bg - b * a.grid_heads;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kvh = grp / a.head_groups, hg = grp - kvh * a.head_groups;
    const int h0 = kvh * a.n_rep + hg * a.heads_per_wave;
    const int nh = min(a.heads_per_wave, a.n_rep - hg * a.heads_per_wave);
    int row, kv_len, start;
    if (b >= a.num_seqs || !decode_row_of<kWindowPages>(a, b, row, kv_len, start)) return;  // a chunk's tiles
    const int npg = pages_seen<kWindowPages>(a, kv_len, start);
    const int per_part = (npg + P - 1) / P;
    const int first = part * per_part, mine = min(npg - first, per_part);
    const int parts = npg > 0 ? (npg + per_part - 1) / per_part : 1;  // with pages
    if (part >= parts) return;
    const int per = (mine + W - 1) / W;
    const int lp0 = min(mine, wave * per), n = min(mine, lp0 + per) - lp0;
    uint8_t* own = lds + wave * kWaveLds;
    HeadState s;
    if (n > 0) {
        mfma_segment<E, FULL, kWindowPages, STAGES>(a, b, kv_len, start, first + lp0, n, row, h0, nh,
                                                    (int64_t)kvh * a.pool_stride_head, own, s);
    } else {
        s.clear();
    }
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
    // Thread i holds dims 4 (i % 32) .. of head i / 32 (and so on).
    char* out = reinterpret_cast<char*>(a.out);
    auto write = [&](int r, int d, f32x4 o, float l) __attribute__((always_inline)) {
        const int64_t at = (int64_t)(h0 + r) * a.out_stride_head + (int64_t)row * a.out_stride_seq + d;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            // no key: zeros in a decode call, 0 / 0 in a row of a prefill call
            const float v = npg > 0 ? o[x] / l : a.cu_seqlens ? __builtin_nanf("") : 0.0f;
            if (FULL || d + x < a.head_dim) store_elem<E>(out, at + x, v);
        }
    };
    const int64_t slot0 = ((int64_t)b * a.n_heads + h0) * P;
    const auto ra = __builtin_amdgcn_make_buffer_rsrc(a.part_acc + slot0 * kDimHead, (short)0, nh * P * kDimHead * 4, 0x00020000);
    const auto rm = __builtin_amdgcn_make_buffer_rsrc(a.part_ml + slot0 * 2, (short)0, nh * P * 8, 0x00020000);
    for (int i = threadIdx.x; i < nh * (kDimHead / 4); i += 64 * W) {
        const int r = i / (kDimHead / 4), d = 4 * (i % (kDimHead / 4));
        float M = kEmptyMax;
#pragma unroll
        for (int w = 0; w < W; ++w) M = fmaxf(M, s_ml[w][r][0]);
        float L = 0.0f;
        f32x4 O = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = fast_exp2(s_ml[w][r][0] - M);
            L = fmaf(s_ml[w][r][1], f, L);
            O += *reinterpret_cast<const f32x4*>(lds + w * kWaveLds + (r * kDimHead + d) * 4) * f;
        }
        if (parts == 1) {
            write(r, d, O, L);
        } else {
            const int sl = r * P + part;
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, O), ra, (sl * kDimHead + d) * 4, 0, 0x11);
            if (d == 0)
                __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(M), __float_as_uint(L)}, rm, sl * 8, 0, 0x11);
        }
    }
    if (parts == 1) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's share is in memory
    __syncthreads();                                    // ... and every wave's, before the count goes up
    int* counter = a.merge_counters + bg;
    if (threadIdx.x == 0) *s_old = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (*s_old != parts - 1) return;  // another part merges
    if (threadIdx.x == 0) __hip_atomic_exchange(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("" ::: "memory");
    constexpr int kAhead = 8;  // slots in flight
    for (int i = threadIdx.x; i < nh * (kDimHead / 4); i += 64 * W) {
        const int r = i / (kDimHead / 4), d = 4 * (i % (kDimHead / 4));
        float M = kEmptyMax, L = 0.0f;
        f32x4 O = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int p0 = 0; p0 < parts; p0 += kAhead) {
            u32x2 ml[kAhead];
            u32x4 v[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int sl = r * P + min(p0 + u, parts - 1);  // past the end: the last slot again, left out below
                ml[u] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rm, sl * 8, 0, 0x11));
                v[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(ra, (sl * kDimHead + d) * 4, 0, 0x11));
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (p0 + u >= parts) break;
                const float mu = __uint_as_float(ml[u][0]), mn = fmaxf(M, mu);
                const float f0 = fast_exp2(M - mn), f1 = fast_exp2(mu - mn);
                L = L * f0 + __uint_as_float(ml[u][1]) * f1;
                O = O * f0 + __builtin_bit_cast(f32x4, v[u]) * f1;
                M = mn;
            }
        }
        write(r, d, O, L);
    }
}

// Tails of a shared-prefix call: the waves of workgroup `block`, as
// decode_waves: slices and partial slots are the same; a.heads_per_wave (at
// most 16) query heads per wave, the last wave of a KV head's groups maybe
// fewer.  lds: the workgroup's 4 * kWorkerLds<STAGES> bytes.
template <typename E, bool FULL, int STAGES>
__device__ __forceinline__ void mfma_waves(const DecodeArgs& a, int block, uint8_t* lds) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int gw = block * 4 + wave;
    const int grp = gw / a.waves_per_group;
    const int wi = gw - grp * a.waves_per_group;
    if (grp >= a.grid_heads) return;  // waves are independent: no barriers below
    const int kvh = grp / a.head_groups;
    const int hg = grp - kvh * a.head_groups;
    const int h0 = kvh * a.n_rep + hg * a.heads_per_wave;
    const int nh = min(a.heads_per_wave, a.n_rep - hg * a.heads_per_wave);
    const int c = lane & 15, g = lane >> 4;
    const int64_t head_off = (int64_t)kvh * a.pool_stride_head;
    walk_slice<kTailPages>(a, wi, [&](int b, int kv_len, int start, int lp0, int n, int qrow, int slot, int count, bool last)
                                __attribute__((always_inline)) {
        HeadState s;
        mfma_segment<E, FULL, kTailPages, STAGES>(a, b, kv_len, start, lp0, n, qrow, h0, nh, head_off, lds + wave * kWorkerLds<STAGES>, s);
        if (c < nh) store_partial(a, ((int64_t)b * a.n_heads + h0 + c) * slot_stride<kTailPages>(a) + slot, g, s);
        if (lane == 0 && grp == 0 && last) a.seq_slots[b] = slot + 1;  // last segment: slot count
    });
}

// Head groups of the workers above: as few as hold kMfmaHeads heads each.
inline void set_mfma_heads(DecodeArgs& a) {
    a.head_groups = (a.n_rep + kMfmaHeads - 1) / kMfmaHeads;
    a.heads_per_wave = (a.n_rep + a.head_groups - 1) / a.head_groups;
    a.grid_heads = a.n_heads / a.n_rep * a.head_groups;
}

}  // namespace femto
