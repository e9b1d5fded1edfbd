// KV cache held in 4 bits: the page layout and the conversions.
//
// A page is 16 tokens of K and V of one KV head, page_bytes contiguous bytes of
// a pool (num_blocks, n_kv_heads, page_bytes).  Dims are in N = ceil(D / 32)
// blocks of 32 (the last may be half full, zeros behind it).  A (token, block) is
// one scale 2^(byte - 127) and 32 values of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} of it,
// 4 bits each, which is what gfx950's scaled matrix instructions multiply: the
// bytes are laid out so that a lane's operand is one 16-byte load and a wave's
// are consecutive.  With r the token's row and P = 256 N:
//   K, block b: 16 bytes at 256 b + 16 r, dim 32 b + i in bits 4 i ..
//     (the A operand of K . Q^T: a lane holds 32 dims of a key);
//   V, dims 8 c .. 8 c + 7: 4 bytes at P + 64 N (r / 4) + 16 c + 4 (r % 4), dim 8 c + i in bits 4 i ..
//     (four keys of a lane's 8 dims side by side: V is wanted by dims);
//   K's scale of block b at 2 P + 4 r + b, V's at 2 P + 64 + 16 (r / 4) + 4 b + r % 4.
// The scale is the smallest power of two for which no magnitude of the block is
// more than 7 of it: past that, saturation to 6 would err by more than half the
// list's largest step.  (Root mean square error over normal, t(5) and uniform
// blocks, of the largest magnitude: 0.0483 / 0.0441 / 0.0630; with 6 for 7
// 0.0501 / 0.0465 / 0.0638, with 8 0.0498 / 0.0452 / 0.0662.)  A block that holds
// an infinity or a NaN gets the byte 255, which the hardware reads as NaN.
#pragma once

#include <type_traits>

#include "common.h"

namespace femto {

constexpr int kFp4Block = 32;      // dims that share a scale
constexpr int kFp4MinScale = 8;    // least scale byte, 2^-119: no value is subnormal in bf16
constexpr int kFp4MaxScale = 252;  // 2^125: none is past its range
constexpr int kFp4NanScale = 255;

__host__ __device__ __forceinline__ constexpr int fp4_blocks(int dim) { return (dim + kFp4Block - 1) / kFp4Block; }
__host__ __device__ __forceinline__ constexpr int fp4_page_bytes(int dim) { return 512 * fp4_blocks(dim) + 128; }

// Offsets inside a page; n: blocks of a row.
__device__ __forceinline__ int fp4_k_at(int row, int c) { return 256 * (c >> 2) + 16 * row + 4 * (c & 3); }  // dims 8 c ..
__device__ __forceinline__ int fp4_v_at(int n, int row, int c) {
    return 256 * n + 64 * n * (row >> 2) + 16 * c + 4 * (row & 3);
}
__device__ __forceinline__ int fp4_k_scale_at(int n, int row, int b) { return 512 * n + 4 * row + b; }
__device__ __forceinline__ int fp4_v_scale_at(int n, int row, int b) {
    return 512 * n + 64 + 16 * (row >> 2) + 4 * b + (row & 3);
}

// Scale byte of a block from the bits of its largest magnitude.
__device__ __forceinline__ int fp4_scale_byte(uint32_t top) {
    return top >= 0x7f800000u ? kFp4NanScale : min(max((int)((top + 0x1fffffu) >> 23) - 2, kFp4MinScale), kFp4MaxScale);
}
__device__ __forceinline__ float fp4_scale(int byte) { return __uint_as_float((uint32_t)byte << 23); }

// Eight values, rounded to the nearest, ties to the even index.
__device__ __forceinline__ uint32_t fp4_pack8(const float (&x)[8], float scale) {
    uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
}

// Values 2 I and 2 I + 1 of a word, as 16-bit storage (exact in bf16; f16
// rounds, and past its range gives infinities).
template <int I>
__device__ __forceinline__ uint32_t fp4_pair(BF16, uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, I));
}
template <int I>
__device__ __forceinline__ uint32_t fp4_pair(F16, uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, I));
}
template <typename E>
__device__ __forceinline__ u32x4 fp4_unpack8(E e, uint32_t w, float scale) {
    return u32x4{fp4_pair<0>(e, w, scale), fp4_pair<1>(e, w, scale), fp4_pair<2>(e, w, scale), fp4_pair<3>(e, w, scale)};
}

// The scale at which P . V takes values, from that of the cache: half of it in f16,
// whose row sums are halved too.  A finite f16 value past 57344 rounds to 65536 in
// the cache, which f16 has no number for; half of it it has, and an average of such
// values may well be in its range.  (Halves are as exact: values have two
// significant bits, and fewer only below 2^-23.  A NaN block's scale stays
// 2^128.)
template <typename E>
__device__ __forceinline__ float fp4_value_scale(float scale) {
    return std::is_same<E, F16>::value ? 0.5f * scale : scale;
}
template <typename E>
__device__ __forceinline__ float fp4_row_sum(float l) {
    return std::is_same<E, F16>::value ? 0.5f * l : l;
}

// Global memory said to be such: an address that went through an asm statement
// has lost it, and its loads would be flat ones (which count as LDS traffic, too).
typedef const __attribute__((address_space(1))) uint8_t* GlobalBytes;
__device__ __forceinline__ GlobalBytes as_global(const void* p) { return (GlobalBytes)(uintptr_t)p; }
template <typename T>
__device__ __forceinline__ T load_global(GlobalBytes p) {
    return *reinterpret_cast<const __attribute__((address_space(1))) T*>(p);
}
template <typename T>
__device__ __forceinline__ T load_global_nt(GlobalBytes p) {
    return __builtin_nontemporal_load(reinterpret_cast<const __attribute__((address_space(1))) T*>(p));
}

}  // namespace femto
