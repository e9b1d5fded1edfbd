// Copies from HBM straight into LDS and the row layout that the transposed
// reads of V want (attention_tiles.h, mfma_decode.h).
#pragma once

#include "common.h"

namespace femto {

// One page of zeros: the source of every copy whose block id lies outside
// the pool (each of its rows is read from row 0), so such a page reads as
// zeros.
static __device__ __attribute__((aligned(16))) uint16_t g_zero_page[kPage * kDimHead];

// 16-byte chunk c of LDS row r lives at chunk position c ^ swz(r).  The V
// swizzle gives the four rows that one transposed read covers (r % 4 = 0..3)
// four XOR values that differ in bits 1-2 and in bits 2-3, and the next four
// rows the same values with bit 0 flipped, so the 16-lane groups of a
// ds_read_b64_tr_b16 spread over all banks (measured 282 vs 244 B/ns per CU
// with (r % 8) << 1).
__device__ __forceinline__ int swz_k(int r) { return r & 15; }
__device__ __forceinline__ int swz_v(int r) { return ((r & 1) ? 6 : 0) ^ ((r & 2) ? 10 : 0) ^ ((r & 4) ? 1 : 0); }

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;

// 16 bytes per lane from global memory (uniform base + per-lane offset)
// straight into LDS at lds_base + 16 * lane.  Issued through asm so the
// compiler does not order later LDS reads of the other stage behind it; the
// kernel waits for these copies itself (vmcnt) before the stage is read.
// base and lds_base must be the same in every lane of the wave.  m0 is on the
// clobber list; clang warns that it is reserved, but nothing else in these
// kernels uses m0 (their assembly sets it only here), so the warning is muted.
//
// The compiler inserts no hazard wait states inside inline asm, so the block
// carries the two that gfx9 requires here: a VMEM instruction may read an
// SGPR only 5 wait states after a VALU instruction wrote it (the base and the
// m0 value usually come straight from v_readfirstlane), and an LDS DMA may
// read m0 only 1 wait state after an SALU instruction wrote it.  Without them
// a copy can use a stale base register and read from a wrong address.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ uint64_t wave_base(const void* base) {
    const uint64_t b = (uint64_t)(uintptr_t)base;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)b);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(b >> 32));
    return ((uint64_t)hi << 32) | lo;
}

// One page of K and one of V: four copies of each, the copy j of K landing
// at kd + 1024 j and of V at vd + 1024 j.  All eight go out from one asm
// block, so the 5 wait states after the SGPR writes are paid once; each m0
// step (an SALU write) is followed by the 1 wait state the DMA needs.
__device__ __forceinline__ void lds_dma_page(const void* kbase, const void* vbase, const uint32_t (&ko)[4],
                                             const uint32_t (&vo)[4], uint32_t kd, uint32_t vd) {
    const uint64_t kb = wave_base(kbase), vb = wave_base(vbase);
    const uint32_t km0 = __builtin_amdgcn_readfirstlane(kd);
    const uint32_t vm0 = __builtin_amdgcn_readfirstlane(vd);
    asm volatile(
        "s_nop 4\n\t"
        "s_mov_b32 m0, %10\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %8\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %8\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %2, %8\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %3, %8\n\t"
        "s_mov_b32 m0, %11\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %4, %9\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %5, %9\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %6, %9\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %7, %9"
        :
        : "v"(ko[0]), "v"(ko[1]), "v"(ko[2]), "v"(ko[3]), "v"(vo[0]), "v"(vo[1]), "v"(vo[2]), "v"(vo[3]),
          "s"(kb), "s"(vb), "s"(km0), "s"(vm0)
        : "memory", "m0", "scc");
}
// One copy of the same kind, for copies issued one at a time between other
// instructions (same wait states as above).
__device__ __forceinline__ void lds_dma_one(uint64_t base_in, uint32_t off, uint32_t m0_in) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)base_in);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(base_in >> 32));
    const uint64_t base = ((uint64_t)hi << 32) | lo;
    const uint32_t m0v = __builtin_amdgcn_readfirstlane(m0_in);
    asm volatile(
        "s_nop 4\n\t"
        "s_mov_b32 m0, %2\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %1"
        :
        : "v"(off), "s"(base), "s"(m0v)
        : "memory", "m0");
}
// Four rows of 64 x 16 bytes to dst, dst + 1024, ..: the copies of a decode
// worker, with the non-temporal hint (each byte is read once per call); from
// base + off[j] per lane, or from an address per lane.  The wait for LDS reads
// keeps a copy from landing on rows that the wave is still reading.
__device__ __forceinline__ void lds_dma_rows(const void* base_in, const uint32_t (&off)[4], uint32_t dst) {
    const uint64_t base = wave_base(base_in);
    const uint32_t m0v = __builtin_amdgcn_readfirstlane(dst);
    asm volatile(
        "s_waitcnt lgkmcnt(0)\n\t"
        "s_nop 4\n\t"
        "s_mov_b32 m0, %5\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %4 nt\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %4 nt\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %2, %4 nt\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %3, %4 nt"
        :
        : "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base), "s"(m0v)
        : "memory", "m0", "scc");
}
__device__ __forceinline__ void lds_dma_rows(const uint64_t (&addr)[4], uint32_t dst) {
    const uint32_t m0v = __builtin_amdgcn_readfirstlane(dst);
    asm volatile(
        "s_waitcnt lgkmcnt(0)\n\t"
        "s_nop 4\n\t"
        "s_mov_b32 m0, %4\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %0, off nt\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, off nt\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %2, off nt\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %3, off nt"
        :
        : "v"(addr[0]), "v"(addr[1]), "v"(addr[2]), "v"(addr[3]), "s"(m0v)
        : "memory", "m0", "scc");
}
#pragma clang diagnostic pop

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

}  // namespace femto
