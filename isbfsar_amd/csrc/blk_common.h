// Device helpers of the stand-alone layer operators (xattn_kernels.hip, ffn_kernels.hip): swizzled LDS tiles, the transposing LDS
// read, the LDS-DMA request with a per-lane validity and division by a launch constant.
#pragma once
#include "conv_common.h"

namespace isb {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_tr_ptr_t;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// ---- n / d for 0 <= n < 2^31 by one multiply (d >= 1): l = ceil(log2 d), m = floor(2^32 (2^l - d) / d) + 1, q = (mulhi(n, m) + n) >> l
struct FastDiv {
    uint32_t d = 1, m = 1, l = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div) {
        while ((1ull << l) < div) ++l;
        m = (uint32_t)(((1ull << 32) * ((1ull << l) - div)) / div + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, m) + n) >> l; }
};

// ---- a tile in LDS: ROWS rows of W 16-bit values (W = 64 or 128 or 256), 16-byte chunk c of row r at chunk position c ^ tile_xor(r).
// Two kinds of reads have to be free of bank conflicts (64 banks of 4 bytes):
//  * a fragment whose lanes walk the ROWS (16 lanes read chunk c of 16 consecutive rows): the XOR takes 16 (W >= 128; 8 per row pair for
//    W = 64) different values over 16 rows;
//  * a transposing read (tr16): 32 lanes read 4 consecutive rows x 64 bytes: the 64-byte block (chunk >> 2) differs over 4 rows.
template <int W>
__device__ __forceinline__ int tile_xor(int r) {
    if constexpr (W == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return ((r & 3) << 2) | ((r >> 2) & 3);
}
template <int W>
__device__ __forceinline__ int tile_at(int r, int c) { return r * (W * 2) + ((c ^ tile_xor<W>(r)) << 4); }

// Fragment of a 32x32x16 product from a tile whose rows are the product's rows (A) or columns (B): lane l holds row (l & 31), values
// 16 ks + 8 (l >> 5) ... + 7.
template <int W>
__device__ __forceinline__ uint4 frag_rows(const unsigned char* t, int row0, int ks, int lane) {
    return *reinterpret_cast<const uint4*>(t + tile_at<W>(row0 + (lane & 31), 2 * ks + (lane >> 5)));
}

// ds_read_b64_tr_b16: in each group of 16 lanes, lane i gives the address of 4 values (row i / 4, columns 4 (i % 4) ...) and receives
// column i of the 4 rows.
__device__ __forceinline__ uint2 tr16(const unsigned char* p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr_t)(p)));
}
// Fragment from a tile whose rows are the summed index: lane l holds column col0 + (l & 31). The 8 summed rows of lane half h are
// r0 + step h ... + 3 and the same + gap: (step, gap) = (8, 4) gives rows 8 h ... 8 h + 7, the order of frag_rows; (4, 8) gives rows
// 4 h + {0 .. 3, 8 .. 11}, the order in which a 32x32 accumulator holds its rows.
template <int W, int STEP, int GAP>
__device__ __forceinline__ uint4 frag_cols(const unsigned char* t, int r0, int col0, int lane) {
    const int r = r0 + STEP * (lane >> 5) + ((lane & 15) >> 2);
    const int c = (col0 >> 3) + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const uint2 lo = tr16(t + tile_at<W>(r, c) + (lane & 1) * 8);
    const uint2 hi = tr16(t + tile_at<W>(r + GAP, c) + (lane & 1) * 8);
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
}

// ---- LDS-DMA through a raw buffer: 16 bytes per lane from base + voff to lds + 16 lane. A lane whose voff is DMA_NONE reads nothing and
// its 16 bytes become zeros (the offset is past num_records), so a masked or absent row costs no data and no branch.
constexpr uint32_t DMA_NONE = 0x80000000u;
constexpr uint32_t DMA_SPAN = 0x7fffffffu;
__device__ __forceinline__ i32x4 dma_desc(const void* base) {
    const uint64_t b = (uint64_t)(uintptr_t)base;
    i32x4 r;
    r.x = __builtin_amdgcn_readfirstlane((int)(uint32_t)b);
    r.y = __builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32));
    r.z = (int)DMA_SPAN;
    r.w = 0x00020000;
    return r;
}
__device__ __forceinline__ void dma16_desc(i32x4 desc, uint32_t voff, uint32_t lds_addr) {
    const uint32_t la = __builtin_amdgcn_readfirstlane(lds_addr);
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(desc), "s"(la) : "memory");
}
// the same from an address of each lane's own
__device__ __forceinline__ void dma16_lane(const void* src, uint32_t lds_addr) {
    const uint32_t la = __builtin_amdgcn_readfirstlane(lds_addr);
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(la) : "memory");
}
__device__ __forceinline__ uint32_t lds_addr_of(const void* p) { return (uint32_t)(uintptr_t)(lds_ptr_t)(void*)p; }

// every request and LDS access of this wave is done; then the workgroup meets
__device__ __forceinline__ void wait_all_and_meet() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Conversions to fp16 saturate from here on (MODE.FP16_OVFL, as T16::enter()), for kernels with matrix products: with the bit set, an fp16
// matrix product takes a NaN operand for 0, so it is set behind the last one. Returns 1.0, and what is converted has to be a product with it:
// that keeps the conversions behind the switch.
template <bool F16>
__device__ __forceinline__ float saturate_from_here() {
    float one = 1.0f;
    if constexpr (F16) asm volatile("s_setreg_imm32_b32 hwreg(HW_REG_MODE, 23, 1), 1\n\ts_nop 1\n\tv_mov_b32 %0, 1.0" : "=v"(one)::"memory");
    return one;
}

// the other half's value of a pair of lanes (l, l ^ 32)
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void both_halves(float x, float& lo, float& hi) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    lo = __uint_as_float(r.x);
    hi = __uint_as_float(r.y);
}
__device__ __forceinline__ float max_halves(float x) { float a, b; both_halves(x, a, b); return fmaxf(a, b); }
__device__ __forceinline__ float sum_halves(float x) { float a, b; both_halves(x, a, b); return a + b; }

// workgroup id -> work item so that the ids of one XCD (id & 7: ids go round the 8 XCDs) take a contiguous range of items: items that
// read the same states or weights then share one L2
__device__ __forceinline__ int xcd_item(int id, int total) {
    const int per = (total + 7) >> 3;
    return (id & 7) * per + (id >> 3);
}

}  // namespace isb
