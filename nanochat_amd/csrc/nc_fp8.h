/*
 * The 8-bit form of matrices (fp8_quant.hip, fp8_gemm.hip, fp8_skinny.hip, fp8_grad.hip): e4m3 codes and one power of two for each block of
 * 128 columns of a row (activations, gradients) or 128 x 128 of a weight, kept as its biased exponent (e8m0, a byte). A value
 * stands for code * 2^(byte - 127).
 *
 * The scale is the least power of two s with amax <= 448 s: amax = m 2^e with m in [1, 2) gives 2^(e - 8), doubled where m >
 * 1.75 (448 = 1.75 2^8). A block of zeros has scale 1. A power of two keeps the codes' relative error at half a step (2^-4)
 * whatever it is, down to amax 2^-15 / 1.75 or less where e4m3 becomes subnormal; it makes x / s exact, so a code is one
 * rounding of x, and code * s exact in bf16, which the matrix cores multiply as it is (but at either end of the range: under s = 2^-124
 * a code's lowest bits fall below bf16's least number, and one that rounds a magnitude above 2^128 (1 - 2^-5) up stands for 2^128).
 * A block with an infinity or a NaN becomes NaN whole (byte 255, every code 0x7F): what is made from it is NaN too.
 */
#pragma once

#include "nc_device.h"

namespace nc {

constexpr int F8_BLOCK = 128;
constexpr uint32_t F8_NAN_BYTE = 255, F8_NAN_CODES = 0x7F7F7F7Fu;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

/* The scale byte for a block's largest magnitude, given as the bits of |x| in fp32 (at or past 0x7F800000: an infinity or a
 * NaN is in the block). At least 1: 2^-126, so that both the scale and its inverse are normal numbers. */
__device__ __forceinline__ uint32_t f8_scale_byte(uint32_t amax) {
    const int e = (int)(amax >> 23) - 8 + ((amax & 0x7FFFFFu) > 0x600000u);
    const uint32_t byte = e < 1 ? 1u : (uint32_t)e;
    return amax >= 0x7F800000u ? F8_NAN_BYTE : amax == 0u ? 127u : byte;
}

__device__ __forceinline__ float f8_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

/* Four codes of two bf16 pairs, or of four fp32, over a scale (one rounding each, to nearest even). The converter divides by
 * the scale's power of two itself; |x| <= 448 s by the choice of s, so nothing saturates. */
__device__ __forceinline__ uint32_t f8_codes(uint32_t lo, uint32_t hi, float s) {
    s16x2 r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, lo), s, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, hi), s, true);
    return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ uint32_t f8_codes(float a, float b, float c, float d, float s) {
    s16x2 r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, s, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, s, true);
    return __builtin_bit_cast(uint32_t, r);
}

/* The values of eight codes at a scale, as bf16. */
__device__ __forceinline__ bf16x8 f8_values(uint32_t a, uint32_t b, float s) {
    return __builtin_bit_cast(bf16x8, u32x4{
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)a, s, false)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)a, s, true)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)b, s, false)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)b, s, true))});
}

/* Two fp32 -> a bf16 pair (to nearest even; NaN stays NaN). */
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}

/* The larger |x| of both halves of two bf16 pairs: their bits without signs order as the magnitudes do. */
__device__ __forceinline__ uint32_t pair_amax(uint32_t m, uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m),
                                                                  __builtin_bit_cast(u16x2, w & 0x7FFF7FFFu)));
}
/* ... and of a pair's own two, as the bits of an fp32. */
__device__ __forceinline__ uint32_t pair_top(uint32_t m) {
    const uint32_t lo = m << 16, hi = m & 0xFFFF0000u;
    return lo > hi ? lo : hi;
}

/* A buffer resource from values that are the same in every lane. A 64-bit comparison or product on the way to them leaves them in
 * vector registers, and each access would then loop over the lanes' resources; a lane's value read back keeps them scalar. */
__device__ __forceinline__ __amdgpu_buffer_rsrc_t f8_rsrc(const void *p, long long bytes) {
    const uint64_t a = (uint64_t)p;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
    return __builtin_amdgcn_make_buffer_rsrc((void *)((uint64_t)hi << 32 | lo), (short)0,
                                             __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}

/* Bytes of the scales of some rows of `blocks` blocks, from the first row's on, that a kernel may read: whole rows to their end, the
 * last one to its own scales' padding to a dword. A tensor may end there, also where its rows lie further apart. */
__host__ __device__ static inline long long f8_scale_range(long long rows, long long stride, int blocks) {
    return (rows - 1) * stride + (blocks + 3) / 4 * 4;
}

/* DMA from memory to LDS of 16 or 4 bytes a lane (lane l's to `to` + 16 l or 4 l), as inline assembly: the compiler makes every
 * LDS read that follows its own form wait for it. The kernels that use it load and store nothing else meanwhile, and keep its
 * waits themselves. An offset past the resource's range reads zeros without an access. */
__device__ __forceinline__ u32x4 f8_words(const void *p, long long bytes) {
    const uint64_t at = (uint64_t)p;
    return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at),
                    (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32)) & 0xFFFFu,
                    (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}
__device__ __forceinline__ void f8_dma16(uint32_t to, uint32_t off, const u32x4 &r) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" :: "s"(to), "v"(off), "s"(r)
                 : "memory");
}
__device__ __forceinline__ void f8_dma4(uint32_t to, uint32_t off, const u32x4 &r) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" :: "s"(to), "v"(off), "s"(r)
                 : "memory");
}
/* f8_dma16 to base + STEP, from off + more, in three instructions. */
template <int STEP> __device__ __forceinline__ void f8_dma16(uint32_t base, uint32_t off, uint32_t more, const u32x4 &r) {
    uint32_t at;
    asm volatile("s_add_u32 m0, %1, %2\n\tv_add_u32 %0, %4, %3\n\tbuffer_load_dwordx4 %0, %5, 0 offen lds"
                 : "=&v"(at) : "s"(base), "i"(STEP), "v"(off), "s"(more), "s"(r) : "memory", "scc");
}
/* f8_dma16 to base + STEP, from off, which then moves on. */
template <int STEP> __device__ __forceinline__ void f8_dma16_on(uint32_t base, uint32_t &off, uint32_t on, const u32x4 &r) {
    asm volatile("s_add_u32 m0, %1, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %3, 0 offen lds\n\tv_add_u32 %0, %4, %0"
                 : "+v"(off) : "s"(base), "i"(STEP), "s"(r), "s"(on) : "memory", "scc");
}
__device__ __forceinline__ uint32_t f8_lds(const void *p) {
    return (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void *)p);
}

/* Largest over lanes L ^ 1, 2, 4 (8 lanes), over L ^ 16 and L ^ 32 (the four groups of 16 lanes). */
template <int M> __device__ __forceinline__ uint32_t lane_max_dpp(uint32_t v) {
    const uint32_t o = __float_as_uint(lane_xor_dpp<M>(__uint_as_float(v)));
    return v > o ? v : o;
}
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = a[0] > a[1] ? a[0] : a[1];
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return b[0] > b[1] ? b[0] : b[1];
}

/* Rows of activations in LDS, 128 bytes each: a row keeps its 16-byte piece b at place b ^ f8_swizzle(row). A 16-byte LDS read serves
 * lanes 0-3, 12-15, 20-23 and 24-27 together, then 4-11, 16-19 and 28-31, and so the upper half. Two rows lie side by side over the 64
 * banks, so 8 rows of one parity, four of one 16-byte piece b and four of b ^ 2, need 8 places. Rows i: i / 2 in {0, 1, 6, 7} gives
 * places 0 to 3 (closed under ^ 2), the others 4 to 7. */
__device__ __forceinline__ int f8_swizzle(int row) {
    const int k = (row >> 1) & 7;
    return (k & 3) | ((k + 2) & 4);
}

/* What the entry points check. */
static inline bool f8_misaligned(const void *p, unsigned n) { return ((uintptr_t)p & (n - 1)) != 0; }
static inline bool f8_bad_scales(const void *p, long long stride, int cols) {
    return f8_misaligned(p, 4) || stride % 4 || stride < (cols + F8_BLOCK - 1) / F8_BLOCK || stride > 1 << 14;
}

/* Rows in the 8-bit form in a workspace: their codes, then their scales at a padded stride. */
static inline long long f8_pitch(int cols) { return ((cols + F8_BLOCK - 1) / F8_BLOCK + 3) / 4 * 4; }
static inline long long f8_form_bytes(long long rows, int cols) { return rows * cols + (rows * f8_pitch(cols) + 15) / 16 * 16; }
struct F8Form {
    unsigned char *codes, *scale;
    long long pitch, bytes;
    F8Form(void *at, long long rows, int cols)
        : codes((unsigned char *)at), scale(codes + rows * cols), pitch(f8_pitch(cols)), bytes(f8_form_bytes(rows, cols)) {}
};

}  // namespace nc
