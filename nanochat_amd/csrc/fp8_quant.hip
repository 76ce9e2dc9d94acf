/*
 * The 8-bit form (nc_fp8.h) of activations and of weights on gfx950.
 *
 * fp8_rows_kernel: 8 lanes a block of 128 columns, 16 adjacent values a lane: their largest magnitude (integer maxima of the
 * bits without signs), the other lanes' by DPP, the scale, 16 codes, one 16-byte store. Bound by memory: 2 or 4 bytes in, 1
 * out (65,536 x 1,664 of bf16 55 us, 5.9 TB/s; a copy of 1 GiB reaches 5.2).
 *
 * fp8_weight_kernel: a workgroup a block of 128 x 128. It holds the block in registers, finds its scale, stores its codes and,
 * where a transpose is asked for (the operand of the input's gradient, whose products run over the weight's rows), turns them
 * in LDS. Both directions share the block's scale. 6,656 x 1,664 of fp32 in both orders: 15 us, 4.5 TB/s.
 */
#include "nanochat_amd.h"
#include "nc_fp8.h"

namespace nc {
namespace {

/* 16 adjacent values of a row as they come: 8 dwords of bf16 pairs, or 16 of fp32. ALIGNED: by 16-byte loads. */
template <bool F32, bool ALIGNED> struct Sixteen {
    uint32_t w[F32 ? 16 : 8];
    __device__ __forceinline__ void load(const void *p) {
        if (ALIGNED) {
#pragma unroll
            for (int i = 0; i < (F32 ? 4 : 2); i++) {
                const u32x4 v = ((const u32x4 *)p)[i];
#pragma unroll
                for (int j = 0; j < 4; j++) w[4 * i + j] = v[j];
            }
        } else if (F32) {
#pragma unroll
            for (int i = 0; i < 16; i++) w[F32 ? i : 0] = ((const uint32_t *)p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                w[i] = (uint32_t)((const uint16_t *)p)[2 * i] | (uint32_t)((const uint16_t *)p)[2 * i + 1] << 16;
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < (F32 ? 16 : 8); i++) w[i] = 0u;
    }
    __device__ __forceinline__ uint32_t amax() const {
        uint32_t m = 0u;
        if (F32) {
#pragma unroll
            for (int i = 0; i < (F32 ? 16 : 8); i++) {
                const uint32_t a = w[i] & 0x7FFFFFFFu;
                m = m > a ? m : a;
            }
            return m;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) m = pair_amax(m, w[i]);
        return pair_top(m);
    }
    __device__ __forceinline__ u32x4 codes(uint32_t byte) const {
        if (byte == F8_NAN_BYTE) return u32x4{F8_NAN_CODES, F8_NAN_CODES, F8_NAN_CODES, F8_NAN_CODES};
        const float s = f8_scale(byte);
        u32x4 c;
#pragma unroll
        for (int i = 0; i < 4; i++)
            c[i] = F32 ? f8_codes(__uint_as_float(w[F32 ? 4 * i : 0]), __uint_as_float(w[F32 ? 4 * i + 1 : 0]),
                                  __uint_as_float(w[F32 ? 4 * i + 2 : 0]), __uint_as_float(w[F32 ? 4 * i + 3 : 0]), s)
                       : f8_codes(w[F32 ? 0 : 2 * i], w[F32 ? 0 : 2 * i + 1], s);
        return c;
    }
};

struct Rows {
    const unsigned char *x;     /* rows of cols values at row_bytes */
    long long row_bytes;
    int cols, blocks;           /* blocks of a row */
    long long items;            /* blocks of all rows */
    unsigned char *codes, *scale;   /* [rows][cols]; [rows] at scale_stride */
    long long scale_stride;
};

template <bool F32, bool ALIGNED>
__global__ void __launch_bounds__(256) fp8_rows_kernel(Rows p) {
    const long long item = (long long)blockIdx.x * 32 + (threadIdx.x >> 3);
    const int lane8 = threadIdx.x & 7;
    const bool live = item < p.items;
    const long long row = live ? (long long)((uint32_t)item / (uint32_t)p.blocks) : 0;   /* items < 2^31, by the host */
    const int block = live ? (int)((uint32_t)item % (uint32_t)p.blocks) : 0, col = block * F8_BLOCK + 16 * lane8;
    const bool in = live && col < p.cols;                     /* cols is a multiple of 16 */
    Sixteen<F32, ALIGNED> v;
    if (in) v.load(p.x + row * p.row_bytes + (long long)col * (F32 ? 4 : 2));
    else v.clear();
    const uint32_t byte = f8_scale_byte(lane_max_dpp<1>(lane_max_dpp<2>(lane_max_dpp<4>(v.amax()))));
    if (in) *(u32x4 *)(p.codes + row * p.cols + col) = v.codes(byte);
    if (live && lane8 == 0) p.scale[row * p.scale_stride + block] = (unsigned char)byte;
}

struct Weight {
    const unsigned char *w;     /* [n][k] at row_bytes */
    long long row_bytes;
    int n, k;
    unsigned char *codes, *scale, *codes_t, *scale_t;   /* [n][k], [ceil(n / 128)] at stride; codes_t NULL, or [k][n] */
    int stride, stride_t;
};

constexpr int TURN_ROW = F8_BLOCK + 4;   /* bytes of a row in LDS: 33 dwords, so a column's bytes lie in 32 banks */

template <bool F32, bool ALIGNED>
__global__ void __launch_bounds__(256) fp8_weight_kernel(Weight p) {
    __shared__ uint32_t most[4];
    __shared__ unsigned char turn[F8_BLOCK * TURN_ROW];
    const int tid = threadIdx.x, kb = blockIdx.x, nb = blockIdx.y;
    const int r0 = tid >> 3, c0 = 16 * (tid & 7), col = kb * F8_BLOCK + c0;
    Sixteen<F32, ALIGNED> v[4];
    uint32_t m = 0u;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int row = nb * F8_BLOCK + r0 + 32 * j;
        if (row < p.n && col < p.k) v[j].load(p.w + row * p.row_bytes + (long long)col * (F32 ? 4 : 2));
        else v[j].clear();
        const uint32_t a = v[j].amax();
        m = m > a ? m : a;
    }
    m = group_max(lane_max_dpp<1>(lane_max_dpp<2>(lane_max_dpp<4>(lane_max_dpp<8>(m)))));
    if ((tid & 63) == 0) most[tid >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) m = m > most[i] ? m : most[i];
    const uint32_t byte = f8_scale_byte(m);
    if (tid == 0) {
        p.scale[(long long)nb * p.stride + kb] = (unsigned char)byte;
        if (p.codes_t) p.scale_t[(long long)kb * p.stride_t + nb] = (unsigned char)byte;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int r = r0 + 32 * j, row = nb * F8_BLOCK + r;
        const u32x4 c = v[j].codes(byte);
        if (row < p.n && col < p.k) *(u32x4 *)(p.codes + (long long)row * p.k + col) = c;
        if (p.codes_t) {
            uint32_t *t = (uint32_t *)(turn + r * TURN_ROW + c0);
#pragma unroll
            for (int i = 0; i < 4; i++) t[i] = c[i];
        }
    }
    if (!p.codes_t) return;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; j++) {   /* thread: column r0 + 32 j, rows c0 .. c0 + 15 */
        const int k = kb * F8_BLOCK + r0 + 32 * j, n = nb * F8_BLOCK + c0;
        if (k >= p.k || n >= p.n) continue;   /* n is a multiple of 16 where a transpose is asked for */
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned char *t = turn + (c0 + 4 * i) * TURN_ROW + r0 + 32 * j;
            o[i] = (uint32_t)t[0] | (uint32_t)t[TURN_ROW] << 8 | (uint32_t)t[2 * TURN_ROW] << 16 |
                   (uint32_t)t[3 * TURN_ROW] << 24;
        }
        *(u32x4 *)(p.codes_t + (long long)k * p.n + n) = o;
    }
}

}  // namespace
}  // namespace nc

using namespace nc;

extern "C" int nc_fp8_quantize_rows(const void *x, int is_f32, long long row_stride, long long rows, int cols, void *codes,
                                    void *scale, long long scale_stride, void *stream) {
    const int blocks = (cols + F8_BLOCK - 1) / F8_BLOCK;
    if (rows < 0 || cols <= 0 || cols % 16 || cols > (1 << 20) || rows > (1LL << 31) / blocks - 32 ||
        (rows > 1 && row_stride < cols) || row_stride > (1LL << 40) || scale_stride < blocks || scale_stride % 4)
        return NC_ERR_SHAPE;
    if (rows == 0) return NC_OK;
    if (!x || !codes || !scale) return NC_ERR_NULL;
    const int size = is_f32 ? 4 : 2;
    if (f8_misaligned(codes, 16) || f8_misaligned(scale, 4) || f8_misaligned(x, size)) return NC_ERR_SHAPE;
    const Rows p = {(const unsigned char *)x, row_stride * size, cols, blocks, rows * blocks, (unsigned char *)codes,
                    (unsigned char *)scale, scale_stride};
    const dim3 grid((unsigned)((p.items + 31) / 32)), block(256);
    const bool fast = !f8_misaligned(x, 16) && p.row_bytes % 16 == 0;
    const auto kernel = is_f32 ? fast ? fp8_rows_kernel<true, true> : fp8_rows_kernel<true, false>
                               : fast ? fp8_rows_kernel<false, true> : fp8_rows_kernel<false, false>;
    hipLaunchKernelGGL(kernel, grid, block, 0, (hipStream_t)stream, p);
    return (int)hipGetLastError();
}

extern "C" int nc_fp8_quantize_weight(const void *w, int is_f32, long long row_stride, int n, int k, void *codes, void *scale,
                                      int scale_stride, void *codes_t, void *scale_t, int scale_t_stride, void *stream) {
    const long long nb = ((long long)n + F8_BLOCK - 1) / F8_BLOCK, kb = ((long long)k + F8_BLOCK - 1) / F8_BLOCK;
    if (n <= 0 || k <= 0 || k % 16 || n > (1 << 20) || k > (1 << 20) || (n > 1 && row_stride < k) ||
        row_stride > (1LL << 40) || scale_stride < kb || scale_stride % 4 ||
        (codes_t && (n % 16 || scale_t_stride < nb || scale_t_stride % 4)))
        return NC_ERR_SHAPE;
    if (!w || !codes || !scale || (codes_t && !scale_t)) return NC_ERR_NULL;
    const int size = is_f32 ? 4 : 2;
    if (f8_misaligned(codes, 16) || f8_misaligned(codes_t, 16) || f8_misaligned(scale, 4) || f8_misaligned(scale_t, 4) ||
        f8_misaligned(w, size))
        return NC_ERR_SHAPE;
    const Weight p = {(const unsigned char *)w, row_stride * size, n, k, (unsigned char *)codes, (unsigned char *)scale,
                      (unsigned char *)codes_t, (unsigned char *)scale_t, scale_stride, scale_t_stride};
    const dim3 grid((unsigned)kb, (unsigned)nb), block(256);   /* at most 8,192 x 8,192 */
    const bool fast = !f8_misaligned(w, 16) && p.row_bytes % 16 == 0;
    const auto kernel = is_f32 ? fast ? fp8_weight_kernel<true, true> : fp8_weight_kernel<true, false>
                               : fast ? fp8_weight_kernel<false, true> : fp8_weight_kernel<false, false>;
    hipLaunchKernelGGL(kernel, grid, block, 0, (hipStream_t)stream, p);
    return (int)hipGetLastError();
}
