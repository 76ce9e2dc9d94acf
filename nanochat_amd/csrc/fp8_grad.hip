/*
 * The gradient of a weight from the 8-bit checkpoint of its layer's input on gfx950: out[i][j] (+)= sum_m dy[m][i] x[m][j] over
 * token rows m, dy bf16 [M][N1], x in the 8-bit form (nc_fp8.h) [M][N2] with a scale for each 128 columns of a token.
 *
 * The scale changes along the summed dimension, so the products cannot be taken in 8 bits. A code times a power of two is
 * exact in bf16, so x is unpacked on its way into LDS and the products are v_mfma_f32_16x16x32_bf16, fp32 sums, as exact as
 * those of a bf16 input: only half of that input's bytes are read.
 *
 * A workgroup owns a 256 x 256 tile of the result and a slice of the tokens, walked in stages of 32. dy's 256 columns go into
 * LDS by DMA, three stages ahead (a ring of four); x's 16 codes a thread into registers, three stages ahead, and as 32 bytes of
 * bf16 into one of two LDS buffers the stage before they are used. Both are read transposed (ds_read_b64_tr_b16: four tokens of
 * one column a lane). A 512-byte row keeps its 32-byte piece s at place s ^ (row % 8), so that the eight rows that half a wave
 * reads meet in different banks. Eight waves hold 128 x 64 results each.
 *
 * The result is small and the sum long: where tiles alone would leave CUs idle the tokens are cut into slices, whose partial
 * tiles fp8_grad_sum_kernel adds in slice order, so the result does not depend on scheduling.
 */
#include "nanochat_amd.h"
#include "nc_fp8.h"
#include "nc_internal.h"

namespace nc {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __amdgpu_buffer_rsrc_t Rsrc;
typedef __attribute__((address_space(3))) void LdsPtr;
typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16 LdsV4;

constexpr int GR_T = 256;                     /* a tile's rows and columns */
constexpr int GR_KC = 32;                     /* tokens of a stage */
constexpr int GR_ROWB = GR_T * 2;
constexpr int GR_OPB = GR_KC * GR_ROWB;       /* a stage's operand in LDS: 16 KiB */
constexpr int GR_WAVES = 8;
constexpr int GR_PAST = 0x7FFF0000;           /* a byte offset past every operand's range */

enum { GR_PART, GR_ADD, GR_F32, GR_BF16 };

struct F8Grad {
    const uint16_t *dy;                       /* [M][N1] */
    const unsigned char *x, *xs;              /* [M][N2], [M] at xs_stride */
    long long xs_stride, M;
    int N1, N2, tiles2, slices, rows;         /* rows: of a slice, a multiple of GR_KC */
    void *out;                                /* PART: fp32 [slices][N1][N2]; else the result [N1][N2] */
};

/* Stage j of dy: instruction q moves rows 2 q, 2 q + 1; lane l row 2 q + l / 32, LDS piece (l % 32) / 2, half l % 2. */
__device__ __forceinline__ void gr_fetch(Rsrc rs, unsigned char *lds, int j, int N, int c0, int wave, int lane) {
#pragma unroll
    for (int k = 0; k < GR_OPB / 1024 / GR_WAVES; k++) {
        const int q = wave + GR_WAVES * k, row = 2 * q + (lane >> 5);
        const int piece = ((lane & 31) >> 1) ^ (row & 7), col = c0 + piece * 16 + (lane & 1) * 8;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (LdsPtr *)(lds + q * 1024), 16,
                                                 col < N ? ((j * GR_KC + row) * N + col) * 2 : GR_PAST, 0, 0, 0);
    }
}

/* A thread's 16 codes of a stage of x and their scale byte: token tid / 16, columns 16 (tid % 16) .. + 15 of the tile. */
struct Codes {
    u32x4 c;
    uint32_t byte;
};
struct XSource {
    Rsrc codes, scales;
    int at, scale_at;        /* this thread's byte offsets in stage 0 (GR_PAST: a column past N2) */
    int step, scale_step;    /* bytes of a stage */
    __device__ __forceinline__ Codes fetch(int j) const {
        Codes f;
        const bool in = at != GR_PAST;
        f.c = __builtin_amdgcn_raw_buffer_load_b128(codes, in ? at + j * step : GR_PAST, 0, 0);
        f.byte = __builtin_amdgcn_raw_buffer_load_b8(scales, in ? scale_at + j * scale_step : GR_PAST, 0, 0);
        return f;
    }
};

/* The codes as bf16 into LDS. Tokens past the slice have codes and byte 0, and stay zeros. */
__device__ __forceinline__ void gr_unpack(unsigned char *lds, const Codes &f, int tid) {
    const int row = tid >> 4, piece = tid & 15;
    const float s = f8_scale(f.byte < 1u ? 1u : f.byte);
    u32x4 o[2];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        o[i >> 1][2 * (i & 1)] =
            __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)f.c[i], s, false));
        o[i >> 1][2 * (i & 1) + 1] =
            __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)f.c[i], s, true));
    }
    u32x4 *to = (u32x4 *)(lds + row * GR_ROWB + ((piece ^ (row & 7)) << 5));
    to[0] = o[0];
    to[1] = o[1];
}

/* The MFMA operand of columns 16 d .. + 15: lane (g, c) gets column 16 d + c of rows 4 g .. + 3, then 16 + 4 g .. + 3. */
__device__ __forceinline__ bf16x8 gr_operand(const unsigned char *lds, int d, int g, int c) {
    const int r0 = 4 * g + (c >> 2), r1 = r0 + 16;   /* both with the same row % 8 */
    const int at = ((d ^ (r0 & 7)) << 5) + ((c & 3) << 3);
    const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsV4 *)(lds + r0 * GR_ROWB + at));
    const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsV4 *)(lds + r1 * GR_ROWB + at));
    const uint2 x = __builtin_bit_cast(uint2, lo), y = __builtin_bit_cast(uint2, hi);
    return __builtin_bit_cast(bf16x8, uint4{x.x, x.y, y.x, y.y});
}

__device__ __forceinline__ void gr_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ void gr_compute(const unsigned char *a, const unsigned char *b, f32x4 (&acc)[8][4], int wm, int wn,
                                           int g, int c) {
    bf16x8 fb[4];
#pragma unroll
    for (int u = 0; u < 4; u++) fb[u] = gr_operand(b, 4 * wn + u, g, c);
#pragma unroll
    for (int t = 0; t < 8; t++) {
        const bf16x8 fa = gr_operand(a, 8 * wm + t, g, c);
#pragma unroll
        for (int u = 0; u < 4; u++) acc[t][u] = mfma16x16x32(fa, fb[u], acc[t][u]);
    }
}

/* All but the 6 memory operations issued last have landed (a stage's fetch is x: 2, dy: 2; stage j needs dy of j, issued three
 * steps ago, and x of j + 1, issued two ago before dy of that stage), and this wave's LDS writes are done. */
__device__ __forceinline__ void gr_wait() { __builtin_amdgcn_s_waitcnt(6 | (0x7 << 4) | (0x0 << 8)); }

/* Step j: dy of stage j in A, x of it in B; x of stage j + 1 goes from X1 into the other buffer; stage j + 3 is fetched (dy into
 * the buffer of stage j - 1, which every wave has left). */
#define GR_STEP(j, A, AFREE, B, BNEXT, X1, X3)                    \
    do {                                                            \
        gr_wait();                                                  \
        gr_barrier();                                               \
        X3 = xsrc.fetch((j) + 3);                                   \
        gr_fetch(ra, AFREE, (j) + 3, p.N1, i0, wave, lane);         \
        gr_unpack(BNEXT, X1, tid);                                  \
        gr_compute(A, B, acc, wm, wn, g, c);                        \
    } while (0)

template <int MODE>
__global__ void __launch_bounds__(GR_WAVES *WAVE, 1) fp8_grad_kernel(F8Grad p) {
    __shared__ __align__(16) unsigned char a0[GR_OPB], a1[GR_OPB], a2[GR_OPB], a3[GR_OPB], b0[GR_OPB], b1[GR_OPB];
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid >> 6, g = lane >> 4, c = lane & 15;
    const int wm = wave >> 2, wn = wave & 3;
    /* slices fastest: the workgroups that run together read different tokens of the same few columns */
    const int slice = blockIdx.x % p.slices, tile = blockIdx.x / p.slices;
    const int i0 = tile / p.tiles2 * GR_T, j0 = tile % p.tiles2 * GR_T;
    const long long m0 = (long long)slice * p.rows;
    const int rows = (int)(p.M - m0 < p.rows ? p.M - m0 : p.rows);   /* > 0: the host makes no empty slice */
    const Rsrc ra = f8_rsrc(p.dy + m0 * p.N1, (long long)rows * p.N1 * 2);
    XSource xsrc;
    xsrc.codes = f8_rsrc(p.x + m0 * p.N2, (long long)rows * p.N2);
    xsrc.scales = f8_rsrc(p.xs + m0 * p.xs_stride, rows * p.xs_stride);
    const int xcol = j0 + 16 * (tid & 15);
    xsrc.at = xcol < p.N2 ? (tid >> 4) * p.N2 + xcol : GR_PAST;
    xsrc.scale_at = (tid >> 4) * (int)p.xs_stride + xcol / F8_BLOCK;
    xsrc.step = GR_KC * p.N2;
    xsrc.scale_step = GR_KC * (int)p.xs_stride;
    const int stages = (rows + GR_KC - 1) / GR_KC;
    f32x4 acc[8][4];
#pragma unroll
    for (int t = 0; t < 8; t++)
#pragma unroll
        for (int u = 0; u < 4; u++) acc[t][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    Codes x0 = xsrc.fetch(0);
    gr_fetch(ra, a0, 0, p.N1, i0, wave, lane);
    Codes x1 = xsrc.fetch(1);
    gr_fetch(ra, a1, 1, p.N1, i0, wave, lane);
    Codes x2 = xsrc.fetch(2), x3;
    gr_fetch(ra, a2, 2, p.N1, i0, wave, lane);
    gr_unpack(b0, x0, tid);
    for (int j = 0; j < stages; j += 4) {   /* stages past the slice read zeros and add nothing */
        GR_STEP(j, a0, a3, b0, b1, x1, x3);
        GR_STEP(j + 1, a1, a0, b1, b0, x2, x0);
        GR_STEP(j + 2, a2, a1, b0, b1, x3, x1);
        GR_STEP(j + 3, a3, a2, b1, b0, x0, x2);
    }
    __builtin_amdgcn_s_waitcnt(0);   /* no DMA may land in LDS after the workgroup ends */
    /* lane (g, c) of result tile (t, u): rows i0 + 128 wm + 16 t + 4 g + e, column j0 + 64 wn + 16 u + c; 32-bit offsets into the
     * tile's rows, those past N1 and columns past N2 outside the range */
    constexpr int SIZE = MODE == GR_BF16 ? 2 : 4;
    const int live = p.N1 - i0 < GR_T ? p.N1 - i0 : GR_T;
    const unsigned row_bytes = (unsigned)p.N2 * SIZE;
    const long long first = ((MODE == GR_PART ? (long long)slice * p.N1 : 0) + i0) * p.N2;
    const Rsrc ro = f8_rsrc((unsigned char *)p.out + first * SIZE, (long long)live * row_bytes);
    unsigned at[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const int col = j0 + 64 * wn + 16 * u + c;
        at[u] = col < p.N2 ? (unsigned)(128 * wm + 4 * g) * row_bytes + (unsigned)col * SIZE : (unsigned)GR_PAST;
    }
    float old[2][4][4];   /* ADD: the result's rows of t, and of t + 1 in flight */
    const auto fetch_old = [&](int t) {
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                old[t & 1][u][e] =
                    __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(ro, at[u] + (16 * t + e) * row_bytes, 0, 0));
    };
    if (MODE == GR_ADD) fetch_old(0);
#pragma unroll
    for (int t = 0; t < 8; t++) {
        if (MODE == GR_ADD && t < 7) fetch_old(t + 1);
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const unsigned to = at[u] + (16 * t + e) * row_bytes;
                const float v = MODE == GR_ADD ? old[t & 1][u][e] + acc[t][u][e] : acc[t][u][e];
                if (MODE == GR_BF16)
                    __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, (__bf16)v), ro, to, 0, 0);
                else
                    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), ro, to, 0, 0);
            }
    }
}

/* The slices' partials added in order, and the result with them (ADD); four elements a thread. */
template <int MODE>
__global__ void __launch_bounds__(256) fp8_grad_sum_kernel(const float4 *part, int slices, long long n4, void *out) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n4) return;
    float4 sum = part[i];
#pragma unroll 8
    for (int s = 1; s < slices; s++) {
        const float4 v = part[s * n4 + i];
        sum.x = sum.x + v.x; sum.y = sum.y + v.y; sum.z = sum.z + v.z; sum.w = sum.w + v.w;
    }
    if (MODE == GR_BF16) {
        ((uint2 *)out)[i] = uint2{bf16_pair(sum.x, sum.y), bf16_pair(sum.z, sum.w)};
        return;
    }
    if (MODE == GR_ADD) {
        const float4 o = ((const float4 *)out)[i];
        sum.x = o.x + sum.x; sum.y = o.y + sum.y; sum.z = o.z + sum.z; sum.w = o.w + sum.w;
    }
    ((float4 *)out)[i] = sum;
}

constexpr int GR_MIN_ROWS = 4 * GR_KC;   /* a shorter slice is mostly the ring's start */

/* Token slices: as many as fill the CUs with tiles, none under GR_MIN_ROWS rows unless it is the only one and none whose
 * operand slice passes 1 GiB. */
void grad_slices(long long M, int N1, int N2, int &slices, int &rows) {
    const long long tiles = (long long)((N1 + GR_T - 1) / GR_T) * ((N2 + GR_T - 1) / GR_T);
    const long long wide = (long long)N1 * 2 > N2 ? (long long)N1 * 2 : N2;
    const long long fit = (1LL << 30) / wide / GR_KC * GR_KC;
    long long s = device_cus() / tiles;
    const long long most = (M + GR_MIN_ROWS - 1) / GR_MIN_ROWS, least = (M + fit - 1) / fit;
    s = s < most ? s : most;
    s = s > 1 ? s : 1;
    s = s > least ? s : least;
    rows = (int)(((M + s - 1) / s + GR_KC - 1) / GR_KC * GR_KC);
    if (rows > fit) rows = (int)fit;
    slices = (int)((M + rows - 1) / rows);
}

/* One slice needs none (never 0 where there is a call). */
long long grad_bytes(int slices, int N1, int N2) { return slices == 1 ? 16 : (long long)slices * N1 * N2 * 4; }

bool grad_fits(long long M, int N1, int N2) {
    return M >= 0 && M < (1LL << 31) && N1 > 0 && N2 > 0 && N1 % 8 == 0 && N2 % 16 == 0 && N1 <= 65536 && N2 <= 65536;
}

}  // namespace
}  // namespace nc

using namespace nc;

extern "C" long long nc_fp8_weight_grad_workspace_bytes(long long rows, int n1, int n2) {
    if (!grad_fits(rows, n1, n2)) return -1;
    if (rows == 0) return 0;
    int slices, per;
    grad_slices(rows, n1, n2, slices, per);
    return grad_bytes(slices, n1, n2);
}

extern "C" int nc_fp8_weight_grad(const void *dy, const void *codes, const void *scale, long long scale_stride, long long rows,
                                  int n1, int n2, int mode, void *out, void *workspace, long long workspace_bytes,
                                  void *stream) {
    if (!grad_fits(rows, n1, n2) || mode < 0 || mode > 2 || scale_stride < (n2 + F8_BLOCK - 1) / F8_BLOCK ||
        scale_stride > n2)   /* a slice's scales take no more bytes than its codes */
        return NC_ERR_SHAPE;
    if (rows == 0) return NC_OK;
    if (!dy || !codes || !scale || !out || !workspace) return NC_ERR_NULL;
    if (((uintptr_t)dy | (uintptr_t)codes | (uintptr_t)out | (uintptr_t)workspace) & 15) return NC_ERR_SHAPE;
    F8Grad p = {(const uint16_t *)dy, (const unsigned char *)codes, (const unsigned char *)scale, scale_stride, rows, n1, n2,
                (n2 + GR_T - 1) / GR_T, 0, 0, out};
    grad_slices(rows, n1, n2, p.slices, p.rows);
    if (workspace_bytes < grad_bytes(p.slices, n1, n2)) return NC_ERR_WORKSPACE;
    const long long tiles = (long long)((n1 + GR_T - 1) / GR_T) * p.tiles2;
    const dim3 grid((unsigned)(tiles * p.slices)), block(GR_WAVES * WAVE);
    const hipStream_t s = (hipStream_t)stream;
    if (p.slices == 1) {
        const auto kernel = mode == 0 ? fp8_grad_kernel<GR_F32> : mode == 1 ? fp8_grad_kernel<GR_ADD> : fp8_grad_kernel<GR_BF16>;
        hipLaunchKernelGGL(kernel, grid, block, 0, s, p);
        return (int)hipGetLastError();
    }
    p.out = workspace;
    hipLaunchKernelGGL(fp8_grad_kernel<GR_PART>, grid, block, 0, s, p);
    const long long n4 = (long long)n1 * n2 / 4;
    const auto sum = mode == 0 ? fp8_grad_sum_kernel<GR_F32> : mode == 1 ? fp8_grad_sum_kernel<GR_ADD>
                                                                           : fp8_grad_sum_kernel<GR_BF16>;
    hipLaunchKernelGGL(sum, dim3((unsigned)((n4 + 255) / 256)), dim3(256), 0, s, (const float4 *)workspace, p.slices, n4, out);
    return (int)hipGetLastError();
}
