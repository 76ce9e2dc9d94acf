/*
 * Products of few results with a weight in the 8-bit form (nc_fp8.h) on gfx950, out[m][n] = epilogue(sum_k x8[m][k] w[n][k]), x8 the
 * 8-bit form of x's rows: a decoding step, draft tokens. Then a layer and an MLP for serving as one call each. Bound by reading w once,
 * and below about 8 MB of it by latency: a launch, a row's way through k, the sums.
 *
 * Up to 64 rows, x as it is (fp8_few_kernel): a workgroup holds 16 rows of w and all of x's, its eight waves take every eighth block of 128
 * k, both operands from memory straight into registers: lane (g = lane / 16, i = lane % 16) takes bytes 16 g .. + 15 and 64 + 16 g ..
 * + 15 of row i's block (w's, and each 16 rows' of x), so that a load instruction reads 64 adjacent bytes a row. Which k stands where in a product does not matter
 * as long as both operands agree. x comes in bf16 or fp32: a row's block lies in four lanes, which find its largest magnitude together
 * and make the codes that nc_fp8_quantize_rows makes. One row: 4,992 x 1,664 5.0 us, 16,384 x 1,664 8.7 us (3.1 TB/s of weights).
 *
 * Few tiles, x in 8 bits (fp8_some_kernel): the tiles of fp8_gemm.hip would leave CUs idle and walk a long k alone. 32 rows of x a
 * workgroup, x's codes in LDS by DMA (a ring of steps), as all eight waves read them; the waves stand RW by 16 rows of w and S by blocks
 * of k, w still straight into registers, up to six blocks ahead. 128 x 1,664 x 6,656 12.4 us (small tiles 21.3), 128 x 1,280 x 1,280
 * 5.5 (6.2), 17 x 4,992 x 1,664 6.4 (7.5).
 *
 * The waves' fp32 sums meet in LDS and are added in a fixed order.
 *
 * Products: v_mfma_scale_f32_16x16x128_f8f6f4 for a bf16 result; before a ReLU^2 exact ones, as fp8_gemm.hip says, by
 * v_mfma_f32_16x16x32_bf16 from the values in bf16.
 */
#include "nanochat_amd.h"
#include "nc_fp8.h"
#include "nc_internal.h"

namespace nc {
namespace {

typedef __amdgpu_buffer_rsrc_t Rsrc;

constexpr int SK_WAVES = 8;
constexpr unsigned SK_PAST = 0x7FFF0000u;   /* a byte offset past every operand's range */

enum { SK_CODES, SK_BF16, SK_F32 };         /* what x is */

struct Skinny {
    const void *x;                          /* [M][K] at row_bytes (codes: dense) */
    long long row_bytes;
    const unsigned char *xs;                /* SK_CODES: [M] scale bytes at xs_stride */
    int xs_stride, ws_stride;
    const unsigned char *w, *ws;            /* [N][K] codes, [ceil(N / 128)] scale bytes at ws_stride */
    int M, N, K, blocks;
    void *out;                              /* [M][N] bf16, or fp32 (RELU2) */
};

/* A lane's 32 codes of a block, and their scale byte. */
struct Codes32 {
    uint32_t c[8];
    uint32_t byte;
};
__device__ __forceinline__ i32x8 sk_operand(const Codes32 &f) {
    return i32x8{(int)f.c[0], (int)f.c[1], (int)f.c[2], (int)f.c[3], (int)f.c[4], (int)f.c[5], (int)f.c[6], (int)f.c[7]};
}
/* Codes 8 Q .. + 7 of a lane as bf16. */
template <int Q> __device__ __forceinline__ bf16x8 sk_exact(const Codes32 &f) {
    const float s = f8_scale(f.byte < 1u ? 1u : f.byte);   /* a row past the last has byte 0, and zeros */
    return f8_values(f.c[2 * Q], f.c[2 * Q + 1], s);
}

/* A lane's part of a block as it comes from memory: 16 values from 16 g and 16 from 64 + 16 g. */
template <int XT> struct Raw {
    static constexpr int SIZE = XT == SK_CODES ? 1 : XT == SK_BF16 ? 2 : 4, N = 2 * SIZE;   /* 16-byte pieces */
    u32x4 p[N];
    uint32_t byte;
    __device__ __forceinline__ void load(Rsrc r, unsigned row, int kb, int g, int K) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int k = kb * F8_BLOCK + 64 * h + 16 * g;
#pragma unroll
            for (int i = 0; i < SIZE; i++)
                p[SIZE * h + i] = __builtin_amdgcn_raw_buffer_load_b128(r, k < K ? row + k * SIZE + 16 * i : SK_PAST, 0, 0);
        }
    }
    /* Codes of a row's block, whose four lanes (16 apart) act together. */
    __device__ __forceinline__ Codes32 codes() const {
        Codes32 f;
        if constexpr (XT == SK_CODES) {
#pragma unroll
            for (int i = 0; i < 8; i++) f.c[i] = p[i >> 2][i & 3];
            f.byte = byte;
            return f;
        }
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (XT == SK_BF16) m = pair_amax(m, p[i][j]);
                else {
                    const uint32_t a = p[i][j] & 0x7FFFFFFFu;
                    m = m > a ? m : a;
                }
            }
        f.byte = f8_scale_byte(group_max(XT == SK_BF16 ? pair_top(m) : m));
        const float s = f8_scale(f.byte);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            uint32_t c;
            if constexpr (XT == SK_BF16) c = f8_codes(p[i / 2][2 * (i % 2)], p[i / 2][2 * (i % 2) + 1], s);
            else
                c = f8_codes(__uint_as_float(p[i % N][0]), __uint_as_float(p[i % N][1]), __uint_as_float(p[i % N][2]),
                             __uint_as_float(p[i % N][3]), s);
            f.c[i] = f.byte == F8_NAN_BYTE ? F8_NAN_CODES : c;
        }
        return f;
    }
};

/* The products of a block: a 16 x 16 tile of results. */
template <bool RELU2> __device__ __forceinline__ void sk_product(f32x4 &acc, const Codes32 &w, const Codes32 &x) {
    if constexpr (RELU2) {
        acc = mfma16x16x32(sk_exact<0>(w), sk_exact<0>(x), acc);
        acc = mfma16x16x32(sk_exact<1>(w), sk_exact<1>(x), acc);
        acc = mfma16x16x32(sk_exact<2>(w), sk_exact<2>(x), acc);
        acc = mfma16x16x32(sk_exact<3>(w), sk_exact<3>(x), acc);
    } else {
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(sk_operand(w), sk_operand(x), acc, 0, 0, 0, (int)w.byte, 0,
                                                               (int)x.byte);
    }
}
/* 16 MT rows of x. */
template <int XT, int MT, bool RELU2>
__global__ void __launch_bounds__(SK_WAVES *WAVE, MT == 1 ? 4 : 2) fp8_few_kernel(Skinny p) {
    __shared__ __align__(16) f32x4 part[SK_WAVES][MT][WAVE];
    const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, i16 = lane & 15;
    const int n0 = blockIdx.x * 16;
    const Rsrc rw = f8_rsrc(p.w + (long long)n0 * p.K, 16LL * p.K);
    const Rsrc rx = f8_rsrc(p.x, p.M * p.row_bytes);
    const unsigned char *ws = p.ws + (long long)(n0 / F8_BLOCK) * p.ws_stride;   /* 16 rows lie in one block */
    f32x4 acc[MT];
#pragma unroll
    for (int u = 0; u < MT; u++) acc[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int AHEAD = 3;   /* blocks of w on their way beside the present one; one of x, but for 64 rows */
    Raw<SK_CODES> w[AHEAD + 1];
    Raw<XT> x[MT], next[MT];
    const auto fetch = [&](int slot, int kb) {
        if (kb >= p.blocks) return;
        w[slot].load(rw, (unsigned)(i16 * p.K), kb, g, p.K);
        w[slot].byte = ws[kb];
    };
    const auto fetch_x = [&](Raw<XT> (&to)[MT], int kb) {
        if (kb >= p.blocks) return;
#pragma unroll
        for (int u = 0; u < MT; u++) to[u].load(rx, (unsigned)((16 * u + i16) * p.row_bytes), kb, g, p.K);
    };
    if (MT < 4) fetch_x(next, wave);
#pragma unroll
    for (int a = 0; a < AHEAD; a++) fetch(a, wave + SK_WAVES * a);
    for (int kb0 = wave; kb0 < p.blocks; kb0 += SK_WAVES * (AHEAD + 1)) {
#pragma unroll
        for (int a = 0; a <= AHEAD; a++) {
            const int kb = kb0 + SK_WAVES * a;
            if (kb >= p.blocks) break;
            if constexpr (MT < 4) {
#pragma unroll
                for (int u = 0; u < MT; u++) x[u] = next[u];
                fetch_x(next, kb + SK_WAVES);
            } else {
                fetch_x(x, kb);
            }
            fetch((a + AHEAD) % (AHEAD + 1), kb + SK_WAVES * AHEAD);
            const Codes32 cw = w[a].codes();
#pragma unroll
            for (int u = 0; u < MT; u++) sk_product<RELU2>(acc[u], cw, x[u].codes());
        }
    }
#pragma unroll
    for (int u = 0; u < MT; u++) part[wave][u][lane] = acc[u];
    __syncthreads();
    const int row = 16 * wave + i16;
    if (wave >= MT || row >= p.M) return;
    f32x4 v = part[0][wave][lane];   /* columns 4 g .. 4 g + 3 of the row */
#pragma unroll
    for (int s = 1; s < SK_WAVES; s++) {
        const f32x4 o = part[s][wave][lane];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = v[e] + o[e];
    }
    const long long at = (long long)row * p.N + n0 + 4 * g;
    if constexpr (RELU2) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float r = __builtin_elementwise_maximum(v[e], 0.0f);   /* a NaN stays one */
            v[e] = r * r;
        }
        *(f32x4 *)((float *)p.out + at) = v;
    } else {
        *(u32x2 *)((uint16_t *)p.out + at) = u32x2{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])};
    }
}

/* Step j: blocks j S + s of k. RW, S 1, 8 and 2, 4, us: 64 x 1,280 x 1,280 4.8, 5.3; 128 x 1,280 x 1,280 8.4, 5.4; 64 x 1,664 x 6,656
 * 9.6, 12.3; 128 x 1,664 x 6,656 17.4, 12.4; 17 x 4,992 x 1,664 8.9, 6.4. */
constexpr int SK_BLOCKS = 128;   /* of a row at most: their scales are kept in LDS */
template <int RW, int S>
__global__ void __launch_bounds__(SK_WAVES *WAVE, S == 8 ? 2 : 4) fp8_some_kernel(Skinny p) {
    static_assert(RW * S == SK_WAVES, "waves");
    constexpr int MT = 2;   /* 32 rows of x */
    constexpr int BLOCK = 16 * MT * F8_BLOCK, STEP = S * BLOCK;              /* bytes of x in LDS: of a block, of a step */
    constexpr int RING = STEP <= 16384 ? 4 : 3, DMAS = STEP / 1024 / SK_WAVES;
    constexpr int SUMS = SK_WAVES * MT * 1024, COLS = 16 * RW, PITCH = SK_BLOCKS + 4;
    static_assert(DMAS >= 1 && STEP <= 32768, "every wave moves a part of a step");
    __shared__ __align__(16) unsigned char lds[RING * STEP > SUMS ? RING * STEP : SUMS];
    __shared__ __align__(16) unsigned char scales[(16 * MT + 1) * PITCH];   /* x's rows', then w's */
    const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, i16 = lane & 15, rw = wave % RW, s = wave / RW;
    /* parts of x fastest, and on one XCD: the second reads w from its L2 */
    const int parts = (p.M + 16 * MT - 1) / (16 * MT), per = gridDim.x / 8, extra = gridDim.x % 8, xcd = blockIdx.x % 8;
    const int id = xcd * per + min(xcd, extra) + blockIdx.x / 8;
    const int m0 = id % parts * 16 * MT, n0 = id / parts * COLS;
    const int rows = min(p.M - m0, 16 * MT), cols = min(p.N - n0, COLS);
    const Rsrc rsw = f8_rsrc(p.w + (long long)n0 * p.K, (long long)cols * p.K);
    const u32x4 rx = f8_words((const unsigned char *)p.x + (long long)m0 * p.K, (long long)rows * p.K);
    const unsigned char *ws = p.ws + (long long)(n0 / F8_BLOCK) * p.ws_stride;   /* COLS rows lie in one block */
    const unsigned w_row = (unsigned)((16 * rw + i16) * p.K);
    const int steps = (p.blocks + S - 1) / S;
    const uint32_t base = f8_lds(lds);
    /* instruction q of a step moves 8 rows of a block: block q / (2 MT), rows 8 (q % (2 MT)) + lane / 8 */
    const auto fetch_x = [&](int j) {
#pragma unroll
        for (int d = 0; d < DMAS; d++) {
            const int q = wave * DMAS + d, row = 8 * (q % (2 * MT)) + (lane >> 3);
            const int k = (j * S + q / (2 * MT)) * F8_BLOCK + (((lane & 7) ^ f8_swizzle(row)) << 4);
            f8_dma16(base + j % RING * STEP + q * 1024, k < p.K ? (unsigned)(row * p.K + k) : SK_PAST, rx);
        }
    };
    f32x4 acc[MT];
#pragma unroll
    for (int u = 0; u < MT; u++) acc[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int AHEAD = 5;
    Raw<SK_CODES> w[AHEAD + 1];
    const auto fetch_w = [&](Raw<SK_CODES> &f, int j) {   /* a block past the last: zeros */
        f.load(rsw, w_row, j * S + s, g, p.K);
    };
    /* the scales, a dword of four blocks a thread (rows past the last: zeros) */
    for (int t = threadIdx.x; t < (16 * MT + 1) * (SK_BLOCKS / 4); t += SK_WAVES * WAVE) {
        const int row = t / (SK_BLOCKS / 4), c = t % (SK_BLOCKS / 4) * 4;
        const unsigned char *from = row == 16 * MT ? ws : p.xs + (long long)(m0 + row) * p.xs_stride;
        if (c < p.blocks) *(uint32_t *)(scales + row * PITCH + c) = row < rows || row == 16 * MT ? *(const uint32_t *)(from + c) : 0u;
    }
#pragma unroll
    for (int j = 0; j < RING - 1; j++) fetch_x(j);
#pragma unroll
    for (int a = 0; a < AHEAD; a++) fetch_w(w[a], a);
    __syncthreads();   /* the scales */
    for (int j0 = 0; j0 < steps; j0 += AHEAD + 1) {
#pragma unroll
        for (int a = 0; a <= AHEAD; a++) {
            const int j = j0 + a;
            if (j >= steps) break;
            const int kb = j * S + s;
            /* x of step j has landed: behind it were issued at least the w of its own step and x and w of the steps since (the
             * last of these w may still be held back by the compiler); this wave's reads of the slot filled next are done */
            constexpr int NEWER = (RING - 2) * (DMAS + 2);
            __builtin_amdgcn_s_waitcnt((NEWER & 0xF) | ((NEWER >> 4) << 14) | (0x7 << 4) | (0x0 << 8));
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            fetch_x(j + RING - 1);
            fetch_w(w[(a + AHEAD) % (AHEAD + 1)], j + AHEAD);
            const unsigned char *xb = lds + j % RING * STEP + s * BLOCK;
            w[a].byte = kb < p.blocks ? scales[16 * MT * PITCH + kb] : 0u;
            const Codes32 cw = w[a].codes();
#pragma unroll
            for (int u = 0; u < MT; u++) {
                const int row = 16 * u + i16;
                Codes32 cx;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const u32x4 v = *(const u32x4 *)(xb + row * F8_BLOCK + (((4 * h + g) ^ f8_swizzle(row)) << 4));
#pragma unroll
                    for (int e = 0; e < 4; e++) cx.c[4 * h + e] = v[e];
                }
                cx.byte = kb < p.blocks ? scales[row * PITCH + kb] : 0u;
                sk_product<false>(acc[u], cw, cx);
            }
        }
    }
    __builtin_amdgcn_s_waitcnt(0);   /* no DMA may land on the sums */
    __syncthreads();
    /* sums[s][row][column], fp32: lane (g, i16) has columns 16 rw + 4 g .. + 3 of row 16 u + i16 */
    float *sums = (float *)lds;
#pragma unroll
    for (int u = 0; u < MT; u++) *(f32x4 *)(sums + (s * 16 * MT + 16 * u + i16) * COLS + 16 * rw + 4 * g) = acc[u];
    __syncthreads();
    for (int t = threadIdx.x; t < 16 * MT * COLS / 8; t += SK_WAVES * WAVE) {
        const int row = t / (COLS / 8), c = t % (COLS / 8) * 8;
        if (row >= rows || c >= cols) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = sums[row * COLS + c + e];
#pragma unroll
        for (int k = 1; k < S; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = v[e] + sums[(k * 16 * MT + row) * COLS + c + e];
        *(u32x4 *)((uint16_t *)p.out + (long long)(m0 + row) * p.N + n0 + c) =
            u32x4{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])};
    }
}

template <int RW, int S> int some_go(const Skinny &p, hipStream_t stream) {
    const int parts = (p.M + 31) / 32;
    hipLaunchKernelGGL((fp8_some_kernel<RW, S>), dim3((unsigned)((p.N + 16 * RW - 1) / (16 * RW) * parts)),
                       dim3(SK_WAVES * WAVE), 0, stream, p);
    return (int)hipGetLastError();
}

/* x bf16 or fp32 taken as it is: rows must be readable 16 bytes at a time. Every workgroup reads x and puts it in 8 bits, which tells
 * with many of them, many rows and long ones; else it is two launches to do that first. Microseconds for 1, 4, 8 and 16 rows, against
 * the two launches:
 *    1,280 x 1,280   3.2   3.3   3.5   3.8 (6.8 to 7.4)     16,384 x 1,664    8.8   9.4  10.5  11.8 (10.0 to 10.4)
 *    4,992 x 1,664   5.0   5.4   5.7   6.7 (8.2 to 9.1)     65,536 x 1,664   25.4  25.9  27.7  31.4 (24.8 to 25.7)
 * and from an MLP's squares in fp32, all of it, 6,656 wide: 14.0  16.4  19.0 (18.0 and more). For 17, 32, 37 and 64 rows:
 *    1,280 x 1,280   4.5   5.5   6.2   7.5 (7.4 to 7.8)      1,664 x 1,664    5.3   6.6   7.8   9.4 (7.5 to 7.9)
 *    4,992 x 1,664   9.2  11.7  14.6  17.7 (9.0 to 10.2)     1,280 x 5,120   10.8  14.0  17.4  22.9 (10.1 to 11.1) */
bool few_takes(const void *x, bool f32, long long row_stride, long long rows, int n, int k) {
    const long long size = f32 ? 4 : 2, tiles = n / 16, cus = device_cus();
    const bool few = f32 ? rows <= 4 : rows <= 16 || (rows <= 64 && tiles <= cus && rows * k <= 640 * F8_BLOCK);
    return few && tiles <= 4 * cus && (rows > 16 || rows * tiles <= 32 * cus) && !((uintptr_t)x & 15) &&
           (rows == 1 || (row_stride * size % 16 == 0 && row_stride <= 1 << 22));
}
int few(const void *x, bool f32, long long row_stride, const void *w, const void *ws, int ws_stride, int rows, int n, int k,
        bool relu2, void *out, hipStream_t stream) {
    const Skinny p = {x, (rows > 1 ? row_stride : k) * (f32 ? 4 : 2), nullptr, 0, ws_stride, (const unsigned char *)w,
                      (const unsigned char *)ws, rows, n, k, (k + F8_BLOCK - 1) / F8_BLOCK, out};
    const auto kernel = relu2        ? fp8_few_kernel<SK_BF16, 1, true>
                        : f32        ? fp8_few_kernel<SK_F32, 1, false>
                        : rows <= 16 ? fp8_few_kernel<SK_BF16, 1, false>
                        : rows <= 32 ? fp8_few_kernel<SK_BF16, 2, false> : fp8_few_kernel<SK_BF16, 4, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(n / 16)), dim3(SK_WAVES * WAVE), 0, stream, p);
    return (int)hipGetLastError();
}

bool serve_sizes(long long rows, int n, int k) {
    return rows >= 0 && n > 0 && k > 0 && n % 16 == 0 && k % 16 == 0 && n <= 1 << 20 && k <= 1 << 20 &&
           rows <= (1LL << 31) / ((k + F8_BLOCK - 1) / F8_BLOCK) - 32;
}
bool weight_pitch(int stride, int k) { return stride >= (k + F8_BLOCK - 1) / F8_BLOCK && stride % 4 == 0 && stride <= 1 << 14; }

int linear(const void *x, int is_f32, long long row_stride, const void *w, const void *ws, int ws_stride, long long rows, int n,
           int k, void *out, void *workspace, hipStream_t stream) {
    if (few_takes(x, is_f32, row_stride, rows, n, k))
        return few(x, is_f32, row_stride, w, ws, ws_stride, (int)rows, n, k, false, out, stream);
    const F8Form f(workspace, rows, k);
    const int status = nc_fp8_quantize_rows(x, is_f32, row_stride, rows, k, f.codes, f.scale, f.pitch, stream);
    return status ? status : nc_fp8_matmul(f.codes, f.scale, f.pitch, w, ws, ws_stride, rows, n, k, out, stream);
}

}  // namespace

/* The number of (16 rows of w) x (32 rows of x): the waves of a workgroup split k eight ways while there are fewer than the CUs, four
 * ways while there are fewer than twice as many. */
static long long some_tiles(long long rows, int n) { return (n + 15) / 16 * ((rows + 31) / 32); }
bool fp8_some_takes(long long rows, int n, int k, long long cus) {
    return k <= SK_BLOCKS * F8_BLOCK && some_tiles(rows, n) < 2 * cus;
}

int fp8_some(const void *codes, const void *scale, long long scale_stride, const void *w, const void *w_scale, int w_scale_stride,
             int rows, int n, int k, void *out, hipStream_t stream) {
    const Skinny p = {codes, k, (const unsigned char *)scale, (int)scale_stride, w_scale_stride, (const unsigned char *)w,
                      (const unsigned char *)w_scale, rows, n, k, (k + F8_BLOCK - 1) / F8_BLOCK, out};
    return some_tiles(rows, n) < device_cus() ? some_go<1, 8>(p, stream) : some_go<2, 4>(p, stream);
}

}  // namespace nc

using namespace nc;

extern "C" long long nc_fp8_linear_workspace_bytes(const void *x, int is_f32, long long row_stride, long long rows, int n, int k) {
    if (!serve_sizes(rows, n, k)) return -1;
    return rows == 0 || few_takes(x, is_f32, row_stride, rows, n, k) ? 0 : f8_form_bytes(rows, k);
}

extern "C" int nc_fp8_linear(const void *x, int is_f32, long long row_stride, const void *w, const void *w_scale,
                             int w_scale_stride, long long rows, int n, int k, void *out, void *workspace,
                             long long workspace_bytes, void *stream) {
    if (!serve_sizes(rows, n, k) || (rows > 1 && row_stride < k) || row_stride > (1LL << 40) ||
        !weight_pitch(w_scale_stride, k))
        return NC_ERR_SHAPE;
    if (rows == 0) return NC_OK;
    if (!x || !w || !w_scale || !out) return NC_ERR_NULL;
    if (f8_misaligned(x, is_f32 ? 4 : 2) || f8_misaligned(w, 16) || f8_misaligned(w_scale, 4) || f8_misaligned(out, 16)) return NC_ERR_SHAPE;
    const long long need = nc_fp8_linear_workspace_bytes(x, is_f32, row_stride, rows, n, k);
    if (need > 0 && !workspace) return NC_ERR_NULL;
    if (need > 0 && (f8_misaligned(workspace, 16) || workspace_bytes < need)) return NC_ERR_WORKSPACE;
    return linear(x, is_f32, row_stride, w, w_scale, w_scale_stride, rows, n, k, out, workspace, (hipStream_t)stream);
}

/* x's form, then the squared activations: in the 8-bit form, or for up to 16 rows in fp32 and then in that form. */
extern "C" long long nc_fp8_mlp_workspace_bytes(long long rows, int c, int hidden) {
    if (!serve_sizes(rows, hidden, c) || !serve_sizes(rows, 16, hidden)) return -1;
    return f8_form_bytes(rows, c) + f8_form_bytes(rows, hidden) + (rows <= 16 ? 4 * rows * hidden : 0);
}

static int mlp(bool fast, const void *x, long long row_stride, const void *fc, const void *fc_scale, int fc_scale_stride,
               const void *proj, const void *proj_scale, int proj_scale_stride, long long rows, int c, int hidden, int n, void *out,
               void *workspace, long long workspace_bytes, void *stream) {
    if (!serve_sizes(rows, hidden, c) || !serve_sizes(rows, n, hidden) || (rows > 1 && row_stride < c) ||
        row_stride > (1LL << 40) || !weight_pitch(fc_scale_stride, c) || !weight_pitch(proj_scale_stride, hidden))
        return NC_ERR_SHAPE;
    if (rows == 0) return NC_OK;
    if (!x || !fc || !fc_scale || !proj || !proj_scale || !out || !workspace) return NC_ERR_NULL;
    if (f8_misaligned(x, 2) || f8_misaligned(fc, 16) || f8_misaligned(fc_scale, 4) || f8_misaligned(proj, 16) || f8_misaligned(proj_scale, 4) ||
        f8_misaligned(out, 16))
        return NC_ERR_SHAPE;
    if (f8_misaligned(workspace, 16) || workspace_bytes < nc_fp8_mlp_workspace_bytes(rows, c, hidden)) return NC_ERR_WORKSPACE;
    const hipStream_t s = (hipStream_t)stream;
    const F8Form f(workspace, rows, c), a(f.codes + f.bytes, rows, hidden);
    if (rows <= 16 && few_takes(x, false, row_stride, rows, hidden, c)) {
        float *const act = (float *)(a.codes + a.bytes);
        const int status = few(x, false, row_stride, fc, fc_scale, fc_scale_stride, (int)rows, hidden, c, true, act, s);
        return status ? status : linear(act, 1, hidden, proj, proj_scale, proj_scale_stride, rows, n, hidden, out, a.codes, s);
    }
    int status = nc_fp8_quantize_rows(x, 0, row_stride, rows, c, f.codes, f.scale, f.pitch, stream);
    if (!status)
        status = (fast ? nc_fp8_matmul_relu2_fast : nc_fp8_matmul_relu2)(f.codes, f.scale, f.pitch, fc, fc_scale, fc_scale_stride,
                                                                           rows, hidden, c, a.codes, a.scale, a.pitch, stream);
    return status ? status : nc_fp8_matmul(a.codes, a.scale, a.pitch, proj, proj_scale, proj_scale_stride, rows, n, hidden, out,
                                           stream);
}

extern "C" int nc_fp8_mlp(const void *x, long long row_stride, const void *fc, const void *fc_scale, int fc_scale_stride,
                          const void *proj, const void *proj_scale, int proj_scale_stride, long long rows, int c, int hidden,
                          int n, void *out, void *workspace, long long workspace_bytes, void *stream) {
    return mlp(false, x, row_stride, fc, fc_scale, fc_scale_stride, proj, proj_scale, proj_scale_stride, rows, c, hidden, n, out,
               workspace, workspace_bytes, stream);
}

extern "C" int nc_fp8_mlp_fast(const void *x, long long row_stride, const void *fc, const void *fc_scale, int fc_scale_stride,
                                const void *proj, const void *proj_scale, int proj_scale_stride, long long rows, int c, int hidden,
                                int n, void *out, void *workspace, long long workspace_bytes, void *stream) {
    return mlp(true, x, row_stride, fc, fc_scale, fc_scale_stride, proj, proj_scale, proj_scale_stride, rows, c, hidden, n, out,
               workspace, workspace_bytes, stream);
}
