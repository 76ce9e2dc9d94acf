/*
 * The gradient of a weight from the 8-bit checkpoint of its layer's input on gfx950: out[i][j] (+)= sum_m dy[m][i] x[m][j] over
 * token rows m, dy bf16 [M][N1], x in the 8-bit form (nc_fp8.h) [M][N2] with a scale for each 128 columns of a token.
 *
 * The scale changes along the summed dimension, so the products cannot be taken in 8 bits. A code times a power of two is
 * exact in bf16, so x is unpacked on its way into LDS and the products are v_mfma_f32_16x16x32_bf16, fp32 sums, as exact as
 * those of a bf16 input: only half of that input's bytes are read.
 *
 * A workgroup owns a 256 x 256 tile of the result and a slice of the tokens, walked in stages of 32: four waves, one a SIMD, of
 * 128 x 128 results each (all 256 AGPRs of a lane), which read the next stage's operands from LDS into the other half of 128
 * registers between this stage's products. dy's 256 columns go into LDS by DMA four stages ahead, x's codes and scales five
 * stages ahead; a thread turns its own 32 codes into bf16 two stages before they are multiplied. Operands are read transposed
 * (ds_read_b64_tr_b16: four tokens of one column a lane). A 512-byte row keeps its 32-byte piece s at place s ^ (row % 8), so
 * that the eight rows that half a wave reads meet in different banks.
 *
 * The result is small and the sum long: where tiles alone would leave CUs idle the tokens are cut into slices, whose partial
 * tiles fp8_grad_sum_kernel adds in slice order, so the result does not depend on scheduling.
 *
 * Bound by the matrix cores at bf16's rate and by the LDS reads beside them: 65,536 x 4,992 x 1,664 943 us (1,154 TFLOP/s; a library
 * product of 8,192^3 reaches 1,530), x 6,656 x 1,664 1,206, x 1,664 x 6,656 1,176; 16,384 x 5,120 x 1,280 199; 1,001 x 5,120 x 1,280
 * 30, mostly its partial tiles. Eight waves of 64 x 128 with operands made by all took 1,444 where this takes 943.
 */
#include "nanochat_amd.h"
#include "nc_fp8.h"
#include "nc_internal.h"

namespace nc {
namespace {

typedef __amdgpu_buffer_rsrc_t Rsrc;
typedef __attribute__((address_space(3))) void LdsPtr;
typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16 LdsV4;

constexpr int GR_T = 256;                     /* a tile's rows and columns */
constexpr int GR_KC = 32;                     /* tokens of a stage */
constexpr int GR_ROWB = GR_T * 2;
constexpr int GR_OPB = GR_KC * GR_ROWB;       /* a stage's operand in LDS: 16 KiB */
constexpr int GR_WAVES = 4;
constexpr int GR_PAST = 0x7FFF0000;           /* a byte offset past every operand's range */

enum { GR_PART, GR_ADD, GR_F32, GR_BF16 };

struct F8Grad {
    const uint16_t *dy;                       /* [M][N1] */
    const unsigned char *x, *xs;              /* [M][N2], [M] at xs_stride */
    long long xs_stride, M;
    int N1, N2, tiles1, tiles2, slices, rows;         /* rows: of a slice, a multiple of GR_KC */
    void *out;                                /* PART: fp32 [slices][N1][N2]; else the result [N1][N2] */
};

/* Two results over the same tokens in one launch: the first workgroups' and the others'. */
struct F8Grads {
    F8Grad of[2];
    int first;                                /* workgroups of the first result */
};

/* LDS: four stages of dy, two of x in bf16, four of x's codes, eight of its scale dwords (a token's two blocks lie in one). */
constexpr int GR_CODES = GR_KC * GR_T;
constexpr int GR_X = 4 * GR_OPB, GR_XC = GR_X + 2 * GR_OPB, GR_XS = GR_XC + 4 * GR_CODES, GR_LDS = GR_XS + 8 * 128;

/* The DMA of a workgroup, a wave's part. dy: instruction s moves rows 2 q, 2 q + 1, q = wave + 4 s; lane l row 2 q + l / 32, LDS
 * piece (l % 32) / 2, half l % 2. x's codes: rows 4 q .. + 3, lane l row 4 q + l / 16, columns 16 (l % 16) .. + 15, q = wave + 4 s.
 * Scales: every wave asks for all 64 tokens' dwords of two stages, lane l token l, so that each waits for its own. */
struct GrDma {
    u32x4 ra, rx, rs;
    uint32_t lds;                 /* the workgroup's LDS */
    uint32_t a, x, s;             /* this lane's offsets of instruction 0 in stage 0 (GR_PAST: a column past the result's) */
    uint32_t s_row;               /* bytes of a token's scales */
    int wave;
    uint32_t lds_a, lds_x;        /* where the next stage's go */
    uint32_t a8, a16, a24, x16;   /* bytes of 8, 16, 24 and 16 tokens */
    __device__ __forceinline__ void at_a(int j) { lds_a = lds + (j & 3) * GR_OPB + wave * 1024; }
    __device__ __forceinline__ void at_x(int j) { lds_x = lds + GR_XC + (j & 3) * GR_CODES + wave * 1024; }
    /* Instruction K of the next stage of dy, of x's codes, and (every other stage) the scale dwords of 64 tokens; after the last
     * one the offsets move on. */
    template <int K> __device__ __forceinline__ void issue_a() {
        f8_dma16<4096 * K>(lds_a, a, K == 0 ? 0u : K == 1 ? a8 : K == 2 ? a16 : a24, ra);
        if constexpr (K == 3) a += 4 * a8;
    }
    template <int K> __device__ __forceinline__ void issue_x() {
        f8_dma16<4096 * K>(lds_x, x, K == 0 ? 0u : x16, rx);
        if constexpr (K == 1) x += 2 * x16;
    }
    __device__ __forceinline__ void issue_s(int j) {   /* stages j and j + 1, j even */
        f8_dma4(lds + GR_XS + (j & 6) * 128, s, rs);
        s += 2 * GR_KC * s_row;
    }
};

/* A thread's 2 x 16 codes of a stage of x (tokens tid / 16 and 16 on, columns 16 (tid % 16) .. + 15) and their scales, as its
 * own wave's DMA left them, on their way to bf16. The empty asm statements keep each conversion where it is written. */
struct GrUnpack {
    u32x4 c[2], o[2];
    float s[2];
    uint32_t byte[2];
    template <int K> __device__ __forceinline__ void read(const unsigned char *lds, int j, int tid, int scale_byte) {
        c[K] = *(const u32x4 *)(lds + GR_XC + (j & 3) * GR_CODES + tid * 16 + 4096 * K);
        byte[K] = lds[GR_XS + (j & 7) * 128 + ((tid >> 4) + 16 * K) * 4 + scale_byte];
    }
    /* Tokens past the slice have codes and byte 0, and stay zeros. */
    template <int K> __device__ __forceinline__ void scale() {
        asm volatile("" : "+v"(byte[K]));
        s[K] = f8_scale(byte[K] < 1u ? 1u : byte[K]);
        asm volatile("" : "+v"(s[K]));
    }
    template <int K, int I> __device__ __forceinline__ void convert() {   /* codes 4 I .. + 3 */
        uint32_t w = c[K][I];
        asm volatile("" : "+v"(w));
        uint32_t lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, s[K], false));
        uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, s[K], true));
        asm volatile("" : "+v"(lo), "+v"(hi));
        o[I >> 1][2 * (I & 1)] = lo;
        o[I >> 1][2 * (I & 1) + 1] = hi;
    }
    template <int K> __device__ __forceinline__ void write(unsigned char *to, int tid) const {
        const int row = (tid >> 4) + 16 * K, piece = tid & 15;
        u32x4 *at = (u32x4 *)(to + row * GR_ROWB + ((piece ^ (row & 7)) << 5));
        at[0] = o[0];
        at[1] = o[1];
    }
    template <int K> __device__ __forceinline__ void all(const unsigned char *lds, int j, int tid, int scale_byte,
                                                         unsigned char *to) {
        read<K>(lds, j, tid, scale_byte);
        scale<K>();
        convert<K, 0>();
        convert<K, 1>();
        convert<K, 2>();
        convert<K, 3>();
        write<K>(to, tid);
    }
};

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

/* A wave's operands of a stage: 128 columns of dy, 128 of x. */
struct Operands {
    bf16x8 a[8], b[8];
};

/* The products as inline assembly: accumulators that stay in their AGPRs for the whole walk ("+a"; all 256). The compiler sees
 * no matrix instructions there and inserts none of their wait states; they are kept by construction: operands are written by LDS
 * reads alone, a step earlier; an accumulator is used again 63 products later, and read 32 wait states after the last one. */
__device__ __forceinline__ void gr_mfma(f32x4 &c, const bf16x8 &a, const bf16x8 &b) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}

/* All but the DMA of the last two steps (6 and 7: an odd one brings scales) has landed, and this wave's LDS reads and writes are
 * done. */
__device__ __forceinline__ void gr_wait() { __builtin_amdgcn_s_waitcnt(13 | (0x7 << 4) | (0x0 << 8)); }

/* What a step does between its products, behind product I of 64: a product keeps the matrix core busy for 16 cycles, in which
 * the wave (one a SIMD) issues up to three more instructions; in a run they would let the core idle. */
struct GrStep {
    const unsigned char *lds, *la, *lb;   /* the workgroup's LDS, dy and x of stage j + 1 */
    unsigned char *to;                    /* where x of stage j + 2 becomes bf16 */
    int j, tid, scale_byte, wm, wn, g, c;
    template <int I, bool EVEN> __device__ __forceinline__ void side(Operands &next, GrUnpack &f, GrDma &dma) const {
        if constexpr (I < 32 && I % 4 == 1) next.b[I / 4] = gr_operand(lb, 8 * wn + I / 4, g, c);
        if constexpr (I < 32 && I % 4 == 3) next.a[I / 4] = gr_operand(la, 8 * wm + I / 4, g, c);
        if constexpr (I == 2) dma.at_a(j + 4);
        if constexpr (I < 32 && I % 8 == 4) dma.issue_a<I / 8>();
        if constexpr (I == 35) dma.at_x(j + 5);
        if constexpr (I == 37) dma.issue_x<0>();
        if constexpr (I == 40) dma.issue_x<1>();
        if constexpr (I == 58 && !EVEN) dma.issue_s(j + 5);
        if constexpr (I == 32) f.read<0>(lds, j + 2, tid, scale_byte);
        if constexpr (I == 34) f.read<1>(lds, j + 2, tid, scale_byte);
        if constexpr (I == 42) f.scale<0>();
        if constexpr (I == 43) f.convert<0, 0>();
        if constexpr (I == 45) f.convert<0, 1>();
        if constexpr (I == 46) f.convert<0, 2>();
        if constexpr (I == 47) f.convert<0, 3>();
        if constexpr (I == 48) f.write<0>(to, tid);
        if constexpr (I == 50) f.scale<1>();
        if constexpr (I == 51) f.convert<1, 0>();
        if constexpr (I == 53) f.convert<1, 1>();
        if constexpr (I == 54) f.convert<1, 2>();
        if constexpr (I == 55) f.convert<1, 3>();
        if constexpr (I == 56) f.write<1>(to, tid);
    }
    template <bool EVEN, int I = 0>
    __device__ __forceinline__ void run(f32x4 (&acc)[8][8], const Operands &cur, Operands &next, GrUnpack &f, GrDma &dma) const {
        if constexpr (I < 64) {
            gr_mfma(acc[I / 8][I % 8], cur.a[I / 8], cur.b[I % 8]);
            side<I, EVEN>(next, f, dma);
            run<EVEN, I + 1>(acc, cur, next, f, dma);
        }
    }
};

/* Step j: the products of stage j, whose operands are in CUR, while NEXT takes those of stage j + 1; x of stage j + 2 becomes
 * bf16; dy of stage j + 4 and x's codes of stage j + 5 are fetched (into the buffers of stages j and j + 1, whose readers are a
 * barrier behind). EVEN: j's parity, that of its bf16 buffer. */
#define GR_STEP(j, EVEN, CUR, NEXT)                                                                               \
    do {                                                                                                           \
        gr_wait();                                                                                                 \
        gr_barrier();                                                                                              \
        const GrStep step = {lds, lds + (((j) + 1) & 3) * GR_OPB, lds + GR_X + (1 - (EVEN)) * GR_OPB,              \
                             lds + GR_X + (EVEN) * GR_OPB, (j), tid, scale_byte, wm, wn, g, c};                    \
        GrUnpack f;                                                                                                \
        step.run<(EVEN) == 0>(acc, CUR, NEXT, f, dma);                                                                          \
    } while (0)

template <int MODE>
__global__ void __launch_bounds__(GR_WAVES *WAVE, 1) fp8_grad_kernel(F8Grads both) {
    __shared__ __align__(16) unsigned char lds[GR_LDS];
    const bool second = (int)blockIdx.x >= both.first;
    const F8Grad &p = both.of[second];
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int wm = wave >> 1, wn = wave & 1;
    /* Workgroup L runs on XCD L % 8: each XCD takes a contiguous run of (slice, band of 4 row tiles, column tile, row tile), so
     * that what it runs at once reads the same tokens of few columns. */
    const int tiles = p.tiles1 * p.tiles2, l = second ? blockIdx.x - both.first : blockIdx.x;
    const int count = second ? gridDim.x - both.first : both.first, per = count / 8, extra = count % 8;
    const int id = l % 8 * per + min(l % 8, extra) + l / 8, slice = id / tiles, tile = id % tiles;
    const int band = tile / (4 * p.tiles2), tall = min(4, p.tiles1 - 4 * band), in = tile - band * 4 * p.tiles2;
    const int i0 = (4 * band + in % tall) * GR_T, j0 = in / tall * GR_T;
    const long long m0 = (long long)slice * p.rows;
    const int rows = (int)(p.M - m0 < p.rows ? p.M - m0 : p.rows);   /* > 0: the host makes no empty slice */
    GrDma dma;
    dma.ra = f8_words(p.dy + m0 * p.N1, (long long)rows * p.N1 * 2);
    dma.rx = f8_words(p.x + m0 * p.N2, (long long)rows * p.N2);
    dma.rs = f8_words(p.xs + m0 * p.xs_stride, f8_scale_range(rows, p.xs_stride, (p.N2 + F8_BLOCK - 1) / F8_BLOCK));
    dma.lds = f8_lds(lds);
    dma.wave = wave;
    dma.s_row = (uint32_t)p.xs_stride;
    dma.a8 = 16 * p.N1;
    dma.a16 = 32 * p.N1;
    dma.a24 = 48 * p.N1;
    dma.x16 = 16 * p.N2;
    {
        const int row = 2 * wave + (lane >> 5), col = i0 + (((lane & 31) >> 1) ^ (row & 7)) * 16 + (lane & 1) * 8;
        dma.a = col < p.N1 ? (uint32_t)(row * p.N1 + col) * 2 : GR_PAST;   /* rows 8 on have the same piece */
        const int xrow = 4 * wave + (lane >> 4), xcol = j0 + 16 * (lane & 15);
        dma.x = xcol < p.N2 ? (uint32_t)(xrow * p.N2 + xcol) : GR_PAST;
        dma.s = lane * dma.s_row + (j0 / F8_BLOCK & ~3);
    }
    const int scale_byte = (j0 / F8_BLOCK & 3) + ((tid & 15) >> 3);
    const int stages = (rows + GR_KC - 1) / GR_KC;
    f32x4 acc[8][8];
#pragma unroll
    for (int t = 0; t < 8; t++)
#pragma unroll
        for (int u = 0; u < 8; u++) asm volatile("" : "=a"(acc[t][u]) : "0"(f32x4{0.0f, 0.0f, 0.0f, 0.0f}));
    const auto fetch_x = [&](int j) {
        if (!(j & 1)) dma.issue_s(j);
        dma.at_x(j);
        dma.issue_x<0>();
        dma.issue_x<1>();
    };
#pragma unroll
    for (int j = 0; j < 4; j++) {
        fetch_x(j);
        dma.at_a(j);
        dma.issue_a<0>();
        dma.issue_a<1>();
        dma.issue_a<2>();
        dma.issue_a<3>();
    }
    __builtin_amdgcn_s_waitcnt((17 & 0xF) | ((17 >> 4) << 14) | (0x7 << 4) | (0xF << 8));   /* x of 0 and 1, dy of 0 */
#pragma unroll
    for (int j = 0; j < 2; j++) {
        GrUnpack f;
        f.all<0>(lds, j, tid, scale_byte, lds + GR_X + j * GR_OPB);
        f.all<1>(lds, j, tid, scale_byte, lds + GR_X + j * GR_OPB);
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);   /* the LDS writes */
    gr_barrier();
    fetch_x(4);
    Operands o0, o1;
#pragma unroll
    for (int t = 0; t < 8; t++) {
        o0.b[t] = gr_operand(lds + GR_X, 8 * wn + t, g, c);
        o0.a[t] = gr_operand(lds, 8 * wm + t, g, c);
    }
    for (int j = 0; j < stages; j += 2) {   /* a stage past the slice reads zeros and adds nothing */
        GR_STEP(j, 0, o0, o1);
        GR_STEP(j + 1, 1, o1, o0);
    }
    __builtin_amdgcn_s_waitcnt(0);   /* no DMA may land in LDS after the workgroup ends */
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");   /* 32 wait states; no read moves above */
#pragma unroll
    for (int t = 0; t < 8; t++)
#pragma unroll
        for (int u = 0; u < 8; u++) asm volatile("" : "+a"(acc[t][u]));
    /* lane (g, c) of result tile (t, u): rows i0 + 128 wm + 16 t + 4 g + e, column j0 + 128 wn + 16 u + c; 32-bit offsets into the
     * tile's rows, those past N1 and columns past N2 outside the range */
    constexpr int SIZE = MODE == GR_BF16 ? 2 : 4;
    const int live = p.N1 - i0 < GR_T ? p.N1 - i0 : GR_T;
    const unsigned row_bytes = (unsigned)p.N2 * SIZE;
    const long long first = ((MODE == GR_PART ? (long long)slice * p.N1 : 0) + i0) * p.N2;
    const Rsrc ro = f8_rsrc((unsigned char *)p.out + first * SIZE, (long long)live * row_bytes);
    unsigned at[8];
#pragma unroll
    for (int u = 0; u < 8; u++) {
        const int col = j0 + 128 * wn + 16 * u + c;
        at[u] = col < p.N2 ? (unsigned)(128 * wm + 4 * g) * row_bytes + (unsigned)col * SIZE : (unsigned)GR_PAST;
    }
    float old[2][8][4];   /* ADD: the result's rows of t, and of t + 1 in flight */
    const auto fetch_old = [&](int t) {
#pragma unroll
        for (int u = 0; u < 8; u++)
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
        for (int u = 0; u < 8; u++)
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

/* What M tokens take in us by a model of measured parts, one workgroup a CU: rounds of workgroups, each a slice's stages and ten
 * more for its start and its end; a stage 0.6 and up to 0.15 more with every CU at work (clock, and the L2s shared); a slice's
 * partial tiles out and back at 4.5 TB/s. One slice has none. */
double grad_time(long long tiles, long long elements, int cus, long long slices, long long rows) {
    const double rounds = (double)((tiles * slices + cus - 1) / cus), busy = (double)(tiles * slices) / (rounds * cus);
    const double partials = slices == 1 ? 0.0 : 3.0 + slices * elements * 8.0 / 4.5e6;
    return rounds * (rows / GR_KC + 10) * (0.6 + 0.15 * busy) + partials;
}

/* How the tokens of one result, or of two in one launch, are cut. */
struct GrPlan {
    int slices, rows;
    double time;
};
/* The best of a few counts by grad_time (small ones, steps of about a quarter above, and those that just fill one to six rounds),
 * no slice under GR_MIN_ROWS rows unless it is the only one and none whose operand slice passes 1 GiB. */
GrPlan grad_plan(long long M, long long tiles, long long elements, long long row_bytes) {
    const long long fit = (1LL << 30) / row_bytes / GR_KC * GR_KC;
    const long long least = (M + fit - 1) / fit, most = (M + GR_MIN_ROWS - 1) / GR_MIN_ROWS;
    const int cus = device_cus();
    GrPlan best = {0, 0, -1.0};
    auto consider = [&](long long s) {
        s = s < most ? s : most;
        s = s > least ? s : least;
        const long long r = ((M + s - 1) / s + GR_KC - 1) / GR_KC * GR_KC;
        if (r > fit) return;
        s = (M + r - 1) / r;   /* no empty slice */
        const double t = grad_time(tiles, elements, cus, s, r);
        if (best.time < 0.0 || t < best.time) best = {(int)s, (int)r, t};
    };
    for (long long s = 1; s <= most && (s == 1 || tiles * s <= 6LL * cus); s += s < 8 ? 1 : s / 4) consider(s);
    for (int k = 1; k <= 6; k++)
        if (k * cus >= tiles) consider(k * cus / tiles);
    return best;
}
int tiles_of(int n) { return (n + GR_T - 1) / GR_T; }
long long row_of(int n1, int n2) { return 2LL * n1 > n2 ? 2LL * n1 : n2; }
GrPlan grad_alone(long long M, int n1, int n2) {
    return grad_plan(M, (long long)tiles_of(n1) * tiles_of(n2), (long long)n1 * n2, row_of(n1, n2));
}
/* Both in one launch, where that takes less time than one after the other (with slices = 0: it does not). 200 tiles for 256 CUs are
 * one round in place of two of 100: 1,001 tokens x (5,120 x 1,280 and 1,280 x 5,120) 64 -> 34 us. */
GrPlan grad_both(long long M, const int (&n1)[2], const int (&n2)[2]) {
    const long long r0 = row_of(n1[0], n2[0]), r1 = row_of(n1[1], n2[1]);
    const GrPlan both = grad_plan(M, (long long)tiles_of(n1[0]) * tiles_of(n2[0]) + (long long)tiles_of(n1[1]) * tiles_of(n2[1]),
                                  (long long)n1[0] * n2[0] + (long long)n1[1] * n2[1], r0 > r1 ? r0 : r1);
    return both.time < 0.95 * (grad_alone(M, n1[0], n2[0]).time + grad_alone(M, n1[1], n2[1]).time) ? both : GrPlan{0, 0, 0.0};
}

/* One slice needs none (never 0 where there is a call). */
long long grad_bytes(int slices, long long elements) { return slices == 1 ? 16 : slices * elements * 4; }

bool grad_fits(long long M, int N1, int N2) {
    return M >= 0 && M < (1LL << 31) && N1 > 0 && N2 > 0 && N1 % 8 == 0 && N2 % 16 == 0 && N1 <= 65536 && N2 <= 65536;
}

int grad_check(const GradOf &g, long long rows, const void *workspace) {
    if (const int e = fp8_weight_grad_refuses(g, rows)) return e;
    if (rows == 0) return NC_OK;
    return !workspace ? NC_ERR_NULL : (uintptr_t)workspace & 15 ? NC_ERR_SHAPE : NC_OK;
}

int grad_launch(const GradOf *g, int results, const GrPlan &plan, long long rows, void *workspace, hipStream_t s) {
    F8Grads both = {};
    int workgroups = 0;
    char *part = (char *)workspace;
    void *parts[2];
    for (int i = 0; i < results; i++) {
        both.of[i] = {(const uint16_t *)g[i].dy, (const unsigned char *)g[i].codes, (const unsigned char *)g[i].scale,
                      g[i].scale_stride, rows, g[i].n1, g[i].n2, tiles_of(g[i].n1), tiles_of(g[i].n2), plan.slices, plan.rows,
                      plan.slices == 1 ? g[i].out : part};
        parts[i] = part;
        part += (long long)plan.slices * g[i].n1 * g[i].n2 * 4;
        workgroups += both.of[i].tiles1 * both.of[i].tiles2 * plan.slices;
        if (i == 0) both.first = workgroups;
    }
    const auto kernel = plan.slices > 1    ? fp8_grad_kernel<GR_PART>
                        : g[0].mode == 0   ? fp8_grad_kernel<GR_F32>
                        : g[0].mode == 1   ? fp8_grad_kernel<GR_ADD> : fp8_grad_kernel<GR_BF16>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)workgroups), dim3(GR_WAVES * WAVE), 0, s, both);
    for (int i = 0; plan.slices > 1 && i < results; i++) {
        const long long n4 = (long long)g[i].n1 * g[i].n2 / 4;
        const auto sum = g[i].mode == 0 ? fp8_grad_sum_kernel<GR_F32> : g[i].mode == 1 ? fp8_grad_sum_kernel<GR_ADD>
                                                                                           : fp8_grad_sum_kernel<GR_BF16>;
        hipLaunchKernelGGL(sum, dim3((unsigned)((n4 + 255) / 256)), dim3(256), 0, s, (const float4 *)parts[i], plan.slices, n4,
                           g[i].out);
    }
    return (int)hipGetLastError();
}

/* Two results can share a launch that writes them itself only in one mode; partials are alike. */
GrPlan grad_shared(long long rows, const int (&n1)[2], const int (&n2)[2], int mode0, int mode1) {
    const GrPlan both = grad_both(rows, n1, n2);
    return both.slices > 1 || mode0 == mode1 ? both : GrPlan{0, 0, 0.0};
}

}  // namespace

/* Sizes first, then pointers, then their alignment. A slice's scales take no more bytes than its codes. */
int fp8_weight_grad_refuses(const GradOf &g, long long rows) {
    if (!grad_fits(rows, g.n1, g.n2) || g.mode < 0 || g.mode > 2 || g.scale_stride < (g.n2 + F8_BLOCK - 1) / F8_BLOCK ||
        g.scale_stride > g.n2 || g.scale_stride % 4)
        return NC_ERR_SHAPE;
    if (rows == 0) return NC_OK;
    if (!g.dy || !g.codes || !g.scale || !g.out) return NC_ERR_NULL;
    return ((uintptr_t)g.dy | (uintptr_t)g.codes | (uintptr_t)g.out) & 15 || (uintptr_t)g.scale & 3 ? NC_ERR_SHAPE : NC_OK;
}

long long fp8_weight_grads_bytes(long long rows, int n1, int n2, int mode, int m1, int m2, int other) {
    if (!grad_fits(rows, n1, n2) || !grad_fits(rows, m1, m2)) return -1;
    if (rows == 0) return 0;
    const int a[2] = {n1, m1}, b[2] = {n2, m2};
    const GrPlan both = grad_shared(rows, a, b, mode, other);
    const long long x = nc_fp8_weight_grad_workspace_bytes(rows, n1, n2), y = nc_fp8_weight_grad_workspace_bytes(rows, m1, m2);
    const long long z = both.slices ? grad_bytes(both.slices, (long long)n1 * n2 + (long long)m1 * m2) : 0;
    return x > y ? x > z ? x : z : y > z ? y : z;   /* both plans: which one it is depends on the results' places */
}

/* Results that overlap (one buffer that both are added to) are not made at once. */
static bool grads_overlap(const GradOf (&g)[2]) {
    const char *at[2], *end[2];
    for (int i = 0; i < 2; i++) {
        at[i] = (const char *)g[i].out;
        end[i] = at[i] + (long long)g[i].n1 * g[i].n2 * (g[i].mode == 2 ? 2 : 4);
    }
    return at[0] < end[1] && at[1] < end[0];
}

int fp8_weight_grads(const GradOf (&g)[2], long long rows, void *workspace, long long workspace_bytes, hipStream_t stream) {
    for (int i = 0; i < 2; i++)
        if (const int e = grad_check(g[i], rows, workspace)) return e;
    if (rows == 0) return NC_OK;
    const int a[2] = {g[0].n1, g[1].n1}, b[2] = {g[0].n2, g[1].n2};
    const GrPlan both = grad_shared(rows, a, b, g[0].mode, g[1].mode);
    if (workspace_bytes < fp8_weight_grads_bytes(rows, a[0], b[0], g[0].mode, a[1], b[1], g[1].mode)) return NC_ERR_WORKSPACE;
    if (both.slices && !grads_overlap(g)) return grad_launch(g, 2, both, rows, workspace, stream);
    const int status = grad_launch(g, 1, grad_alone(rows, a[0], b[0]), rows, workspace, stream);
    return status ? status : grad_launch(g + 1, 1, grad_alone(rows, a[1], b[1]), rows, workspace, stream);
}

}  // namespace nc

using namespace nc;

extern "C" long long nc_fp8_weight_grad_workspace_bytes(long long rows, int n1, int n2) {
    if (!grad_fits(rows, n1, n2)) return -1;
    return rows == 0 ? 0 : grad_bytes(grad_alone(rows, n1, n2).slices, (long long)n1 * n2);
}

extern "C" int nc_fp8_weight_grad(const void *dy, const void *codes, const void *scale, long long scale_stride, long long rows,
                                  int n1, int n2, int mode, void *out, void *workspace, long long workspace_bytes,
                                  void *stream) {
    const GradOf g = {dy, codes, scale, scale_stride, n1, n2, mode, out};
    const int e = grad_check(g, rows, workspace);
    if (e != NC_OK || rows == 0) return e;
    const GrPlan plan = grad_alone(rows, n1, n2);
    if (workspace_bytes < grad_bytes(plan.slices, (long long)n1 * n2)) return NC_ERR_WORKSPACE;
    return grad_launch(&g, 1, plan, rows, workspace, (hipStream_t)stream);
}
