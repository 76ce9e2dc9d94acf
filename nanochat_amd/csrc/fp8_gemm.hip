/*
 * Products of two matrices in the 8-bit form (nc_fp8.h) on gfx950: out[m][n] = epilogue(sum_k a[m][k] w[n][k]), a with a scale
 * for each 128 columns of a row, w for each 128 x 128.
 *
 * v_mfma_scale_f32_16x16x128_f8f6f4 takes one block a step and applies both scales itself: its A operand holds 16 weight rows,
 * its B operand 16 activation rows, lane (g = lane / 16, i = lane % 16) bytes 32 g .. + 31 of row i and that row's scale byte.
 * A wave owns 128 columns n (a block of w, so its scale is one number) and 16 NU rows m. Which weight row is which row of an
 * A operand is free: rows 4 q + e of two operands are 8 adjacent columns, so that a lane holds whole 16-byte pieces of a row of
 * the result, and a row's block of 128 meets across four lanes where the epilogue needs its largest magnitude. The results go
 * through LDS once more, so that a store instruction writes four whole rows of 256 bytes.
 *
 * Operands go from memory to LDS by DMA in stages of 128 k (128 bytes a row: rows of 64 took twice as long for a byte). A row keeps
 * its 16-byte piece b at place b ^ swizzle(row), so that the 16 lanes that an LDS read serves at a time meet in different banks.
 *
 * Full tiles, 256 x 256 (two stages in LDS, one workgroup a CU): four waves, one a SIMD, of 128 x 128 results each (all 256 AGPRs of a
 * lane), which take their next operands from LDS between this stage's products. Bound by the matrix core: a stage takes 1.4 us (3,100
 * TFLOP/s over 256 CUs; a library product of 8,192^3 reaches 3,040), a tile about 4 more for its results, beside which the next
 * tile's first stage is fetched: 8,192^3 375 to 378 us (2,930 to 2,910 TFLOP/s); 65,536 x 4,992 x 1,664 441 to 447 (2,470 to 2,435);
 * 65,536 x 1,664 x 6,656 531 (2,734); the fast ReLU^2 form of 65,536 x 6,656 x 1,664 583 to 602; its backward, which moves 1.7 GB
 * besides, 811 to 835. Eight waves of 64 x 128 that took turns at the core read half as much again from LDS and took 417, 508, 611, 642 and
 * 822 us. Results leave by buffer stores, whose range takes the place of masks and 64-bit addresses (the five took 376, 453, 534, 594
 * and 852 us with those).
 * Half tiles, 128 x 128, two workgroups a CU, and small ones, 64 x 128, three stages in LDS: for results that make fewer tiles.
 * Bound by LDS, 0.5 to 0.65 and 0.35 to 0.42 us a stage: 1,001 x 5,120 x 1,280 11 us; 128 x 65,536 x 1,664 26 us (4.2 TB/s of
 * weights); 128 x 4,992 x 1,664 7.6. Rings of six stages in small tiles and of four in half tiles leave room for one workgroup a CU:
 * 256 x 4,992 x 1,664 7.7 -> 8.8 us, 1,001 x 4,992 13.4 -> 19.9.
 *
 * Rows past M and N and columns past K read zeros (offsets past the buffer resource), and are not stored.
 *
 * The instruction adds the eight products of a lane's adjacent bytes at 13 bits below the largest of them (measured: beside
 * 2^16, 2^3 is kept and 2^2 is not, of either sign; products of other eights keep theirs) and everything else in fp32: 1.5e-5
 * relative error for normal values, 3e-5 with a few channels far above the others, against the 2e-3 of a bf16 result. Before a
 * ReLU^2, whose result is rounded to 8 bits next, such an error lands on another code now and then: an MLP's result was 0.0024 to
 * 0.0037 off float64's in place of 0.0017. So those products are taken exactly, from the values in bf16: in small tiles, which have the
 * time, in half tiles, and in wide ones, 256 x 256 by eight waves of 64 x 128, which convert 1.5 times a product where half tiles do
 * 2.5 times. Bound by the matrix cores at bf16's rate and the conversions beside them: 65,536 x 6,656 x 1,664 1,087 to 1,098 us (1,320
 * TFLOP/s; by half tiles 1,240), 16,384 x 5,120 x 1,280 168 (190), 9,995 x 5,120 x 1,280 117 (121; all in wide tiles 123), 1,001 x 5,120
 * x 1,280 20 (wide 30). A caller may ask for the products by eights all the same (_fast): these four take 597, 99, 70 and 12 us then.
 */
#include "nanochat_amd.h"
#include "nc_fp8.h"
#include "nc_internal.h"

namespace nc {
namespace {

constexpr int FG_ROWB = F8_BLOCK;        /* bytes of a row of a stage: one block */
constexpr int FG_PAST = 0x7FFF0000;      /* a byte offset past every operand's range */
constexpr int FG_NT = 2;                 /* a store past the caches */

enum { FG_STORE, FG_RELU2, FG_RELU2_BWD, FG_RELU2_EXACT };

struct F8Gemm {
    const unsigned char *a, *as;         /* [M][K] codes, [M] scale bytes at as_stride */
    const unsigned char *w, *ws;         /* [N][K] codes, [ceil(N / 128)] scale bytes at ws_stride */
    long long as_stride;
    int ws_stride;
    long long M;
    int N, K;
    uint16_t *out;                       /* [M][N] bf16 (STORE, RELU2_BWD) */
    unsigned char *q, *qs;               /* [M][N] codes and their scales at qs_stride (RELU2, RELU2_BWD: written) */
    const unsigned char *act, *acts;     /* [M][N] codes and scales at act_stride (RELU2_BWD: read) */
    long long qs_stride, act_stride;
};

template <int NU_, int WN_, int WM_, int RING_> struct FgTile {
    static constexpr int NU = NU_, WN = WN_, WM = WM_, RING = RING_, WAVES = WN * WM, TM = 16 * NU * WM, TN = F8_BLOCK * WN;
    static constexpr bool FULL = NU == 8;
    static constexpr int ROWS = TM + TN, STAGE = ROWS * FG_ROWB, LOADS = ROWS / 8 / WAVES, A_LOADS = TM / 8 / WAVES;
    static_assert(TM % (8 * WAVES) == 0 && TN % (8 * WAVES) == 0, "DMA split");
};
typedef FgTile<8, 2, 2, 2> FgFull;   /* 256 x 256, 4 waves of 128 x 128, two stages in LDS */
typedef FgTile<4, 2, 4, 2> FgWide;   /* 256 x 256, 8 waves of 64 x 128: exact products alone */
typedef FgTile<2, 1, 4, 2> FgHalf;   /* 128 x 128, 4 waves */
typedef FgTile<1, 1, 4, 3> FgSmall;  /* 64 x 128, 4 waves */

/* Activation rows lie in LDS by f8_swizzle. A weight row that stands for row i = 4 q + c of an operand has the same by q (0, 3 or 1, 2)
 * and c / 2, whichever operand t it belongs to. */
/* The column (0 .. 127 of a wave's block) of row 4 q of operand t, rows on being columns on. */
__host__ __device__ constexpr int fg_column(int t, int q) { return 32 * (t / 2) + 8 * q + 4 * (t % 2); }
__device__ __forceinline__ int fg_swizzle_w(int row) {
    const int q = (row >> 3) & 3, u = ((q << 1) & 3) ^ ((q >> 1) * 3);   /* 0, 2, 3, 1 */
    return ((row >> 1) & 1) | (u << 1);
}

__device__ __forceinline__ void fg_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int I> struct FgIndex { static constexpr int value = I; };
template <int N, int I = 0, class F> __device__ __forceinline__ void fg_unroll(F &&f) {
    if constexpr (I < N) {
        f(FgIndex<I>{});
        fg_unroll<N, I + 1>(f);
    }
}

__device__ __forceinline__ i32x8 fg_operand(const unsigned char *buf, int lo, int hi) {
    const u32x4 x = *(const u32x4 *)(buf + lo), y = *(const u32x4 *)(buf + hi);
    return i32x8{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
}

/* A stage's products; BYTE: which byte of the scale dwords is its block's. EXACT: from the values in bf16, four instructions in
 * place of one (codes 8 Q .. + 7 of each lane's 32 in instruction Q). */
template <int BYTE> __device__ __forceinline__ float fg_scale(uint32_t s) { return f8_scale((s >> (8 * BYTE)) & 0xFFu); }
template <int Q> __device__ __forceinline__ bf16x8 fg_values(const i32x8 &c, float s) {
    return f8_values((uint32_t)c[2 * Q], (uint32_t)c[2 * Q + 1], s);
}
template <class P, int BYTE, bool EXACT>
__device__ __forceinline__ void fg_compute(const unsigned char *buf, f32x4 (&acc)[8][P::NU], const uint32_t (&sa)[P::NU],
                                           uint32_t sw, int a_at, int w_at) {
    i32x8 fb[P::NU];
#pragma unroll
    for (int u = 0; u < P::NU; u++) fb[u] = fg_operand(buf, a_at + u * 16 * FG_ROWB, (a_at ^ 16) + u * 16 * FG_ROWB);
    if constexpr (EXACT) {
        const float t_s = fg_scale<BYTE>(sw);
        bf16x8 b[P::NU][4];
        fg_unroll<P::NU>([&](auto u) {
            constexpr int U = decltype(u)::value;
            const float s = fg_scale<BYTE>(sa[U]);
            fg_unroll<4>([&](auto q) { b[U][decltype(q)::value] = fg_values<decltype(q)::value>(fb[U], s); });
        });
#pragma unroll
        for (int t = 0; t < 8; t++) {
            const i32x8 fa = fg_operand(buf, w_at + fg_column(t, 0) * FG_ROWB, (w_at ^ 16) + fg_column(t, 0) * FG_ROWB);
            fg_unroll<4>([&](auto q) {
                const bf16x8 v = fg_values<decltype(q)::value>(fa, t_s);
#pragma unroll
                for (int u = 0; u < P::NU; u++) acc[t][u] = mfma16x16x32(v, b[u][decltype(q)::value], acc[t][u]);
            });
        }
    } else {
#pragma unroll
        for (int t = 0; t < 8; t++) {
            const i32x8 fa = fg_operand(buf, w_at + fg_column(t, 0) * FG_ROWB, (w_at ^ 16) + fg_column(t, 0) * FG_ROWB);
#pragma unroll
            for (int u = 0; u < P::NU; u++)
                acc[t][u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fa, fb[u], acc[t][u], 0, 0, BYTE, (int)sw, BYTE,
                                                                             (int)sa[u]);
        }
    }
}

/* What a wave knows of its tile. */
struct FgPlace {
    int lane, wave, grp, i, wn, wm;
    int rows, cols;              /* of the tile that exist */
    int row0, nb;                /* the wave's first row of a (this lane's), and its block of w */
    bool some;                   /* the wave has columns */
};

template <class P>
__device__ __forceinline__ FgPlace fg_place(const F8Gemm &g, long long m0, int n0) {
    FgPlace p;
    p.lane = threadIdx.x & (WAVE - 1);
    p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    p.grp = p.lane >> 4;
    p.i = p.lane & 15;
    p.wn = p.wave % P::WN;
    p.wm = p.wave / P::WN;
    p.rows = __builtin_amdgcn_readfirstlane((int)(g.M - m0 < P::TM ? g.M - m0 : P::TM));
    p.cols = g.N - n0 < P::TN ? g.N - n0 : P::TN;
    p.row0 = 16 * P::NU * p.wm + p.i;
    p.nb = n0 / F8_BLOCK + p.wn;
    p.some = F8_BLOCK * p.wn < p.cols;
    return p;
}

/* The K walk of all but the full tile: P::RING stages in LDS, the DMA of the next RING - 1 on its way. Each wave moves 8 rows of every 32
 * (64 with eight waves), and every fourth stage the scale dwords of its own operands' next four blocks (its rows of a by lane, its block of w). */
constexpr int FG_OWN = 512;   /* bytes of a wave's scales of four stages: 64 dwords of a, then w's */
template <class P, bool EXACT>
__device__ __forceinline__ void fg_walk_ring(const F8Gemm &g, const FgPlace &p, long long m0, int n0, unsigned char *lds,
                                             f32x4 (&acc)[8][P::NU]) {
    const int stages = (g.K + F8_BLOCK - 1) / F8_BLOCK, K = g.K;
    const u32x4 ra = f8_words(g.a + m0 * K, (long long)p.rows * K), rw = f8_words(g.w + (long long)n0 * K, (long long)p.cols * K);
    /* stages past the last ask for dwords behind their rows' scales: zeros, or the next row's */
    const u32x4 rsa = f8_words(g.as + m0 * g.as_stride, f8_scale_range(p.rows, g.as_stride, stages));
    const u32x4 rsw = f8_words(g.ws + (long long)(p.some ? p.nb : 0) * g.ws_stride, f8_scale_range(1, g.ws_stride, stages));
    const uint32_t base = f8_lds(lds) + p.wave * 1024;
    unsigned char *const scales = lds + P::RING * P::STAGE + p.wave * 2 * FG_OWN;
    const uint32_t scale_to = f8_lds(scales);
    const int row = 8 * p.wave + (p.lane >> 3), first = row * K;   /* rows 32 on have the same pieces */
    const int ca = ((p.lane & 7) ^ f8_swizzle(row)) << 4, cw = ((p.lane & 7) ^ fg_swizzle_w(row)) << 4;
    const int scale_at = p.lane < 16 * P::NU ? (16 * P::NU * p.wm + p.lane) * (int)g.as_stride : FG_PAST;
    const auto fetch = [&](int j, int slot) {   /* a stage past the last: zeros, without an access */
        const int k = j * FG_ROWB;
        const int oa = k + ca < K ? first + ca + k : FG_PAST, ow = k + cw < K ? first + cw + k : FG_PAST;
        const uint32_t to = base + slot * P::STAGE;
        if ((j & 3) == 0) {
            f8_dma4(scale_to + ((j >> 2) & 1) * FG_OWN, scale_at + j, rsa);
            f8_dma4(scale_to + ((j >> 2) & 1) * FG_OWN + 256, j, rsw);
        }
        constexpr int STEP = 8 * P::WAVES;   /* rows that all waves move at a time */
#pragma unroll
        for (int s = 0; s < P::A_LOADS; s++) f8_dma16(to + STEP * FG_ROWB * s, oa + STEP * s * K, ra);
#pragma unroll
        for (int s = 0; s < P::LOADS - P::A_LOADS; s++)
            f8_dma16(to + STEP * FG_ROWB * (P::A_LOADS + s), ow + STEP * s * K, rw);
    };
#pragma unroll
    for (int j = 0; j < P::RING - 1; j++) fetch(j, j);
    const int a_at = p.row0 * FG_ROWB + (((2 * p.grp) ^ f8_swizzle(p.row0)) << 4);
    const int w_row = F8_BLOCK * p.wn + fg_column(0, p.i >> 2) + (p.i & 3);
    const int w_at = (P::TM + w_row) * FG_ROWB + (((2 * p.grp) ^ fg_swizzle_w(w_row)) << 4);
    uint32_t sa[P::NU], sw = 0;
    int slot = 0, last = P::RING - 1;
    for (int j0 = 0; j0 < stages; j0 += 4)
        fg_unroll<4>([&](auto which) {
            constexpr int BYTE = decltype(which)::value;
            const int j = j0 + BYTE;
            if (j >= stages) return;
            /* all but the RING - 2 newest stages has landed, and what this wave read of the slot filled next is in registers */
            constexpr int NEWER = (P::RING - 2) * P::LOADS + 2 * ((BYTE + P::RING - 2) / 4);
            __builtin_amdgcn_s_waitcnt((NEWER & 0xF) | ((NEWER >> 4) << 14) | (0x7 << 4) | (0x0 << 8));
            fg_barrier();
            fetch(j + P::RING - 1, last);
            if constexpr (BYTE == 0) {
                const unsigned char *own = scales + ((j >> 2) & 1) * FG_OWN;
#pragma unroll
                for (int u = 0; u < P::NU; u++) sa[u] = *(const uint32_t *)(own + 4 * (16 * u + p.i));
                sw = *(const uint32_t *)(own + 256);
            }
            fg_compute<P, BYTE, EXACT>(lds + slot * P::STAGE, acc, sa, sw, a_at, w_at);
            last = slot;
            slot = slot + 1 == P::RING ? 0 : slot + 1;
        });
    __builtin_amdgcn_s_waitcnt(0);
    fg_barrier();   /* the epilogue writes where other waves may still read and DMA may still land */
}

/* The products as inline assembly: accumulators that stay in the same four AGPRs for the whole walk ("+a"; all 256 of a wave, one a
 * SIMD), where the compiler moved them about. It does not see matrix instructions there and inserts none of their wait states; they
 * are kept by construction: operands and scales are written by LDS reads alone, a quarter of a stage ahead; an accumulator is used
 * again 63 products later, and read only 32 wait states after the last product. */
__device__ __forceinline__ void fg_mfma(f32x4 &c, const i32x8 &w, const i32x8 &a, uint32_t sw, uint32_t sa) {
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]"
                 : "+a"(c) : "v"(w), "v"(a), "v"(sw), "v"(sa));
}

/* ... and from nothing: a tile's first stage needs no cleared accumulators. */
__device__ __forceinline__ void fg_mfma_new(f32x4 &c, const i32x8 &w, const i32x8 &a, uint32_t sw, uint32_t sa) {
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, 0, %3, %4 op_sel_hi:[0,0,0]"
                 : "=a"(c) : "v"(w), "v"(a), "v"(sw), "v"(sa));
}

/* The full tile's DMA: instruction s = 0 .. 7 of w and of a moves rows 32 s + 8 wave + lane / 8; every fourth stage three more bring the
 * scale dwords of four blocks that the wave itself needs (its 128 rows of a, its block of w). */
constexpr int FG_SCALES = 768;    /* bytes of a wave's scales of four blocks: 128 dwords of a, then w's in each lane's place */
struct FgDma {
    u32x4 ra, rw, rsa, rsw;
    uint32_t lds, scales;         /* this wave's addresses in stage buffer 0 and of its first scales */
    int ca, cw, first, K;         /* the lane's pieces and its row of s = 0 */
    int scale_at, more;           /* the offset of its row's scales, and of 64 rows */
    uint32_t oa, ow, to;          /* the stage being fetched */
    int flip;                     /* the buffer of even stages */
    __device__ __forceinline__ FgDma(const F8Gemm &g, const FgPlace &p, long long m0, int n0, unsigned char *b0, int flip)
        : flip(flip) {
        ra = f8_words(g.a + m0 * g.K, (long long)p.rows * g.K);
        rw = f8_words(g.w + (long long)n0 * g.K, (long long)p.cols * g.K);
        const int stages = (g.K + F8_BLOCK - 1) / F8_BLOCK;
        rsa = f8_words(g.as + m0 * g.as_stride, f8_scale_range(p.rows, g.as_stride, stages));
        rsw = f8_words(g.ws + (long long)(p.some ? p.nb : 0) * g.ws_stride, f8_scale_range(1, g.ws_stride, stages));
        scale_at = (128 * p.wm + p.lane) * (int)g.as_stride;
        more = 64 * (int)g.as_stride;
        lds = f8_lds(b0) + p.wave * 1024;
        scales = f8_lds(b0) + 2 * FgFull::STAGE + p.wave * 2 * FG_SCALES;
        K = g.K;
        const int row = 8 * p.wave + (p.lane >> 3), pos = p.lane & 7;
        first = row * K;
        ca = (pos ^ f8_swizzle(row)) << 4;
        cw = (pos ^ fg_swizzle_w(row)) << 4;   /* rows 32 on have the same */
    }
    /* Stage j's offsets, and its scales' DMA where it is the first of four. Past K they lie past the range, also with 224 K added. */
    __device__ __forceinline__ void stage(int j) {
        const int k = j * FG_ROWB;
        oa = k + ca < K ? first + ca + k : FG_PAST;
        ow = k + cw < K ? first + cw + k : FG_PAST;
        to = lds + ((j & 1) ^ flip) * FgFull::STAGE;
        if ((j & 3) == 0) {
            const uint32_t own = scales + ((j >> 2) & 1) * FG_SCALES;
            f8_dma4(own, scale_at + j, rsa);
            f8_dma4(own + 256, scale_at + more + j, rsa);
            f8_dma4(own + 512, j, rsw);
        }
    }
    /* in order of S */
    template <int S> __device__ __forceinline__ void issue_w() { f8_dma16_on<FgFull::TM * FG_ROWB + S * 4096>(to, ow, 32 * K, rw); }
    template <int S> __device__ __forceinline__ void issue_a() { f8_dma16_on<S * 4096>(to, oa, 32 * K, ra); }
    __device__ __forceinline__ void fetch(int j) {
        stage(j);
        fg_unroll<8>([&](auto s) { issue_w<decltype(s)::value>(); });
        fg_unroll<8>([&](auto s) { issue_a<decltype(s)::value>(); });
    }
};

/* RELU2_BWD: a wave's 128 x 128 codes of a, which come as a stage behind the last, into the buffer that is free by then: 8 rows an
 * instruction, their places fg_code_place's. From memory behind the walk they took 4 us more a tile (65,536 x 6,656 x 1,664 861 us
 * -> 829). */
struct FgAct {
    u32x4 r;
    uint32_t at, to;
    int N;
    __device__ __forceinline__ FgAct(const F8Gemm &g, const FgPlace &p, long long m0, int n0, const unsigned char *buffer) {
        r = f8_words(g.act + m0 * g.N + n0, (long long)p.rows * g.N - n0);
        const int row = p.lane >> 3, col = F8_BLOCK * p.wn + 16 * ((p.lane & 7) ^ row);
        N = g.N;
        at = col < p.cols ? (uint32_t)((128 * p.wm + row) * N + col) : (uint32_t)FG_PAST;   /* also with 120 N added */
        to = f8_lds(buffer) + p.wave * 16384;
    }
    template <int S> __device__ __forceinline__ void issue() const { f8_dma16(to + S * 1024, at + 8 * S * N, r); }
};

/* All but the N newest DMA have landed, and this wave's LDS reads are done. */
template <int N> __device__ __forceinline__ void fg_wait() {
    __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4) | (0x0 << 8));
}

/*
 * The K walk of the full tile: a wave a SIMD, its 64 products of a stage in four quarters of 16, each of four of w's eight operands
 * with four of a's: (w low, first of a), (low, second), (high, second), (high, first); what is "first" changes from stage to stage.
 * So half of w's registers are free from the middle of a stage on and half of a's for its last quarter, and take the next stage's
 * operands there; the other halves come in the next stage's first half. A stage's buffer has been read by the middle of the stage:
 * the DMA of the stage after next goes there, w's part in the third quarter, a's in the fourth. Two barriers a stage: in the middle
 * (everyone has read w of this buffer; w of the next stage has landed) and before the last quarter (a of the next stage has).
 */
struct FgWalk {
    const unsigned char *lds, *own;       /* the workgroup's LDS, this wave's scales */
    int a_at, w_at, i, flip;
    i32x8 w[8], a[8];
    uint32_t sa[2][8], sw[2];             /* scale bytes of even and of odd stages */
    template <int T> __device__ __forceinline__ void read_w(const unsigned char *buf) {
        w[T] = fg_operand(buf, w_at + fg_column(T, 0) * FG_ROWB, (w_at ^ 16) + fg_column(T, 0) * FG_ROWB);
    }
    template <int U> __device__ __forceinline__ void read_a(const unsigned char *buf) {
        a[U] = fg_operand(buf, a_at + U * 16 * FG_ROWB, (a_at ^ 16) + U * 16 * FG_ROWB);
    }
    template <int U, int ODD> __device__ __forceinline__ void read_scale(int j) {   /* of stage j; U = 8: w's */
        const unsigned char *sc = own + ((j >> 2) & 1) * FG_SCALES + (j & 3);
        if constexpr (U == 8) sw[ODD] = sc[512];
        else sa[ODD][U] = sc[(16 * U + i) * 4];
    }
    /* The bytes as whole registers from their reads on: else the compiler clears their upper bits right before the products. */
    template <int ODD> __device__ __forceinline__ void pin() {
#pragma unroll
        for (int u = 0; u < 8; u++) asm volatile("" : "+v"(sa[ODD][u]));
        asm volatile("" : "+v"(sw[ODD]));
    }
    /* What is done behind product I: of stage j, FIRST (its parity) which half of a comes first. act_next: the
     * DMA is not of stage j + 2 but of act. */
    template <int I, int FIRST> __device__ __forceinline__ void side(int j, FgDma &dma, bool act_next, const FgAct *act) {
        const unsigned char *cur = lds + ((j & 1) ^ flip) * FgFull::STAGE, *next = lds + ((j & 1) ^ flip ^ 1) * FgFull::STAGE;
        if constexpr (I < 8 && I % 2 == 1) read_a<4 * (1 - FIRST) + I / 2>(cur);
        if constexpr (I >= 8 && I < 24 && I % 4 == 1) read_w<4 + (I - 8) / 4>(cur);
        if constexpr (I >= 32 && I < 40 && I % 2 == 1) read_w<(I - 32) / 2>(next);
        if constexpr (I >= 48 && I < 56 && I % 2 == 1) read_a<4 * (1 - FIRST) + (I - 48) / 2>(next);
        if constexpr (I >= 56 && I < 62 && I % 2 == 1) {
            read_scale<3 * ((I - 56) / 2), 1 - FIRST>(j + 1);
            read_scale<3 * ((I - 56) / 2) + 1, 1 - FIRST>(j + 1);
            read_scale<3 * ((I - 56) / 2) + 2, 1 - FIRST>(j + 1);
        }
        if constexpr (I == 63) pin<1 - FIRST>();
        if constexpr (I >= 32 && I % 2 == 0) {
            constexpr int S = (I - 32) / 2;   /* 0 .. 7 w, 8 .. 15 a */
            if (act_next) act->template issue<S>();
            else if constexpr (S < 8) dma.template issue_w<S>();
            else dma.template issue_a<S - 8>();
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    template <int I, int FIRST, bool NEW = false>
    __device__ __forceinline__ void run(f32x4 (&acc)[8][8], int j, FgDma &dma, bool act_next, const FgAct *act) {
        if constexpr (I < 64) {
            constexpr int Q = I / 16, T = 4 * (Q / 2) + I % 16 / 4, U = 4 * ((Q == 0 || Q == 3) ? FIRST : 1 - FIRST) + I % 4;
            if constexpr (I == 32) {
                fg_wait<8>();       /* w of stage j + 1; a's eight are newer */
                fg_barrier();
                dma.stage(j + 2);
            }
            if constexpr (I == 48) {
                if ((j & 3) == 2) fg_wait<11>();   /* a of stage j + 1; w of stage j + 2 is newer, its scales too where it brought any */
                else fg_wait<8>();
                fg_barrier();
            }
            if constexpr (NEW) fg_mfma_new(acc[T][U], w[T], a[U], sw[FIRST], sa[FIRST][U]);
            else fg_mfma(acc[T][U], w[T], a[U], sw[FIRST], sa[FIRST][U]);
            side<I, FIRST>(j, dma, act_next, act);
            run<I + 1, FIRST, NEW>(acc, j, dma, act_next, act);
        }
    }
};

/* Stage 0 is on its way, and NEWER memory instructions behind it. */
template <bool ACT, int NEWER>
__device__ __forceinline__ void fg_walk_full(const F8Gemm &g, const FgPlace &p, long long m0, int n0, unsigned char *lds, FgDma &dma,
                                             bool newer, f32x4 (&acc)[8][8]) {
    const int stages = (g.K + F8_BLOCK - 1) / F8_BLOCK;
    const FgAct act(ACT ? g : F8Gemm{}, p, ACT ? m0 : 0, ACT ? n0 : 0, lds + ((stages & 1) ^ dma.flip) * FgFull::STAGE);
    if (ACT && stages == 1) fg_unroll<16>([&](auto s) { act.template issue<decltype(s)::value>(); });
    else dma.fetch(1);
    FgWalk k;
    k.lds = lds;
    k.own = lds + 2 * FgFull::STAGE + p.wave * 2 * FG_SCALES;
    k.i = p.i;
    k.flip = dma.flip;
    k.a_at = p.row0 * FG_ROWB + (((2 * p.grp) ^ f8_swizzle(p.row0)) << 4);
    const int w_row = F8_BLOCK * p.wn + fg_column(0, p.i >> 2) + (p.i & 3);
    k.w_at = (FgFull::TM + w_row) * FG_ROWB + (((2 * p.grp) ^ fg_swizzle_w(w_row)) << 4);
    if (newer) fg_wait<16 + NEWER>();
    else fg_wait<16>();
    fg_barrier();
    const unsigned char *b0 = lds + dma.flip * FgFull::STAGE;
    fg_unroll<4>([&](auto t) {
        k.template read_w<decltype(t)::value>(b0);
        k.template read_a<decltype(t)::value>(b0);
    });
    fg_unroll<9>([&](auto u) { k.template read_scale<decltype(u)::value, 0>(0); });
    k.template pin<0>();
    k.template run<0, 0, true>(acc, 0, dma, ACT && stages == 2, &act);
    for (int j = 1; j < stages; j += 2) {
        k.template run<0, 1>(acc, j, dma, ACT && j + 2 == stages, &act);
        if (j + 1 >= stages) break;
        k.template run<0, 0>(acc, j + 1, dma, ACT && j + 3 == stages, &act);
    }
    __builtin_amdgcn_s_waitcnt(0);
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");   /* 32 wait states; no read moves above */
    fg_barrier();   /* what follows writes where other waves may still read and DMA may still land */
#pragma unroll
    for (int t = 0; t < 8; t++)
#pragma unroll
        for (int u = 0; u < 8; u++) asm volatile("" : "+a"(acc[t][u]));
}

/* A wave's parts of LDS behind its walk, two in turn: 16 rows of 256 bytes, then 16 of 128. */
constexpr int FG_TURN = 16 * 384;
__device__ __forceinline__ int fg_code_place(int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }
/* Lanes of one wave exchange values through LDS, which serves a wave's accesses in order; the compiler keeps the order too. */
__device__ __forceinline__ void fg_wave_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

/* An offset moves on, here and now: the compiler would keep every sum of them in a register of its own. */
__device__ __forceinline__ void fg_on(uint32_t &at, uint32_t by) { asm volatile("v_add_u32 %0, %1, %0" : "+v"(at) : "s"(by)); }

/* A wave's results. turns: the workgroup's part of LDS for them; acts, act_bytes: ACT_STAGE's codes of a, in LDS, and the scale bytes
 * of the wave's rows `lane` and 64 on. */
template <class P, int EPI>
__device__ __forceinline__ void fg_results(const F8Gemm &g, const FgPlace &p, long long m0, int n0, f32x4 (&acc)[8][P::NU],
                                           unsigned char *turns, const unsigned char *acts, const uint32_t (&act_bytes)[2]) {
    constexpr bool ACT_STAGE = P::FULL && EPI == FG_RELU2_BWD;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));   /* made again, not kept through the walk */
    const int grp = (tid & (WAVE - 1)) >> 4;
    const int rows = p.rows, cols = p.cols, nb = p.nb, wn = p.wn;
    if (!p.some) return;
    const int lane = tid & (WAVE - 1), rows_left = rows - 16 * P::NU * p.wm, col = F8_BLOCK * wn;   /* this wave's */
    const long long first = m0 + 16 * P::NU * p.wm;
    unsigned char *mine = turns + (threadIdx.x >> 6) * FG_TURN;
    const unsigned char *act_at = acts + (threadIdx.x >> 6) * 16384;
    const int r16 = lane & 15;
    /* RELU2_BWD: a's scales, and in the smaller tiles its codes, a piece of 16 columns a lane of rows 8 k + lane / 8 of each 16; all on
     * their way at once */
    u32x4 act[P::NU][2];
    uint32_t act_byte[P::NU];
    if constexpr (ACT_STAGE) {
#pragma unroll
        for (int u = 0; u < P::NU; u++) act_byte[u] = __shfl(act_bytes[u / 4], 16 * (u % 4) + r16);
    } else if constexpr (EPI == FG_RELU2_BWD) {
#pragma unroll
        for (int u = 0; u < P::NU; u++) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int r = 16 * u + 8 * k + (lane >> 3), c = col + 16 * (lane & 7);
                act[u][k] = r < rows_left && c < cols ? *(const u32x4 *)(g.act + (first + r) * g.N + n0 + c) : u32x4{0, 0, 0, 0};
            }
            const int r = 16 * u + r16;
            act_byte[u] = r < rows_left ? g.acts[(first + r) * g.act_stride + nb] : 127u;
        }
    }
    /* Stores by way of a buffer's range: rows past the last fall behind it, columns past the last have offsets behind it. So each is an
     * addition and a store, without masks, and all of them are issued. */
    const auto rsrc = [&](void *base, long long row_bytes) {
        return f8_rsrc((unsigned char *)base + m0 * row_bytes, rows * row_bytes);
    };
    const uint32_t top = (uint32_t)(16 * P::NU * p.wm);   /* the wave's first row */
    __amdgpu_buffer_rsrc_t r_out, r_q, r_qs;
    uint32_t out_at = 0, q_at = 0, qs_at = 0;
    if constexpr (EPI != FG_RELU2) {
        r_out = rsrc(g.out, 2LL * g.N);
        const int c = col + 8 * (lane & 15);
        out_at = c < cols ? ((top + (lane >> 4)) * (uint32_t)g.N + n0 + c) * 2u : (uint32_t)FG_PAST;
    }
    if constexpr (EPI != FG_STORE) {
        r_q = rsrc(g.q, g.N);
        r_qs = rsrc(g.qs, g.qs_stride);
        const int c = col + 16 * (lane & 7);
        q_at = c < cols ? (top + (lane >> 3)) * (uint32_t)g.N + n0 + c : (uint32_t)FG_PAST;
        qs_at = grp == 0 ? (top + r16) * (uint32_t)g.qs_stride + nb : (uint32_t)FG_PAST;
    }
    /* Rows 16 u + r16: this lane's results, columns 32 h + 8 grp + 0 .. 7, into the wave's turn buffer u % 2 */
    u32x2 c_next[4];   /* ACT_STAGE: a's codes of the rows after next */
    const auto read_act = [&](int u) {
#pragma unroll
        for (int h = 0; h < 4; h++)
            c_next[h] = *(const u32x2 *)(act_at + u * 16 * 128 + fg_code_place(r16, 2 * h + (grp >> 1)) + 8 * (grp & 1));
    };
    if constexpr (ACT_STAGE) read_act(0);
    const auto make = [&](int u) {
        unsigned char *const turn = mine + u % 2 * P::WAVES * FG_TURN, *const codes = turn + 16 * 256;
        float v[32];
#pragma unroll
        for (int t = 0; t < 8; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[4 * t + e] = acc[t][u][e];
        u32x2 q[4];
        uint32_t o[16];
        if constexpr (EPI == FG_RELU2) {
            uint32_t m = 0u;
#pragma unroll
            for (int k = 0; k < 32; k++) {
                const float x = __builtin_elementwise_maximum(v[k], 0.0f);   /* a NaN stays one */
                v[k] = x * x;
                const uint32_t b = __float_as_uint(v[k]);                     /* no sign but a NaN's, which is above all */
                m = m > b ? m : b;
            }
            const uint32_t byte = f8_scale_byte(group_max(m));
            const float s = f8_scale(byte);
#pragma unroll
            for (int h = 0; h < 4; h++)
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const int z = 8 * h + 4 * k;
                    q[h][k] = byte == F8_NAN_BYTE ? F8_NAN_CODES : f8_codes(v[z], v[z + 1], v[z + 2], v[z + 3], s);
                }
            __builtin_amdgcn_raw_buffer_store_b8((unsigned char)byte, r_qs, qs_at, 0, 0);
            fg_on(qs_at, 16u * (uint32_t)g.qs_stride);
        } else if constexpr (EPI == FG_RELU2_BWD) {
            /* dh = da 2 sqrt(a) */
            u32x2 c[4];
            if constexpr (ACT_STAGE) {
#pragma unroll
                for (int h = 0; h < 4; h++) c[h] = c_next[h];
                if (u + 1 < P::NU) read_act(u + 1);
            } else {
                fg_wave_order();
#pragma unroll
                for (int k = 0; k < 2; k++) *(u32x4 *)(codes + fg_code_place(8 * k + (lane >> 3), lane & 7)) = act[u][k];
                fg_wave_order();
#pragma unroll
                for (int h = 0; h < 4; h++)
                    c[h] = *(const u32x2 *)(codes + fg_code_place(r16, 2 * h + (grp >> 1)) + 8 * (grp & 1));
            }
            /* 2 sqrt(a) = sqrt(4 a). Where 4 a may leave fp32's normal range (which v_sqrt_f32 takes for 0, or is infinite) it is
             * taken times 2^32 or 2^-32, and the sum times the inverse of the root of that. */
            const bool low = act_byte[u] < 16u, high = act_byte[u] >= 240u;
            const float s = 4.0f * (f8_scale(act_byte[u]) * (low ? 0x1p32f : high ? 0x1p-32f : 1.0f));
            if (__any(low || high)) {
                const float p = low ? 0x1p-16f : high ? 0x1p16f : 1.0f;
#pragma unroll
                for (int k = 0; k < 32; k++) v[k] = v[k] * p;
            }
            float m = 0.0f;   /* the largest before its rounding, which keeps the order */
#pragma unroll
            for (int h = 0; h < 4; h++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const auto a = (k & 1) ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[h][k >> 1], s, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[h][k >> 1], s, false);
                    /* v_sqrt_f32 is within an ulp; the result is rounded to bf16 right away */
                    const float x = v[8 * h + 2 * k] * __builtin_amdgcn_sqrtf(a[0]);
                    const float y = v[8 * h + 2 * k + 1] * __builtin_amdgcn_sqrtf(a[1]);
                    o[4 * h + k] = bf16_pair(x, y);
                    m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(__builtin_fabsf(x), __builtin_fabsf(y)), m);
                }
            const uint32_t byte = f8_scale_byte(group_max((bf16_pair(m, m) & 0x7FFFu) << 16));
            const float qs = f8_scale(byte);
#pragma unroll
            for (int h = 0; h < 4; h++)
                q[h] = byte == F8_NAN_BYTE ? u32x2{F8_NAN_CODES, F8_NAN_CODES}
                                           : u32x2{f8_codes(o[4 * h], o[4 * h + 1], qs), f8_codes(o[4 * h + 2], o[4 * h + 3], qs)};
            __builtin_amdgcn_raw_buffer_store_b8((unsigned char)byte, r_qs, qs_at, 0, 0);
            fg_on(qs_at, 16u * (uint32_t)g.qs_stride);
        } else {
#pragma unroll
            for (int k = 0; k < 16; k++) o[k] = bf16_pair(v[2 * k], v[2 * k + 1]);
        }
        fg_wave_order();
        if constexpr (EPI != FG_RELU2) {
#pragma unroll
            for (int h = 0; h < 4; h++)
                *(u32x4 *)(turn + r16 * 256 + (((4 * h + grp) ^ r16) << 4)) =
                    u32x4{o[4 * h], o[4 * h + 1], o[4 * h + 2], o[4 * h + 3]};
        }
        if constexpr (EPI != FG_STORE) {
#pragma unroll
            for (int h = 0; h < 4; h++) *(u32x2 *)(codes + fg_code_place(r16, 2 * h + (grp >> 1)) + 8 * (grp & 1)) = q[h];
        }
        fg_wave_order();
    };
    /* ... and from there whole rows to memory */
    const auto send = [&](int u) {
        const unsigned char *const turn = mine + u % 2 * P::WAVES * FG_TURN, *const codes = turn + 16 * 256;
        if constexpr (EPI != FG_RELU2) {
#pragma unroll
            for (int k = 0; k < 4; k++) {   /* four rows an instruction, past the caches: larger than they are, and read much later */
                const int r = 4 * k + (lane >> 4), c = lane & 15;
                const u32x4 d = *(const u32x4 *)(turn + r * 256 + ((c ^ r) << 4));
                __builtin_amdgcn_raw_buffer_store_b128(d, r_out, out_at, 0, FG_NT);
                fg_on(out_at, 8u * g.N);   /* four rows */
            }
        }
        if constexpr (EPI != FG_STORE) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int r = 8 * k + (lane >> 3), c = lane & 7;
                const u32x4 d = *(const u32x4 *)(codes + fg_code_place(r, c));
                /* through the caches: the next product reads them (an MLP of 9,995 x 1,280/5,120 170 us past them, 157; the training of
                 * 65,536 x 1,664/6,656, whose 436 MB do not fit, 5,108 and 5,170) */
                __builtin_amdgcn_raw_buffer_store_b128(d, r_q, q_at, 0, 0);
                fg_on(q_at, 8u * g.N);
            }
        }
    };
    make(0);
#pragma unroll
    for (int u = 1; u < P::NU; u++) {   /* the next rows are made while these are on their way through LDS */
        make(u);
        send(u - 1);
    }
    send(P::NU - 1);
}

/* The order workgroups take tiles in. Workgroup L runs on XCD L % 8, each with its own L2: XCD k gets a contiguous run of the
 * tiles, numbered in bands of 4 m-tiles walked m first, so that what an XCD runs at once shares operand tiles. */
__device__ __forceinline__ int2 fg_tile(int l, int count, int nx) {
    const int k = l % 8, r = l / 8, per = count / 8, extra = count % 8;
    const int id = k * per + min(k, extra) + r, band = 4 * nx, y0 = id / band * 4, ny = count / nx - y0;
    const int tall = ny < 4 ? ny : 4, in = id - id / band * band;
    return int2{in / tall, y0 + in % tall};
}

template <class P, int EPI> __device__ __forceinline__ void fg_run(const F8Gemm &g, unsigned char *lds) {
    const int2 t = fg_tile(blockIdx.x, gridDim.x, (g.N + P::TN - 1) / P::TN);
    const long long m0 = (long long)t.y * P::TM;
    const FgPlace p = fg_place<P>(g, m0, t.x * P::TN);
    f32x4 acc[8][P::NU];
#pragma unroll
    for (int t = 0; t < 8; t++)
#pragma unroll
        for (int u = 0; u < P::NU; u++) acc[t][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    fg_walk_ring<P, EPI == FG_RELU2_EXACT || (P::NU == 1 && EPI == FG_RELU2)>(g, p, m0, t.x * P::TN, lds, acc);
    const uint32_t none[2] = {0u, 0u};
    fg_results<P, EPI == FG_RELU2_EXACT ? FG_RELU2 : EPI>(g, p, m0, t.x * P::TN, acc, lds, lds, none);
}

/* The kernel's arguments with the codes' places read anew: kept over the walk they are four scalar registers too many. */
__device__ __forceinline__ F8Gemm fg_again(F8Gemm g) {
    typedef __attribute__((address_space(4))) const F8Gemm Args;
    Args *at = (Args *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    g.q = at->q;
    g.qs = at->qs;
    return g;
}

/* Full tiles: a workgroup a CU takes every gridDim.x-th of them, and the first stage of the next is fetched while the last one's results
 * are written (into the buffer that they do not pass through). RELU2_BWD has a's codes in that buffer: a workgroup a tile. */
template <int EPI> __device__ __forceinline__ void fg_run_full(const F8Gemm &g, int tiles, unsigned char *lds) {
    constexpr bool ACT_STAGE = EPI == FG_RELU2_BWD;
    constexpr int STORES = EPI == FG_STORE ? 32 : 24;   /* of a whole tile, a wave's instructions: 4 a 16 rows, or 2 and a scale's */
    typedef FgFull P;
    const int nx = (g.N + P::TN - 1) / P::TN, stages = (g.K + F8_BLOCK - 1) / F8_BLOCK;
    int2 t = fg_tile(blockIdx.x, tiles, nx);
    FgPlace p = fg_place<P>(g, (long long)t.y * P::TM, t.x * P::TN);
    FgDma dma(g, p, (long long)t.y * P::TM, t.x * P::TN, lds, 0);
    dma.fetch(0);
    bool stores = false;
    for (int l = blockIdx.x;;) {
        const long long m0 = (long long)t.y * P::TM;
        const int n0 = t.x * P::TN;
        uint32_t act_bytes[2] = {127u, 127u};
        if constexpr (ACT_STAGE) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int row = 128 * p.wm + 64 * h + p.lane;
                if (row < p.rows && p.some) act_bytes[h] = g.acts[(m0 + row) * g.act_stride + p.nb];
            }
        }
        f32x4 acc[8][8];
        fg_walk_full<ACT_STAGE, STORES>(g, p, m0, n0, lds, dma, stores, acc);
        const int flip = (stages & 1) ^ dma.flip;   /* the buffer of a stage behind the last */
        const FgPlace done = p;
        l += gridDim.x;
        const bool more = !ACT_STAGE && l < tiles;
        if (more) {
            t = fg_tile(l, tiles, nx);
            p = fg_place<P>(g, (long long)t.y * P::TM, t.x * P::TN);
            dma = FgDma(g, p, (long long)t.y * P::TM, t.x * P::TN, lds, flip);
            dma.fetch(0);
        }
        fg_results<P, EPI>(fg_again(g), done, m0, n0, acc, lds + (flip ^ 1) * P::STAGE, lds + flip * P::STAGE, act_bytes);
        if (!more) return;
        stores = done.some;   /* then all were issued */
        __builtin_amdgcn_s_waitcnt(0xC07F);   /* the LDS reads */
        fg_barrier();
    }
}

template <class P, int EPI>
__global__ void __launch_bounds__(P::WAVES *WAVE, P::FULL ? 1 : 2) fp8_gemm_kernel(F8Gemm g, int tiles) {
    __shared__ __align__(16) unsigned char lds[P::RING * P::STAGE + P::WAVES * 2 * (P::FULL ? FG_SCALES : FG_OWN)];
    if constexpr (P::FULL) fg_run_full<EPI>(g, tiles, lds);
    else fg_run<P, EPI>(g, lds);
}

template <class P>
int fg_launch(const F8Gemm &g, int epi, hipStream_t stream) {
    const long long tiles = (g.M + P::TM - 1) / P::TM * ((g.N + P::TN - 1) / P::TN);
    if (tiles >= (1LL << 31)) return NC_ERR_SHAPE;
    void (*kernel)(F8Gemm, int) = nullptr;
    if constexpr (P::NU == 4)
        kernel = fp8_gemm_kernel<P, FG_RELU2_EXACT>;
    else
        kernel = epi == FG_STORE ? fp8_gemm_kernel<P, FG_STORE>
                 : epi == FG_RELU2 ? fp8_gemm_kernel<P, FG_RELU2> : fp8_gemm_kernel<P, FG_RELU2_BWD>;
    if constexpr (P::NU == 2)
        if (epi == FG_RELU2_EXACT) kernel = fp8_gemm_kernel<P, FG_RELU2_EXACT>;
    const long long cus = device_cus(), grid = P::FULL && epi != FG_RELU2_BWD && tiles > cus ? cus : tiles;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(P::WAVES * WAVE), 0, stream, g, (int)tiles);
    return (int)hipGetLastError();
}

/* Sizes first, then pointers, then their alignment. */
int fg_check(const F8Gemm &g, int epi) {
    if (epi == FG_RELU2_EXACT) epi = FG_RELU2;
    if (g.M < 0 || g.M > (1LL << 31) || g.N <= 0 || g.K <= 0 || g.N % 16 || g.K % 16 || g.N > (1 << 20) || g.K > (1 << 20))
        return NC_ERR_SHAPE;
    if (g.M == 0) return NC_OK;
    if (!g.a || !g.as || !g.w || !g.ws || (epi != FG_RELU2 && !g.out) || (epi != FG_STORE && (!g.q || !g.qs)) ||
        (epi == FG_RELU2_BWD && (!g.act || !g.acts)))
        return NC_ERR_NULL;
    if (f8_misaligned(g.a, 16) || f8_misaligned(g.w, 16) || f8_misaligned(g.out, 16) || f8_misaligned(g.q, 16) || f8_misaligned(g.act, 16) ||
        f8_bad_scales(g.as, g.as_stride, g.K) || f8_bad_scales(g.ws, g.ws_stride, g.K) ||
        (epi != FG_STORE && f8_bad_scales(g.qs, g.qs_stride, g.N)) ||
        (epi == FG_RELU2_BWD && f8_bad_scales(g.acts, g.act_stride, g.N)))
        return NC_ERR_SHAPE;
    return NC_OK;
}

/* The first rows of g, or those behind them. */
F8Gemm fg_rows(F8Gemm g, long long from, long long count) {
    g.a += from * g.K;
    g.as += from * g.as_stride;
    if (g.out) g.out += from * g.N;
    if (g.q) g.q += from * g.N, g.qs += from * g.qs_stride;
    if (g.act) g.act += from * g.N, g.acts += from * g.act_stride;
    g.M = count;
    return g;
}

/*
 * Small tiles while they all run at once; else by rounds, of a full tile a CU (8 parts of time), of two half tiles a CU (5; one alone
 * 4), or whole rounds of full tiles and half tiles for the rows left, a launch more (1). Microseconds of full and half tiles of 1,664 k:
 * 515 x 16,384 21.0, 24.5; 300 x 16,384 20.4, 14.1; 200 x 65,536 29.3, 37.4; 128 x 65,536 28.1, 25.5; 2,500 x 4,992 20.7, 25.4;
 * 1,001 x 4,992 20.2, 14.1; alone and split, 9,995 x 5,120 x 1,280 73.7, 66.5; 1,500 x 16,384 45.0, 40.6. Of small and half: 256 x
 * 4,992 8.0, 11.0; 128 x 16,384 8.6, 11.8; 515 x 4,992, 351 small ones, 11.6, 11.5; 300 x 16,384, 640, 18.6, 14.1. Before a ReLU^2 wide
 * tiles take the full ones' place: 41 us to a pair of halves' 24 (1,664 k), much the same proportion; alone and split, 5,000 x 6,656
 * 105, 102. Full and half tiles sum in the same order, wide, half and small ones of exact products do too; few results
 * (fp8_skinny.hip) are summed in parts of k.
 */
int fg_whole(const F8Gemm &g, int epi, hipStream_t s) {
    return epi == FG_RELU2_EXACT ? fg_launch<FgWide>(g, epi, s) : fg_launch<FgFull>(g, epi, s);
}
long long fg_half_time(long long tiles, long long cus) { return tiles <= cus ? 4 : 5 * ((tiles + 2 * cus - 1) / (2 * cus)); }
int fg_gemm(const F8Gemm &g, int epi, void *stream) {
    const int e = fg_check(g, epi);
    if (e != NC_OK || g.M == 0) return e;
    const hipStream_t s = (hipStream_t)stream;
    const long long cus = device_cus(), nx = (g.N + 255) / 256, full = (g.M + 255) / 256 * nx, half_nx = (g.N + 127) / 128;
    const long long small = (g.M + 63) / 64 * half_nx;
    if (epi == FG_STORE && fp8_some_takes(g.M, g.N, g.K, cus))
        return fp8_some(g.a, g.as, g.as_stride, g.w, g.ws, g.ws_stride, (int)g.M, g.N, g.K, g.out, s);
    if (small <= cus) return fg_launch<FgSmall>(g, epi == FG_RELU2_EXACT ? FG_RELU2 : epi, s);
    const long long full_time = 8 * ((full + cus - 1) / cus), half_time = fg_half_time((g.M + 127) / 128 * half_nx, cus);
    const long long rounds = full / cus, top = rounds * cus / nx * 256;   /* rows of whole rounds: less than M, or all are whole */
    if (top > 0 && top < g.M) {
        const long long split = 8 * rounds + fg_half_time((g.M - top + 127) / 128 * half_nx, cus) + 1;
        if (split < full_time && split < half_time) {
            const int status = fg_whole(fg_rows(g, 0, top), epi, s);
            return status ? status : fg_launch<FgHalf>(fg_rows(g, top, g.M - top), epi, s);
        }
    }
    return full_time <= half_time ? fg_whole(g, epi, s) : fg_launch<FgHalf>(g, epi, s);
}

}  // namespace
}  // namespace nc

using namespace nc;

extern "C" int nc_fp8_matmul(const void *a, const void *a_scale, long long a_scale_stride, const void *w, const void *w_scale,
                             int w_scale_stride, long long rows, int n, int k, void *out, void *stream) {
    const F8Gemm g = {(const unsigned char *)a, (const unsigned char *)a_scale, (const unsigned char *)w,
                      (const unsigned char *)w_scale, a_scale_stride, w_scale_stride, rows, n, k, (uint16_t *)out,
                      nullptr, nullptr, nullptr, nullptr, 0, 0};
    return fg_gemm(g, FG_STORE, stream);
}

extern "C" int nc_fp8_matmul_relu2_fast(const void *a, const void *a_scale, long long a_scale_stride, const void *w,
                                   const void *w_scale, int w_scale_stride, long long rows, int n, int k, void *codes,
                                   void *scale, long long scale_stride, void *stream) {
    const F8Gemm g = {(const unsigned char *)a, (const unsigned char *)a_scale, (const unsigned char *)w,
                      (const unsigned char *)w_scale, a_scale_stride, w_scale_stride, rows, n, k, nullptr,
                      (unsigned char *)codes, (unsigned char *)scale, nullptr, nullptr, scale_stride, 0};
    return fg_gemm(g, FG_RELU2, stream);
}

extern "C" int nc_fp8_matmul_relu2(const void *a, const void *a_scale, long long a_scale_stride, const void *w,
                                         const void *w_scale, int w_scale_stride, long long rows, int n, int k, void *codes,
                                         void *scale, long long scale_stride, void *stream) {
    const F8Gemm g = {(const unsigned char *)a, (const unsigned char *)a_scale, (const unsigned char *)w,
                      (const unsigned char *)w_scale, a_scale_stride, w_scale_stride, rows, n, k, nullptr,
                      (unsigned char *)codes, (unsigned char *)scale, nullptr, nullptr, scale_stride, 0};
    return fg_gemm(g, FG_RELU2_EXACT, stream);
}

extern "C" int nc_fp8_matmul_relu2_bwd(const void *a, const void *a_scale, long long a_scale_stride, const void *w,
                                       const void *w_scale, int w_scale_stride, long long rows, int n, int k,
                                       const void *act, const void *act_scale, long long act_scale_stride, void *out,
                                       void *codes, void *scale, long long scale_stride, void *stream) {
    const F8Gemm g = {(const unsigned char *)a, (const unsigned char *)a_scale, (const unsigned char *)w,
                      (const unsigned char *)w_scale, a_scale_stride, w_scale_stride, rows, n, k, (uint16_t *)out,
                      (unsigned char *)codes, (unsigned char *)scale, (const unsigned char *)act,
                      (const unsigned char *)act_scale, scale_stride, act_scale_stride};
    return fg_gemm(g, FG_RELU2_BWD, stream);
}
