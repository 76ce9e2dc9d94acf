/*
 * Attention of packed query rows over the paged fp8 cache on gfx950: each sequence brings any number of new tokens (one to
 * decode, a few drafts to verify, a chunk of a prompt), all already in the cache, and its row t attends the keys
 * [max(p - window, 0), p] of its own sequence, p = seq_len - n + t. One launch serves the whole mix; lengths and row
 * offsets stay on the device. (The reference runs such rows as separate kernels, model/kernels/decode.cu:567-675 and
 * 1041-1051; the padded forms are attention.hip's.)
 *
 *   o = sum_j exp2(s_j - m) v_j / sum_j exp2(s_j - m),  s_j = (q . k_j) sm_scale log2(e),  m a running maximum
 *
 * The step over two pages (pk_pair) is this file's own; the query operand, the softmax state and the accesses across
 * workgroups are nc_attend.h's. Scores, softmax, sums and O are held in 32 bits; a probability times its key's V scale is
 * rounded to bf16 for the second product, whose matrix instruction takes bf16 (V codes are exact there), and the output once
 * more: against float64 about 1.4 times the error of one rounding. What bounds a sequence depends on its rows: a page of a
 * KV head is 2 KiB of K, 2 KiB of V and 128 bytes of scales for 16 keys, and each query column costs 512 flops a key, so
 * below about 80 columns (rows times the heads of a KV head) the pages' bytes take longer than the products. Hence two
 * kinds of work items, both streaming pages into LDS by asynchronous copies:
 *
 *   narrow  at most 32 columns: one wave takes a chunk of the keys by itself, page pairs through a ring of its own in LDS
 *           with two pairs in flight; waves meet at no barrier, so one's start or merge hides behind the others' streams.
 *           A sequence of at most PK_SHORT pages is not cut but shared by the four waves of a workgroup, which merge
 *           through LDS ("alone": it costs no round trips through memory, which is what a short one's time is made of)
 *   wide    a tile of up to 128 columns, 32 a wave: the four waves of a workgroup walk the same pairs, each fetched once
 *           (two stages of two pairs ahead); of at most 64 columns two waves take one pair of a stage and two the other,
 *           so that no wave idles (64 sequences of 64 columns over 8,192 keys: 169 us, and 209 by two waves of the four)
 *
 * A sequence's keys are cut into chunks (pk_plan), so that few rows over many keys still fill the chip; a (tile, KV head)
 * of several chunks leaves one partial (O, max, sum) in fp32 a chunk, and whoever finishes its last chunk merges them in
 * order. The cuts depend on nothing but the sequence's own numbers, so its output bits do not depend on the rest of the
 * launch. A workgroup takes wide and alone items while there are any, then its waves narrow ones: the first by workgroup
 * index, later ones from eight queues (an XCD's workgroups take every eighth item, which keeps a KV head's pages in that
 * XCD's L2), so that unequal items even out.
 *
 * Measured (16 query heads, 4 KV heads): 64 sequences of 8,192 keys, one row each 100 us (5.5 TB/s of pages), 4 rows each
 * 111 us (5.0), 16 rows each 169 us; 8 prompt chunks of 512 rows, each over 4,096 keys, 174 us (740 TFLOP/s of the
 * keys a row may see), 2 prompts of 4,096 rows 175 us (787). One sequence, 5 rows of 6 heads over 1,029 keys: 14.5 us, most
 * of it round trips to memory one after the other (the plan, the block table, pages, the output). These are times of calls in
 * a row; the first hundred launches after a pause run at a lower clock and take up to a fifth longer where products bound
 * them (the 8 chunks 213 -> 174 us).
 */
#include <limits.h>

#include "nc_attend.h"
#include "nanochat_amd.h"

namespace nc {

constexpr int PK_NT = 2;                       /* 16-column tiles a wave */
constexpr int PK_NARROW_COLS = 16 * PK_NT;
constexpr int PK_WIDE_COLS = WAVES * 16 * PK_NT;
constexpr int PK_MAX_BATCH = 1024;
constexpr int PK_QUEUES = 8;                   /* XCDs */
/* Pages of a narrow chunk: 64 sequences of 8,192 keys, 4 rows each, take 112 us with 64 pages and 158 with 32 (twice the
 * partials); one of 32,768 keys 35.6 and 33.2. */
constexpr int PK_NARROW_SPLIT = 64;
constexpr int PK_MIN_TAIL = 4;                 /* a last chunk of fewer pages joins the one before it */
/* A narrow sequence of at most so many pages is not cut: 1,029 keys take 14.4 us whole, 30.4 in two partials. */
constexpr int PK_SHORT = 2 * PK_NARROW_SPLIT;
/* Least and most pages of a wide chunk, and the items that a wide sequence is cut into at most if its chunks stay that long.
 * Short chunks fill the chip when a sequence is alone, and cost partials when it is not: one chunk of 512 rows over 8,192 keys
 * takes 71 us with 128 pages at least and 113 with 256, eight of them over 4,096 keys 175 and 152 (64 pages: 70 and
 * 201). A cut by what else the launch holds would make a sequence's bits depend on it. 128 items: 111 us for the first, and
 * 253 instead of 179 for 4 chunks of 200 to 700 rows among 60 decoding sequences. */
constexpr int PK_WIDE_MIN = 128, PK_WIDE_MAX = 1024, PK_WIDE_ITEMS = 256;
constexpr int PK_AHEAD = 2;                    /* wide: stages of two pairs in flight */
static_assert(PK_SHORT <= 2 * WAVE && PK_NARROW_SPLIT + PK_MIN_TAIL <= 2 * WAVE,
              "a narrow item's block-table entries: two a lane");

/* A pair in a stage: K (2 x 2 KiB), V (2 x 2 KiB), and its scales, per page 16 of K, then 16 of V. A narrow stage is one
 * pair, scales last; a wide one two pairs, then both pairs' scales for each wave. */
constexpr int PK_SCALE_AT = 4 * PAGE_BYTES, PK_SCALE_BYTES = 256;
constexpr int PK_WIDE_STAGE = 2 * PK_SCALE_AT + WAVES * 2 * PK_SCALE_BYTES, PK_WIDE_BUFS = PK_AHEAD + 1;
constexpr int PK_NARROW_STAGE = PK_SCALE_AT + PK_SCALE_BYTES;
constexpr int PK_BUFS = 2;                     /* pairs of a narrow wave's ring */
constexpr int PK_STAGES = WAVES * PK_BUFS * PK_NARROW_STAGE;   /* bytes of LDS */
static_assert(PK_WIDE_BUFS * PK_WIDE_STAGE <= PK_STAGES, "the wide stages fit");
typedef __attribute__((address_space(3))) void LdsVoid;

struct PackedArgs {
    AttnArgs a;                 /* q, pools, block_table, seq_lens, B, Hq, Hkv, G, window, scale_log2, max_len, out */
    const int32_t *cu;          /* [B + 1] */
    int rows;                   /* rows of q and out */
    float *part_wide, *part_narrow;   /* [slots][cols][128] O, then [slots][cols][2] (max, sum) */
    long long wide_slots, narrow_slots;
    int units;                  /* arrival counts */
    int tpt;                    /* tokens of a 16-column tile: 16 / G */
    int *tickets, *done, *arrived;    /* [2][8][PK_LINE] (workgroups, waves), [PK_LINE], [units]; zero between launches */
};

/* A sequence's rows, its pages [pg0, pg0 + np) (pg0 even) and how they are cut: nch chunks of s pages from pg0. tiles = 0:
 * no rows; < 0: a length that does not fit (its rows become NaN). */
struct PkSeq {
    int row0, n, len, pg0, np, tiles, s, nch;
    bool narrow, alone;   /* narrow; and of at most PK_SHORT pages: one item, four waves */
};

__device__ __forceinline__ PkSeq pk_plan(const PackedArgs &p, int row0, int n, int len) {
    const AttnArgs &a = p.a;
    PkSeq q = {};
    q.row0 = row0;
    q.n = n;
    if (q.n == 0) return q;
    q.len = len;
    if (q.len < q.n || q.len > a.max_len) {
        q.tiles = -1;
        return q;
    }
    const int first = a.window >= 0 ? max(q.len - q.n - a.window, 0) : 0;
    q.pg0 = (first / PAGE) & ~1;
    q.np = (q.len - 1) / PAGE + 1 - q.pg0;
    const int tpw = p.tpt * PK_NT;
    q.narrow = q.n <= tpw;
    if (q.narrow) {
        q.tiles = 1;
        q.alone = q.np <= PK_SHORT;
        q.s = PK_NARROW_SPLIT;
        q.nch = q.alone ? 1 : (q.np - 1) / q.s + 1;
        q.nch -= q.nch > 1 && q.np - (q.nch - 1) * q.s < PK_MIN_TAIL;
    } else {
        q.tiles = (int)((unsigned)(q.n - 1) / (unsigned)(WAVES * tpw)) + 1;
        const unsigned want = max((unsigned)PK_WIDE_ITEMS / (unsigned)(q.tiles * a.Hkv), 1u);
        q.s = min(max((int)(((unsigned)(q.np - 1) / want + 1 + 31) & ~31u), PK_WIDE_MIN), PK_WIDE_MAX);
        q.nch = (int)((unsigned)(q.np - 1) / (unsigned)q.s) + 1;
    }
    return q;
}

/* This lane, as a value the compiler cannot compute ahead: nothing made of it is kept in registers across items. */
__device__ __forceinline__ int pk_lane() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t & (WAVE - 1);
}

/* A value that is the same in every lane, as a scalar register's. */
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

constexpr int PK_SUMS = 6;   /* of the sequences before each: wide, alone and narrow items, units, wide and narrow slots */

/* a + b, at most INT_MAX (a, b >= 0): counts that only overlapping row offsets could make so large. */
__device__ __forceinline__ int pk_add(int a, int b) { return (int)min((unsigned)a + (unsigned)b, (unsigned)INT_MAX); }

/* Exclusive prefix sums of PK_SUMS values a thread over the workgroup's 256 threads. Within a wave by DPP: shifts by 1, 2,
 * 4 and 8 within rows of 16 lanes, then a row's last sum added to the next row's, and the lower half's to the upper's. */
__device__ __forceinline__ void pk_scan(int (&v)[PK_SUMS], int (&part)[PK_SUMS][WAVES]) {
    const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < PK_SUMS; k++) {
        int s = v[k];
        s = pk_add(s, __builtin_amdgcn_update_dpp(0, s, 0x111, 0xF, 0xF, false));
        s = pk_add(s, __builtin_amdgcn_update_dpp(0, s, 0x112, 0xF, 0xF, false));
        s = pk_add(s, __builtin_amdgcn_update_dpp(0, s, 0x114, 0xF, 0xF, false));
        s = pk_add(s, __builtin_amdgcn_update_dpp(0, s, 0x118, 0xF, 0xF, false));
        s = pk_add(s, __builtin_amdgcn_update_dpp(0, s, 0x142, 0xA, 0xF, false));
        s = pk_add(s, __builtin_amdgcn_update_dpp(0, s, 0x143, 0xC, 0xF, false));
        if (lane == WAVE - 1) part[k][wave] = s;
        v[k] = (int)__builtin_amdgcn_update_dpp(0, s, 0x138, 0xF, 0xF, false);   /* the lane before's, 0 in lane 0 */
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PK_SUMS; k++)
#pragma unroll
        for (int w = 0; w < WAVES; w++) v[k] = pk_add(v[k], w < wave ? part[k][w] : 0);
}

/* A workgroup barrier that drains no asynchronous copy; memory accesses do not move across it. */
__device__ __forceinline__ void pk_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ int pk_lds_offset(const unsigned char *p) {
    return (int)(uintptr_t)(__attribute__((address_space(3))) const unsigned char *)p;
}

/* s_waitcnt operands (gfx9 encoding: vmcnt in bits 3:0 and 15:14, expcnt 6:4, lgkmcnt 11:8). */
constexpr int pk_wait(int vmcnt, int lgkmcnt) { return (vmcnt & 15) | (vmcnt >> 4) << 14 | 7 << 4 | lgkmcnt << 8; }

/* One partial's O [cols][128] and (max, sum) [cols][2]. */
struct PkPart {
    float *o, *ml;
};
__device__ __forceinline__ PkPart pk_part(float *base, long long slots, int cols, long long slot) {
    return PkPart{base + slot * cols * HEAD_DIM, base + slots * cols * HEAD_DIM + slot * cols * 2};
}

/* What an item works on: the KV head, its tokens t0 .. t0 + tn - 1 of the sequence, pages [pg0, pg1) of its chunk. */
struct PkItem {
    PkSeq q;
    int b, kvh, t0, tn, pg0, pg1;
};

/* Column c of wave tile t (first token wt0) -> its token (< 0: not live). */
__device__ __forceinline__ int pk_token(const PackedArgs &p, int wt0, int end, int t, int c) {
    const int tok = wt0 + t * p.tpt + (int)((unsigned)c / (unsigned)p.a.G);
    return c < p.tpt * p.a.G && tok < end ? tok : -1;
}

__device__ __forceinline__ long long pk_row(const PackedArgs &p, const PkItem &it, int tok, int c) {
    return ((long long)it.q.row0 + tok) * p.a.Hq + it.kvh * p.a.G + (int)((unsigned)c % (unsigned)p.a.G);
}

/* Keys of a wave: in tile t a lane's column sees [lo[t], hi[t]]; the pairs from page in0 (even) up to in1 are seen whole by
 * every column. No column sees keys outside [first, last], which need not be cache contents: the sequence may end inside
 * the pair, and a window's first page may be its second, the page before having left the block table. */
template <int NT>
struct PkBounds {
    int lo[NT], hi[NT];
    int in0, in1, first, last;
};

/* The first key that the sequence's row t sees. */
__device__ __forceinline__ int pk_first_key(const PackedArgs &p, const PkSeq &q, int t) {
    return p.a.window >= 0 ? max(q.len - q.n + t - p.a.window, 0) : 0;
}

/* Per-column key bounds of a wave whose first token is wt0 (end: one past the item's last), its query operand and the
 * columns' references. */
template <int NT>
__device__ __forceinline__ void pk_columns(const PackedArgs &p, const PkItem &it, int wt0, int end, int lane,
                                           PkBounds<NT> &kb, uint4 (&raw)[NT][4], WaveState<NT> &st) {
    const AttnArgs &a = p.a;
    const int c = lane & 15, g = lane >> 4, start = it.q.len - it.q.n, tpt = p.tpt;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int tok = pk_token(p, wt0, end, t, c), pos = start + tok;
        kb.hi[t] = tok >= 0 ? pos : -1;
        /* a column that is not live has zero scores: with a finite reference they never ask for a rescale (one that did, on
         * every pair, took half the time of a wave with few columns) */
        st.m[t] = tok >= 0 ? -INFINITY : 0.0f;
        kb.lo[t] = tok >= 0 && a.window >= 0 ? max(pos - a.window, 0) : 0;
#pragma unroll
        for (int cc = 0; cc < 4; cc++)
            raw[t][cc] = tok >= 0 ? *reinterpret_cast<const uint4 *>(a.q + pk_row(p, it, tok, c) * HEAD_DIM + g * 32 + cc * 8)
                                  : uint4{0u, 0u, 0u, 0u};
    }
    const int last = min(wt0 + NT * tpt, end) - 1;
    kb.first = pk_first_key(p, it.q, wt0);
    kb.last = start + last;
    const int whole_lo = pk_first_key(p, it.q, last), whole_hi = start + wt0;
    kb.in0 = ((whole_lo + PAGE - 1) / PAGE + 1) & ~1;
    kb.in1 = min((whole_hi + 1) / PAGE, it.pg1) & ~1;
}

/* A pair's operands from a stage: four 16-byte reads a lane (K: at = the stage's LDS byte, V: 4 KiB on) and the lane's
 * scales of both pages (K: sc = the scales' LDS byte, V: 64 on), in registers when this returns. The compiler would make
 * ordinary reads of the stages wait for every copy in flight into any of them (it cannot tell one stage from another);
 * these wait for nothing but themselves, the caller having waited for the stage's own copies. */
__device__ __forceinline__ void pk_read(int at, int sc, int lane, PairRegs &k) {
    u32x4 a0, a1, b0, b1, sa, sb;
    asm volatile("ds_read_b128 %0, %6\n\t"
                 "ds_read_b128 %1, %6 offset:1024\n\t"
                 "ds_read_b128 %2, %6 offset:2048\n\t"
                 "ds_read_b128 %3, %6 offset:0xc00\n\t"
                 "ds_read_b128 %4, %7\n\t"
                 "ds_read_b128 %5, %7 offset:128\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(a0), "=&v"(a1), "=&v"(b0), "=&v"(b1), "=&v"(sa), "=&v"(sb)
                 : "v"(at + lane * 16), "v"(sc + (lane >> 4) * 16)
                 : "memory");
    k.a0 = uint4{a0[0], a0[1], a0[2], a0[3]};
    k.a1 = uint4{a1[0], a1[1], a1[2], a1[3]};
    k.b0 = uint4{b0[0], b0[1], b0[2], b0[3]};
    k.b1 = uint4{b1[0], b1[1], b1[2], b1[3]};
    k.sa = float4{__uint_as_float(sa[0]), __uint_as_float(sa[1]), __uint_as_float(sa[2]), __uint_as_float(sa[3])};
    k.sb = float4{__uint_as_float(sb[0]), __uint_as_float(sb[1]), __uint_as_float(sb[2]), __uint_as_float(sb[3])};
}

/* Four zeros in registers of their own, for the products that start a sum (the compiler would set them anew each time). */
__device__ __forceinline__ f32x4 pk_zero() {
    f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
    asm volatile("" : "+v"(z));
    return z;
}

/* x, of which nothing is computed before this point (work of rare paths would move ahead of their branches). */
__device__ __forceinline__ int pk_here(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

/* A stage's place in LDS, for one wave. */
struct PkAt {
    int at, scales;
};

constexpr float PK_RESCALE = 2048.0f;

/* One pair's scores, softmax and PV. The lazy rescale, as in nc_attend.h: a column keeps its reference maximum m, and its
 * exponentials p = exp2(s - m) grow past one, until the sum of a lane's eight passes PK_RESCALE (the sum is made anyway,
 * where the largest would take eight more instructions); then the column moves to its new maximum. The decision and what
 * it does depend on the column's own scores. A pair that holds keys which some column does not see is masked: what is not
 * seen takes no part whatever its bytes (its exponential and its product with the V scale are replaced by zero, and the V
 * codes of keys that no column sees are cleared; the cache's own codes are never NaN, whatever was appended). freed() is
 * called once the stage's bytes are in registers. */
template <int NT, typename Freed>
__device__ __forceinline__ void pk_pair(int lpa, bool has_b, PkAt stage, const QOp (&qb)[NT], const PkBounds<NT> &kb,
                                        const f32x4 &zero, WaveState<NT> &st, int lane, Freed freed) {
    const int key_a = lpa * PAGE + (lane >> 4) * 4;
    PairRegs k, v;
    pk_read(stage.at, stage.scales, lane, k);
    f32x4 sc[NT][2];
    {
        const i32x8 a = {(int)k.a0.x, (int)k.a0.y, (int)k.a0.z, (int)k.a0.w, (int)k.a1.x, (int)k.a1.y, (int)k.a1.z, (int)k.a1.w};
        const i32x8 b = {(int)k.b0.x, (int)k.b0.y, (int)k.b0.z, (int)k.b0.w, (int)k.b1.x, (int)k.b1.y, (int)k.b1.z, (int)k.b1.w};
        __builtin_amdgcn_s_setprio(1);   /* the other wave of the SIMD runs its VALU while these products issue */
#pragma unroll
        for (int t = 0; t < NT; t++) {   /* independent products between two that add up */
            sc[t][0] = mfma_fp8(a, qb[t].hi, qb[t].scale, zero);
            sc[t][1] = mfma_fp8(b, qb[t].hi, qb[t].scale, zero);
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            sc[t][0] = mfma_fp8(a, qb[t].lo, qb[t].scale, sc[t][0]);
            sc[t][1] = mfma_fp8(b, qb[t].lo, qb[t].scale, sc[t][1]);
        }
        __builtin_amdgcn_s_setprio(0);
    }
    __builtin_amdgcn_sched_barrier(0);   /* K's registers are free, and V's reads take less than the products */
    const float ks[8] = {k.sa.x * st.sl2, k.sa.y * st.sl2, k.sa.z * st.sl2, k.sa.w * st.sl2,
                         k.sb.x * st.sl2, k.sb.y * st.sl2, k.sb.z * st.sl2, k.sb.w * st.sl2};
    const auto vs = [&](int i) { return i < 4 ? (&v.sa.x)[i] : (&v.sb.x)[i - 4]; };
    /* key: the lane's first key of page a */
    const auto seen = [&](int key, int t, int i) {
        key += (i < 4 ? 0 : PAGE) + (i & 3);
        return (i < 4 || has_b) && key >= kb.lo[t] && key <= kb.hi[t];
    };
    const auto sum8 = [](const float (&x)[8]) {
        return ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
    };
    float pv[NT][8], sum[NT];
    if (lpa >= kb.in0 && lpa < kb.in1) {   /* V is read on both paths: one path's changes to it cost the other no copy */
        pk_read(stage.at + 2 * PAGE_BYTES, stage.scales + PAGE * 4, lane, v);
        freed();
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const float negm = -st.m[t];   /* +inf before the first key: every p is +inf, the slow path */
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; i++) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i >> 2][i & 3], ks[i], negm));
            sum[t] = sum8(e);
#pragma unroll
            for (int i = 0; i < 8; i++) pv[t][i] = e[i] * vs(i);
        }
    } else {
        const int key = pk_here(key_a);
        pk_read(stage.at + 2 * PAGE_BYTES, stage.scales + PAGE * 4, lane, v);
        freed();
        const auto upto = [&](int k) {   /* the codes of a lane's four keys, a byte each, that lie below the k-th */
            const int n = min(max(k, 0), 4);
            return n >= 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1u;
        };
        const uint32_t ma = upto(kb.last - key + 1) & ~upto(kb.first - key);
        const uint32_t mb = has_b ? upto(kb.last - key - PAGE + 1) & ~upto(kb.first - key - PAGE) : 0u;
        v.a0 = and4(v.a0, ma); v.a1 = and4(v.a1, ma);
        v.b0 = and4(v.b0, mb); v.b1 = and4(v.b1, mb);
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const float negm = -st.m[t];
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i >> 2][i & 3], ks[i], negm));
                e[i] = seen(key, t, i) ? e[i] : 0.0f;
                pv[t][i] = seen(key, t, i) ? e[i] * vs(i) : 0.0f;
            }
            sum[t] = sum8(e);
        }
    }
    bool fine = true;
#pragma unroll
    for (int t = 0; t < NT; t++) fine = fine && sum[t] <= PK_RESCALE;
    if (__any(!fine)) {
        const int key = pk_here(key_a);
#pragma unroll
        for (int t = 0; t < NT; t++) {
            /* by selections, not a branch a lane */
            const bool move = pair_max32(pair_max16(sum[t])) > PK_RESCALE;   /* the column's largest over its four groups */
            float mt = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; i++) mt = fmaxf(mt, seen(key, t, i) ? sc[t][i >> 2][i & 3] * ks[i] : -INFINITY);
            mt = pair_max32(pair_max16(mt));
            const float mnew = move ? fmaxf(st.m[t], mt) : st.m[t];
            const float alpha = mnew == st.m[t] ? 1.0f : __builtin_amdgcn_exp2f(st.m[t] - mnew);
            const float base = mnew == -INFINITY ? 0.0f : mnew;
#pragma unroll
            for (int d = 0; d < 8; d++) st.o[t][d] *= alpha;
            st.l[t] *= alpha;
            st.m[t] = mnew;
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i >> 2][i & 3], ks[i], -base));
                e[i] = seen(key, t, i) ? e[i] : 0.0f;
                pv[t][i] = seen(key, t, i) ? e[i] * vs(i) : 0.0f;
            }
            sum[t] = sum8(e);
        }
    }
    bf16x8 pb[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        st.l[t] += sum[t];
#pragma unroll
        for (int i = 0; i < 8; i++) pb[t][i] = (__bf16)pv[t][i];
    }
#pragma unroll
    for (int d = 0; d < 8; d++) {
        const bf16x8 va = fp8x8_to_bf16(dword(d < 4 ? v.a0 : v.a1, d & 3), dword(d < 4 ? v.b0 : v.b1, d & 3));
#pragma unroll
        for (int t = 0; t < NT; t++) st.o[t][d] = mfma16x16x32(va, pb[t], st.o[t][d]);
    }
}

/* A column of tile t (c of it, token tok): its bf16 row; or its part of a partial, column `col` there. l: of all groups. */
template <int NT>
__device__ __forceinline__ void pk_store_row(const PackedArgs &p, const PkItem &it, const WaveState<NT> &ws, int t, int tok, int c,
                                             int g) {
    uint16_t *dst = p.a.out + pk_row(p, it, tok, c) * HEAD_DIM;
    const float inv = 1.0f / ws.l[t];
#pragma unroll
    for (int d = 0; d < 8; d++) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = ws.bad ? NAN : ws.o[t][d][i] * inv;
        store_bf16x4(dst + 16 * d + 4 * g, v);
    }
}

template <int NT>
__device__ __forceinline__ void pk_store_part(const WaveState<NT> &ws, int t, int col, int g, Rsrc ro, Rsrc rm) {
#pragma unroll
    for (int d = 0; d < 8; d++)
        part_store(ro, (col * HEAD_DIM + 16 * d + 4 * g) * 4,
                   float4{ws.o[t][d][0], ws.o[t][d][1], ws.o[t][d][2], ws.o[t][d][3]});
    if (g == 0)
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(ws.bad ? NAN : ws.m[t]), __float_as_uint(ws.l[t])}, rm,
                                              col * 8, 0, SC1);
}

/* Tickets: queue x holds the items first + x, first + x + 8, ... below N, its count on a line of its own (atomics on one
 * line wait for each other, wherever they come from). pk_draw takes a ticket of queue x. pk_next makes an item of one drawn
 * from queue `own`, or draws from whichever queue has some left (INT_MAX: none has); a whole wave calls it. Items are drawn
 * when the one before is done: drawn earlier, an item would wait for it. */
constexpr int PK_LINE = 32;   /* ints of a 128-byte line */

__device__ __forceinline__ int pk_draw(int *tickets, int x) {
    return __hip_atomic_fetch_add(tickets + x * PK_LINE, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ int pk_have(int first, int N, int x) {   /* items of queue x */
    return N - first > x ? (N - first - x - 1) / PK_QUEUES + 1 : 0;
}

__device__ __forceinline__ int pk_next(int *tickets, int first, int N, int own, int got, int lane) {
    int x = own;
    got = uni(got);
    for (;;) {
        if (got < pk_have(first, N, x)) return first + x + got * PK_QUEUES;
        /* lane i < 8: queue own + i */
        const int y = (own + lane) % PK_QUEUES;
        const int taken = lane < PK_QUEUES ? __hip_atomic_load(tickets + y * PK_LINE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                                           : INT_MAX;
        const unsigned long long left = __ballot(taken < pk_have(first, N, y));
        if (!left) return INT_MAX;
        x = (own + __ffsll(left) - 1) % PK_QUEUES;
        got = 0;
        if (lane == 0) got = pk_draw(tickets, x);
        got = uni(got);
    }
}

/* --- wide items */

/* One stage's copies, two pairs (pages 4 s .. 4 s + 3 of the chunk; past its end, its last one again): wave w page w's K and
 * V (two of 1 KiB each) and all four pages' scales into its own slot (two of 256 bytes); every wave always issues six. */
__device__ __forceinline__ void pk_fetch_wide(const AttnArgs &a, const int *tab, int npages, int s, int kvh, unsigned char *st,
                                              int wave, int lane) {
    const int pg = uni(tab[min(4 * s + wave, npages - 1)]);
    const long long ph = (long long)pg * a.Hkv + kvh;
    /* pair wave / 2: K of its pages, then V */
    unsigned char *k = st + (wave >> 1) * PK_SCALE_AT + (wave & 1) * PAGE_BYTES, *v = k + 2 * PAGE_BYTES;
    __builtin_amdgcn_global_load_lds((const void *)(a.k_pages + ph * PAGE_BYTES + lane * 16), (LdsVoid *)k, 16, 0, 0);
    __builtin_amdgcn_global_load_lds((const void *)(a.k_pages + ph * PAGE_BYTES + 1024 + lane * 16), (LdsVoid *)(k + 1024), 16, 0, 0);
    __builtin_amdgcn_global_load_lds((const void *)(a.v_pages + ph * PAGE_BYTES + lane * 16), (LdsVoid *)v, 16, 0, 0);
    __builtin_amdgcn_global_load_lds((const void *)(a.v_pages + ph * PAGE_BYTES + 1024 + lane * 16), (LdsVoid *)(v + 1024), 16, 0, 0);
    unsigned char *sc = st + 2 * PK_SCALE_AT + wave * 2 * PK_SCALE_BYTES;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const long long sh = (long long)tab[min(4 * s + 2 * h + (lane >> 5), npages - 1)] * a.Hkv + kvh;
        __builtin_amdgcn_global_load_lds((const void *)(a.kv_scale + sh * 2 * PAGE + (lane & 31)),
                                         (LdsVoid *)(sc + h * PK_SCALE_BYTES), 4, 0, 0);
    }
}

/* The merge of a tile's partials by the workgroup that finishes last, in chunk order, from its own state (chunk `own`) and
 * the others' in slots slot0 ..: a lane loads what it holds itself, eight dims a tile of its columns, a chunk at a time. */
__device__ __forceinline__ void pk_join(const PackedArgs &p, const PkItem &it, int chunks, int own, long long slot0,
                                        const WaveState<PK_NT> &ws, const int (&tok)[PK_NT], int wcol, int c, int g) {
    float m[PK_NT], l[PK_NT];
    f32x4 o[PK_NT][8];
#pragma unroll
    for (int t = 0; t < PK_NT; t++) {
        m[t] = -INFINITY;
        l[t] = 0.0f;
#pragma unroll
        for (int d = 0; d < 8; d++) o[t][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    for (int j = 0; j < chunks; j++) {
        float mj[PK_NT], lj[PK_NT];
        f32x4 oj[PK_NT][8];
        if (j == own) {
#pragma unroll
            for (int t = 0; t < PK_NT; t++) {
                mj[t] = ws.bad ? NAN : ws.m[t];
                lj[t] = ws.l[t];
#pragma unroll
                for (int d = 0; d < 8; d++) oj[t][d] = ws.o[t][d];
            }
        } else {   /* sc1: past this XCD's L2, where another workgroup's stores are not seen */
            const PkPart part = pk_part(p.part_wide, p.wide_slots, PK_WIDE_COLS, slot0 + j);
            const Rsrc ro = page_rsrc(part.o, PK_WIDE_COLS * HEAD_DIM * 4), rm = page_rsrc(part.ml, PK_WIDE_COLS * 8);
#pragma unroll
            for (int t = 0; t < PK_NT; t++) {
                const int col = (wcol * PK_NT + t) * 16 + c;
                const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(rm, col * 8, 0, SC1);
                mj[t] = __uint_as_float(w[0]);
                lj[t] = __uint_as_float(w[1]);
#pragma unroll
                for (int d = 0; d < 8; d++) oj[t][d] = part_load(ro, (col * HEAD_DIM + 16 * d + 4 * g) * 4);
            }
        }
#pragma unroll
        for (int t = 0; t < PK_NT; t++) {
            const float mb = fmaxf(m[t], mj[t]);
            const float keep = m[t] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[t] - mb);
            const float f = mj[t] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mj[t] - mb);   /* NaN: a bad page */
            l[t] = l[t] * keep + lj[t] * f;
            m[t] = mb;
#pragma unroll
            for (int d = 0; d < 8; d++) o[t][d] = o[t][d] * keep + oj[t][d] * f;
        }
    }
#pragma unroll
    for (int t = 0; t < PK_NT; t++) {
        if (tok[t] < 0) continue;
        uint16_t *dst = p.a.out + pk_row(p, it, tok[t], c) * HEAD_DIM;
        const float inv = 1.0f / l[t];
#pragma unroll
        for (int d = 0; d < 8; d++) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = o[t][d][i] * inv;
            store_bf16x4(dst + 16 * d + 4 * g, v);
        }
    }
}

/* own: this item's place among its tile's chunks, whose partials are in slots slot0 ..; arrived: their count. queue: NULL, or
 * where thread 0 draws the workgroup's next ticket while its partial is on its way (returned). */
__device__ __forceinline__ int pk_wide(const PackedArgs &p, const PkItem &it, int chunks, int own, long long slot0, int *arrived,
                                       unsigned char *stages, int *tab, int &shared, int *queue) {
    const AttnArgs &a = p.a;
    const int lane = pk_lane(), wave = uni((int)threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int tpw = p.tpt * PK_NT, start = it.q.len - it.q.n;
    /* at most two waves' columns: waves w and w + 2 share them, one the first pair of every stage, one the second */
    const bool halves = it.tn <= 2 * tpw;
    const int wcol = halves ? wave & 1 : wave;
    const int wt0 = it.t0 + wcol * tpw, end = it.t0 + it.tn, npages = it.pg1 - it.pg0;
    const bool on = wt0 < end;
    const int last = min(wt0 + tpw, end) - 1;
    /* the wave's own pages, and pairs, within the chunk's */
    const int w0 = max(pk_first_key(p, it.q, wt0) / PAGE, it.pg0);
    const int w1 = on ? min((start + last) / PAGE + 1, it.pg1) : 0, count = (npages + 1) / 2;
    const int s0 = min(max(w0 - it.pg0, 0) / 2, count), s1 = min(max(w1 - it.pg0 + 1, 0) / 2, count);
    PkBounds<PK_NT> kb;
    uint4 raw[PK_NT][4];
    WaveState<PK_NT> ws;
    state_init(ws);
    ws.sl2 = a.scale_log2;
    pk_columns<PK_NT>(p, it, wt0, end, lane, kb, raw, ws);
    /* every wave looks at all the entries (is one outside the pool among its pages'?) and stores a quarter of them */
    const int32_t *bt = a.block_table + (long long)it.b * a.max_pages + it.pg0;
    bool bad = false;
    for (int i = lane; i < npages; i += WAVE) {
        const int e = bt[i];
        const bool ok = (unsigned)e < (unsigned)a.num_pages;
        bad = bad || (!ok && i >= w0 - it.pg0 && i < w1 - it.pg0);
        if (((i >> 6) & (WAVES - 1)) == wave) tab[i] = ok ? e : 0;   /* only read: a wave that needs it reports NaN */
    }
    ws.bad = __any(bad);
    __syncthreads();
    const f32x4 zero = pk_zero();
    const int lds = pk_lds_offset(stages), steps = (count + 1) / 2;
    for (int s = 0; s < PK_AHEAD; s++) pk_fetch_wide(a, tab, npages, s, it.kvh, stages + s * PK_WIDE_STAGE, wave, lane);
    QOp qb[PK_NT];
    q8_from_raw<PK_NT>(raw, qb);
    /* step s: this wave's copies of stage s have landed (then everyone's, after the barrier, and everyone's reads of the
     * stage before are done); refill that buffer with stage s + PK_AHEAD; compute the stage's pairs that meet this wave's */
    for (int s = 0, buf = 0; s < steps; s++) {
        __builtin_amdgcn_s_waitcnt(pk_wait(6 * (PK_AHEAD - 1), 15));
        pk_barrier();
        const int into = buf == 0 ? PK_WIDE_BUFS - 1 : buf - 1;   /* (s + PK_AHEAD) % PK_WIDE_BUFS */
        pk_fetch_wide(a, tab, npages, s + PK_AHEAD, it.kvh, stages + into * PK_WIDE_STAGE, wave, lane);
        const int st = lds + buf * PK_WIDE_STAGE;
        const int from = max(2 * s + (halves ? wave >> 1 : 0), s0), until = min(2 * s + (halves ? (wave >> 1) + 1 : 2), s1);
        for (int i = from; i < until; i++) {
            const int at = st + (i & 1) * PK_SCALE_AT, lpa = it.pg0 + 2 * i;
            pk_pair<PK_NT>(lpa, lpa + 1 < it.pg1, PkAt{at, st + 2 * PK_SCALE_AT + (2 * wave + (i & 1)) * PK_SCALE_BYTES}, qb, kb,
                           zero, ws, lane, [] {});
        }
        buf = buf == PK_WIDE_BUFS - 1 ? 0 : buf + 1;
    }
    int prior = 0, got = -1;
    if (chunks > 1 && threadIdx.x == 0) prior = __hip_atomic_load(arrived, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_s_waitcnt(0);   /* every copy has landed before the stages and the table are used again */
    if (threadIdx.x == 0) shared = prior;
    __syncthreads();
    int tok[PK_NT];
#pragma unroll
    for (int t = 0; t < PK_NT; t++) {
        ws.l[t] = pair_sum32(pair_sum16(ws.l[t]));
        tok[t] = pk_token(p, wt0, end, t, c);
    }
    if (halves) {   /* waves 2 and 3 hand their states over: O [wave][column][O_PITCH] in the stages, (max, sum) in the table */
        float *o2 = reinterpret_cast<float *>(stages) + wcol * 16 * PK_NT * O_PITCH;
        float *ml2 = reinterpret_cast<float *>(tab) + wcol * 16 * PK_NT * 2;
        if (wave >= 2)
#pragma unroll
            for (int t = 0; t < PK_NT; t++) {
                const int col = t * 16 + c;
                if (g == 0) {
                    ml2[2 * col] = ws.bad ? NAN : ws.m[t];
                    ml2[2 * col + 1] = ws.l[t];
                }
#pragma unroll
                for (int d = 0; d < 8; d++) *reinterpret_cast<f32x4 *>(o2 + col * O_PITCH + 16 * d + 4 * g) = ws.o[t][d];
                tok[t] = -1;
            }
        __syncthreads();
        if (wave < 2)
#pragma unroll
            for (int t = 0; t < PK_NT; t++) {
                const int col = t * 16 + c;
                const float m2 = ml2[2 * col], mb = fmaxf(ws.m[t], m2);
                const float f1 = ws.m[t] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ws.m[t] - mb);
                const float f2 = m2 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m2 - mb);   /* NaN: a bad page */
                ws.l[t] = ws.l[t] * f1 + ml2[2 * col + 1] * f2;
                ws.m[t] = mb;
#pragma unroll
                for (int d = 0; d < 8; d++)
                    ws.o[t][d] = ws.o[t][d] * f1 + *reinterpret_cast<const f32x4 *>(o2 + col * O_PITCH + 16 * d + 4 * g) * f2;
            }
    }
    if (chunks == 1) {
#pragma unroll
        for (int t = 0; t < PK_NT; t++)
            if (tok[t] >= 0) pk_store_row<PK_NT>(p, it, ws, t, tok[t], c, g);
        return got;
    }
    if (uni(shared) != chunks - 1) {   /* others are not done: leave a partial */
        const PkPart part = pk_part(p.part_wide, p.wide_slots, PK_WIDE_COLS, slot0 + own);
        const Rsrc ro = page_rsrc(part.o, PK_WIDE_COLS * HEAD_DIM * 4), rm = page_rsrc(part.ml, PK_WIDE_COLS * 8);
#pragma unroll
        for (int t = 0; t < PK_NT; t++)
            if (tok[t] >= 0) pk_store_part<PK_NT>(ws, t, (wcol * PK_NT + t) * 16 + c, g, ro, rm);
        if (queue && threadIdx.x == 0) got = pk_draw(queue, 0);
        __builtin_amdgcn_s_waitcnt(pk_wait(0, 15));   /* this wave's part of the partial is out; then everyone's */
        __syncthreads();
        if (threadIdx.x == 0) shared = __hip_atomic_fetch_add(arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (uni(shared) != chunks - 1) return got;
    }
    pk_join(p, it, chunks, own, slot0, ws, tok, wcol, c, g);
    if (threadIdx.x == 0) __hip_atomic_store(arrived, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return got;
}

/* --- narrow items */

/* One pair's copies into a wave's stage: four of 1 KiB a page, through descriptors of one page (live false: of no range, so
 * nothing is read), and the 256 scale bytes. Nine in all. */
__device__ __forceinline__ void pk_fetch_narrow(const AttnArgs &a, int pa, int pb, bool live, int kvh, unsigned char *st,
                                                int lane) {
    const long long ha = (long long)pa * a.Hkv + kvh, hb = (long long)pb * a.Hkv + kvh;
    const int bytes = live ? PAGE_BYTES : 0;
    const Rsrc ka = page_rsrc(a.k_pages + ha * PAGE_BYTES, bytes), kb = page_rsrc(a.k_pages + hb * PAGE_BYTES, bytes);
    const Rsrc va = page_rsrc(a.v_pages + ha * PAGE_BYTES, bytes), vb = page_rsrc(a.v_pages + hb * PAGE_BYTES, bytes);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(ka, (LdsVoid *)st, 16, lane * 16, 0, 0, 2);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(ka, (LdsVoid *)(st + 1024), 16, lane * 16 + 1024, 0, 0, 2);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(kb, (LdsVoid *)(st + 2048), 16, lane * 16, 0, 0, 2);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(kb, (LdsVoid *)(st + 3 * 1024), 16, lane * 16 + 1024, 0, 0, 2);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(va, (LdsVoid *)(st + 4096), 16, lane * 16, 0, 0, 2);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(va, (LdsVoid *)(st + 5120), 16, lane * 16 + 1024, 0, 0, 2);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(vb, (LdsVoid *)(st + 6144), 16, lane * 16, 0, 0, 2);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(vb, (LdsVoid *)(st + 7168), 16, lane * 16 + 1024, 0, 0, 2);
    __builtin_amdgcn_global_load_lds((const void *)(a.kv_scale + (lane < 32 ? ha : hb) * 2 * PAGE + (lane & 31)),
                                     (LdsVoid *)(st + PK_SCALE_AT), 4, 0, 0);
}

/* The item's page pairs first, first + stride, ... by one wave. ALONE: the four waves of a workgroup share the item so and
 * merge their states through LDS (stages, ml); else one wave has a chunk to itself and leaves a partial. */
template <int NT, bool ALONE>
__device__ __forceinline__ void pk_narrow(const PackedArgs &p, const PkItem &it, long long slot, unsigned char *ring, int first,
                                          unsigned char *stages, float *ml) {
    constexpr int stride = ALONE ? WAVES : 1;
    const AttnArgs &a = p.a;
    const int lane = pk_lane(), c = lane & 15, g = lane >> 4;
    const int npages = it.pg1 - it.pg0, pairs = max(((npages + 1) / 2 - first + stride - 1) / stride, 0);
    /* lane j: entries j and 64 + j of the item's pages */
    const int32_t *bt = a.block_table + (long long)it.b * a.max_pages + it.pg0;
    const int before = pk_first_key(p, it.q, 0) / PAGE - it.pg0;   /* a page that no row sees */
    int e0 = lane < npages && lane >= before ? bt[lane] : 0, e1 = WAVE + lane < npages ? bt[WAVE + lane] : 0;
    WaveState<NT> ws;
    state_init(ws);
    ws.sl2 = a.scale_log2;
    ws.bad = __any((unsigned)e0 >= (unsigned)a.num_pages || (unsigned)e1 >= (unsigned)a.num_pages);
    if ((unsigned)e0 >= (unsigned)a.num_pages) e0 = 0;   /* only read: if a row needs it the item reports NaN */
    if ((unsigned)e1 >= (unsigned)a.num_pages) e1 = 0;
    const auto entry = [&](int e) {
        const int lo = __builtin_amdgcn_readlane(e0, e & (WAVE - 1)), hi = __builtin_amdgcn_readlane(e1, e & (WAVE - 1));
        return e < WAVE ? lo : hi;
    };
    PkBounds<NT> kb;
    uint4 raw[NT][4];
    pk_columns<NT>(p, it, 0, it.tn, lane, kb, raw, ws);
    const f32x4 zero = pk_zero();
    const int lds = pk_lds_offset(ring);
    const auto fetch = [&](int i, int buf) {
        const int la = i < pairs ? 2 * (first + stride * i) : 0, lb = la + 1 < npages ? la + 1 : la;   /* no second page: the
                                                                                                       * first again */
        pk_fetch_narrow(a, entry(la), entry(lb), i < pairs, it.kvh, ring + buf * PK_NARROW_STAGE, lane);
    };
#pragma unroll
    for (int i = 0; i < PK_BUFS; i++) fetch(i, i);
    QOp qb[NT];
    q8_from_raw<NT>(raw, qb);
    for (int i = 0; i < pairs; i++) {
        const int buf = i & (PK_BUFS - 1), at = lds + buf * PK_NARROW_STAGE, lpa = it.pg0 + 2 * (first + stride * i);
        /* all but the younger pairs' copies have landed */
        __builtin_amdgcn_s_waitcnt(pk_wait(9 * (PK_BUFS - 1), 15));
        asm volatile("" ::: "memory");
        pk_pair<NT>(lpa, lpa + 1 < it.pg1, PkAt{at, at + PK_SCALE_AT}, qb, kb, zero, ws, lane,
                    [&] { fetch(i + PK_BUFS, buf); });
    }
    if constexpr (!ALONE) {
        const PkPart part = pk_part(p.part_narrow, p.narrow_slots, PK_NARROW_COLS, slot);
        const Rsrc ro = page_rsrc(part.o, PK_NARROW_COLS * HEAD_DIM * 4), rm = page_rsrc(part.ml, PK_NARROW_COLS * 8);
#pragma unroll
        for (int t = 0; t < NT; t++) {
            ws.l[t] = pair_sum32(pair_sum16(ws.l[t]));
            if (pk_token(p, 0, it.tn, t, c) >= 0) pk_store_part<NT>(ws, t, t * 16 + c, g, ro, rm);
        }
        return;   /* the caller waits for the stores, and for the copies that read nothing */
    }
    float *merged = reinterpret_cast<float *>(stages), *sums = ml + WAVES * PK_NARROW_COLS;
    __builtin_amdgcn_s_waitcnt(0);   /* no copy of this wave's is in flight into the stages; then no one's */
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; t++) {
        ws.l[t] = pair_sum32(pair_sum16(ws.l[t]));
        const int row = (first * NT + t) * 16 + c;
        if (g == 0) {
            ml[row] = ws.bad ? NAN : ws.m[t];
            sums[row] = ws.l[t];
        }
#pragma unroll
        for (int d = 0; d < 8; d++) *reinterpret_cast<f32x4 *>(merged + row * O_PITCH + 16 * d + 4 * g) = ws.o[t][d];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 16 * (HEAD_DIM / 4); i += 256) {
        const int col = i >> 5, quad = i & 31, tok = pk_token(p, 0, it.tn, col >> 4, col & 15);
        if (tok < 0) continue;
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) m = fmaxf(m, ml[w * NT * 16 + col]);
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float mw = ml[w * NT * 16 + col];
            const float f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - m);   /* NaN: a bad page */
            o += *reinterpret_cast<const f32x4 *>(merged + (w * NT * 16 + col) * O_PITCH + 4 * quad) * f;
            l += sums[w * NT * 16 + col] * f;
        }
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = o[k] / l;
        store_bf16x4(a.out + pk_row(p, it, tok, col & 15) * HEAD_DIM + 4 * quad, v);
    }
}

/* The merge of a narrow unit's partials in slots slot0 .. slot0 + chunks - 1, in chunk order, into its bf16 rows, by one
 * wave, each lane P pieces of four dims at a time and NB chunks' loads of them in flight: the merge is bound by their
 * latency, so few columns take many chunks at a time and many columns few. */
template <int P, int NB>
__device__ __forceinline__ void pk_merge(const PackedArgs &p, const PkItem &it, int chunks, long long slot0, int lane) {
    const AttnArgs &a = p.a;
    constexpr int cols = PK_NARROW_COLS, pieces = cols * (HEAD_DIM / 4);
    const PkPart part = pk_part(p.part_narrow, p.narrow_slots, cols, slot0);
    for (int i0 = lane; i0 < pieces; i0 += P * WAVE) {
        int tok[P];
        bool some = false;
        float m[P], l[P];
        f32x4 o[P];
#pragma unroll
        for (int k = 0; k < P; k++) {
            const int col = (i0 + k * WAVE) >> 5;
            tok[k] = col < cols ? pk_token(p, it.t0, it.t0 + it.tn, col >> 4, col & 15) : -1;
            some = some || tok[k] >= 0;
            m[k] = -INFINITY;
            l[k] = 0.0f;
            o[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        if (!__any(some)) continue;
        for (int j0 = 0; j0 < chunks; j0 += NB) {
            f32x4 oj[NB][P];
            float mj[NB][P], lj[NB][P];
#pragma unroll
            for (int n = 0; n < NB; n++) {
                /* sc1: past this XCD's L2, where another workgroup's stores are not seen. Past the last chunk: descriptors
                 * of no range (zeros, no access) */
                const bool live = j0 + n < chunks;
                const long long j = live ? j0 + n : 0;
                const Rsrc ro = page_rsrc(part.o + j * cols * HEAD_DIM, live ? cols * HEAD_DIM * 4 : 0);
                const Rsrc rm = page_rsrc(part.ml + j * cols * 2, live ? cols * 8 : 0);
#pragma unroll
                for (int k = 0; k < P; k++) {
                    const int i = i0 + k * WAVE;
                    oj[n][k] = part_load(ro, i * 16);
                    const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(rm, (i >> 5) * 8, 0, SC1);
                    mj[n][k] = __uint_as_float(w[0]);
                    lj[n][k] = __uint_as_float(w[1]);
                }
            }
#pragma unroll
            for (int k = 0; k < P; k++)
#pragma unroll
                for (int n = 0; n < NB; n++) {
                    if (j0 + n >= chunks) continue;
                    const float mb = fmaxf(m[k], mj[n][k]);
                    const float keep = m[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[k] - mb);
                    const float f = mj[n][k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mj[n][k] - mb);   /* NaN: a bad page */
                    o[k] = o[k] * keep + oj[n][k] * f;
                    l[k] = l[k] * keep + lj[n][k] * f;
                    m[k] = mb;
                }
        }
#pragma unroll
        for (int k = 0; k < P; k++) {
            if (tok[k] < 0) continue;
            const int i = i0 + k * WAVE, col = i >> 5;
            float v[4];
#pragma unroll
            for (int d = 0; d < 4; d++) v[d] = o[k][d] / l[k];
            store_bf16x4(a.out + pk_row(p, it, tok[k], col & 15) * HEAD_DIM + 4 * (i & 31), v);
        }
    }
}

__global__ void __launch_bounds__(256, 2) packed_attn_kernel(PackedArgs p) {
    /* the stages, PK_STAGES bytes; [PK_SUMS][B + 1] prefix sums; [3][B]: row0, n, len. Two workgroups fit a CU up to 281
     * sequences; beyond, one: 512 of 2,049 keys take 210 us (5.3 TB/s of pages), 256 take 99 (5.6). */
    extern __shared__ __align__(16) unsigned char stages[];
    int *pk_lds = reinterpret_cast<int *>(stages + PK_STAGES);
    __shared__ int tab[PK_WIDE_MAX];
    __shared__ int scan[PK_SUMS][WAVES];
    __shared__ int sh_next;
    const AttnArgs &a = p.a;
    const int B = a.B;
    int *wide = pk_lds, *alone = wide + B + 1, *narrow = alone + B + 1, *units = narrow + B + 1, *wslots = units + B + 1,
        *nslots = wslots + B + 1, *row0 = nslots + B + 1, *count = row0 + B, *length = count + B;
    bool fits = true;
    {
        const int per = (B + 255) / 256, b0 = min((int)threadIdx.x * per, B), b1 = min(b0 + per, B);
        int sum[PK_SUMS] = {0, 0, 0, 0, 0, 0};
        for (int b = b0; b < b1; b++) {
            const int c0 = p.cu[b], c1 = p.cu[b + 1], len = a.seq_lens[b];
            row0[b] = min(max(c0, 0), p.rows);
            count[b] = min(max(c1, row0[b]), p.rows) - row0[b];
            length[b] = len;
            const PkSeq q = pk_plan(p, row0[b], count[b], len);
            const long long u64 = (long long)max(q.tiles, 0) * a.Hkv;
            const int u = (int)min(u64, (long long)INT_MAX), n = (int)min(u64 * q.nch, (long long)INT_MAX);
            const int cut = q.nch > 1 ? n : 0;
            const int v[PK_SUMS] = {q.narrow ? 0 : n, q.narrow && q.alone ? n : 0, q.narrow && !q.alone ? n : 0,
                                    q.nch > 1 ? u : 0, q.narrow ? 0 : cut, q.narrow ? cut : 0};
#pragma unroll
            for (int k = 0; k < PK_SUMS; k++) {
                wide[k * (B + 1) + b] = v[k];
                sum[k] = pk_add(sum[k], v[k]);
            }
        }
        pk_scan(sum, scan);
        for (int b = b0; b < b1; b++) {
            int v[PK_SUMS];
#pragma unroll
            for (int k = 0; k < PK_SUMS; k++) v[k] = wide[k * (B + 1) + b];
#pragma unroll
            for (int k = 0; k < PK_SUMS; k++) {
                wide[k * (B + 1) + b] = sum[k];
                sum[k] = pk_add(sum[k], v[k]);
            }
        }
        if (b1 == B && b0 < b1)
#pragma unroll
            for (int k = 0; k < PK_SUMS; k++) wide[k * (B + 1) + B] = sum[k];
        __syncthreads();
        /* row offsets that overlap could ask for more than the host sized the workspace for */
        fits = wslots[B] <= p.wide_slots && nslots[B] <= p.narrow_slots && units[B] <= p.units &&
               (long long)wide[B] + alone[B] < INT_MAX / 2 && narrow[B] < INT_MAX / 2;
    }
    /* rows of sequences whose length does not fit */
    for (int b = blockIdx.x; b < B; b += gridDim.x) {
        if (fits && (count[b] == 0 || (length[b] >= count[b] && length[b] <= a.max_len))) continue;
        uint2 *dst = reinterpret_cast<uint2 *>(a.out + (long long)row0[b] * a.Hq * HEAD_DIM);
        const long long quads = (long long)count[b] * a.Hq * (HEAD_DIM / 4);
        for (long long i = threadIdx.x; i < quads; i += 256) dst[i] = uint2{0x7FC07FC0u, 0x7FC07FC0u};
    }
    if (!fits) return;   /* every workgroup: no ticket is taken */

    /* wide and alone items, by workgroups */
    const int NW = uni(wide[B]), N = uni(NW + alone[B]), NN = uni(narrow[B]), G = gridDim.x, own = blockIdx.x % PK_QUEUES;
    const auto plan = [&](int b) { return pk_plan(p, uni(row0[b]), uni(count[b]), uni(length[b])); };
    for (int k = blockIdx.x; k < N;) {
        int got = -1;   /* in thread 0: a ticket already drawn */
        PkItem it;
        if (k < NW) {
            it.b = uni(find_sequence(wide, B, k));
            it.q = plan(it.b);
            /* a sequence's items: the last tiles first, then the chunks, its KV heads fastest */
            const int local = uni(k - wide[it.b]), rest = (int)((unsigned)local / (unsigned)a.Hkv);
            it.kvh = local - rest * a.Hkv;
            const int back = (int)((unsigned)rest / (unsigned)it.q.nch);
            const int tile = it.q.tiles - 1 - back, j = rest - back * it.q.nch, tokens = WAVES * PK_NT * p.tpt;
            it.t0 = tile * tokens;
            it.tn = min(it.q.n - it.t0, tokens);
            /* the tile's own pages, its chunks [j0, j1), this chunk's pages within */
            const int start = it.q.len - it.q.n;
            const int lo = ((a.window >= 0 ? max(start + it.t0 - a.window, 0) : 0) / PAGE) & ~1;
            const int hi = (start + it.t0 + it.tn - 1) / PAGE + 1;
            const int j0 = (lo - it.q.pg0) / it.q.s, j1 = (hi - 1 - it.q.pg0) / it.q.s + 1;
            it.pg0 = max(it.q.pg0 + j * it.q.s, lo);
            it.pg1 = min(it.q.pg0 + (j + 1) * it.q.s, hi);
            if (it.pg0 < it.pg1) {
                const long long slot0 = uni(wslots[it.b]) + ((long long)tile * a.Hkv + it.kvh) * it.q.nch;
                got = pk_wide(p, it, j1 - j0, j - j0, slot0, p.arrived + uni(units[it.b]) + tile * a.Hkv + it.kvh, stages, tab,
                              sh_next, N > G ? p.tickets + own * PK_LINE : nullptr);
            }
        } else {
            it.b = uni(find_sequence(alone, B, k - NW));
            it.q = plan(it.b);
            it.kvh = uni(k - NW - alone[it.b]);
            it.t0 = 0;
            it.tn = it.q.n;
            it.pg0 = it.q.pg0;
            it.pg1 = it.q.pg0 + it.q.np;
            const int wave = uni((int)threadIdx.x >> 6);
            unsigned char *ring = stages + wave * PK_BUFS * PK_NARROW_STAGE;
            if (it.tn <= p.tpt)
                pk_narrow<1, true>(p, it, 0, ring, wave, stages, reinterpret_cast<float *>(tab));
            else
                pk_narrow<2, true>(p, it, 0, ring, wave, stages, reinterpret_cast<float *>(tab));
        }
        if (N <= G) break;
        __syncthreads();   /* sh_next, the stages and the table are used again */
        if (threadIdx.x < WAVE) {
            if (got < 0 && threadIdx.x == 0) got = pk_draw(p.tickets, own);
            sh_next = pk_next(p.tickets, G, N, own, got, threadIdx.x);
        }
        __syncthreads();
        k = uni(sh_next);
    }
    __syncthreads();

    /* narrow items by the waves on their own, the first by index in the workgroups that had none of the others (so that
     * not every wave of the chip starts with a ticket) */
    const int lane = threadIdx.x & (WAVE - 1), wave = uni((int)threadIdx.x >> 6);
    const int free = max(G - N, 0), first = WAVES * free;
    unsigned char *ring = stages + wave * PK_BUFS * PK_NARROW_STAGE;
    int *tickets = p.tickets + PK_QUEUES * PK_LINE;
    const bool queued = NN > first;
    int k = (int)blockIdx.x - N + free * wave;
    if ((int)blockIdx.x < N) {
        int got = 0;
        if (queued && lane == 0) got = pk_draw(tickets, own);
        k = queued ? pk_next(tickets, first, NN, own, got, lane) : NN;
    }
    while (k < NN) {
        PkItem it;
        it.b = uni(find_sequence(narrow, B, k));
        it.q = plan(it.b);
        const int local = uni(k - narrow[it.b]), j = (int)((unsigned)local / (unsigned)a.Hkv);   /* the chunks, its KV heads fastest */
        it.kvh = local - j * a.Hkv;
        it.t0 = 0;
        it.tn = it.q.n;
        it.pg0 = it.q.pg0 + j * it.q.s;
        it.pg1 = j == it.q.nch - 1 ? it.q.pg0 + it.q.np : it.pg0 + it.q.s;
        const int chunks = it.q.nch;
        const long long slot0 = uni(nslots[it.b]) + (long long)it.kvh * chunks;
        if (it.tn <= p.tpt)
            pk_narrow<1, false>(p, it, slot0 + j, ring, 0, nullptr, nullptr);
        else
            pk_narrow<2, false>(p, it, slot0 + j, ring, 0, nullptr, nullptr);
        int got = 0;
        if (queued && lane == 0) got = pk_draw(tickets, own);
        __builtin_amdgcn_s_waitcnt(pk_wait(0, 15));   /* nothing is in flight into the ring, and the partial is out */
        int *arrived = p.arrived + uni(units[it.b]) + it.kvh;   /* an uncut sequence is an "alone" item: there are others */
        int prior = 0;
        if (lane == 0) prior = __hip_atomic_fetch_add(arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (uni(prior) == chunks - 1) {
            if (it.tn * a.G <= 4)
                pk_merge<2, 16>(p, it, chunks, slot0, lane);
            else
                pk_merge<4, 8>(p, it, chunks, slot0, lane);
            if (lane == 0) __hip_atomic_store(arrived, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (!queued) break;
        k = pk_next(tickets, first, NN, own, got, lane);
    }
    /* where tickets were taken, the last workgroup to leave returns them */
    if (N <= G && !queued) return;
    __syncthreads();
    if (threadIdx.x == 0 &&
        __hip_atomic_fetch_add(p.done, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == G - 1) {
        for (int x = 0; x < 2 * PK_QUEUES; x++)
            __hip_atomic_store(p.tickets + x * PK_LINE, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(p.done, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

/* The most partials and arrival counts a launch of these sizes can need, whatever its lengths (pk_plan): a narrow sequence
 * longer than PK_SHORT pages is Hkv units of at most ceil(pages / PK_NARROW_SPLIT) chunks. A wide one has at least tpw + 1
 * rows; all of them together have at most rows / (WAVES tpw) + their number tiles, each Hkv units, cut into at most
 * ceil(pages / PK_WIDE_MIN) chunks, and no sequence into more than PK_WIDE_ITEMS items unless its chunks would pass
 * PK_WIDE_MAX pages. */
struct PkSizes {
    long long wide_slots, narrow_slots, units;
};

static PkSizes pk_sizes(long long rows, int B, int Hq, int Hkv, int max_seq_len, int window) {
    const int tpt = 16 / (Hq / Hkv), tpw = tpt * PK_NT;
    long long np = ((long long)max_seq_len - 1) / PAGE + 1;
    /* a windowed sequence of n rows sees n + window keys, from an even page */
    if (window >= 0) np = min(np, (rows + window) / PAGE + 3);
    const long long nw = min((long long)B, rows / (tpw + 1)), tiles = rows / (WAVES * tpw) + nw;
    PkSizes z = {};
    const long long nch = np <= PK_SHORT ? 1 : (np - 1) / PK_NARROW_SPLIT + 1;
    const long long wch = (np - 1) / PK_WIDE_MIN + 1, most = (np - 1) / PK_WIDE_MAX + 1;
    if (nch > 1) z.narrow_slots = min((long long)B, rows) * Hkv * nch;
    if (wch > 1) z.wide_slots = min(tiles * Hkv * wch, nw * PK_WIDE_ITEMS + (most > 1 ? tiles * Hkv * most : 0));
    z.units = (nch > 1 ? min((long long)B, rows) : 0) * Hkv + (wch > 1 ? tiles * Hkv : 0);
    return z;
}

static size_t pk_part_bytes(const PkSizes &z) {
    return (size_t)(z.wide_slots * PK_WIDE_COLS + z.narrow_slots * PK_NARROW_COLS) * (HEAD_DIM + 2) * sizeof(float);
}

/* As attention.hip's decode workspace: partials from the start, int32 counts (tickets, done, arrivals) in the last 1/256,
 * whose place depends on the workspace's size alone. */
static size_t pk_count_region(size_t bytes) { return (bytes - ((bytes >> 8) & ~(size_t)3)) & ~(size_t)3; }
static size_t pk_count_bytes(const PkSizes &z) { return (size_t)(z.units + (2 * PK_QUEUES + 1) * PK_LINE) * sizeof(int); }

static bool pk_shape_ok(long long rows, int B, int Hq, int Hkv, int max_seq_len) {
    return rows > 0 && rows <= 1LL << 24 && B > 0 && B <= PK_MAX_BATCH && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 &&
           Hq / Hkv <= 16 && Hkv <= 1024 && max_seq_len > 0;
}

}  // namespace nc

using namespace nc;

extern "C" size_t nc_packed_workspace_bytes(long long rows, int B, int Hq, int Hkv, int max_seq_len, int window) {
    if (!pk_shape_ok(rows, B, Hq, Hkv, max_seq_len)) return 0;
    const PkSizes z = pk_sizes(rows, B, Hq, Hkv, max_seq_len, window);
    if (z.wide_slots > INT_MAX || z.narrow_slots > INT_MAX || z.units > INT_MAX / 2) return 0;
    size_t k = max((pk_part_bytes(z) + 254) / 255, pk_count_bytes(z));
    return 256 * ((k + 3) & ~(size_t)3);
}

extern "C" int nc_packed_attn_fp8(const void *q, const void *k_pages, const void *v_pages, const float *kv_scale,
                                  const int32_t *block_table, int max_pages, int num_pages, const int32_t *cu_seqlens,
                                  const int32_t *seq_lens, long long rows, int B, int Hq, int Hkv, int max_seq_len,
                                  int window, float sm_scale, void *out, void *workspace, size_t workspace_bytes,
                                  void *stream) {
    if (!q || !k_pages || !v_pages || !kv_scale || !block_table || !cu_seqlens || !seq_lens || !out || !workspace)
        return NC_ERR_NULL;
    if (!pk_shape_ok(rows, B, Hq, Hkv, max_seq_len) || max_pages <= 0 || num_pages <= 0 ||
        (long long)max_pages * PAGE < max_seq_len)
        return NC_ERR_SHAPE;
    const size_t need = nc_packed_workspace_bytes(rows, B, Hq, Hkv, max_seq_len, window);
    if (need == 0) return NC_ERR_SHAPE;
    const PkSizes z = pk_sizes(rows, B, Hq, Hkv, max_seq_len, window);
    const size_t counts = pk_count_region(workspace_bytes);
    if ((uintptr_t)workspace % 16 || pk_part_bytes(z) > counts || pk_count_bytes(z) > workspace_bytes - counts)
        return NC_ERR_WORKSPACE;
    PackedArgs p = {};
    AttnArgs &a = p.a;
    a.q = (const uint16_t *)q;
    a.k_pages = (const uint8_t *)k_pages; a.v_pages = (const uint8_t *)v_pages; a.kv_scale = kv_scale;
    a.block_table = block_table; a.max_pages = max_pages; a.num_pages = num_pages;
    a.seq_lens = seq_lens;
    a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.G = Hq / Hkv; a.window = window;
    a.scale_log2 = sm_scale * LOG2E;
    a.max_len = max_seq_len;
    a.out = (uint16_t *)out;
    p.cu = cu_seqlens;
    p.rows = (int)rows;
    p.part_wide = (float *)workspace;
    p.part_narrow = p.part_wide + z.wide_slots * PK_WIDE_COLS * (HEAD_DIM + 2);
    p.wide_slots = z.wide_slots; p.narrow_slots = z.narrow_slots;
    p.units = (int)z.units;
    p.tpt = 16 / a.G;
    p.tickets = (int *)((char *)workspace + counts);
    p.done = p.tickets + 2 * PK_QUEUES * PK_LINE;
    p.arrived = p.done + PK_LINE;
    const size_t lds = PK_STAGES + (PK_SUMS * (B + 1) + 3 * B) * sizeof(int);
    const int cus = device_cus() / PK_QUEUES * PK_QUEUES;
    hipLaunchKernelGGL(packed_attn_kernel, dim3(max(2 * cus, PK_QUEUES)), dim3(256), lds, (hipStream_t)stream, p);
    return (int)hipGetLastError();
}
