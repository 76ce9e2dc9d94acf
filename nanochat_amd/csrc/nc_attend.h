/*
 * What the attention kernels over the paged fp8 cache share (attention.hip, packed_attn.hip): a wave's query operands, its
 * softmax state, and the accesses that cross workgroups. The step over two 16-token pages (page_scores to pair_step_k:
 * scores, softmax update and PV) is attention.hip's, whose header describes it; packed_attn.hip has one of its own.
 */
#pragma once

#include <math.h>

#include "nc_device.h"
#include "nc_internal.h"

namespace nc {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int WAVES = 4;
constexpr int O_PITCH = HEAD_DIM + 4;  /* LDS row pitch of a wave's merged output (floats) */
constexpr float RESCALE_LOG2 = 8.0f;   /* lazy rescale threshold: exponentials stay <= 2^8 */

struct AttnArgs {
    const uint16_t *q;        /* [B][T][Hq][128] bf16 (T = 1 in decode) */
    const uint8_t *k_pages, *v_pages;
    const float *kv_scale;    /* [num_pages][Hkv][2][16]: K scales, then V scales */
    const int32_t *block_table;
    int max_pages, num_pages;
    const int32_t *seq_lens;  /* decode */
    const int32_t *start_pos; /* prefill: the first position of each sequence's (or run's) rows */
    const int32_t *run_row0;  /* NULL, or prefill runs: run b's rows are q/out rows run_row0[b] .. + run_count[b] */
    const int32_t *run_count;
    const int32_t *run_slot;  /* run b's block-table row */
    int B, T, Hq, Hkv, G, window;
    float scale_log2;         /* sm_scale * log2(e) */
    int workers;              /* decode: waves launched (whole work-groups of 4) */
    int max_len;              /* decode: the longest sequence the launch accepts (its workspace bound) */
    float *part_o;            /* decode partials [items][G][128] */
    float *part_ml;           /* [items][G][2]: reference max (log2 domain), sum */
    int *arrived;             /* [B*Hkv]: chunks of each (sequence, KV head) finished so far; zero between launches */
    uint16_t *out;            /* [B][T][Hq][128] bf16 */
    StepArgs step;            /* the fused decode step's append (decode_kernel<true>) */
};

/* A wave's running state for NT tiles of 16 query columns; lane (g, c) = (lane >> 4, lane & 15) holds column c
 * of every tile. */
template <int NT>
struct WaveState {
    f32x4 o[NT][8];  /* O^T tile d: dims 16d + 4g + i of column c, scaled by 2^-m */
    float m[NT];     /* column c's reference max (log2 domain, equal in the four groups); exponentials use it */
    float l[NT];     /* sum of exp2(s - m) over the keys this lane's group holds */
    float sl2;       /* score multiplier: sm_scale log2(e) */
    bool bad;        /* a block-table entry fell outside the page pool */
};

template <int NT>
__device__ __forceinline__ void state_init(WaveState<NT> &st) {
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int d = 0; d < 8; d++) st.o[t][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        st.m[t] = -INFINITY;
        st.l[t] = 0.0f;
    }
    st.bad = false;
}

/* The query operand of column c (B operand of the fp8 score MFMA v_mfma_scale_f32_16x16x128_f8f6f4): lane (g, c) holds
 * dims 32 g .. 32 g + 31 of its row as bytes 0..31, the same (lane, byte) -> k mapping as the K page's A operand
 * (lane (g, key) holds that key's dims 32 g .. + 31). The row times 2^e (e chosen per column, from the column's own
 * largest |q|, which lands in [128, 256)) is split into two e4m3 parts, hi = e4m3(x), lo = e4m3(x - hi): a bf16 value
 * has 8 significant bits and each part 4, so hi + lo = x exactly unless |x| < 2^-2 (then lo may lose bits below 2^-10,
 * at most 2^-18 of the column's largest element). The MFMA's E8M0 scale of the B operand, one per lane (a lane holds
 * exactly one 32-element block of one column), is 2^-e, so the products come out unscaled and one score multiplier
 * serves every column. The score MFMAs read the cache's K codes as they are, with no conversion. Since e depends on
 * the column alone, so do its scores: a row's result does not depend on the rows that share its wave. */
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct QOp {
    i32x8 hi, lo;
    int scale;   /* E8M0 code of 2^-e: 127 - e */
};

__device__ __forceinline__ f32x4 mfma_fp8(const i32x8 &a, const i32x8 &b, int scale_b, const f32x4 &c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 127, 0, scale_b);   /* A: unit scale */
}

/* QOp of NT tiles from this lane's raw bf16 (raw[t][cc] = dims 32 g + 8 cc .. + 7 of its column in tile t). Every lane
 * of the wave must call it (a column's maximum combines its four row groups). */
template <int NT>
__device__ __forceinline__ void q8_from_raw(const uint4 (&raw)[NT][4], QOp (&q)[NT]) {
    float amax[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        amax[t] = 0.0f;
#pragma unroll
        for (int cc = 0; cc < 4; cc++) {
            const uint32_t w[4] = {raw[t][cc].x, raw[t][cc].y, raw[t][cc].z, raw[t][cc].w};
#pragma unroll
            for (int i = 0; i < 4; i++)
                amax[t] = fmaxf(amax[t], fmaxf(fabsf(bf16_to_f32((uint16_t)w[i])), fabsf(bf16_to_f32((uint16_t)(w[i] >> 16)))));
        }
        amax[t] = pair_max32(pair_max16(amax[t]));   /* the column's four row groups */
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int E = amax[t] > 0.0f ? (int)((__float_as_uint(amax[t]) >> 23) & 0xFFu) - 127 : 0;
        const int e = min(max(7 - E, -120), 120);
        const float up = __uint_as_float((uint32_t)(127 + e) << 23);
        q[t].scale = 127 - e;
#pragma unroll
        for (int cc = 0; cc < 4; cc++) {
            const uint32_t w[4] = {raw[t][cc].x, raw[t][cc].y, raw[t][cc].z, raw[t][cc].w};
#pragma unroll
            for (int h = 0; h < 2; h++) {   /* dwords 2 cc + h of the operand: dims 32 g + 8 cc + 4 h .. + 3 */
                float x[4];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    x[2 * i] = bf16_to_f32((uint16_t)w[2 * h + i]) * up;
                    x[2 * i + 1] = bf16_to_f32((uint16_t)(w[2 * h + i] >> 16)) * up;
                }
                int hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
                hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], hi, true);
                const float r[4] = {x[0] - __builtin_amdgcn_cvt_f32_fp8(hi, 0), x[1] - __builtin_amdgcn_cvt_f32_fp8(hi, 1),
                                    x[2] - __builtin_amdgcn_cvt_f32_fp8(hi, 2), x[3] - __builtin_amdgcn_cvt_f32_fp8(hi, 3)};
                int lo = __builtin_amdgcn_cvt_pk_fp8_f32(r[0], r[1], 0, false);
                lo = __builtin_amdgcn_cvt_pk_fp8_f32(r[2], r[3], lo, true);
                q[t].hi[2 * cc + h] = hi;
                q[t].lo[2 * cc + h] = lo;
            }
        }
    }
}

/* Stages NT rows (NULL: zeros) as QOp; every lane of the wave must call it. */
template <int NT>
__device__ __forceinline__ void load_q8(const uint16_t *const (&rows)[NT], int g, QOp (&q)[NT]) {
    uint4 raw[NT][4];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int cc = 0; cc < 4; cc++)
            raw[t][cc] = rows[t] ? *reinterpret_cast<const uint4 *>(rows[t] + g * 32 + cc * 8) : uint4{0u, 0u, 0u, 0u};
    q8_from_raw<NT>(raw, q);
}

/* Scores S^T (keys 4g + i of one page, column c of tile t) = K Q^T for every tile from one page's two K loads
 * (dims 32 g .. + 15, then + 16 .. + 31): two fp8 MFMAs a tile, hi then lo. */
template <int NT>
__device__ __forceinline__ void page_scores(const uint4 &k0, const uint4 &k1, const QOp (&qb)[NT], f32x4 (&s)[NT]) {
    const i32x8 k = {(int)k0.x, (int)k0.y, (int)k0.z, (int)k0.w, (int)k1.x, (int)k1.y, (int)k1.z, (int)k1.w};
#pragma unroll
    for (int t = 0; t < NT; t++) {
        s[t] = mfma_fp8(k, qb[t].hi, qb[t].scale, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
        s[t] = mfma_fp8(k, qb[t].lo, qb[t].scale, s[t]);
    }
}

__device__ __forceinline__ uint32_t dword(const uint4 &u, int i) {
    return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
}

__device__ __forceinline__ uint4 and4(const uint4 &u, uint32_t m) { return uint4{u.x & m, u.y & m, u.z & m, u.w & m}; }

/* Two consecutive logical pages (lpa, lpa + 1) of one KV head: their (page, head) indices. Without a second
 * page in range (has_b false) the first is read twice and every key of the copy is masked. */
struct PairAddr {
    long long ha, hb;
    int lpa;
    bool has_b;
};

__device__ __forceinline__ PairAddr pair_addr(const AttnArgs &a, const int32_t *bt, int kvh, int lpa, int end,
                                              bool &bad) {
    PairAddr p;
    p.lpa = lpa;
    p.has_b = lpa + 1 < end;
    int pa = bt[lpa];
    int pb = p.has_b ? bt[lpa + 1] : pa;
    if ((unsigned)pa >= (unsigned)a.num_pages) { bad = true; pa = 0; }
    if ((unsigned)pb >= (unsigned)a.num_pages) { bad = true; pb = 0; }
    p.ha = (long long)pa * a.Hkv + kvh;
    p.hb = (long long)pb * a.Hkv + kvh;
    return p;
}

/* One operand (K or V) of a page pair as this lane loads it: two 1 KiB-contiguous 16-byte loads per page and
 * the four scales of the lane's keys 4g..4g+3. */
struct PairRegs {
    uint4 a0, a1, b0, b1;
    float4 sa, sb;
};

/* Page bytes are streamed once per launch: non-temporal loads (measured ~7 TB/s for a plain stream on MI355X,
 * against ~6.4 TB/s for ordinary loads). */
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint4 load_nt(const uint8_t *p) {
    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
    return uint4{v[0], v[1], v[2], v[3]};
}

__device__ __forceinline__ float4 load_nt(const float *p) {
    const f32x4v v = __builtin_nontemporal_load(reinterpret_cast<const f32x4v *>(p));
    return float4{v[0], v[1], v[2], v[3]};
}

/* scales: the K (or V) half of kv_scale, i.e. kv_scale (+ 16 for V); a (page, head)'s scales are 32 floats apart. */
__device__ __forceinline__ void load_pair(const uint8_t *pages, const float *scales, const PairAddr &p, int lane,
                                          PairRegs &r) {
    const uint8_t *A = pages + p.ha * PAGE_BYTES + lane * 16;
    const uint8_t *Bp = pages + p.hb * PAGE_BYTES + lane * 16;
    r.a0 = load_nt(A);
    r.a1 = load_nt(A + 1024);
    r.b0 = load_nt(Bp);
    r.b1 = load_nt(Bp + 1024);
    r.sa = load_nt(scales + p.ha * 2 * PAGE + (lane >> 4) * 4);
    r.sb = load_nt(scales + p.hb * 2 * PAGE + (lane >> 4) * 4);
}

/* Key bounds of a wave: in tile t a lane's column sees keys [lo[t], hi[t]]; pairs inside [full_lo, full_hi]
 * are unmasked for every column; V codes of keys past written_hi are not cache contents and are zeroed. */
template <int NT>
struct KeyBounds {
    int lo[NT], hi[NT];
    int full_lo, full_hi, written_hi;
};

/* Softmax update and PV of one pair from its scores. The lazy rescale keeps each column's reference max m until a
 * score passes it by RESCALE_LOG2 (so p <= 2^8). The common case costs one FMA and one exponential a score:
 * p = exp2(acc ks - m) against the current m. Only a column some of whose p exceed 2^8 (or whose m is still -inf) takes
 * the slow path, which moves the column to its new max, rescales it and recomputes its p; the wave enters the slow
 * block when any of its columns needs it, but every column's update depends on its own scores alone, so a query row's
 * result does not depend on the rows that share its wave. The pair's exponentials and PV MFMAs then form one straight
 * block. Each converted V operand feeds NT MFMAs. */
template <int NT, bool MASKED>
__device__ __forceinline__ void pair_update(const AttnArgs &a, const PairAddr &p, const f32x4 (&sa)[NT],
                                            const f32x4 (&sb)[NT], const float4 &ksa, const float4 &ksb, PairRegs &v,
                                            const KeyBounds<NT> &kb, WaveState<NT> &st, int lane) {
    const int g = lane >> 4;
    const int key_a = p.lpa * PAGE + g * 4, key_b = key_a + PAGE;
    if (MASKED) {
        const int na = min(max(kb.written_hi - key_a + 1, 0), 4), nb = p.has_b ? min(max(kb.written_hi - key_b + 1, 0), 4) : 0;
        const uint32_t ma = na >= 4 ? 0xFFFFFFFFu : ((1u << (8 * na)) - 1u);
        const uint32_t mb = nb >= 4 ? 0xFFFFFFFFu : ((1u << (8 * nb)) - 1u);
        v.a0 = and4(v.a0, ma); v.a1 = and4(v.a1, ma);
        v.b0 = and4(v.b0, mb); v.b1 = and4(v.b1, mb);
    }
    const float ks[8] = {ksa.x * st.sl2, ksa.y * st.sl2, ksa.z * st.sl2, ksa.w * st.sl2,
                         ksb.x * st.sl2, ksb.y * st.sl2, ksb.z * st.sl2, ksb.w * st.sl2};
    const float vs[8] = {v.sa.x, v.sa.y, v.sa.z, v.sa.w, v.sb.x, v.sb.y, v.sb.z, v.sb.w};
    bool ok[NT][8];
    float pr[NT][8];
    float pmax = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const float negm = -st.m[t];   /* +inf before the first key: every live p is +inf, the slow path */
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float acc = i < 4 ? sa[t][i] : sb[t][i - 4];
            if (MASKED) {
                const int key = (i < 4 ? key_a : key_b) + (i & 3);
                ok[t][i] = (i < 4 || p.has_b) && key >= kb.lo[t] && key <= kb.hi[t];
            } else {
                ok[t][i] = true;
            }
            pr[t][i] = ok[t][i] ? __builtin_amdgcn_exp2f(__builtin_fmaf(acc, ks[i], negm)) : 0.0f;
            pmax = fmaxf(pmax, pr[t][i]);
        }
    }
    if (__any(!(pmax <= 256.0f))) {   /* some column's max passed its reference by more than 2^8 (or has none yet) */
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float pc = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) pc = fmaxf(pc, pr[t][i]);
            pc = pair_max32(pair_max16(pc));   /* the column's largest p over its four row groups */
            if (pc <= 256.0f) continue;        /* this column keeps its reference and its p (NaN-free: pc >= 0) */
            float s[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float acc = i < 4 ? sa[t][i] : sb[t][i - 4];
                s[i] = ok[t][i] ? acc * ks[i] : -INFINITY;
            }
            float mt = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
            mt = pair_max32(pair_max16(mt));   /* the column's max over the four row groups */
            const float mnew = fmaxf(st.m[t], mt);
            const float alpha = mnew == st.m[t] ? 1.0f : __builtin_amdgcn_exp2f(st.m[t] - mnew);
#pragma unroll
            for (int d = 0; d < 8; d++) st.o[t][d] *= alpha;
            st.l[t] *= alpha;
            st.m[t] = mnew;
            const float mbase = mnew == -INFINITY ? 0.0f : mnew;  /* no key yet: every s is -inf */
#pragma unroll
            for (int i = 0; i < 8; i++) pr[t][i] = __builtin_amdgcn_exp2f(s[i] - mbase);
        }
    }
    bf16x8 pv[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        float psum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            psum += pr[t][i];
            pv[t][i] = (__bf16)(pr[t][i] * vs[i]);
        }
        st.l[t] += psum;
    }
#pragma unroll
    for (int d = 0; d < 8; d++) {
        const bf16x8 va = fp8x8_to_bf16(dword(d < 4 ? v.a0 : v.a1, d & 3), dword(d < 4 ? v.b0 : v.b1, d & 3));
#pragma unroll
        for (int t = 0; t < NT; t++) st.o[t][d] = mfma16x16x32(va, pv[t], st.o[t][d]);
    }
}

template <int NT>
__device__ __forceinline__ void pair_step(const AttnArgs &a, const PairAddr &cur, const f32x4 (&sa)[NT],
                                          const f32x4 (&sb)[NT], const float4 &ksa, const float4 &ksb, PairRegs &vr,
                                          const KeyBounds<NT> &kb, WaveState<NT> &st, int lane) {
    const bool interior = cur.has_b && cur.lpa * PAGE >= kb.full_lo && cur.lpa * PAGE + 2 * PAGE - 1 <= kb.full_hi &&
                          cur.lpa * PAGE + 2 * PAGE - 1 <= kb.written_hi;
    if (interior)
        pair_update<NT, false>(a, cur, sa, sb, ksa, ksb, vr, kb, st, lane);
    else
        pair_update<NT, true>(a, cur, sa, sb, ksa, ksb, vr, kb, st, lane);
}

/* pair_step with the scores made inside each branch from the pair's K operands (k0, k1: page a; k2, k3: page b), so
 * the score MFMAs share a scheduling block with the exponentials: page a's products first, then page b's, one at a
 * time between groups of page a's softmax instructions, which do not wait for them (c4: 830-843 -> 868-875 TFLOP/s
 * against all eight products issued before the branch). The wave raises its priority while it issues them, so the
 * SIMD's other wave, when it is in its softmax, issues between them (870 -> 882 TFLOP/s; the same around the PV
 * products added nothing). */
template <int NT, bool MASKED>
__device__ __forceinline__ void pair_update_k(const AttnArgs &a, const PairAddr &p, const uint4 &k0, const uint4 &k1,
                                              const uint4 &k2, const uint4 &k3, const QOp (&qb)[NT],
                                              const float4 &ksa, const float4 &ksb, PairRegs &v,
                                              const KeyBounds<NT> &kb, WaveState<NT> &st, int lane) {
    f32x4 sa[NT], sb[NT];
    __builtin_amdgcn_s_setprio(1);   /* the other wave of the SIMD runs its VALU while these products issue */
    page_scores<NT>(k0, k1, qb, sa);
    page_scores<NT>(k2, k3, qb, sb);
    __builtin_amdgcn_sched_group_barrier(0x008, 2 * NT, 0);
#pragma unroll
    for (int i = 0; i < 2 * NT; i++) {   /* groups of 2 to 10 VALU instructions measured the same */
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
    }
    __builtin_amdgcn_s_setprio(0);
    pair_update<NT, MASKED>(a, p, sa, sb, ksa, ksb, v, kb, st, lane);
}

template <int NT>
__device__ __forceinline__ void pair_step_k(const AttnArgs &a, const PairAddr &cur, const uint4 &k0, const uint4 &k1,
                                            const uint4 &k2, const uint4 &k3, const QOp (&qb)[NT], const float4 &ksa,
                                            const float4 &ksb, PairRegs &vr, const KeyBounds<NT> &kb,
                                            WaveState<NT> &st, int lane) {
    const bool interior = cur.has_b && cur.lpa * PAGE >= kb.full_lo && cur.lpa * PAGE + 2 * PAGE - 1 <= kb.full_hi &&
                          cur.lpa * PAGE + 2 * PAGE - 1 <= kb.written_hi;
    if (interior)
        pair_update_k<NT, false>(a, cur, k0, k1, k2, k3, qb, ksa, ksb, vr, kb, st, lane);
    else
        pair_update_k<NT, true>(a, cur, k0, k1, k2, k3, qb, ksa, ksb, vr, kb, st, lane);
}

typedef __amdgpu_buffer_rsrc_t Rsrc;


/* A descriptor over `bytes` bytes from p, p the same in every lane (its halves are read from the first lane, so the
 * descriptor lives in scalar registers and no load needs a per-lane loop). */
__device__ __forceinline__ Rsrc page_rsrc(const void *p, int bytes) {
    const unsigned long long u = (unsigned long long)p;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)u), hi = __builtin_amdgcn_readfirstlane((unsigned)(u >> 32));
    void *q = (void *)(((unsigned long long)hi << 32) | lo);
    return __builtin_amdgcn_make_buffer_rsrc(q, (short)0, __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

/* The last b in [0, B) with cum[b] <= k (cum non-decreasing, cum[0] = 0 <= k). */
__device__ __forceinline__ int find_sequence(const int *cum, int B, int k) {
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cum[mid] <= k) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ void store_bf16x4(uint16_t *dst, const float *v) {
    uint2 u;
    u.x = (uint32_t)f32_to_bf16(v[0]) | ((uint32_t)f32_to_bf16(v[1]) << 16);
    u.y = (uint32_t)f32_to_bf16(v[2]) | ((uint32_t)f32_to_bf16(v[3]) << 16);
    *reinterpret_cast<uint2 *>(dst) = u;
}

/* Partials cross work-groups (and XCDs, whose L2 caches are not coherent with each other) inside one launch. They
 * are written and read with the sc1 cache policy, the encoding of agent-scope atomic stores and loads (coherent
 * across the device: stores write through, loads miss stale lines), and the writer waits for its stores to complete
 * (vmcnt 0) before it counts its chunk, so the wave that sees the last count reads every partial as written. This
 * costs no cache-wide writeback or invalidate, which an agent-scope fence would (measured: twice the kernel time). */
constexpr int SC1 = 16;   /* cache-policy operand of the buffer builtins: sc1 */
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ void part_store(Rsrc r, int off, const float4 &v) {
    __builtin_amdgcn_raw_buffer_store_b128(u32x4{__float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z),
                                                 __float_as_uint(v.w)}, r, off, 0, SC1);
}

__device__ __forceinline__ f32x4 part_load(Rsrc r, int off) {
    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, SC1);
    return f32x4{__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]), __uint_as_float(v[3])};
}

}  // namespace nc
