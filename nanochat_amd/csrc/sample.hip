/*
 * A token a row from its logits, by temperature, top-k, top-p and min-p, from one given uniform number a row: the token
 * choice of the decoder runtime (decoder.hip, whose noise comes from a seed) for callers with logits of their own.
 *
 *   weight   w_i = exp((z_i - max z) / T), for allowed tokens (the mask's bit set, z_i neither NaN nor -inf)
 *   top-k    the k largest, the lower index first among equals
 *   top-p    of those, the tokens with less than top_p of their weight strictly above them (equals stay together)
 *   min-p    of those, the tokens with w_i >= min_p
 *   choice   the first token, in index order, whose running weight exceeds u times the weight of all that are left
 *
 * Weights are integers: exp in float64 (2^x by a polynomial after splitting off the integer part), times 2^S and rounded.
 * Sums of integers depend on no order, so the LDS histograms may be filled by atomics, and the sums of a row are as exact as
 * its weights (2^-47 of the largest at 65,536 tokens): a border between two tokens moves by less than that share. In float32 a
 * border among many small weights would move by about their size.
 *
 * No sort: the place where a running count (top-k) or weight (top-p) in order of value reaches its target is found by a
 * histogram over ranges of the value, then among the few tokens of the range that holds it, or by finer histograms where it
 * holds many.
 *
 * split_kernel takes up to 512 / ceil(vocab / 8,192) rows of up to 262,144 tokens, a workgroup for every 8,192 (or
 * 4,096), which stay in its registers. What bounds it is neither bytes nor operations (a row of 65,536 fp32 logits is
 * 256 KiB) but the steps one after the other, each ending where the row's workgroups need one another: the largest logit; the
 * histogram; the list; about 2.5 us a meeting through memory. Greedy rows and a top-k of at most 128 need no meeting: every
 * slice leaves its k largest in order, and the last workgroup to arrive does the rest on k tokens. No meeting waits without
 * bound: where the others do not come, because the device is crowded, a row is given up and one workgroup does it
 * (nc_meeting.h). Measured: one row of 65,536 fp32 logits with top-p 22 us, with top-k 13; 64 rows 36 and 20.
 *
 * row_kernel takes a row by one workgroup that reads it again for every step, for more rows and for longer ones. With top-p
 * it is bound by the exponentials, twice for every token (about 180 cycles of a SIMD for a wave's 64, most of them float64
 * at half rate): 256 rows of 65,536 tokens 94 us, 333 rows of 32,768 masked bf16 logits 85. With a top-k it reads the row
 * twice and the rest is k tokens: 128 rows of 65,536 fp32 logits, a quarter of them greedy, 25 us (1.3 TB/s of logits).
 */
#include <math.h>

#include "nc_device.h"
#include "nc_internal.h"
#include "nc_meeting.h"
#include "nanochat_amd.h"

namespace nc {

typedef unsigned long long u64;

struct SampleArgs {
    const void *logits;
    long long stride;                    /* elements between rows */
    int vocab, bf16, wide;               /* wide: rows start at multiples of four elements' bytes */
    const float *uniform, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    const uint32_t *mask;
    long long mask_stride;
    int32_t *out;
};

/* Order-preserving integer of a float (no NaN, no -0) and back. */
__device__ __forceinline__ uint32_t order_key(float z) {
    const uint32_t u = __float_as_uint(z);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

/* a b + c with c, a constant, in scalar registers: the compiler would move it into vector registers first, each time. */
__device__ __forceinline__ double fma_by(double a, double b, double c) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}

/* round(2^S 2^x) for x <= 0; x below -100 or NaN: 0. 2^f, |f| <= 1/2, by a polynomial of degree 10 fitted for the least
 * relative error, 2^-52. The sum with 2^52 leaves the rounded integer in the low 52 bits (S <= 46). No branch: elements'
 * chains run side by side. */
__device__ __forceinline__ u64 fixed_exp2(double x, int S) {
    x = fmax(x, -100.0);
    const double n = __builtin_rint(x), f = x - n;
    double p = fma_by(f, 7.037259617627914e-09, 1.0208538206271505e-07);
    p = fma_by(p, f, 1.3215662976568588e-06);
    p = fma_by(p, f, 1.525265811546915e-05);
    p = fma_by(p, f, 0.00015403529960773235);
    p = fma_by(p, f, 0.0013333558228561912);
    p = fma_by(p, f, 0.009618129108034947);
    p = fma_by(p, f, 0.055504108664458846);
    p = fma_by(p, f, 0.24022650695908768);
    p = fma_by(p, f, 0.6931471805599497);
    p = __builtin_fma(p, f, 1.0);
    const double v = __builtin_ldexp(p, (int)n + S) + 0x1p52;
    return (u64)__builtin_bit_cast(long long, v) & 0xFFFFFFFFFFFFFull;
}

/* A value that is the same in every lane, as a scalar register's: branches on it are the wave's. */
__device__ __forceinline__ int alike(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ u64 alike(u64 x) {
    return (u64)(uint32_t)alike((int)(uint32_t)(x >> 32)) << 32 | (uint32_t)alike((int)(uint32_t)x);
}
__device__ __forceinline__ float alike(float x) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x))); }

/* What a row's token is chosen by. */
struct Choice {
    float T, u, p, zmax;
    double per_log2;
    u64 least_w;
    int S;   /* a weight of 1 is 2^S */

    __device__ __forceinline__ Choice(const SampleArgs &a, long long r, float temperature, float largest)
        : T(temperature), u(alike(a.uniform[r])), p(a.top_p ? alike(a.top_p[r]) : 1.0f), zmax(largest),
          per_log2(1.4426950408889634 / (double)temperature) {
        S = 62;   /* the row's weights sum below 2^62 */
        while (S > 0 && (1LL << (62 - S)) < a.vocab) S--;
        S = min(S, 46);
        const double floor_w = a.min_p ? fmin(fmax((double)alike(a.min_p[r]), 0.0), 1.0) : 0.0;   /* NaN: 0 */
        least_w = (u64)ceil(__builtin_ldexp(floor_w, S));
    }
    __device__ __forceinline__ u64 weight(float z) const {
        /* the largest's equals: 2^S, infinite ones too; -inf: 0 */
        return fixed_exp2(z == zmax ? 0.0 : ((double)z - (double)zmax) * per_log2, S);
    }
    /* The nucleus: tokens with less than this above them. */
    __device__ __forceinline__ u64 mass(u64 total) const {
        return max((u64)ceil(fmax((double)p, 0.0) * (double)total), 1ull);
    }
    /* The first running sum above u total. */
    __device__ __forceinline__ u64 choice(u64 total) const {
        const u64 at = u > 0.0f ? (u < 1.0f ? (u64)((double)u * (double)total) : total) : 0ull;
        return min(at, total - 1) + 1;
    }
    /* Values further below the largest than T ln(vocab / (1 - p)) weigh less than 1 - p of it together: the nucleus' border is
     * not among them, nor 47 log2 units below, where they weigh nothing. The first ranges need not tell them apart. */
    __device__ __forceinline__ float range(int vocab) const {
        return T * fminf(__logf((float)vocab / (1.0f - fmaxf(p, 0.0f))), 33.0f);
    }
};

/* Where a running sum reaches its target: its tokens' key, the last index taken among that key's equals, and whether the
 * sum reaches it at all. */
struct Cut {
    bool some;
    uint32_t key;
    int idx;
};

/* --- Rows of up to ST_MAX_GROUPS slices of 8,192 or 4,096 tokens, a workgroup each: the slice stays in its registers, E (16
 * or 8) tokens a thread, and the workgroups of a row exchange what the next step needs through memory. 512 threads of at most
 * 128 registers and the weights in LDS leave room for two workgroups a CU, one working while the other waits: measured side by
 * side, one workgroup a CU (149 registers, none spilled) took 25 us for one row instead of 27, but 124 instead of 88 for 333
 * rows, and slices of 1,024 threads with 8 tokens each 30 and 150. */

constexpr int ST_WAVES = 8, ST_THREADS = ST_WAVES * WAVE;
constexpr int ST_STEP = 4 * ST_THREADS;   /* element 4 c + j of thread t: index slice + c ST_STEP + 4 t + j */
constexpr int ST_MAX_GROUPS = 32;
constexpr int ST_BINS = 2 * ST_THREADS;
constexpr int ST_LIST = 256;              /* tokens a range may hold to be settled pairwise */
constexpr int ST_TOP = 128;               /* the largest top-k settled by lists of candidates */
constexpr int ST_CAND = 4096;             /* candidates: at most ST_TOP of 32 tokens, or of ST_MAX_GROUPS lists */
constexpr int ST_LINE = 32;               /* ints of a 128-byte line: counts that several workgroups add to share none */
constexpr int ST_QUEUES = 8;              /* XCDs */
constexpr int ST_MAX_WORKGROUPS = 512;    /* of rows that are cut: as many as run at once on 256 CUs, two a CU */
/* Looks at a row's word, each a round trip past the L2, before it is given up. The longest meeting is the first, which waits for
 * the last workgroups to start: 16 looks were enough for 64 rows of 65,536 tokens (42 us; given up after 8 looks 150), not for
 * 16 rows of 262,144 (71 us; given up 700). What giving up costs is the row done by one workgroup, so waiting about as long
 * as that takes is at most twice the better choice. */
constexpr int ST_PATIENCE = 400;
static_assert(ST_MAX_GROUPS <= MT_MOST_LEFT, "workgroups of a row that have left are counted");
constexpr int ST_MAX_E = 16;              /* tokens a thread: this many, or half */
static_assert(ST_TOP * (ST_MAX_E * ST_THREADS / 256) <= ST_CAND && ST_TOP * ST_MAX_GROUPS <= ST_CAND, "candidates fit");

enum { HD_BEST, HD_COUNT, HD_ABOVE, HD_LEAST, HD_MOST, HD_SUM, HD_WORDS };
constexpr int ST_PART = ST_BINS + 2 * ST_LIST + HD_WORDS;   /* words a workgroup publishes: histogram, list, head */

struct SplitArgs {
    SampleArgs a;
    int rows, groups;      /* slices a row */
    u64 *part;             /* [rows][groups][ST_PART] */
    int *tickets, *done, *count;   /* [ST_QUEUES], [ST_QUEUES], [rows] lines; zero between launches */
    int patience;
};

/* A row's word (nc_meeting.h). */
struct RowWord {
    int *p;
    __device__ __forceinline__ int add(int n) { return __hip_atomic_fetch_add(p, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
    __device__ __forceinline__ int look() const { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
    __device__ __forceinline__ bool swap(int &expected, int desired) {
        return __hip_atomic_compare_exchange_strong(p, &expected, desired, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                                    __HIP_MEMORY_SCOPE_AGENT);
    }
};

template <int E>
struct SplitShared {
    union {
        u64 weight[E * ST_THREADS];   /* element e of thread t: [e ST_THREADS + t] */
        struct {
            u64 cand[ST_CAND];
            u64 top[ST_TOP], top_w[ST_TOP], kept_w[ST_TOP];
            u64 most[256];
            int rank[ST_THREADS];
        };
    };
    union {
        u64 hist[ST_BINS];
        u64 above[ST_LIST];
    };
    u64 code[ST_LIST], w[ST_LIST];
    u64 sum[ST_MAX_E / 4 * ST_WAVES];
    u64 kept[ST_MAX_GROUPS], head[ST_MAX_GROUPS];
    int start[ST_MAX_GROUPS + 1];
    u64 found, least_code, lo, hi;
    int bin, n, token, flag;
};
static_assert(2 * sizeof(SplitShared<ST_MAX_E>) <= 160 * 1024, "two workgroups a CU");

/* A token as one integer: larger for the larger logit, and among equals for the lower index; 0: not allowed. */
__device__ __forceinline__ u64 token_code(float z, int i) {
    return z > -INFINITY ? (u64)order_key(z) << 32 | (0xFFFFFFFFu - (uint32_t)i) : 0ull;
}
__device__ __forceinline__ int code_index(u64 c) { return (int)(0xFFFFFFFFu - (uint32_t)c); }

/* Words that other workgroups read: past this XCD's L2 (sc1), where another's stores are not seen. */
__device__ __forceinline__ void publish(u64 *p, u64 v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ u64 peek(const u64 *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

/* Inclusive sums over the lanes by DPP: shifts by 1, 2, 4 and 8 within rows of 16 lanes, then a row's last sum added to the
 * next row's, and the lower half's to the upper's. */
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_add(u64 v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
    return v + ((u64)hi << 32 | lo);
}
__device__ __forceinline__ u64 lane_scan64(u64 v) {
    v = dpp_add<0x111, 0xF>(v);
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);
    return dpp_add<0x143, 0xC>(v);
}
__device__ __forceinline__ u64 lane64(u64 v, int lane) {
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
__device__ __forceinline__ u64 lane_sum64(u64 v) { return lane64(lane_scan64(v), WAVE - 1); }

template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_max(u64 v) {
    const uint32_t lo = (uint32_t)v, hi = (uint32_t)(v >> 32);
    const uint32_t l = __builtin_amdgcn_update_dpp((int)lo, (int)lo, CTRL, ROWS, 0xF, false);
    const uint32_t h = __builtin_amdgcn_update_dpp((int)hi, (int)hi, CTRL, ROWS, 0xF, false);
    return max(v, (u64)h << 32 | l);
}
__device__ __forceinline__ u64 lane_max64(u64 v) {
    v = dpp_max<0x111, 0xF>(v);
    v = dpp_max<0x112, 0xF>(v);
    v = dpp_max<0x114, 0xF>(v);
    v = dpp_max<0x118, 0xF>(v);
    v = dpp_max<0x142, 0xA>(v);
    v = dpp_max<0x143, 0xC>(v);
    return lane64(v, WAVE - 1);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_max(float v) {
    const int u = __float_as_int(v);
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(u, u, CTRL, ROWS, 0xF, false)));
}
__device__ __forceinline__ float lane_max(float v) {
    v = dpp_max<0x111, 0xF>(v);
    v = dpp_max<0x112, 0xF>(v);
    v = dpp_max<0x114, 0xF>(v);
    v = dpp_max<0x118, 0xF>(v);
    v = dpp_max<0x142, 0xA>(v);
    v = dpp_max<0x143, 0xC>(v);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), WAVE - 1));
}

/* Room for this lane's `count` entries at the end of a list of n: one addition a wave. */
__device__ __forceinline__ int reserve(int *n, int count, int lane) {
    const int at = (int)lane_scan64((u64)count);
    int first = 0;
    if (lane == WAVE - 1) first = __hip_atomic_fetch_add(n, at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    return __builtin_amdgcn_readlane(first, WAVE - 1) + at - count;
}

template <int E>
struct Split {
    const SplitArgs &s;
    SplitShared<E> &sh;
    int t, lane, wave;
    int row, g, G;         /* row, slice, slices */
    int first;             /* index of this thread's element 0 */
    int reached;           /* arrivals that the last wait of this row asked for */
    int gone;              /* the row was given up */
    u64 *mine;

    __device__ __forceinline__ int index(int e) const { return first + (e >> 2) * ST_STEP + (e & 3); }
    __device__ __forceinline__ u64 *part(int of) const { return s.part + ((long long)row * G + of) * ST_PART; }
    __device__ __forceinline__ int *counter() const { return s.count + (long long)row * ST_LINE; }

    /* Until every thread's stores are out. */
    __device__ __forceinline__ void arrive() {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
    /* Until every workgroup of the row has come as far: what they published is there. False: the row was given up, by this
     * workgroup or another, and is to be left at once. Every wait ends (nc_meeting.h), whatever else the device runs. */
    __device__ __forceinline__ bool meet() {
        arrive();
        if (G == 1) return true;
        reached += G;
        if (t == 0) {
            RowWord word{counter()};
            int seen = word.add(1) + 1, patience = s.patience;
            Meeting m;
            while ((m = meeting_look(word, seen, reached, patience)) == MT_WAIT) {
                __builtin_amdgcn_s_sleep(1);
                seen = word.look();
            }
            sh.flag = m == MT_GONE;
        }
        __syncthreads();
        gone = __builtin_amdgcn_readfirstlane(sh.flag);
        return !gone;
    }
    /* A word of a head: of workgroup t's by thread t, after a meeting, and this workgroup's own. */
    __device__ __forceinline__ u64 head_of(int word) const { return peek(part(t) + ST_BINS + 2 * ST_LIST + word); }
    __device__ __forceinline__ void tell(int word, u64 v) const { publish(mine + ST_BINS + 2 * ST_LIST + word, v); }

    /* The last of a row's workgroups to leave clears its word, the last row's of a queue clears the queue. By thread 0;
     * whether it is the last. `alone`: nobody else of the row is there. */
    __device__ __forceinline__ bool leave(bool alone) {
        if (!alone && !meeting_last(RowWord{counter()}.add(MT_LEFT), G)) return false;
        __hip_atomic_store(counter(), 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const int y = row % ST_QUEUES, rows = (s.rows - y + ST_QUEUES - 1) / ST_QUEUES;
        if (__hip_atomic_fetch_add(s.done + y * ST_LINE, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == rows - 1) {
            __hip_atomic_store(s.tickets + y * ST_LINE, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(s.done + y * ST_LINE, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        return true;
    }
};

/* Values that the compiler takes as new: what an earlier step made of them is not kept in registers for a later one. */
template <typename V, int E>
__device__ __forceinline__ void anew(V (&v)[E]) {
#pragma unroll
    for (int e = 0; e < E; e++) asm volatile("" : "+v"(v[e]));
}

/* This thread's tokens; those not allowed and those past the row's end are -inf. */
template <int E>
__device__ __forceinline__ void split_load(const Split<E> &q, const SampleArgs &a, long long r, float (&x)[E]) {
    const char *p = (const char *)a.logits + r * a.stride * (a.bf16 ? 2 : 4);
    uint32_t allowed = (1u << E) - 1;
    if (a.mask) {
        allowed = 0;
        const uint32_t *mask = a.mask + r * a.mask_stride;
        const int words = (a.vocab + 31) >> 5;
#pragma unroll
        for (int c = 0; c < E / 4; c++) {
            const int i = q.first + c * ST_STEP;
            allowed |= (mask[min(i >> 5, words - 1)] >> (i & 31) & 0xFu) << (4 * c);
        }
    }
    if (a.wide && (q.g + 1) * E * ST_THREADS <= a.vocab) {
        if (a.bf16) {
            uint2 u[E / 4];
#pragma unroll
            for (int c = 0; c < E / 4; c++) u[c] = *reinterpret_cast<const uint2 *>(p + 2LL * (q.first + c * ST_STEP));
#pragma unroll
            for (int c = 0; c < E / 4; c++) {
                x[4 * c] = __uint_as_float(u[c].x << 16); x[4 * c + 1] = __uint_as_float(u[c].x & 0xFFFF0000u);
                x[4 * c + 2] = __uint_as_float(u[c].y << 16); x[4 * c + 3] = __uint_as_float(u[c].y & 0xFFFF0000u);
            }
        } else {
#pragma unroll
            for (int c = 0; c < E / 4; c++) {
                const float4 u = *reinterpret_cast<const float4 *>(p + 4LL * (q.first + c * ST_STEP));
                x[4 * c] = u.x; x[4 * c + 1] = u.y; x[4 * c + 2] = u.z; x[4 * c + 3] = u.w;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) {   /* past the end: the last token's, dropped below */
            const int i = min(q.index(e), a.vocab - 1);
            x[e] = a.bf16 ? bf16_to_f32(reinterpret_cast<const uint16_t *>(p)[i]) : reinterpret_cast<const float *>(p)[i];
        }
#pragma unroll
        for (int e = 0; e < E; e++) allowed &= ~((uint32_t)(q.index(e) >= a.vocab) << e);
    }
#pragma unroll
    for (int e = 0; e < E; e++)   /* NaN fails the comparison; -0 becomes +0, its equal */
        x[e] = (allowed >> e & 1) && x[e] > -INFINITY ? x[e] + 0.0f : -INFINITY;
}

/* The `want` largest of the n codes of sh.cand, in order, in sh.top; returns how many. Every one of THREADS threads must call
 * it, after a __syncthreads. */
template <int THREADS, typename Shared>
__device__ __forceinline__ int sort_codes(Shared &sh, int n, int want) {
    const int t = threadIdx.x;
    if (n <= THREADS) {   /* a code's comparisons spread over THREADS / n threads */
        int lanes = 1;
        while (lanes < n) lanes <<= 1;
        sh.rank[t] = 0;
        __syncthreads();
        const int i = t & (lanes - 1);
        if (i < n) {
            const u64 c = sh.cand[i];
            int above = 0;
#pragma unroll 4
            for (int j = t / lanes; j < n; j += THREADS / lanes) above += sh.cand[j] > c;
            __hip_atomic_fetch_add(&sh.rank[i], above, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
        __syncthreads();
        if (t < n && sh.rank[t] < want) sh.top[sh.rank[t]] = sh.cand[t];
    } else {
        for (int i = t; i < n; i += THREADS) {
            const u64 c = sh.cand[i];
            int above = 0;
            for (int j = 0; j < n && above < want; j++) above += sh.cand[j] > c;
            if (above < want) sh.top[above] = c;
        }
    }
    __syncthreads();
    return min(n, want);
}

/* By one wave: a code that k of the 256 maxima of sh.most reach (0: a group without a token), by bisection k to k + 8 of
 * them, but at most ST_TOP; 1 if fewer than k groups have a token. */
template <typename Shared>
__device__ __forceinline__ u64 least_of_top(const Shared &sh, int lane, int k) {
    u64 m[4], hi = 0, none = ~0ull;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        m[j] = sh.most[j * WAVE + lane];
        hi = max(hi, m[j]);
        none = min(none, m[j] - 1);   /* a group without a token: the largest */
    }
    const auto reach = [&](u64 code) {
        int n = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) n += __popcll(__ballot(m[j] >= code));
        return n;
    };
    hi = lane_max64(hi);
    const int most = min(k + 8, ST_TOP);
    u64 lo = ~lane_max64(~none) + 1;   /* the least of the maxima */
    if (lo == 0 || reach(lo) < k) lo = 1;
    for (int n = reach(lo); n > most && lo < hi;) {
        const u64 mid = lo + (hi - lo + 1) / 2;
        const int of = reach(mid);
        if (of >= k) {
            lo = mid;
            n = of;
        } else {
            hi = mid - 1;
        }
    }
    return lo;
}

/* The choice among the n <= ST_TOP tokens of sh.top, in order of value: top-p, min-p, then the first in index order at which
 * the running weight reaches its goal. Every thread must call it, after a __syncthreads. */
template <typename Shared, typename Weight, typename Goal, typename Choice>
__device__ __forceinline__ void choose_top(Shared &sh, int n, Weight weight, bool nucleus, Goal mass_goal, u64 least_w,
                                           Choice choice, int32_t *out) {
    const int t = threadIdx.x;
    if (t < n) sh.top_w[t] = weight(key_value((uint32_t)(sh.top[t] >> 32)));
    __syncthreads();
    if (t < n) {
        const u64 c = sh.top[t];
        u64 more = 0, total = 0;
        for (int j = 0; j < n; j++) {
            const u64 w = sh.top_w[j];
            more += sh.top[j] >> 32 > c >> 32 ? w : 0;
            total += w;
        }
        const u64 w = sh.top_w[t];
        sh.kept_w[t] = w >= least_w && (!nucleus || more < mass_goal(total)) ? w : 0;
    }
    __syncthreads();
    if (t < n) {
        const int idx = code_index(sh.top[t]);
        u64 before = 0, total = 0;
        for (int j = 0; j < n; j++) {
            const u64 w = sh.kept_w[j];
            before += code_index(sh.top[j]) < idx ? w : 0;
            total += w;
        }
        const u64 goal = choice(total);
        if (before < goal && goal <= before + sh.kept_w[t]) *out = idx;
    }
}

/* Adds `v` to the candidates if `take`. */
template <int E>
__device__ __forceinline__ void split_collect(SplitShared<E> &sh, u64 v, bool take) {
    if (take) sh.cand[__hip_atomic_fetch_add(&sh.n, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)] = v;
}

/* The k <= ST_TOP largest of this slice, in order, in sh.top; returns how many. A code that k of the maxima of 256 groups of
 * 2 E tokens reach is a lower bound of the k-th largest: only the tokens that reach it (in random order about 51 for k = 50,
 * 177 for 128) are compared pairwise. */
template <int E>
__device__ __forceinline__ int split_top(const Split<E> &q, float (&x)[E], int k) {
    SplitShared<E> &sh = q.sh;
    const int t = q.t;
    u64 best = 0;
#pragma unroll
    for (int e = 0; e < E; e++) best = max(best, token_code(x[e], q.index(e)));
    best = max(best, (u64)__shfl_xor(best, 1, WAVE));
    if (k == 1) {
        best = lane_max64(best);
        if (q.lane == 0) sh.sum[q.wave] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < ST_WAVES; w++) best = max(best, sh.sum[w]);
        if (t == 0) sh.top[0] = best;
        __syncthreads();
        return best != 0;
    }
    if (t == 0) sh.n = 0;
    if ((t & 1) == 0) sh.most[t >> 1] = best;
    __syncthreads();
    if (q.wave == 0) {
        const u64 least = least_of_top(sh, q.lane, k);
        if (q.lane == 0) sh.least_code = least;
    }
    __syncthreads();
    const u64 least = sh.least_code;
    anew(x);
    int count = 0;
#pragma unroll
    for (int e = 0; e < E; e++) count += token_code(x[e], q.index(e)) >= least;
    int at = reserve(&sh.n, count, q.lane);
    if (count) {
#pragma unroll
        for (int e = 0; e < E; e++) {
            const u64 c = token_code(x[e], q.index(e));
            if (c >= least) sh.cand[at++] = c;
        }
    }
    __syncthreads();
    return sort_codes<ST_THREADS>(sh, alike(sh.n), k);
}

/* The smallest of this slice's tokens, in index order, whose running sum of m(e), over the elements of the set `in`, reaches
 * `goal`, which its total does. Every thread must call it. */
template <int E, typename M>
__device__ __forceinline__ int split_pick(const Split<E> &q, uint32_t in, M m, u64 goal) {
    SplitShared<E> &sh = q.sh;
    u64 own[E / 4], scan[E / 4];
    asm volatile("" : "+v"(in));
#pragma unroll
    for (int c = 0; c < E / 4; c++) {
        own[c] = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) own[c] += in >> (4 * c + j) & 1 ? m(4 * c + j) : 0;
        scan[c] = lane_scan64(own[c]);
        if (q.lane == WAVE - 1) sh.sum[c * ST_WAVES + q.wave] = scan[c];
        __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    const u64 part = q.lane < E / 4 * ST_WAVES ? sh.sum[q.lane] : 0, upto = lane_scan64(part) - part;
#pragma unroll
    for (int c = 0; c < E / 4; c++) {
        u64 before = lane64(upto, c * ST_WAVES + q.wave) + scan[c] - own[c];
        if (before < goal && goal <= before + own[c]) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const u64 v = in >> (4 * c + j) & 1 ? m(4 * c + j) : 0;
                if (before < goal && goal <= before + v) sh.token = q.index(4 * c + j);
                before += v;
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    return sh.token;
}

/* Over the slices of a row: where the running sum of m(e), over the elements of the sets `live`, the larger value
 * first, reaches target(total). Ranges of values are narrowed by histograms, which the workgroups publish and each adds up,
 * until the tokens of the one that holds the cut fit a list, which each settles pairwise. Between two histograms, and between
 * two lists, there is always a meeting after the first is read. sh.kept: per slice the weight of the tokens down to the cut
 * that weigh least_w or more (not SPLIT). Every thread of every workgroup of the row calls it, and looks at q.gone after it. */
template <bool SPLIT, int E, typename Target>
__device__ __forceinline__ Cut split_cut(Split<E> &q, float (&x)[E], uint32_t live, float zmax, float range, u64 least_w,
                                         Target target) {
    SplitShared<E> &sh = q.sh;
    const int lane = q.lane, wave = q.wave, G = q.G;
    int t = q.t;
    u64 *base_part = q.part(0);
    const auto m = [&](int e) { return SPLIT ? 1ull : sh.weight[e * ST_THREADS + t]; };
    const float scale = range > 0.0f && range < INFINITY ? (ST_BINS - 1) / range : 0.0f;
    /* a range whose products are NaN or past the last bin: the last bin; monotone in z in every case */
    const auto bin_of = [&](float z) { return z == zmax ? 0 : (int)fminf((zmax - z) * scale, (float)(ST_BINS - 1)); };
    u64 goal = 0, base = 0;
    /* once a range of values is split again: by its keys, or its tokens' codes where equals are told apart */
    u64 lo = 0, hi = ~0ull;
    const auto key = [&](int e) { return SPLIT ? token_code(x[e], q.index(e)) : (u64)order_key(x[e]); };
    int keyed = 0;
    u64 base_above = 0;
    for (;;) {
        /* one body for the first level and the others, and no address or set kept in registers from one to the next */
        asm volatile("" : "+s"(keyed), "+s"(base_part), "+v"(t), "+v"(q.first), "+v"(live));
        const auto part = [&](int o) { return base_part + (long long)o * ST_PART; };
        const auto listed = [&](u64 code) {   /* what a token of this slice counts */
            const int i = code_index(code) - q.g * E * ST_THREADS;
            return SPLIT ? 1ull : sh.weight[(i / ST_STEP * 4 + i % 4) * ST_THREADS + i % ST_STEP / 4];
        };
        const auto head_of = [&](int word) { return peek(part(lane) + ST_BINS + 2 * ST_LIST + word); };
        const auto tell = [&](int word, u64 v) { publish(part(q.g) + ST_BINS + 2 * ST_LIST + word, v); };
        int shift = 0;
        if (keyed)
            while ((hi - lo) >> shift >= ST_BINS) shift++;
        anew(x);
        __syncthreads();
        sh.hist[t] = sh.hist[t + ST_THREADS] = 0;
        if (t == 0) {
            sh.n = 0;
            sh.least_code = ~0ull;
            sh.lo = ~0ull;
            sh.hi = 0;
        }
        __syncthreads();
        u64 rest_of = 0, w4[4];
        uint32_t bins[E / 2];   /* two elements' a register; ST_BINS: not live */
#pragma unroll
        for (int e = 0; e < E; e++) {
            int b = keyed ? (int)min((hi - key(e)) >> shift, (u64)ST_BINS) : bin_of(x[e]);
            b = live >> e & 1 ? b : ST_BINS;
            bins[e / 2] = e & 1 ? bins[e / 2] | (uint32_t)b << 16 : (uint32_t)b;
            if (e % 4 == 0) {   /* four weights' loads in flight */
#pragma unroll
                for (int k = 0; k < 4; k++) w4[k] = m(e + k);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (b < ST_BINS - 1)
                __hip_atomic_fetch_add(&sh.hist[b], w4[e % 4], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            rest_of += b == ST_BINS - 1 ? w4[e % 4] : 0;   /* many may be past the range: one addition a wave */
            if (e & 1) asm volatile("" : "+v"(bins[e / 2]), "+v"(rest_of));
        }
        rest_of = lane_sum64(rest_of);
        if (lane == 0 && rest_of)
            __hip_atomic_fetch_add(&sh.hist[ST_BINS - 1], rest_of, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        __syncthreads();
        u64 v[2] = {sh.hist[2 * t], sh.hist[2 * t + 1]};
        if (G > 1) {
            publish(part(q.g) + 2 * t, v[0]);
            publish(part(q.g) + 2 * t + 1, v[1]);
            if (!q.meet()) return Cut{false, 0u, 0};
            v[0] = v[1] = 0;
            for (int o = 0; o < G; o += 8) {   /* eight workgroups' loads in flight */
                u64 other[8][2];
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const u64 *p = part(min(o + k, G - 1)) + 2 * t;
                    other[k][0] = peek(p);
                    other[k][1] = peek(p + 1);
                }
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    v[0] += o + k < G ? other[k][0] : 0;
                    v[1] += o + k < G ? other[k][1] : 0;
                }
            }
        }
        const u64 scan = lane_scan64(v[0] + v[1]);
        if (lane == WAVE - 1) sh.sum[wave] = scan;
        __syncthreads();
        u64 before = scan - v[0] - v[1], total = 0;
#pragma unroll
        for (int o = 0; o < ST_WAVES; o++) {
            before += o < wave ? sh.sum[o] : 0;
            total += sh.sum[o];
        }
        if (!keyed) {
            goal = target(total);
            if (alike((int)(goal > total))) {
                q.meet();   /* the histograms are published over by the next cut: not before everyone has read these */
                return Cut{false, 0u, 0};   /* or the row was given up */
            }
        }
        const u64 rest = goal - base;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            if (before < rest && rest <= before + v[k]) {
                sh.bin = 2 * t + k;
                sh.found = before;
            }
            before += v[k];
        }
        __syncthreads();
        const int bin = alike(sh.bin);
        base += sh.found;

        anew(x);
        asm volatile("" : "+v"(t), "+v"(live), "+v"(q.first));
        u64 above = 0;
        u64 least = ~0ull, most = 0;
        const auto slot = [&](int e) { return (int)(bins[e / 2] >> (e & 1) * 16 & 0xFFFFu); };
        live = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int b = slot(e);
            live |= (uint32_t)(b == bin) << e;
            if (!SPLIT) {   /* on top of the levels' before */
                const u64 v = m(e);
                base_above += b < bin && v >= least_w ? v : 0;
            }
            if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("" : "+v"(base_above));
        above = base_above;
        const int count = __popc(live);
        int at = reserve(&sh.n, count, lane);
        if (count) {
#pragma unroll
            for (int e = 0; e < E; e++) {
                if (live >> e & 1) {
                    const u64 k = key(e);
                    if (at < ST_LIST) sh.code[at] = token_code(x[e], q.index(e));
                    at++;
                    least = min(least, k);
                    most = max(most, k);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        asm volatile("" : "+v"(live));
        if (most) {
            __hip_atomic_fetch_min(&sh.lo, least, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            __hip_atomic_fetch_max(&sh.hi, most, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
        if (!SPLIT) {
            above = lane_sum64(above);
            if (lane == 0) sh.sum[wave] = above;
        }
        __syncthreads();
        int n = alike(sh.n);
        if (!SPLIT) {
            above = 0;
#pragma unroll
            for (int v = 0; v < ST_WAVES; v++) above += sh.sum[v];
        }
        if (G > 1) {
            if (t < min(n, ST_LIST)) {
                publish(part(q.g) + ST_BINS + t, sh.code[t]);
                publish(part(q.g) + ST_BINS + ST_LIST + t, listed(sh.code[t]));
            }
            if (t == 0) {
                tell(HD_COUNT, (u64)n);
                tell(HD_ABOVE, above);
                tell(HD_LEAST, sh.lo);
                tell(HD_MOST, sh.hi);
            }
            if (!q.meet()) return Cut{false, 0u, 0};
            if (wave == 0) {
                int count = 0;
                u64 l = ~0ull, h = 0;
                if (lane < G) {
                    count = (int)head_of(HD_COUNT);
                    l = head_of(HD_LEAST);
                    h = head_of(HD_MOST);
                    sh.kept[lane] = head_of(HD_ABOVE);
                    sh.head[lane] = (u64)count;
                }
                int end = count;
#pragma unroll
                for (int o = 1; o < WAVE; o <<= 1) {
                    const int up = __shfl_up(end, o, WAVE);
                    if (lane >= o) end += up;
                }
                l = ~lane_max64(~l);
                h = lane_max64(h);
                if (lane < G) sh.start[lane + 1] = end;
                if (lane == 0) {
                    sh.start[0] = 0;
                    sh.lo = l;
                    sh.hi = h;
                }
            }
            __syncthreads();
            n = alike(sh.start[G]);
            if (n <= ST_LIST) {
                if (t < n) {   /* entry t: of the last workgroup that starts at or before it */
                    int o = 0;
#pragma unroll
                    for (int k = ST_MAX_GROUPS / 2; k; k >>= 1)
                        if (o + k < G && sh.start[o + k] <= t) o += k;
                    const u64 *entry = part(o) + ST_BINS + t - sh.start[o];
                    const u64 code = peek(entry), of = peek(entry + ST_LIST);
                    sh.code[t] = code;
                    sh.w[t] = of;
                }
            }
        } else {
            if (t < min(n, ST_LIST)) sh.w[t] = listed(sh.code[t]);
            if (t == 0) {
                sh.kept[0] = above;
                sh.head[0] = (u64)n;
                sh.start[0] = 0;
                sh.start[1] = n;
            }
        }
        __syncthreads();
        lo = alike(sh.lo);
        hi = alike(sh.hi);
        keyed = 1;
        if (n <= ST_LIST) {
            if (t < ST_LIST) sh.above[t] = 0;
            __syncthreads();
            int lanes = 1;
            while (lanes < n) lanes <<= 1;
            const int i = t & (lanes - 1);
            if (i < n) {
                const u64 c = sh.code[i];
                u64 more = 0;
#pragma unroll 4
                for (int j = t / lanes; j < n; j += ST_THREADS / lanes)
                    more += (SPLIT ? sh.code[j] > c : (uint32_t)(sh.code[j] >> 32) > (uint32_t)(c >> 32)) ? sh.w[j] : 0;
                __hip_atomic_fetch_add(&sh.above[i], more, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            }
            __syncthreads();
            if (t < n) {
                const bool in = base + sh.above[t] < goal;
                if (in) __hip_atomic_fetch_min(&sh.least_code, sh.code[t], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                if (!SPLIT && in && sh.w[t] >= least_w)
                    __hip_atomic_fetch_add(&sh.kept[code_index(sh.code[t]) / (E * ST_THREADS)], sh.w[t], __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_WORKGROUP);
            }
            __syncthreads();
            const u64 last = sh.least_code;
            return Cut{true, (uint32_t)(last >> 32), SPLIT ? code_index(last) : 0x7FFFFFFF};
        }
        if (!SPLIT && lo == hi) {   /* one value */
            if (t < G && sh.head[t]) {
                const u64 of = G > 1 ? peek(part(t) + ST_BINS + ST_LIST) : sh.w[0];   /* every one's weight */
                if (of >= least_w) sh.kept[t] += sh.head[t] * of;
            }
            __syncthreads();
            return Cut{true, (uint32_t)lo, 0x7FFFFFFF};
        }
    }
}

/* This workgroup's part of its row. Returns whether it is still to leave the row; q.gone: the row was given up, and has no
 * token. */
template <int E>
__device__ __forceinline__ bool split_row(Split<E> &q) {
    SplitShared<E> &sh = q.sh;
    const SampleArgs &a = q.s.a;
    q.first = q.g * E * ST_THREADS + 4 * q.t;
    q.reached = q.gone = 0;
    q.mine = q.part(q.g);
    const int t = q.t, lane = q.lane, wave = q.wave, G = q.G;
    const long long r = q.row;
    float x[E];
    split_load(q, a, r, x);
    const float T = alike(a.temperature[r]);
    const bool greedy = !(T > 0.0f);
    const int k = greedy ? 1 : a.top_k ? alike(a.top_k[r]) : 0;
    Choice with(a, r, T, 0.0f);
    const auto weight = [&](float z) { return with.weight(z); };
    const auto mass_goal = [&](u64 total) { return with.mass(total); };
    const auto choice = [&](u64 total) { return with.choice(total); };

    if (k > 0 && k <= ST_TOP) {
        __syncthreads();   /* sh.n held the ticket */
        int n = alike(split_top(q, x, k));
        if (G > 1) {
            if (t < n) publish(q.mine + ST_BINS + t, sh.top[t]);
            if (t == 0) q.tell(HD_COUNT, (u64)n);
            q.arrive();
            if (t == 0) {
                sh.flag = __hip_atomic_fetch_add(q.counter(), 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == G - 1;
                sh.n = 0;
            }
            __syncthreads();
            if (!alike(sh.flag)) return false;
            /* every list's ceil(k / G)-th: k tokens reach the least of them */
            const int quota = (k + G - 1) / G;
            if (wave == 0) {
                u64 least = ~0ull;
                if (lane < G) {
                    const int count = (int)q.head_of(HD_COUNT);
                    sh.head[lane] = (u64)count;
                    least = count >= quota ? peek(q.part(lane) + ST_BINS + quota - 1) : 1ull;
                }
#pragma unroll
                for (int o = 1; o < WAVE; o <<= 1) least = min(least, (u64)__shfl_xor(least, o, WAVE));
                if (lane == 0) sh.least_code = least;
            }
            __syncthreads();
            const u64 least = sh.least_code;
            for (int o = wave; o < G; o += ST_WAVES)
                for (int i = lane; i < (int)sh.head[o]; i += WAVE) {
                    const u64 c = peek(q.part(o) + ST_BINS + i);
                    split_collect(sh, c, c >= least);
                }
            __syncthreads();
            n = alike(sort_codes<ST_THREADS>(sh, alike(sh.n), k));
            if (t == 0) q.leave(true);
        }
        if (n == 0 || k == 1) {
            if (t == 0) a.out[r] = n == 0 ? -1 : code_index(sh.top[0]);
            return false;
        }
        with.zmax = key_value((uint32_t)(sh.top[0] >> 32));
        choose_top(sh, n, weight, with.p < 1.0f, mass_goal, with.least_w, choice, a.out + r);
        return false;
    }

    /* the largest allowed logit and the smallest */
    float most = -INFINITY, least = INFINITY;
#pragma unroll
    for (int e = 0; e < E; e++) {
        most = fmaxf(most, x[e]);
        least = fminf(least, x[e] > -INFINITY ? x[e] : INFINITY);
    }
    for (int round = 0; round < (G > 1 ? 2 : 1); round++) {
        if (round) {
            if (t == 0) q.tell(HD_BEST, (u64)__float_as_uint(most) << 32 | __float_as_uint(least));
            if (!q.meet()) return true;
            if (t < G) {
                const u64 of = q.head_of(HD_BEST);
                most = __uint_as_float((uint32_t)(of >> 32));
                least = __uint_as_float((uint32_t)of);
            }
        }
        most = lane_max(most);
        least = -lane_max(-least);
        if (lane == 0) sh.sum[wave] = (u64)__float_as_uint(most) << 32 | __float_as_uint(least);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < ST_WAVES; w++) {
            most = fmaxf(most, __uint_as_float((uint32_t)(sh.sum[w] >> 32)));
            least = fminf(least, __uint_as_float((uint32_t)sh.sum[w]));
        }
        __syncthreads();
    }
    most = alike(most);
    least = alike(least);
    if (most == -INFINITY) {
        if (t == 0 && q.g == 0) a.out[r] = -1;
        return true;
    }
    with.zmax = most;
    anew(x);

    if (k > 0 && k < a.vocab) {
        uint32_t live = 0;
#pragma unroll
        for (int e = 0; e < E; e++) live |= (uint32_t)(x[e] > -INFINITY) << e;
        const Cut top = split_cut<true>(q, x, live, with.zmax, with.zmax - least, 0ull,
                                        [&](u64) { return (u64)k; });
        if (q.gone) return true;
        if (top.some) {
            const float z = key_value(top.key);
#pragma unroll
            for (int e = 0; e < E; e++)   /* past the k largest: dropped */
                if (!(x[e] > z || (x[e] == z && q.index(e) <= top.idx))) x[e] = -INFINITY;
        }
    }
    anew(x);
    uint32_t live = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const u64 v = weight(x[e]);
        sh.weight[e * ST_THREADS + t] = v;   /* read by this thread alone */
        live |= (uint32_t)(v != 0) << e;
        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);   /* four at a time: more would need more registers */
    }
    float least_z = -INFINITY;   /* the nucleus' smallest logit */
    if (with.p < 1.0f) {
        const Cut mass = split_cut<false>(q, x, live, with.zmax, fminf(with.zmax - least, with.range(a.vocab)), with.least_w,
                                          mass_goal);
        if (q.gone) return true;
        if (mass.some) least_z = key_value(mass.key);
    } else {
        u64 own = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const u64 v = sh.weight[e * ST_THREADS + t];
            own += v >= with.least_w ? v : 0;
        }
        own = lane_sum64(own);
        if (lane == 0) sh.sum[wave] = own;
        __syncthreads();
        if (t == 0) {
            own = 0;
#pragma unroll
            for (int v = 0; v < ST_WAVES; v++) own += sh.sum[v];
            if (G > 1) q.tell(HD_SUM, own);
            else sh.kept[0] = own;
        }
        if (!q.meet()) return true;
        if (G > 1) {
            if (t < G) sh.kept[t] = q.head_of(HD_SUM);
            __syncthreads();
        }
    }
    u64 total = 0, before = 0;
    for (int o = 0; o < G; o++) {
        before += o < q.g ? sh.kept[o] : 0;
        total += sh.kept[o];
    }
    const u64 goal = choice(total), ours = sh.kept[q.g];
    __syncthreads();
    if (alike((int)(before < goal && goal <= before + ours))) {
        uint32_t kept = 0;
#pragma unroll
        for (int e = 0; e < E; e++) kept |= (uint32_t)(x[e] >= least_z && sh.weight[e * ST_THREADS + t] >= with.least_w) << e;
        const int token = split_pick(q, kept, [&](int e) { return sh.weight[e * ST_THREADS + t]; }, goal - before);
        if (t == 0) a.out[r] = token;
    }
    return true;
}

/* --- Rows by one workgroup each, read again for every step: where rows are many, or longer than the slices allow. Wave w
 * takes a contiguous run of the row, so that a sum in index order is a sum over waves, then over one wave. */

constexpr int RW_WAVES = 16, RW_THREADS = RW_WAVES * WAVE;   /* of row_kernel; W: of whoever takes a row */
constexpr int RW_CHUNK = 4 * WAVE;       /* elements of a wave's chunk: four a lane */

template <int W>
struct RowShared {
    static constexpr int THREADS = W * WAVE;
    static constexpr int BINS = 4 * THREADS;
    static constexpr int LIST = THREADS / 2;   /* tokens a range may hold to be settled pairwise */
    union {
        u64 hist[BINS];
        u64 cand[ST_CAND];
    };
    u64 top[ST_TOP], top_w[ST_TOP], kept_w[ST_TOP], most[256];
    int rank[THREADS];
    u64 code[LIST], w[LIST];
    u64 sum[W];
    u64 found, least_code, lo, hi;
    int bin, n, token;
};
static_assert(sizeof(RowShared<ST_WAVES>) <= sizeof(SplitShared<ST_MAX_E / 2>), "a row that was given up fits");

/* Element j of lane l of chunk c of wave w is index (w per + c) RW_CHUNK + 4 l + j. */
template <int AHEAD, int W>   /* chunks in flight, waves */
struct Row {
    const SampleArgs &a;
    const char *p;
    const uint32_t *mask;
    int per, base, lane;

    __device__ __forceinline__ Row(const SampleArgs &args, long long row)
        : a(args), p((const char *)args.logits + row * args.stride * (args.bf16 ? 2 : 4)),
          mask(args.mask ? args.mask + row * args.mask_stride : nullptr) {
        per = (a.vocab + W * RW_CHUNK - 1) / (W * RW_CHUNK);
        lane = threadIdx.x & (WAVE - 1);
        base = alike((int)(threadIdx.x >> 6)) * per * RW_CHUNK;
    }

    __device__ __forceinline__ int index(int c, int j) const { return base + c * RW_CHUNK + 4 * lane + j; }

    /* Chunks c .. c + AHEAD - 1. Elements that are not allowed, those past the row's end and those of the next wave are -inf. */
    __device__ __forceinline__ void fetch(int c, float (&x)[4 * AHEAD]) const {
        constexpr uint32_t all = (1u << 4 * AHEAD) - 1;
        uint32_t allowed = all;
        if (mask) {
            allowed = 0;
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
                const int i = min(index(c + k, 0), a.vocab - 1) & ~3;
                allowed |= (mask[i >> 5] >> (i & 31) & 0xFu) << (4 * k);
            }
        }
        if (a.wide && c + AHEAD <= per && base + (c + AHEAD) * RW_CHUNK <= a.vocab) {
            if (a.bf16) {
                uint2 u[AHEAD];
#pragma unroll
                for (int k = 0; k < AHEAD; k++) u[k] = *reinterpret_cast<const uint2 *>(p + 2LL * index(c + k, 0));
#pragma unroll
                for (int k = 0; k < AHEAD; k++) {
                    x[4 * k] = __uint_as_float(u[k].x << 16); x[4 * k + 1] = __uint_as_float(u[k].x & 0xFFFF0000u);
                    x[4 * k + 2] = __uint_as_float(u[k].y << 16); x[4 * k + 3] = __uint_as_float(u[k].y & 0xFFFF0000u);
                }
            } else {
#pragma unroll
                for (int k = 0; k < AHEAD; k++) {
                    const float4 u = *reinterpret_cast<const float4 *>(p + 4LL * index(c + k, 0));
                    x[4 * k] = u.x; x[4 * k + 1] = u.y; x[4 * k + 2] = u.z; x[4 * k + 3] = u.w;
                }
            }
        } else {
            const int end = min(base + per * RW_CHUNK, a.vocab);
#pragma unroll
            for (int e = 0; e < 4 * AHEAD; e++) {
                const int i = index(c + e / 4, e % 4), at = min(i, a.vocab - 1);
                x[e] = a.bf16 ? bf16_to_f32(reinterpret_cast<const uint16_t *>(p)[at]) : reinterpret_cast<const float *>(p)[at];
                allowed &= ~((uint32_t)(i >= end) << e);
            }
        }
        if (allowed != all)
#pragma unroll
            for (int e = 0; e < 4 * AHEAD; e++)   /* not allowed: NaN */
                x[e] = __int_as_float(__float_as_int(x[e]) | ~((int)(allowed << (31 - e)) >> 31));
#pragma unroll
        for (int e = 0; e < 4 * AHEAD; e++)   /* NaN fails the comparison; -0 becomes +0, its equal */
            x[e] = (x[e] > -INFINITY ? x[e] : -INFINITY) + 0.0f;
    }

    /* f(value, index) for every element of this wave. */
    template <typename F>
    __device__ __forceinline__ void each(F &&f) const {
        for (int c = 0; c < per; c += AHEAD) {
            float x[4 * AHEAD];
            fetch(c, x);
#pragma unroll
            for (int e = 0; e < 4 * AHEAD; e++) f(x[e], index(c + e / 4, e % 4));
        }
    }
};

/* The bins' sums in order: sh.bin is the first bin at which the running sum reaches target(total), sh.found the sum
 * before it. Returns whether there is one. Every thread must call it. */
template <int W, typename Target>
__device__ __forceinline__ bool row_bin(RowShared<W> &sh, Target target) {
    const int t = threadIdx.x, lane = t & (WAVE - 1), wave = t >> 6;
    u64 v[4], own = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; k++) {
        v[k] = sh.hist[4 * t + k];
        own += v[k];
    }
    const u64 scan = lane_scan64(own);
    if (lane == WAVE - 1) sh.sum[wave] = scan;
    __syncthreads();
    u64 before = scan - own, total = 0;
#pragma unroll
    for (int w = 0; w < W; w++) {
        before += w < wave ? sh.sum[w] : 0;
        total += sh.sum[w];
    }
    const u64 goal = target(total);
    if (before < goal && goal <= before + own) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (before < goal && goal <= before + v[k]) {
                sh.bin = 4 * t + k;
                sh.found = before;
            }
            before += v[k];
        }
    }
    __syncthreads();
    return alike((int)(goal <= total));
}

/* Over the elements that in(z, index) keeps, in order of value, the larger first: where the running sum of m(z) reaches
 * target(total). SPLIT: equals are taken one by one, the lower index first (m is 1), and the cut's idx is the last one
 * taken; else they are taken together. `range`: the values below zmax - range need no telling apart. Every thread must
 * call it. */
template <bool SPLIT, int AHEAD, int W, typename In, typename M, typename Target>
__device__ __forceinline__ Cut row_cut(RowShared<W> &sh, const Row<AHEAD, W> &row, float zmax, float range, In in, M m,
                                       Target target) {
    constexpr int THREADS = RowShared<W>::THREADS, BINS = RowShared<W>::BINS, LIST = RowShared<W>::LIST;
    const int t = threadIdx.x, lane = row.lane;
    const float scale = range > 0.0f && range < INFINITY ? (BINS - 1) / range : 0.0f;
    /* a range whose products are NaN or past the last bin: the last bin; monotone in z in every case */
    const auto bin_of = [&](float z) { return z == zmax ? 0 : (int)fminf((zmax - z) * scale, (float)(BINS - 1)); };
    const auto key = [&](float z, int i) { return SPLIT ? token_code(z, i) : (u64)order_key(z); };
    const auto clear = [&]() {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; k++) sh.hist[t + k * THREADS] = 0;
        if (t == 0) {
            sh.n = 0;
            sh.least_code = sh.lo = ~0ull;
            sh.hi = 0;
        }
        __syncthreads();
    };
    u64 goal = 0;
    clear();
    u64 rest = 0;   /* of the last bin: many may be past the range */
    row.each([&](float z, int i) {
        const u64 w = in(z, i) ? m(z) : 0;
        const int b = bin_of(z);
        if (b < BINS - 1)
            __hip_atomic_fetch_add(&sh.hist[b], w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        rest += b == BINS - 1 ? w : 0;
    });
    rest = lane_sum64(rest);
    if (lane == 0) __hip_atomic_fetch_add(&sh.hist[BINS - 1], rest, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    if (!row_bin(sh, [&](u64 total) { return goal = target(total); })) return Cut{false, 0u, 0};
    const int bin = alike(sh.bin);
    u64 base = sh.found, lo = 0, hi = ~0ull;   /* once a range of values is split again: its keys */
    bool keyed = false;
    for (;;) {
        const auto member = [&](float z, int i) {
            if (!in(z, i)) return false;
            if (!keyed) return bin_of(z) == bin;
            const u64 k = key(z, i);
            return k >= lo && k <= hi;
        };
        row.each([&](float z, int i) {
            if (member(z, i)) {
                const int at = __hip_atomic_fetch_add(&sh.n, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                if (at < LIST) {
                    sh.code[at] = token_code(z, i);
                    sh.w[at] = m(z);
                }
            }
        });
        __syncthreads();
        const int n = alike(sh.n);
        if (n <= LIST) {   /* pairwise, up to 16 neighbours a token */
            int parts = 16;
            while (parts > 2 && parts * n > THREADS) parts >>= 1;
            const int i = t / parts;
            const u64 c = i < n ? sh.code[i] : ~0ull;
            u64 more = 0;
#pragma unroll 4
            for (int j = t % parts; j < n; j += parts)
                more += (SPLIT ? sh.code[j] > c : (uint32_t)(sh.code[j] >> 32) > (uint32_t)(c >> 32)) ? sh.w[j] : 0;
            for (int o = 1; o < parts; o <<= 1) more += (u64)__shfl_xor(more, o, WAVE);
            /* the cut is the last that less than the goal lies above */
            if (i < n && t % parts == 0 && base + more < goal)
                __hip_atomic_fetch_min(&sh.least_code, c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            __syncthreads();
            const u64 last = sh.least_code;
            return Cut{true, (uint32_t)(last >> 32), SPLIT ? code_index(last) : 0x7FFFFFFF};
        }
        if (!keyed) {   /* the least and largest key of the range */
            u64 least = ~0ull, most = 0;
            row.each([&](float z, int i) {
                if (member(z, i)) {
                    least = min(least, key(z, i));
                    most = max(most, key(z, i));
                }
            });
            least = ~lane_max64(~least);
            most = lane_max64(most);
            if (lane == 0) {
                __hip_atomic_fetch_min(&sh.lo, least, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                __hip_atomic_fetch_max(&sh.hi, most, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            }
            __syncthreads();
            lo = alike(sh.lo);
            hi = alike(sh.hi);
            keyed = true;
        }
        if (!SPLIT && lo == hi) return Cut{true, (uint32_t)lo, 0x7FFFFFFF};   /* one value */
        int shift = 0;
        while ((hi - lo) >> shift >= BINS) shift++;
        clear();
        row.each([&](float z, int i) {   /* the larger keys first */
            if (member(z, i))
                __hip_atomic_fetch_add(&sh.hist[(hi - key(z, i)) >> shift], m(z), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_WORKGROUP);
        });
        const u64 still = goal - base;
        row_bin(sh, [&](u64) { return still; });
        base += sh.found;
        const u64 top = hi - ((u64)alike(sh.bin) << shift), span = (1ull << shift) - 1;
        lo = top - lo > span ? top - span : lo;
        hi = top;
    }
}

/* The first element in index order at which the running sum of m(z, index) reaches goal(total). Every thread must call it. */
template <int AHEAD, int W, typename M, typename Goal>
__device__ __forceinline__ int row_pick(RowShared<W> &sh, const Row<AHEAD, W> &row, M m, Goal goal) {
    const int lane = row.lane, wave = threadIdx.x >> 6;
    u64 s = 0;
    row.each([&](float z, int i) { s += m(z, i); });
    s = lane_sum64(s);
    __syncthreads();
    if (lane == 0) sh.sum[wave] = s;
    __syncthreads();
    u64 before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < W; w++) {
        before += w < wave ? sh.sum[w] : 0;
        total += sh.sum[w];
    }
    const u64 g = goal(total);
    if (alike((int)(before < g && g <= before + s))) {   /* this wave holds it */
        for (int c = 0; c < row.per; c += AHEAD) {
            float x[4 * AHEAD];
            row.fetch(c, x);
            u64 scan[AHEAD];
            bool found = false;
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
                u64 v[4], own = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) own += v[j] = m(x[4 * k + j], row.index(c + k, j));
                scan[k] = lane_scan64(own);
                u64 run = before + scan[k] - own;
                if (run < g && g <= run + own) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if (run < g && g <= run + v[j]) sh.token = row.index(c + k, j);
                        run += v[j];
                    }
                }
                before += lane64(scan[k], WAVE - 1);
                found = found || before >= g;
            }
            if (alike((int)found)) break;
        }
    }
    __syncthreads();
    return sh.token;
}

/* A row's token by W waves of one workgroup. */
template <int AHEAD, int W>
__device__ __forceinline__ void row_choose(const SampleArgs &a, long long r, RowShared<W> &sh) {
    constexpr int THREADS = RowShared<W>::THREADS;
    const int t = threadIdx.x, lane = t & (WAVE - 1), wave = t >> 6;
    const Row<AHEAD, W> row(a, r);

    /* the largest allowed logit (the lowest index among equals) and the smallest */
    float most = -INFINITY, least = INFINITY;
    int at = 0;
    row.each([&](float z, int i) {
        at = z > most ? i : at;
        most = fmaxf(most, z);
        least = fminf(least, z > -INFINITY ? z : INFINITY);
    });
    u64 best = token_code(most, at);
    const u64 own = best;
    best = lane_max64(best);
    least = -lane_max(-least);
    if (lane == 0) {
        sh.sum[wave] = best;
        sh.rank[wave] = __float_as_int(least);
    }
    if (t == 0) sh.n = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; w++) {
        best = max(best, sh.sum[w]);
        least = fminf(least, __int_as_float(sh.rank[w]));
    }
    best = alike(best);
    least = alike(least);
    const float T = alike(a.temperature[r]);
    int k = a.top_k ? alike(a.top_k[r]) : 0;
    if (best == 0 || !(T > 0.0f) || k == 1) {   /* nothing allowed; or the largest logit */
        if (t == 0) a.out[r] = best == 0 ? -1 : code_index(best);
        return;
    }
    const Choice with(a, r, T, key_value((uint32_t)(best >> 32)));

    if (k > 0 && k <= ST_TOP) {
        /* as split_top: the tokens that reach a bound which k of 256 groups of threads reach */
        constexpr int PER = THREADS / 256;
        u64 group = own;
#pragma unroll
        for (int o = 1; o < PER; o <<= 1) group = max(group, (u64)__shfl_xor(group, o, WAVE));
        if (t % PER == 0) sh.most[t / PER] = group;
        __syncthreads();
        if (wave == 0) {
            const u64 bound = least_of_top(sh, lane, k);
            if (lane == 0) sh.least_code = bound;
        }
        __syncthreads();
        const u64 bound = alike(sh.least_code);
        row.each([&](float z, int i) {
            const u64 c = token_code(z, i);
            if (c >= bound) {
                const int slot = __hip_atomic_fetch_add(&sh.n, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                if (slot < ST_CAND) sh.cand[slot] = c;
            }
        });
        __syncthreads();
        const int n = alike(sh.n);
        if (n <= ST_CAND) {   /* more only where the largest tokens crowd in few groups */
            choose_top(sh, sort_codes<THREADS>(sh, n, k), [&](float z) { return with.weight(z); }, with.p < 1.0f,
                       [&](u64 total) { return with.mass(total); }, with.least_w, [&](u64 total) { return with.choice(total); },
                       a.out + r);
            return;
        }
    }

    Cut top = {false, 0u, 0};
    if (k > 0 && k < a.vocab)
        top = row_cut<true>(sh, row, with.zmax, with.zmax - least, [&](float z, int) { return z > -INFINITY; },
                            [&](float) { return 1ull; }, [&](u64) { return (u64)k; });
    const float top_z = top.some ? key_value(top.key) : -INFINITY;
    const auto ranked = [&](float z, int i) {   /* among the k largest */
        return z > top_z || (top.some && z == top_z && i <= top.idx);
    };
    float least_z = -INFINITY;   /* the nucleus' smallest logit */
    if (with.p < 1.0f) {
        const Cut mass = row_cut<false>(sh, row, with.zmax, fminf(with.zmax - least, with.range(a.vocab)), ranked,
                                        [&](float z) { return with.weight(z); }, [&](u64 total) { return with.mass(total); });
        if (mass.some) least_z = key_value(mass.key);
    }
    const int token = row_pick(
        sh, row,
        [&](float z, int i) {
            const u64 w = z >= least_z && ranked(z, i) ? with.weight(z) : 0ull;
            return w >= with.least_w ? w : 0ull;
        },
        [&](u64 total) { return with.choice(total); });
    if (t == 0) a.out[r] = token;
}

/* Two forms, with the same results: four chunks in flight, 93 registers, a workgroup a CU; or two chunks and 64 registers, two
 * workgroups a CU, where there are more rows than CUs: 333 rows of 32,768 tokens with top-p 102 and 85 us, 256 of 65,536 94 and
 * 95, 128 of them with a top-k 23.6 and 25.0. */
template <int AHEAD>
__global__ void __launch_bounds__(RW_THREADS, AHEAD == 4 ? 4 : 8) row_kernel(SampleArgs a) {
    __shared__ RowShared<RW_WAVES> sh;
    row_choose<AHEAD>(a, blockIdx.x, sh);
}

/* split_kernel's arguments, read once more: those that only a row that was given up needs would be kept in scalar registers
 * all along (100 of them spilled, and one row of 65,536 tokens took 23.4 us instead of 21.7). */
__device__ __forceinline__ SampleArgs sample_args_again() {
    const __attribute__((address_space(4))) SplitArgs *p =
        (const __attribute__((address_space(4))) SplitArgs *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    SampleArgs a;
    a.logits = p->a.logits; a.stride = p->a.stride; a.vocab = p->a.vocab; a.bf16 = p->a.bf16; a.wide = p->a.wide;
    a.uniform = p->a.uniform; a.temperature = p->a.temperature; a.top_p = p->a.top_p; a.min_p = p->a.min_p;
    a.top_k = p->a.top_k; a.mask = p->a.mask; a.mask_stride = p->a.mask_stride; a.out = p->a.out;
    return a;
}

/* Rows in slices. A row that was given up is done by the last of its workgroups to leave. */
template <int E>
__global__ void __launch_bounds__(ST_THREADS, 4) split_kernel(SplitArgs s) {
    __shared__ SplitShared<E> sh;
    Split<E> q = {s, sh};
    q.t = threadIdx.x;
    q.lane = q.t & (WAVE - 1);
    q.wave = q.t >> 6;
    q.G = s.groups;
    q.row = blockIdx.x;
    q.g = 0;
    if (q.G > 1) {   /* every eighth workgroup, which one XCD runs, draws on one queue, and a row is one queue's */
        const int y = blockIdx.x % ST_QUEUES, rows = (s.rows - y + ST_QUEUES - 1) / ST_QUEUES;
        if ((int)(blockIdx.x / ST_QUEUES) >= rows * q.G) return;
        if (q.t == 0)
            sh.n = __hip_atomic_fetch_add(s.tickets + y * ST_LINE, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        const int ticket = alike(sh.n);
        q.row = y + ticket / q.G * ST_QUEUES;
        if (q.row >= s.rows) return;   /* counts that were not zero: no access out of bounds */
        q.g = ticket % q.G;
    }
    if (!split_row(q) || q.G == 1) return;
    if (q.t == 0) {
        const bool last = q.leave(false);
        sh.token = last;
    }
    if (!q.gone) return;
    __syncthreads();
    if (!alike(sh.token)) return;
    __syncthreads();   /* sh.token is read; the same LDS serves the whole row */
    row_choose<2>(sample_args_again(), alike(q.row), reinterpret_cast<RowShared<ST_WAVES> &>(sh));
}

}  // namespace nc

using namespace nc;

/* Slices of a row, of e tokens a thread, or 0 for row_kernel: rows too long for slices, or so many that not all slices run at
 * once. A round of slices takes 17 to 37 us whatever the rows ask for, most of it waiting for one another, and row_kernel as
 * long as a row's own work: 128 rows of 65,536 tokens (two rounds of slices) take 35 us in slices and 24 whole with a top-k of
 * 40, 21 and 10 greedily, 75 and 84 with top-p; 256 rows with top-p 142 and 94, and 64 rows (one round) with a top-k 20 and 23.
 * Half slices where one suffices, or where they are at most one a CU and few to a row: one row of 3,000 tokens 15 -> 11 us,
 * 16 rows of 32,768 tokens 25.6 -> 23.5; but two a CU, for 32 rows of 65,536 tokens, took 37 us and whole slices 31. */
static int split_groups(long long rows, int vocab, int &e) {
    const int half = ST_MAX_E / 2 * ST_THREADS, halves = (vocab + half - 1) / half;
    e = halves == 1 || (halves > 2 && halves <= ST_MAX_GROUPS / 2 && rows * halves <= ST_MAX_WORKGROUPS / 2) ? ST_MAX_E / 2
                                                                                                    : ST_MAX_E;
    const int slice = e * ST_THREADS, groups = (vocab + slice - 1) / slice;
    return groups == 1 || (groups <= ST_MAX_GROUPS && rows * groups <= ST_MAX_WORKGROUPS) ? groups : 0;
}

/* The counts come first, in the same place whatever the sizes, so that every call finds them as the one before left them. */
constexpr size_t ST_COUNT_BYTES = (2 * ST_QUEUES + ST_MAX_WORKGROUPS / 2) * ST_LINE * sizeof(int);
static_assert(ST_COUNT_BYTES <= 64 * 1024, "callers zero no more than 64 KiB");

extern "C" size_t nc_sample_workspace_bytes(long long rows, int vocab) {
    if (rows < 0 || rows > 1LL << 22 || vocab <= 0 || vocab > 1 << 24) return 0;
    int e;
    const int groups = split_groups(rows, vocab, e);
    return groups <= 1 ? 16 : ST_COUNT_BYTES + (size_t)rows * groups * ST_PART * sizeof(u64);
}

static int sample_tokens(const void *logits, int is_bf16, long long row_stride, long long rows, int vocab,
                         const float *uniform, const float *temperature, const int32_t *top_k, const float *top_p,
                         const float *min_p, const uint32_t *mask, long long mask_stride, int32_t *tokens, void *workspace,
                         size_t workspace_bytes, int patience, void *stream) {
    if (!logits || !uniform || !temperature || !tokens || !workspace) return NC_ERR_NULL;
    if (rows < 0 || rows > 1LL << 22 || vocab <= 0 || vocab > 1 << 24 || row_stride < vocab ||
        (mask && mask_stride < ((long long)vocab + 31) / 32) || (uintptr_t)workspace % 16 ||
        workspace_bytes < nc_sample_workspace_bytes(rows, vocab))
        return NC_ERR_SHAPE;
    if (rows == 0) return NC_OK;
    SampleArgs a = {};
    a.logits = logits; a.stride = row_stride; a.vocab = vocab; a.bf16 = is_bf16 != 0;
    a.wide = (uintptr_t)logits % (is_bf16 ? 8 : 16) == 0 && (row_stride % 4 == 0 || rows == 1);
    a.uniform = uniform; a.temperature = temperature; a.top_p = top_p; a.min_p = min_p; a.top_k = top_k;
    a.mask = mask; a.mask_stride = mask_stride;
    a.out = tokens;
    int e, groups = split_groups(rows, vocab, e);
    const int cus = device_cus();
    if (groups > 1 && rows * groups > 2 * cus) groups = 0;   /* a device of fewer CUs: slices would give rows up */
    if (groups == 0) {
        hipLaunchKernelGGL(rows > cus ? row_kernel<2> : row_kernel<4>, dim3((unsigned)rows), dim3(RW_THREADS), 0,
                           (hipStream_t)stream, a);
        return (int)hipGetLastError();
    }
    SplitArgs s = {};
    s.a = a;
    s.rows = (int)rows;
    s.groups = groups;
    s.patience = patience;
    s.tickets = (int *)workspace;
    s.done = s.tickets + ST_QUEUES * ST_LINE;
    s.count = s.done + ST_QUEUES * ST_LINE;
    s.part = (u64 *)((char *)workspace + ST_COUNT_BYTES);
    const long long grid = groups == 1 ? rows : (rows + ST_QUEUES - 1) / ST_QUEUES * ST_QUEUES * groups;
    hipLaunchKernelGGL(e == ST_MAX_E ? split_kernel<ST_MAX_E> : split_kernel<ST_MAX_E / 2>, dim3((unsigned)grid), dim3(ST_THREADS), 0, (hipStream_t)stream, s);
    return (int)hipGetLastError();
}

extern "C" int nc_sample_tokens(const void *logits, int is_bf16, long long row_stride, long long rows, int vocab,
                                const float *uniform, const float *temperature, const int32_t *top_k, const float *top_p,
                                const float *min_p, const uint32_t *mask, long long mask_stride, int32_t *tokens,
                                void *workspace, size_t workspace_bytes, void *stream) {
    return sample_tokens(logits, is_bf16, row_stride, rows, vocab, uniform, temperature, top_k, top_p, min_p, mask, mask_stride,
                         tokens, workspace, workspace_bytes, ST_PATIENCE, stream);
}

extern "C" int nc_debug_sample_tokens(const void *logits, int is_bf16, long long row_stride, long long rows, int vocab,
                                      const float *uniform, const float *temperature, const int32_t *top_k,
                                      const float *top_p, const float *min_p, const uint32_t *mask, long long mask_stride,
                                      int32_t *tokens, void *workspace, size_t workspace_bytes, int patience, void *stream) {
    if (patience < 0 || patience > 1 << 16) return NC_ERR_SHAPE;
    return sample_tokens(logits, is_bf16, row_stride, rows, vocab, uniform, temperature, top_k, top_p, min_p, mask, mask_stride,
                         tokens, workspace, workspace_bytes, patience, stream);
}
