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
 * Weights are integers: exp in float64 (2^x by its Taylor polynomial after splitting off the integer part), times 2^S and
 * rounded. Sums of integers depend on no order, so the LDS histograms may be filled by atomics, and the sums of a row are
 * as exact as its weights (2^-47 of the largest at 65,536 tokens): a border between two tokens moves by less than that
 * share. In float32 a border among many small weights would move by about their size.
 *
 * One workgroup of 16 waves takes a row, wave w a contiguous run of it, so that a sum in index order is a sum over waves,
 * then over one wave. No sort: the place where a running count (top-k) or
 * weight (top-p) in order of value reaches its target is found by a histogram over 4,096 ranges of the value, then among
 * the few tokens of the range that holds it, or by finer histograms where it holds many.
 */
#include <math.h>

#include "nc_device.h"
#include "nanochat_amd.h"

namespace nc {

typedef unsigned long long u64;

constexpr int SM_WAVES = 16, SM_THREADS = SM_WAVES * WAVE;
constexpr int SM_CHUNK = 4 * WAVE;       /* elements of a wave's chunk: four a lane */
constexpr int SM_BINS = 4 * SM_THREADS;
constexpr int SM_LIST = SM_THREADS;      /* tokens a range may hold to be settled pairwise */

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

struct SampleShared {
    u64 hist[SM_BINS];
    u64 sum[SM_WAVES];
    u64 found;                           /* a running sum before the range or token that was found */
    u64 w[SM_LIST], above[SM_LIST], equal[SM_LIST];
    u64 chunk[16][WAVE];
    uint32_t key[SM_LIST];
    int idx[SM_LIST];
    uint32_t lo, hi;
    int bin, n, token;
    uint32_t cut;
};

/* Order-preserving integer of a float (no NaN, no -0) and back. */
__device__ __forceinline__ uint32_t order_key(float z) {
    const uint32_t u = __float_as_uint(z);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
    for (int o = WAVE / 2; o; o >>= 1) v += __shfl_xor(v, o, WAVE);
    return v;
}
__device__ __forceinline__ u64 wave_scan64(u64 v, int lane) {   /* inclusive */
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const u64 t = __shfl_up(v, o, WAVE);
        if (lane >= o) v += t;
    }
    return v;
}

/* round(2^S 2^x) for x <= 0; x below -100 or NaN: 0. 2^f, |f| <= 1/2, by sum_k (f ln 2)^k / k! up to k = 11, whose rest is
 * below 2^-47 of it. The sum with 2^52 leaves the rounded integer in the low 52 bits (S <= 46). */
__device__ __forceinline__ u64 fixed_exp2(double x, int S) {
    x = fmax(x, -100.0);
    const double n = __builtin_rint(x), f = x - n;
    double p = 4.44553827187081e-10;
    p = __builtin_fma(p, f, 7.054911620801121e-09);
    p = __builtin_fma(p, f, 1.0178086009239696e-07);
    p = __builtin_fma(p, f, 1.3215486790144305e-06);
    p = __builtin_fma(p, f, 1.5252733804059838e-05);
    p = __builtin_fma(p, f, 0.00015403530393381606);
    p = __builtin_fma(p, f, 0.0013333558146428441);
    p = __builtin_fma(p, f, 0.009618129107628477);
    p = __builtin_fma(p, f, 0.055504108664821576);
    p = __builtin_fma(p, f, 0.2402265069591007);
    p = __builtin_fma(p, f, 0.6931471805599453);
    p = __builtin_fma(p, f, 1.0);
    const double v = __builtin_ldexp(p, (int)n + S) + 0x1p52;
    return (u64)__builtin_bit_cast(long long, v) & 0xFFFFFFFFFFFFFull;
}

/* One row, read again for each pass. Element j of lane l of chunk c of wave w is index (w per + c) SM_CHUNK + 4 l + j.
 * Elements that are not allowed, and those past the row's end, are -inf. */
struct Row {
    const SampleArgs &a;
    const char *p;
    const uint32_t *mask;
    int per, base, lane;

    __device__ __forceinline__ Row(const SampleArgs &args, long long row)
        : a(args), p((const char *)args.logits + row * args.stride * (args.bf16 ? 2 : 4)),
          mask(args.mask ? args.mask + row * args.mask_stride : nullptr) {
        per = (a.vocab + SM_WAVES * SM_CHUNK - 1) / (SM_WAVES * SM_CHUNK);
        lane = threadIdx.x & (WAVE - 1);
        base = (int)(threadIdx.x >> 6) * per * SM_CHUNK;
    }

    __device__ __forceinline__ int index(int c) const { return base + c * SM_CHUNK + 4 * lane; }

    __device__ __forceinline__ void fetch(int c, float (&x)[4]) const {
        const int i = index(c);
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = -INFINITY;
        if (i >= a.vocab) return;
        if (a.wide && i + 3 < a.vocab) {
            if (a.bf16) {
                const uint2 u = *reinterpret_cast<const uint2 *>(p + 2LL * i);
                x[0] = __uint_as_float(u.x << 16); x[1] = __uint_as_float(u.x & 0xFFFF0000u);
                x[2] = __uint_as_float(u.y << 16); x[3] = __uint_as_float(u.y & 0xFFFF0000u);
            } else {
                const float4 u = *reinterpret_cast<const float4 *>(p + 4LL * i);
                x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j < a.vocab)
                    x[j] = a.bf16 ? bf16_to_f32(reinterpret_cast<const uint16_t *>(p)[i + j])
                                  : reinterpret_cast<const float *>(p)[i + j];
        }
        const uint32_t allowed = mask ? mask[i >> 5] >> (i & 31) : 0xFu;
#pragma unroll
        for (int j = 0; j < 4; j++)   /* NaN fails the comparison; -0 becomes +0, its equal */
            x[j] = (allowed >> j & 1) && x[j] > -INFINITY ? x[j] + 0.0f : -INFINITY;
    }

    /* f(c, values) for every chunk of this wave. */
    template <typename F>
    __device__ __forceinline__ void each(F &&f) const {
        for (int c = 0; c < per; c++) {
            float x[4];
            fetch(c, x);
            f(c, x);
        }
    }
};

/* Where a running sum reaches its target: its tokens' key, the last index taken among that key's equals, and whether the
 * sum reaches it at all. */
struct Cut {
    bool some;
    uint32_t key;
    int idx;
};

/* The bins' sums in order: sh.bin is the first bin at which the running sum reaches target(total), sh.found the sum
 * before it. Returns whether there is one. Every thread must call it. */
template <typename Target>
__device__ __forceinline__ bool find_bin(SampleShared &sh, Target target) {
    const int t = threadIdx.x, lane = t & (WAVE - 1), wave = t >> 6;
    u64 v[4], own = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; k++) {
        v[k] = sh.hist[4 * t + k];
        own += v[k];
    }
    const u64 scan = wave_scan64(own, lane);
    if (lane == WAVE - 1) sh.sum[wave] = scan;
    __syncthreads();
    u64 before = scan - own, total = 0;
#pragma unroll
    for (int w = 0; w < SM_WAVES; w++) {
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
    return goal <= total;
}

/* The smallest index whose running sum of m(z, index), in index order, reaches goal(total); -1 without one. Every thread
 * must call it. */
template <typename M, typename Goal>
__device__ __forceinline__ int select_in_order(SampleShared &sh, const Row &row, M m, Goal goal) {
    const int lane = row.lane, wave = threadIdx.x >> 6;
    u64 s = 0;
    row.each([&](int c, const float (&x)[4]) {
#pragma unroll
        for (int j = 0; j < 4; j++) s += m(x[j], row.index(c) + j);
    });
    s = wave_sum64(s);
    __syncthreads();
    if (lane == 0) sh.sum[wave] = s;
    if (threadIdx.x == 0) sh.token = -1;
    __syncthreads();
    u64 before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < SM_WAVES; w++) {
        before += w < wave ? sh.sum[w] : 0;
        total += sh.sum[w];
    }
    const u64 g = goal(total);
    if (before < g && g <= before + s) {   /* this wave holds it: its chunks, 16 at a time */
        for (int c0 = 0; c0 < row.per; c0 += 16) {
#pragma unroll
            for (int k = 0; k < 16; k++) sh.chunk[k][lane] = 0;
            row.each([&](int c, const float (&x)[4]) {
                if (c < c0 || c >= c0 + 16) return;
                u64 v = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) v += m(x[j], row.index(c) + j);
                sh.chunk[c - c0][lane] = v;
            });
            __builtin_amdgcn_wave_barrier();   /* one wave's LDS accesses complete in order */
            u64 part = 0;                      /* chunk lane / 4: 16 of its lanes, then the four quarters */
#pragma unroll
            for (int k = 0; k < 16; k++) part += sh.chunk[lane >> 2][(lane & 3) * 16 + k];
            part += __shfl_xor(part, 1, WAVE);
            part += __shfl_xor(part, 2, WAVE);
            const u64 upto = before + wave_scan64((lane & 3) == 3 ? part : 0, lane);
            const u64 hit = __ballot((lane & 3) == 3 && upto - part < g && g <= upto);
            if (!hit) {
                before = __shfl(upto, WAVE - 1, WAVE);
                continue;
            }
            const int at = __ffsll(hit) - 1, c1 = at >> 2;
            const u64 base = __shfl(upto - part, at, WAVE);
            const u64 v = sh.chunk[c1][lane], end = base + wave_scan64(v, lane);
            row.each([&](int c, const float (&x)[4]) {
                if (c != c0 + c1 || !(end - v < g && g <= end)) return;
                u64 run = end - v;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const u64 w = m(x[j], row.index(c) + j);
                    if (run < g && g <= run + w) sh.token = row.index(c) + j;
                    run += w;
                }
            });
            break;
        }
    }
    __syncthreads();
    return sh.token;
}

/* Over the elements that in(z, index) keeps, in order of value, the larger first: where the running sum of m(z) reaches
 * target(total). SPLIT: equals are taken one by one, the lower index first (m is 1), and the cut's idx is the last one
 * taken; else they are taken together. `range`: the values below zmax - range need no telling apart. Every thread must
 * call it. */
template <bool SPLIT, typename In, typename M, typename Target>
__device__ __forceinline__ Cut find_cut(SampleShared &sh, const Row &row, float zmax, float range, In in, M m, Target target) {
    const int t = threadIdx.x, lane = row.lane, wave = t >> 6;
    const float scale = range > 0.0f && range < INFINITY ? (SM_BINS - 1) / range : 0.0f;
    /* a range whose products are NaN or past the last bin: the last bin; monotone in z in every case */
    const auto bin_of = [&](float z) { return z == zmax ? 0 : (int)fminf((zmax - z) * scale, (float)(SM_BINS - 1)); };
    const auto clear = [&]() {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; k++) sh.hist[t + k * SM_THREADS] = 0;
        if (t == 0) sh.n = 0;
        __syncthreads();
    };
    u64 goal = 0;
    clear();
    row.each([&](int c, const float (&x)[4]) {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (in(x[j], row.index(c) + j))
                __hip_atomic_fetch_add(&sh.hist[bin_of(x[j])], m(x[j]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    });
    const bool some = find_bin(sh, [&](u64 total) { return goal = target(total); });
    if (!some) return Cut{false, 0u, 0};
    const int bin = sh.bin;
    u64 base = sh.found;
    uint32_t lo = 0u, hi = 0xFFFFFFFFu;   /* once a range of values is split again: its keys */
    bool keyed = false;
    for (;;) {
        const auto member = [&](float z, int i) {
            if (!in(z, i)) return false;
            const uint32_t k = order_key(z);
            return keyed ? k >= lo && k <= hi : bin_of(z) == bin;
        };
        row.each([&](int c, const float (&x)[4]) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (member(x[j], row.index(c) + j)) {
                    const int at = __hip_atomic_fetch_add(&sh.n, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                    if (at < SM_LIST) {
                        sh.key[at] = order_key(x[j]);
                        sh.idx[at] = row.index(c) + j;
                        sh.w[at] = m(x[j]);
                    }
                }
        });
        sh.above[t] = sh.equal[t] = 0;
        __syncthreads();
        const int n = sh.n;
        if (n <= SM_LIST) {   /* pairwise, every token's list split over 1,024 / n threads */
            int lanes = 1;
            while (lanes < n) lanes <<= 1;
            const int i = t & (lanes - 1);
            if (i < n) {
                const uint32_t k = sh.key[i];
                const int id = sh.idx[i];
                u64 above = 0, equal = 0;
                for (int j = t / lanes; j < n; j += SM_THREADS / lanes) {
                    const uint32_t kj = sh.key[j];
                    const u64 w = sh.w[j];
                    above += kj > k || (SPLIT && kj == k && sh.idx[j] < id) ? w : 0;
                    equal += !SPLIT && kj == k ? w : 0;
                }
                __hip_atomic_fetch_add(&sh.above[i], above, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                if (!SPLIT) __hip_atomic_fetch_add(&sh.equal[i], equal, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            }
            __syncthreads();
            if (t < n) {
                const u64 above = base + sh.above[t], own = SPLIT ? sh.w[t] : sh.equal[t];
                if (above < goal && goal <= above + own) {   /* one token, or one value's equals, who write the same */
                    sh.cut = sh.key[t];
                    sh.token = SPLIT ? sh.idx[t] : 0x7FFFFFFF;
                }
            }
            __syncthreads();
            return Cut{true, sh.cut, sh.token};
        }
        if (!keyed) {   /* the least and largest key of the range */
            uint32_t least = 0xFFFFFFFFu, most = 0u;
            row.each([&](int c, const float (&x)[4]) {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (member(x[j], row.index(c) + j)) {
                        least = min(least, order_key(x[j]));
                        most = max(most, order_key(x[j]));
                    }
            });
            __syncthreads();
            if (t == 0) sh.lo = 0xFFFFFFFFu, sh.hi = 0u;
            __syncthreads();
            __hip_atomic_fetch_min(&sh.lo, least, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            __hip_atomic_fetch_max(&sh.hi, most, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            __syncthreads();
            lo = sh.lo;
            hi = sh.hi;
            keyed = true;
        }
        if (lo == hi) {   /* one value */
            int idx = 0x7FFFFFFF;
            if (SPLIT) {
                const u64 rest = goal - base;
                idx = select_in_order(sh, row, [&](float z, int i) { return (u64)(in(z, i) && order_key(z) == lo); },
                                      [&](u64) { return rest; });
            }
            return Cut{true, lo, idx};
        }
        int shift = 0;
        while ((hi - lo) >> shift >= SM_BINS) shift++;
        clear();
        row.each([&](int c, const float (&x)[4]) {   /* the larger keys first */
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (member(x[j], row.index(c) + j))
                    __hip_atomic_fetch_add(&sh.hist[(hi - order_key(x[j])) >> shift], m(x[j]), __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_WORKGROUP);
        });
        const u64 rest = goal - base;
        find_bin(sh, [&](u64) { return rest; });
        base += sh.found;
        const uint32_t top = hi - ((uint32_t)sh.bin << shift);
        const uint32_t span = (1u << shift) - 1u;
        lo = top - lo > span ? top - span : lo;
        hi = top;
    }
}

__global__ void __launch_bounds__(SM_THREADS) sample_kernel(SampleArgs a) {
    __shared__ SampleShared sh;
    const long long r = blockIdx.x;
    const int t = threadIdx.x, lane = t & (WAVE - 1), wave = t >> 6;
    const Row row(a, r);

    /* the largest allowed logit (the lowest index among equals) and the smallest */
    u64 best = 0;
    float least = INFINITY;
    row.each([&](int c, const float (&x)[4]) {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (x[j] > -INFINITY) {
                best = max(best, (u64)order_key(x[j]) << 32 | (0xFFFFFFFFu - (uint32_t)(row.index(c) + j)));
                least = fminf(least, x[j]);
            }
    });
#pragma unroll
    for (int o = WAVE / 2; o; o >>= 1) {
        best = max(best, (u64)__shfl_xor(best, o, WAVE));
        least = fminf(least, __shfl_xor(least, o, WAVE));
    }
    if (lane == 0) {
        sh.sum[wave] = best;
        sh.idx[wave] = (int)__float_as_uint(least);
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SM_WAVES; w++) {
        best = max(best, sh.sum[w]);
        least = fminf(least, __uint_as_float((uint32_t)sh.idx[w]));
    }
    const float T = a.temperature[r];
    if (best == 0 || !(T > 0.0f)) {   /* nothing allowed; or the largest logit */
        if (t == 0) a.out[r] = best == 0 ? -1 : (int)(0xFFFFFFFFu - (uint32_t)best);
        return;
    }

    const float zmax = key_value((uint32_t)(best >> 32));
    const double zmaxd = zmax, per_log2 = 1.4426950408889634 / (double)T;
    int S = 62;   /* the row's weights sum below 2^62 */
    while (S > 0 && (1LL << (62 - S)) < a.vocab) S--;
    S = min(S, 46);
    const auto weight = [&](float z) {
        return z == zmax ? 1ull << S : z == -INFINITY ? 0ull : fixed_exp2(((double)z - zmaxd) * per_log2, S);
    };

    Cut top = {false, 0u, 0};
    const int k = a.top_k ? a.top_k[r] : 0;
    if (k > 0 && k < a.vocab)
        top = find_cut<true>(sh, row, zmax, zmax - least, [&](float z, int) { return z > -INFINITY; },
                             [&](float) { return 1ull; }, [&](u64) { return (u64)k; });
    const float top_z = top.some ? key_value(top.key) : -INFINITY;
    const auto ranked = [&](float z, int i) {   /* among the k largest */
        return z > top_z || (top.some && z == top_z && i <= top.idx);
    };

    float least_z = -INFINITY;   /* the nucleus' smallest logit */
    const float p = a.top_p ? a.top_p[r] : 1.0f;
    if (p < 1.0f) {
        /* values 47 log2 units below the largest weigh nothing: one bin for them all */
        const Cut mass = find_cut<false>(sh, row, zmax, fminf(zmax - least, 33.0f * T), ranked, weight, [&](u64 total) {
            return max((u64)ceil(fmax((double)p, 0.0) * (double)total), 1ull);
        });
        if (mass.some) least_z = key_value(mass.key);
    }
    const double floor_w = a.min_p ? fmin(fmax((double)a.min_p[r], 0.0), 1.0) : 0.0;   /* NaN: 0 */
    const u64 least_w = (u64)ceil(__builtin_ldexp(floor_w, S));
    const float u = a.uniform[r];
    const int token = select_in_order(
        sh, row,
        [&](float z, int i) {
            if (!(z >= least_z && ranked(z, i))) return 0ull;
            const u64 w = weight(z);
            return w >= least_w ? w : 0ull;
        },
        [&](u64 total) {   /* the first running sum above u total */
            const u64 at = u > 0.0f ? (u < 1.0f ? (u64)((double)u * (double)total) : total) : 0ull;
            return min(at, total - 1) + 1;
        });
    if (t == 0) a.out[r] = token;
}

}  // namespace nc

using namespace nc;

extern "C" int nc_sample_tokens(const void *logits, int is_bf16, long long row_stride, long long rows, int vocab,
                                const float *uniform, const float *temperature, const int32_t *top_k, const float *top_p,
                                const float *min_p, const uint32_t *mask, long long mask_stride, int32_t *tokens,
                                void *stream) {
    if (!logits || !uniform || !temperature || !tokens) return NC_ERR_NULL;
    if (rows < 0 || rows > 1LL << 22 || vocab <= 0 || vocab > 1 << 24 || row_stride < vocab ||
        (mask && mask_stride < ((long long)vocab + 31) / 32))
        return NC_ERR_SHAPE;
    if (rows == 0) return NC_OK;
    SampleArgs a = {};
    a.logits = logits; a.stride = row_stride; a.vocab = vocab; a.bf16 = is_bf16 != 0;
    a.wide = (uintptr_t)logits % (is_bf16 ? 8 : 16) == 0 && row_stride % 4 == 0;
    a.uniform = uniform; a.temperature = temperature; a.top_p = top_p; a.min_p = min_p; a.top_k = top_k;
    a.mask = mask; a.mask_stride = mask_stride;
    a.out = tokens;
    hipLaunchKernelGGL(sample_kernel, dim3((unsigned)rows), dim3(SM_THREADS), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}
