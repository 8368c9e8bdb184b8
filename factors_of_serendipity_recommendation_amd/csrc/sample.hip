// Draws from score rows: temperature, top-k, top-p and min-p, from given random numbers.
//
// The kept columns are a prefix of the row's ranking (score descending, ties to the lower column), so they are
// described by one 64-bit key (wave_topk.h's make_key): column i is kept iff its key is at least the cut.
// A cut is found through a histogram of 2048 equal steps of the distance to the row's best score, of counts for
// top_k and of weights for top_p: the bin in which the running sum reaches its target is gathered and sorted.
// A top_k of at most ~kList columns gathers all of them, and what follows works on that list alone.  A bin that
// holds more than kList columns (many equal scores, scores of very different sizes) is opened by a descent
// over the 32 score bits instead.
//
// Which column a given number draws depends on every weight before it, and with a million columns the borders
// between columns lie 1e-6 of the total apart, so 24 bits are not enough: weights are computed in f64 and
// summed in f64 in a fixed order, and the histogram holds them as integers (so that the order of its atomic
// additions does not matter).
#include "wave_topk.h"

#include <algorithm>

namespace lgx {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kList = 2048;  // columns that are sorted in LDS
constexpr int kSegs = 1024;  // column segments with sums of their own: a draw scans one of them

struct SampleArgs {
    const void* S;
    int64_t rows, cols, ld;
    const void* u;
    int u_f64;
    int64_t n_draws;
    double T, top_p, min_p;
    int64_t top_k;
    const float *T_rows, *p_rows, *m_rows;
    const int32_t* k_rows;
    int32_t* out_idx;
    float* out_prob;
};

// ------------------------------------------------------------------------------------ scores and weights
template <bool BF16>
__device__ __forceinline__ float load_score(const void* s, int64_t i) {
    return BF16 ? bf16_to_f32(static_cast<const uint16_t*>(s)[i]) : static_cast<const float*>(s)[i];
}

// four scores from any element offset
template <bool BF16>
struct Vec {
    static constexpr int N = 4;
    float v[N];
    __device__ __forceinline__ void load(const void* s, int64_t i) {
        if (BF16) {
            using U = uint32_t __attribute__((ext_vector_type(2), aligned(2)));
            const U q = *reinterpret_cast<const U*>(static_cast<const uint16_t*>(s) + i);
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                v[j] = __uint_as_float(q[j / 2] << 16);
                v[j + 1] = __uint_as_float(q[j / 2] & 0xffff0000u);
            }
        } else {
            using F = float __attribute__((ext_vector_type(4), aligned(4)));
            const F q = *reinterpret_cast<const F*>(static_cast<const float*>(s) + i);
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = q[j % 4];
        }
    }
    // columns at or past `end` as -inf, which no step takes
    __device__ __forceinline__ void load_tail(const void* s, int64_t i, int64_t end) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = i + j < end ? load_score<BF16>(s, i + j) : -INFINITY;
    }
};

// f(four scores, column of the first) over columns [lo, hi) by `width` lanes, this one being `me`; a lane takes
// its columns in ascending order, U groups at a time; columns past the end come as -inf
template <bool BF16, int U, typename F>
__device__ __forceinline__ void for_groups(const void* s, int64_t lo, int64_t hi, int me, int width, F f) {
    constexpr int N = Vec<BF16>::N;
    int64_t i = lo + (int64_t)me * N;
    const int64_t step = (int64_t)width * N;
    if (U > 1)
        for (; i + (U - 1) * step + N <= hi; i += U * step) {
            Vec<BF16> v[U];
#pragma unroll
            for (int k = 0; k < U; ++k) v[k].load(s, i + k * step);
#pragma unroll
            for (int k = 0; k < U; ++k) f(v[k].v, (int)(i + k * step));
        }
#pragma unroll 1
    for (; i < hi; i += step) {
        Vec<BF16> v;
        if (i + N <= hi)
            v.load(s, i);
        else
            v.load_tail(s, i, hi);
        f(v.v, (int)i);
    }
}

// the order key of a score; 0 for the excluded ones (NaN, -inf).  -0 ranks with +0
__device__ __forceinline__ uint32_t score_key(float s) {
    return s > -INFINITY ? ord_f32(s + 0.0f) : 0u;
}
__device__ __forceinline__ uint64_t column_key(float s, int i) {
    return (uint64_t)score_key(s) << 32 | (0xffffffffu - (uint32_t)i);
}

// where the ranking is cut: columns scoring above s, and those scoring s up to column i
struct Cut {
    float s;
    int i;
    __device__ __forceinline__ bool keeps(float v, int col) const { return (v > s) | ((v == s) & (col <= i)); }
};
constexpr float kNone = -INFINITY;  // Cut{kNone, -1}: every column with a score

// one f64 multiply-add with its addend in scalar registers (the compiler copies a constant addend into vector
// registers before every step: 10 more instructions a weight)
__device__ __forceinline__ double fma_const(double a, double b, double c) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}

// Weights exp((s - m) / T) against the row's best score m, a finite one; 0 for -inf and NaN, which the maximum turns into
// a distance of 2^-1100.  2^y = 2^n 2^f with n = rint(y) and for 2^f, |f| <= 1/2, the polynomial that equals it at 0 and
// at nine Chebyshev nodes (within 4e-14 relative, exact at f = 0: equal scores weigh the same power of two)
struct Weigh {
    double m, c;   // c = log2(e) / T
    double floor;  // the distance whose weight underflows
    int unit;      // log2 of the fixed-point unit
    __device__ __forceinline__ Weigh(float top, double T, int cols) {
        m = (double)top;
        c = 1.4426950408889634074 / fmin(T, 1e300);
        floor = -1100.0 / c;
        unit = 62;  // the sum of all weights is at most cols
        while (unit > 0 && (1ll << (62 - unit)) < (int64_t)cols) --unit;
        unit = min(unit, 51);
    }
    __device__ __forceinline__ double scaled(float s, int e) const {
        const double d = fmax((double)s - m, floor);
        const double big = fma(d, c, 6755399441055744.0);  // 1.5 * 2^52: the low word is n
        const double f = fma(d, c, 6755399441055744.0 - big);
        double r = fma_const(f, 1.0203121063391729e-07, 1.3255224878668817e-06);
        r = fma_const(r, f, 1.525268684626772e-05);
        r = fma_const(r, f, 0.00015403455852453838);
        r = fma_const(r, f, 0.0013333558179043112);
        r = fma_const(r, f, 0.009618129159402558);
        r = fma_const(r, f, 0.055504108664760424);
        r = fma_const(r, f, 0.2402265069581299);
        r = fma_const(r, f, 0.6931471805599453);
        r = fma(r, f, 1.0);
        return ldexp(r, (int)(uint32_t)__double_as_longlong(big) + e);
    }
    __device__ __forceinline__ double operator()(float s) const { return scaled(s, 0); }
    // w in units of 2^-unit, rounded; w 2^unit <= 2^51, so that adding 2^52 leaves it in the low bits
    __device__ __forceinline__ uint64_t fixed(float s) const {
        const double w = scaled(s, unit) + 4503599627370496.0;
        return (uint64_t)__double_as_longlong(w) & 0xfffffffffffffull;
    }
};

// ------------------------------------------------------------------------------------ wave and workgroup steps
__device__ __forceinline__ double shfl_f64(double v, int src) { return __longlong_as_double((int64_t)shfl_u64(__double_as_longlong(v), src)); }
__device__ __forceinline__ double shfl_xor_f64(double v, int m) { return __longlong_as_double((int64_t)shfl_xor_u64(__double_as_longlong(v), m)); }

// v from the lane that a DPP row operation names, 0 where it names none
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
    return (uint64_t)hi << 32 | lo;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_f64(double v) {
    return __longlong_as_double((int64_t)dpp_u64<CTRL, ROWS>((uint64_t)__double_as_longlong(v)));
}
// inclusive sums over the lanes: shifts within a row of 16, then the last lane of row 0 into row 1 and of row 2 into row
// 3, then lane 31 into the upper half
__device__ __forceinline__ double wave_scan_f64(double v) {
    v += dpp_f64<0x111, 0xf>(v);
    v += dpp_f64<0x112, 0xf>(v);
    v += dpp_f64<0x114, 0xf>(v);
    v += dpp_f64<0x118, 0xf>(v);
    v += dpp_f64<0x142, 0xa>(v);
    v += dpp_f64<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {
    v += dpp_u64<0x111, 0xf>(v);
    v += dpp_u64<0x112, 0xf>(v);
    v += dpp_u64<0x114, 0xf>(v);
    v += dpp_u64<0x118, 0xf>(v);
    v += dpp_u64<0x142, 0xa>(v);
    v += dpp_u64<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
    v = max(v, dpp_u64<0x111, 0xf>(v));
    v = max(v, dpp_u64<0x112, 0xf>(v));
    v = max(v, dpp_u64<0x114, 0xf>(v));
    v = max(v, dpp_u64<0x118, 0xf>(v));
    v = max(v, dpp_u64<0x142, 0xa>(v));
    v = max(v, dpp_u64<0x143, 0xc>(v));
    return v;  // lane 63 holds it
}

struct Shared {
    uint64_t hist[kBins];
    uint64_t key[kList];    // gathered columns
    double w[kList];        // their weights, then the running sums of the kept ones
    double seg[kSegs + 1];
    uint64_t part[kWaves];
    uint64_t below;
    uint32_t bin, n;
};

// sum / maximum over the workgroup, the same value in every thread
__device__ uint64_t block_sum_u64(uint64_t v, Shared& sh) {
    v = wave_scan_u64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t s = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) s += sh.part[i];
    return s;
}
__device__ uint64_t block_max_u64(uint64_t v, Shared& sh) {
    v = wave_max_u64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t s = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) s = max(s, sh.part[i]);
    return s;
}

__device__ __forceinline__ void clear_hist(Shared& sh) {
    __syncthreads();
    for (int j = threadIdx.x; j < kBins; j += kThreads) sh.hist[j] = 0;
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
}

// The bin in which the running sum of hist, from bin 0 on, reaches `target`: sum before it < target <= sum with
// it; the last bin that holds anything if the whole falls short, bin 0 of an empty histogram.
// -> sh.bin, sh.below = the sum before it
__device__ void find_bin(double target, Shared& sh) {
    constexpr int per = kBins / kThreads;
    const int tid = threadIdx.x;
    if (tid == 0) {
        sh.bin = 0;
        sh.below = 0;
    }
    __syncthreads();
    uint64_t h[per], own = 0;
#pragma unroll
    for (int j = 0; j < per; ++j) own += h[j] = sh.hist[tid * per + j];
    const uint64_t incl = wave_scan_u64(own);
    if ((tid & 63) == 63) sh.part[tid >> 6] = incl;
    __syncthreads();
    uint64_t run = incl - own, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < (tid >> 6)) run += sh.part[w];
        all += sh.part[w];
    }
    target = fmin(target, (double)all);
#pragma unroll
    for (int j = 0; j < per; ++j) {
        const uint64_t next = run + h[j];
        // the first bin that reaches it (a target of 0 or less: the first that holds anything)
        if (h[j] && (double)next >= target && (run == 0 || (double)run < target)) {
            sh.bin = (uint32_t)(tid * per + j);
            sh.below = run;
        }
        run = next;
    }
    __syncthreads();
}

// bitonic sort of sh.key[0, n), descending, n <= kList; keys past n become 0
__device__ void sort_keys(int n, Shared& sh) {
    int size = 64;
    while (size < n) size <<= 1;
    __syncthreads();
    for (int j = threadIdx.x; j < size; j += kThreads)
        if (j >= n) sh.key[j] = 0;
    for (int k = 2; k <= size; k <<= 1)
        for (int d = k >> 1; d > 0; d >>= 1) {
            __syncthreads();
            for (int t = threadIdx.x; t < size / 2; t += kThreads) {
                const int i = (t / d) * 2 * d + t % d;
                const uint64_t x = sh.key[i], y = sh.key[i + d];
                if ((x < y) == ((i & k) == 0)) {
                    sh.key[i] = y;
                    sh.key[i + d] = x;
                }
            }
        }
    __syncthreads();
}

// sh.w[0, n) -> its inclusive running sums, in order
__device__ void scan_list(int n, Shared& sh) {
    constexpr int per = kList / 64;
    __syncthreads();
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x, lo = lane * per, hi = min(n, lo + per);
        double own = 0.0;
        for (int j = lo; j < hi; ++j) own += sh.w[j];
        double run = wave_scan_f64(own) - own;
        for (int j = lo; j < hi; ++j) sh.w[j] = run += sh.w[j];
    }
    __syncthreads();
}

// ------------------------------------------------------------------------------------ one row
struct Row {
    double T, top_p, min_p;
    int64_t top_k;
};
__device__ __forceinline__ Row row_settings(const SampleArgs& a, int64_t row) {
    Row r;
    r.T = a.T_rows ? (double)a.T_rows[row] : a.T;
    r.top_p = a.p_rows ? (double)a.p_rows[row] : a.top_p;
    const double m = a.m_rows ? (double)a.m_rows[row] : a.min_p;
    r.min_p = m > 0.0 ? fmin(m, 1.0) : 0.0;
    r.top_k = a.k_rows ? (int64_t)a.k_rows[row] : a.top_k;
    return r;
}
__device__ __forceinline__ double draw_number(const SampleArgs& a, int64_t row, int64_t j) {
    const int64_t i = row * a.n_draws + j;
    const double u = a.u_f64 ? static_cast<const double*>(a.u)[i] : (double)static_cast<const float*>(a.u)[i];
    return fmin(fmax(u, 0.0), 1.0);
}

// one reading of the columns [lo, hi): the best one as a key (0 without one), and the lowest score above -1e30 (lower
// ones are masks, and share the last bin)
struct Top {
    uint64_t best;
    float low;
};
template <bool BF16>
__device__ __forceinline__ Top scan_top(const void* s, int64_t lo, int64_t hi, int me, int width) {
    float best = -INFINITY, low = INFINITY;
    int at = -1;
    for_groups<BF16, 4>(s, lo, hi, me, width, [&](const float (&v)[4], int i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) low = fminf(low, v[j] > -1e30f ? v[j] : INFINITY);
        if (fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) > best) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (v[j] > best) {
                    best = v[j];
                    at = i + j;
                }
        }
    });
    return Top{at < 0 ? 0ull : column_key(best, at), low};
}

// equal steps of the distance to the best score.  A score belongs to bin b < kBins - 1 iff b <= at(s) < b + 1,
// what is farther (and NaN) to the last one
struct Binning {
    float top, inv;
    __device__ __forceinline__ float at(float s) const { return (top - s) * inv; }
    __device__ __forceinline__ int operator()(float s) const { return (int)fminf(at(s), (float)(kBins - 1)); }
};
__device__ __forceinline__ Binning make_binning(float top, double range) {
    const double inv = (double)(kBins - 1) / range;  // a range of 0: all the best score's equals in bin 0
    return Binning{top, (float)fmin(inv, 1e30)};
}

// The cut of top_k (MASS false: `target` columns) or top_p (`target` of the fixed weights), among the columns of
// key >= cut, by descent over the score bits; ties are counted off in column order
template <bool BF16, bool MASS>
__device__ Cut descend(const void* s, int cols, const Cut& cut, double target, const Weigh& weigh, Shared& sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t above = 0;   // counted in better bins than this digit's
    uint32_t prefix = 0;  // the score bits found so far
#pragma unroll 1
    for (int digit = 0; digit < 3; ++digit) {
        const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
        const int open = digit == 0 ? 32 : digit == 1 ? 21 : 10;  // bits not yet found
        const uint32_t mask = (1u << (open - shift)) - 1u;
        clear_hist(sh);
        for_groups<BF16, 1>(s, 0, cols, tid, kThreads, [&](const float (&v)[4], int i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t k = score_key(v[j]);
                if (cut.keeps(v[j], i + j) && (open == 32 || (k >> open) == (prefix >> open)))
                    atomicAdd((unsigned long long*)&sh.hist[mask - ((k >> shift) & mask)],
                              (unsigned long long)(MASS ? weigh.fixed(v[j]) : 1ull));
            }
        });
        find_bin(target - (double)above, sh);
        prefix |= (mask - sh.bin) << shift;
        above += sh.below;
    }
    __syncthreads();
    const float value = unord_f32(prefix);
    const uint64_t each = MASS ? max(weigh.fixed(value), (uint64_t)1) : 1ull;
    const double want_f = ceil((target - (double)above) / (double)each);
    int64_t want = want_f < 1.0 ? 1 : (int64_t)fmin(want_f, (double)cols);
    int found = -1;  // the column of the last one taken
    for (int64_t i0 = 0; i0 < cols; i0 += kThreads) {
        const int64_t i = i0 + tid;
        const float v = i < cols ? load_score<BF16>(s, i) : kNone;
        const bool eq = v == value && cut.keeps(v, (int)i);
        const uint64_t m = __ballot(eq);
        __syncthreads();
        if (lane == 0) sh.part[wave] = (uint64_t)__popcll(m);
        __syncthreads();
        int64_t before = 0, all = 0;
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) before += (int64_t)sh.part[w];
            all += (int64_t)sh.part[w];
        }
        before += __popcll(m & ((1ull << lane) - 1));
        if (eq && before < want) found = (int)i;
        want -= all;
        if (want <= 0) break;
    }
    return Cut{value, (int)block_max_u64((uint64_t)(found + 1), sh) - 1};
}

// sh.key[0, n) holds the row's best n columns, unsorted, n <= kList, at least min(top_k, live) of them: the
// restrictions and the draws on that list
__device__ void finish_list(const SampleArgs& a, int64_t row, const Row& r, int n, const Weigh& weigh, Shared& sh) {
    sort_keys(n, sh);
    n = (int)min((int64_t)n, r.top_k);
    for (int j = threadIdx.x; j < n; j += kThreads) sh.w[j] = weigh(key_score(sh.key[j]));
    __syncthreads();
    // min_p cuts a prefix of the ranking; top_p looks at all of top_k
    int keep = n;
    if (r.top_p < 1.0) {
        scan_list(n, sh);
        const double target = r.top_p * sh.w[n - 1];
        // column j stays iff the sum before it is below the target
        int lo = 1, hi = n;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (sh.w[mid - 1] < target) lo = mid + 1; else hi = mid;
        }
        keep = lo;
        // (lo is the first count whose sum reaches the target)
        __syncthreads();
    }
    // the kept ones in column order
    for (int j = threadIdx.x; j < keep; j += kThreads) {
        const uint64_t key = sh.key[j];
        const double w = weigh(key_score(key));
        // ~column descending = column ascending; the score rides along in the low half
        sh.hist[j] = w >= r.min_p ? (uint64_t)(uint32_t)key << 32 | (uint32_t)(key >> 32) : 0ull;
    }
    __syncthreads();
    for (int j = threadIdx.x; j < keep; j += kThreads) sh.key[j] = sh.hist[j];
    sort_keys(keep, sh);
    for (int j = threadIdx.x; j < keep; j += kThreads) {
        const uint64_t key = sh.key[j];
        sh.w[j] = key ? weigh(unord_f32((uint32_t)key)) : 0.0;
    }
    scan_list(keep, sh);
    const double total = sh.w[keep - 1];
    int end = keep - 1;  // the last column with any weight
    while (end > 0 && !(sh.w[end] > sh.w[end - 1])) --end;
    for (int64_t j = threadIdx.x; j < a.n_draws; j += kThreads) {
        const double target = draw_number(a, row, j) * total;
        int lo = 0, hi = end;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (sh.w[mid] > target) hi = mid; else lo = mid + 1;
        }
        const uint64_t key = sh.key[lo];
        a.out_idx[row * a.n_draws + j] = (int32_t)(0xffffffffu - (uint32_t)(key >> 32));
        if (a.out_prob) a.out_prob[row * a.n_draws + j] = (float)(weigh(unord_f32((uint32_t)key)) / total);
    }
}

// A row with infinite scores: those columns share it equally, and their ranking is the column order
template <bool BF16>
__device__ void draw_infinite(const SampleArgs& a, int64_t row, const Row& r, const void* s, Shared& sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t n = 0;
    for (int64_t i = tid; i < a.cols; i += kThreads) n += load_score<BF16>(s, i) == INFINITY;
    int64_t keep = (int64_t)block_sum_u64(n, sh);
    if (r.top_k > 0) keep = min(keep, r.top_k);
    if (r.top_p < 1.0) keep = max((int64_t)1, (int64_t)ceil(r.top_p * (double)keep));
    for (int64_t j = wave; j < a.n_draws; j += kWaves) {
        int64_t rank = min((int64_t)(draw_number(a, row, j) * (double)keep), keep - 1), at = -1;
        for (int64_t i0 = 0; i0 < a.cols && at < 0; i0 += 64) {
            const uint64_t m = __ballot(i0 + lane < a.cols && load_score<BF16>(s, min(i0 + lane, a.cols - 1)) == INFINITY);
            const bool mine = (m >> lane & 1) && __popcll(m & ((1ull << lane) - 1)) == rank;
            const uint64_t hit = __ballot(mine);
            if (hit) at = i0 + __builtin_ctzll(hit);
            rank -= __popcll(m);
        }
        if (lane == 0) {
            a.out_idx[row * a.n_draws + j] = (int32_t)at;
            if (a.out_prob) a.out_prob[row * a.n_draws + j] = (float)(1.0 / (double)keep);
        }
    }
}

template <bool BF16>
__global__ __launch_bounds__(kThreads, 4) void sample_rows_kernel(SampleArgs a) {
    __shared__ Shared sh;
    constexpr int N = Vec<BF16>::N;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const void* s = BF16 ? (const void*)(static_cast<const uint16_t*>(a.S) + row * a.ld)
                         : (const void*)(static_cast<const float*>(a.S) + row * a.ld);
    const int cols = (int)a.cols;
    const Row r = row_settings(a, row);

    const Top mine = scan_top<BF16>(s, 0, cols, tid, kThreads);
    const uint64_t best = block_max_u64(mine.best, sh);
    if (best == 0 || !(r.T > 0.0) || r.top_k == 1) {
        for (int64_t j = tid; j < a.n_draws; j += kThreads) {
            a.out_idx[row * a.n_draws + j] = best ? key_index(best) : -1;
            if (a.out_prob) a.out_prob[row * a.n_draws + j] = best ? 1.0f : 0.0f;
        }
        return;
    }
    const float top = key_score(best);
    if (top == INFINITY) {
        draw_infinite<BF16>(a, row, r, s, sh);
        return;
    }
    const Weigh weigh(top, r.T, cols);

    Cut cut{kNone, -1};
    if (r.top_k > 0 && r.top_k < cols) {
        const float low = unord_f32(~(uint32_t)block_max_u64((uint64_t)(~ord_f32(mine.low)), sh));
        const Binning bin = make_binning(top, fmax((double)top - (double)low, 0.0));
        clear_hist(sh);
        for_groups<BF16, 2>(s, 0, cols, tid, kThreads, [&](const float (&v)[4], int) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (v[j] > kNone) atomicAdd((unsigned*)&sh.hist[bin(v[j])], 1u);
        });
        find_bin((double)r.top_k, sh);
        const int b = (int)sh.bin;
        const uint64_t before = sh.below, in_bin = sh.hist[b];
        const bool list = before + in_bin <= kList;
        if (list || in_bin <= kList) {
            const float from = list ? -INFINITY : (float)b, to = b == kBins - 1 ? NAN : (float)(b + 1);
            for_groups<BF16, 2>(s, 0, cols, tid, kThreads, [&](const float (&v)[4], int i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = bin.at(v[j]);
                    if ((x >= from) & !(x >= to) & (v[j] > kNone)) sh.key[atomicAdd(&sh.n, 1u)] = column_key(v[j], i + j);
                }
            });
            __syncthreads();
            if (list) {
                finish_list(a, row, r, (int)sh.n, weigh, sh);
                return;
            }
            sort_keys((int)in_bin, sh);
            const uint64_t key = sh.key[min((uint64_t)r.top_k - before, in_bin) - 1];
            cut = Cut{key_score(key), key_index(key)};
        } else {
            cut = descend<BF16, false>(s, cols, cut, (double)r.top_k, weigh, sh);
        }
    }
    if (r.top_p < 1.0) {
        // a column of weight below (1 - p) Z / cols is never kept (all such together weigh less than the
        // (1 - p) Z that are dropped), and Z >= 1; they share the last bin, summed in registers
        const Binning bin = make_binning(top, fmin(r.T, 1e30) * (log((double)cols / (1.0 - r.top_p)) + 1e-3));
        const bool all = cut.s == kNone;
        clear_hist(sh);
        uint64_t rest = 0;
        for_groups<BF16, 1>(s, 0, cols, tid, kThreads, [&](const float (&v)[4], int i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!all && !cut.keeps(v[j], i + j)) continue;
                const uint64_t w = weigh.fixed(v[j]);
                const int b = bin(v[j]);
                if (b < kBins - 1)
                    atomicAdd((unsigned long long*)&sh.hist[b], (unsigned long long)w);
                else
                    rest += w;
            }
        });
        if (rest) atomicAdd((unsigned long long*)&sh.hist[kBins - 1], (unsigned long long)rest);
        __syncthreads();
        uint64_t sum = 0;
        for (int j = tid; j < kBins; j += kThreads) sum += sh.hist[j];
        const double target = r.top_p * (double)block_sum_u64(sum, sh);
        find_bin(target, sh);
        const int b = (int)sh.bin;
        const uint64_t before = sh.below;
        const float from = (float)b, to = b == kBins - 1 ? NAN : (float)(b + 1);
        for_groups<BF16, 4>(s, 0, cols, tid, kThreads, [&](const float (&v)[4], int i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x = bin.at(v[j]);
                if ((x >= from) & !(x >= to) & cut.keeps(v[j], i + j)) {
                    const uint32_t at = atomicAdd(&sh.n, 1u);
                    if (at < kList) sh.key[at] = column_key(v[j], i + j);
                }
            }
        });
        __syncthreads();
        const int n = (int)min(sh.n, (uint32_t)kList + 1);
        if (n > 0 && n <= kThreads) {
            // each thread adds up what ranks before its column: the last one below the target is the cut
            if (tid < n) sh.hist[tid] = weigh.fixed(key_score(sh.key[tid]));
            __syncthreads();
            uint64_t mine = ~0ull;
            if (tid < n) {
                mine = sh.key[tid];
                uint64_t sum = before;
                bool first = true;
                for (int j = 0; j < n; ++j) {
                    const bool better = sh.key[j] > mine;
                    sum += better ? sh.hist[j] : 0;
                    first &= !better;
                }
                if (!((double)sum < target) && !(first && before == 0)) mine = ~0ull;
            }
            const uint64_t key = ~block_max_u64(~mine, sh);
            cut = Cut{key_score(key), key_index(key)};
        } else if (n > 0 && n <= kList) {
            sort_keys(n, sh);
            // the last column whose sum before it is below the target
            for (int j = tid; j < n; j += kThreads) sh.hist[j] = weigh.fixed(key_score(sh.key[j]));
            __syncthreads();
            if (tid < 64) {
                constexpr int per = kList / 64;
                const int lo = lane * per, hi = min(n, lo + per);
                uint64_t own = 0;
                for (int j = lo; j < hi; ++j) own += sh.hist[j];
                uint64_t run = before + wave_scan_u64(own) - own;
                int last = 0;
                for (int j = lo; j < hi; ++j) {
                    if ((double)run < target) last = j;
                    run += sh.hist[j];
                }
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) last = max(last, __shfl_xor(last, o, 64));
                if (lane == 0) sh.bin = (uint32_t)last;
            }
            __syncthreads();
            const uint64_t key = sh.key[sh.bin];
            cut = Cut{key_score(key), key_index(key)};
        } else {
            cut = descend<BF16, true>(s, cols, cut, target, weigh, sh);
        }
    }

    // weights of the kept columns, summed per segment
    constexpr int kStep = 64 * N;  // at least four steps of a wave, so that their one reduction is shared
    const int64_t seg_len = max(((int64_t)cols + kSegs * kStep - 1) / (kSegs * kStep), (int64_t)(cols > 16 * kStep * kWaves ? 4 : 1)) * kStep;
    const int n_segs = (int)(((int64_t)cols + seg_len - 1) / seg_len);
    auto kept = [&](float v, int i) -> double {
        const double w = weigh(v);
        return (cut.keeps(v, i) & (w >= r.min_p)) ? w : 0.0;
    };
    __syncthreads();
    for (int g = wave; g < n_segs; g += kWaves) {
        double w = 0.0;
        for_groups<BF16, 1>(s, g * seg_len, min((int64_t)cols, (g + 1) * seg_len), lane, 64, [&](const float (&v)[4], int i) {
            if (fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= cut.s)
                w += (kept(v[0], i) + kept(v[1], i + 1)) + (kept(v[2], i + 2) + kept(v[3], i + 3));
        });
        w = wave_scan_f64(w);
        if (lane == 63) sh.seg[g + 1] = w;
    }
    __syncthreads();
    if (tid < 64) {
        constexpr int per = kSegs / 64;
        const int lo = lane * per, hi = min(n_segs, lo + per);
        double own = 0.0;
        for (int j = lo; j < hi; ++j) own += sh.seg[j + 1];
        double run = wave_scan_f64(own) - own;
        for (int j = lo; j < hi; ++j) sh.seg[j + 1] = run += sh.seg[j + 1];
        if (lane == 0) sh.seg[0] = 0.0;
    }
    __syncthreads();
    const double total = sh.seg[n_segs];
    int last_seg = n_segs - 1;  // the last segment with any weight
    while (last_seg > 0 && !(sh.seg[last_seg + 1] > sh.seg[last_seg])) --last_seg;
    for (int64_t j = wave; j < a.n_draws; j += kWaves) {
        const double target = draw_number(a, row, j) * total;
        int lo = 0, hi = last_seg;  // the first segment whose end passes the target
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (sh.seg[mid + 1] > target) hi = mid; else lo = mid + 1;
        }
        const int64_t end = min((int64_t)cols, (lo + 1) * seg_len);
        double run = sh.seg[lo];
        int64_t pick = -1;
        double wp = 0.0;
        for (int64_t i0 = lo * seg_len; i0 < end; i0 += kStep) {
            Vec<BF16> v;
            const int64_t i = i0 + lane * N;
            if (i + N <= end)
                v.load(s, i);
            else
                v.load_tail(s, i, end);
            double w[N], own = 0.0;
#pragma unroll
            for (int k = 0; k < N; ++k) own += w[k] = kept(v.v[k], (int)i + k);
            double c = run + wave_scan_f64(own) - own;
            // this lane's first column past the target, or without one its last of any weight
            int at = -1, tail = -1;
            double wa = 0.0, wt = 0.0;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                c += w[k];
                if (w[k] > 0.0) {
                    tail = k;
                    wt = w[k];
                    if (at < 0 && c > target) {
                        at = k;
                        wa = w[k];
                    }
                }
            }
            const uint64_t pass = __ballot(at >= 0), any = __ballot(tail >= 0);
            if (any) {
                const int l = pass ? __builtin_ctzll(pass) : 63 - __builtin_clzll(any);
                pick = i0 + l * N + __shfl(pass ? at : tail, l, 64);
                wp = shfl_f64(pass ? wa : wt, l);
                if (pass) break;
            }
            run = shfl_f64(c, 63);
        }
        if (lane == 0) {
            a.out_idx[row * a.n_draws + j] = (int32_t)pick;
            if (a.out_prob) a.out_prob[row * a.n_draws + j] = (float)(wp / total);
        }
    }
}

}  // namespace
}  // namespace lgx

using namespace lgx;

extern "C" int lgx_sample_rows_workspace(int64_t rows, int64_t cols, int64_t n_draws, size_t* ws_bytes) {
    LGX_REQUIRE(ws_bytes && rows >= 0 && cols >= 1 && n_draws >= 0, LGX_ERR_INVALID_ARG,
                "lgx_sample_rows_workspace: bad arguments");
    *ws_bytes = 0;
    return LGX_OK;
}

extern "C" int lgx_sample_rows(const void* S, int dtype, int64_t rows, int64_t cols, int64_t ld, const void* u, int u_dtype,
                               int64_t n_draws, double temperature, const float* temperature_rows, int64_t top_k,
                               const int32_t* top_k_rows, double top_p, const float* top_p_rows, double min_p,
                               const float* min_p_rows, int32_t* out_idx, float* out_prob, void* ws, size_t ws_bytes,
                               lgx_stream_t stream_) {
    hipStream_t stream = as_hip(stream_);
    LGX_REQUIRE(dtype == LGX_DTYPE_F32 || dtype == LGX_DTYPE_BF16, LGX_ERR_INVALID_ARG, "lgx_sample_rows: dtype");
    LGX_REQUIRE(u_dtype == LGX_DTYPE_F32 || u_dtype == LGX_DTYPE_F64, LGX_ERR_INVALID_ARG, "lgx_sample_rows: dtype of u");
    LGX_REQUIRE(rows >= 0 && n_draws >= 0, LGX_ERR_INVALID_ARG, "lgx_sample_rows: negative size");
    LGX_REQUIRE(cols >= 1 && cols < INT32_MAX && ld >= cols, LGX_ERR_INVALID_ARG,
                "lgx_sample_rows: cols=%lld outside [1, 2^31) or ld=%lld < cols", (long long)cols, (long long)ld);
    if (rows == 0 || n_draws == 0) return LGX_OK;
    LGX_REQUIRE(rows < (1LL << 31), LGX_ERR_UNSUPPORTED, "lgx_sample_rows: %lld rows is too many", (long long)rows);
    LGX_REQUIRE(S && u && out_idx, LGX_ERR_INVALID_ARG, "lgx_sample_rows: null pointer");
    (void)ws;
    (void)ws_bytes;
    const SampleArgs a{S, rows, cols, ld, u, u_dtype == LGX_DTYPE_F64, n_draws, temperature, top_p, min_p, top_k,
                       temperature_rows, top_p_rows, min_p_rows, top_k_rows, out_idx, out_prob};
    if (dtype == LGX_DTYPE_BF16)
        sample_rows_kernel<true><<<(unsigned)rows, kThreads, 0, stream>>>(a);
    else
        sample_rows_kernel<false><<<(unsigned)rows, kThreads, 0, stream>>>(a);
    LGX_LAUNCH_CHECK();
    return LGX_OK;
}
