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

// f(score, column) over columns [lo, hi) by `width` lanes, this one being `me`; a lane takes its columns in
// ascending order
template <bool BF16, int U, typename F>
__device__ __forceinline__ void for_columns(const void* s, int64_t lo, int64_t hi, int me, int width, F f) {
    constexpr int N = Vec<BF16>::N;
    int64_t i = lo + (int64_t)me * N;
    const int64_t step = (int64_t)width * N;
    for (; i + (U - 1) * step + N <= hi; i += U * step) {
        Vec<BF16> v[U];
#pragma unroll
        for (int k = 0; k < U; ++k) v[k].load(s, i + k * step);
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j) f(v[k].v[j], i + k * step + j);
    }
#pragma unroll 1
    for (; i < hi; i += step) {
        Vec<BF16> v;
        if (i + N <= hi)
            v.load(s, i);
        else
            v.load_tail(s, i, hi);
#pragma unroll
        for (int j = 0; j < N; ++j) f(v.v[j], i + j);
    }
}

// the order key of a score; 0 for the excluded ones (NaN, -inf).  -0 ranks with +0
__device__ __forceinline__ uint32_t score_key(float s) {
    return s > -INFINITY ? ord_f32(s + 0.0f) : 0u;
}
__device__ __forceinline__ uint64_t column_key(float s, int64_t i) {
    return (uint64_t)score_key(s) << 32 | (0xffffffffu - (uint32_t)i);
}

// 2^(y + e) for y <= 0: y = n + f, |f| <= 1/2, and the Taylor polynomial of e^(f ln 2) of degree 11, whose
// coefficients are ln(2)^k / k! (remainder below 0.347^12 / 12! < 7e-15)
__device__ __forceinline__ double exp2_f64(double y, int e) {
    y = fmax(y, -1100.0);
    const double big = y + 6755399441055744.0;  // 1.5 * 2^52: the low word is rint(y)
    const double f = y - (big - 6755399441055744.0);
    constexpr double L = 0.69314718055994530942;
    constexpr double c2 = L * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5, c6 = c5 * L / 6, c7 = c6 * L / 7,
                     c8 = c7 * L / 8, c9 = c8 * L / 9, c10 = c9 * L / 10, c11 = c10 * L / 11;
    double r = fma(c11, f, c10);
    r = fma(r, f, c9);
    r = fma(r, f, c8);
    r = fma(r, f, c7);
    r = fma(r, f, c6);
    r = fma(r, f, c5);
    r = fma(r, f, c4);
    r = fma(r, f, c3);
    r = fma(r, f, c2);
    r = fma(r, f, L);
    r = fma(r, f, 1.0);
    return ldexp(r, (int)(uint32_t)__double_as_longlong(big) + e);
}

// Weights against the row's best score m: exp((s - m) / T), 1 for s == m (an infinite m too), 0 for excluded ones
struct Weigh {
    double m, c;  // c = log2(e) / T
    float top;
    int unit;     // log2 of the fixed-point unit
    __device__ __forceinline__ double operator()(float s) const {
        const double w = exp2_f64(((double)s - m) * c, 0);
        return s == top ? 1.0 : s > -INFINITY ? w : 0.0;
    }
    // w in units of 2^-unit, rounded; w 2^unit <= 2^51, so that adding 2^52 leaves it in the low bits
    __device__ __forceinline__ uint64_t fixed(float s) const {
        const double w = exp2_f64(((double)s - m) * c, unit) + 4503599627370496.0;
        const uint64_t v = (uint64_t)__double_as_longlong(w) & 0xfffffffffffffull;
        return s == top ? 1ull << unit : s > -INFINITY ? v : 0ull;
    }
};

// ------------------------------------------------------------------------------------ wave and workgroup steps
__device__ __forceinline__ double shfl_f64(double v, int src) { return __longlong_as_double((int64_t)shfl_u64(__double_as_longlong(v), src)); }
__device__ __forceinline__ double shfl_xor_f64(double v, int m) { return __longlong_as_double((int64_t)shfl_xor_u64(__double_as_longlong(v), m)); }

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += shfl_xor_f64(v, o);
    return v;
}
__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += shfl_xor_u64(v, o);
    return v;
}
// inclusive prefix sums over the lanes
__device__ __forceinline__ double wave_scan_f64(double v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double t = shfl_f64(v, lane >= o ? lane - o : lane);
        if (lane >= o) v += t;
    }
    return v;
}
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t t = shfl_u64(v, lane >= o ? lane - o : lane);
        if (lane >= o) v += t;
    }
    return v;
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
    v = wave_sum_u64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t s = 0;
    for (int i = 0; i < kWaves; ++i) s += sh.part[i];
    return s;
}
__device__ uint64_t block_max_u64(uint64_t v, Shared& sh) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, shfl_xor_u64(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t s = 0;
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
// it; the last bin that holds anything if the whole falls short.  -> sh.bin, sh.below = the sum before it
__device__ void find_bin(double target, Shared& sh) {
    __syncthreads();
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        constexpr int per = kBins / 64;
        uint64_t own = 0;
        for (int j = 0; j < per; ++j) own += sh.hist[lane * per + j];
        const uint64_t incl = wave_scan_u64(own, lane);
        const uint64_t hit = __ballot(own > 0 && (double)incl >= target);
        const uint64_t any = __ballot(own > 0);
        const int pick = hit ? __builtin_ctzll(hit) : any ? 63 - __builtin_clzll(any) : 0;
        if (lane == pick) {
            uint64_t run = incl - own;
            int last = lane * per;
            uint64_t at = run;
            for (int j = 0; j < per; ++j) {
                const uint64_t h = sh.hist[lane * per + j];
                if (!h) continue;
                last = lane * per + j;
                at = run;
                if ((double)(run + h) >= target) break;
                run += h;
            }
            sh.bin = (uint32_t)last;
            sh.below = at;
        }
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
        double run = wave_scan_f64(own, lane) - own;
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

// what one reading of a row (or a part of it) gives
struct Top {
    uint64_t best;  // largest column key
    uint64_t live;  // columns that are not excluded
    float low;      // smallest live score above -1e30 (lower ones are masks, and share the last bin)
};
template <bool BF16>
__device__ __forceinline__ Top scan_top(const void* s, int64_t lo, int64_t hi, int me, int width) {
    float best = -INFINITY, low = INFINITY;
    int64_t at = -1;
    uint32_t live = 0;
    for_columns<BF16, 2>(s, lo, hi, me, width, [&](float v, int64_t i) {
        if (v > best) {
            best = v;
            at = i;
        }
        live += v > -INFINITY;
        if (v > -1e30f) low = fminf(low, v);
    });
    return Top{at < 0 ? 0ull : column_key(best, at), live, low};
}

// equal steps of the distance to the best score; 0 is the best bin
struct Binning {
    float top, inv;
    __device__ __forceinline__ int operator()(float s) const {
        // NaN and -inf never get here; top - s is inf at most
        return s == top ? 0 : (int)fminf((top - s) * inv, (float)(kBins - 1));
    }
};
__device__ __forceinline__ Binning make_binning(float top, float low, double reach) {
    const double range = fmin((double)top - (double)low, reach);
    // at least one f32 step per bin; an infinite or undefined range leaves all in bin 0 or the last one
    const double inv = (double)(kBins - 1) / range;
    return Binning{top, inv < 1e37 && inv > 0.0 ? (float)inv : inv > 0.0 ? 1e37f : 0.0f};
}

// The cut of top_k (MASS false: `target` columns) or top_p (`target` of the fixed weights), among the columns of
// key >= cut, by descent over the score bits; ties are counted off in column order
template <bool BF16, bool MASS>
__device__ uint64_t descend(const void* s, int cols, uint64_t cut, double target, const Weigh& weigh, Shared& sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t above = 0;   // counted in better bins than this digit's
    uint32_t prefix = 0;  // the score bits found so far
#pragma unroll 1
    for (int digit = 0; digit < 3; ++digit) {
        const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
        const int open = digit == 0 ? 32 : digit == 1 ? 21 : 10;  // bits not yet found
        const uint32_t mask = (1u << (open - shift)) - 1u;
        clear_hist(sh);
        for_columns<BF16, 1>(s, 0, cols, tid, kThreads, [&](float v, int64_t i) {
            const uint64_t key = column_key(v, i);
            const uint32_t k = (uint32_t)(key >> 32);
            if (k && key >= cut && (open == 32 || (k >> open) == (prefix >> open)))
                atomicAdd((unsigned long long*)&sh.hist[mask - ((k >> shift) & mask)],
                          (unsigned long long)(MASS ? weigh.fixed(v) : 1ull));
        });
        find_bin(target - (double)above, sh);
        prefix |= (mask - sh.bin) << shift;
        above += sh.below;
    }
    __syncthreads();
    const uint64_t each = MASS ? max(weigh.fixed(unord_f32(prefix)), (uint64_t)1) : 1ull;
    const double want_f = ceil((target - (double)above) / (double)each);
    int64_t want = want_f < 1.0 ? 1 : (int64_t)fmin(want_f, (double)cols);
    int64_t found = -1;  // the column of the last one taken
    for (int64_t i0 = 0; i0 < cols; i0 += kThreads) {
        const int64_t i = i0 + tid;
        const uint64_t key = i < cols ? column_key(load_score<BF16>(s, i), i) : 0ull;
        const bool eq = (uint32_t)(key >> 32) == prefix && key >= cut;
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
        if (eq && before < want) found = i;
        want -= all;
        if (want <= 0) break;
    }
    const uint64_t last = block_max_u64((uint64_t)(found + 1), sh);
    return max(cut, (uint64_t)prefix << 32 | (0xffffffffu - (uint32_t)(last - 1)));
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
    const uint64_t live = block_sum_u64(mine.live, sh);
    if (live == 0 || !(r.T > 0.0) || r.top_k == 1) {
        for (int64_t j = tid; j < a.n_draws; j += kThreads) {
            a.out_idx[row * a.n_draws + j] = live ? key_index(best) : -1;
            if (a.out_prob) a.out_prob[row * a.n_draws + j] = live ? 1.0f : 0.0f;
        }
        return;
    }
    const float low = unord_f32(~(uint32_t)block_max_u64((uint64_t)(~ord_f32(mine.low)), sh));
    const float top = key_score(best);
    int unit = 62;  // the sum of all weights is at most cols
    while (unit > 0 && (1ll << (62 - unit)) < (int64_t)cols) --unit;
    const Weigh weigh{(double)top, 1.4426950408889634074 / r.T, top, min(unit, 51)};

    uint64_t cut = 1ull << 32;  // every column with a score
    if (r.top_k > 0 && (uint64_t)r.top_k < live) {
        const Binning bin = make_binning(top, low, INFINITY);
        clear_hist(sh);
        for_columns<BF16, 2>(s, 0, cols, tid, kThreads, [&](float v, int64_t) {
            if (v > -INFINITY) atomicAdd((unsigned*)&sh.hist[bin(v)], 1u);
        });
        find_bin((double)r.top_k, sh);
        const int b = (int)sh.bin;
        const uint64_t before = sh.below, in_bin = sh.hist[b];
        const bool list = before + in_bin <= kList;
        if (list || in_bin <= kList) {
            for_columns<BF16, 2>(s, 0, cols, tid, kThreads, [&](float v, int64_t i) {
                if (v > -INFINITY) {
                    const int at = bin(v);
                    if (list ? at <= b : at == b) sh.key[atomicAdd(&sh.n, 1u)] = column_key(v, i);
                }
            });
            __syncthreads();
            if (list) {
                finish_list(a, row, r, (int)(before + in_bin), weigh, sh);
                return;
            }
            sort_keys((int)in_bin, sh);
            cut = sh.key[(uint64_t)r.top_k - before - 1];
        } else {
            cut = descend<BF16, false>(s, cols, cut, (double)r.top_k, weigh, sh);
        }
    }
    if (r.top_p < 1.0) {
        // a column of weight below (1 - p) Z / cols is never kept (all such together weigh less than the
        // (1 - p) Z that are dropped), and Z >= 1
        const double reach = r.T * (log((double)cols / (1.0 - r.top_p)) + 1e-3);
        const Binning bin = make_binning(top, low, reach);
        clear_hist(sh);
        for_columns<BF16, 1>(s, 0, cols, tid, kThreads, [&](float v, int64_t i) {
            if (column_key(v, i) >= cut) atomicAdd((unsigned long long*)&sh.hist[bin(v)], (unsigned long long)weigh.fixed(v));
        });
        __syncthreads();
        uint64_t sum = 0;
        for (int j = tid; j < kBins; j += kThreads) sum += sh.hist[j];
        const double target = r.top_p * (double)block_sum_u64(sum, sh);
        find_bin(target, sh);
        const int b = (int)sh.bin;
        const uint64_t before = sh.below;
        for_columns<BF16, 2>(s, 0, cols, tid, kThreads, [&](float v, int64_t i) {
            const uint64_t key = column_key(v, i);
            if (key >= cut && bin(v) == b) {
                const uint32_t at = atomicAdd(&sh.n, 1u);
                if (at < kList) sh.key[at] = key;
            }
        });
        __syncthreads();
        const int n = (int)min(sh.n, (uint32_t)kList + 1);
        if (n <= kList) {
            sort_keys(n, sh);
            // the last column whose sum before it is below the target
            for (int j = tid; j < n; j += kThreads) sh.hist[j] = weigh.fixed(key_score(sh.key[j]));
            __syncthreads();
            if (tid < 64) {
                constexpr int per = kList / 64;
                const int lo = lane * per, hi = min(n, lo + per);
                uint64_t own = 0;
                for (int j = lo; j < hi; ++j) own += sh.hist[j];
                uint64_t run = before + wave_scan_u64(own, lane) - own;
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
            cut = max(cut, sh.key[sh.bin]);
        } else {
            cut = descend<BF16, true>(s, cols, cut, target, weigh, sh);
        }
    }

    // weights of the kept columns, summed per segment
    constexpr int kStep = 64 * N;
    const int64_t seg_len = ((int64_t)cols + kSegs * kStep - 1) / (kSegs * kStep) * kStep;
    const int n_segs = (int)(((int64_t)cols + seg_len - 1) / seg_len);
    auto kept = [&](float v, int64_t i) -> double {
        const double w = column_key(v, i) >= cut ? weigh(v) : 0.0;
        return w >= r.min_p ? w : 0.0;
    };
    __syncthreads();
    for (int g = wave; g < n_segs; g += kWaves) {
        double w = 0.0;
        for_columns<BF16, 1>(s, g * seg_len, min((int64_t)cols, (g + 1) * seg_len), lane, 64,
                             [&](float v, int64_t i) { w += kept(v, i); });
        w = wave_sum_f64(w);
        if (lane == 0) sh.seg[g + 1] = w;
    }
    __syncthreads();
    if (tid < 64) {
        constexpr int per = kSegs / 64;
        const int lo = lane * per, hi = min(n_segs, lo + per);
        double own = 0.0;
        for (int j = lo; j < hi; ++j) own += sh.seg[j + 1];
        double run = wave_scan_f64(own, lane) - own;
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
            for (int k = 0; k < N; ++k) own += w[k] = kept(v.v[k], i + k);
            double c = run + wave_scan_f64(own, lane) - own;
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
