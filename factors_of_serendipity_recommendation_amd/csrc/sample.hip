// Draws from score rows: temperature, top-k, top-p and min-p, from given random numbers.
//
// The kept columns are a prefix of the row's ranking (score descending, ties to the lower column), so they are
// described by one 64-bit key (wave_topk.h's make_key): column i is kept iff its key is at least the cut.
// top_k: the columns (or one chunk in several) are cut into kThreads x 4 classes; the top_k-th largest of the classes' best
// scores is at most the row's top_k-th largest score, so that what reaches it holds the top_k columns.  One reading of the row
// gathers those as a list in LDS, and everything else happens on that list.
// top_p: a histogram of the distances to the best score, in 4096 equal steps, counts columns; a count times the weight
// at the columns' mean place in the step is close enough to name the step or two in which the running weight reaches its target.
// The next reading sums the exact weights of everything better, and gathers those steps' columns, among which the cut is
// found.  What does not fit (a top_k of thousands, sums that show the cut elsewhere) takes a descent over the 32 score bits, by
// one workgroup also where several share a row: 1 x 1M f32 with top_k 1024 37 us, 1025 333, 5000 415; 64 x 1M 117, 470, 512; 2048 x
// 40,981 with top_k 1000 132, 5000 210.
// Without restrictions one reading does, each segment of the row weighed against its own best score.
//
// Which column a given number draws depends on every weight before it, and with a million columns the borders
// between columns lie 1e-6 of the total apart, so 24 bits are not enough: weights are computed in f64 and
// summed in f64 in a fixed order, and what atomics add are integers (so that their order does not matter): the columns of a list
// or of top_p's window in units of 2^-51 and 2^-49 of the best weight, which 64 bits hold thousands of, rows of any length in 2^-84.
//
// Bounds: a reading runs at up to 5.6 TB/s; the exact sums take 29 vector instructions a step of 64 columns, 16 of them the
// weight (2 of the difference, 4 of the exponent's split, a polynomial of degree 9, the scaling), 4 cycles each at the 2.0 GHz that
// this arithmetic holds: 512 x 1M f32 with top_p in 0.5 ms against 0.36 for reading it.
#include "wave_topk.h"

#include <algorithm>

namespace lgx {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 4096;  // of 32 bits, or half as many of 64
constexpr int kTopBins = 512;  // the first of them, whose columns' places within the step are summed too
constexpr int kList = 2048;  // columns that are gathered in LDS
constexpr int kFar = 8192;   // and in the workspace, of a row that several workgroups share
constexpr int kAim = 384;  // columns a list is made of, where one chunk in several is looked at first
constexpr int kShort = 160;  // columns that are compared with each other, a step per pair, instead of placed
constexpr int kSegs = 1024;  // column segments with sums of their own: a draw scans one of them

// The columns' segments, at most kSegs: of up to eight steps of a wave each (so that their one reduction is shared), and as
// many for every wave of the `parts` workgroups of a row
struct Segments {
    static constexpr int64_t kStep = 64 * 4;
    int64_t len;
    int n, part;  // a workgroup's
    Segments(int64_t cols, int64_t n_draws, int parts = 1) {
        const int64_t waves = kWaves * parts, steps = (cols + kStep * waves - 1) / (kStep * waves);
        // a segment's reduction costs about a third of a step of its sum, and a draw scans one segment
        int64_t most = 8;
        while (most > 1 && 3 * most * most * n_draws > steps * waves) --most;
        int64_t each = (steps + most - 1) / most;
        if (most > 1) {
            const int64_t more = (steps + most - 2) / (most - 1);  // a step shorter, if that leaves a wave fewer empty ones
            if (more * ((steps + more - 1) / more) < each * ((steps + each - 1) / each)) each = more;
        }
        if (each > kSegs / waves) each = kSegs / waves;
        len = (steps + each - 1) / each * kStep;
        n = (int)((cols + len - 1) / len);
        part = kWaves * (int)each;
    }
    int parts() const { return (n + part - 1) / part; }
};

// whether a row that one workgroup takes is drawn from by running weights of groups of columns instead of segments
constexpr int kGroup = 16;
__host__ __device__ __forceinline__ bool grouped(int64_t cols, int64_t n_draws) {
    return cols <= kList || (cols <= kGroup * kList && n_draws > kWaves);
}

struct SampleArgs {
    const void* S;
    int64_t rows, cols, ld;
    const void* u;
    int u_f64, rows_f64;
    int64_t n_draws;
    double T, top_p, min_p;
    int64_t top_k;
    const void *T_rows, *p_rows, *m_rows;  // f32, or f64 (rows_f64)
    const int32_t* k_rows;
    int32_t* out_idx;
    float* out_prob;
    Segments segs;  // of a row that one workgroup takes
};

// ------------------------------------------------------------------------------------ scores and weights
template <bool BF16>
__device__ __forceinline__ float load_score(const void* s, int64_t i) {
    return BF16 ? bf16_to_f32(static_cast<const uint16_t*>(s)[i]) : static_cast<const float*>(s)[i];
}

// four scores from any element offset, as they lie in memory: what is on its way is not looked at
template <bool BF16>
struct Vec {
    static constexpr int N = 4;
    using F = float __attribute__((ext_vector_type(4), aligned(4)));
    using U = uint32_t __attribute__((ext_vector_type(2), aligned(2)));
    F f;
    U u;
    __device__ __forceinline__ void load(const void* s, int64_t i) {
        if (BF16)
            u = *reinterpret_cast<const U*>(static_cast<const uint16_t*>(s) + i);
        else
            f = *reinterpret_cast<const F*>(static_cast<const float*>(s) + i);
    }
    __device__ __forceinline__ void none() {  // four excluded scores
        f = F{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        u = U{0xff80ff80u, 0xff80ff80u};
    }
    // the values are there from here on (a loop that enters with loads on their way would wait for its own first thing)
    __device__ __forceinline__ void arrive() {
        if (BF16)
            asm volatile("" : "+v"(u));
        else
            asm volatile("" : "+v"(f));
    }
    __device__ __forceinline__ void values(float (&v)[4]) const {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = BF16 ? __uint_as_float(j % 2 ? u[j / 2] & 0xffff0000u : u[j / 2] << 16) : f[j];
    }
};
// columns at or past `end` as -inf, which no step takes
template <bool BF16>
__device__ __forceinline__ void load_tail(float (&v)[4], const void* s, int64_t i, int64_t end) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i + j < end ? load_score<BF16>(s, i + j) : -INFINITY;
}

// f(four scores, column of the first) over columns [lo, hi) by `width` lanes, this one being `me`; a lane takes
// its columns in ascending order.  U = 1, 2: so many groups at a time with the next ones on their way (f takes long); U = 4, 8:
// so many on their way at once (8 bytes each of bf16 rows: 1024 x 91,599, top_k 100, 73.5 us with eight, 78.6 with four).  What is
// past the end comes as -inf
template <bool BF16, int U, typename F>
__device__ __forceinline__ void for_groups(const void* s, int64_t lo, int64_t hi, int me, int width, F f) {
    constexpr int N = Vec<BF16>::N;
    const int64_t step = (int64_t)width * N, whole = lo + (hi - lo) / N * N;  // the end of the whole groups
    int64_t i = lo + (int64_t)me * N;
    Vec<BF16> v[U];
    auto take = [&](const Vec<BF16>& g, int64_t at) {
        float x[4];
        g.values(x);
        f(x, (int)at);
    };
    if (U >= 4) {
#pragma unroll 1
        for (; i < whole; i += U * step) {
#pragma unroll
            for (int k = 0; k < U; ++k) {
                v[k].none();
                if (i + k * step < whole) v[k].load(s, i + k * step);
            }
#pragma unroll
            for (int k = 0; k < U; ++k) take(v[k], i + k * step);
        }
    } else {
        const int64_t last = whole - N - (U - 1) * step;  // the last place of U whole groups
        bool more = i <= last;
        if (more) {
            for (int k = 0; k < U; ++k) v[k].load(s, i + k * step);
            for (int k = 0; k < U; ++k) v[k].arrive();
        }
#pragma unroll 1
        while (more) {
            Vec<BF16> next[U];
            const int64_t at = i;
            i += U * step;
            more = i <= last;
            if (more)
                for (int k = 0; k < U; ++k) next[k].load(s, i + k * step);
            for (int k = 0; k < U; ++k) take(v[k], at + k * step);
            for (int k = 0; k < U; ++k) v[k] = next[k];
        }
        if (U > 1 && i < whole) {  // one group less
            v[0].load(s, i);
            take(v[0], i);
        }
    }
    if (whole < hi && (whole - lo) / N % width == me) {  // the lane whose turn it is takes the last columns
        float x[4];
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = whole + j < hi ? load_score<BF16>(s, whole + j) : -INFINITY;
        f(x, (int)whole);
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
    int unit;      // log2 of the fixed-point unit of a list's weights, of which 64 bits hold 2^12
    __device__ __forceinline__ Weigh(float top, double T) {
        m = (double)top;
        c = 1.4426950408889634074 / fmin(T, 1e300);
        floor = -1100.0 / c;
        unit = 51;
    }
    template <int N>
    __device__ __forceinline__ void scaled(const float (&s)[N], int e, double (&w)[N]) const {
        if (N > 2) {
            const float s0[2] = {s[0], s[1 % N]}, s1[2] = {s[2 % N], s[3 % N]};
            double w0[2], w1[2];
            scaled<2>(s0, e, w0);
            scaled<2>(s1, e, w1);
            w[0] = w0[0]; w[1 % N] = w0[1]; w[2 % N] = w1[0]; w[3 % N] = w1[1];
            return;
        }
        double f[N];
        int n[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const double d = fmax((double)s[j] - m, floor);
            const double big = fma(d, c, 6755399441055744.0);  // 1.5 * 2^52: the low word is n
            f[j] = fma(d, c, 6755399441055744.0 - big);
            n[j] = (int)(uint32_t)__double_as_longlong(big) + e;
            w[j] = 1.0203121063391729e-07;
        }
        // step by step over all of them: one after the other they would wait for each step
        constexpr double k[8] = {1.3255224878668817e-06, 1.525268684626772e-05, 0.00015403455852453838, 0.0013333558179043112,
                                 0.009618129159402558, 0.055504108664760424, 0.2402265069581299, 0.6931471805599453};
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) w[j] = fma_const(w[j], f[j], k[i]);
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = ldexp(fma(w[j], f[j], 1.0), n[j]);
    }
    __device__ __forceinline__ double scaled(float s, int e) const {
        const float v[1] = {s};
        double w[1];
        scaled<1>(v, e, w);
        return w[0];
    }
    __device__ __forceinline__ double operator()(float s) const { return scaled(s, 0); }
    // w in units of 2^-unit, rounded; w 2^unit <= 2^51, so that adding 2^52 leaves it in the low bits
    __device__ __forceinline__ uint64_t fixed(float s) const {
        const double w = scaled(s, unit) + 4503599627370496.0;
        return (uint64_t)__double_as_longlong(w) & 0xfffffffffffffull;
    }
    // the same, but at least 1 for a weight that f64 does not round to 0: a column that is kept can be drawn
    __device__ __forceinline__ uint64_t fixed_kept(float s) const {
        return max(fixed(s), (uint64_t)(scaled(s, 0) > 0.0 ? 1 : 0));
    }
};

// ------------------------------------------------------------------------------------ wave and workgroup steps
__device__ __forceinline__ double shfl_f64(double v, int src) { return __longlong_as_double((int64_t)shfl_u64(__double_as_longlong(v), src)); }

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

struct alignas(16) Pair {
    uint64_t w, key;
};
struct Shared {
    union {
        uint64_t wide[kBins / 2];
        uint32_t count[kBins];
        struct {
            Pair pair[kShort];
            float prob[kShort];
        };
        float seg_top[kSegs];  // the segments' own best scores
    };
    uint64_t place[kTopBins];  // in 2^-16 of a step
    uint64_t key[kList];       // gathered columns
    union {
        double w[kList];  // their weights, then the running sums of the kept ones
        double seg[kSegs + 1];
    };
    uint64_t part[kWaves];
    double dpart[kWaves];
    uint64_t below, below2;
    uint32_t bin, bin2, bin3, n;
};

// sum / maximum over the workgroup, the same value in every thread
__device__ __forceinline__ uint64_t block_sum_u64(uint64_t v, Shared& sh) {
    v = wave_scan_u64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t s = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) s += sh.part[i];
    return s;
}
__device__ __forceinline__ uint64_t block_max_u64(uint64_t v, Shared& sh) {
    v = wave_max_u64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t s = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) s = max(s, sh.part[i]);
    return s;
}

// the maximum of a and of b
__device__ __forceinline__ void block_max2(uint32_t& a, uint32_t& b, Shared& sh) {
    const uint64_t x = wave_max_u64(a), y = wave_max_u64(b);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.part[threadIdx.x >> 6] = x << 32 | y;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        a = max(a, (uint32_t)(sh.part[i] >> 32));
        b = max(b, (uint32_t)sh.part[i]);
    }
}
__device__ __forceinline__ double block_sum_f64(double v, Shared& sh) {
    v = wave_scan_f64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.dpart[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) s += sh.dpart[i];
    return s;
}

__device__ __forceinline__ void clear_hist(Shared& sh) {
    __syncthreads();
    for (int j = threadIdx.x; j < kBins / 2; j += kThreads) sh.wide[j] = 0;
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
}

// The bin in which the running sum of the histogram, from bin 0 on, reaches `target`: sum before it < target <= sum with
// it; the last bin that holds anything if the whole falls short, bin 0 of an empty histogram.
// -> sh.bin, sh.below = the sum before it
template <typename C>
__device__ __forceinline__ void find_bin(const C* hist, double target, Shared& sh) {
    constexpr int per = kBins * 4 / (int)sizeof(C) / kThreads;
    const int tid = threadIdx.x;
    if (tid == 0) {
        sh.bin = 0;
        sh.below = 0;
    }
    __syncthreads();
    uint64_t own = 0;
    for (int j = 0; j < per; ++j) own += hist[tid * per + j];
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
    // one thread holds it (with a target of 0 or less: the first bin that holds anything)
    if (own && (double)(run + own) >= target && (run == 0 || (double)run < target))
        for (int j = 0; j < per; ++j) {
            const uint64_t h = hist[tid * per + j], next = run + h;
            if (h && (double)next >= target) {
                sh.bin = (uint32_t)(tid * per + j);
                sh.below = run;
                break;
            }
            run = next;
        }
    __syncthreads();
}

// The same over kThreads bins of 64 bits in sh.wide, a thread each; needs a sum above 0.  A target past the sum counts as
// the sum.
__device__ __forceinline__ void clear_fine(Shared& sh) {
    __syncthreads();
    sh.wide[threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
}
__device__ __forceinline__ void find_fine(double target, Shared& sh) {
    const int tid = threadIdx.x;
    __syncthreads();
    const uint64_t own = sh.wide[tid], incl = wave_scan_u64(own);
    if ((tid & 63) == 63) sh.part[tid >> 6] = incl;
    __syncthreads();
    uint64_t run = incl - own, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < (tid >> 6)) run += sh.part[w];
        all += sh.part[w];
    }
    target = fmin(target, (double)all);
    if (own && (double)(run + own) >= target && (run == 0 || (double)run < target)) {
        sh.bin = (uint32_t)tid;
        sh.below = run;
    }
    __syncthreads();
}

// what the wave's lanes wrote to LDS is there for its other lanes (its LDS instructions run in order)
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// bitonic sort of sh.key[0, n), descending, n <= kList; keys past n become 0
__device__ __forceinline__ void sort_keys(int n, Shared& sh) {
    int size = 64;
    while (size < n) size <<= 1;
    __syncthreads();
    for (int j = threadIdx.x; j < size; j += kThreads)
        if (j >= n) sh.key[j] = 0;
    for (int k = 2; k <= size; k <<= 1)
        for (int d = k >> 1; d > 0; d >>= 1) {
            // up to a distance of 64 a wave works on 128 keys of its own
            if (k == 2 || d >= 64)
                __syncthreads();
            else
                wave_lds_order();
            for (int t = threadIdx.x; t < size / 2; t += kThreads) {
                const int i = 2 * t - (t & (d - 1));
                const uint64_t x = sh.key[i], y = sh.key[i + d];
                if ((x < y) == ((i & k) == 0)) {
                    sh.key[i] = y;
                    sh.key[i + d] = x;
                }
            }
        }
    __syncthreads();
}

// v[0, n), n <= PER * kThreads, in LDS -> its inclusive running sums, in order; the last place above 0 (0 without one)
template <int PER>
__device__ __forceinline__ int running_sums(double* v, int n, Shared& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lo = threadIdx.x * PER;
    double x[PER], own = 0.0;
    uint32_t last = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        x[j] = lo + j < n ? v[lo + j] : 0.0;
        own += x[j];
        if (x[j] > 0.0) last = lo + j;
    }
    const double incl = wave_scan_f64(own);
    if (lane == 63) sh.dpart[wave] = incl;
    __syncthreads();
    double run = incl - own;
    for (int w = 0; w < wave; ++w) run += sh.dpart[w];
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (lo + j < n) v[lo + j] = run += x[j];
    return (int)block_max_u64(last, sh);
}

// ------------------------------------------------------------------------------------ one row
struct Row {
    double T, top_p, min_p;
    int64_t top_k;
};
__device__ __forceinline__ Row row_settings(const SampleArgs& a, int64_t row) {
    Row r;
    const auto setting = [&](const void* of_rows, double all) {
        return !of_rows ? all : a.rows_f64 ? static_cast<const double*>(of_rows)[row] : (double)static_cast<const float*>(of_rows)[row];
    };
    r.T = setting(a.T_rows, a.T);
    if (r.T > 0.0) r.T = fmax(r.T, 1e-300);  // below it 1 / T is none, and no two f32 scores lie so near anyway
    r.top_p = setting(a.p_rows, a.top_p);
    // within 1e-15 of top_p is reached: of equal weights that lie on it to the last bit (0.9 of ten), a sum's order and what weighs
    // next to nothing would decide
    if (r.top_p < 1.0) r.top_p *= 1.0 - 1e-15;
    const double m = setting(a.m_rows, a.min_p);
    r.min_p = m > 0.0 ? fmin(m, 1.0) : 0.0;
    r.top_k = a.k_rows ? (int64_t)a.k_rows[row] : a.top_k;
    return r;
}
__device__ __forceinline__ double draw_number(const SampleArgs& a, int64_t row, int64_t j) {
    const int64_t i = row * a.n_draws + j;
    const double u = a.u_f64 ? static_cast<const double*>(a.u)[i] : (double)static_cast<const float*>(a.u)[i];
    return fmin(fmax(u, 0.0), 1.0);
}

// The larger of two scores, the number of a number and a NaN; NaN of two NaN, which the next maximum with a number drops
__device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }

// the best of the columns [lo, hi) as a key, 0 without one
template <bool BF16>
__device__ __forceinline__ uint64_t scan_best(const void* s, int64_t lo, int64_t hi, int me, int width) {
    float best = kNone;
    int at = -1;
    for_groups<BF16, BF16 ? 8 : 4>(s, lo, hi, me, width, [&](const float (&v)[4], int i) {
        if (max_of(max_of(v[0], v[1]), max_of(v[2], v[3])) > best) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (v[j] > best) {
                    best = v[j];
                    at = i + j;
                }
        }
    });
    return at < 0 ? 0ull : column_key(best, at);
}

// equal steps of the distance to the best score.  A score belongs to bin b < kBins - 1 iff b <= at(s) < b + 1,
// what is farther (and NaN) to the last one
struct Binning {
    float top, inv;
    // of kThreads bins
    __device__ __forceinline__ int fine(float s) const { return (int)fminf(at(s), (float)(kThreads - 1)); }
    __device__ __forceinline__ float at(float s) const { return (top - s) * inv; }
    __device__ __forceinline__ int operator()(float s) const { return (int)fminf(at(s), (float)(kBins - 1)); }
};
// the largest score whose distance is at least x steps: at(s) < x iff s is above it (the distance falls with the score)
__device__ __forceinline__ float score_at(const Binning& bin, float x) {
    if (!(bin.at(bin.top) < x)) return bin.top;
    // at(lo) >= x > at(hi); scores above top lie at less than any x > 0.  Every lane tries a place between them
    uint32_t lo = ord_f32(-INFINITY), hi = __builtin_amdgcn_readfirstlane(ord_f32(bin.top));
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 64) / 65, mine = lo + step * ((threadIdx.x & 63) + 1);
        const int n = __popcll(__ballot(mine < hi && !(bin.at(unord_f32(mine)) < x)));
        hi = min(hi, lo + step * (n + 1));
        lo += step * n;
    }
    return unord_f32(lo);
}
__device__ __forceinline__ Binning make_binning(float top, double range, int bins = kBins) {
    const double inv = (double)(bins - 1) / range;  // a range of 0: all the best score's equals in bin 0
    return Binning{top, (float)fmin(inv, 1e30)};
}

// Sums of weights by atomics, for rows of any length: integers, whose order does not matter, of 128 bits in units of 2^-84.  2^31
// weights fit, and what all of them lose to the unit is 2^-53 of the best one (in 64 bits a unit would have to grow with the row:
// of 12M columns that share a score the cut lay 33 off, of 100M 22,743).  A bin's low word is in sh.wide, its high one in sh.key
using u128 = unsigned __int128;
constexpr int kMassUnit = 84;
__device__ __forceinline__ double mass_value(u128 x) {  // in units; never falls as x grows (the high word is below 2^53)
    return fma((double)(uint64_t)(x >> 64), 0x1p64, (double)(uint64_t)x);
}
__device__ __forceinline__ void add_mass(int bin, double w, Shared& sh) {  // w in units
    const uint32_t hi = (uint32_t)(w * 0x1p-64);
    const uint64_t lo = (uint64_t)fma(-(double)hi, 0x1p64, w);
    const uint64_t sum = atomicAdd((unsigned long long*)&sh.wide[bin], (unsigned long long)lo) + lo;
    const uint32_t up = hi + (sum < lo ? 1 : 0);
    if (up) atomicAdd((unsigned long long*)&sh.key[bin], (unsigned long long)up);
}
__device__ __forceinline__ void clear_mass(Shared& sh) {
    static_assert(kList == kBins / 2, "a high word a bin");
    __syncthreads();
    for (int j = threadIdx.x; j < kList; j += kThreads) sh.wide[j] = sh.key[j] = 0;
    __syncthreads();
}
__device__ __forceinline__ u128 bin_mass(int bin, const Shared& sh) { return (u128)sh.key[bin] << 64 | sh.wide[bin]; }
// find_bin over these sums with `base` before them.  The first time the target is that part of the whole
// -> sh.bin, sh.below2 and sh.below = the sum before it, base included
__device__ __forceinline__ void find_mass(double& target, u128 base, bool first, Shared& sh) {
    constexpr int per = kBins / 2 / kThreads;
    const int tid = threadIdx.x, wave = tid >> 6;
    __syncthreads();
    u128 own = 0;
    for (int j = 0; j < per; ++j) own += bin_mass(tid * per + j, sh);
    const u128 incl = ((u128)wave_scan_u64((uint64_t)(own >> 64)) << 64) + ((u128)wave_scan_u64((uint64_t)own >> 32) << 32) +
                      wave_scan_u64((uint32_t)own);
    if ((tid & 63) == 63) {
        sh.part[wave] = (uint64_t)incl;
        sh.dpart[wave] = __longlong_as_double((int64_t)(incl >> 64));
    }
    __syncthreads();
    u128 run = base + incl - own, all = base;
    for (int w = 0; w < kWaves; ++w) {
        const u128 x = (u128)(uint64_t)__double_as_longlong(sh.dpart[w]) << 64 | sh.part[w];
        if (w < wave) run += x;
        all += x;
    }
    const double whole = mass_value(all);
    target = fmin(first ? target * whole : target, whole);
    if (own && mass_value(run + own) >= target && (run == base || mass_value(run) < target))
        for (int j = 0; j < per; ++j) {
            const u128 h = bin_mass(tid * per + j, sh), next = run + h;
            if (h && mass_value(next) >= target) {
                sh.bin = (uint32_t)(tid * per + j);
                sh.below = (uint64_t)run;
                sh.below2 = (uint64_t)(run >> 64);
                break;
            }
            run = next;
        }
    __syncthreads();
}

// The cut of top_k (MASS false: `target` columns) or top_p (that part of the weights), among the columns that `cut`
// keeps, by descent over the score bits; ties are counted off in column order
template <bool BF16, bool MASS>
__device__ __forceinline__ Cut descend(const void* s, int cols, const Cut& cut, double target, const Weigh& weigh, Shared& sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    u128 above = 0;       // counted in better bins than this digit's
    uint32_t prefix = 0;  // the score bits found so far
#pragma unroll 1
    for (int digit = 0; digit < 3; ++digit) {
        const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
        const int open = digit == 0 ? 32 : digit == 1 ? 21 : 10;  // bits not yet found
        const uint32_t mask = (1u << (open - shift)) - 1u;
        if (MASS) clear_mass(sh); else clear_hist(sh);
        for_groups<BF16, 1>(s, 0, cols, tid, kThreads, [&](const float (&v)[4], int i) {
#pragma unroll 1  // (four copies of it cost the callers registers)
            for (int j = 0; j < 4; ++j) {
                const uint32_t k = score_key(v[j]);
                if (!cut.keeps(v[j], i + j) || (open < 32 && (k >> open) != (prefix >> open))) continue;
                const int bin = (int)(mask - ((k >> shift) & mask));
                if (MASS)
                    add_mass(bin, weigh.scaled(v[j], kMassUnit), sh);
                else
                    atomicAdd((unsigned long long*)&sh.wide[bin], 1ull);
            }
        });
        if (MASS)
            find_mass(target, above, digit == 0, sh);
        else
            find_bin(sh.wide, target - (double)(uint64_t)above, sh);
        prefix |= (mask - sh.bin) << shift;
        if (MASS)
            above = (u128)sh.below2 << 64 | sh.below;
        else
            above += sh.below;
    }
    __syncthreads();
    const float value = unord_f32(prefix);
    const double each = MASS ? weigh.scaled(value, kMassUnit) : 1.0;
    const double want_f = ceil((target - mass_value(above)) / each);
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
// restrictions and the draws on that list, a column per thread.  A column's rank, the weight that ranks before it, and
// the kept weight up to it in column order are sums over the list.
__device__ __forceinline__ void finish_short(const SampleArgs& a, int64_t row, const Row& r, int n, const Weigh& weigh, Shared& sh) {
    const int tid = threadIdx.x;
    const int n_wave = __builtin_amdgcn_readfirstlane(tid) < n ? n : 0;  // waves without a column skip the loops
    const uint64_t mine = tid < n ? sh.key[tid] : 0;
    const double weight = weigh(key_score(mine));
    const uint64_t plain = tid < n ? weigh.fixed(key_score(mine)) : 0;
    const uint64_t w = max(plain, (uint64_t)(tid < n && weight > 0.0 ? 1 : 0));  // to be drawn
    // (weight, key) pairs side by side: a step of the loops is one read
    if (tid < n) sh.pair[tid] = Pair{plain, mine};
    __syncthreads();
    int rank = 0;
    uint64_t better = 0;
#pragma unroll 8
    for (int j = 0; j < n_wave; ++j) {
        const Pair p = sh.pair[j];
        const bool b = p.key > mine;
        rank += b;
        better += b ? p.w : 0;
    }
    bool keep = tid < n && rank < r.top_k;
    if (r.top_p < 1.0) {
        const double target = r.top_p * (double)block_sum_u64(keep ? plain : 0, sh);
        keep &= rank == 0 || (double)better < target;
    }
    keep &= (w > 0) & (weight >= r.min_p);
    __syncthreads();
    if (tid < n) sh.pair[tid].w = keep ? w : 0;
    __syncthreads();
    uint64_t upto = 0;
#pragma unroll 8
    for (int j = 0; j < n_wave; ++j) {
        const Pair p = sh.pair[j];
        upto += (uint32_t)p.key >= (uint32_t)mine ? p.w : 0;  // the low half falls with the column
    }
    const uint64_t total = block_max_u64(keep ? upto : 0, sh);  // (the barriers also end the loop above)
    const float prob = (float)(ldexp(weight, weigh.unit) / (double)total);
    const auto put = [&](int64_t j, uint64_t key, float p) {
        a.out_idx[row * a.n_draws + j] = key_index(key);
        if (a.out_prob) a.out_prob[row * a.n_draws + j] = p;
    };
    // a draw is the column with upto - w <= target < upto; a number at the end of the range counts as the last column's
    if (a.n_draws <= n) {
        for (int j = tid; j < (int)a.n_draws; j += kThreads) sh.pair[j].w = min((uint64_t)(draw_number(a, row, j) * (double)total), total - 1);
        __syncthreads();
        if (keep)
#pragma unroll 4
            for (int j = 0; j < (int)a.n_draws; ++j) {
                const uint64_t target = sh.pair[j].w;
                if ((target < upto) & (target >= upto - w)) put(j, mine, prob);
            }
        return;
    }
    if (tid < n) sh.pair[tid].w = keep ? upto : 0;
    if (tid < n) sh.prob[tid] = prob;
    __syncthreads();
    for (int64_t j = tid; j < a.n_draws; j += kThreads) {
        const uint64_t target = min((uint64_t)(draw_number(a, row, j) * (double)total), total - 1);
        uint64_t least = ~0ull;
        int at = 0;
#pragma unroll 4
        for (int c = 0; c < n; ++c) {
            const uint64_t x = sh.pair[c].w;
            const bool nearer = (x > target) & (x < least);
            least = nearer ? x : least;
            at = nearer ? c : at;
        }
        put(j, sh.pair[at].key, sh.prob[at]);
    }
}

// A longer list is cut to little more than its best top_k: a histogram of its scores names the step of the top_k-th
__device__ __forceinline__ int shrink_list(int n, int64_t top_k, Shared& sh) {
    const int tid = threadIdx.x;
    constexpr int per = kList / kThreads;
    uint64_t mine[per];
    uint32_t most = 0, least = 0;  // order bits, reversed ones
#pragma unroll
    for (int j = 0; j < per; ++j) {
        mine[j] = tid + j * kThreads < n ? sh.key[tid + j * kThreads] : 0;
        const uint32_t order = (uint32_t)(mine[j] >> 32);
        most = max(most, order);
        if (order) least = max(least, ~order);
    }
    block_max2(most, least, sh);
    const float top = unord_f32(most);
    const Binning bin = make_binning(top, (double)top - (double)unord_f32(~least), kThreads);
    clear_fine(sh);
#pragma unroll
    for (int j = 0; j < per; ++j)
        if (mine[j]) atomicAdd((unsigned long long*)&sh.wide[bin.fine(key_score(mine[j]))], 1ull);
    find_fine((double)top_k, sh);
#pragma unroll
    for (int j = 0; j < per; ++j)
        if (mine[j] && bin.fine(key_score(mine[j])) <= (int)sh.bin) sh.key[atomicAdd(&sh.n, 1u)] = mine[j];
    __syncthreads();
    return (int)sh.n;
}

// Of the keys `mine` (each thread's, 0 for none) the last in rank before which less than `target` lies: columns, or MASS: fixed
// weights.  kThreads steps of the score name the step that holds it, whose keys are compared with each other
template <bool MASS>
__device__ __forceinline__ uint64_t list_cut(const uint64_t (&mine)[kList / kThreads], double target, const Weigh& weigh, Shared& sh) {
    constexpr int per = kList / kThreads;
    uint64_t* members = reinterpret_cast<uint64_t*>(sh.w);
    const auto measure = [&](uint64_t key) { return MASS ? weigh.fixed(key_score(key)) : 1ull; };
    uint32_t most = 0, least = 0;  // order bits, reversed ones
#pragma unroll
    for (int j = 0; j < per; ++j)
        if (mine[j]) {
            most = max(most, (uint32_t)(mine[j] >> 32));
            least = max(least, ~(uint32_t)(mine[j] >> 32));
        }
    block_max2(most, least, sh);
    const float top = unord_f32(most);
    const Binning bin = make_binning(top, (double)top - (double)unord_f32(~least), kThreads);
    clear_fine(sh);
#pragma unroll
    for (int j = 0; j < per; ++j)
        if (mine[j]) atomicAdd((unsigned long long*)&sh.wide[bin.fine(key_score(mine[j]))], (unsigned long long)measure(mine[j]));
    find_fine(target, sh);
    const int b = (int)sh.bin;
    const double before = (double)sh.below;
#pragma unroll
    for (int j = 0; j < per; ++j)
        if (mine[j] && bin.fine(key_score(mine[j])) == b) members[atomicAdd(&sh.n, 1u)] = mine[j];
    __syncthreads();
    const int m = (int)sh.n;
    uint64_t last = 0;  // of the keys below the target the smallest, complemented
    for (int c = threadIdx.x; c < m; c += kThreads) {
        uint64_t sum = 0;
        for (int j = 0; j < m; ++j) sum += members[j] > members[c] ? measure(members[j]) : 0;
        if (before + (double)sum < target) last = max(last, ~members[c]);
    }
    return ~block_max_u64(last, sh);
}

// the same for longer lists: cut by rank, and placed in column order by kThreads runs of columns
__device__ __forceinline__ void finish_list(const SampleArgs& a, int64_t row, const Row& r, int n, const Weigh& weigh, Shared& sh) {
    // comparing takes two steps a column, and four times that a draw: 256 x 100 f32, one draw: 10 us, 100 draws: 17; placing 12
    const auto few = [&](int n) { return n + 2 * min((int64_t)n, a.n_draws) <= kShort; };
    if (!few(n) && r.top_k < n) n = shrink_list(n, r.top_k, sh);
    if (few(n)) {
        finish_short(a, row, r, n, weigh, sh);
        return;
    }
    constexpr int per = kList / kThreads;
    uint64_t mine[per], cut = 1;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < per; ++j) mine[j] = threadIdx.x + j * kThreads < n ? sh.key[threadIdx.x + j * kThreads] : 0;
    const auto keep = [&](auto f) {
#pragma unroll
        for (int j = 0; j < per; ++j)
            if (!f(mine[j])) mine[j] = 0;
    };
    if (r.top_k < n) {
        cut = list_cut<false>(mine, (double)r.top_k, weigh, sh);
        keep([&](uint64_t key) { return key >= cut; });
    }
    // min_p cuts a prefix of the ranking; top_p looks at all of top_k
    if (r.top_p < 1.0) {
        uint64_t whole = 0;
#pragma unroll
        for (int j = 0; j < per; ++j) whole += mine[j] ? weigh.fixed(key_score(mine[j])) : 0;
        whole = block_sum_u64(whole, sh);
        cut = list_cut<true>(mine, r.top_p * (double)whole, weigh, sh);
        keep([&](uint64_t key) { return key >= cut; });
    }
    if (r.min_p > 0.0) keep([&](uint64_t key) { return key && weigh(key_score(key)) >= r.min_p; });
    uint32_t last = 0, first = 0;  // columns, the first complemented
#pragma unroll
    for (int j = 0; j < per; ++j)
        if (mine[j]) {
            last = max(last, (uint32_t)key_index(mine[j]));
            first = max(first, ~(uint32_t)key_index(mine[j]));
        }
    block_max2(last, first, sh);
    first = ~first;
    const uint32_t run = (last - first) / kThreads + 1;
    const auto place = [&](uint64_t key) { return ((uint32_t)key_index(key) - first) / run; };
    clear_fine(sh);
#pragma unroll
    for (int j = 0; j < per; ++j)
        if (mine[j]) atomicAdd((unsigned long long*)&sh.wide[place(mine[j])], 1ull);
    __syncthreads();
    const uint64_t own = sh.wide[threadIdx.x], incl = wave_scan_u64(own);
    if ((threadIdx.x & 63) == 63) sh.part[threadIdx.x >> 6] = incl;
    __syncthreads();
    uint64_t begin = incl - own;
    n = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < (int)(threadIdx.x >> 6)) begin += sh.part[w];
        n += (int)sh.part[w];
    }
    sh.wide[threadIdx.x] = begin;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < per; ++j)
        if (mine[j]) sh.key[atomicAdd((unsigned long long*)&sh.wide[place(mine[j])], 1ull)] = mine[j];
    __syncthreads();
    int at[per];
#pragma unroll
    for (int j = 0; j < per; ++j) {
        if (!mine[j]) continue;
        const uint32_t p = place(mine[j]);
        const int end = (int)sh.wide[p];
        at[j] = p ? (int)sh.wide[p - 1] : 0;
        const int begins = at[j];
        for (int c = begins; c < end; ++c) at[j] += key_index(sh.key[c]) < key_index(mine[j]);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < per; ++j)
        if (mine[j]) {
            sh.key[at[j]] = mine[j];
            sh.w[at[j]] = weigh(key_score(mine[j]));
        }
    const int end = running_sums<kList / kThreads>(sh.w, n, sh);  // the last column with any weight
    const double total = sh.w[n - 1];
    for (int64_t j = threadIdx.x; j < a.n_draws; j += kThreads) {
        const double target = draw_number(a, row, j) * total;
        int lo = 0, hi = end;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (sh.w[mid] > target) hi = mid; else lo = mid + 1;
        }
        const uint64_t key = sh.key[lo];
        a.out_idx[row * a.n_draws + j] = key_index(key);
        if (a.out_prob) a.out_prob[row * a.n_draws + j] = (float)(weigh(key_score(key)) / total);
    }
}

// A row with infinite scores: those columns share it equally, and their ranking is the column order
template <bool BF16>
__device__ __forceinline__ void draw_infinite(const SampleArgs& a, int64_t row, const Row& r, const void* s, Shared& sh) {
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

// f(four scores, column of the first) over the segments [g0, g1), done(segment) behind each.  A wave takes a run of them as
// one stream: its addresses are a scalar and the lane's place, and the next step is on its way across their ends
template <bool BF16, typename F, typename D>
__device__ __forceinline__ void for_segments(const void* s, int64_t cols, const Segments& segs, int g0, int g1, F f, D done) {
    constexpr int N = Vec<BF16>::N, kStep = Segments::kStep;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int each = (g1 - g0 + kWaves - 1) / kWaves, last = min(g1, g0 + (wave + 1) * each), per = (int)segs.len / kStep;
    int g = g0 + wave * each, left = per;
    if (g >= last) return;
    const int64_t lo = g * segs.len, hi = min(cols, last * segs.len);
    const int steps = (int)((hi - lo) / kStep);
    const char* at = static_cast<const char*>(s) + lo * (BF16 ? 2 : 4);
    Vec<BF16> v;
    if (steps) {
        v.load(at, lane * N);
        v.arrive();
    }
#pragma unroll 1
    for (int k = 0; k < steps; ++k) {
        Vec<BF16> next;
        at += kStep * (BF16 ? 2 : 4);
        if (k + 1 < steps) next.load(at, lane * N);
        float x[4];
        v.values(x);
        f(x, (int)lo + k * kStep + lane * N);
        if (--left == 0) {
            done(g++);
            left = per;
        }
        v = next;
    }
    if (lo + (int64_t)steps * kStep < hi) {
        const int64_t i = lo + (int64_t)steps * kStep + lane * N;
        float x[4];
        load_tail<BF16>(x, s, i, hi);
        f(x, (int)min(i, hi));
        left = 0;
    }
    if (left < per) done(g);
}

// what the first reading finds: the best scores of the thread's four classes of columns, and a low score that sets the
// width of the steps (of a quarter of the columns, masks of the type's lowest value left out)
struct Maxima {
    float best[4], low;
};
constexpr int64_t kChunk = kThreads * 4;  // columns of one step of the workgroup
// of every `stride`-th chunk of [lo, hi)
template <bool BF16>
__device__ __forceinline__ Maxima scan_maxima(const void* s, int64_t lo, int64_t hi, int64_t stride) {
    Maxima m{{kNone, kNone, kNone, kNone}, INFINITY};
    for_groups<BF16, BF16 ? 8 : 4>(s, lo, hi, threadIdx.x, kThreads * stride, [&](const float (&v)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; ++j) m.best[j] = max_of(m.best[j], v[j]);
        m.low = v[0] > -1e30f ? fminf(m.low, v[0]) : m.low;
    });
    return m;
}
// For a list of about kAim columns of those that reach the top_k-th of the chunks looked at, at least two of them (sorted
// and periodic rows look like others this way)
__device__ __forceinline__ int64_t list_stride(int64_t lo, int64_t hi, int64_t top_k) {
    return max((int64_t)1, min((int64_t)kAim / top_k, (hi - lo) / (2 * kChunk)));
}
__device__ __forceinline__ uint64_t order_of(float f) { return ord_f32(f); }
__device__ __forceinline__ uint64_t reverse_order_of(float f) { return (uint32_t)~ord_f32(f); }
__device__ __forceinline__ float of_reverse_order(uint64_t o) { return unord_f32(~(uint32_t)o); }

// a score that at least k of the workgroup's classes reach, so at least k columns do; kNone without k classes
__device__ __forceinline__ float class_bound(const Maxima& m, int64_t k, Shared& sh) {
    uint32_t least = 0, most = 0;  // reversed order bits, order bits
    uint64_t classes = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (m.best[j] > kNone) {
            ++classes;
            least = max(least, (uint32_t)reverse_order_of(m.best[j]));
            most = max(most, (uint32_t)order_of(m.best[j]));
        }
    if (block_sum_u64(classes, sh) < (uint64_t)k) return kNone;
    block_max2(least, most, sh);
    const float top = unord_f32(most);
    const Binning bin = make_binning(top, (double)top - (double)of_reverse_order(least), kThreads);
    clear_fine(sh);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (m.best[j] > kNone) atomicAdd((unsigned long long*)&sh.wide[bin.fine(m.best[j])], 1ull);
    find_fine((double)k, sh);
    // the least class at or before that bin
    uint64_t bound = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (m.best[j] > kNone && bin.fine(m.best[j]) <= (int)sh.bin) bound = max(bound, reverse_order_of(m.best[j]));
    return of_reverse_order(block_max_u64(bound, sh));
}

// a list keys[0, kList), counted in n beyond that
template <typename Keys, typename Count>
__device__ __forceinline__ void push(Keys keys, Count n, uint64_t key) {
    const uint32_t at = atomicAdd(n, 1u);
    if (at < kList) keys[at] = key;
}
// put(key) for the columns of [lo, hi) that `take` names
template <bool BF16, typename Take, typename Put>
__device__ __forceinline__ void gather(const void* s, int64_t lo, int64_t hi, Take take, Put put) {
    for_groups<BF16, BF16 ? 8 : 4>(s, lo, hi, threadIdx.x, kThreads, [&](const float (&v)[4], int i) {
        if ((int)take(v[0]) | (int)take(v[1]) | (int)take(v[2]) | (int)take(v[3])) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (take(v[j])) put(column_key(v[j], i + j));
        }
    });
}

// Steps of the distance to the best score for top_p.  A column of weight below (1 - p) Z / cols is never kept (all such
// together weigh less than the (1 - p) Z that are dropped), and Z >= 1: that far below the best score is the reach.  What
// lies 12 T below that shares the last step, and adds at most e^-12 (1 - p) to the sums; so does what lies a tenth of the
// range below the low score, which is that of some of the columns.
struct Steps {
    double range, reach, margin;
    // top, low: of the columns looked at.  margin: room above them for the others
    __device__ __forceinline__ Steps(float top, float low, const Row& r, int64_t cols) {
        range = fmax((double)top - (double)low, 0.0);
        reach = fmin(r.T, 1e30) * (log((double)cols / (1.0 - r.top_p)) + 12.0);
        margin = fmin(0.25 * range, 0.25 * reach);
    }
    __device__ __forceinline__ Binning bins(float top, double room) const {
        const float first = (float)((double)top + room);
        return make_binning(first, (double)first - (double)top + fmin(1.1 * range, reach));
    }
};

// counts of the columns [lo, hi) that the cut keeps, without the last step, into sh.count, and the first steps' places.
// top: this thread's best score (one above the first step counts there, and shows by that)
template <bool BF16>
__device__ __forceinline__ void count_steps(const void* s, int64_t lo, int64_t hi, const Binning& bin, const Cut& cut, Shared& sh, float* top = nullptr) {
    const bool all = cut.s == kNone;
    clear_hist(sh);
    for (int j = threadIdx.x; j < kTopBins; j += kThreads) sh.place[j] = 0;
    __syncthreads();
    float best = kNone;
    for_groups<BF16, 2>(s, lo, hi, threadIdx.x, kThreads, [&](const float (&v)[4], int i) {
        if (top) best = max_of(best, max_of(max_of(v[0], v[1]), max_of(v[2], v[3])));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float x = fmaxf(fminf(bin.at(v[j]), (float)(kBins - 1)), 0.0f);  // NaN goes to the last
            const int b = (int)x;
            if ((all | cut.keeps(v[j], i + j)) & (b < kBins - 1)) {
                atomicAdd(&sh.count[b], 1u);
                if (b < kTopBins) atomicAdd((unsigned long long*)&sh.place[b], (unsigned long long)((x - (float)b) * 65536.0f));
            }
        }
    });
    if (top) *top = best;
}

// The steps [first, last] that may hold the column in which the running weight reaches top_p of the whole, and the columns
// in them.  The weight w at the mean place of a step's columns stands for each of them.  Past the first steps, where single
// columns weigh little, the middle is their place: they lie anywhere in the step's width of d, an error of w d / (T sqrt 12)
// each, or of that for all of a step's columns together where they share a score, as bf16 ones do.  Four times its root of
// squares, and 5e-6 of the whole (the slope of their number within a step), are allowed for.  Where that is more than `limit`
// columns, f32 ones fill their step evenly enough for a part of it to do: at most a step to both sides of where the target lies
// in it (0.35 of the limit; they lie 0.01 of a step off).
__device__ __forceinline__ double exp2_step(double distance, const Weigh& weigh) {
    Weigh one = weigh;
    one.m = 0.0;
    return one((float)-distance);
}
struct Window {
    int first, last;
    uint64_t columns;
    float from, to;
    __device__ __forceinline__ bool usable(int limit) const { return last < kBins - 1 && columns > 0 && columns <= limit; }
};
template <bool BF16>
__device__ __forceinline__ Window mass_window(const Binning& bin, double T, double top_p, const Weigh& weigh, int limit, Shared& sh) {
    constexpr int per = kBins / kThreads;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const double wide = 1.0 / (double)bin.inv;
    const int b0 = tid * per;
    double w[per], own = 0.0, square = 0.0;
    uint32_t count[per];
#pragma unroll
    for (int j = 0; j < per; ++j) count[j] = sh.count[b0 + j];
    if (b0 < kTopBins) {
#pragma unroll
        for (int j = 0; j < per; ++j) {
            const float place = (float)sh.place[b0 + j] / (65536.0f * (float)max(count[j], 1u));
            // an empty step above the best score may weigh too much for a number
            w[j] = count[j] ? (double)count[j] * weigh((float)((double)bin.top - wide * (b0 + j + (double)place))) : 0.0;
        }
    } else {
        double x = weigh((float)((double)bin.top - wide * (b0 + 0.5)));
        const double ratio = exp2_step(wide, weigh);
#pragma unroll
        for (int j = 0; j < per; ++j) {
            w[j] = count[j] ? (double)count[j] * x : 0.0;
            square = fma(w[j], BF16 ? w[j] : count[j] ? x : 0.0, square);
            x *= ratio;
        }
    }
#pragma unroll
    for (int j = 0; j < per; ++j) own += w[j];
    const double error = 4.0 * wide / (T * sqrt(12.0)) * sqrt(block_sum_f64(square, sh));
    const double incl = wave_scan_f64(own);
    __syncthreads();
    if (lane == 63) sh.dpart[wave] = incl;
    if (tid == 0) sh.bin = sh.bin2 = sh.bin3 = kBins - 1;
    __syncthreads();
    double run = incl - own, sum = 0.0;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
        if (v < wave) run += sh.dpart[v];
        sum += sh.dpart[v];
    }
    const double all = (1.0 - 1e-13) * sum, t3 = fmin(top_p * sum, all);
    const double t1 = fmax(t3 - 5e-6 * sum - error, 1e-300), t2 = fmin(t3 + 5e-6 * sum + error, all);
#pragma unroll
    for (int j = 0; j < per; ++j) {
        const double next = run + w[j];
        if (next >= t1 && run < t1) sh.bin = b0 + j;
        if (next >= t2 && run < t2) sh.bin2 = b0 + j;
        if (next >= t3 && run < t3) {
            sh.bin3 = b0 + j;
            sh.below = (uint64_t)__double_as_longlong(b0 + j + (t3 - run) / w[j]);
        }
        run = next;
    }
    __syncthreads();
    Window win{(int)sh.bin, (int)sh.bin2, 0, (float)sh.bin, (float)(sh.bin2 + 1)};
    uint64_t inside = 0;
#pragma unroll
    for (int j = 0; j < per; ++j) inside += b0 + j >= win.first && b0 + j <= win.last ? count[j] : 0;
    win.columns = block_sum_u64(inside, sh);
    if (win.columns > (uint64_t)limit) {
        const int b = (int)sh.bin3;
        win = Window{b, b, sh.count[b], (float)b, (float)(b + 1)};
        if (!BF16 && b > 0 && b < kBins - 2) {
            const float at = (float)__longlong_as_double((int64_t)sh.below);
            const uint32_t most = max(max(sh.count[b - 1], sh.count[b + 1]), sh.count[b]);
            const float half = fminf(1.0f, 0.35f * (float)limit / (float)most);
            win = Window{(int)(at - half), (int)(at + half), min((uint64_t)limit, (uint64_t)most), at - half, at + half};
        }
    }
    return win;
}

// One reading of the segments [g0, g1) with exact weights: z = all that the cut keeps, better = what lies before the
// window, sum(g, .) = of that what min_p keeps.  The window's columns are put.  z and better of this lane.
template <bool BF16, bool ALL, bool MASKS, typename Put, typename Sum>
__device__ __forceinline__ void sum_window(const void* s, int64_t cols, const Segments& segs, int g0, int g1, float above, float least,
                                           const Cut& cut, const Weigh& weigh, double min_p, Put put, Sum sum, double& z, double& better) {
    const int lane = threadIdx.x & 63;
    double w = 0.0;
    z = better = 0.0;
    for_segments<BF16>(s, cols, segs, g0, g1, [&](const float (&v)[4], int i) {
        double x[4];
        weigh.scaled<4>(v, 0, x);
        uint64_t in[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool before = v[j] > above;
            if (ALL || cut.keeps(v[j], i + j)) z += x[j];
            if (before) {
                if (MASKS) better += x[j];
                if (!MASKS || x[j] >= min_p) w += x[j];
            }
            in[j] = __ballot(v[j] > least) & ~__ballot(before);
        }
        if (in[0] | in[1] | in[2] | in[3]) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if ((in[j] >> lane & 1) && (ALL || cut.keeps(v[j], i + j))) put(column_key(v[j], i + j));
        }
    }, [&](int g) {
        if (!MASKS) better += w;
        w = wave_scan_f64(w);
        if (lane == 63) sum(g, w);
        w = 0.0;
    });
}
template <bool BF16, bool ALL, typename Put, typename Sum>
__device__ __forceinline__ void sum_window(const void* s, int64_t cols, const Segments& segs, int g0, int g1, const Binning& bin,
                                           const Window& win, const Cut& cut, const Weigh& weigh, double min_p, Put put,
                                           Sum sum, double& z, double& better) {
    const float above = win.from > 0.0f ? score_at(bin, win.from) : INFINITY, least = score_at(bin, win.to);
    if (min_p > 0.0)
        sum_window<BF16, ALL, true>(s, cols, segs, g0, g1, above, least, cut, weigh, min_p, put, sum, z, better);
    else
        sum_window<BF16, ALL, false>(s, cols, segs, g0, g1, above, least, cut, weigh, min_p, put, sum, z, better);
}

// The cut of top_p among the window's columns, and their kept weights added to the segments.  each(f): f(key) for this
// thread's of them.  False if the exact sums show that the cut lies elsewhere.
template <typename Each>
__device__ __forceinline__ bool resolve_window(Each each, int64_t cols, double z, double better, const Binning& bin, const Window& win,
                                               const Row& r, const Segments& segs, Weigh weigh, Cut& cut, Shared& sh) {
    static_assert(kFar <= 1 << 13, "units of 2^-49");
    weigh.unit = 49;  // these columns' weights add up to at most kFar
    const int tid = threadIdx.x;
    const double target = r.top_p * z, scale = ldexp(1.0, -weigh.unit);
    // kThreads smaller steps within the window, of weights, and the columns of the one that reaches the target
    const float fine = (float)kThreads / (win.to - win.from);
    const auto step = [&](float v) { return min(kThreads - 1, max(0, (int)((bin.at(v) - win.from) * fine))); };
    uint64_t whole = 0;
    clear_fine(sh);
    each([&](uint64_t key) {
        const float v = key_score(key);
        const uint64_t w = weigh.fixed(v);
        whole += w;
        atomicAdd((unsigned long long*)&sh.wide[step(v)], (unsigned long long)w);
    });
    whole = block_sum_u64(whole, sh);
    if (!whole || !(better < target && better + (double)whole * scale >= target)) return false;
    find_fine((target - better) / scale, sh);
    const int b = (int)sh.bin;
    const double before = better + (double)sh.below * scale;
    uint32_t most = 0, least = 0;  // order bits, reversed ones
    __syncthreads();
    each([&](uint64_t key) {
        if (step(key_score(key)) != b) return;
        const uint32_t order = (uint32_t)order_of(key_score(key));
        most = max(most, order);
        least = max(least, ~order);
        const uint32_t k = atomicAdd(&sh.n, 1u);
        if (k < kList) sh.key[k] = key;
    });
    block_max2(most, least, sh);
    int m = (int)sh.n;
    uint64_t last = 0;  // of the keys below the target the smallest, complemented
    if (m > 64 && most == ~least) {
        // equal scores: the first `want` of them in column order, found in kThreads runs of columns
        const double each_w = (double)weigh.fixed(unord_f32(most)) * scale;
        double want = floor((target - before) / each_w);
        if (!(before + want * each_w < target)) want -= 1.0;
        if (before + (want + 1.0) * each_w < target) want += 1.0;
        const uint32_t run = (uint32_t)((cols + kThreads - 1) / kThreads);
        const int equals = m;
        clear_fine(sh);
        each([&](uint64_t key) {
            if (step(key_score(key)) == b) atomicAdd((unsigned long long*)&sh.wide[(uint32_t)key_index(key) / run], 1ull);
        });
        find_fine(fmin(want + 1.0, (double)equals), sh);
        const uint32_t piece = sh.bin;
        const int64_t rank = (int64_t)fmin(want, (double)(equals - 1)) - (int64_t)sh.below;
        __syncthreads();
        each([&](uint64_t key) {
            if (step(key_score(key)) != b || (uint32_t)key_index(key) / run != piece) return;
            const uint32_t k = atomicAdd(&sh.n, 1u);
            if (k < kList) sh.key[k] = key;
        });
        __syncthreads();
        m = (int)sh.n;
        if (m > kList) return false;
        for (int c = tid; c < m; c += kThreads) {
            int64_t n = 0;
            for (int j = 0; j < m; ++j) n += sh.key[j] > sh.key[c];
            if (n == rank) last = ~sh.key[c];
        }
    } else {
        if (m > kList) return false;
        for (int c = tid; c < m; c += kThreads) sh.wide[c] = weigh.fixed(key_score(sh.key[c]));
        __syncthreads();
        // each thread adds up what ranks before its columns: the last one below the target is the cut
        for (int c = tid; c < m; c += kThreads) {
            uint64_t sum = 0;
            for (int j = 0; j < m; ++j) sum += sh.key[j] > sh.key[c] ? sh.wide[j] : 0;
            if (before + (double)sum * scale < target) last = max(last, ~sh.key[c]);
        }
    }
    last = block_max_u64(last, sh);
    if (!last) return false;
    const uint64_t key = ~last;
    cut = Cut{key_score(key), key_index(key)};
    __syncthreads();
    for (int j = tid; j < segs.n; j += kThreads) sh.wide[j] = 0;
    __syncthreads();
    each([&](uint64_t k) {
        const float v = key_score(k);
        if (k >= key && weigh(v) >= r.min_p)
            atomicAdd((unsigned long long*)&sh.wide[(uint32_t)key_index(k) / (uint32_t)segs.len], (unsigned long long)weigh.fixed_kept(v));
    });
    __syncthreads();
    for (int j = tid; j < segs.n; j += kThreads) sh.seg[j + 1] += (double)sh.wide[j] * scale;
    return true;
}

__device__ __forceinline__ void kept_weights(const float (&v)[4], int i, const Cut& cut, const Weigh& weigh, double min_p, double (&w)[4]) {
    weigh.scaled<4>(v, 0, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = (cut.keeps(v[j], i + j) & (w[j] >= min_p)) ? w[j] : 0.0;
}

// weights of the kept columns of segments [g0, g1) -> sum(g, .)
template <bool BF16, bool ALL, typename Sum>
__device__ __forceinline__ void sum_segments(const void* s, int64_t cols, const Segments& segs, int g0, int g1, const Cut& cut,
                                             const Weigh& weigh, double min_p, Sum sum) {
    const bool masks = min_p > 0.0;
    double w = 0.0;
    for_segments<BF16>(s, cols, segs, g0, g1, [&](const float (&v)[4], int i) {
        if (!ALL && !(max_of(max_of(v[0], v[1]), max_of(v[2], v[3])) >= cut.s)) return;
        double x[4];
        if (ALL && !masks)
            weigh.scaled<4>(v, 0, x);
        else
            kept_weights(v, i, cut, weigh, min_p, x);
        w += (x[0] + x[1]) + (x[2] + x[3]);
    }, [&](int g) {
        w = wave_scan_f64(w);
        if ((threadIdx.x & 63) == 63) sum(g, w);
        w = 0.0;
    });
}

// The same without any restriction, in one reading: a segment's weights against the segment's own best score,
// sum(g, weights, best score).  A wave keeps 1024 columns in registers between finding their best and weighing them.
// Against a reading for the best score and one for the sums: 2048 x 91,599 f32 190 us (295), 64 x 1M 65 us (104), 64 x 40,981
// bf16 15 us (21).  A segment's sum is above 0 iff its best column's weight is, so no draw meets a segment without columns
template <bool BF16, typename Sum>
__device__ __forceinline__ void sum_own(const void* s, int64_t cols, const Segments& segs, int g0, int g1, const Weigh& like, Sum sum) {
    constexpr int U = 4, N = Vec<BF16>::N;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int g = g0 + wave; g < g1; g += kWaves) {
        const int64_t end = min(cols, (g + 1) * segs.len);
        double w = 0.0;
        float top = kNone;
        for (int64_t i0 = g * segs.len; i0 < end; i0 += U * 64 * N) {
            float v[U][4], best = kNone;
            const bool whole = i0 + U * 64 * N <= end;
            if (whole) {
                Vec<BF16> x[U];
#pragma unroll
                for (int k = 0; k < U; ++k) x[k].load(s, i0 + (k * 64 + lane) * N);
#pragma unroll
                for (int k = 0; k < U; ++k) x[k].values(v[k]);
            } else {
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    const int64_t i = i0 + (k * 64 + lane) * N;
                    Vec<BF16> x;
                    x.none();
                    if (i + N <= end) x.load(s, i);
                    x.values(v[k]);
                    if (i < end && i + N > end) load_tail<BF16>(v[k], s, i, end);
                }
            }
#pragma unroll
            for (int k = 0; k < U; ++k) best = max_of(best, max_of(max_of(v[k][0], v[k][1]), max_of(v[k][2], v[k][3])));
            const uint32_t order = (uint32_t)wave_max_u64(order_of(best));
            best = unord_f32((uint32_t)__builtin_amdgcn_readlane((int)order, 63));
            if (!(best > kNone)) continue;
            Weigh weigh = like;
            if (best > top) {
                weigh.m = (double)best;
                w = top > kNone ? w * weigh(top) : 0.0;
                top = best;
            }
            weigh.m = (double)top;
            if (top == INFINITY) continue;
            auto add = [&](const float (&s)[4]) {
                double x[4];
                weigh.scaled<4>(s, 0, x);
                w += (x[0] + x[1]) + (x[2] + x[3]);
            };
            if (whole) {
#pragma unroll
                for (int k = 0; k < U; ++k) add(v[k]);
            } else {
#pragma unroll
                for (int k = 0; k < U; ++k)
                    if (i0 + k * 64 * N < end) add(v[k]);
            }
        }
        w = wave_scan_f64(w);
        if (lane == 63) sum(g, w, top);
    }
}

// A row of at most kGroup x kList columns by one workgroup: the running weights of groups of columns in LDS, which every thread
// searches for a draw of its own: 256 x 14,687 f32 with min_p, 100 draws 12.8 us (a wave a draw, on segments, 35), 20 draws 12.6 (16);
// one draw of 1000 columns 7.3 (7.0), of 14,687 a wave's still: the groups take another reading
template <bool BF16>
__device__ __forceinline__ bool draw_groups(const SampleArgs& a, int64_t row, const Row& r, const void* s, const Cut& cut,
                                            const Weigh& weigh, Shared& sh) {
    constexpr int N = Vec<BF16>::N;
    if (!grouped(a.cols, a.n_draws)) return false;
    const int cols = (int)a.cols, size = (cols + N * kList - 1) / (N * kList) * N, n = (cols + size - 1) / size;
    const auto weights = [&](int i, double (&w)[N]) {
        float v[N];
        if (i + N <= cols) {
            Vec<BF16> x;
            x.load(s, i);
            x.values(v);
        } else {
            load_tail<BF16>(v, s, i, cols);
        }
        kept_weights(v, i, cut, weigh, r.min_p, w);
    };
    __syncthreads();
    for (int g = threadIdx.x; g < n; g += kThreads) {
        double sum = 0.0;
        for (int i = g * size; i < min(cols, (g + 1) * size); i += N) {
            double w[N];
            weights(i, w);
            sum += (w[0] + w[1]) + (w[2] + w[3]);
        }
        sh.w[g] = sum;
    }
    const int end = running_sums<kList / kThreads>(sh.w, n, sh);
    const double total = sh.w[n - 1];
    for (int64_t j = threadIdx.x; j < a.n_draws; j += kThreads) {
        const double target = draw_number(a, row, j) * total;
        int lo = 0, hi = end;  // the first group whose end passes the target
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (sh.w[mid] > target) hi = mid; else lo = mid + 1;
        }
        double run = lo ? sh.w[lo - 1] : 0.0, weight = 0.0;
        int pick = -1;  // its first column past the target, or without one its last of any weight
        bool past = false;
        for (int i = lo * size; i < min(cols, (lo + 1) * size) && !past; i += N) {
            double w[N];
            weights(i, w);
#pragma unroll
            for (int k = 0; k < N; ++k) {
                run += w[k];
                if (w[k] > 0.0 && !past) {
                    pick = i + k;
                    weight = w[k];
                    past = run > target;
                }
            }
        }
        a.out_idx[row * a.n_draws + j] = pick;
        if (a.out_prob) a.out_prob[row * a.n_draws + j] = (float)(weight / total);
    }
    return true;
}

// the draws part, part + parts, ... (in groups of kWaves) from the segment sums sh.seg[1, n]
template <bool BF16>
__device__ __forceinline__ void draw_columns(const SampleArgs& a, int64_t row, const Row& r, const void* s, const Segments& segs, const Cut& cut,
                             const Weigh& weigh, int part, int parts, Shared& sh) {
    constexpr int N = Vec<BF16>::N, kStep = 64 * N;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int last_seg = running_sums<kSegs / kThreads>(sh.seg + 1, segs.n, sh);  // the last segment with any weight
    if (tid == 0) sh.seg[0] = 0.0;
    __syncthreads();
    const double total = sh.seg[segs.n];
    for (int64_t j = wave + (int64_t)part * kWaves; j < a.n_draws; j += (int64_t)parts * kWaves) {
        const double target = draw_number(a, row, j) * total;
        int lo = 0, hi = last_seg;  // the first segment whose end passes the target
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (sh.seg[mid + 1] > target) hi = mid; else lo = mid + 1;
        }
        const int64_t end = min(a.cols, (lo + 1) * segs.len);
        double run = sh.seg[lo];
        int64_t pick = -1, fallback = -1;  // without a column past the target: the segment's last of any weight
        double wp = 0.0;
        // four steps of the wave on their way at once
        constexpr int kAhead = 4;
        for (int64_t i0 = lo * segs.len; i0 < end && pick < 0; i0 += kAhead * kStep) {
            float v[kAhead][4];
#pragma unroll
            for (int t = 0; t < kAhead; ++t) {
                const int64_t i = i0 + t * kStep + lane * N;
                if (i + N <= end) {
                    Vec<BF16> x;
                    x.load(s, i);
                    x.values(v[t]);
                } else {
                    load_tail<BF16>(v[t], s, i, end);
                }
            }
#pragma unroll
            for (int t = 0; t < kAhead; ++t) {
                if (pick >= 0) break;
                const int64_t i = i0 + t * kStep + lane * N;
                double w[N], own = 0.0;
                kept_weights(v[t], (int)i, cut, weigh, r.min_p, w);
#pragma unroll
                for (int k = 0; k < N; ++k) own += w[k];
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
                    const int64_t col = i0 + t * kStep + l * N + __shfl(pass ? at : tail, l, 64);
                    wp = shfl_f64(pass ? wa : wt, l);
                    if (pass) pick = col; else fallback = col;
                }
                run = shfl_f64(c, 63);
            }
        }
        if (pick < 0) pick = fallback;
        if (lane == 0) {
            a.out_idx[row * a.n_draws + j] = (int32_t)pick;
            if (a.out_prob) a.out_prob[row * a.n_draws + j] = (float)(wp / total);
        }
    }
}

__device__ __forceinline__ void all_draws(const SampleArgs& a, int64_t row, int32_t idx, float prob) {
    for (int64_t j = threadIdx.x; j < a.n_draws; j += kThreads) {
        a.out_idx[row * a.n_draws + j] = idx;
        if (a.out_prob) a.out_prob[row * a.n_draws + j] = prob;
    }
}
__device__ __forceinline__ bool best_only(const Row& r) { return !(r.T > 0.0) || r.top_k == 1 || r.top_p <= 0.0; }

template <bool BF16>
__device__ __forceinline__ const void* row_scores(const SampleArgs& a, int64_t row) {
    return BF16 ? (const void*)(static_cast<const uint16_t*>(a.S) + row * a.ld)
                : (const void*)(static_cast<const float*>(a.S) + row * a.ld);
}

__device__ __forceinline__ bool listed(const SampleArgs& a, const Row& r) { return r.top_k > 0 && r.top_k < a.cols; }
__device__ __forceinline__ bool unrestricted(const SampleArgs& a, const Row& r) {
    return !listed(a, r) && !(r.top_p < 1.0) && !(r.min_p > 0.0);
}

__device__ __forceinline__ float best_of(const Maxima& m, Shared& sh) {
    return unord_f32((uint32_t)block_max_u64(order_of(max_of(max_of(m.best[0], m.best[1]), max_of(m.best[2], m.best[3]))), sh));
}

// the draws of a row whose top_k columns are among sh.key[0, n)
template <bool BF16>
__device__ __forceinline__ void draw_list(const SampleArgs& a, int64_t row, const Row& r, const void* s, int n, Shared& sh) {
    uint64_t best = 0;
    for (int j = threadIdx.x; j < n; j += kThreads) best = max(best, sh.key[j]);
    best = block_max_u64(best, sh);
    if (!best)
        all_draws(a, row, -1, 0.0f);
    else if (key_score(best) == INFINITY)
        draw_infinite<BF16>(a, row, r, s, sh);
    else
        finish_list(a, row, r, n, Weigh(key_score(best), r.T), sh);
}

// the draws of a row without restrictions, from its segments' weights against their own best scores (sh.seg, sh.seg_top)
template <bool BF16>
__device__ __forceinline__ void draw_own(const SampleArgs& a, int64_t row, const Row& r, const void* s, const Segments& segs, int part,
                                         int parts, Shared& sh) {
    float top = kNone;
    __syncthreads();
    for (int j = threadIdx.x; j < segs.n; j += kThreads) top = max_of(top, sh.seg_top[j]);
    top = unord_f32((uint32_t)block_max_u64(order_of(top), sh));
    if (top == kNone) {
        if (part == 0) all_draws(a, row, -1, 0.0f);
    } else if (top == INFINITY) {
        if (part == 0) draw_infinite<BF16>(a, row, r, s, sh);
    } else {
        const Weigh weigh(top, r.T);
        for (int j = threadIdx.x; j < segs.n; j += kThreads) sh.seg[j + 1] *= weigh(sh.seg_top[j]);
        draw_columns<BF16>(a, row, r, s, segs, Cut{kNone, -1}, weigh, part, parts, sh);
    }
}

// A whole row by one workgroup.  K, P: there may be a top_k, a top_p (a kernel without the one's steps keeps its weights in
// registers)
template <bool BF16, bool K, bool P>
__device__ __forceinline__ void sample_row(const SampleArgs& a, int64_t row, const Row& r, Shared& sh) {
    const int tid = threadIdx.x;
    const void* s = row_scores<BF16>(a, row);
    const int cols = (int)a.cols;
    if (best_only(r)) {
        const uint64_t best = block_max_u64(scan_best<BF16>(s, 0, cols, tid, kThreads), sh);
        all_draws(a, row, best ? key_index(best) : -1, best ? 1.0f : 0.0f);
        return;
    }
    const bool by_k = K && listed(a, r), by_p = P && r.top_p < 1.0;
    if (!K && !P && !(r.min_p > 0.0) && !grouped(cols, a.n_draws)) {
        sum_own<BF16>(s, cols, a.segs, 0, a.segs.n, Weigh(0.0f, r.T), [&](int g, double w, float t) {
            sh.seg[g + 1] = w;
            sh.seg_top[g] = t;
        });
        draw_own<BF16>(a, row, r, s, a.segs, 0, 1, sh);
        return;
    }
    const auto to_list = [&](uint64_t key) { push(sh.key, &sh.n, key); };
    // the list of the columns that reach the bound of the first ones, or of all of a short row
    if (K && (by_k ? r.top_k <= kList / 2 : by_p && cols <= kList)) {
        Row first = r;
        if (!by_k) first.top_k = cols;
        float bound = kNone;
        if (cols > kList) {
            const Maxima m = scan_maxima<BF16>(s, 0, cols, list_stride(0, cols, r.top_k));
            bound = class_bound(m, r.top_k, sh);
        }
        // without a bound there are few scores
        __syncthreads();
        if (tid == 0) sh.n = 0;
        __syncthreads();
        gather<BF16>(s, 0, cols, [&](float v) { return (v >= bound) & (v > kNone); }, to_list);
        __syncthreads();
        if (sh.n <= kList) {
            draw_list<BF16>(a, row, first, s, (int)sh.n, sh);
            return;
        }
    }
    // for top_p alone an eighth of the row is enough to lay out the steps, and the reading that counts them finds the best
    // score; a best score above them (by more than a quarter of the range, or a T so low that there is no such room) costs
    // a reading more
    const bool sample = by_p && !by_k && cols >= 16 * kChunk;
    Maxima m = scan_maxima<BF16>(s, 0, cols, sample ? 8 : 1);
    float top = best_of(m, sh), low = of_reverse_order(block_max_u64(reverse_order_of(m.low), sh));
    Binning bin{top, 0.0f};
    bool counted = false;
    if (sample && top > kNone && top < INFINITY) {
        const Steps steps(top, low, r, cols);
        if (steps.margin > 0.1 * steps.range) {
            bin = steps.bins(top, steps.margin);
            count_steps<BF16>(s, 0, cols, bin, Cut{kNone, -1}, sh, &m.best[0]);
            top = unord_f32((uint32_t)block_max_u64(order_of(m.best[0]), sh));
            counted = top <= bin.top;
        }
    }
    if (sample && !counted) {
        m = scan_maxima<BF16>(s, 0, cols, 1);
        top = best_of(m, sh);
        low = of_reverse_order(block_max_u64(reverse_order_of(m.low), sh));
    }
    if (top == kNone) {
        all_draws(a, row, -1, 0.0f);
        return;
    }
    if (top == INFINITY) {
        draw_infinite<BF16>(a, row, r, s, sh);
        return;
    }
    const Weigh weigh(top, r.T);
    Cut cut{kNone, -1};
    if (by_k) {
        // the step of the top_k-th column
        bin = make_binning(top, fmax((double)top - (double)low, 0.0));
        clear_hist(sh);
        for_groups<BF16, 2>(s, 0, cols, tid, kThreads, [&](const float (&v)[4], int) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (v[j] > kNone) atomicAdd(&sh.count[bin(v[j])], 1u);
        });
        __syncthreads();
        find_bin(sh.count, (double)r.top_k, sh);
        const int b = (int)sh.bin;
        const uint64_t before = sh.below, in_bin = sh.count[b];
        if (in_bin > 0 && in_bin <= kList) {
            gather<BF16>(s, 0, cols, [&](float v) { return (v > kNone) & (bin(v) == b); }, to_list);
            sort_keys((int)in_bin, sh);
            const uint64_t key = sh.key[min((uint64_t)r.top_k - before, in_bin) - 1];
            cut = Cut{key_score(key), key_index(key)};
        } else {
            cut = descend<BF16, false>(s, cols, cut, (double)r.top_k, weigh, sh);
        }
    }
    const Segments& segs = a.segs;
    const auto to_seg = [&](int g, double w) { sh.seg[g + 1] = w; };
    bool summed = false;
    if (by_p) {
        if (!counted) {
            bin = Steps(top, low, r, cols).bins(top, 0.0);
            count_steps<BF16>(s, 0, cols, bin, cut, sh);
        }
        __syncthreads();
        const Window win = mass_window<BF16>(bin, r.T, r.top_p, weigh, kList, sh);
        if (win.usable(kList)) {
            double z, better;
            if (K && by_k)
                sum_window<BF16, false>(s, cols, segs, 0, segs.n, bin, win, cut, weigh, r.min_p, to_list, to_seg, z, better);
            else
                sum_window<BF16, true>(s, cols, segs, 0, segs.n, bin, win, cut, weigh, r.min_p, to_list, to_seg, z, better);
            z = block_sum_f64(z, sh);
            better = block_sum_f64(better, sh);
            const uint32_t n = sh.n;
            uint64_t mine[kList / kThreads];
#pragma unroll
            for (int j = 0; j < kList / kThreads; ++j) mine[j] = tid + j * kThreads < n ? sh.key[tid + j * kThreads] : 0;
            summed = n <= kList && resolve_window([&](auto f) {
#pragma unroll
                for (int j = 0; j < kList / kThreads; ++j)
                    if (mine[j]) f(mine[j]);
            }, cols, z, better, bin, win, r, segs, weigh, cut, sh);
        }
        if (!summed) cut = descend<BF16, true>(s, cols, cut, r.top_p, weigh, sh);
    }
    if (draw_groups<BF16>(a, row, r, s, cut, weigh, sh)) return;
    if (!summed) {
        __syncthreads();
        sum_segments<BF16, !K && !P>(s, cols, segs, 0, segs.n, cut, weigh, r.min_p, to_seg);
    }
    draw_columns<BF16>(a, row, r, s, segs, cut, weigh, 0, 1, sh);
}

// 2048 x 40,981 f32, top_p: 166 to 173 us (2 1/8 readings, of which the memory's share is 126), min_p 117; 1024 x 91,599 bf16, top_k 100: 74 us (one
// reading and a third, 44).  Held to 80 registers (three workgroups a CU) with 8 to 13 spilled
template <bool BF16, bool K, bool P>
__global__ __launch_bounds__(kThreads, 6) void sample_rows_kernel(SampleArgs a) {
    __shared__ Shared sh;
    sample_row<BF16, K, P>(a, blockIdx.x, row_settings(a, blockIdx.x), sh);
}

// ------------------------------------------------------------------------------------ few long rows
// The same steps with a row cut into `parts` runs of segments, a workgroup each, and a launch per reading; what the
// workgroups of a row tell each other goes through the workspace, in integers whose order does not matter or in slots
// of their own.  A row that needs one of the rare ways is left to its first workgroup in the last launch.
// 512 x 1M f32 with settings per row: top 194 us (a third of the rows is read whole: 0.7 GB), find 267 (62 %), again 11, sum 281
// (a quarter with top_p, a twelfth without restrictions), draw 35, clear 7.
struct Counted {
    uint32_t count[kBins];
    uint64_t place[kTopBins];
};
// the best and a low score of what the first reading looked at
struct Extent {
    float top, low;
};
struct RowState {   // cleared at the start
    uint32_t n;     // columns gathered
    uint32_t top;   // order bits of the best score, of rows of which an eighth was looked at first
    Extent extent;  // where there is a second launch
    Counted steps;
};
struct SplitArgs {
    RowState* state;
    Counted* again;  // [rows], cleared too: where the steps laid out from an eighth of the row missed its best score
    bool sample;     // top_p's steps are laid out from an eighth of the row
    bool clear;      // by the first reading
    bool find;       // there is a second launch
    uint64_t* keys;  // [rows, list]
    int list;
    double* seg;     // [rows, kSegs + 1]
    uint64_t* first;  // [rows, parts], what the part's first reading found: the class bound's order bits (top_k), the best column
                      // key (rows that draw it only), or the best score's order bits above the low score's reversed ones
    double* sums;     // [rows, parts, 2]: z, better (top_p)
    float* seg_top;  // [rows, kSegs]
    Segments segs;
    int parts;       // of them, a workgroup each
};

__global__ __launch_bounds__(256) void sample_clear(uint32_t* p, int64_t n) {
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += gridDim.x * (int64_t)256) p[i] = 0;
}

// the segments of this workgroup
struct Part {
    int g0, g1;
    int64_t lo, hi;
    __device__ __forceinline__ Part(const Segments& segs, int64_t cols, int part) {
        g0 = part * segs.part;
        g1 = min(segs.n, g0 + segs.part);
        lo = g0 * segs.len;
        hi = min(cols, g1 * segs.len);
    }
};
__device__ __forceinline__ void load_steps(const Counted& c, Shared& sh) {
    for (int j = threadIdx.x; j < kBins; j += kThreads) sh.count[j] = c.count[j];
    for (int j = threadIdx.x; j < kTopBins; j += kThreads) sh.place[j] = c.place[j];
}
__device__ __forceinline__ void add_steps(Counted& c, const Shared& sh) {
    for (int j = threadIdx.x; j < kBins; j += kThreads)
        if (sh.count[j]) atomicAdd(&c.count[j], sh.count[j]);
    for (int j = threadIdx.x; j < kTopBins; j += kThreads)
        if (sh.place[j]) atomicAdd((unsigned long long*)&c.place[j], (unsigned long long)sh.place[j]);
}
__device__ __forceinline__ bool finite(float top) { return top > kNone && top < INFINITY; }
__device__ __forceinline__ Extent first_extent(const SplitArgs& p, int64_t row, Shared& sh) {
    uint32_t top = 0, low = 0;
    for (int j = threadIdx.x; j < p.parts; j += kThreads) {
        const uint64_t x = p.first[row * p.parts + j];
        top = max(top, (uint32_t)(x >> 32));
        low = max(low, (uint32_t)x);
    }
    block_max2(top, low, sh);
    return Extent{unord_f32(top), of_reverse_order(low)};
}
__device__ __forceinline__ Extent known_extent(const SplitArgs& p, int64_t row, Shared& sh) {
    return p.find ? p.state[row].extent : first_extent(p, row, sh);
}
__device__ __forceinline__ bool eighth(const SplitArgs& p, const Row& r) { return p.sample && r.top_p < 1.0; }
__device__ __forceinline__ float best_score(const SplitArgs& p, int64_t row, const Row& r, const Extent& e) {
    return eighth(p, r) ? unord_f32(p.state[row].top) : e.top;
}
// steps with room above what an eighth of the row showed; false without them
__device__ __forceinline__ bool eighth_steps(const Extent& e, const Row& r, int64_t cols, Binning& bin) {
    if (!finite(e.top)) return false;
    const Steps steps(e.top, e.low, r, cols);
    bin = steps.bins(e.top, steps.margin);
    return steps.margin > 0.1 * steps.range;
}
// what the columns were counted by, and the counts
__device__ __forceinline__ const Counted& counted_steps(const SplitArgs& p, int64_t row, const Row& r, int64_t cols, const Extent& e,
                                                        Binning& bin) {
    const float top = best_score(p, row, r, e);
    if (p.sample && eighth_steps(e, r, cols, bin) && top <= bin.top) return p.state[row].steps;
    bin = Steps(top, e.low, r, cols).bins(top, 0.0);
    return p.sample ? p.again[row] : p.state[row].steps;
}

__device__ __forceinline__ void load_own(const SplitArgs& p, int64_t row, const Segments& segs, Shared& sh) {
    for (int j = threadIdx.x; j < segs.n; j += kThreads) {
        sh.seg[j + 1] = p.seg[row * (kSegs + 1) + j + 1];
        sh.seg_top[j] = p.seg_top[row * kSegs + j];
    }
}

__device__ __forceinline__ void draw_best(const SampleArgs& a, const SplitArgs& p, int64_t row, Shared& sh) {
    uint64_t best = 0;
    for (int j = threadIdx.x; j < p.parts; j += kThreads) best = max(best, p.first[row * p.parts + j]);
    best = block_max_u64(best, sh);
    all_draws(a, row, best ? key_index(best) : -1, best ? 1.0f : 0.0f);
}

// Without any restriction two launches do: the segments' own weights, and the draws
template <bool BF16>
__global__ __launch_bounds__(kThreads, 6) void sample_own_sum(SampleArgs a, SplitArgs p) {
    __shared__ Shared sh;
    const int64_t row = blockIdx.y;
    const Row r = row_settings(a, row);
    const Segments& segs = p.segs;
    const Part part(segs, a.cols, blockIdx.x);
    const void* s = row_scores<BF16>(a, row);
    if (best_only(r)) {
        const uint64_t best = block_max_u64(scan_best<BF16>(s, part.lo, part.hi, threadIdx.x, kThreads), sh);
        if (threadIdx.x == 0) p.first[row * p.parts + blockIdx.x] = best;
        return;
    }
    sum_own<BF16>(s, a.cols, segs, part.g0, part.g1, Weigh(0.0f, r.T), [&](int g, double w, float t) {
        p.seg[row * (kSegs + 1) + g + 1] = w;
        p.seg_top[row * kSegs + g] = t;
    });
}
template <bool BF16>
__global__ __launch_bounds__(kThreads, 4) void sample_own_draw(SampleArgs a, SplitArgs p) {
    __shared__ Shared sh;
    const int64_t row = blockIdx.y;
    const Row r = row_settings(a, row);
    const Segments& segs = p.segs;
    if (best_only(r)) {
        if (blockIdx.x) return;
        draw_best(a, p, row, sh);
        return;
    }
    load_own(p, row, segs, sh);
    draw_own<BF16>(a, row, r, row_scores<BF16>(a, row), segs, blockIdx.x, gridDim.x, sh);
}

// Every part gives the score of its j-th best class; the ceil(top_k / j)-th best of those is one that top_k columns reach.
// j is a little more than their average share.
__device__ __forceinline__ int64_t part_rank(int64_t top_k, int parts) { return 5 * top_k / (4 * parts) + 1; }

template <bool BF16>
__global__ __launch_bounds__(kThreads, 6) void sample_split_top(SampleArgs a, SplitArgs p) {
    __shared__ Shared sh;
    const int64_t row = blockIdx.y;
    const Row r = row_settings(a, row);
    const Part part(p.segs, a.cols, blockIdx.x);
    const void* s = row_scores<BF16>(a, row);
    const bool by_k = listed(a, r);
    uint64_t found = 0;
    if (best_only(r)) {
        found = block_max_u64(scan_best<BF16>(s, part.lo, part.hi, threadIdx.x, kThreads), sh);
    } else if (by_k ? r.top_k <= kList / 2 : !unrestricted(a, r)) {
        const int64_t stride = by_k ? list_stride(part.lo, part.hi, r.top_k) : eighth(p, r) ? 8 : 1;
        const Maxima m = scan_maxima<BF16>(s, part.lo, part.hi, stride);
        if (by_k) {
            found = order_of(class_bound(m, part_rank(r.top_k, p.parts), sh));
        } else {
            const uint64_t top = order_of(best_of(m, sh));
            found = top << 32 | block_max_u64(reverse_order_of(m.low), sh);
        }
    }
    if (threadIdx.x == 0) p.first[row * p.parts + blockIdx.x] = found;
    if (!p.clear) return;
    const auto clear = [&](void* at, int words) {
        for (int j = blockIdx.x * kThreads + threadIdx.x; j < words; j += p.parts * kThreads) static_cast<uint32_t*>(at)[j] = 0;
    };
    clear(p.state + row, sizeof(RowState) / 4);
    if (p.sample) clear(p.again + row, sizeof(Counted) / 4);
}

// a column to the workgroup's list in LDS, to the row's `list` ones in the workspace once that is full
__device__ __forceinline__ void push_far(uint64_t* keys, uint32_t* count, uint32_t list, Shared& sh, uint64_t key) {
    const uint32_t at = atomicAdd(&sh.n, 1u);
    if (at < kList) {
        sh.key[at] = key;
    } else {
        const uint32_t far = atomicAdd(count, 1u);
        if (far < list) keys[far] = key;
    }
}
// the workgroup's list behind the row's
__device__ __forceinline__ void append_list(uint64_t* keys, uint32_t* count, uint32_t list, Shared& sh) {
    __syncthreads();
    const uint32_t n = min(sh.n, (uint32_t)kList);
    if (threadIdx.x == 0) sh.bin = atomicAdd(count, n);
    __syncthreads();
    const uint32_t at = sh.bin;
    for (uint32_t j = threadIdx.x; j < n; j += kThreads)
        if (at + j < list) keys[at + j] = sh.key[j];
}

template <bool BF16>
__global__ __launch_bounds__(kThreads, 6) void sample_split_find(SampleArgs a, SplitArgs p) {
    __shared__ Shared sh;
    const int64_t row = blockIdx.y;
    const Row r = row_settings(a, row);
    const Part part(p.segs, a.cols, blockIdx.x);
    RowState* st = p.state + row;
    if (best_only(r)) return;
    const void* s = row_scores<BF16>(a, row);
    if (listed(a, r)) {
        if (r.top_k > kList / 2) return;
        for (int j = threadIdx.x; j < p.parts; j += kThreads)
            sh.key[j] = p.first[row * p.parts + j];
        sort_keys(p.parts, sh);
        const int64_t j = part_rank(r.top_k, p.parts);
        const float bound = unord_f32((uint32_t)sh.key[(r.top_k + j - 1) / j - 1]);  // without one there are few scores
        __syncthreads();
        if (threadIdx.x == 0) sh.n = 0;
        __syncthreads();
        gather<BF16>(s, part.lo, part.hi, [&](float v) { return (v >= bound) & (v > kNone); }, [&](uint64_t key) { push_far(p.keys + row * p.list, &st->n, kList, sh, key); });
        append_list(p.keys + row * p.list, &st->n, kList, sh);
        return;
    }
    if (unrestricted(a, r) || (blockIdx.x && !(r.top_p < 1.0))) return;
    const Extent e = first_extent(p, row, sh);
    if (blockIdx.x == 0 && threadIdx.x == 0) st->extent = e;
    if (eighth(p, r)) {
        Binning bin;
        float top;
        if (eighth_steps(e, r, a.cols, bin)) {
            count_steps<BF16>(s, part.lo, part.hi, bin, Cut{kNone, -1}, sh, &top);
            __syncthreads();
            add_steps(st->steps, sh);
        } else {
            const Maxima m = scan_maxima<BF16>(s, part.lo, part.hi, 1);
            top = max_of(max_of(m.best[0], m.best[1]), max_of(m.best[2], m.best[3]));
        }
        const uint32_t order = (uint32_t)block_max_u64(order_of(top), sh);
        if (threadIdx.x == 0) atomicMax(&st->top, order);
    } else if (r.top_p < 1.0 && finite(e.top)) {
        count_steps<BF16>(s, part.lo, part.hi, Steps(e.top, e.low, r, a.cols).bins(e.top, 0.0), Cut{kNone, -1}, sh);
        __syncthreads();
        add_steps(st->steps, sh);
    }
}

// The rows whose best score lies above the steps that a part of them laid out (by more than a quarter of the range), or
// whose T is so low that no room could be left
template <bool BF16>
__global__ __launch_bounds__(kThreads, 6) void sample_split_again(SampleArgs a, SplitArgs p) {
    __shared__ Shared sh;
    const int64_t row = blockIdx.y;
    const Row r = row_settings(a, row);
    const Part part(p.segs, a.cols, blockIdx.x);
    if (best_only(r) || listed(a, r) || !(r.top_p < 1.0) || !finite(unord_f32(p.state[row].top))) return;
    Binning bin;
    if (&counted_steps(p, row, r, a.cols, p.state[row].extent, bin) != p.again + row) return;
    count_steps<BF16>(row_scores<BF16>(a, row), part.lo, part.hi, bin, Cut{kNone, -1}, sh);
    __syncthreads();
    add_steps(p.again[row], sh);
}

template <bool BF16>
__global__ __launch_bounds__(kThreads, 6) void sample_split_sum(SampleArgs a, SplitArgs p) {
    __shared__ Shared sh;
    const int64_t row = blockIdx.y;
    const Row r = row_settings(a, row);
    const Segments& segs = p.segs;
    const Part part(segs, a.cols, blockIdx.x);
    RowState* st = p.state + row;
    if (best_only(r) || listed(a, r)) return;
    const void* s = row_scores<BF16>(a, row);
    double* seg = p.seg + row * (kSegs + 1);
    if (unrestricted(a, r)) {
        sum_own<BF16>(s, a.cols, segs, part.g0, part.g1, Weigh(0.0f, r.T), [&](int g, double w, float t) {
            seg[g + 1] = w;
            p.seg_top[row * kSegs + g] = t;
        });
        return;
    }
    const Extent extent = known_extent(p, row, sh);
    const float top = best_score(p, row, r, extent);
    if (!finite(top)) return;
    const Weigh weigh(top, r.T);
    if (!(r.top_p < 1.0)) {
        sum_segments<BF16, true>(s, a.cols, segs, part.g0, part.g1, Cut{kNone, -1}, weigh, r.min_p, [&](int g, double w) { seg[g + 1] = w; });
        return;
    }
    Binning bin;
    load_steps(counted_steps(p, row, r, a.cols, extent, bin), sh);
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    const Window win = mass_window<BF16>(bin, r.T, r.top_p, weigh, p.list, sh);
    if (!win.usable(p.list)) return;
    double z, better;
    sum_window<BF16, true>(s, a.cols, segs, part.g0, part.g1, bin, win, Cut{kNone, -1}, weigh, r.min_p,
                           [&](uint64_t key) { push_far(p.keys + row * p.list, &st->n, p.list, sh, key); },
                           [&](int g, double w) { seg[g + 1] = w; }, z, better);
    append_list(p.keys + row * p.list, &st->n, p.list, sh);
    z = block_sum_f64(z, sh);
    better = block_sum_f64(better, sh);
    if (threadIdx.x == 0) {
        double* o = p.sums + (row * p.parts + blockIdx.x) * 2;
        o[0] = z;
        o[1] = better;
    }
}

template <bool BF16>
__global__ __launch_bounds__(kThreads, 4) void sample_split_draw(SampleArgs a, SplitArgs p) {
    __shared__ Shared sh;
    const int64_t row = blockIdx.y;
    const int tid = threadIdx.x;
    const bool first = blockIdx.x == 0;
    const Row r = row_settings(a, row);
    const Segments& segs = p.segs;
    const RowState* st = p.state + row;
    const void* s = row_scores<BF16>(a, row);
    if (best_only(r)) {
        if (first) draw_best(a, p, row, sh);
        return;
    }
    if (unrestricted(a, r)) {
        load_own(p, row, segs, sh);
        draw_own<BF16>(a, row, r, s, segs, blockIdx.x, gridDim.x, sh);
        return;
    }
    const bool by_k = listed(a, r);
    const int list = by_k ? kList : p.list, n = (int)min(st->n, (uint32_t)list + 1);
    bool alone = n > list;
    const uint64_t* keys = p.keys + row * p.list;
    if (by_k && r.top_k <= kList / 2 && !alone) {
        if (!first) return;
        for (int j = tid; j < n; j += kThreads) sh.key[j] = keys[j];
        __syncthreads();
        draw_list<BF16>(a, row, r, s, n, sh);
        return;
    }
    alone |= by_k;
    Cut cut{kNone, -1};
    const double* seg = p.seg + row * (kSegs + 1);
    const bool by_p = r.top_p < 1.0;
    const Extent extent = by_k ? Extent{0.0f, 0.0f} : known_extent(p, row, sh);  // (a top_k row comes here with no list)
    const float top = best_score(p, row, r, extent);
    const Weigh weigh(top, r.T);
    if (!by_k && !finite(top)) {
        if (!first) return;
        if (top == INFINITY) draw_infinite<BF16>(a, row, r, s, sh); else all_draws(a, row, -1, 0.0f);
        return;
    }
    if (!alone && by_p) {
        Binning bin;
        load_steps(counted_steps(p, row, r, a.cols, extent, bin), sh);
        __syncthreads();
        const Window win = mass_window<BF16>(bin, r.T, r.top_p, weigh, p.list, sh);
        alone = !win.usable(p.list);
        if (!alone) {
            __syncthreads();
            for (int j = tid; j < segs.n; j += kThreads) sh.seg[j + 1] = seg[j + 1];
            double z = 0.0, better = 0.0;
            for (int j = 0; j < p.parts; ++j) {
                z += p.sums[(row * p.parts + j) * 2];
                better += p.sums[(row * p.parts + j) * 2 + 1];
            }
            __syncthreads();
            alone = !resolve_window([&](auto f) {
                for (int j = tid; j < n; j += kThreads) f(keys[j]);
            }, a.cols, z, better, bin, win, r, segs, weigh, cut, sh);
        }
    } else if (!alone) {
        for (int j = tid; j < segs.n; j += kThreads) sh.seg[j + 1] = seg[j + 1];
    }
    if (alone) {
        __syncthreads();
        if (first) sample_row<BF16, true, true>(a, row, r, sh);
        return;
    }
    draw_columns<BF16>(a, row, r, s, segs, cut, weigh, blockIdx.x, gridDim.x, sh);
}

// How many workgroups share a row: none where a workgroup per row fills the chip (three fit a CU; 1024 x 300,000 f32, top_p: 523
// us, by two of them 633), except that of rows past 2^19 columns more bf16 ones share a score than a workgroup can list
// (1024 x 1M bf16, top_p: 3.5 ms, by three of them 1.8; f32 2.0 and 2.1).  Else enough to fill it four times over (rows with
// other settings cost other amounts), of at least two steps for every wave
// (more than 16 kFill rows again none: their lists would take gigabytes)
constexpr int64_t kFill = 768, kSplitGroups = 4 * kFill;
Segments split_segments(int64_t rows, int64_t cols, int64_t n_draws) {
    int64_t parts = 1;
    if (rows > 0 && rows < (cols > 1 << 19 ? 16 * kFill : kFill) && cols > 32768)
        parts = std::min({std::max<int64_t>(2, kSplitGroups / rows), cols / (2 * kWaves * Segments::kStep), (int64_t)kSegs / kWaves});
    return Segments(cols, n_draws, (int)parts);
}

// parts of a row that are long enough for an eighth of them to show what the row is like
bool split_sample(const Segments& segs) { return segs.part * segs.len >= 16 * kChunk; }
int split_list(int64_t cols) { return cols > 131072 ? kFar : kList; }

// the workspace: states, second counts, keys, segment sums, first findings, sums, segments' best scores
struct SplitLayout {
    size_t again, keys, seg, first, sums, seg_top, bytes;
    SplitLayout(int64_t rows, int64_t cols, const Segments& segs) {
        const int parts = segs.parts();
        again = (size_t)rows * sizeof(RowState);
        keys = align_up(again + (split_sample(segs) ? (size_t)rows * sizeof(Counted) : 0));
        seg = keys + align_up((size_t)rows * split_list(cols) * 8);
        first = seg + align_up((size_t)rows * (kSegs + 1) * 8);
        sums = first + align_up((size_t)rows * parts * 8);
        seg_top = sums + align_up((size_t)rows * parts * 16);
        bytes = parts > 1 ? seg_top + align_up((size_t)rows * kSegs * 4) : 0;
    }
};

// the rows from `first` on
SampleArgs rows_from(SampleArgs a, bool bf16, int64_t first) {
    a.S = static_cast<const char*>(a.S) + first * a.ld * (bf16 ? 2 : 4);
    a.u = static_cast<const char*>(a.u) + first * a.n_draws * (a.u_f64 ? 8 : 4);
    for (const void** p : {&a.T_rows, &a.p_rows, &a.m_rows})
        if (*p) *p = static_cast<const char*>(*p) + first * (a.rows_f64 ? 8 : 4);
    if (a.k_rows) a.k_rows += first;
    a.out_idx += first * a.n_draws;
    if (a.out_prob) a.out_prob += first * a.n_draws;
    a.rows -= first;
    return a;
}

template <bool BF16>
int launch_sample(const SampleArgs& a, void* ws, const Segments& segs, hipStream_t stream) {
    const int parts = segs.parts();
    if (parts == 1) {
        const bool by_p = a.p_rows || a.top_p < 1.0;
        constexpr int64_t kMost = 1 << 22;  // rows of a launch: a grid has less than 2^32 threads
        for (int64_t first = 0; first < a.rows; first += kMost) {
            const SampleArgs b = rows_from(a, BF16, first);
            const unsigned grid = (unsigned)std::min(kMost, b.rows);
            if (a.k_rows || (a.top_k > 0 && a.top_k < a.cols) || (by_p && a.cols <= kList))
                sample_rows_kernel<BF16, true, true><<<grid, kThreads, 0, stream>>>(b);
            else if (by_p)
                sample_rows_kernel<BF16, false, true><<<grid, kThreads, 0, stream>>>(b);
            else
                sample_rows_kernel<BF16, false, false><<<grid, kThreads, 0, stream>>>(b);
            LGX_LAUNCH_CHECK();
        }
        return LGX_OK;
    }
    const SplitLayout l(a.rows, a.cols, segs);
    const bool by_p = a.p_rows || a.top_p < 1.0, sample = by_p && split_sample(segs);
    const bool find = by_p || a.k_rows || (a.top_k > 0 && a.top_k < a.cols);
    // a launch more costs a small batch 2 us (64 x 131,072, top_k 50: 57, 55 without), the clearing inside a reading of many rows 10
    // (512 x 1M with settings per row: 738 us, 727 with the launch)
    const int64_t words = a.rows * (int64_t)((sizeof(RowState) + (sample ? sizeof(Counted) : 0)) / 4);
    const bool clear = words <= 1 << 21;
    char* w = static_cast<char*>(ws);
    const SplitArgs p{reinterpret_cast<RowState*>(w), reinterpret_cast<Counted*>(w + l.again), sample, clear, find, reinterpret_cast<uint64_t*>(w + l.keys), split_list(a.cols), reinterpret_cast<double*>(w + l.seg),
                      reinterpret_cast<uint64_t*>(w + l.first), reinterpret_cast<double*>(w + l.sums), reinterpret_cast<float*>(w + l.seg_top), segs, parts};
    const dim3 grid((unsigned)parts, (unsigned)a.rows);
    const dim3 draws((unsigned)std::min<int64_t>(ceil_div(a.n_draws, (int64_t)kWaves), parts), (unsigned)a.rows);
    if (!find && !a.m_rows && !(a.min_p > 0.0)) {
        sample_own_sum<BF16><<<grid, kThreads, 0, stream>>>(a, p);
        LGX_LAUNCH_CHECK();
        sample_own_draw<BF16><<<draws, kThreads, 0, stream>>>(a, p);
        LGX_LAUNCH_CHECK();
        return LGX_OK;
    }
    if (!clear) {
        sample_clear<<<1024, 256, 0, stream>>>(reinterpret_cast<uint32_t*>(w), words);
        LGX_LAUNCH_CHECK();
    }
    sample_split_top<BF16><<<grid, kThreads, 0, stream>>>(a, p);
    LGX_LAUNCH_CHECK();
    if (find) {
        sample_split_find<BF16><<<grid, kThreads, 0, stream>>>(a, p);
        LGX_LAUNCH_CHECK();
    }
    if (sample) {
        sample_split_again<BF16><<<grid, kThreads, 0, stream>>>(a, p);
        LGX_LAUNCH_CHECK();
    }
    sample_split_sum<BF16><<<grid, kThreads, 0, stream>>>(a, p);
    LGX_LAUNCH_CHECK();
    sample_split_draw<BF16><<<draws, kThreads, 0, stream>>>(a, p);
    LGX_LAUNCH_CHECK();
    return LGX_OK;
}

}  // namespace
}  // namespace lgx

using namespace lgx;

extern "C" int lgx_sample_rows_workspace(int64_t rows, int64_t cols, int64_t n_draws, size_t* ws_bytes) {
    LGX_REQUIRE(ws_bytes && rows >= 0 && cols >= 1 && n_draws >= 0, LGX_ERR_INVALID_ARG,
                "lgx_sample_rows_workspace: bad arguments");
    *ws_bytes = SplitLayout(rows, cols, split_segments(rows, cols, n_draws)).bytes;
    return LGX_OK;
}

namespace lgx {
namespace {

int sample_entry(const void* S, int dtype, int64_t rows, int64_t cols, int64_t ld, const void* u, int u_dtype, int64_t n_draws,
                 double temperature, const void* temperature_rows, int64_t top_k, const int32_t* top_k_rows, double top_p,
                 const void* top_p_rows, double min_p, const void* min_p_rows, bool rows_f64, int32_t* out_idx, float* out_prob,
                 void* ws, size_t ws_bytes, lgx_stream_t stream_) {
    hipStream_t stream = as_hip(stream_);
    LGX_REQUIRE(dtype == LGX_DTYPE_F32 || dtype == LGX_DTYPE_BF16, LGX_ERR_INVALID_ARG, "lgx_sample_rows: dtype");
    LGX_REQUIRE(u_dtype == LGX_DTYPE_F32 || u_dtype == LGX_DTYPE_F64, LGX_ERR_INVALID_ARG, "lgx_sample_rows: dtype of u");
    LGX_REQUIRE(rows >= 0 && n_draws >= 0, LGX_ERR_INVALID_ARG, "lgx_sample_rows: negative size");
    LGX_REQUIRE(cols >= 1 && cols < INT32_MAX && ld >= cols, LGX_ERR_INVALID_ARG,
                "lgx_sample_rows: cols=%lld outside [1, 2^31) or ld=%lld < cols", (long long)cols, (long long)ld);
    if (rows == 0 || n_draws == 0) return LGX_OK;
    LGX_REQUIRE(rows < (1LL << 31), LGX_ERR_UNSUPPORTED, "lgx_sample_rows: %lld rows is too many", (long long)rows);
    LGX_REQUIRE(S && u && out_idx, LGX_ERR_INVALID_ARG, "lgx_sample_rows: null pointer");
    const Segments segs = split_segments(rows, cols, n_draws);
    const size_t need = SplitLayout(rows, cols, segs).bytes;
    LGX_REQUIRE(need == 0 || (ws && ws_bytes >= need && reinterpret_cast<uintptr_t>(ws) % 16 == 0), LGX_ERR_WORKSPACE,
                "lgx_sample_rows: workspace %zu < %zu", ws_bytes, need);
    const SampleArgs a{S, rows, cols, ld, u, u_dtype == LGX_DTYPE_F64, rows_f64, n_draws, temperature, top_p, min_p, top_k,
                       temperature_rows, top_p_rows, min_p_rows, top_k_rows, out_idx, out_prob,
                       Segments(cols, grouped(cols, n_draws) ? 1 : n_draws)};
    return dtype == LGX_DTYPE_BF16 ? launch_sample<true>(a, ws, segs, stream) : launch_sample<false>(a, ws, segs, stream);
}

}  // namespace
}  // namespace lgx

extern "C" int lgx_sample_rows(const void* S, int dtype, int64_t rows, int64_t cols, int64_t ld, const void* u, int u_dtype,
                               int64_t n_draws, double temperature, const float* temperature_rows, int64_t top_k,
                               const int32_t* top_k_rows, double top_p, const float* top_p_rows, double min_p,
                               const float* min_p_rows, int32_t* out_idx, float* out_prob, void* ws, size_t ws_bytes,
                               lgx_stream_t stream) {
    return sample_entry(S, dtype, rows, cols, ld, u, u_dtype, n_draws, temperature, temperature_rows, top_k, top_k_rows, top_p,
                        top_p_rows, min_p, min_p_rows, false, out_idx, out_prob, ws, ws_bytes, stream);
}

extern "C" int lgx_sample_rows_f64(const void* S, int dtype, int64_t rows, int64_t cols, int64_t ld, const void* u, int u_dtype,
                                   int64_t n_draws, double temperature, const double* temperature_rows, int64_t top_k,
                                   const int32_t* top_k_rows, double top_p, const double* top_p_rows, double min_p,
                                   const double* min_p_rows, int32_t* out_idx, float* out_prob, void* ws, size_t ws_bytes,
                                   lgx_stream_t stream) {
    return sample_entry(S, dtype, rows, cols, ld, u, u_dtype, n_draws, temperature, temperature_rows, top_k, top_k_rows, top_p,
                        top_p_rows, min_p, min_p_rows, true, out_idx, out_prob, ws, ws_bytes, stream);
}
