// Draws from score rows: temperature, top-k, top-p and min-p, from given random numbers.
//
// One workgroup per row.  The kept columns are a prefix of the row's ranking (score descending, ties to the lower
// column), so they are described by one 64-bit key (wave_topk.h's make_key): column i is kept iff its key is at
// least the cut.  top_k and top_p find their cut by a descent over the 32 score bits, a digit at a time,
// through a histogram of counts (top_k) or of weights (top_p); ties at the cut are counted off in column order.
//
// Which column a given number draws depends on every weight before it, and with a million columns the borders
// between columns lie 1e-6 of the total apart, so 24 bits are not enough: weights are computed in f64 and
// summed in f64 in a fixed order, and the histogram holds them as integers of 2^-62 of the row's total (so that
// the order of its atomic additions does not matter).
#include "wave_topk.h"

#include <algorithm>

namespace lgx {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;
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

template <bool BF16>
__device__ __forceinline__ float load_score(const void* s, int64_t i) {
    return BF16 ? bf16_to_f32(static_cast<const uint16_t*>(s)[i]) : static_cast<const float*>(s)[i];
}

// the order key of a score; 0 for the excluded ones (NaN, -inf).  -0 ranks with +0
__device__ __forceinline__ uint32_t score_key(float s) {
    return s > -INFINITY ? ord_f32(s + 0.0f) : 0u;
}

// 2^y for y <= 0: y = n + f, |f| <= 1/2, the Taylor polynomial of e^(f ln 2) of degree 13
// (remainder below 0.35^14 / 14! < 5e-18)
__device__ __forceinline__ double exp2_f64(double y) {
    y = fmax(y, -1100.0);
    const double n = __builtin_rint(y);
    const double x = (y - n) * 0.69314718055994530942;
    double r = 1.0 / 6227020800.0;
    r = fma(r, x, 1.0 / 479001600.0);
    r = fma(r, x, 1.0 / 39916800.0);
    r = fma(r, x, 1.0 / 3628800.0);
    r = fma(r, x, 1.0 / 362880.0);
    r = fma(r, x, 1.0 / 40320.0);
    r = fma(r, x, 1.0 / 5040.0);
    r = fma(r, x, 1.0 / 720.0);
    r = fma(r, x, 1.0 / 120.0);
    r = fma(r, x, 1.0 / 24.0);
    r = fma(r, x, 1.0 / 6.0);
    r = fma(r, x, 0.5);
    r = fma(r, x, 1.0);
    r = fma(r, x, 1.0);
    return ldexp(r, (int)n);
}

struct Weigh {
    double m;      // the row's largest score
    double c;      // log2(e) / T
    uint32_t top;  // its key
    __device__ __forceinline__ double operator()(float s, uint32_t key) const {
        return key == top ? 1.0 : key == 0u ? 0.0 : exp2_f64(((double)s - m) * c);
    }
};

// a weight in units of 2^-62 of the row's total; a weight above 0 counts at least 1
__device__ __forceinline__ uint64_t to_fixed(double w, double unit) {
    if (!(w > 0.0)) return 0ull;
    const double x = w * unit;  // <= 2^62
    const double hi = floor(x * (1.0 / 4294967296.0));
    const double lo = fma(hi, -4294967296.0, x);
    const uint64_t v = ((uint64_t)(uint32_t)hi << 32) + (uint64_t)(uint32_t)(lo + 0.5);
    return v ? v : 1ull;
}

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
    double seg[kSegs + 1];
    uint64_t part[kWaves];
    double dpart[kWaves];
    uint64_t u64;
    uint64_t below;
    uint32_t bin;
};

// sum over the workgroup, the same value in every thread
__device__ uint64_t block_sum_u64(uint64_t v, Shared& sh) {
    v = wave_sum_u64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t s = 0;
    for (int i = 0; i < kWaves; ++i) s += sh.part[i];
    return s;
}
__device__ double block_sum_f64(double v, Shared& sh) {
    v = wave_sum_f64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.dpart[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0;
    for (int i = 0; i < kWaves; ++i) s += sh.dpart[i];
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

// The bin (from the top) in which the running sum of hist reaches `target`: sum above it < target <= sum
// with it; the last bin that holds anything if the whole falls short.  -> sh.bin, sh.below = the sum above it
__device__ void find_bin(double target, Shared& sh) {
    __syncthreads();
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        constexpr int per = kBins / 64;
        uint64_t own = 0;  // lane 0 holds the highest bins
        for (int j = 0; j < per; ++j) own += sh.hist[kBins - 1 - (lane * per + j)];
        const uint64_t incl = wave_scan_u64(own, lane);
        const uint64_t hit = __ballot(own > 0 && (double)incl >= target);
        const uint64_t any = __ballot(own > 0);
        const int pick = hit ? __builtin_ctzll(hit) : any ? 63 - __builtin_clzll(any) : 0;
        if (lane == pick) {
            uint64_t run = incl - own;
            int last = kBins - 1 - lane * per;
            uint64_t at = run;
            for (int j = 0; j < per; ++j) {
                const int b = kBins - 1 - (lane * per + j);
                const uint64_t h = sh.hist[b];
                if (!h) continue;
                last = b;
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

template <bool BF16>
__global__ __launch_bounds__(kThreads) void sample_rows_kernel(SampleArgs a) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const void* s = BF16 ? (const void*)(static_cast<const uint16_t*>(a.S) + row * a.ld)
                         : (const void*)(static_cast<const float*>(a.S) + row * a.ld);
    const int cols = (int)a.cols;
    const double T = a.T_rows ? (double)a.T_rows[row] : a.T;
    const double top_p = a.p_rows ? (double)a.p_rows[row] : a.top_p;
    const double min_given = a.m_rows ? (double)a.m_rows[row] : a.min_p;
    const double min_p = min_given > 0.0 ? fmin(min_given, 1.0) : 0.0;
    const int64_t top_k = a.k_rows ? (int64_t)a.k_rows[row] : a.top_k;
    int32_t* out_idx = a.out_idx + row * a.n_draws;
    float* out_prob = a.out_prob ? a.out_prob + row * a.n_draws : nullptr;

    // the best column and the number of columns that can be drawn
    uint64_t best = 0, live = 0;
    for (int64_t i = tid; i < cols; i += kThreads) {
        const uint32_t k = score_key(load_score<BF16>(s, i));
        if (k) {
            ++live;
            best = max(best, (uint64_t)k << 32 | (0xffffffffu - (uint32_t)i));
        }
    }
    best = block_max_u64(best, sh);
    live = block_sum_u64(live, sh);
    if (live == 0 || !(T > 0.0) || top_k == 1) {
        for (int64_t j = tid; j < a.n_draws; j += kThreads) {
            out_idx[j] = live ? key_index(best) : -1;
            if (out_prob) out_prob[j] = live ? 1.0f : 0.0f;
        }
        return;
    }
    const uint32_t top = (uint32_t)(best >> 32);
    const Weigh weigh{(double)unord_f32(top), 1.4426950408889634074 / T, top};

    uint64_t cut = 1ull << 32;  // every column with a score
    const bool by_k = top_k > 0 && (uint64_t)top_k < live, by_p = top_p < 1.0;
    double unit = 0.0;
    if (by_p) {
        double z = 0.0;
        for (int64_t i = tid; i < cols; i += kThreads) {
            const float v = load_score<BF16>(s, i);
            z += weigh(v, score_key(v));
        }
        unit = 4611686018427387904.0 / block_sum_f64(z, sh);
    }
    for (int step = 0; step < 2; ++step) {
        const bool mass = step == 1;
        if (mass ? !by_p : !by_k) continue;
        double target = (double)top_k;
        if (mass) {
            uint64_t sum = 0;
            for (int64_t i = tid; i < cols; i += kThreads) {
                const float v = load_score<BF16>(s, i);
                const uint32_t k = score_key(v);
                if (((uint64_t)k << 32 | (0xffffffffu - (uint32_t)i)) >= cut) sum += to_fixed(weigh(v, k), unit);
            }
            target = top_p * (double)block_sum_u64(sum, sh);
        }
        uint64_t above = 0;     // counted above the bins of this digit
        uint32_t prefix = 0;    // the score bits found so far
#pragma unroll 1
        for (int digit = 0; digit < 3; ++digit) {
            const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
            const uint32_t mask = digit == 2 ? 1023u : 2047u;
            const int done = digit == 0 ? 32 : digit == 1 ? 21 : 10;  // bits still open before this digit
            __syncthreads();
            for (int j = tid; j < kBins; j += kThreads) sh.hist[j] = 0;
            __syncthreads();
            for (int64_t i = tid; i < cols; i += kThreads) {
                const float v = load_score<BF16>(s, i);
                const uint32_t k = score_key(v);
                if (!k || ((uint64_t)k << 32 | (0xffffffffu - (uint32_t)i)) < cut) continue;
                if (done < 32 && (k >> done) != (prefix >> done)) continue;
                atomicAdd((unsigned long long*)&sh.hist[(k >> shift) & mask],
                          (unsigned long long)(mass ? to_fixed(weigh(v, k), unit) : 1ull));
            }
            find_bin(target - (double)above, sh);
            prefix |= sh.bin << shift;
            above += sh.below;
        }
        // the columns of score `prefix`: as many of the first as the target asks for
        __syncthreads();
        const uint64_t each = mass ? to_fixed(weigh(unord_f32(prefix), prefix), unit) : 1ull;
        const double want_f = ceil((target - (double)above) / (double)each);
        int64_t want = want_f < 1.0 ? 1 : (int64_t)fmin(want_f, (double)cols);
        int64_t found = -1;  // the column of the last one taken
        for (int64_t i0 = 0; i0 < cols; i0 += kThreads) {
            const int64_t i = i0 + tid;
            const uint32_t k = i < cols ? score_key(load_score<BF16>(s, i)) : 0u;
            const bool eq = k == prefix && ((uint64_t)k << 32 | (0xffffffffu - (uint32_t)i)) >= cut;
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
            if (eq && before < want) found = i;  // the largest wins below
            want -= all;
            if (want <= 0) break;
        }
        const uint64_t last = block_max_u64((uint64_t)(found + 1), sh);
        cut = max(cut, (uint64_t)prefix << 32 | (0xffffffffu - (uint32_t)(last - 1)));
    }

    // weights of the kept columns, summed per segment
    const int64_t seg_len = ((int64_t)cols + kSegs * 64 - 1) / (kSegs * 64) * 64;
    const int n_segs = (int)((cols + seg_len - 1) / seg_len);
    auto kept = [&](int64_t i) -> double {
        const float v = load_score<BF16>(s, i);
        const uint32_t k = score_key(v);
        if (((uint64_t)k << 32 | (0xffffffffu - (uint32_t)i)) < cut) return 0.0;
        const double w = weigh(v, k);
        return w >= min_p ? w : 0.0;
    };
    __syncthreads();
    for (int g = wave; g < n_segs; g += kWaves) {
        double w = 0.0;
        const int64_t end = min((int64_t)cols, (g + 1) * seg_len);
        for (int64_t i = g * seg_len + lane; i < end; i += 64) w += kept(i);
        w = wave_sum_f64(w);
        if (lane == 0) sh.seg[g + 1] = w;
    }
    __syncthreads();
    if (tid == 0) {
        double run = 0.0;
        sh.seg[0] = 0.0;
        for (int g = 0; g < n_segs; ++g) sh.seg[g + 1] = run += sh.seg[g + 1];
    }
    __syncthreads();
    const double total = sh.seg[n_segs];
    for (int64_t j = wave; j < a.n_draws; j += kWaves) {
        double u = a.u_f64 ? static_cast<const double*>(a.u)[row * a.n_draws + j]
                           : (double)static_cast<const float*>(a.u)[row * a.n_draws + j];
        u = fmin(fmax(u, 0.0), 1.0);
        const double target = u * total;
        int lo = 0, hi = n_segs - 1;  // the first segment whose end passes the target, the last with any weight
        while (hi > 0 && !(sh.seg[hi + 1] > sh.seg[hi])) --hi;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (sh.seg[mid + 1] > target) hi = mid; else lo = mid + 1;
        }
        const int64_t end = min((int64_t)cols, (lo + 1) * seg_len);
        double run = sh.seg[lo];
        int64_t pick = -1;
        double wp = 0.0;
        for (int64_t i0 = lo * seg_len; i0 < end; i0 += 64) {
            const int64_t i = i0 + lane;
            const double w = i < end ? kept(i) : 0.0;
            const double c = run + wave_scan_f64(w, lane);
            const uint64_t pass = __ballot(w > 0.0 && c > target), any = __ballot(w > 0.0);
            if (any) {  // without a column past the target: the last one of the segment
                const int l = pass ? __builtin_ctzll(pass) : 63 - __builtin_clzll(any);
                pick = i0 + l;
                wp = shfl_f64(w, l);
                if (pass) break;
            }
            run = shfl_f64(c, 63);
        }
        if (lane == 0) {
            out_idx[j] = (int32_t)pick;
            if (out_prob) out_prob[j] = (float)(wp / total);
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
