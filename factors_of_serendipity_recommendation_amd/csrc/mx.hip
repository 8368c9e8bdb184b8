// Microscaled 4-bit floating point tables: quantisation, its inverse, and full-catalog scoring over them.
//
// A row of d elements is cut into blocks of 32.  A block with largest magnitude a is stored as one byte
// b = max(E(a) - 2, 0), E the f32 exponent field, standing for the scale 2^(b - 127), and 32 e2m1 codes of
// x * 2^(127 - b): 4.25 bits an element, 1/7.5 of f32.  lgx_score_mx multiplies such rows on the block-scaled
// matrix instructions, which take the codes and scale bytes as they are stored.
#include "lgx_common.h"

#include <algorithm>
#include <type_traits>

namespace lgx {
namespace {

constexpr int kBlock = 32;       // elements under one scale
constexpr int64_t kMaxD = 65536;

using u32x4 = uint32_t __attribute__((ext_vector_type(4)));
using f32x4 = float __attribute__((ext_vector_type(4)));
using f32x2 = float __attribute__((ext_vector_type(2)));
using f32x16 = float __attribute__((ext_vector_type(16)));
using i32x8 = int __attribute__((ext_vector_type(8)));
// at any multiple of an element
using f32x4u = float __attribute__((ext_vector_type(4), aligned(4)));
using u32x2u = uint32_t __attribute__((ext_vector_type(2), aligned(2)));
using u32x4u = uint32_t __attribute__((ext_vector_type(4), aligned(2)));

// the codes of 8 scaled elements, element 0 in the low nibble of byte 0 (v_cvt_scalef32_pk_fp4_f32 rounds
// to nearest even and saturates at 6; the scale is applied by the caller, so its own is 1)
__device__ __forceinline__ uint32_t pack8(const float (&y)[8]) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[0], y[1], 1.0f, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[2], y[3], 1.0f, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[4], y[5], 1.0f, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[6], y[7], 1.0f, 3);
    return r;
}

// 8 elements from 16-byte boundaries (VEC) or anywhere
template <bool VEC>
__device__ __forceinline__ void load8_f32(const float* p, float (&x)[8]) {
    using V = std::conditional_t<VEC, f32x4, f32x4u>;
    const f32x4 a = *reinterpret_cast<const V*>(p), b = *reinterpret_cast<const V*>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = a[j], x[4 + j] = b[j];
}
template <bool VEC>
__device__ __forceinline__ void load8_bf16(const uint16_t* p, float (&x)[8]) {
    using V = std::conditional_t<VEC, u32x4, u32x4u>;
    const u32x4 a = *reinterpret_cast<const V*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[2 * j] = __uint_as_float(a[j] << 16);
        x[2 * j + 1] = __uint_as_float(a[j] & 0xffff0000u);
    }
}

// two values to bf16, round to nearest even (one instruction)
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    using B2 = __bf16 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), B2));
}

// the scale byte of a block whose largest magnitude has the bits a
__device__ __forceinline__ uint32_t scale_byte(uint32_t a) {
    const uint32_t e = a >> 23;
    return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}

// 4 lanes per block, 8 elements a lane.  VEC: rows are 16-byte aligned and d % 8 == 0.  rows_of (optional):
// the source row of every output row, a row outside [0, n_src) gives NaN blocks.  Bound by memory: 1M x 256 f32, 1.16 GB, in
// 234 us (5.0 TB/s, a copy's rate); 70,839 x 64 in 4.5 us.  Rows at odd addresses are loaded as wide, at any multiple of an
// element (100,000 x 601 f32 43 us, element by element 101).
template <bool BF16, bool VEC>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const void* __restrict__ X, const int64_t* __restrict__ rows_of,
                                                          int64_t n_src, int64_t units, int64_t nb, int64_t d, int64_t ld,
                                                          uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int64_t unit = blockIdx.x * (int64_t)64 + (threadIdx.x >> 2);
    const int sub = threadIdx.x & 3;
    if (unit >= units) return;
    const int64_t row = units <= UINT32_MAX ? (int64_t)((uint32_t)unit / (uint32_t)nb) : unit / nb;
    const int64_t c0 = (unit - row * nb) * kBlock + sub * 8;
    int64_t src = row;
    bool bad = false;
    if (rows_of) {
        src = rows_of[row];
        bad = src < 0 || src >= n_src;
    }
    float x[8] = {};
    if (!bad) {
        if (c0 + 8 <= d) {
            if (BF16)
                load8_bf16<VEC>(static_cast<const uint16_t*>(X) + src * ld + c0, x);
            else
                load8_f32<VEC>(static_cast<const float*>(X) + src * ld + c0, x);
        } else if (!VEC) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c0 + j < d)
                    x[j] = BF16 ? bf16_to_f32(static_cast<const uint16_t*>(X)[src * ld + c0 + j])
                                : static_cast<const float*>(X)[src * ld + c0 + j];
        }
    }
    uint32_t a = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) a = max(a, __float_as_uint(x[j]) & 0x7fffffffu);
    a = max(a, (uint32_t)__shfl_xor((int)a, 1));
    a = max(a, (uint32_t)__shfl_xor((int)a, 2));
    const uint32_t b = bad ? 255u : scale_byte(a);
    bad |= b == 255u;
    const float inv = __uint_as_float((254u - b) << 23);  // 2^(127 - b), b <= 252
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = x[j] * inv;
    reinterpret_cast<uint32_t*>(codes)[unit * 4 + sub] = bad ? 0u : pack8(y);
    if (sub == 0) scales[unit] = (uint8_t)b;
}

__device__ __forceinline__ float scale_value(uint32_t b) {  // 2^(b - 127); b = 0 is the subnormal 2^-127
    return b == 255u ? __builtin_nanf("") : __uint_as_float(b ? b << 23 : 0x00400000u);
}

// 4 lanes per block, 8 elements a lane (the layout of the quantiser).  1M x 256 to f32: 237 us (in a loop of calls 214, the quantiser 201); 100,000 x 601 50 us
// (element by element 146)
template <bool BF16, bool VEC>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales, int64_t units, int64_t nb,
                                                            int64_t d, void* __restrict__ out) {
    const int64_t unit = blockIdx.x * (int64_t)64 + (threadIdx.x >> 2);
    const int sub = threadIdx.x & 3;
    if (unit >= units) return;
    const int64_t row = units <= UINT32_MAX ? (int64_t)((uint32_t)unit / (uint32_t)nb) : unit / nb;
    const int64_t c0 = (unit - row * nb) * kBlock + sub * 8;
    if (c0 >= d) return;
    const uint32_t c = reinterpret_cast<const uint32_t*>(codes)[unit * 4 + sub];
    const float s = scale_value(scales[unit]);
    f32x2 p[4];
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[j / 2][j % 2] * s;
    if (BF16) {
        uint16_t* o = static_cast<uint16_t*>(out) + row * d + c0;
        if (VEC || c0 + 8 <= d) {
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
            *reinterpret_cast<std::conditional_t<VEC, u32x4, u32x4u>*>(o) = w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c0 + j < d) o[j] = f32_to_bf16(v[j]);
        }
    } else {
        float* o = static_cast<float*>(out) + row * d + c0;
        if (VEC || c0 + 8 <= d) {
            using V = std::conditional_t<VEC, f32x4, f32x4u>;
            *reinterpret_cast<V*>(o) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<V*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c0 + j < d) o[j] = v[j];
        }
    }
}

// ------------------------------------------------------------------------------------ product
// v_mfma_scale_f32_32x32x64 on e2m1 operands: lane l gives row l % 32 of A (users) and column l % 32 of B
// (items), 32 consecutive codes of that row (16 bytes: one block, so one scale byte a lane), the lane's half
// l / 32 picking the first or second 32 of the 64 products; result element i of lane l is user
// 8 (i / 4) + 4 (l / 32) + i % 4, item l % 32.  Any assignment of a row's blocks to (step, half) gives the
// same sum as long as both operands use it.
struct MxArgs {
    const uint8_t* q;
    const uint8_t* qs;
    const int64_t* user_rows;
    int64_t n_q;
    const uint8_t* it;
    const uint8_t* its;
    int64_t B, n_items, nb;
    void* out;
    int64_t d, q_ld;  // of f32 / bf16 queries
    bool q_vec;       // their rows start at multiples of 16 bytes and d % 8 == 0
};

__device__ __forceinline__ i32x8 frag(u32x4 v) {
    return i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
}

template <int KK>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c, uint32_t sa, uint32_t sb) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(frag(a), frag(b), c, 4, 4, KK, (int)sa, KK, (int)sb);
}

// e^-x by one instruction, |x| 2^-24 off for the rounding of x log2(e): below 2^-17 where the result is not 0, enough for
// bf16 results.  f32 ones take the product's rest in: within 2^-22 with the reciprocal's 1 ulp.  A call of 2048 x 40,981 with expf: bf16
// 59 us (34), f32 79 (74); an IEEE division made the stores wait
template <bool BF16>
__device__ __forceinline__ float sigmoid(float x) {
    constexpr float c = -1.44269502f, c_rest = (float)(-1.4426950408889634074 - (double)c);  // -log2(e)
    const float t = x * c;
    float e = __builtin_amdgcn_exp2f(t);
    if (!BF16) {
        const float rest = __builtin_amdgcn_fmed3f(fmaf(x, c_rest, fmaf(x, c, -t)), -0.01f, 0.01f);  // infinite x: of a NaN the lower bound, which leaves 0 and infinity as they are
        e *= fmaf(rest, 0.69314718f, 1.0f);
    }
    return __builtin_amdgcn_rcpf(1.0f + e);
}

using u32u = uint32_t __attribute__((aligned(1)));
using u16u = uint16_t __attribute__((aligned(1)));

// HB steps of 64 products of one row: 16 bytes of codes and one scale byte a step
template <int HB>
struct Frag {
    u32x4 c[HB];
    uint32_t s;
};

// blocks [first, first + HB) of one row; the ones at or past nb, and all of them without `valid`, are zeros.
// The row is `row` rows behind codes / scales (for items a wave-uniform address, so that a lane holds 32-bit
// offsets only: 128 rows of at most 2048 blocks).
template <int HB, typename Row>
__device__ __forceinline__ void load_frag(Frag<HB>& f, const uint8_t* codes, const uint8_t* scales, Row row, int nb, int first,
                                          bool valid) {
    const Row blk = row * (Row)nb + (Row)first;
    const u32x4* src = reinterpret_cast<const u32x4*>(codes + blk * 16);
    const uint8_t* ss = scales + blk;
    f.s = 0x7f7f7f7fu;
    if (valid && first + HB <= nb) {
#pragma unroll
        for (int kk = 0; kk < HB; ++kk) f.c[kk] = src[kk];
        if (HB == 4) {
            f.s = *reinterpret_cast<const u32u*>(ss);
        } else if (HB == 2) {
            f.s = *reinterpret_cast<const u16u*>(ss);
        } else {
            f.s = 0;
#pragma unroll
            for (int kk = 0; kk < HB; ++kk) f.s |= (uint32_t)ss[kk] << (8 * kk);
        }
    } else {
#pragma unroll
        for (int kk = 0; kk < HB; ++kk) {
            f.c[kk] = u32x4{0, 0, 0, 0};
            if (valid && first + kk < nb) {
                f.c[kk] = src[kk];
                f.s ^= (0x7fu ^ ss[kk]) << (8 * kk);
            }
        }
    }
}

template <int HB>
__device__ __forceinline__ void copy_frag(Frag<HB>& to, const Frag<HB>& from) {
#pragma unroll
    for (int kk = 0; kk < HB; ++kk) to.c[kk] = from.c[kk];
    to.s = from.s;
}

// the row of Q behind query b: -1 without one, -2 for an id outside the table
__device__ __forceinline__ int64_t query_row(const MxArgs& a, int64_t b) {
    if (b >= a.B) return -1;
    if (!a.user_rows) return b;
    const int64_t r = a.user_rows[b];
    return r >= 0 && r < a.n_q ? r : -2;
}
// QD: the queries' type.  f32 and bf16 ones are quantised here, 32 elements of a row by one lane
template <int QD, int HB>
__device__ __forceinline__ void load_query(Frag<HB>& f, const MxArgs& a, int64_t row, int first) {
    if (QD != LGX_DTYPE_MXFP4) {
        f.s = 0x7f7f7f7fu;
#pragma unroll
        for (int kk = 0; kk < HB; ++kk) {
            f.c[kk] = u32x4{0, 0, 0, 0};
            const int c0 = (first + kk) * kBlock;
            if (row < 0 || c0 >= a.d) continue;
            float x[4][8] = {};
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t at = row * a.q_ld + c0 + 8 * i;
                if (a.q_vec) {
                    if (c0 + 8 * i < a.d) {
                        if (QD == LGX_DTYPE_BF16)
                            load8_bf16<true>(reinterpret_cast<const uint16_t*>(a.q) + at, x[i]);
                        else
                            load8_f32<true>(reinterpret_cast<const float*>(a.q) + at, x[i]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (c0 + 8 * i + j < a.d)
                            x[i][j] = QD == LGX_DTYPE_BF16 ? bf16_to_f32(reinterpret_cast<const uint16_t*>(a.q)[at + j])
                                                           : reinterpret_cast<const float*>(a.q)[at + j];
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(x[i][j]) & 0x7fffffffu);
            }
            const uint32_t b = scale_byte(most);
            const float inv = __uint_as_float((254u - b) << 23);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[i][j] *= inv;
                f.c[kk][i] = b == 255u ? 0u : pack8(x[i]);
            }
            f.s ^= (0x7fu ^ b) << (8 * kk);
        }
        if (row == -2) f.s = 0xffffffffu;
        return;
    }
    load_frag<HB, int64_t>(f, a.q, a.qs, row, (int)a.nb, first, row >= 0);
    if (row == -2) f.s = 0xffffffffu;  // NaN scales
}

// items past the end repeat the last one
__device__ __forceinline__ uint32_t item_row(const MxArgs& a, int64_t base, int j) {
    return (uint32_t)min((int64_t)j, a.n_items - 1 - base);
}

template <int HB>
__device__ __forceinline__ void mma_steps(f32x16 (&acc)[4], const Frag<HB>& q, const Frag<HB> (&it)[4]) {
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] = mma<0>(q.c[0], it[t].c[0], acc[t], q.s, it[t].s);
    if (HB > 1)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t] = mma<1>(q.c[HB > 1 ? 1 : 0], it[t].c[HB > 1 ? 1 : 0], acc[t], q.s, it[t].s);
    if (HB > 2)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t] = mma<2>(q.c[HB > 2 ? 2 : 0], it[t].c[HB > 2 ? 2 : 0], acc[t], q.s, it[t].s);
    if (HB > 3)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t] = mma<3>(q.c[HB > 3 ? 3 : 0], it[t].c[HB > 3 ? 3 : 0], acc[t], q.s, it[t].s);
}

// 32 users x 128 items of results.  The items' tile t of lane l is item base + 4 (l % 32) + t, so that a lane's
// four results of one user are neighbours in the output row: one 16-byte store (512 bytes of a row per
// half-wave).
// NT: past the caches
template <bool NT, typename V, typename P>
__device__ __forceinline__ void put(V v, P* p) {
    if (NT)
        __builtin_nontemporal_store(v, p);
    else
        *p = v;
}

template <bool BF16, bool SIG, bool NT>
__device__ __forceinline__ void store_tile(const MxArgs& a, const f32x16 (&acc)[4], int64_t u0, int64_t base, int lane) {
    const int64_t left = a.n_items - base - 4 * (lane & 31);
    if (left <= 0) return;
    // a wave-uniform row plus a 32-bit lane offset (n_items < 2^27)
    const uint32_t off = (uint32_t)(4 * (lane >> 5)) * (uint32_t)a.n_items + 4u * (lane & 31);
    const int64_t u_lane = u0 + 4 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int64_t r = 8 * (i / 4) + i % 4;
        if (u_lane + r >= a.B) continue;
        float v[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) v[t] = SIG ? sigmoid<BF16>(acc[t][i]) : acc[t][i];
        if (BF16) {
            uint16_t* o = static_cast<uint16_t*>(a.out) + (u0 + r) * a.n_items + base + off;
            if (left >= 4) {
                put<NT>(u32x2u{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])}, reinterpret_cast<u32x2u*>(o));
            } else {
                o[0] = f32_to_bf16(v[0]);
                if (left > 1) o[1] = f32_to_bf16(v[1]);
                if (left > 2) o[2] = f32_to_bf16(v[2]);
            }
        } else {
            float* o = static_cast<float*>(a.out) + (u0 + r) * a.n_items + base + off;
            if (left >= 4) {
                put<NT>(f32x4u{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4u*>(o));
            } else {
                o[0] = v[0];
                if (left > 1) o[1] = v[1];
                if (left > 2) o[2] = v[2];
            }
        }
    }
}

constexpr int kUserTiles = 8;  // tiles of 32 users a workgroup of score_mx_short walks

// Rows of at most 8 blocks (d <= 256), HB = ceil(nb / 2): a wave keeps 128 items in registers and walks the
// users' tiles; the next tile's rows are loaded before this one's scores are stored, so that no load waits
// behind a store.  Bound by the writes of the score matrix: 1024 x 1M x 256 f32, 4.1 GB, in 0.76 ms (the same stores
// without loads and products 0.755); 2048 x 40,981 x 64 with the sigmoid 70 us (62 at best; a call 74 to 78).
template <int HB, bool BF16, bool SIG, bool NT>
__global__ __launch_bounds__(256, 2) void score_mx_short(MxArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31;
    const int first = HB * (lane >> 5);
    // workgroups go to the 8 XCDs in turn; rows whose stores share lines put neighbours on one XCD, so that one
    // L2 sees both parts of a line (2048 x 40,981: 94 -> 75 us; whole-line rows 793 -> 804)
    const uint32_t bx = NT ? blockIdx.x : blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8;
    const int64_t base = (bx * (int64_t)4 + wave) * 128;
    if (base >= a.n_items) return;
    const int64_t u_end = min(a.B, (blockIdx.y + (int64_t)1) * (kUserTiles * 32));
    int64_t u0 = blockIdx.y * (int64_t)(kUserTiles * 32);
    Frag<HB> it[4], q;
#pragma unroll
    for (int t = 0; t < 4; ++t)
        load_frag<HB, uint32_t>(it[t], a.it + base * a.nb * 16, a.its + base * a.nb, item_row(a, base, 4 * col + t), (int)a.nb,
                                first, true);
    load_query<LGX_DTYPE_MXFP4, HB>(q, a, query_row(a, u0 + col), first);
    for (; u0 < u_end; u0 += 32) {
        Frag<HB> next;
        if (u0 + 32 < u_end) load_query<LGX_DTYPE_MXFP4, HB>(next, a, query_row(a, u0 + 32 + col), first);
        f32x16 acc[4] = {};
        mma_steps<HB>(acc, q, it);
        store_tile<BF16, SIG, NT>(a, acc, u0, base, lane);
        copy_frag<HB>(q, next);
    }
}

// The same for one tile of users: a wave keeps that, quantised by itself, and walks the items, the next 128 on their way.
// Bound by the reading of the table: 1 x 1M x 256, 136 MB, in 29 us.  Four steps (d of 193 to 256) take all 256 registers and
// spill 12 to 28 of them, 64 where it packs the queries and writes bf16 scores without the sigmoid: a call of 1 x 1M x 256 takes 36 us
// there, 31 with the sigmoid, 30 with f32 scores.
template <int QD, int HB, bool BF16, bool SIG, bool NT>
__global__ __launch_bounds__(256, 2) void score_mx_few(MxArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31;
    const int first = HB * (lane >> 5);
    const int64_t stride = gridDim.x * (int64_t)512;
    int64_t base = (blockIdx.x * (int64_t)4 + wave) * 128;
    if (base >= a.n_items) return;
    auto load_items = [&](Frag<HB> (&it)[4], int64_t at) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
            load_frag<HB, uint32_t>(it[t], a.it + at * a.nb * 16, a.its + at * a.nb, item_row(a, at, 4 * col + t), (int)a.nb, first, true);
    };
    Frag<HB> it[4], q;
    load_items(it, base);
    load_query<QD, HB>(q, a, query_row(a, col), first);
#pragma unroll 1
    for (;;) {
        const int64_t next_base = base + stride;
        Frag<HB> next[4];
        if (next_base < a.n_items) load_items(next, next_base);
        f32x16 acc[4] = {};
        mma_steps<HB>(acc, q, it);
        store_tile<BF16, SIG, NT>(a, acc, 0, base, lane);
        if (next_base >= a.n_items) break;
        base = next_base;
#pragma unroll
        for (int t = 0; t < 4; ++t) copy_frag<HB>(it[t], next[t]);
    }
}

// Longer rows.  A workgroup holds UW x NU x 32 users against 4 / UW x 128 items, a wave NU x 32 x 128 of them, and walks the
// blocks 8 at a time through LDS: read from there a row's 16 bytes a lane cost a line each (333 x 91,599 x 1000: 93 us, its
// address unit busy throughout), while 8 lanes fetch the 128 bytes of a row together.  The next 8 blocks are on their way
// in registers during the products.  Block b of a row lies at slot b ^ (r % 8) of the row's 128 bytes, of an item's at b ^ (r / 4 %
// 8), so that 8 lanes that read one block of 8 rows (items: every fourth) touch all banks.  333 x 91,599 x 1000 bf16: 43 to 45 us, for 49 MB of
// codes (23 us of memory time with the 61 MB of scores): 1080 workgroups of two a CU are 2.1 fillings of the chip, of 384 users.  Few
// users leave CUs idle (184 workgroups): 1 x 91,599 x 1000 12 us with packed queries, 15 with f32 ones, which a launch of its own packs;
// 8 x 200,000 x 768 16 and 19 (17 us of memory time).
template <int UW, int NU, bool BF16, bool SIG, bool NT>
__global__ __launch_bounds__(256, 2) void score_mx_long(MxArgs a, int user_tiles) {
    constexpr int kUsers = UW * NU * 32, kItems = 4 / UW * 128, kRows = kUsers + kItems;
    constexpr int kUnits = kRows / 32, kScales = (kRows + 255) / 256;
    __shared__ u32x4 codes[kRows * 8];
    __shared__ uint32_t scales[kRows * 2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the user tiles of one item tile run side by side on one XCD (workgroups go to the 8 XCDs in turn)
    const int64_t turn = blockIdx.x / 8;
    const int64_t base = (turn / user_tiles * 8 + blockIdx.x % 8) * kItems, u0 = turn % user_tiles * kUsers;
    if (base >= a.n_items) return;
    const int nb = (int)a.nb, blk = tid & 7, row0 = tid >> 3;
    const uint8_t* it = a.it + base * nb * 16;
    const uint8_t* its = a.its + base * nb;
    const int last_item = (int)min((int64_t)kItems, a.n_items - base) - 1;  // rows past it repeat it
    int64_t q_row[UW * NU];
#pragma unroll
    for (int j = 0; j < UW * NU; ++j) q_row[j] = query_row(a, u0 + row0 + 32 * j);
    int64_t s_row[kScales];  // users: as query_row; items: the row
#pragma unroll
    for (int j = 0; j < kScales; ++j) {
        const int r = tid + 256 * j;
        s_row[j] = r < kUsers ? query_row(a, u0 + r) : min(r - kUsers, last_item);
    }
    u32x4 c[kUnits];
    uint32_t sc[kScales][2];
    auto fetch = [&](int k0) {
        const bool in = k0 + blk < nb;
#pragma unroll
        for (int j = 0; j < kUnits; ++j) {
            c[j] = u32x4{0, 0, 0, 0};
            if (j < UW * NU) {
                if (in && q_row[j < UW * NU ? j : 0] >= 0)
                    c[j] = *reinterpret_cast<const u32x4*>(a.q + (q_row[j < UW * NU ? j : 0] * nb + k0 + blk) * 16);
            } else if (in) {
                const uint32_t r = (uint32_t)min(row0 + 32 * (j - UW * NU), last_item);
                c[j] = *reinterpret_cast<const u32x4*>(it + (r * (uint32_t)nb + (uint32_t)(k0 + blk)) * 16u);
            }
        }
#pragma unroll
        for (int j = 0; j < kScales; ++j) {
            const int r = tid + 256 * j;
            const bool user = r < kUsers;
            sc[j][0] = sc[j][1] = user && s_row[j] == -2 ? 0xffffffffu : 0x7f7f7f7fu;
            if (r >= kRows || s_row[j] < 0) continue;
            const uint8_t* p = user ? a.qs + s_row[j] * nb + k0 : its + s_row[j] * nb + k0;
            if (k0 + 8 <= nb) {
                sc[j][0] = *reinterpret_cast<const u32u*>(p);
                sc[j][1] = *reinterpret_cast<const u32u*>(p + 4);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (k0 + k < nb) sc[j][k / 4] ^= (0x7fu ^ p[k]) << (8 * (k % 4));
            }
        }
    };
    auto stage = [&]() {
#pragma unroll
        for (int j = 0; j < kUnits; ++j) codes[(row0 + 32 * j) * 8 + (blk ^ ((j < UW * NU ? row0 : row0 >> 2) & 7))] = c[j];
#pragma unroll
        for (int j = 0; j < kScales; ++j)
            if (tid + 256 * j < kRows) {
                scales[(tid + 256 * j) * 2] = sc[j][0];
                scales[(tid + 256 * j) * 2 + 1] = sc[j][1];
            }
    };
    const int col = lane & 31, half = lane >> 5;
    const int users = wave % UW * NU * 32, items = wave / UW * 128;  // this wave's within the workgroup's
    f32x16 acc[NU][4] = {};
    fetch(0);
    for (int k0 = 0; k0 < nb; k0 += 8) {
        __syncthreads();
        stage();
        __syncthreads();
        if (k0 + 8 < nb) fetch(k0 + 8);
        uint32_t sq[NU], si[4];
#pragma unroll
        for (int u = 0; u < NU; ++u) sq[u] = scales[(users + 32 * u + col) * 2 + half];
#pragma unroll
        for (int t = 0; t < 4; ++t) si[t] = scales[(kUsers + items + 4 * col + t) * 2 + half];
        auto step = [&](auto kk) {
            constexpr int KK = decltype(kk)::value;
            u32x4 q[NU];
#pragma unroll
            for (int u = 0; u < NU; ++u) q[u] = codes[(users + 32 * u + col) * 8 + ((4 * half + KK) ^ (col & 7))];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int r = kUsers + items + 4 * col + t;
                const u32x4 x = codes[r * 8 + ((4 * half + KK) ^ (col & 7))];
#pragma unroll
                for (int u = 0; u < NU; ++u) acc[u][t] = mma<KK>(q[u], x, acc[u][t], sq[u], si[t]);
            }
        };
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
        step(std::integral_constant<int, 2>{});
        step(std::integral_constant<int, 3>{});
    }
    if (base + items >= a.n_items) return;
#pragma unroll
    for (int u = 0; u < NU; ++u)
        if (u0 + users + 32 * u < a.B) store_tile<BF16, SIG, NT>(a, acc[u], u0 + users + 32 * u, base + items, lane);
}

#define LGX_MX_STEPS(KERNEL, ...)                                        \
    switch ((a.nb + 1) / 2) {                                            \
        case 1: KERNEL(1, __VA_ARGS__); break;                           \
        case 2: KERNEL(2, __VA_ARGS__); break;                           \
        case 3: KERNEL(3, __VA_ARGS__); break;                           \
        default: KERNEL(4, __VA_ARGS__); break;                          \
    }
#define LGX_MX_FEW(HB, QD) score_mx_few<QD, HB, BF16, SIG, NT><<<grid, 256, 0, stream>>>(a)
#define LGX_MX_SHORT(HB, ...) score_mx_short<HB, BF16, SIG, NT><<<grid, 256, 0, stream>>>(a)

template <bool BF16, bool SIG, bool NT>
int launch_score(const MxArgs& a, int q_dtype, hipStream_t stream) {
    if (a.nb <= 8 && a.B <= 32) {
        // two workgroups a CU
        const dim3 grid((unsigned)std::min<int64_t>(512, ceil_div(a.n_items, (int64_t)512)));
        if (q_dtype == LGX_DTYPE_F32) { LGX_MX_STEPS(LGX_MX_FEW, LGX_DTYPE_F32) }
        else if (q_dtype == LGX_DTYPE_BF16) { LGX_MX_STEPS(LGX_MX_FEW, LGX_DTYPE_BF16) }
        else { LGX_MX_STEPS(LGX_MX_FEW, LGX_DTYPE_MXFP4) }
    } else if (a.nb <= 8) {
        const int64_t gy = ceil_div(a.B, (int64_t)(kUserTiles * 32));
        const int64_t gx = ceil_div(a.n_items, (int64_t)512);
        const dim3 grid((unsigned)(NT ? gx : 8 * ceil_div(gx, (int64_t)8)), (unsigned)gy);
        LGX_MX_STEPS(LGX_MX_SHORT, 0)
    } else {
        // Two waves side by side over the users where there are enough of them, and from the third tile of users on two tiles
        // a wave, which read an item's codes half as often.  Against one tile: 2048 x 30,000 x 4096 f32 206 us (254),
        // 128 x 100,000 x 512 14.7 (17.1), 1024 x 100,000 x 512 85.5 (83.6), 1024 x 20,000 x 300 24.2 (22.8)
        const int uw = a.B > 32 ? 2 : 1, nu = a.B > 64 ? 2 : 1;
        const int64_t user_tiles = ceil_div(a.B, (int64_t)(uw * nu * 32));
        const int64_t grid = 8 * ceil_div(ceil_div(a.n_items, (int64_t)(512 / uw)), (int64_t)8) * user_tiles;
        // (scores of so many tiles would not fit the memory)
        LGX_REQUIRE(grid < (1LL << 24), LGX_ERR_UNSUPPORTED, "lgx_score_mx: %lld queries of %lld items is too many", (long long)a.B,
                    (long long)a.n_items);
        if (nu == 2) score_mx_long<2, 2, BF16, SIG, NT><<<(unsigned)grid, 256, 0, stream>>>(a, (int)user_tiles);
        else if (uw == 2) score_mx_long<2, 1, BF16, SIG, NT><<<(unsigned)grid, 256, 0, stream>>>(a, (int)user_tiles);
        else score_mx_long<1, 1, BF16, SIG, NT><<<(unsigned)grid, 256, 0, stream>>>(a, (int)user_tiles);
    }
    LGX_LAUNCH_CHECK();
    return LGX_OK;
}

// One tile of users over rows of at most 8 blocks: every wave of score_mx_few quantises it for itself (a launch less: 57 ->
// 52 us for a call of 1 x 1 M x 256 by itself); with more of them, once for all by a launch of its own
bool quantised_inside(int64_t B, int64_t d) { return B <= 32 && d <= 8 * kBlock; }

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Rows (queries) of a launch: a grid holds less than 2^32 threads, and 64 blocks take 256
constexpr int64_t kMostBlocks = 1 << 28, kMostQueries = 1 << 22;

int launch_quantize(const void* X, const int64_t* rows_of, int64_t n_src, int64_t rows, int64_t d, int64_t ld, int dtype,
                    uint8_t* codes, uint8_t* scales, hipStream_t stream) {
    const int64_t nb = ceil_div(d, (int64_t)kBlock), most = kMostBlocks / nb;
    const int size = dtype == LGX_DTYPE_BF16 ? 2 : 4;
    const bool vec = d % 8 == 0 && (ld * size) % 16 == 0 && aligned(X, 16);
#define LGX_MXQ(BF, V)                                                                                                  \
    mx_quantize_kernel<BF, V><<<grid, 256, 0, stream>>>(static_cast<const char*>(X) + (rows_of ? 0 : first * ld * size),  \
                                                        rows_of ? rows_of + first : nullptr, n_src, units, nb, d, ld,     \
                                                        codes + first * nb * 16, scales + first * nb)
    for (int64_t first = 0; first < rows; first += most) {
        const int64_t units = std::min(most, rows - first) * nb;
        const unsigned grid = (unsigned)ceil_div(units, (int64_t)64);
        if (dtype == LGX_DTYPE_BF16) {
            if (vec) LGX_MXQ(true, true); else LGX_MXQ(true, false);
        } else {
            if (vec) LGX_MXQ(false, true); else LGX_MXQ(false, false);
        }
        LGX_LAUNCH_CHECK();
    }
#undef LGX_MXQ
    return LGX_OK;
}

}  // namespace
}  // namespace lgx

using namespace lgx;

extern "C" int lgx_mx_quantize(const void* X, int64_t rows, int64_t d, int64_t ld, int dtype, uint8_t* codes,
                               uint8_t* scales, lgx_stream_t stream) {
    LGX_REQUIRE(rows >= 0 && (rows == 0 || (X && codes && scales)), LGX_ERR_INVALID_ARG, "lgx_mx_quantize: bad arguments");
    LGX_REQUIRE(dtype == LGX_DTYPE_F32 || dtype == LGX_DTYPE_BF16, LGX_ERR_INVALID_ARG, "lgx_mx_quantize: dtype");
    LGX_REQUIRE(d >= 1 && d <= kMaxD && ld >= d, LGX_ERR_UNSUPPORTED, "lgx_mx_quantize: d=%lld outside [1, %lld] or ld=%lld < d",
                (long long)d, (long long)kMaxD, (long long)ld);
    LGX_REQUIRE(aligned(codes, 16), LGX_ERR_INVALID_ARG, "lgx_mx_quantize: codes must be 16-byte aligned");
    LGX_REQUIRE(rows < (1LL << 36), LGX_ERR_UNSUPPORTED, "lgx_mx_quantize: %lld rows is too many", (long long)rows);
    return launch_quantize(X, nullptr, rows, rows, d, ld, dtype, codes, scales, as_hip(stream));
}

extern "C" int lgx_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t d, int dtype, void* out,
                                 lgx_stream_t stream_) {
    hipStream_t stream = as_hip(stream_);
    LGX_REQUIRE(rows >= 0 && (rows == 0 || (codes && scales && out)), LGX_ERR_INVALID_ARG,
                "lgx_mx_dequantize: bad arguments");
    LGX_REQUIRE(dtype == LGX_DTYPE_F32 || dtype == LGX_DTYPE_BF16, LGX_ERR_INVALID_ARG, "lgx_mx_dequantize: dtype");
    LGX_REQUIRE(d >= 1 && d <= kMaxD, LGX_ERR_UNSUPPORTED, "lgx_mx_dequantize: d=%lld outside [1, %lld]", (long long)d,
                (long long)kMaxD);
    LGX_REQUIRE(aligned(codes, 16), LGX_ERR_INVALID_ARG, "lgx_mx_dequantize: codes must be 16-byte aligned");
    if (rows == 0) return LGX_OK;
    LGX_REQUIRE(rows < (1LL << 36), LGX_ERR_UNSUPPORTED, "lgx_mx_dequantize: %lld rows is too many", (long long)rows);
    const int64_t nb = ceil_div(d, (int64_t)kBlock), most = kMostBlocks / nb;
    const int size = dtype == LGX_DTYPE_BF16 ? 2 : 4;
    const bool vec = d % 8 == 0 && aligned(out, 16);
#define LGX_MXD(BF, V)                                                                                              \
    mx_dequantize_kernel<BF, V><<<grid, 256, 0, stream>>>(codes + first * nb * 16, scales + first * nb, units, nb, d, \
                                                          static_cast<char*>(out) + first * d * size)
    for (int64_t first = 0; first < rows; first += most) {
        const int64_t units = std::min(most, rows - first) * nb;
        const unsigned grid = (unsigned)ceil_div(units, (int64_t)64);
        if (dtype == LGX_DTYPE_BF16) {
            if (vec) LGX_MXD(true, true); else LGX_MXD(true, false);
        } else {
            if (vec) LGX_MXD(false, true); else LGX_MXD(false, false);
        }
        LGX_LAUNCH_CHECK();
    }
#undef LGX_MXD
    return LGX_OK;
}

extern "C" int lgx_score_mx_workspace(int64_t B, int64_t d, int q_dtype, size_t* ws_bytes) {
    LGX_REQUIRE(ws_bytes && B >= 0 && d >= 1 && d <= kMaxD, LGX_ERR_INVALID_ARG, "lgx_score_mx_workspace: bad arguments");
    const size_t nb = (size_t)ceil_div(d, (int64_t)kBlock);
    *ws_bytes = q_dtype == LGX_DTYPE_MXFP4 || quantised_inside(B, d) ? 0 : align_up((size_t)B * nb * 16) + align_up((size_t)B * nb);
    return LGX_OK;
}

extern "C" int lgx_score_mx(const void* Q, const uint8_t* q_scales, int q_dtype, int64_t n_q, int64_t q_ld,
                            const int64_t* user_rows, const uint8_t* item_codes, const uint8_t* item_scales, int64_t B,
                            int64_t n_items, int64_t d, int apply_sigmoid, int out_dtype, void* scores, void* ws,
                            size_t ws_bytes, lgx_stream_t stream_) {
    hipStream_t stream = as_hip(stream_);
    LGX_REQUIRE(B >= 0 && n_items >= 0 && n_q >= 0, LGX_ERR_INVALID_ARG, "lgx_score_mx: negative size");
    LGX_REQUIRE(q_dtype == LGX_DTYPE_F32 || q_dtype == LGX_DTYPE_BF16 || q_dtype == LGX_DTYPE_MXFP4, LGX_ERR_INVALID_ARG,
                "lgx_score_mx: query dtype");
    LGX_REQUIRE(out_dtype == LGX_DTYPE_F32 || out_dtype == LGX_DTYPE_BF16, LGX_ERR_INVALID_ARG, "lgx_score_mx: out dtype");
    LGX_REQUIRE(d >= 1 && d <= kMaxD, LGX_ERR_UNSUPPORTED, "lgx_score_mx: d=%lld outside [1, %lld]", (long long)d,
                (long long)kMaxD);
    LGX_REQUIRE(n_items < (1LL << 27), LGX_ERR_UNSUPPORTED, "lgx_score_mx: %lld items is too many (< 2^27)",
                (long long)n_items);
    if (B == 0 || n_items == 0) return LGX_OK;
    LGX_REQUIRE((Q || n_q == 0) && item_codes && item_scales && scores, LGX_ERR_INVALID_ARG, "lgx_score_mx: null pointer");
    LGX_REQUIRE(user_rows || B <= n_q, LGX_ERR_INVALID_ARG, "lgx_score_mx: %lld queries of %lld rows", (long long)B,
                (long long)n_q);
    LGX_REQUIRE(aligned(item_codes, 16), LGX_ERR_INVALID_ARG, "lgx_score_mx: codes must be 16-byte aligned");
    const int64_t nb = ceil_div(d, (int64_t)kBlock);
    MxArgs a{static_cast<const uint8_t*>(Q), q_scales, user_rows, n_q, item_codes, item_scales, B, n_items, nb, scores, d, q_ld, false};
    if (q_dtype == LGX_DTYPE_MXFP4) {
        LGX_REQUIRE((q_scales || n_q == 0) && aligned(Q, 16), LGX_ERR_INVALID_ARG, "lgx_score_mx: query codes must be 16-byte aligned, with scales");
    } else {
        LGX_REQUIRE(q_ld >= d, LGX_ERR_INVALID_ARG, "lgx_score_mx: q_ld=%lld < d", (long long)q_ld);
        size_t need = 0;
        lgx_score_mx_workspace(B, d, q_dtype, &need);
        a.q_vec = d % 8 == 0 && q_ld * (q_dtype == LGX_DTYPE_BF16 ? 2 : 4) % 16 == 0 && aligned(Q, 16);
        LGX_REQUIRE(need == 0 || (ws && ws_bytes >= need && aligned(ws, 16)), LGX_ERR_WORKSPACE, "lgx_score_mx: workspace %zu < %zu", ws_bytes, need);
        if (!quantised_inside(B, d)) {
            uint8_t* codes = static_cast<uint8_t*>(ws);
            uint8_t* scales = codes + align_up((size_t)B * nb * 16);
            const int rc = launch_quantize(Q, user_rows, n_q, B, d, q_ld, q_dtype, codes, scales, stream);
            if (rc) return rc;
            a.q = codes;
            a.qs = scales;
            a.user_rows = nullptr;
            a.n_q = B;
            q_dtype = LGX_DTYPE_MXFP4;
        }
    }
    // Rows that start on a 128-byte line write whole lines, which go past the L2 (1024 x 1 M f32: 0.79 against
    // 0.94 ms); the ends of other rows' stores share lines, which the L2 merges (2048 x 40,981: 119 us past it).
    const bool nt = aligned(scores, 128) && n_items * (out_dtype == LGX_DTYPE_BF16 ? 2 : 4) % 128 == 0;
#define LGX_SMX(BF, SG) (nt ? launch_score<BF, SG, true>(b, q_dtype, stream) : launch_score<BF, SG, false>(b, q_dtype, stream))
    for (int64_t first = 0; first < B; first += kMostQueries) {
        MxArgs b = a;
        b.B = std::min(kMostQueries, B - first);
        b.out = static_cast<char*>(scores) + first * n_items * (out_dtype == LGX_DTYPE_BF16 ? 2 : 4);
        if (b.user_rows) {
            b.user_rows += first;
        } else if (first) {  // packed rows: more of them than a wave quantises by itself
            b.q += first * nb * 16;
            b.qs += first * nb;
        }
        const int rc = out_dtype == LGX_DTYPE_BF16 ? (apply_sigmoid ? LGX_SMX(true, true) : LGX_SMX(true, false))
                                                   : (apply_sigmoid ? LGX_SMX(false, true) : LGX_SMX(false, false));
        if (rc) return rc;
    }
#undef LGX_SMX
    return LGX_OK;
}
