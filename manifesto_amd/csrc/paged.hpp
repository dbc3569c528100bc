// paged.hpp — what the paged-cache kernels share: the cache's checks, exact
// division by a launch's constants, 16-bit and FP8 pieces, matrix products.
#ifndef MFH_PAGED_HPP
#define MFH_PAGED_HPP

#include "common.hpp"
#include "launch.hpp"
#include "../../include/mfh_attention.h"

namespace mfh {

int check_cache(const mfh_kv_cache* cache, const char* what);  // decode.hip
int check_attention(const mfh_attention_shape* shape, const mfh_kv_cache* cache, const char* what);

// Tokens of a request, and rows of a call, at most: sums and differences of two
// positions and a window fit 32 bits.
constexpr int kLongest = 1 << 30;

// A descriptor's pair of strides, where two zeros stand for [tokens][heads][dim].
struct Strides {
    int64_t token, head;
    Strides(int64_t t, int64_t h, int64_t heads, int64_t dim)
        : token(t || h ? t : heads * dim), head(t || h ? h : dim)
    {
    }
};

// n / d for n below 2^31 and a d known at launch: n * ceil(2^(31 + s) / d) >>
// (31 + s) with 2^s >= d, where the rounding adds n * d * 2^-(31 + s) < 1 to
// the quotient's numerator.
struct Divider {
    mfh_u32 m, shift, d;
    Divider() = default;
    explicit Divider(mfh_u32 by) : d(by)
    {
        mfh_u32 s = 0;
        while (((mfh_u64)1 << s) < by) s++;
        shift = 31 + s;
        m = (mfh_u32)((((mfh_u64)1 << shift) + by - 1) / by);
    }
    __device__ mfh_u32 quotient(mfh_u32 n) const { return (mfh_u32)((mfh_u64)n * m >> shift); }
    __device__ mfh_i64 quotient64(mfh_i64 n) const { return n >> 31 ? n / (mfh_i64)d : (mfh_i64)quotient((mfh_u32)n); }
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <int DT>
MFH_DEV float dec16(mfh_u32 h)
{
    return DT == kBFloat16 ? mfh_bf16_to_f32(h) : mfh_f16_to_f32(h);
}

template <int DT>
MFH_DEV mfh_u32 enc16x2(float lo, float hi)
{
    if constexpr (DT == kBFloat16) return mfh_bf16x2_rne(lo, hi);
    else return mfh_f16x2_rne(lo, hi);
}

// Four E4M3 codes by the hardware's conversion (nearest, ties to even, into
// subnormals too; the codec of mfh_convert keeps the reference's subnormal
// rule instead), limited to the largest finite value first.  NaN stays NaN.
MFH_DEV float e4m3_limit(float v) { return v > 448.0f ? 448.0f : v < -448.0f ? -448.0f : v; }

MFH_DEV mfh_u32 e4m3x4(float v0, float v1, float v2, float v3)
{
    mfh_u32 w = (mfh_u32)__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_limit(v0), e4m3_limit(v1), 0, false);
    return (mfh_u32)__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_limit(v2), e4m3_limit(v3), (int)w, true);
}

// Two of a dword's four E4M3 codes as bf16 or f16 (both hold every code exactly).
template <int DT, bool HIGH>
MFH_DEV mfh_u32 e4m3_pair(mfh_u32 codes)
{
    if constexpr (DT == kBFloat16)
        return __builtin_bit_cast(mfh_u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, HIGH));
    else return __builtin_bit_cast(mfh_u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, HIGH));
}

// c + a b with eight 16-bit values of a's row and of b's column per lane.
// 16 x 16 x 32: row / column lane % 16, values 8 * (lane / 16) ..; c: column
// lane % 16, rows 4 * (lane / 16) ...
template <int DT>
MFH_DEV f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c)
{
    if constexpr (DT == kBFloat16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// 32 x 32 x 16: row / column lane % 32, values 8 * (lane / 32) ..; c: column
// lane % 32, element i is row 8 * (i / 4) + 4 * (lane / 32) + i % 4.
template <int DT>
MFH_DEV f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c)
{
    if constexpr (DT == kBFloat16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

MFH_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The softmax's running reference moves where a score passes `limit`, which is
// 2^kStep above the largest score at the last move; weights are 2^(score - reference).
// In f16 the reference stands kBelow under that score, so that weights fill the
// type's range (up to 2^15) and the smallest ones, of which a long context can have
// many, keep their bits down to 2^-21 of the largest; from 1 down they would lose
// them from 2^-14 on.  In bf16, which has f32's exponents, it stands at the limit:
// weights are 1 at most, and products with the largest values stay finite where the
// result is.  (Eight-bit values are at most 448, their scale is the result's.)
constexpr float kStep = 8.0f;
template <int DT, bool FP8>
constexpr float kBelow = DT == kFloat16 ? 7.0f : FP8 ? 0.0f : -kStep;

// Scores are in units of log2(e) on the way to exp2: scaled * tanh(x / scaled) with
// scaled = cap log2(e), from twice = 2 / cap: tanh y = 1 - 2 / (1 + e^2y), which ends
// at -1 and 1 without a case of its own.
MFH_DEV float capped(float x, float twice, float scaled)
{
    return scaled * (1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + exp2_fast(x * twice)));
}

// That difference is off by up to 2^-22 of the cap, however small the score: under
// 2^-16 for caps up to kWideCap, far below a weight's rounding to 16 bits.  Above it
// scores of less than an eighth of the cap take tanh's series, x (1 - y^2 / 3 +
// 2 y^4 / 15), whose first missing term is 2^-22 of the first; the others are within
// 2^-19 of themselves.  Both have to be computed: a prompt of 4096, 32 heads over 8
// of 128, 303 us, and 218 with `capped`, which caps that models have in use keep.
constexpr float kWideCap = 64.0f;

MFH_DEV float wide_capped(float x, float scaled_inverse, float scaled)
{
    const float y = x * scaled_inverse, z = y * y;
    const float near = __builtin_fmaf(__builtin_fmaf(z, 2.0f / 15.0f, -1.0f / 3.0f) * z, x, x);
    return z < 1.0f / 64.0f ? near : capped(y, 2.0f * kLog2e, scaled);
}

// Pages a kernel reads: strides in bytes, of keys and of values alike.
struct PageArgs {
    const char* k;
    const char* v;
    const int32_t* table;
    int64_t table_stride;
    int64_t page_bytes, head_bytes;
    mfh_u32 token_bytes;  // 0 where a page holds one token
    mfh_u32 pages;
    mfh_u32 page_span;    // bytes of a page from its first element of a head to the last one
    Divider by_page;      // page size
    mfh_u32 width;
    PageArgs() = default;
    PageArgs(const mfh_kv_cache& c, const void* keys, const void* values, const int32_t* block_table, int64_t stride,
             int32_t table_width)
        : k((const char*)keys), v((const char*)values), table(block_table), table_stride(stride)
    {
        const int bytes = c.dtype == kF8E4M3 ? 1 : 2;
        page_bytes = c.page_stride * bytes, head_bytes = c.head_stride * bytes;
        token_bytes = c.page_size > 1 ? (mfh_u32)(c.token_stride * bytes) : 0;
        pages = (mfh_u32)c.pages;
        page_span = (mfh_u32)(c.page_size - 1) * token_bytes + (mfh_u32)(c.head_dim * bytes);
        by_page = Divider((mfh_u32)c.page_size);
        width = (mfh_u32)table_width;
    }
};

MFH_DEV mfh_i64 shuffle64(mfh_i64 v, int lane)
{
    const mfh_u32 lo = __shfl((int)(mfh_u32)v, lane), hi = __shfl((int)(v >> 32), lane);
    return (mfh_i64)((mfh_u64)hi << 32 | lo);
}

// A value that is the same in every lane, as the compiler may know it.
MFH_DEV mfh_u32 uniform(mfh_u32 v) { return (mfh_u32)__builtin_amdgcn_readfirstlane((int)v); }

// Sum of the lanes up to and with this one, by moves between lanes of a row of
// 16 and then from the rows before.
MFH_DEV mfh_u32 lanes_upto(mfh_u32 v)
{
    v += (mfh_u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, true);  // row_shr 1, 2, 4, 8
    v += (mfh_u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, true);
    v += (mfh_u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, true);
    v += (mfh_u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, true);
    v += (mfh_u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
    v += (mfh_u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
    return v;
}

MFH_DEV mfh_u32 last_lane(mfh_u32 v) { return (mfh_u32)__builtin_amdgcn_readlane((int)v, 63); }

}  // namespace mfh

#endif  // MFH_PAGED_HPP
