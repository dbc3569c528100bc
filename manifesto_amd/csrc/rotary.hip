// rotary.hip — rotary positions of queries and keys, with keys and values
// written to their slots of a paged cache in the same launch, and the host's
// table of frequencies (mfh_rotary, mfh_rotary_append, mfh_rotary_frequencies).
//
// A stream: every element is read and written once, so the HBM rate bounds
// it.  A workgroup takes one token, or more where a token has few heads.  Its
// threads load a unit of 2 E elements each (two 16-byte pieces where the head's
// parts allow it): E pairs of one head, or elements that are only copied (the
// head behind rotary_dim, and values).  While these are on their way they
// compute the tokens' cosines and sines, each once for all heads, into LDS.
// 16381 tokens of 32 + 8 + 8 heads of 128, half of each turned, bf16 into a cache
// of e4m3: 62 us, 5.9 TB/s; with the two pieces of whole pairs side by side, so
// that a load of the wave has gaps, and the loads behind the angles, 83 us.
//
// The phase position * frequency is reduced to one turn in f64: at position
// 2^24 its error is below 2^-28 of a turn, under the step of the f32 phase that
// the polynomials take.  A phase in f32 would be off by 2^-7 of a radian at
// position 2^17.
// Cosine and sine are Taylor polynomials on an eighth of a turn either way,
// whose first missing terms are below 2^-33.
#include "common.hpp"
#include "launch.hpp"
#include "paged.hpp"
#include "../../include/mfh_attention.h"

#include <cmath>

namespace mfh {
namespace {

constexpr int kThreads = 256;
constexpr int kMostBlocks = 1 << 23;  // of a launch dimension, which holds fewer than 2^32 threads
constexpr int kMaxPairs = 1024;  // cosines and sines in LDS: tokens of a workgroup * rotary_dim / 2

struct RotaryArgs {
    const void* q;
    void* q_out;
    const void* k;
    void* k_out;  // the result, or the key pages
    const void* v;
    void* v_out;  // the value pages
    const int32_t* positions;
    const int64_t* slots;  // NULL without a cache
    const double* frequencies;
    int64_t tokens;
    int64_t q_t, q_h, qo_t, qo_h, k_t, k_h, ko_t, ko_h, v_t, v_h;
    int64_t page_stride, slot_count;
    float factor, sine_factor, k_by, v_by;  // the last two: reciprocals of the cache's scales
    int32_t tokens_per_block;
    mfh_u32 half;          // rotary_dim / 2
    mfh_u32 q_units, k_units, units;  // running: of q, of q and k, of q, k and v
    Divider by_half, by_units, by_head, by_page;
    mfh_u32 units_per_head, turned_units;
};

// Cosine and sine of `turn` turns, |turn| <= 1/2.
MFH_DEV void cos_sin(float turn, float* c, float* s)
{
    const float quarters = __builtin_rintf(turn * 4.0f);
    const float x = (turn - quarters * 0.25f) * 6.28318530717958647692f;  // the difference is exact; |x| <= pi/4
    const float y = x * x;
    float p = -1.0f / 39916800.0f;
    p = __builtin_fmaf(p, y, 1.0f / 362880.0f);
    p = __builtin_fmaf(p, y, -1.0f / 5040.0f);
    p = __builtin_fmaf(p, y, 1.0f / 120.0f);
    p = __builtin_fmaf(p, y, -1.0f / 6.0f);
    const float sine = __builtin_fmaf(p * y, x, x);
    float q = -1.0f / 3628800.0f;
    q = __builtin_fmaf(q, y, 1.0f / 40320.0f);
    q = __builtin_fmaf(q, y, -1.0f / 720.0f);
    q = __builtin_fmaf(q, y, 1.0f / 24.0f);
    q = __builtin_fmaf(q, y, -0.5f);
    const float cosine = __builtin_fmaf(q, y, 1.0f);
    const int n = (int)quarters & 3;
    const float a = n & 1 ? sine : cosine, b = n & 1 ? cosine : sine;
    *c = n == 1 || n == 2 ? -a : a;
    *s = n >= 2 ? -b : b;
}

// E consecutive elements at any element alignment, and as f32.
template <int DT, int E>
struct Piece {
    static constexpr int kWords = DT == kFloat32 ? E : (E + 1) / 2;
    mfh_u32 w[kWords];
    MFH_DEV void load(const void* base, int64_t at)
    {
        const char* p = static_cast<const char*>(base) + at * (DT == kFloat32 ? 4 : 2);
        if constexpr (kWords == 4) {
            const u32x4 t = load16<true>(p);
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = t[i];
        } else if constexpr (kWords == 2) {
            const u32x2 t = load8<true>(p);
            w[0] = t[0], w[1] = t[1];
        } else if constexpr (DT == kFloat32 || E == 2) {
            w[0] = load4(p);
        } else {
            w[0] = load2(p);
        }
    }
    MFH_DEV float operator[](int j) const
    {
        if constexpr (DT == kFloat32) return mfh_f32(w[j]);
        else return dec16<DT>((w[j >> 1] >> (16 * (j & 1))) & 0xffffu);
    }
};

template <int DT, int E>
MFH_DEV void store(void* base, int64_t at, const float (&x)[E])
{
    if constexpr (DT == kFloat32) {
        float* p = static_cast<float*>(base) + at;
        if constexpr (E % 4 == 0) {
#pragma unroll
            for (int j = 0; j < E; j += 4)
                store16(p + j, u32x4{mfh_bits(x[j]), mfh_bits(x[j + 1]), mfh_bits(x[j + 2]), mfh_bits(x[j + 3])});
        } else {
#pragma unroll
            for (int j = 0; j < E; j++) store4(p + j, mfh_bits(x[j]));
        }
    } else if constexpr (DT == kF8E4M3) {
        mfh_u8* p = static_cast<mfh_u8*>(base) + at;
        if constexpr (E == 8) store8(p, u32x2{e4m3x4(x[0], x[1], x[2], x[3]), e4m3x4(x[4], x[5], x[6], x[7])});
        else if constexpr (E == 4) store4(p, e4m3x4(x[0], x[1], x[2], x[3]));
        else if constexpr (E == 2) store2(p, e4m3x4(x[0], x[1], 0.0f, 0.0f));
        else *p = (mfh_u8)e4m3x4(x[0], 0.0f, 0.0f, 0.0f);
    } else {
        mfh_u16* p = static_cast<mfh_u16*>(base) + at;
        if constexpr (E == 8)
            store16(p, u32x4{enc16x2<DT>(x[0], x[1]), enc16x2<DT>(x[2], x[3]), enc16x2<DT>(x[4], x[5]),
                             enc16x2<DT>(x[6], x[7])});
        else if constexpr (E == 4) store8(p, u32x2{enc16x2<DT>(x[0], x[1]), enc16x2<DT>(x[2], x[3])});
        else if constexpr (E == 2) store4(p, enc16x2<DT>(x[0], x[1]));
        else store2(p, enc16x2<DT>(x[0], 0.0f));
    }
}

// DT: of q, k, v and their results; CACHE: of the pages (DT without a cache).
template <int DT, int CACHE, int E, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void k_rotary(RotaryArgs a)
{
    __shared__ float s_cos[kMaxPairs], s_sin[kMaxPairs];
    const int64_t first = ((int64_t)blockIdx.y * kMostBlocks + blockIdx.x) * a.tokens_per_block;
    if (first >= a.tokens) return;
    const mfh_u32 tokens = (mfh_u32)min((int64_t)a.tokens_per_block, a.tokens - first);
    const mfh_u32 total = tokens * a.units;
    constexpr mfh_u32 kNone = 0xffffffffu;
    for (mfh_u32 base = 0; base < total; base += kThreads) {
        // The unit is on its way before the angles are ready.
        const mfh_u32 u = base + threadIdx.x;
        Piece<DT, E> first_piece, second_piece;
        mfh_u32 angles = kNone, second_angles = kNone;  // kNone: copied
        bool write = u < total, into_cache = false;
        float by = 1.0f;
        void* dst = nullptr;
        int64_t to = 0, second_to = 0;
        if (write) {
            const mfh_u32 t = a.by_units.quotient(u), in_token = u - t * a.units;
            const bool is_q = in_token < a.q_units, is_v = in_token >= a.k_units;
            const mfh_u32 of = in_token - (is_q ? 0 : is_v ? a.k_units : a.q_units);
            const mfh_u32 head = a.by_head.quotient(of), unit = of - head * a.units_per_head;
            const int64_t token = first + t;
            const void* src = is_q ? a.q : is_v ? a.v : a.k;
            const int64_t from = is_q   ? token * a.q_t + head * a.q_h
                                 : is_v ? token * a.v_t + head * a.v_h
                                        : token * a.k_t + head * a.k_h;
            // The pieces are those of the pairs' two halves; or, where a piece holds
            // whole pairs or is only copied, they stand half of that part of the head
            // apart, so that neighbouring lanes hold neighbouring pieces.
            mfh_u32 first_at, second_at;
            if (INTERLEAVED && E == 1 && !is_v) {
                first_at = 2 * unit, second_at = first_at + 1;
                if (unit < a.turned_units) angles = t * a.half + unit;
            } else if (INTERLEAVED || is_v) {
                first_at = unit * E, second_at = first_at + a.units_per_head * E;
                if (!is_v && first_at < 2 * a.half) angles = t * a.half + first_at / 2;
                if (!is_v && second_at < 2 * a.half) second_angles = t * a.half + second_at / 2;
            } else if (unit < a.turned_units) {
                first_at = unit * E, second_at = first_at + a.half;
                angles = t * a.half + first_at;
            } else {
                first_at = 2 * a.half + (unit - a.turned_units) * E;
                second_at = first_at + (a.units_per_head - a.turned_units) * E;
            }
            first_piece.load(src, from + first_at);
            second_piece.load(src, from + second_at);
            dst = is_q ? a.q_out : is_v ? a.v_out : a.k_out;
            to = is_q ? token * a.qo_t + head * a.qo_h : token * a.ko_t + head * a.ko_h;
            if (a.slots && !is_q) {
                const int64_t slot = a.slots[token];
                write = slot >= 0 && slot < a.slot_count;
                const int64_t page = write ? a.by_page.quotient64(slot) : 0;
                to = page * a.page_stride + (slot - page * a.by_page.d) * a.ko_t + head * a.ko_h;
                into_cache = true;
                by = is_v ? a.v_by : a.k_by;
            }
            second_to = to + second_at, to += first_at;
        }
        if (base == 0) {
            for (mfh_u32 i = threadIdx.x; i < tokens * a.half; i += kThreads) {
                const mfh_u32 t = a.by_half.quotient(i), pair = i - t * a.half;
                // turns; the product's rounding is 2^-53 of it
                double turns = (double)a.positions[first + t] * (a.frequencies[pair] * 0.15915494309189533577);
                turns -= __builtin_rint(turns);
                float c, s;
                cos_sin((float)turns, &c, &s);
                s_cos[i] = c * a.factor;
                s_sin[i] = s * a.sine_factor;
            }
            __syncthreads();
        }
        if (!write) continue;
        float x[E], y[E];
#pragma unroll
        for (int j = 0; j < E; j++) x[j] = first_piece[j], y[j] = second_piece[j];
        if constexpr (INTERLEAVED && E >= 2) {
            auto turn = [&](float (&z)[E], mfh_u32 at) {
#pragma unroll
                for (int j = 0; j < E / 2; j++) {
                    const float c = s_cos[at + j], s = s_sin[at + j], p = z[2 * j], q = z[2 * j + 1];
                    z[2 * j] = p * c - q * s;
                    z[2 * j + 1] = q * c + p * s;
                }
            };
            if (angles != kNone) turn(x, angles);
            if (second_angles != kNone) turn(y, second_angles);
        } else if (angles != kNone) {
#pragma unroll
            for (int j = 0; j < E; j++) {
                const float c = s_cos[angles + j], s = s_sin[angles + j], p = x[j], q = y[j];
                x[j] = p * c - q * s;
                y[j] = q * c + p * s;
            }
        }
        if (CACHE == kF8E4M3 && into_cache) {
#pragma unroll
            for (int j = 0; j < E; j++) x[j] *= by, y[j] *= by;
            store<CACHE, E>(dst, to, x);
            store<CACHE, E>(dst, second_to, y);
        } else {
            store<DT, E>(dst, to, x);
            store<DT, E>(dst, second_to, y);
        }
    }
}

template <int DT, int CACHE, int E>
void launch_width(bool interleaved, dim3 grid, hipStream_t s, const RotaryArgs& a)
{
    if (interleaved) k_rotary<DT, CACHE, E, true><<<grid, kThreads, 0, s>>>(a);
    else k_rotary<DT, CACHE, E, false><<<grid, kThreads, 0, s>>>(a);
}

template <int DT, int CACHE>
void launch_types(int e, bool interleaved, dim3 grid, hipStream_t s, const RotaryArgs& a)
{
    switch (e) {
    case 8:
        if constexpr (DT != kFloat32) return launch_width<DT, CACHE, 8>(interleaved, grid, s, a);
        [[fallthrough]];
    case 4: return launch_width<DT, CACHE, 4>(interleaved, grid, s, a);
    case 2: return launch_width<DT, CACHE, 2>(interleaved, grid, s, a);
    default: return launch_width<DT, CACHE, 1>(interleaved, grid, s, a);
    }
}

int check_shape(const mfh_rotary_shape* shape, int64_t tokens, const char* what)
{
    if (!shape) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL shape", what);
    const int dt = shape->dtype;
    if (dt != kFloat32 && dt != kFloat16 && dt != kBFloat16)
        return fail(MFH_ERR_DTYPE_UNSUPPORTED, "%s: dtype %s is not f32/bf16/f16", what, dtype_name(dt));
    if (shape->head_dim < 2 || shape->head_dim > 1024 || shape->head_dim % 2)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: head dim %d is not an even number in 2..1024", what,
                    shape->head_dim);
    if (shape->rotary_dim < 0 || shape->rotary_dim > shape->head_dim || shape->rotary_dim % 2)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: rotary dim %d is not an even number in 0..%d", what,
                    shape->rotary_dim, shape->head_dim);
    if (shape->q_heads < 0 || shape->kv_heads < 0 || shape->q_heads > 4096 || shape->kv_heads > 4096)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d query and %d key-value heads are not within 0..4096", what,
                    shape->q_heads, shape->kv_heads);
    if (tokens < 0 || tokens > (int64_t(1) << 30))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %lld tokens are not within 0..2^30", what, (long long)tokens);
    return MFH_OK;
}

int launch(const mfh_rotary_shape& sh, RotaryArgs a, int cache, hipStream_t s)
{
    const Strides qs(sh.q_token_stride, sh.q_head_stride, sh.q_heads, sh.head_dim);
    const Strides qo(sh.q_out_token_stride, sh.q_out_head_stride, sh.q_heads, sh.head_dim);
    const Strides ks(sh.k_token_stride, sh.k_head_stride, sh.kv_heads, sh.head_dim);
    const Strides ko(sh.k_out_token_stride, sh.k_out_head_stride, sh.kv_heads, sh.head_dim);
    const Strides vs(sh.v_token_stride, sh.v_head_stride, sh.kv_heads, sh.head_dim);
    a.q_t = qs.token, a.q_h = qs.head, a.qo_t = qo.token, a.qo_h = qo.head, a.k_t = ks.token, a.k_h = ks.head;
    a.v_t = vs.token, a.v_h = vs.head;
    if (!a.slots) a.ko_t = ko.token, a.ko_h = ko.head;
    const mfh_u32 half = (mfh_u32)sh.rotary_dim / 2, rest = (mfh_u32)(sh.head_dim - sh.rotary_dim) / 2;
    // The widest piece that divides the pairs and what is copied behind them:
    // 16 bytes where both allow it.
    int e = sh.dtype == kFloat32 ? 4 : 8;
    while (half % e || rest % e) e >>= 1;
    a.half = half;
    a.units_per_head = (half + rest) / e;
    a.turned_units = half / e;
    a.q_units = a.q ? (mfh_u32)sh.q_heads * a.units_per_head : 0;
    a.k_units = a.q_units + (a.k ? (mfh_u32)sh.kv_heads * a.units_per_head : 0);
    a.units = a.k_units + (a.v ? (mfh_u32)sh.kv_heads * a.units_per_head : 0);
    if (a.units == 0) return MFH_OK;
    // One unit a thread, or one token where that is more: 62 us for 16381 tokens of
    // 32 + 8 + 8 heads of 128, bf16 into a cache of e4m3; with 2, 3 or 4 units in flight 66.
    int64_t per = std::max<int64_t>(1, kThreads / a.units);
    if (half) per = std::min<int64_t>(per, kMaxPairs / half);
    a.tokens_per_block = (int32_t)std::max<int64_t>(1, per);
    a.by_half = Divider(std::max<mfh_u32>(half, 1));
    a.by_units = Divider(a.units);
    a.by_head = Divider(a.units_per_head);
    a.factor = sh.factor;
    a.sine_factor = sh.inverse ? -sh.factor : sh.factor;
    const int64_t blocks = (a.tokens + a.tokens_per_block - 1) / a.tokens_per_block;
    const dim3 grid((unsigned)std::min<int64_t>(blocks, kMostBlocks), (unsigned)((blocks + kMostBlocks - 1) / kMostBlocks));
    const bool il = sh.interleaved != 0;
    switch (sh.dtype) {
    case kFloat32: launch_types<kFloat32, kFloat32>(e, il, grid, s, a); break;
    case kFloat16:
        if (cache == kF8E4M3) launch_types<kFloat16, kF8E4M3>(e, il, grid, s, a);
        else launch_types<kFloat16, kFloat16>(e, il, grid, s, a);
        break;
    default:
        if (cache == kF8E4M3) launch_types<kBFloat16, kF8E4M3>(e, il, grid, s, a);
        else launch_types<kBFloat16, kBFloat16>(e, il, grid, s, a);
        break;
    }
    return launch_status("k_rotary");
}

}  // namespace
}  // namespace mfh

using namespace mfh;

extern "C" {

int mfh_rotary_frequencies(double* out, int32_t rotary_dim, double base, int32_t scaling, double factor,
                           double original_length, double low, double high)
{
    const char* what = "mfh_rotary_frequencies";
    if (rotary_dim < 0 || rotary_dim % 2)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: rotary dim %d is not an even number", what, rotary_dim);
    if (rotary_dim > 0 && !out) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL buffer", what);
    if (!(base > 0.0) || !std::isfinite(base))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: base %g is not a positive number", what, base);
    if (scaling < MFH_ROTARY_PLAIN || scaling > MFH_ROTARY_BANDS)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: unknown scaling %d", what, scaling);
    if (scaling != MFH_ROTARY_PLAIN && (!(factor > 0.0) || !std::isfinite(factor)))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: factor %g is not a positive number", what, factor);
    if (scaling == MFH_ROTARY_BANDS && (!(original_length > 0.0) || !std::isfinite(original_length) || !(high > low)))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: bands %g..%g over a length of %g", what, low, high,
                    original_length);
    if (scaling == MFH_ROTARY_BASE && rotary_dim > 2)
        base *= std::pow(factor, (double)rotary_dim / (rotary_dim - 2));
    for (int32_t i = 0; i < rotary_dim / 2; i++) {
        double f = std::pow(base, -2.0 * i / rotary_dim);
        if (scaling == MFH_ROTARY_LINEAR) f /= factor;
        if (scaling == MFH_ROTARY_BANDS) {
            const double turns = original_length * f / 6.28318530717958647692;
            const double keep = std::min(1.0, std::max(0.0, (turns - low) / (high - low)));
            f *= keep + (1.0 - keep) / factor;
        }
        out[i] = f;
    }
    return MFH_OK;
}

int mfh_rotary(const mfh_rotary_shape* shape, int64_t tokens, const void* q, void* q_out, const void* k, void* k_out,
               const int32_t* positions, const double* frequencies, void* stream)
{
    const char* what = "mfh_rotary";
    const Device* dev;
    MFH_TRY(bind_device(&dev));
    MFH_TRY(check_shape(shape, tokens, what));
    if (tokens == 0) return MFH_OK;
    if (!positions || (shape->rotary_dim > 0 && !frequencies))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL positions or frequencies", what);
    if ((!q) != (!q_out) || (!k) != (!k_out))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: an input without its result, or a result without its input", what);
    RotaryArgs a{};
    a.q = q, a.q_out = q_out, a.k = k, a.k_out = k_out;
    a.positions = positions, a.frequencies = frequencies, a.tokens = tokens;
    a.by_page = Divider(1);
    return launch(*shape, a, shape->dtype, (hipStream_t)stream);
}

int mfh_rotary_append(const mfh_rotary_shape* shape, const mfh_kv_cache* cache, int64_t tokens, const void* q,
                      void* q_out, const void* k, const void* v, const int32_t* positions, const int64_t* slots,
                      const double* frequencies, void* k_cache, void* v_cache, void* stream)
{
    const char* what = "mfh_rotary_append";
    const Device* dev;
    MFH_TRY(bind_device(&dev));
    MFH_TRY(check_shape(shape, tokens, what));
    MFH_TRY(check_cache(cache, what));
    if (shape->kv_heads != cache->kv_heads || shape->head_dim != cache->head_dim)
        return fail(MFH_ERR_SHAPE_MISMATCH, "%s: %d heads of %d do not match the cache's %d of %d", what,
                    shape->kv_heads, shape->head_dim, cache->kv_heads, cache->head_dim);
    if (cache->dtype != shape->dtype && !(cache->dtype == kF8E4M3 && shape->dtype != kFloat32))
        return fail(MFH_ERR_DTYPE_UNSUPPORTED, "%s: dtype %s into a cache of %s", what, dtype_name(shape->dtype),
                    dtype_name(cache->dtype));
    if (shape->inverse)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: the inverse is a gradient's and has no place in a cache", what);
    if (tokens == 0) return MFH_OK;
    if (!positions || !slots || !k || !v || !k_cache || !v_cache || (shape->rotary_dim > 0 && !frequencies))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL buffer", what);
    if ((!q) != (!q_out))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: an input without its result, or a result without its input", what);
    RotaryArgs a{};
    a.q = q, a.q_out = q_out, a.k = k, a.k_out = k_cache, a.v = v, a.v_out = v_cache;
    a.positions = positions, a.slots = slots, a.frequencies = frequencies, a.tokens = tokens;
    a.ko_t = cache->token_stride, a.ko_h = cache->head_stride;
    a.page_stride = cache->page_stride;
    a.slot_count = cache->pages * cache->page_size;
    a.by_page = Divider((mfh_u32)cache->page_size);
    a.k_by = 1.0f / cache->k_scale, a.v_by = 1.0f / cache->v_scale;
    return launch(*shape, a, cache->dtype, (hipStream_t)stream);
}

}  // extern "C"
