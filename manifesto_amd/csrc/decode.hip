// decode.hip — attention of one new token per request over a paged cache
// (mfh_paged_decode), split over the context's length and joined.
//
// Each key and value is read once for the heads that share it: bytes bound it,
// 2 * length * kv_heads * head_dim of them, so everything serves to keep loads
// in flight.  A workgroup is four waves on one request, one key-value head
// (16 of its query heads at most) and one part of the context; the waves take
// tiles of 32 tokens in turn and meet in LDS only at the end, so none waits
// for another.
//
// In a wave nothing goes through LDS at all:
//   scores^T [tokens][heads] = K Q^T   two products of 16 tokens, K straight from
//                                      memory in the matrix operand's layout
//   out^T [dims][heads] += V^T P^T     32 tokens at once
// A lane holds the scores of head lane % 16 for the tokens 4 * (lane / 16) + i
// of both halves; taken in that order as the product's 32 steps they are its P^T
// operand as they stand.  V^T needs eight tokens of one dim per lane: a lane
// loads eight dims of its eight tokens (16 bytes each, whole rows across the
// lanes) and turns the 8 x 8 block in registers, one byte permute per dword.
//
// Softmax runs over the tiles with a running reference instead of the running
// maximum: it moves, and the sums are rescaled, only where a score passes it by
// 2^8.  Weights are at most 2^8 and the reference divides out; sums and
// products stay in f32, weights are rounded to the queries' 16 bits for the
// product with V alone, whose terms have that rounding already.
#include "paged.hpp"

namespace mfh {

int check_cache(const mfh_kv_cache* c, const char* what)
{
    if (!c) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL cache", what);
    const int dt = c->dtype;
    if (dt != kFloat16 && dt != kBFloat16 && dt != kF8E4M3)
        return fail(MFH_ERR_DTYPE_UNSUPPORTED, "%s: a cache of %s is not f16/bf16/f8e4m3", what, dtype_name(dt));
    if (c->page_size < 1) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: page size %d is not positive", what, c->page_size);
    if (c->kv_heads < 1 || c->kv_heads > 4096)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d key-value heads are not within 1..4096", what, c->kv_heads);
    const int step = dt == kF8E4M3 ? 16 : 8;
    if (c->head_dim < step || c->head_dim > 256 || c->head_dim % step)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: head dim %d is not a multiple of %d up to 256", what, c->head_dim, step);
    if (c->pages < 1 || c->pages > 0x7fffffff)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %lld pages are not within 1..2^31-1", what, (long long)c->pages);
    if (c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: negative stride", what);
    const __int128 span = ((__int128)(c->page_size - 1) * c->token_stride + (__int128)(c->kv_heads - 1) * c->head_stride +
                           c->head_dim) * (dt == kF8E4M3 ? 1 : 2);
    if (span >= ((__int128)1 << 31))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: a page spans 2 GiB or more", what);
    if ((__int128)(c->pages - 1) * c->page_stride >= ((__int128)1 << 61))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: the pages span too far", what);
    for (float s : {c->k_scale, c->v_scale}) {
        if (!__builtin_isnormal(s) || !__builtin_isnormal(1.0f / s))
            return fail(MFH_ERR_INVALID_ARGUMENT, "%s: scale %g has no reciprocal", what, (double)s);
        if (dt != kF8E4M3 && s != 1.0f)
            return fail(MFH_ERR_INVALID_ARGUMENT, "%s: scale %g of a cache that is not in 8 bits", what, (double)s);
    }
    return MFH_OK;
}

int check_attention(const mfh_attention_shape* sh, const mfh_kv_cache* c, const char* what)
{
    if (!sh) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL shape", what);
    MFH_TRY(check_cache(c, what));
    if (sh->dtype != kFloat16 && sh->dtype != kBFloat16)
        return fail(MFH_ERR_DTYPE_UNSUPPORTED, "%s: queries of %s are not f16/bf16", what, dtype_name(sh->dtype));
    if (c->dtype != sh->dtype && c->dtype != kF8E4M3)
        return fail(MFH_ERR_DTYPE_UNSUPPORTED, "%s: queries of %s over a cache of %s", what, dtype_name(sh->dtype),
                    dtype_name(c->dtype));
    if (sh->q_heads < 1 || sh->q_heads > (1 << 16) || sh->q_heads % c->kv_heads)
        return fail(MFH_ERR_SHAPE_MISMATCH, "%s: %d query heads do not share %d key-value heads evenly", what,
                    sh->q_heads, c->kv_heads);
    if (!__builtin_isfinite(sh->scale)) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: scale %g", what, (double)sh->scale);
    if (!(sh->softcap >= 0.0f) || (sh->softcap > 0.0f && !(__builtin_isnormal(sh->softcap) && __builtin_isnormal(1.0f / sh->softcap))))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: cap %g is not 0 or a positive number", what, (double)sh->softcap);
    if (sh->window < 0) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: window %d is negative", what, sh->window);
    return MFH_OK;
}

namespace {

constexpr int kTile = 32;    // tokens of a wave's step
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kHeads = 16;   // query heads of a workgroup
constexpr float kStep = 8.0f;  // the reference moves where a score passes it by 2^kStep

struct DecodeArgs {
    PageArgs pages;
    const char* q;
    char* out;
    float* lse;
    float* part_out;   // [requests * q_heads][parts][head_dim]
    float2* part_sum;  // [requests * q_heads][parts]: reference and sum
    const int32_t* lengths;
    const float* slopes;
    int64_t q_t, q_h, out_t, out_h;  // elements
    float scale, cap_twice, cap_scaled, v_scale;
    int32_t window, requests, kv_heads, q_heads, group, head_groups, dim;
    mfh_u32 parts, least;  // of a request; tiles of a part at least
    Divider by_parts, by_head_groups, by_kv_heads;
};

MFH_DEV mfh_u32 low_halves(mfh_u32 a, mfh_u32 b) { return __builtin_amdgcn_perm(b, a, 0x05040100); }
MFH_DEV mfh_u32 high_halves(mfh_u32 a, mfh_u32 b) { return __builtin_amdgcn_perm(b, a, 0x07060302); }

// The tokens of a request that its new token sees: [first, length).
struct Context {
    mfh_u32 length, first, tile0, tiles;
    __device__ Context(const DecodeArgs& a, mfh_u32 r)
    {
        const mfh_u64 most = min((mfh_u64)a.pages.width * a.pages.by_page.d, (mfh_u64)kLongest);
        length = min((mfh_u32)max(a.lengths[r], 0), (mfh_u32)most);
        first = a.window > 0 && length > (mfh_u32)a.window ? length - a.window : 0;
        tile0 = first / kTile;
        tiles = length > first ? (length + kTile - 1) / kTile - tile0 : 0;
    }
};

// Where a tile's 32 tokens stand.  Where a page holds whole groups of 16 tokens
// (FAST) the two halves have a uniform offset each and the lanes' own offsets
// never change; else lane i % 32 looks token i up and the others ask for it.
template <bool FAST>
struct TileAt {
    int64_t half[2];
    int64_t mine;
    mfh_u32 valid;  // bit i: token i is seen and has a page
};

MFH_DEV int64_t uniform64(int64_t v)
{
    const mfh_u32 lo = __builtin_amdgcn_readfirstlane((int)(mfh_u32)v);
    const mfh_u32 hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
    return (int64_t)((mfh_u64)hi << 32 | lo);
}

MFH_DEV int64_t shuffle64(int64_t v, int lane)
{
    const mfh_u32 lo = __shfl((int)(mfh_u32)v, lane), hi = __shfl((int)(v >> 32), lane);
    return (int64_t)((mfh_u64)hi << 32 | lo);
}

template <bool FAST>
MFH_DEV TileAt<FAST> locate(const PageArgs& p, const int32_t* table, const Context& c, mfh_u32 t0, int lane)
{
    TileAt<FAST> at;
    if constexpr (FAST) {
        at.valid = 0;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const mfh_u32 t = t0 + 16 * h;
            const mfh_u32 row = p.by_page.quotient(t), in_page = t - row * p.by_page.d;
            const int32_t page = __builtin_amdgcn_readfirstlane(t < c.length ? table[row] : -1);
            const bool ok = page >= 0 && page < p.pages;
            at.half[h] = (ok ? page : 0) * p.page_bytes + in_page * p.token_bytes;
            if (ok) {
                const mfh_u32 below = c.length - t;  // > 0
                mfh_u32 bits = below >= 16 ? 0xffffu : (1u << below) - 1;
                if (c.first > t) bits &= c.first - t >= 16 ? 0 : 0xffffu << (c.first - t);
                at.valid |= (bits & 0xffffu) << (16 * h);
            }
        }
    } else {
        const mfh_u32 t = t0 + (lane & 31);
        const mfh_u32 row = p.by_page.quotient(t), in_page = t - row * p.by_page.d;
        const bool seen = t < c.length && t >= c.first;
        const int32_t page = seen ? table[row] : -1;
        const bool ok = page >= 0 && page < p.pages;
        at.mine = (ok ? page : 0) * p.page_bytes + (ok ? in_page : 0) * p.token_bytes;
        at.valid = (mfh_u32)__ballot(ok);
    }
    return at;
}

template <int DT, bool FP8>
MFH_DEV u32x4 load_eight(const char* p)
{
    if constexpr (FP8) {
        const u32x2 w = load8<true>(p);
        return u32x4{e4m3_pair<DT, false>(w[0]), e4m3_pair<DT, true>(w[0]), e4m3_pair<DT, false>(w[1]),
                     e4m3_pair<DT, true>(w[1])};
    } else {
        return load16<true>(p);
    }
}

// DP: head_dim rounded up to 64, 128 or 256.
template <int DT, bool FP8, int DP, bool FAST>
__global__ __launch_bounds__(kThreads) void k_decode(DecodeArgs a)
{
    constexpr int kSteps = DP / 32;               // of the product with K
    constexpr int kSets = DP == 64 ? 1 : DP / 128;  // of 16 lanes' dims in V
    constexpr int kDims = DP == 64 ? 4 : 8;       // of a lane in a set
    constexpr int kBytes = FP8 ? 1 : 2;
    constexpr int kSetDims = 16 * kDims;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    mfh_u32 at = blockIdx.x;
    mfh_u32 rest = a.by_parts.quotient(at);
    const mfh_u32 part = at - rest * a.parts;
    at = rest;
    rest = a.by_head_groups.quotient(at);
    const mfh_u32 head_group = at - rest * a.head_groups;
    const mfh_u32 r = a.by_kv_heads.quotient(rest), kv = rest - r * a.kv_heads;

    const Context c(a, r);
    const mfh_u32 size = part_tiles(c.tiles, a.least, a.parts);
    const mfh_u32 used = max(1u, (c.tiles + size - 1) / size);
    if (part >= used) return;
    const mfh_u32 begin = c.tile0 + part * size, end = min(begin + size, c.tile0 + c.tiles);

    const int heads = min(kHeads, a.group - (int)head_group * kHeads);
    const int head0 = kv * a.group + head_group * kHeads;
    const int32_t* table = a.pages.table + (int64_t)r * a.pages.table_stride;
    const char* k_base = a.pages.k + kv * a.pages.head_bytes;
    const char* v_base = a.pages.v + kv * a.pages.head_bytes;
    const mfh_u32 token_bytes = (mfh_u32)a.pages.token_bytes;

    // Q^T: head `col`, dims 32 s + 8 quad ..
    u32x4 q[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; s++) {
        const int d = 32 * s + 8 * quad;
        q[s] = u32x4{0, 0, 0, 0};
        if (col < heads && d < a.dim)
            q[s] = load16<false>(a.q + ((int64_t)r * a.q_t + (int64_t)(head0 + col) * a.q_h + d) * 2);
    }
    const float slope = a.slopes && col < heads ? a.slopes[head0 + col] * kLog2e : 0.0f;

    f32x4 acc[kSets][kDims];
#pragma unroll
    for (int u = 0; u < kSets; u++)
#pragma unroll
        for (int d = 0; d < kDims; d++) acc[u][d] = f32x4{0, 0, 0, 0};
    float ref = 0.0f, limit = -INFINITY, sum = 0.0f;

    // Lanes past head_dim read its last dims again, inside the row: their
    // steps have zeros in Q (and, below, in K), their results are not written.
    mfh_u32 k_lane[kSteps], v_lane[kSets];
#pragma unroll
    for (int s = 0; s < kSteps; s++)
        k_lane[s] = (FAST ? col * token_bytes : 0) + min(32 * s + 8 * quad, a.dim - 8) * kBytes;
#pragma unroll
    for (int u = 0; u < kSets; u++)
        v_lane[u] = (FAST ? 4 * quad * token_bytes : 0) + min(u * kSetDims + kDims * col, a.dim - kDims) * kBytes;
    const bool ragged = a.dim != DP;

    u32x4 k[2][kSteps];
    auto load_k = [&](const TileAt<FAST>& w) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const char* row;
            if constexpr (FAST) row = k_base + w.half[h];
            else row = k_base + shuffle64(w.mine, 16 * h + col);
#pragma unroll
            for (int s = 0; s < kSteps; s++) k[h][s] = load_eight<DT, FP8>(row + k_lane[s]);
        }
    };

    mfh_u32 tile = begin + wave;
    TileAt<FAST> now, next;
    if (tile < end) {
        now = locate<FAST>(a.pages, table, c, tile * kTile, lane);
        load_k(now);
    }
    for (; tile < end; tile += kWaves) {
        const bool more = tile + kWaves < end;
        u32x4 v[kSets][8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const char* row;
            if constexpr (FAST) row = v_base + (now.half[j >> 2] + (j & 3) * (int64_t)token_bytes);
            else row = v_base + shuffle64(now.mine, 16 * (j >> 2) + 4 * quad + (j & 3));
#pragma unroll
            for (int u = 0; u < kSets; u++) {
                if constexpr (kDims == 8) {
                    v[u][j] = load_eight<DT, FP8>(row + v_lane[u]);
                } else if constexpr (FP8) {
                    const mfh_u32 w = load4(row + v_lane[u]);
                    v[u][j] = u32x4{e4m3_pair<DT, false>(w), e4m3_pair<DT, true>(w), 0, 0};
                } else {
                    const u32x2 w = load8<true>(row + v_lane[u]);
                    v[u][j] = u32x4{w[0], w[1], 0, 0};
                }
            }
        }
        if (ragged) {
#pragma unroll
            for (int s = 0; s < kSteps; s++)
                if (32 * s + 8 * quad >= a.dim) k[0][s] = k[1][s] = u32x4{0, 0, 0, 0};
        }
        f32x4 s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < kSteps; s++) {
            s0 = mfma16<DT>(k[0][s], q[s], s0);
            s1 = mfma16<DT>(k[1][s], q[s], s1);
        }
        if (more) {
            next = locate<FAST>(a.pages, table, c, (tile + kWaves) * kTile, lane);
            load_k(next);
        }

        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = (j < 4 ? s0[j & 3] : s1[j & 3]) * a.scale;
        if (a.cap_scaled != 0.0f) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = capped(x[j], a.cap_twice, a.cap_scaled);
        }
        if (a.slopes) {
            const int back = (int)(c.length - 1) - (int)(tile * kTile + 4 * quad);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] -= slope * (float)(back - (16 * (j >> 2) + (j & 3)));
        }
        if (now.valid != 0xffffffffu) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (!(now.valid >> (16 * (j >> 2) + 4 * quad + (j & 3)) & 1)) {
                    x[j] = -INFINITY;
#pragma unroll
                    for (int u = 0; u < kSets; u++) v[u][j] = u32x4{0, 0, 0, 0};  // 0 * NaN would be NaN
                }
            }
        }
        float top = x[0];
#pragma unroll
        for (int j = 1; j < 8; j++) top = fmaxf(top, x[j]);
        if (__any(top > limit)) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            if (top > limit) {
                const float alpha = limit == -INFINITY ? 0.0f : exp2_fast(ref - top);
                ref = top;
                limit = top + kStep;
                sum *= alpha;
#pragma unroll
                for (int u = 0; u < kSets; u++)
#pragma unroll
                    for (int d = 0; d < kDims; d++) acc[u][d] *= alpha;
            }
        }
        u32x4 p;
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = exp2_fast(x[j] - ref);
#pragma unroll
        for (int j = 0; j < 4; j++) p[j] = enc16x2<DT>(x[2 * j], x[2 * j + 1]);
        sum += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
#pragma unroll
        for (int u = 0; u < kSets; u++) {
#pragma unroll
            for (int d = 0; d < kDims; d += 2) {
                const int w = d / 2;
                const u32x4 even = {low_halves(v[u][0][w], v[u][1][w]), low_halves(v[u][2][w], v[u][3][w]),
                                    low_halves(v[u][4][w], v[u][5][w]), low_halves(v[u][6][w], v[u][7][w])};
                const u32x4 odd = {high_halves(v[u][0][w], v[u][1][w]), high_halves(v[u][2][w], v[u][3][w]),
                                   high_halves(v[u][4][w], v[u][5][w]), high_halves(v[u][6][w], v[u][7][w])};
                acc[u][d] = mfma16<DT>(even, p, acc[u][d]);
                acc[u][d + 1] = mfma16<DT>(odd, p, acc[u][d + 1]);
            }
        }
        now = next;
    }

    // The waves' results meet: a common reference, then sums weighted by it.
    __shared__ float s_ref[kWaves][kHeads], s_sum[kWaves][kHeads];
    __shared__ float s_out[kWaves][kHeads][kSetDims + 4];
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (quad == 0) {
        s_ref[wave][col] = limit == -INFINITY ? -INFINITY : ref;
        s_sum[wave][col] = sum;
    }
    for (int u = 0; u < kSets; u++) {
        if (u) __syncthreads();
#pragma unroll
        for (int uu = 0; uu < kSets; uu++) {
            if (uu != u) continue;
#pragma unroll
            for (int d = 0; d < kDims; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) s_out[wave][col][kDims * (4 * quad + i) + d] = acc[uu][d][i];
        }
        __syncthreads();
        const int pairs = min(kSetDims, a.dim - u * kSetDims) / 2;
        for (int i = threadIdx.x; i < heads * (kSetDims / 2); i += kThreads) {
            const int h = i / (kSetDims / 2), d = 2 * (i % (kSetDims / 2));
            if (d >= 2 * pairs) continue;
            float top = s_ref[0][h];
#pragma unroll
            for (int w = 1; w < kWaves; w++) top = fmaxf(top, s_ref[w][h]);
            float total = 0.0f, o0 = 0.0f, o1 = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                const float f = s_ref[w][h] == -INFINITY ? 0.0f : exp2_fast(s_ref[w][h] - top);
                total += f * s_sum[w][h];
                o0 += f * s_out[w][h][d];
                o1 += f * s_out[w][h][d + 1];
            }
            const int64_t row = (int64_t)r * a.q_heads + head0 + h;
            const int dim = u * kSetDims + d;
            if (used > 1) {
                const int64_t slot = row * a.parts + part;
                float2* o = reinterpret_cast<float2*>(a.part_out + slot * a.dim + dim);
                *o = make_float2(o0, o1);
                if (dim == 0) a.part_sum[slot] = make_float2(top, total);
            } else {
                const float f = total == 0.0f ? 0.0f : a.v_scale / total;
                store4(a.out + ((int64_t)r * a.out_t + (int64_t)(head0 + h) * a.out_h + dim) * 2, enc16x2<DT>(o0 * f, o1 * f));
                if (dim == 0 && a.lse) a.lse[row] = total == 0.0f ? -INFINITY : top * kLn2 + logf(total);
            }
        }
    }
}

// Joins a request's parts, one wave per query head; lane l takes the dims
// 2 l + 128 u.
template <int DT>
__global__ __launch_bounds__(64) void k_decode_join(DecodeArgs a)
{
    const mfh_u32 r = blockIdx.x / a.q_heads, h = blockIdx.x - r * a.q_heads;
    const Context c(a, r);
    const mfh_u32 size = part_tiles(c.tiles, a.least, a.parts);
    const mfh_u32 used = (c.tiles + size - 1) / size;
    if (used <= 1) return;
    const int lane = threadIdx.x;
    const int64_t row = (int64_t)r * a.q_heads + h;
    const float2* sums = a.part_sum + row * a.parts;
    float top = -INFINITY;
    for (mfh_u32 i = lane; i < used; i += 64) top = fmaxf(top, sums[i].x);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    float total = 0.0f, o[4] = {0, 0, 0, 0};
    for (mfh_u32 i = 0; i < used; i++) {
        const float2 s = sums[i];
        const float f = s.x == -INFINITY ? 0.0f : exp2_fast(s.x - top);
        total += f * s.y;
        const float* from = a.part_out + (row * a.parts + i) * a.dim;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int d = 128 * u + 2 * lane;
            if (d < a.dim) {
                const float2 w = *reinterpret_cast<const float2*>(from + d);
                o[2 * u] += f * w.x;
                o[2 * u + 1] += f * w.y;
            }
        }
    }
    const float f = total == 0.0f ? 0.0f : a.v_scale / total;
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const int d = 128 * u + 2 * lane;
        if (d < a.dim)
            store4(a.out + ((int64_t)r * a.out_t + (int64_t)h * a.out_h + d) * 2, enc16x2<DT>(o[2 * u] * f, o[2 * u + 1] * f));
    }
    if (lane == 0 && a.lse) a.lse[row] = total == 0.0f ? -INFINITY : top * kLn2 + logf(total);
}

template <int DT, bool FP8, int DP>
void launch_pages(bool fast, unsigned grid, hipStream_t s, const DecodeArgs& a)
{
    if (fast) k_decode<DT, FP8, DP, true><<<grid, kThreads, 0, s>>>(a);
    else k_decode<DT, FP8, DP, false><<<grid, kThreads, 0, s>>>(a);
}

template <int DT, bool FP8>
void launch_dims(int dim, bool fast, unsigned grid, hipStream_t s, const DecodeArgs& a)
{
    if (dim <= 64) launch_pages<DT, FP8, 64>(fast, grid, s, a);
    else if (dim <= 128) launch_pages<DT, FP8, 128>(fast, grid, s, a);
    else launch_pages<DT, FP8, 256>(fast, grid, s, a);
}

// Parts of a request and tiles of a part at least.  The parts fill the card
// four workgroups deep; below 128 tokens (a tile a wave) a part is not worth
// its workgroup.
constexpr int kDeep = 4;
constexpr mfh_u32 kLeast = kWaves;

void split(const Device* dev, int64_t rows, int64_t longest, mfh_u32* parts, mfh_u32* least)
{
    const int64_t tiles = std::min<int64_t>((std::max<int64_t>(longest, 1) + kTile - 1) / kTile, kLongest / kTile);
    const int64_t wanted = std::max<int64_t>(1, (int64_t)dev->compute_units * kDeep / std::max<int64_t>(rows, 1));
    const int64_t most = std::max<int64_t>(1, (tiles + kLeast - 1) / kLeast);
    const int64_t n = std::min(wanted, most);
    const int64_t size = ((tiles + n - 1) / n + kWaves - 1) / kWaves * kWaves;
    *least = (mfh_u32)size;
    *parts = (mfh_u32)((tiles + size - 1) / size);
}

size_t part_bytes(int64_t rows, mfh_u32 parts, int dim)
{
    return parts > 1 ? (size_t)rows * parts * (dim + 2) * sizeof(float) : 0;
}

}  // namespace
}  // namespace mfh

using namespace mfh;

extern "C" {

int mfh_paged_decode_workspace(const mfh_attention_shape* shape, const mfh_kv_cache* cache, int32_t requests,
                               int64_t longest, size_t* bytes)
{
    const char* what = "mfh_paged_decode_workspace";
    const Device* dev;
    MFH_TRY(bind_device(&dev));
    MFH_TRY(check_attention(shape, cache, what));
    if (requests < 0) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: negative number of requests %d", what, requests);
    if (!bytes) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL result", what);
    const int group = shape->q_heads / cache->kv_heads;
    mfh_u32 parts, least;
    split(dev, (int64_t)requests * cache->kv_heads * ((group + kHeads - 1) / kHeads), longest, &parts, &least);
    *bytes = part_bytes((int64_t)requests * shape->q_heads, parts, cache->head_dim);
    return MFH_OK;
}

int mfh_paged_decode(const mfh_attention_shape* shape, const mfh_kv_cache* cache, int32_t requests, const void* q,
                     const void* k_cache, const void* v_cache, const int32_t* table, int64_t table_stride,
                     int32_t table_width, const int32_t* lengths, int64_t longest, const float* slopes, void* out,
                     float* lse, void* workspace, size_t workspace_bytes, void* stream)
{
    const char* what = "mfh_paged_decode";
    const Device* dev;
    MFH_TRY(bind_device(&dev));
    MFH_TRY(check_attention(shape, cache, what));
    if (requests < 0) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: negative number of requests %d", what, requests);
    if (table_width < 0 || table_stride < table_width)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: table width %d does not fit its stride %lld", what, table_width,
                    (long long)table_stride);
    if (requests == 0) return MFH_OK;
    if (!q || !out || !k_cache || !v_cache || !lengths || (table_width > 0 && !table))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL buffer", what);
    if (workspace_bytes > 0 && (!workspace || (uintptr_t)workspace % 16))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: the workspace is NULL or not 16-byte aligned", what);
    const int bytes = cache->dtype == kF8E4M3 ? 1 : 2;
    DecodeArgs a{};
    a.pages = PageArgs{(const char*)k_cache, (const char*)v_cache, table, table_stride, cache->page_stride * bytes,
                       cache->token_stride * bytes, cache->head_stride * bytes, cache->pages,
                       Divider((mfh_u32)cache->page_size), (mfh_u32)table_width};
    a.q = (const char*)q, a.out = (char*)out, a.lse = lse;
    a.lengths = lengths, a.slopes = slopes;
    const Strides qs(shape->q_token_stride, shape->q_head_stride, shape->q_heads, cache->head_dim);
    const Strides os(shape->out_token_stride, shape->out_head_stride, shape->q_heads, cache->head_dim);
    a.q_t = qs.token, a.q_h = qs.head, a.out_t = os.token, a.out_h = os.head;
    a.scale = shape->scale * cache->k_scale;
    if (shape->softcap > 0.0f) {
        a.cap_twice = 2.0f * kLog2e / shape->softcap;
        a.cap_scaled = shape->softcap * kLog2e;
    } else {
        a.scale *= kLog2e;
    }
    a.v_scale = cache->v_scale;
    a.window = shape->window, a.requests = requests, a.kv_heads = cache->kv_heads, a.q_heads = shape->q_heads;
    a.group = shape->q_heads / cache->kv_heads;
    a.head_groups = (a.group + kHeads - 1) / kHeads;
    a.dim = cache->head_dim;
    const int64_t rows = (int64_t)requests * cache->kv_heads * a.head_groups;
    split(dev, rows, std::min<int64_t>(longest, (int64_t)table_width * cache->page_size), &a.parts, &a.least);
    const int64_t heads = (int64_t)requests * shape->q_heads;
    while (a.parts > 1 && part_bytes(heads, a.parts, a.dim) > workspace_bytes) {
        a.least *= 2;
        a.parts = (a.parts + 1) / 2;
    }
    const int64_t grid = rows * a.parts;
    if (grid >= (int64_t(1) << 32) / kThreads || heads >= 0x7fffffff)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d requests of %d heads are too many for one call", what, requests,
                    shape->q_heads);
    if (a.parts > 1) {
        a.part_out = (float*)workspace;
        a.part_sum = (float2*)(a.part_out + heads * a.parts * a.dim);
    }
    a.by_parts = Divider(a.parts), a.by_head_groups = Divider((mfh_u32)a.head_groups), a.by_kv_heads = Divider((mfh_u32)a.kv_heads);
    hipStream_t s = (hipStream_t)stream;
    const bool fast = cache->page_size % 16 == 0, fp8 = cache->dtype == kF8E4M3;
    if (shape->dtype == kBFloat16) {
        if (fp8) launch_dims<kBFloat16, true>(a.dim, fast, (unsigned)grid, s, a);
        else launch_dims<kBFloat16, false>(a.dim, fast, (unsigned)grid, s, a);
    } else {
        if (fp8) launch_dims<kFloat16, true>(a.dim, fast, (unsigned)grid, s, a);
        else launch_dims<kFloat16, false>(a.dim, fast, (unsigned)grid, s, a);
    }
    MFH_TRY(launch_status("k_decode"));
    if (a.parts > 1) {
        if (shape->dtype == kBFloat16) k_decode_join<kBFloat16><<<(unsigned)heads, 64, 0, s>>>(a);
        else k_decode_join<kFloat16><<<(unsigned)heads, 64, 0, s>>>(a);
        MFH_TRY(launch_status("k_decode_join"));
    }
    return MFH_OK;
}

}  // extern "C"
