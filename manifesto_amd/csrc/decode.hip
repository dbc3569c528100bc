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
// maximum: it moves, and the sums are rescaled, only where a score passes the last
// move's largest by 2^8 (kBelow in paged.hpp says where it stands); it divides out.
// Sums and products stay in f32.  The matrix units multiply 16-bit numbers, so
// weights are rounded to the queries' type for the product with V; their sum is
// that of the unrounded ones.
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

enum Cap { kNone, kNarrow, kWide };

// A row is a request's key-value head with up to 16 of its query heads.
struct DecodeArgs {
    PageArgs pages;
    const char* q;
    char* out;
    float* lse;
    float* part_out;     // [slots][part_heads][head_dim]
    float2* part_sum;    // [slots][part_heads]: reference and sum
    const int32_t* lengths;
    const float* slopes;
    int64_t q_t, q_h, out_t, out_h;  // elements
    float scale, cap_scaled, cap_factor, v_scale;  // cap_factor: `twice` of a cap, `scaled_inverse` of a wide one
    int cap;
    int32_t window, requests, kv_heads, q_heads, group, head_groups, dim, part_heads;
    mfh_u32 request_rows;  // kv_heads * head_groups
    mfh_u32 blocks, uneven;  // of the split form, where requests are alike and where not
    Divider by_head_groups, by_request_rows, by_blocks, by_uneven, by_q_heads;
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

// The split form: all rows' tiles go to `blocks` (or `uneven`) workgroups, a piece each; a
// row's pieces are its own, of equal size, so that there are `rows` workgroups
// more at most.  Short rows end early and make room for the next workgroup.
// The host takes this form only where the number of all tiles fits 31 bits.
MFH_DEV mfh_u32 lane_tiles(const DecodeArgs& a, mfh_u32 r) { return r < (mfh_u32)a.requests ? Context(a, r).tiles : 0; }

MFH_DEV mfh_u32 piece_of(const DecodeArgs& a, int lane)
{
    mfh_u32 sum = 0, most = 0;
    for (mfh_u32 base = 0; base < (mfh_u32)a.requests; base += 64) {
        const mfh_u32 tiles = lane_tiles(a, base + lane);
        sum += tiles, most = max(most, tiles);
    }
    const mfh_u32 all = last_lane(lanes_upto(sum)), total = all * a.request_rows;
    const bool uneven = __any((mfh_u64)most * (mfh_u32)a.requests * 4 > (mfh_u64)all * 5);
    const mfh_u32 piece = uneven ? a.by_uneven.quotient(total + a.uneven - 1) : a.by_blocks.quotient(total + a.blocks - 1);
    return max(piece, (mfh_u32)kWaves);
}

MFH_DEV mfh_u32 parts_of(mfh_u32 tiles, mfh_u32 piece) { return (tiles + piece - 1) / piece; }

// Where a tile's 32 tokens stand.  Where a page holds whole groups of 16 tokens
// (FAST) the two halves have a uniform offset each and the lanes' own offsets
// never change; else lane i % 32 looks token i up and the others ask for it.
// The table is read a tile before its pages are.
template <bool FAST>
struct TileAt {
    mfh_i64 page[2];    // FAST: of each half, its page
    mfh_u32 in_page[2]; // and its first row there, in bytes
    mfh_i64 mine;
    mfh_u32 valid;  // bit i: token i is seen and has a page
};

// Bit i: whether first + i is in [from, to), for 16 i.
MFH_DEV mfh_u32 range_bits(mfh_u32 first, mfh_u32 from, mfh_u32 to)
{
    const mfh_u32 low = from > first ? min(from - first, 16u) : 0, high = to > first ? min(to - first, 16u) : 0;
    return (1u << high) - 1 & ~((1u << low) - 1);
}

template <bool FAST>
struct Pages {
    int32_t page[2];
    __device__ void ask(const PageArgs& p, const int32_t* table, const Context& c, mfh_u32 t0, int lane)
    {
        // past the length its last page again
#pragma unroll
        for (int h = 0; h < (FAST ? 2 : 1); h++)
            page[h] = table[p.by_page.quotient(min(t0 + (FAST ? 16 * h : lane & 31), c.length - 1))];
    }
    // `real`: the tile is one of the wave's; else nothing of it is valid.
    __device__ TileAt<FAST> place(const PageArgs& p, const Context& c, mfh_u32 t0, int lane, bool real) const
    {
        TileAt<FAST> at;
        if constexpr (FAST) {
            at.valid = 0;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const mfh_u32 t = t0 + 16 * h;
                const mfh_u32 n = uniform((mfh_u32)page[h]);
                const bool ok = real && t < c.length && n < p.pages;
                at.page[h] = ok ? (mfh_i64)n : -1;
                at.in_page[h] = (t - p.by_page.quotient(t) * p.by_page.d) * p.token_bytes;
                if (ok) at.valid |= range_bits(t, c.first, c.length) << (16 * h);
            }
        } else {
            const mfh_u32 t = t0 + (lane & 31);
            const bool ok = real && t < c.length && t >= c.first && (mfh_u32)page[0] < p.pages;
            at.mine = ok ? (mfh_u32)page[0] * p.page_bytes + (t - p.by_page.quotient(t) * p.by_page.d) * p.token_bytes : 0;
            at.valid = (mfh_u32)__ballot(ok);
        }
        return at;
    }
};

// A page's rows of one head as a buffer; without a page one that has no bytes,
// from which loads give zeros and move nothing.
MFH_DEV __amdgpu_buffer_rsrc_t page_buffer(const char* base, mfh_i64 page, const PageArgs& p)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base + max(page, (mfh_i64)0) * p.page_bytes), 0,
                                             page < 0 ? 0 : (int)p.page_span, 0x00020000);
}

constexpr int kStreamed = 2;  // nt: keys and values are read once

template <typename T>
MFH_DEV T buffer_piece(__amdgpu_buffer_rsrc_t r, mfh_u32 lane_at, mfh_u32 at)
{
    if constexpr (sizeof(T) == 16) return __builtin_amdgcn_raw_buffer_load_b128(r, (int)lane_at, (int)at, kStreamed);
    else if constexpr (sizeof(T) == 8) return __builtin_amdgcn_raw_buffer_load_b64(r, (int)lane_at, (int)at, kStreamed);
    else return __builtin_amdgcn_raw_buffer_load_b32(r, (int)lane_at, (int)at, kStreamed);
}

// Eight codes as 16-bit values.
template <int DT>
MFH_DEV u32x4 widen(mfh_u32 lo, mfh_u32 hi)
{
    return u32x4{e4m3_pair<DT, false>(lo), e4m3_pair<DT, true>(lo), e4m3_pair<DT, false>(hi), e4m3_pair<DT, true>(hi)};
}

// What a lane loads of a token of V: 8 dims (4 where head_dim is at most 64).
template <bool FP8, int DIMS> struct Piece { typedef u32x4 type; };
template <> struct Piece<false, 4> { typedef u32x2 type; };
template <> struct Piece<true, 8> { typedef u32x2 type; };
template <> struct Piece<true, 4> { typedef mfh_u32 type; };

template <typename T>
MFH_DEV T load_piece(const char* p)
{
    if constexpr (sizeof(T) == 16) return load16<true>(p);
    else if constexpr (sizeof(T) == 8) return load8<true>(p);
    else return load4(p);
}

template <int DT, bool FP8, int DIMS>
MFH_DEV u32x4 dims_of(typename Piece<FP8, DIMS>::type w)
{
    if constexpr (!FP8 && DIMS == 8) return w;
    else if constexpr (!FP8) return u32x4{w[0], w[1], 0, 0};
    else if constexpr (DIMS == 8) return widen<DT>(w[0], w[1]);
    else return u32x4{e4m3_pair<DT, false>(w), e4m3_pair<DT, true>(w), 0, 0};
}

// DP: head_dim rounded up to 64, 128 or 256.  SPLIT: the line of all tiles in
// equal pieces, joined by k_decode_join; else a workgroup takes one row.
template <int DT, bool FP8, int DP, bool FAST, bool SPLIT>
__global__ __launch_bounds__(kThreads, DP == 64 ? 3 : DP == 128 ? 2 : 1) void k_decode(DecodeArgs a)
{
    constexpr int kSteps = DP / 32;                 // of the product with K
    constexpr int kLoads = FP8 ? kSteps / 2 : kSteps;  // of 16 bytes of a token of K
    constexpr int kSets = DP == 64 ? 1 : DP / 128;  // of 16 lanes' dims in V
    constexpr int kDims = DP == 64 ? 4 : 8;         // of a lane in a set
    constexpr int kBytes = FP8 ? 1 : 2;
    constexpr int kSetDims = 16 * kDims;
    typedef typename Piece<FP8, kDims>::type VPiece;

    __shared__ float s_ref[kWaves][kHeads], s_sum[kWaves][kHeads];
    __shared__ float s_out[kWaves][kHeads][kSetDims + 4];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;

    // This workgroup's row and its tiles.  Every wave finds them by itself.
    mfh_u32 r, row_of, part = 0, parts = 1;
    if constexpr (!SPLIT) {
        r = a.by_request_rows.quotient(blockIdx.x);
        row_of = blockIdx.x - r * a.request_rows;
    } else {
        const mfh_u32 piece = piece_of(a, lane);
        mfh_u32 before = 0;
        r = ~0u, row_of = 0;
        for (mfh_u32 base = 0; base < (mfh_u32)a.requests; base += 64) {
            const mfh_u32 its = parts_of(lane_tiles(a, base + lane), piece), upto = before + lanes_upto(its);
            const mfh_u64 past = __ballot(upto * a.request_rows > blockIdx.x);
            if (past) {  // the first request whose workgroups end past this one
                const int at = __ffsll((unsigned long long)past) - 1;
                parts = (mfh_u32)__builtin_amdgcn_readlane((int)its, at);
                const mfh_u32 in_request = blockIdx.x - ((mfh_u32)__builtin_amdgcn_readlane((int)upto, at) - parts) * a.request_rows;
                r = base + at;
                row_of = in_request / parts;
                part = in_request - row_of * parts;
                break;
            }
            before = last_lane(upto);
        }
        if (r == ~0u) return;
        // known to be uniform, the tables are read as scalars: their loads and
        // those of the pages are then not waited for together
        r = uniform(r), row_of = uniform(row_of), part = uniform(part), parts = uniform(parts);
    }
    const Context c(a, r);
    const mfh_u32 share = uniform((c.tiles + parts - 1) / parts);
    const mfh_u32 begin = c.tile0 + min(part * share, c.tiles), end = c.tile0 + min((part + 1) * share, c.tiles);

    const mfh_u32 token_bytes = a.pages.token_bytes;
    // Lanes past head_dim read its last dims again, inside the row: their
    // steps have zeros in Q (and, below, in K), their results are not written.
    // A step of K takes eight dims of each quad; an 8-bit load holds two steps'.
    auto dim_of = [&](int s) { return FP8 ? 64 * (s / 2) + 16 * quad + 8 * (s & 1) : 32 * s + 8 * quad; };
    mfh_u32 k_lane[kLoads], v_lane[kSets];
#pragma unroll
    for (int s = 0; s < kLoads; s++)
        k_lane[s] = (FAST ? col * token_bytes : 0) + (FP8 ? min(64 * s + 16 * quad, a.dim - 16) : min(32 * s + 8 * quad, a.dim - 8) * 2);
#pragma unroll
    for (int u = 0; u < kSets; u++)
        v_lane[u] = (FAST ? 4 * quad * token_bytes : 0) + min(u * kSetDims + kDims * col, a.dim - kDims) * kBytes;
    const bool ragged = a.dim != DP;

    const mfh_u32 head_group = row_of % a.head_groups, kv = a.by_head_groups.quotient(row_of);
    const int heads = min(kHeads, a.group - (int)head_group * kHeads);
    const int head0 = kv * a.group + head_group * kHeads;
    const int32_t* table = a.pages.table + (int64_t)r * a.pages.table_stride;
    const char* k_base = a.pages.k + kv * a.pages.head_bytes;
    const char* v_base = a.pages.v + kv * a.pages.head_bytes;

    Pages<FAST> pages;
    auto load = [&](u32x4 (&k)[2][kLoads], VPiece (&v)[kSets][8], mfh_u32& valid, mfh_u32 tile) {
        const TileAt<FAST> at = pages.place(a.pages, c, tile * kTile, lane, tile < end);
        valid = at.valid;
        if constexpr (FAST) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const __amdgpu_buffer_rsrc_t rows = page_buffer(k_base, at.page[h], a.pages);
#pragma unroll
                for (int s = 0; s < kLoads; s++) k[h][s] = buffer_piece<u32x4>(rows, k_lane[s], at.in_page[h]);
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const __amdgpu_buffer_rsrc_t rows = page_buffer(v_base, at.page[h], a.pages);
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int u = 0; u < kSets; u++)
                        v[u][4 * h + j] = buffer_piece<VPiece>(rows, v_lane[u], at.in_page[h] + j * token_bytes);
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const char* row = k_base + shuffle64(at.mine, 16 * h + col);
#pragma unroll
                for (int s = 0; s < kLoads; s++) k[h][s] = load16<true>(row + k_lane[s]);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const char* row = v_base + shuffle64(at.mine, 16 * (j >> 2) + 4 * quad + (j & 3));
#pragma unroll
                for (int u = 0; u < kSets; u++) v[u][j] = load_piece<VPiece>(row + v_lane[u]);
            }
        }
    };
    mfh_u32 tile = begin + wave;
    // Two tiles' registers: one is on its way while the other is computed.
    u32x4 k_a[2][kLoads], k_b[2][kLoads];
    VPiece v_a[kSets][8], v_b[kSets][8];
    mfh_u32 valid_a = 0, valid_b = 0;
    if (tile < end) {
        pages.ask(a.pages, table, c, tile * kTile, lane);
        load(k_a, v_a, valid_a, tile);
        pages.ask(a.pages, table, c, (tile + kWaves) * kTile, lane);
    }

    // Q^T: head `col`, the dims of each step
    u32x4 q[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; s++) {
        const int d = dim_of(s);
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

    auto compute = [&](u32x4 (&k)[2][kLoads], VPiece (&v)[kSets][8], mfh_u32 valid) {
        f32x4 s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
        auto product = [&](auto cut) {
#pragma unroll
            for (int s = 0; s < kSteps; s++) {
                u32x4 k0, k1;
                if constexpr (FP8) {
                    const int w = 2 * (s & 1);
                    k0 = widen<DT>(k[0][s / 2][w], k[0][s / 2][w + 1]);
                    k1 = widen<DT>(k[1][s / 2][w], k[1][s / 2][w + 1]);
                } else {
                    k0 = k[0][s], k1 = k[1][s];
                }
                if (cut.value && dim_of(s) >= a.dim) k0 = k1 = u32x4{0, 0, 0, 0};
                s0 = mfma16<DT>(k0, q[s], s0);
                s1 = mfma16<DT>(k1, q[s], s1);
            }
        };
        if (ragged) product(std::true_type{});
        else product(std::false_type{});

        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = (j < 4 ? s0[j & 3] : s1[j & 3]) * a.scale;
        if (a.cap == kNarrow) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = capped(x[j], a.cap_factor, a.cap_scaled);
        } else if (a.cap == kWide) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = wide_capped(x[j], a.cap_factor, a.cap_scaled);
        }
        if (a.slopes) {
            const int back = (int)(c.length - 1) - (int)(tile * kTile + 4 * quad);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] -= slope * (float)(back - (16 * (j >> 2) + (j & 3)));
        }
        if (valid != 0xffffffffu) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (!(valid >> (16 * (j >> 2) + 4 * quad + (j & 3)) & 1)) {
                    x[j] = -INFINITY;
#pragma unroll
                    for (int u = 0; u < kSets; u++) v[u][j] = VPiece{};  // 0 * NaN would be NaN
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
                const float next = top - kBelow<DT, FP8>;
                const float alpha = limit == -INFINITY ? 0.0f : exp2_fast(ref - next);
                ref = next;
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
            u32x4 t[8];
#pragma unroll
            for (int j = 0; j < 8; j++) t[j] = dims_of<DT, FP8, kDims>(v[u][j]);
#pragma unroll
            for (int d = 0; d < kDims; d += 2) {
                const int i = d / 2;
                const u32x4 even = {low_halves(t[0][i], t[1][i]), low_halves(t[2][i], t[3][i]),
                                    low_halves(t[4][i], t[5][i]), low_halves(t[6][i], t[7][i])};
                const u32x4 odd = {high_halves(t[0][i], t[1][i]), high_halves(t[2][i], t[3][i]),
                                   high_halves(t[4][i], t[5][i]), high_halves(t[6][i], t[7][i])};
                acc[u][d] = mfma16<DT>(even, p, acc[u][d]);
                acc[u][d + 1] = mfma16<DT>(odd, p, acc[u][d + 1]);
            }
        }
    };
    // Loads of a tile past the last one are made too, and move nothing:
    // behind loads that only some iterations make, the compiler waits for
    // all that are on their way.
    while (tile < end) {
        load(k_b, v_b, valid_b, tile + kWaves);
        pages.ask(a.pages, table, c, (tile + 2 * kWaves) * kTile, lane);
        compute(k_a, v_a, valid_a);
        tile += kWaves;
        if (tile >= end) break;
        load(k_a, v_a, valid_a, tile + kWaves);
        pages.ask(a.pages, table, c, (tile + 2 * kWaves) * kTile, lane);
        compute(k_b, v_b, valid_b);
        tile += kWaves;
    }

    // The waves' results meet: a common reference, then sums weighted by it.  A
    // wave without a reference has seen nothing, and its sum is 0, or nothing but
    // NaN, and its sum is NaN: it is added as it stands, for the row is NaN then.
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    const float wave_ref = limit == -INFINITY ? -INFINITY : ref;
    if (quad == 0) {
        s_ref[wave][col] = wave_ref;
        s_sum[wave][col] = sum;
    }
    __syncthreads();
    float top = s_ref[0][col];
#pragma unroll
    for (int w = 1; w < kWaves; w++) top = fmaxf(top, s_ref[w][col]);
    const float weight = wave_ref == -INFINITY ? 0.0f : exp2_fast(wave_ref - top);
#pragma unroll
    for (int u = 0; u < kSets; u++) {
        if (u) __syncthreads();
#pragma unroll
        for (int d = 0; d < kDims; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) s_out[wave][col][kDims * (4 * quad + i) + d] = weight * acc[u][d][i];
        __syncthreads();
        const int dims = min(kSetDims, a.dim - u * kSetDims);
        for (int i = threadIdx.x; i < heads * (kSetDims / 2); i += kThreads) {
            const int h = i / (kSetDims / 2), d = 2 * (i % (kSetDims / 2)), dim = u * kSetDims + d;
            if (d >= dims) continue;
            float all = s_ref[0][h], total = 0.0f, o0 = 0.0f, o1 = 0.0f;
#pragma unroll
            for (int w = 1; w < kWaves; w++) all = fmaxf(all, s_ref[w][h]);
#pragma unroll
            for (int w = 0; w < kWaves; w++)
                total += s_ref[w][h] == -INFINITY ? s_sum[w][h] : exp2_fast(s_ref[w][h] - all) * s_sum[w][h];  // 0, or NaN
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                o0 += s_out[w][h][d];
                o1 += s_out[w][h][d + 1];
            }
            if (!SPLIT || parts == 1) {
                const float f = total == 0.0f ? 0.0f : a.v_scale / total;
                store4(a.out + ((int64_t)r * a.out_t + (int64_t)(head0 + h) * a.out_h + dim) * 2, enc16x2<DT>(o0 * f, o1 * f));
                if (dim == 0 && a.lse)
                    a.lse[(int64_t)r * a.q_heads + head0 + h] = total == 0.0f ? -INFINITY : all * kLn2 + logf(total);
            } else {
                const int64_t slot = (int64_t)blockIdx.x * a.part_heads + h;
                *reinterpret_cast<float2*>(a.part_out + slot * a.dim + dim) = make_float2(o0, o1);
                if (dim == 0) a.part_sum[slot] = make_float2(all, total);
            }
        }
    }
}

// Joins the parts of the rows that have several, and writes the rows of
// requests without tokens.  A workgroup takes 128 dims of a query head, a
// quarter of the parts in each wave; lanes take two dims each.
constexpr int kJoinWaves = 4;

template <int DT>
__global__ __launch_bounds__(64 * kJoinWaves) void k_decode_join(DecodeArgs a)
{
    __shared__ float s_all[kJoinWaves];
    __shared__ float2 s_out[kJoinWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int chunks = (a.dim + 127) / 128;
    const mfh_u32 head_row = blockIdx.x / chunks, chunk = blockIdx.x - head_row * chunks;
    const mfh_u32 r = a.by_q_heads.quotient(head_row), head = head_row - r * a.q_heads;
    const mfh_u32 kv = head / a.group, in_group = head - kv * a.group;
    const mfh_u32 row_of = kv * a.head_groups + in_group / kHeads, h = in_group % kHeads;
    const Context c(a, r);
    const mfh_u32 piece = piece_of(a, lane), parts = parts_of(c.tiles, piece);
    if (parts == 1) return;  // one workgroup had it all
    mfh_u32 before = 0;
    for (mfh_u32 base = 0; base < r; base += 64)
        if (base + lane < r) before += parts_of(lane_tiles(a, base + lane), piece);
    const int64_t slot0 = (int64_t)last_lane(lanes_upto(before)) * a.request_rows + (mfh_u64)row_of * parts;
    const int d = 128 * chunk + 2 * lane;
    const float2* sums = a.part_sum + slot0 * a.part_heads + h;
    const float* from = a.part_out + (slot0 * a.part_heads + h) * a.dim + min(d, a.dim - 2);
    float top = -INFINITY;
    for (mfh_u32 n = lane; n < parts; n += 64) top = fmaxf(top, sums[(int64_t)n * a.part_heads].x);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
    float all = 0.0f, o0 = 0.0f, o1 = 0.0f;
#pragma unroll 4
    for (mfh_u32 n = wave; n < parts; n += kJoinWaves) {
        const float2 s = sums[(int64_t)n * a.part_heads];
        const float2 w = *reinterpret_cast<const float2*>(from + (int64_t)n * a.part_heads * a.dim);
        const float f = s.x == -INFINITY ? 0.0f : exp2_fast(s.x - top);
        all += s.x == -INFINITY ? s.y : f * s.y;  // without a reference 0, or NaN
        o0 += f * w.x;
        o1 += f * w.y;
    }
    if (lane == 0) s_all[wave] = all;
    s_out[wave][lane] = make_float2(o0, o1);
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < kJoinWaves; w++) {
        all += s_all[w];
        o0 += s_out[w][lane].x;
        o1 += s_out[w][lane].y;
    }
    if (d >= a.dim) return;
    const float f = all == 0.0f ? 0.0f : a.v_scale / all;
    store4(a.out + ((int64_t)r * a.out_t + (int64_t)head * a.out_h + d) * 2, enc16x2<DT>(o0 * f, o1 * f));
    if (d == 0 && a.lse) a.lse[(int64_t)r * a.q_heads + head] = all == 0.0f ? -INFINITY : top * kLn2 + logf(all);
}

// How a call is laid out, from what the host knows: the number of rows and the
// lengths' upper bound.
struct Layout {
    bool split;
    int64_t rows;
    mfh_u32 blocks, uneven;  // workgroups aimed at
    int part_heads;
    size_t bytes;
};

// One workgroup a row where rows are short, and no second kernel: up to 16
// tiles (8 rows of 512 tokens 10.7 us, split 12.8), and up to 32 where the rows
// alone fill the card (256 rows of 1024 tokens 24.2 us, split 27.6).  Beyond,
// and where lengths may differ much, the split wins: 8 rows of 2048 tokens 28.6
// and 12.6 us, 512 rows of 1..4096 74 and 44.  The split aims at one workgroup
// per CU: two come out slower at 256 dims (33.5 us, 39.7) and for 64 rows
// (14.9, 15.8), and equal or 8% faster elsewhere.  Where requests differ in length
// by so much that the longest is a quarter over the mean, which only the device
// knows, a row's last cut leaves much uneven, and half as many workgroups again
// even it out: 48 rows of 1..16384, e4m3, 33.5 us and 38, the same in bf16 47 and
// 57; 128 rows of 1..3000 73.6 and 76.8 (rows of 256 dims 19.1 and 18.6).
Layout layout(const Device* dev, const mfh_attention_shape& sh, const mfh_kv_cache& c, int32_t requests, int64_t longest)
{
    Layout l{};
    const int group = sh.q_heads / c.kv_heads;
    l.rows = (int64_t)requests * c.kv_heads * ((group + kHeads - 1) / kHeads);
    l.part_heads = std::min(group, kHeads);
    const int64_t tiles = (std::min<int64_t>(std::max<int64_t>(longest, 1), kLongest) + kTile - 1) / kTile;
    l.blocks = (mfh_u32)dev->compute_units, l.uneven = l.blocks + l.blocks / 2;
    l.split = tiles > (l.rows >= dev->compute_units ? 32 : 16);
    l.bytes = l.split ? (size_t)(l.uneven + l.rows) * l.part_heads * (c.head_dim + 2) * sizeof(float) : 0;
    return l;
}

template <int DT, bool FP8, int DP, bool FAST>
void launch_form(const Layout& l, hipStream_t s, const DecodeArgs& a)
{
    if (l.split) k_decode<DT, FP8, DP, FAST, true><<<(unsigned)(l.uneven + l.rows), kThreads, 0, s>>>(a);
    else k_decode<DT, FP8, DP, FAST, false><<<(unsigned)l.rows, kThreads, 0, s>>>(a);
}

template <int DT, bool FP8>
void launch_dims(bool fast, const Layout& l, hipStream_t s, const DecodeArgs& a)
{
    if (fast) {
        if (a.dim <= 64) launch_form<DT, FP8, 64, true>(l, s, a);
        else if (a.dim <= 128) launch_form<DT, FP8, 128, true>(l, s, a);
        else launch_form<DT, FP8, 256, true>(l, s, a);
    } else {
        if (a.dim <= 64) launch_form<DT, FP8, 64, false>(l, s, a);
        else if (a.dim <= 128) launch_form<DT, FP8, 128, false>(l, s, a);
        else launch_form<DT, FP8, 256, false>(l, s, a);
    }
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
    *bytes = layout(dev, *shape, *cache, requests, longest).bytes;
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
    DecodeArgs a{};
    a.pages = PageArgs(*cache, k_cache, v_cache, table, table_stride, table_width);
    a.q = (const char*)q, a.out = (char*)out, a.lse = lse;
    a.lengths = lengths, a.slopes = slopes;
    const Strides qs(shape->q_token_stride, shape->q_head_stride, shape->q_heads, cache->head_dim);
    const Strides os(shape->out_token_stride, shape->out_head_stride, shape->q_heads, cache->head_dim);
    a.q_t = qs.token, a.q_h = qs.head, a.out_t = os.token, a.out_h = os.head;
    a.scale = shape->scale * cache->k_scale * kLog2e;
    if (shape->softcap > 0.0f) {
        a.cap_scaled = shape->softcap * kLog2e;
        a.cap = shape->softcap > kWideCap ? kWide : kNarrow;
        a.cap_factor = a.cap == kWide ? 1.0f / a.cap_scaled : 2.0f / shape->softcap;
    }
    a.v_scale = cache->v_scale;
    a.window = shape->window, a.requests = requests, a.kv_heads = cache->kv_heads, a.q_heads = shape->q_heads;
    a.group = shape->q_heads / cache->kv_heads;
    a.head_groups = (a.group + kHeads - 1) / kHeads;
    a.dim = cache->head_dim;
    a.request_rows = (mfh_u32)(a.kv_heads * a.head_groups);
    Layout l = layout(dev, *shape, *cache, requests, longest);
    // all tiles, and the join's grid, in fewer than 31 bits
    const int64_t most = std::min<int64_t>((int64_t)table_width * cache->page_size, kLongest) / kTile + 1;
    if (l.bytes > workspace_bytes || l.rows * most > kLongest || (int64_t)requests * shape->q_heads > (1 << 22))
        l.split = false;
    if (l.rows + l.uneven >= (int64_t(1) << 32) / kThreads)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d requests of %d heads are too many for one call", what, requests,
                    shape->q_heads);
    a.blocks = l.blocks, a.uneven = l.uneven;
    a.part_heads = l.part_heads;
    if (l.split) {
        a.part_out = (float*)workspace;
        a.part_sum = (float2*)(a.part_out + (l.uneven + l.rows) * l.part_heads * a.dim);
    }
    a.by_head_groups = Divider((mfh_u32)a.head_groups), a.by_request_rows = Divider(a.request_rows);
    a.by_blocks = Divider(l.blocks), a.by_uneven = Divider(l.uneven), a.by_q_heads = Divider((mfh_u32)a.q_heads);
    hipStream_t s = (hipStream_t)stream;
    // whole groups of 16 tokens, and dwords for buffer loads
    const bool fast = cache->page_size % 16 == 0 &&
                      ((uintptr_t)k_cache | (uintptr_t)v_cache | a.pages.page_bytes | a.pages.head_bytes | a.pages.token_bytes) % 4 == 0;
    const bool fp8 = cache->dtype == kF8E4M3;
    if (shape->dtype == kBFloat16) {
        if (fp8) launch_dims<kBFloat16, true>(fast, l, s, a);
        else launch_dims<kBFloat16, false>(fast, l, s, a);
    } else {
        if (fp8) launch_dims<kFloat16, true>(fast, l, s, a);
        else launch_dims<kFloat16, false>(fast, l, s, a);
    }
    MFH_TRY(launch_status("k_decode"));
    if (l.split) {
        const unsigned grid = (unsigned)((int64_t)requests * shape->q_heads * ((a.dim + 127) / 128));
        if (shape->dtype == kBFloat16) k_decode_join<kBFloat16><<<grid, 64 * kJoinWaves, 0, s>>>(a);
        else k_decode_join<kFloat16><<<grid, 64 * kJoinWaves, 0, s>>>(a);
        MFH_TRY(launch_status("k_decode_join"));
    }
    return MFH_OK;
}

}  // extern "C"
