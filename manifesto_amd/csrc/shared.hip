// shared.hip — attention of one new token per request over a paged cache, where
// the requests of a group have their first tokens in common
// (mfh_paged_decode_shared).
//
// As decode.hip, with the shared tokens' keys and values read once for all of a
// group: a column of the matrix products is then a query head of any of the
// group's requests, and a workgroup takes 16, 32 or 64 of them.  Below some 64
// columns bytes bound it, above the matrix units and the exponentials beside
// them.  A request's own tokens are a group of one request.  Both kinds of
// parts run in one launch, the shared ones first, and a second one joins them; where
// a group has so many columns that prefill's kernels compute the shared parts, these
// are a launch of their own in front.
//
// A wave takes tiles of 32 tokens on its own: whole rows of K and V into registers
// while the tile before is worked on, from there to its part of LDS, and out of it
// as matrix operands, V turned on the way, once for all columns.  Columns see
// different tokens (a window, a request shorter than its group's shared
// tokens), so that a value that is not finite may be seen by some only: it is
// cut to zero in the product and added to those columns by itself.
#include "decode.hpp"

#include <numeric>

namespace mfh {

int check_attention(const mfh_attention_shape* shape, const mfh_kv_cache* cache, const char* what);  // decode.hip

namespace {

using namespace decode;

constexpr int kMostGroups = 4096;

struct SharedArgs {
    PageArgs pages;
    const char* q;
    char* out;
    float* lse;
    float* part_out;   // [requests * q_heads][parts][head_dim]
    float2* part_sum;  // [requests * q_heads][parts]: reference and sum
    const int32_t* lengths;
    const int32_t* starts;
    const int32_t* shared;
    const float* slopes;
    int64_t q_t, q_h, out_t, out_h;  // elements
    float scale, cap_scaled, cap_factor, v_scale;
    int cap;
    int32_t window, kv_heads, q_heads, group, head_groups, dim;
    mfh_u32 requests, groups, group_step;  // group_step: groups between two that are looked at first
    mfh_u32 shared_blocks;
    mfh_u32 shared_parts, own_parts, parts, shared_piece, own_piece;  // piece: tiles of a part
    bool all_parts;  // every request of a group has as many shared parts as there are
    bool alone;      // a wave takes a request's own part alone
    Divider by_group, by_kv_parts, by_shared_parts, by_own_parts, by_kv_heads, by_head_groups, by_shared_piece, by_own_piece, by_q_heads;
};

MFH_DEV mfh_u32 limited(const SharedArgs& a, int32_t tokens)
{
    const mfh_u64 most = min((mfh_u64)a.pages.width * a.pages.by_page.d, (mfh_u64)kLongest);
    return min((mfh_u32)max(tokens, 0), (mfh_u32)most);
}

MFH_DEV mfh_u32 length_of(const SharedArgs& a, mfh_u32 r) { return limited(a, a.lengths[r]); }

// The first token that a request of this length sees.
MFH_DEV mfh_u32 first_of(const SharedArgs& a, mfh_u32 length)
{
    return a.window > 0 && length > (mfh_u32)a.window ? length - a.window : 0;
}

// Requests that share tokens, and those that some of them see: [first, length).
struct Group : Seen {
    mfh_u32 begin, members;
    // 64 groups from `base` on, one a lane
    struct Lanes {
        mfh_u32 begin, end, length;
        MFH_DEV Lanes(const SharedArgs& a, mfh_u32 base, int lane)
        {
            const mfh_u32 g = base + lane;
            begin = end = length = 0;
            if (g >= a.groups) return;
            const int32_t from = a.starts[g], to = a.starts[g + 1], tokens = a.shared[g];
            begin = (mfh_u32)min(max(from, 0), (int)a.requests);
            end = (mfh_u32)min(max(to, (int)begin), (int)a.requests);
            length = limited(a, tokens);
        }
    };
    MFH_DEV void of(const SharedArgs& a, const Lanes& lanes, int at, int lane)
    {
        begin = (mfh_u32)__builtin_amdgcn_readlane((int)lanes.begin, at);
        members = (mfh_u32)__builtin_amdgcn_readlane((int)lanes.end, at) - begin;
        length = (mfh_u32)__builtin_amdgcn_readlane((int)lanes.length, at);
        first = 0;
        if (a.window > 0) {
            first = length;
            for (mfh_u32 m = lane; m < members; m += 64) {
                const mfh_u32 its = length_of(a, begin + m);
                if (its > 0) first = min(first, first_of(a, its));
            }
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) first = min(first, (mfh_u32)__shfl_xor((int)first, x));
            first = uniform(first);
        }
    }
    // Looks for the group of request r; without one it has no members and shares nothing.
    MFH_DEV void with(const SharedArgs& a, mfh_u32 r, int lane)
    {
        begin = members = length = first = 0;
        mfh_u32 base = 0;
        if (a.group_step > 1) {  // every group_step-th group first
            const mfh_u32 g = lane * a.group_step;
            const mfh_u64 upto = __ballot(g < a.groups && a.starts[min(g, a.groups)] <= (int64_t)r);
            if (!upto) return;
            base = ((mfh_u32)__popcll(upto) - 1) * a.group_step;
        }
        const Lanes lanes(a, base, lane);
        const mfh_u64 its = __ballot(lanes.begin <= r && r < lanes.end);
        if (its) of(a, lanes, __ffsll((unsigned long long)its) - 1, lane);
    }
};

// Tiles of the seen tokens, and how many parts they have.
struct Tiles {
    mfh_u32 first, count, parts;
    MFH_DEV Tiles(const Seen& s, const Divider& by_piece, mfh_u32 most_parts)
    {
        first = s.first / kTile;
        count = s.length > s.first ? (s.length + kTile - 1) / kTile - first : 0;
        parts = min(by_piece.quotient(count + by_piece.d - 1), most_parts);
    }
};

// One part: the tiles begin .. end of `seen`, read through `table`, for the
// columns column0 .. of `members` requests from `request0` on.  WAVES: of the
// workgroup that take the tiles in turn; 1: the wave is alone.
template <int DT, bool FP8, int DP, bool FAST, int SETS, int WAVES>
struct Part {
    static constexpr int kBytes = FP8 ? 1 : 2;
    static constexpr int kSteps = DP / 32;                    // of the product with K
    static constexpr int kLoads = FP8 ? kSteps / 2 : kSteps;  // of 16 bytes of a token of K
    static constexpr int kDimTiles = DP / 16;
    static constexpr int kSums = SETS * kDimTiles;            // registers of four sums
    static constexpr int kGiven = kSums / kWaves;             // of a wave where all meet
    static constexpr int kPieces = DP * kBytes / 16;          // of 16 bytes in a row
    static constexpr int kRowsAtOnce = 64 / kPieces;          // of a load
    static constexpr int kRaw = 32 / kRowsAtOnce;
    static constexpr int kKinds = 16 / kRowsAtOnce;           // of lanes' places in a page
    static constexpr int kPitch = DP * 2;                     // of a row of V in LDS, in bytes
    // Shared tokens are read by several workgroups where their columns fill more than
    // one: nt would keep them out of the L2.
    static constexpr int kPolicy = SETS > 1 ? 0 : kStreamed;
    struct Lds {
        float ref[kWaves][SETS][kHeads], sum[kWaves][SETS][kHeads];
        union {
            struct {
                u32x4 k[32 * kPieces];
                u32x4 v[32 * kPitch / 16];
            } tile[kWaves];
            f32x4 given[WAVES > 1 ? kWaves - 1 : 1][WAVES > 1 ? kSums : 1][64];
        };
    };
    // Where piece c of row r stands in LDS among the PIECES of the row: 16 rows'
    // pieces in 16 different places, as K is read, and so two of each in V.
    template <int PIECES>
    static MFH_DEV int place(int r, int c)
    {
        if constexpr (PIECES >= 16) return c ^ (r & 15);
        else return c ^ (r / (16 / PIECES) & (PIECES - 1));
    }

    static MFH_DEV void run(const SharedArgs& a, Lds& lds, mfh_u32 request0, mfh_u32 members, mfh_u32 column0, mfh_u32 kv,
                            const Seen& seen, mfh_u32 table_row, mfh_u32 begin, mfh_u32 end, mfh_u32 slot)
    {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int col = lane & 15, quad = lane >> 4;
        const mfh_u32 columns = members * a.group;

        // (the table is read as scalars)
        typedef const __attribute__((address_space(4))) int32_t* Table;
        const Table table = (Table)(uintptr_t)(a.pages.table + (int64_t)table_row * a.pages.table_stride);
        Pages<FAST> pages;
        mfh_u32 tile = begin + (WAVES > 1 ? wave : 0);
        pages.ask(a.pages, table, seen, tile * kTile, lane);

        // This lane's columns: their queries, and the tokens they see.
        u32x4 q[SETS][kSteps];
        float slope[SETS];
        mfh_u32 its_first[SETS], its_length[SETS];
        mfh_u32 all_first = 0, all_length = ~0u;
        auto dim_of = [&](int s) { return FP8 ? 64 * (s / 2) + 16 * quad + 8 * (s & 1) : 32 * s + 8 * quad; };
        auto column = [&](int n) { return column0 + 16 * n + col; };
        auto row_of = [&](int n) {  // request * q_heads + head, of the first column where there is no such one
            const mfh_u32 c = column(n) < columns ? column(n) : 0, member = a.by_group.quotient(c);
            return (int64_t)(request0 + member) * a.q_heads + kv * a.group + (c - member * a.group);
        };
#pragma unroll
        for (int n = 0; n < SETS; n++) {
            const bool real = column(n) < columns;
            const mfh_u32 c = real ? column(n) : 0, member = a.by_group.quotient(c), head = kv * a.group + (c - member * a.group);
            const mfh_u32 r = request0 + member;
            its_length[n] = length_of(a, r);
            slope[n] = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; s++) {
                const int d = dim_of(s);
                q[n][s] = u32x4{0, 0, 0, 0};
                if (real && d < a.dim) q[n][s] = load16<false>(a.q + ((int64_t)r * a.q_t + (int64_t)head * a.q_h + d) * 2);
            }
        }

        // A load takes whole rows, a piece a lane; where it goes to LDS as it is, the
        // lane takes the piece whose place it fills.  Pieces past head_dim are zeros, which
        // buffer loads past every page's end give, or else the row's last one again,
        // cut below.
        const mfh_u32 token_bytes = a.pages.token_bytes;
        mfh_u32 k_lane[kKinds], v_lane[kKinds];
        const int last = a.dim * kBytes - 16;
#pragma unroll
        for (int s = 0; s < kKinds; s++) {
            const int row = lane / kPieces, own = lane % kPieces;
            auto at_piece = [&](int c) {
                return FAST ? 16 * c <= last ? row * token_bytes + 16 * c : 1u << 31 : (mfh_u32)min(16 * c, last);
            };
            k_lane[s] = at_piece(place<kPieces>(kRowsAtOnce * s + row, own));
            v_lane[s] = FP8 ? at_piece(own) : k_lane[s];
        }
        const bool ragged = a.dim != DP;
        const char* k_base = a.pages.k + kv * a.pages.head_bytes;
        const char* v_base = a.pages.v + kv * a.pages.head_bytes;
        typedef u32x4 Rows[kRaw];
        auto load = [&](Rows& raw, const char* base, const mfh_u32 (&at_lane)[kKinds], const TileAt<FAST>& at) {
            if constexpr (FAST) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const __amdgpu_buffer_rsrc_t rows = page_buffer(base, at.page[h], a.pages);
#pragma unroll
                    for (int s = 0; s < kKinds; s++)
                        raw[h * kKinds + s] = buffer_piece<u32x4, kPolicy>(rows, at_lane[s], at.in_page[h] + s * kRowsAtOnce * token_bytes);
                }
            } else {
#pragma unroll
                for (int i = 0; i < kRaw; i++)
                    raw[i] = load16<kPolicy == kStreamed>(base + shuffle64(at.mine, i * kRowsAtOnce + lane / kPieces) + at_lane[i % kKinds]);
            }
        };
        // One tile's registers: the next tile sets out when this one is in LDS.  Loads of
        // a tile past the last one are made too, and move nothing: behind loads that only
        // some waves or rounds make, the compiler waits for all that are on their way.
        Rows k, v;
        TileAt<FAST> at = pages.place(a.pages, seen, tile * kTile, lane, tile < end);
        load(k, k_base, k_lane, at);
        load(v, v_base, v_lane, at);
        pages.ask(a.pages, table, seen, (tile + WAVES) * kTile, lane);

#pragma unroll
        for (int n = 0; n < SETS; n++) {
            its_first[n] = first_of(a, its_length[n]);
            if (column(n) < columns) all_first = max(all_first, its_first[n]), all_length = min(all_length, its_length[n]);
        }
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) {
            all_first = max(all_first, (mfh_u32)__shfl_xor((int)all_first, x));
            all_length = min(all_length, (mfh_u32)__shfl_xor((int)all_length, x));
        }
        all_first = uniform(all_first), all_length = uniform(all_length);
        // Queries of several sets wait in accumulation registers, where the products take
        // them from.
        if constexpr (SETS > 1) {
#pragma unroll
            for (int n = 0; n < SETS; n++)
#pragma unroll
                for (int s = 0; s < kSteps; s++) asm volatile("" : "+a"(q[n][s]));
        }

        f32x4 acc[kSums];  // [set][tile of 16 dims]: dims 4 quad .. of the tile
        float ref[SETS], limit[SETS], sum[SETS];
#pragma unroll
        for (int n = 0; n < SETS; n++) ref[n] = 0.0f, limit[n] = -INFINITY, sum[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < kSums; i++) acc[i] = f32x4{0, 0, 0, 0};

        auto& mine = lds.tile[wave];
        const int k_at = col * kPieces + place<kPieces>(col, quad);  // pieces 4 s + quad of rows col and 16 + col
        auto scores = [&](float (&x)[SETS][8]) {
            f32x4 s0[SETS], s1[SETS];
#pragma unroll
            for (int n = 0; n < SETS; n++) s0[n] = s1[n] = f32x4{0, 0, 0, 0};
            u32x4 from[2][kLoads];
#pragma unroll
            for (int s = 0; s < kLoads; s++)
#pragma unroll
                for (int h = 0; h < 2; h++) from[h][s] = mine.k[16 * kPieces * h + (k_at ^ (4 * s))];
            // (left to itself the compiler reads right ahead of each product, and waits there)
            __builtin_amdgcn_sched_barrier(0);
            auto product = [&](auto cut) {
#pragma unroll
                for (int s = 0; s < kSteps; s++) {
                    u32x4 k0, k1;
                    if constexpr (FP8) {
                        const int w = 2 * (s & 1);
                        k0 = widen<DT>(from[0][s / 2][w], from[0][s / 2][w + 1]);
                        k1 = widen<DT>(from[1][s / 2][w], from[1][s / 2][w + 1]);
                    } else {
                        k0 = from[0][s], k1 = from[1][s];
                    }
                    if (cut.value && dim_of(s) >= a.dim) k0 = k1 = u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int n = 0; n < SETS; n++) {
                        s0[n] = mfma16<DT>(k0, q[n][s], s0[n]);
                        s1[n] = mfma16<DT>(k1, q[n][s], s1[n]);
                    }
                }
            };
            if (!FAST && ragged) product(std::true_type{});
            else product(std::false_type{});
#pragma unroll
            for (int n = 0; n < SETS; n++)
#pragma unroll
                for (int j = 0; j < 8; j++) x[n][j] = j < 4 ? s0[n][j & 3] : s1[n][j & 3];
        };
        // Where scores need more than their scale, they get it here.
        const bool simple = a.cap == kNone && !a.slopes && a.scale > 0.0f;
        const float scale = simple ? a.scale : 1.0f;
        auto shape = [&](float (&x)[SETS][8], mfh_u32 t0) {
#pragma unroll
            for (int n = 0; n < SETS; n++)
#pragma unroll
                for (int j = 0; j < 8; j++) x[n][j] *= a.scale;
            if (a.cap == kNarrow) {
#pragma unroll
                for (int n = 0; n < SETS; n++)
#pragma unroll
                    for (int j = 0; j < 8; j++) x[n][j] = capped(x[n][j], a.cap_factor, a.cap_scaled);
            } else if (a.cap == kWide) {
#pragma unroll
                for (int n = 0; n < SETS; n++)
#pragma unroll
                    for (int j = 0; j < 8; j++) x[n][j] = wide_capped(x[n][j], a.cap_factor, a.cap_scaled);
            }
            if (a.slopes) {
#pragma unroll
                for (int n = 0; n < SETS; n++) {
                    const int back = (int)(its_length[n] - 1) - (int)(t0 + 4 * quad);
#pragma unroll
                    for (int j = 0; j < 8; j++) x[n][j] -= slope[n] * (float)(back - (16 * (j >> 2) + (j & 3)));
                }
            }
        };
        // The weights of x * scale.
        auto soften = [&](float (&x)[SETS][8], u32x4 (&p)[SETS]) {
            float top[SETS];
            bool above = false;
#pragma unroll
            for (int n = 0; n < SETS; n++) {
                top[n] = x[n][0];
#pragma unroll
                for (int j = 1; j < 8; j++) top[n] = fmaxf(top[n], x[n][j]);
                top[n] *= scale;
                above |= top[n] > limit[n];
            }
            if (__any(above)) {
                // (the sums are taken out of the accumulation registers here, and not, for all
                // tiles, ahead of the question)
                if constexpr (SETS > 1) {
#pragma unroll
                    for (int i = 0; i < kSums; i++) asm volatile("" : "+a"(acc[i]));
                }
#pragma unroll
                for (int n = 0; n < SETS; n++) {
                    top[n] = fmaxf(top[n], __shfl_xor(top[n], 16));
                    top[n] = fmaxf(top[n], __shfl_xor(top[n], 32));
                    if (top[n] > limit[n]) {
                        const float next = top[n] - kBelow<DT, FP8>;
                        const float alpha = limit[n] == -INFINITY ? 0.0f : exp2_fast(ref[n] - next);
                        ref[n] = next;
                        limit[n] = top[n] + kStep;
                        sum[n] *= alpha;
#pragma unroll
                        for (int i = 0; i < kDimTiles; i++) acc[n * kDimTiles + i] *= alpha;
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < SETS; n++) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[n][j] = exp2_fast(__builtin_fmaf(x[n][j], scale, -ref[n]));
#pragma unroll
                for (int j = 0; j < 4; j++) p[n][j] = enc16x2<DT>(x[n][2 * j], x[n][2 * j + 1]);
                sum[n] += ((x[n][0] + x[n][1]) + (x[n][2] + x[n][3])) + ((x[n][4] + x[n][5]) + (x[n][6] + x[n][7]));
            }
        };
        auto mask = [&](float (&x)[SETS][8], mfh_u32 t0, mfh_u32 valid) {
#pragma unroll
            for (int n = 0; n < SETS; n++) {
                const mfh_u32 low = its_first[n] > t0 ? min(its_first[n] - t0, 32u) : 0;
                const mfh_u32 high = its_length[n] > t0 ? min(its_length[n] - t0, 32u) : 0;
                const mfh_u32 sees = high > low ? (mfh_u32)(((mfh_u64)1 << high) - ((mfh_u64)1 << low)) & valid : 0;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (!(sees >> (16 * (j >> 2) + 4 * quad + (j & 3)) & 1)) x[n][j] = -INFINITY;
            }
        };
        // Cuts values to zero that are of no token (0 * NaN would be NaN) or not
        // finite; whether there are any of those.
        auto cut = [&](mfh_u32 valid) {
            bool odd = false;
#pragma unroll
            for (int i = 0; i < kRaw; i++) {
                const bool keep = valid >> (i * kRowsAtOnce + lane / kPieces) & 1;
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    mfh_u32 whole;
                    if constexpr (FP8) {
                        const mfh_u32 tops = ((v[i][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                        whole = tops | (tops - (tops >> 7));
                    } else {
                        const mfh_u32 tops = not_finite<DT>(v[i][w]);
                        whole = tops | (tops - (tops >> 15));
                    }
                    odd |= keep && whole != 0;
                    v[i][w] &= keep ? ~whole : 0u;
                }
            }
            return __any(odd);
        };
        auto stage = [&]() {
#pragma unroll
            for (int i = 0; i < kRaw; i++) mine.k[i * 64 + lane] = k[i];
#pragma unroll
            for (int i = 0; i < kRaw; i++) {
                if constexpr (FP8) {
                    const int row = i * kRowsAtOnce + lane / kPieces, c = 2 * (lane % kPieces);
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        mine.v[row * 2 * kPieces + place<2 * kPieces>(row, c + e)] = widen<DT>(v[i][2 * e], v[i][2 * e + 1]);
                } else {
                    mine.v[i * 64 + lane] = v[i];
                }
            }
        };
        // V^T of 32 tokens, in the order of the weights, and 16 dims: see read_column.
        const int v_row = 4 * quad + (lane & 15) / 4;
        const int v_at = v_row * kPitch + place<DP / 8>(v_row, (lane & 3) / 2) * 16 + 8 * (lane & 1);
        auto add = [&](const u32x4 (&p)[SETS]) {
            const char* from = reinterpret_cast<const char*>(mine.v);
            constexpr int kAhead = kDimTiles < 4 ? kDimTiles : 4;
            u32x4 piece[kDimTiles];
            auto read = [&](int d) {
                const u32x2 lo = read_column(from + (v_at ^ (32 * d))), hi = read_column(from + 16 * kPitch + (v_at ^ (32 * d)));
                piece[d] = u32x4{lo[0], lo[1], hi[0], hi[1]};
            };
#pragma unroll
            for (int d = 0; d < kAhead; d++) read(d);
#pragma unroll
            for (int d = 0; d < kDimTiles; d++) {
                if (d + kAhead < kDimTiles) read(d + kAhead);
                if constexpr (SETS > 1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = 0; n < SETS; n++) acc[n * kDimTiles + d] = mfma16<DT>(piece[d], p[n], acc[n * kDimTiles + d]);
                if constexpr (SETS > 1) __builtin_amdgcn_sched_barrier(0);
            }
        };

        bool odd = false;  // some tile had values that are not finite, and columns that do not see it
        for (; tile < end; tile += WAVES) {
            const mfh_u32 t0 = tile * kTile, valid = at.valid;
            const bool open = valid == 0xffffffffu && t0 >= all_first && t0 + kTile <= all_length;  // to every column
            float x[SETS][8];
            u32x4 p[SETS];
            if (!open) odd |= cut(valid);
            stage();
            at = pages.place(a.pages, seen, t0 + WAVES * kTile, lane, tile + WAVES < end);
            load(k, k_base, k_lane, at);
            load(v, v_base, v_lane, at);
            scores(x);
            pages.ask(a.pages, table, seen, t0 + 2 * WAVES * kTile, lane);
            if (!simple) shape(x, t0);
            if (!open) mask(x, t0, valid);
            soften(x, p);
            add(p);
        }

        // Those values, added to the columns that see them (here, and not in their
        // tile: what the loop holds beside the sums leaves no registers for it).
        auto page_of = [&](mfh_u32 t) { return (mfh_u32)table[a.pages.by_page.quotient(t)]; };
        for (tile = odd ? begin + (WAVES > 1 ? wave : 0) : end; tile < end; tile += WAVES) {
            const mfh_u32 t0 = tile * kTile;
            // a tile that every column sees whole was not cut
            bool whole = t0 >= max(all_first, seen.first) && t0 + kTile <= min(all_length, seen.length);
            for (mfh_u32 i = 0; i < kTile && whole; i++) whole = page_of(t0 + i) < a.pages.pages;
            for (mfh_u32 t = max(t0, seen.first); t < min(t0 + kTile, seen.length) && !whole; t++) {
                const mfh_u32 page = page_of(t);
                if (page >= a.pages.pages) continue;
                const char* row = v_base + (mfh_u64)page * a.pages.page_bytes +
                                  (t - a.pages.by_page.quotient(t) * a.pages.by_page.d) * token_bytes;
#pragma unroll
                for (int d = 0; d < kDimTiles; d++)
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        const int dim = 16 * d + 4 * quad + x;
                        if (dim >= a.dim) continue;
                        mfh_u32 code;
                        if constexpr (FP8) code = e4m3_pair<DT, false>(*reinterpret_cast<const uint8_t*>(row + dim)) & 0xffffu;
                        else code = load2(row + dim * 2);
                        const float value = dec16<DT>(code);
                        if (__builtin_isfinite(value)) continue;
#pragma unroll
                        for (int n = 0; n < SETS; n++)
                            if (t >= its_first[n] && t < its_length[n]) acc[n * kDimTiles + d][x] += value;
                    }
            }
        }

        auto store = [&](int i, const f32x4& x) {  // register i of acc
            const int n = i / kDimTiles, dim = 16 * (i % kDimTiles) + 4 * quad;
            if (column(n) < columns && dim < a.dim)
                *reinterpret_cast<f32x4*>(a.part_out + (row_of(n) * a.parts + slot) * a.dim + dim) = x;
        };
#pragma unroll
        for (int n = 0; n < SETS; n++) {
            sum[n] += __shfl_xor(sum[n], 16);
            sum[n] += __shfl_xor(sum[n], 32);
            if (limit[n] == -INFINITY) ref[n] = -INFINITY;  // nothing seen, or nothing but NaN
        }
        if constexpr (WAVES == 1) {
#pragma unroll
            for (int n = 0; n < SETS; n++) {
#pragma unroll
                for (int d = 0; d < kDimTiles; d++) store(n * kDimTiles + d, acc[n * kDimTiles + d]);
                if (quad == 0 && column(n) < columns) a.part_sum[row_of(n) * a.parts + slot] = make_float2(ref[n], sum[n]);
            }
            return;
        }
        // The waves' results meet: a common reference, and sums weighted by it, of which
        // each wave adds up a quarter.  A wave without a reference has seen nothing,
        // and its sum is 0, or nothing but NaN, and its sum is NaN: it is added as it
        // stands, for the row is NaN then.
        if (quad == 0) {
#pragma unroll
            for (int n = 0; n < SETS; n++) lds.ref[wave][n][col] = ref[n], lds.sum[wave][n][col] = sum[n];
        }
        __syncthreads();
        float weight[SETS];
#pragma unroll
        for (int n = 0; n < SETS; n++) {
            float all = lds.ref[0][n][col], total = 0.0f;
#pragma unroll
            for (int w = 1; w < kWaves; w++) all = fmaxf(all, lds.ref[w][n][col]);
            weight[n] = ref[n] == -INFINITY ? 0.0f : exp2_fast(ref[n] - all);
            if (n % kWaves != wave) continue;
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                const float its = lds.ref[w][n][col];
                total += its == -INFINITY ? lds.sum[w][n][col] : exp2_fast(its - all) * lds.sum[w][n][col];  // 0, or NaN
            }
            if (quad == 0 && column(n) < columns) a.part_sum[row_of(n) * a.parts + slot] = make_float2(all, total);
        }
        f32x4 total[kGiven];
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
#pragma unroll
            for (int c = 0; c < kGiven; c++) {
                const int i = w * kGiven + c;
                const f32x4 x = acc[i] * weight[i / kDimTiles];
                if (w == wave) total[c] = x;
                else lds.given[wave < w ? wave : wave - 1][i][lane] = x;
            }
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kGiven; c++) {
#pragma unroll
            for (int g = 0; g < kWaves - 1; g++) total[c] += lds.given[g][wave * kGiven + c][lane];
            store(wave * kGiven + c, total[c]);
        }
    }
};

// DP: head_dim rounded up to 64, 128 or 256.  SETS: of 16 columns, of the shared tokens.
template <int DT, bool FP8, int DP, bool FAST, int SETS>
__global__ __launch_bounds__(kThreads, SETS > 2 || DP == 256 ? 1 : SETS > 1 || DP == 128 ? 2 : 3) void k_shared(SharedArgs a)
{
    typedef Part<DT, FP8, DP, FAST, SETS, kWaves> Common;
    typedef Part<DT, FP8, DP, FAST, 1, kWaves> Own;
    typedef Part<DT, FP8, DP, FAST, 1, 1> Alone;
    __shared__ union {
        typename Common::Lds common;
        typename Own::Lds own;
        typename Alone::Lds alone;
    } lds;
    const int lane = threadIdx.x & 63;
    if (blockIdx.x < a.shared_blocks) {
        // Workgroups of one head and part, which read the same keys if they are of
        // one group, are on one XCD (every eighth is).  Lines that no group has come
        // last: workgroups go to an XCD's shader engines in turn, and with every fourth
        // an empty one 240 others took two rounds on 256 CUs, 100 us for 67.
        const mfh_u32 line = a.by_kv_parts.quotient(blockIdx.x), kv_part = blockIdx.x - line * a.by_kv_parts.d;
        const mfh_u32 kv = a.by_shared_parts.quotient(kv_part), part = kv_part - kv * a.shared_parts;
        if (kv >= (mfh_u32)a.kv_heads) return;
        constexpr mfh_u32 kColumns = kHeads * SETS;
        Group group;
        mfh_u32 before = 0, tile_of = ~0u;
        for (mfh_u32 base = 0; base < a.groups; base += 64) {
            const typename Group::Lanes lanes(a, base, lane);
            const mfh_u32 its = ((lanes.end - lanes.begin) * a.group + kColumns - 1) / kColumns, upto = before + lanes_upto(its);
            const mfh_u64 past = __ballot(upto > line);
            if (past) {
                const int at = __ffsll((unsigned long long)past) - 1;
                tile_of = line - ((mfh_u32)__builtin_amdgcn_readlane((int)upto, at) - (mfh_u32)__builtin_amdgcn_readlane((int)its, at));
                group.of(a, lanes, at, lane);
                break;
            }
            before = last_lane(upto);
        }
        if (tile_of == ~0u) return;
        tile_of = uniform(tile_of);
        const Tiles tiles(group, a.by_shared_piece, a.shared_parts);
        if (part >= tiles.parts) return;
        const mfh_u32 share = uniform((tiles.count + tiles.parts - 1) / tiles.parts);
        Common::run(a, lds.common, group.begin, group.members, tile_of * kColumns, kv, group, group.begin,
                    tiles.first + min(part * share, tiles.count), tiles.first + min((part + 1) * share, tiles.count), part);
        return;
    }
    // A request's own tokens: a row (request, key-value head, 16 of its query heads) and
    // part each, of a workgroup or, of many rows, of a wave.
    mfh_u32 rest = blockIdx.x - a.shared_blocks;
    if (a.alone) rest = rest * kWaves + uniform(threadIdx.x >> 6);
    mfh_u32 line = a.by_own_parts.quotient(rest);
    const mfh_u32 part = rest - line * a.own_parts;
    rest = line, line = a.by_head_groups.quotient(rest);
    const mfh_u32 head_group = rest - line * a.head_groups;
    const mfh_u32 r = a.by_kv_heads.quotient(line), kv = line - r * a.kv_heads;
    if (r >= a.requests) return;
    Group group;
    group.with(a, r, lane);
    Seen own;
    own.length = uniform(length_of(a, r));
    own.first = max(first_of(a, own.length), group.length);
    const Tiles tiles(own, a.by_own_piece, a.own_parts);
    if (part >= tiles.parts) return;
    const mfh_u32 share = uniform((tiles.count + tiles.parts - 1) / tiles.parts);
    const mfh_u32 begin = tiles.first + min(part * share, tiles.count), end = tiles.first + min((part + 1) * share, tiles.count);
    if (a.alone) Alone::run(a, lds.alone, r, 1, head_group * kHeads, kv, own, r, begin, end, a.shared_parts + part);
    else Own::run(a, lds.own, r, 1, head_group * kHeads, kv, own, r, begin, end, a.shared_parts + part);
}

// Joins a row's parts, of the shared tokens and of its own.  A wave takes 128 dims
// of a query head, two a lane; or, of many parts, four waves a quarter of them each.
constexpr int kJoinWaves = 4;

template <int DT, int WAVES>
__global__ __launch_bounds__(64 * kJoinWaves) void k_shared_join(SharedArgs a, mfh_u32 units)
{
    __shared__ float s_all[kJoinWaves];
    __shared__ float2 s_out[kJoinWaves][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const mfh_u32 chunks = (a.dim + 127) / 128;
    const mfh_u32 unit = WAVES > 1 ? blockIdx.x : blockIdx.x * kJoinWaves + wave;
    if (WAVES == 1 && unit >= units) return;
    const mfh_u32 row = chunks > 1 ? unit / 2 : unit, chunk = unit - row * chunks;
    const mfh_u32 r = a.by_q_heads.quotient(row), head = row - r * a.q_heads;
    Group group;
    group.with(a, r, lane);
    Seen own;
    own.length = length_of(a, r);
    own.first = max(first_of(a, own.length), group.length);
    const mfh_u32 common = group.members == 0 ? 0 : a.all_parts ? a.shared_parts : Tiles(group, a.by_shared_piece, a.shared_parts).parts;
    const mfh_u32 parts = common + Tiles(own, a.by_own_piece, a.own_parts).parts;
    const float2* sums = a.part_sum + (int64_t)row * a.parts;
    const int d = 128 * chunk + 2 * lane;
    const float* from = a.part_out + (int64_t)row * a.parts * a.dim + min(d, a.dim - 2);
    auto slot = [&](mfh_u32 n) { return n < common ? n : a.shared_parts + (n - common); };
    float top = -INFINITY;
    for (mfh_u32 n = lane; n < parts; n += 64) top = fmaxf(top, sums[slot(n)].x);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
    float all = 0.0f, o0 = 0.0f, o1 = 0.0f;
#pragma unroll 8
    for (mfh_u32 n = WAVES > 1 ? wave : 0; n < parts; n += WAVES) {
        const float2 s = sums[slot(n)];
        const bool seen = s.x != -INFINITY || s.y != 0.0f;  // else there is nothing
        const float2 w = seen ? *reinterpret_cast<const float2*>(from + (int64_t)slot(n) * a.dim) : make_float2(0.0f, 0.0f);
        const float f = s.x == -INFINITY ? 0.0f : exp2_fast(s.x - top);
        all += s.x == -INFINITY ? s.y : f * s.y;  // without a reference 0, or NaN
        o0 += f * w.x;
        o1 += f * w.y;
    }
    if constexpr (WAVES > 1) {
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
    }
    if (d >= a.dim) return;
    const float f = all == 0.0f ? 0.0f : a.v_scale / all;
    store4(a.out + ((int64_t)r * a.out_t + (int64_t)head * a.out_h + d) * 2, enc16x2<DT>(o0 * f, o1 * f));
    if (d == 0 && a.lse) a.lse[row] = all == 0.0f ? -INFINITY : top * kLn2 + logf(all);
}

// A wave a row; four of them where there are many parts, or too few rows to fill the
// card (`few`): 16 requests of 32 heads and 17 parts 43.7 us in all, by a wave a row
// 44.6; 190 of them and 4 parts 51.3 us, by a wave a row 48.9.  Many: 1200 rows of 52
// parts 56.3 us, by a wave a row 58.7; 2000 of 33 63.2 and 63.1; 4000 of 17 88.9 and 84.5.
template <int DT>
void launch_join(const SharedArgs& a, mfh_u32 few, hipStream_t s)
{
    const mfh_u32 units = a.requests * a.q_heads * ((a.dim + 127) / 128);
    if (a.parts > 24 || units <= few) k_shared_join<DT, kJoinWaves><<<units, 64 * kJoinWaves, 0, s>>>(a, units);
    else k_shared_join<DT, 1><<<(units + kJoinWaves - 1) / kJoinWaves, 64 * kJoinWaves, 0, s>>>(a, units);
}

// How a call is laid out, from what the host knows.
//
// Shared tokens: sets of 16 columns, as many as a group has on average, up to 64
// columns, with which a workgroup fills a CU (24 groups of 4 to 32 columns over up
// to 6000 e4m3 tokens: by 64 columns 94 us, by 32 48), and to 32 where there is less
// to share than each request has for itself, whose workgroups a CU then holds two
// of: 24 groups of up to 96 columns over up to 500 e4m3 tokens, 1000 of their own,
// 112 us, by 64 columns 143; one group is as fast by either, 64 requests of 32 heads
// over 8 behind 400 bf16 tokens, 1000 of their own, 44 and 43.
//
// Of 256 columns on and long shared tokens prefill's kernels, whose tiles serve 256
// columns, are faster.  32 heads over 8, bf16, by them and by 64 columns:
//   256 requests over 16384 tokens    120 us  145      64 over 65536    122 us  146
//   over 8192                         100     120      over 16384        62      68
//   over 4096                          84      73      over 8192         52      43
// The rule changes over at 2^22 columns times tokens: the third line left, the second
// right.
// Up to 16 groups, from which on 64 columns fill the card too: groups of 64 such
// requests over 16384, 8 of them 242 us and 301, 16 560 and 555, 24 1428 and 814.
//
// Parts: as many as fill half of the card, so that the requests' own parts run beside
// them on the other half; where the shared tokens take the waves many rounds (`rounds`,
// against those of the own tokens), as many as fill the card, and the own parts come
// after them.  Half: 64 requests over 8192 tokens and 512 of their own 42 us, a full
// card 54; 32 over 4000 and 500 in four groups 55 and 64.  A full card: 48 requests
// over 30000 and 30 67, half of it 92.  Two parts at least where groups may differ
// (those 24: 50 us, with one 63), eight tiles at least.  Of a request's own tokens two
// workgroups a CU, or, where there are four rows a CU and more, a wave a row: 256
// requests of up to 300 own tokens 39 us, by workgroups 44.
struct Layout {
    bool prefill, alone;
    int sets;
    int64_t shared_blocks, own_blocks;
    mfh_u32 kv_parts;  // key-value heads times shared parts, in eights
    mfh_u32 shared_parts, own_parts, shared_piece, own_piece;
    size_t bytes;
};

bool prefill_pays(int64_t columns, int64_t tokens) { return columns >= 256 && columns * tokens >= (1 << 22); }

// Rows of parts (requests * q_heads, times the parts of each) at most, of these sizes
// and of all smaller ones: fewer rows, or fewer own tokens, may have more parts each.
// A row has as many parts as tokens give, a part for eight tiles, and a call:
//   own parts     2 * cus / (requests * kv_heads) a row, so 2 * cus * group, or one each;
//   shared parts  held / (max(1, columns / wide) * kv_heads) a row, of columns * kv_heads
//                 rows: less than 2 * wide * held, which is 128 * cus; or two each;
//   prefill's     cus / (each / P * kv_heads * groups) a row, P its workgroup's rows, of less
//                 than (each + 1) * groups * kv_heads rows, where `each` is at least 256:
//                 less than 257 * cus for its 256 rows.
int64_t part_rows(int64_t cus, int64_t requests, int64_t groups, int64_t group, int64_t kv_heads, int64_t tokens, int64_t own)
{
    const int64_t rows = requests * group * kv_heads, columns = requests * group;
    auto by_tokens = [&](int64_t t) { return rows * (((t + kTile - 1) / kTile + 1 + 7) / 8); };
    const int64_t card = (prefill_pays(columns, tokens) ? 257 : 128) * cus;
    const int64_t own_rows = std::min(by_tokens(own), std::max(rows, 2 * cus * group));
    return own_rows + (groups > 0 ? std::min(by_tokens(tokens), std::max(2 * rows, card)) : 0);
}

Layout layout(const Device* dev, const mfh_attention_shape& sh, const mfh_kv_cache& c, int32_t requests, int32_t groups,
              int64_t most_shared, int64_t most_own)
{
    Layout l{};
    const int group = sh.q_heads / c.kv_heads, cus = dev->compute_units;
    const int64_t columns = (int64_t)requests * group, each = groups > 0 ? columns / groups : 0;
    const int64_t tokens = std::min<int64_t>(std::max<int64_t>(most_shared, 1), kLongest);
    const int64_t own = std::min<int64_t>(std::max<int64_t>(most_own, 1), kLongest);
    l.prefill = prefill_pays(each, tokens) && groups <= 16;
    l.sets = each <= 16 || l.prefill ? 1 : each <= 32 || c.head_dim > 128 || tokens < most_own ? 2 : 4;
    // Columns in 16, 32 or 64, of all groups, at most: a group's number of columns is a
    // multiple of `step`, so that its last line leaves at most that much less than a line.
    const int64_t wide = kHeads * l.sets, step = std::gcd((int64_t)group, wide);
    const int64_t lines = (columns + std::min<int64_t>(groups, requests) * (wide - step)) / wide;
    auto split = [](int64_t blocks, int64_t rows, int64_t tokens, mfh_u32& piece, mfh_u32& parts) {
        const int64_t tiles = (tokens + kTile - 1) / kTile + 1, wanted = std::max<int64_t>(1, blocks / std::max<int64_t>(rows, 1));
        piece = (mfh_u32)std::max<int64_t>(8, (tiles + wanted - 1) / wanted);
        parts = (mfh_u32)((tiles + piece - 1) / piece);
    };
    if (l.prefill) {
        const int64_t rows = (each + prefill_rows(c.head_dim) - 1) / prefill_rows(c.head_dim) * groups * c.kv_heads;
        l.shared_parts = (mfh_u32)std::max<int64_t>(1, std::min<int64_t>({cus / rows, tokens / 256, 64}));
        l.shared_piece = 1;
    } else {
        // Rounds of tiles that the waves take if shared parts have all workgroups that
        // the card holds, and those of the own parts after them.
        const int64_t held = l.sets > 2 || c.head_dim > 128 ? cus : 2 * cus, waves = held * kWaves;
        const int64_t rows = std::max<int64_t>(groups, columns / wide) * c.kv_heads;
        const int64_t heads = (int64_t)requests * c.kv_heads * ((group + kHeads - 1) / kHeads);
        const int64_t rounds = rows * (tokens / kTile) / waves, after = heads * (own / kTile + 1) / waves;
        const int64_t blocks = rounds > 8 + 2 * after ? held : held / 2;
        split(groups > 1 ? std::max(blocks, 2 * rows) : blocks, rows, tokens, l.shared_piece, l.shared_parts);
    }
    split(2 * cus, (int64_t)requests * c.kv_heads, own, l.own_piece, l.own_parts);
    if (groups == 0) l.shared_parts = 0;
    l.kv_parts = (mfh_u32)(((int64_t)c.kv_heads * l.shared_parts + 7) / 8 * 8);
    l.shared_blocks = l.prefill ? 0 : l.kv_parts * lines;
    l.own_blocks = (int64_t)requests * c.kv_heads * ((group + kHeads - 1) / kHeads) * l.own_parts;
    l.alone = l.own_blocks >= 4 * cus;
    if (l.alone) l.own_blocks = (l.own_blocks + kWaves - 1) / kWaves;
    l.bytes = (size_t)part_rows(cus, requests, groups, group, c.kv_heads, tokens, own) * (c.head_dim + 2) * sizeof(float);
    return l;
}

template <int DT, bool FP8, int DP, bool FAST>
void launch_sets(int sets, unsigned grid, hipStream_t s, const SharedArgs& a)
{
    if (sets == 1) k_shared<DT, FP8, DP, FAST, 1><<<grid, kThreads, 0, s>>>(a);
    else if (sets == 2 || DP == 256) k_shared<DT, FP8, DP, FAST, 2><<<grid, kThreads, 0, s>>>(a);
    else k_shared<DT, FP8, DP, FAST, DP == 256 ? 2 : 4><<<grid, kThreads, 0, s>>>(a);
}

template <int DT, bool FP8>
void launch_dims(bool fast, int sets, unsigned grid, hipStream_t s, const SharedArgs& a)
{
    if (fast) {
        if (a.dim <= 64) launch_sets<DT, FP8, 64, true>(sets, grid, s, a);
        else if (a.dim <= 128) launch_sets<DT, FP8, 128, true>(sets, grid, s, a);
        else launch_sets<DT, FP8, 256, true>(sets, grid, s, a);
    } else {
        if (a.dim <= 64) launch_sets<DT, FP8, 64, false>(sets, grid, s, a);
        else if (a.dim <= 128) launch_sets<DT, FP8, 128, false>(sets, grid, s, a);
        else launch_sets<DT, FP8, 256, false>(sets, grid, s, a);
    }
}

int check_shared(const Device* dev, const mfh_attention_shape* shape, const mfh_kv_cache* cache, int32_t requests,
                 int32_t groups, int64_t most_shared, int64_t most_own, const char* what, Layout* l)
{
    MFH_TRY(check_attention(shape, cache, what));
    if (requests < 0) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: negative number of requests %d", what, requests);
    if (groups < 0 || groups > kMostGroups)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d groups are not within 0..%d", what, groups, kMostGroups);
    bool many = (int64_t)requests * shape->q_heads > (1 << 22);
    if (!many) {
        *l = layout(dev, *shape, *cache, requests, groups, most_shared, most_own);
        many = l->shared_blocks + l->own_blocks >= (int64_t(1) << 32) / kThreads;
    }
    if (many)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d requests of %d heads are too many for one call", what, requests,
                    shape->q_heads);
    return MFH_OK;
}

}  // namespace
}  // namespace mfh

using namespace mfh;

extern "C" {

int mfh_paged_decode_shared_workspace(const mfh_attention_shape* shape, const mfh_kv_cache* cache, int32_t requests,
                                      int32_t groups, int64_t most_shared, int64_t most_own, size_t* bytes)
{
    const char* what = "mfh_paged_decode_shared_workspace";
    const Device* dev;
    MFH_TRY(bind_device(&dev));
    Layout l;
    MFH_TRY(check_shared(dev, shape, cache, requests, groups, most_shared, most_own, what, &l));
    if (!bytes) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL result", what);
    *bytes = l.bytes;
    return MFH_OK;
}

int mfh_paged_decode_shared(const mfh_attention_shape* shape, const mfh_kv_cache* cache, int32_t requests,
                            int32_t groups, const void* q, const void* k_cache, const void* v_cache,
                            const int32_t* table, int64_t table_stride, int32_t table_width, const int32_t* starts,
                            const int32_t* shared, int64_t most_shared, const int32_t* lengths, int64_t most_own,
                            const float* slopes, void* out, float* lse, void* workspace, size_t workspace_bytes,
                            void* stream)
{
    const char* what = "mfh_paged_decode_shared";
    const Device* dev;
    MFH_TRY(bind_device(&dev));
    Layout l;
    MFH_TRY(check_shared(dev, shape, cache, requests, groups, most_shared, most_own, what, &l));
    if (table_width < 0 || table_stride < table_width)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: table width %d does not fit its stride %lld", what, table_width,
                    (long long)table_stride);
    if (requests == 0) return MFH_OK;
    if (!q || !out || !k_cache || !v_cache || !lengths || (table_width > 0 && !table) || (groups > 0 && (!starts || !shared)))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL buffer", what);
    if (workspace_bytes < l.bytes || !workspace || (uintptr_t)workspace % 16)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: a workspace of %zu bytes is NULL, not 16-byte aligned or less than %zu",
                    what, workspace_bytes, l.bytes);
    SharedArgs a{};
    a.pages = PageArgs(*cache, k_cache, v_cache, table, table_stride, table_width);
    a.q = (const char*)q, a.out = (char*)out, a.lse = lse;
    a.lengths = lengths, a.starts = starts, a.shared = shared, a.slopes = slopes;
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
    a.window = shape->window, a.kv_heads = cache->kv_heads, a.q_heads = shape->q_heads;
    a.group = shape->q_heads / cache->kv_heads;
    a.head_groups = (a.group + kHeads - 1) / kHeads;
    a.dim = cache->head_dim;
    a.requests = (mfh_u32)requests, a.groups = (mfh_u32)groups, a.group_step = (mfh_u32)(groups + 63) / 64;
    a.shared_blocks = (mfh_u32)l.shared_blocks;
    a.shared_parts = l.shared_parts, a.own_parts = l.own_parts, a.parts = l.shared_parts + l.own_parts;
    a.part_out = (float*)workspace;
    a.part_sum = (float2*)(a.part_out + (int64_t)requests * a.q_heads * a.parts * a.dim);
    a.by_group = Divider((mfh_u32)a.group), a.by_kv_parts = Divider(std::max(l.kv_parts, 1u));
    a.by_shared_parts = Divider(std::max(a.shared_parts, 1u)), a.by_own_parts = Divider(a.own_parts);
    a.by_kv_heads = Divider((mfh_u32)a.kv_heads), a.by_head_groups = Divider((mfh_u32)a.head_groups);
    a.by_shared_piece = Divider(l.shared_piece), a.by_own_piece = Divider(l.own_piece), a.by_q_heads = Divider((mfh_u32)a.q_heads);
    hipStream_t s = (hipStream_t)stream;
    // whole groups of 16 tokens, and dwords for buffer loads
    const bool fast = cache->page_size % 16 == 0 &&
                      ((uintptr_t)k_cache | (uintptr_t)v_cache | a.pages.page_bytes | a.pages.head_bytes | a.pages.token_bytes) % 4 == 0;
    const bool fp8 = cache->dtype == kF8E4M3;
    const unsigned grid = (unsigned)(l.shared_blocks + l.own_blocks);
    a.all_parts = l.prefill, a.alone = l.alone;
    if (l.prefill)
        MFH_TRY(prefill_shared(*shape, *cache, a.pages, requests, groups, q, starts, shared, lengths, slopes, l.shared_parts, a.parts,
                               a.part_out, a.part_sum, s));
    if (shape->dtype == kBFloat16) {
        if (fp8) launch_dims<kBFloat16, true>(fast, l.sets, grid, s, a);
        else launch_dims<kBFloat16, false>(fast, l.sets, grid, s, a);
    } else {
        if (fp8) launch_dims<kFloat16, true>(fast, l.sets, grid, s, a);
        else launch_dims<kFloat16, false>(fast, l.sets, grid, s, a);
    }
    MFH_TRY(launch_status("k_shared"));
    const mfh_u32 few = (mfh_u32)(4 * dev->compute_units);
    if (shape->dtype == kBFloat16) launch_join<kBFloat16>(a, few, s);
    else launch_join<kFloat16>(a, few, s);
    return launch_status("k_shared_join");
}

}  // extern "C"
