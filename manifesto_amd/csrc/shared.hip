// shared.hip — attention of one new token per request over a paged cache, where
// the requests of a group have their first tokens in common
// (mfh_paged_decode_shared).
//
// As decode.hip, with the shared tokens' keys and values read once for all of a
// group: a column of the matrix products is then a query head of any of the
// group's requests, and a workgroup takes 16, 32 or 64 of them.  Below some 64
// columns bytes bound it, above the matrix units and the exponentials beside
// them.  A request's own tokens are a group of one request.  Both kinds of
// parts run in one launch, the shared ones first, and a second one joins them.
//
// A wave takes tiles of 32 tokens on its own, from memory straight into the
// matrix operands (decode.hpp); V is turned once for all columns.  Columns see
// different tokens (a window, a request shorter than its group's shared
// tokens), so that a value that is not finite may be seen by some only: it is
// cut to zero in the product and added to those columns by itself.
#include "decode.hpp"

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
    mfh_u32 lines;                         // columns in 16, 32 or 64, of all groups, at most
    mfh_u32 shared_blocks;
    mfh_u32 shared_parts, own_parts, parts, shared_piece, own_piece;  // piece: tiles of a part
    Divider by_group, by_lines, by_shared_parts, by_own_parts, by_kv_heads, by_head_groups, by_shared_piece, by_own_piece, by_q_heads;
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
    MFH_DEV void of(const SharedArgs& a, mfh_u32 g, int lane)
    {
        begin = uniform((mfh_u32)min(max(a.starts[g], 0), (int)a.requests));
        members = uniform((mfh_u32)min(max(a.starts[g + 1], (int)begin), (int)a.requests)) - begin;
        length = uniform(limited(a, a.shared[g]));
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
        auto upto = [&](mfh_u32 g, mfh_u32 end) {
            return (mfh_u32)__popcll(__ballot(g < end && a.starts[min(g, a.groups)] <= (int64_t)r));
        };
        mfh_u32 found = upto(lane * a.group_step, a.groups);
        if (found == 0) return;
        mfh_u32 g = (found - 1) * a.group_step;
        if (a.group_step > 1) {
            found = upto(g + lane, min(g + a.group_step, a.groups));
            if (found == 0) return;
            g += found - 1;
        }
        if ((int64_t)a.starts[g + 1] > (int64_t)r) of(a, g, lane);
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
// columns column0 .. of `members` requests from `request0` on.
template <int DT, bool FP8, int DP, bool FAST, int SETS>
struct Part {
    static constexpr int kSteps = DP / 32;                    // of the product with K
    static constexpr int kLoads = FP8 ? kSteps / 2 : kSteps;  // of 16 bytes of a token of K
    static constexpr int kSets = DP == 64 ? 1 : DP / 128;     // of 16 lanes' dims in V
    static constexpr int kDims = DP == 64 ? 4 : 8;            // of a lane in a set
    static constexpr int kBytes = FP8 ? 1 : 2;
    static constexpr int kSetDims = 16 * kDims;
    typedef typename Piece<FP8, kDims>::type VPiece;
    // The queries of several sets leave no registers for the rest: they are read from
    // LDS in each tile.
    static constexpr bool kQueriesInLds = SETS > 1;
    // Shared tokens are read by several workgroups where their columns fill more than
    // one: nt would keep them out of the L2.
    static constexpr int kPolicy = SETS > 1 ? 0 : kStreamed;
    struct Lds {
        u32x4 q[kQueriesInLds ? SETS * kSteps : 1][64];
        float ref[kWaves][kHeads], sum[kWaves][kHeads];
        float out[kWaves][kHeads][kSetDims + 4];
    };

    static MFH_DEV void run(const SharedArgs& a, Lds& lds, mfh_u32 request0, mfh_u32 members, mfh_u32 column0, mfh_u32 kv,
                            const Seen& seen, mfh_u32 table_row, mfh_u32 begin, mfh_u32 end, mfh_u32 slot)
    {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int col = lane & 15, quad = lane >> 4;
        const mfh_u32 columns = members * a.group;

        // This lane's columns: their queries, and the tokens they see.
        u32x4 q[kQueriesInLds ? 1 : SETS][kSteps];
        float slope[SETS];
        mfh_u32 its_first[SETS], its_length[SETS];
        mfh_u32 all_first = 0, all_length = ~0u;
        auto dim_of = [&](int s) { return FP8 ? 64 * (s / 2) + 16 * quad + 8 * (s & 1) : 32 * s + 8 * quad; };
#pragma unroll
        for (int n = 0; n < SETS; n++) {
            const mfh_u32 c = column0 + 16 * n + col;
            const bool real = c < columns;
            const mfh_u32 member = a.by_group.quotient(real ? c : 0), head = kv * a.group + ((real ? c : 0) - member * a.group);
            const mfh_u32 r = request0 + member;
            its_length[n] = length_of(a, r);
            its_first[n] = first_of(a, its_length[n]);
            if (real) all_first = max(all_first, its_first[n]), all_length = min(all_length, its_length[n]);
            slope[n] = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; s++) {
                const int d = dim_of(s);
                if (kQueriesInLds && n % kWaves != wave) continue;
                u32x4 x = {0, 0, 0, 0};
                if (real && d < a.dim) x = load16<false>(a.q + ((int64_t)r * a.q_t + (int64_t)head * a.q_h + d) * 2);
                if constexpr (kQueriesInLds) lds.q[n * kSteps + s][lane] = x;
                else q[n][s] = x;
            }
        }
        if (kQueriesInLds) __syncthreads();
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) {
            all_first = max(all_first, (mfh_u32)__shfl_xor((int)all_first, x));
            all_length = min(all_length, (mfh_u32)__shfl_xor((int)all_length, x));
        }
        all_first = uniform(all_first), all_length = uniform(all_length);

        const mfh_u32 token_bytes = a.pages.token_bytes;
        // Lanes past head_dim have zeros in Q and in K: buffer loads past every page's
        // end give them, else they read its last dims again, inside the row, and
        // are cut.  In V they do so too, their results are not written.
        mfh_u32 k_lane[kLoads], v_lane[kSets];
#pragma unroll
        for (int s = 0; s < kLoads; s++) {
            const int d = FP8 ? 64 * s + 16 * quad : 32 * s + 8 * quad, last = a.dim - 16 / kBytes;
            k_lane[s] = FAST ? d <= last ? col * token_bytes + d * kBytes : 1u << 31 : min(d, last) * kBytes;
        }
#pragma unroll
        for (int u = 0; u < kSets; u++)
            v_lane[u] = (FAST ? 4 * quad * token_bytes : 0) + min(u * kSetDims + kDims * col, a.dim - kDims) * kBytes;
        const bool ragged = a.dim != DP;
        // (read as scalars)
        typedef const __attribute__((address_space(4))) int32_t* Table;
        const Table table = (Table)(uintptr_t)(a.pages.table + (int64_t)table_row * a.pages.table_stride);
        const char* k_base = a.pages.k + kv * a.pages.head_bytes;
        const char* v_base = a.pages.v + kv * a.pages.head_bytes;

        // One tile's registers: the next tile's keys set out when this one's scores
        // are there, its values when this one's are used up.
        Pages<FAST> pages;
        u32x4 k[2][kLoads];
        VPiece v[kSets][8];
        auto load_k = [&](const TileAt<FAST>& at) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if constexpr (FAST) {
                    const __amdgpu_buffer_rsrc_t rows = page_buffer(k_base, at.page[h], a.pages);
#pragma unroll
                    for (int s = 0; s < kLoads; s++) k[h][s] = buffer_piece<u32x4, kPolicy>(rows, k_lane[s], at.in_page[h]);
                } else {
                    const char* row = k_base + shuffle64(at.mine, 16 * h + col);
#pragma unroll
                    for (int s = 0; s < kLoads; s++) k[h][s] = load16<kPolicy == kStreamed>(row + k_lane[s]);
                }
            }
        };
        auto load_v = [&](const TileAt<FAST>& at) {
            if constexpr (FAST) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const __amdgpu_buffer_rsrc_t rows = page_buffer(v_base, at.page[h], a.pages);
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int u = 0; u < kSets; u++)
                            v[u][4 * h + j] = buffer_piece<VPiece, kPolicy>(rows, v_lane[u], at.in_page[h] + j * token_bytes);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const char* row = v_base + shuffle64(at.mine, 16 * (j >> 2) + 4 * quad + (j & 3));
#pragma unroll
                    for (int u = 0; u < kSets; u++) v[u][j] = load_piece<VPiece, kPolicy == kStreamed>(row + v_lane[u]);
                }
            }
        };

        f32x4 acc[SETS][kSets][kDims];
        float ref[SETS], limit[SETS], sum[SETS];
#pragma unroll
        for (int n = 0; n < SETS; n++) {
            ref[n] = 0.0f, limit[n] = -INFINITY, sum[n] = 0.0f;
#pragma unroll
            for (int u = 0; u < kSets; u++)
#pragma unroll
                for (int d = 0; d < kDims; d++) acc[n][u][d] = f32x4{0, 0, 0, 0};
        }
        // The tokens of a tile from t0 on that a column sees, a bit each.
        auto sees = [&](int n, mfh_u32 t0) {
            const mfh_u32 low = its_first[n] > t0 ? min(its_first[n] - t0, 32u) : 0;
            const mfh_u32 high = its_length[n] > t0 ? min(its_length[n] - t0, 32u) : 0;
            return high > low ? (mfh_u32)(((mfh_u64)1 << high) - ((mfh_u64)1 << low)) : 0;
        };
        int q_lane = lane;
        auto scores = [&](int n, float (&x)[8]) {
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
                    u32x4 x;
                    if constexpr (kQueriesInLds) x = lds.q[n * kSteps + s][q_lane];
                    else x = q[n][s];
                    s0 = mfma16<DT>(k0, x, s0);
                    s1 = mfma16<DT>(k1, x, s1);
                }
            };
            if (!FAST && ragged) product(std::true_type{});
            else product(std::false_type{});
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = j < 4 ? s0[j & 3] : s1[j & 3];
        };
        // Scores as the softmax takes them: scaled, capped, biased, masked.
        auto shape = [&](int n, float (&x)[8], mfh_u32 t0, mfh_u32 valid, bool open) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] *= a.scale;
            if (a.cap == kNarrow) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = capped(x[j], a.cap_factor, a.cap_scaled);
            } else if (a.cap == kWide) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = wide_capped(x[j], a.cap_factor, a.cap_scaled);
            }
            if (a.slopes) {
                const int back = (int)(its_length[n] - 1) - (int)(t0 + 4 * quad);
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] -= slope[n] * (float)(back - (16 * (j >> 2) + (j & 3)));
            }
            if (!open) {
                const mfh_u32 bits = valid & sees(n, t0);
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (!(bits >> (16 * (j >> 2) + 4 * quad + (j & 3)) & 1)) x[j] = -INFINITY;
            }
        };
        // The weights of x * scale.
        auto soften = [&](float (&x)[SETS][8], float scale, u32x4 (&p)[SETS]) {
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
                    for (int n = 0; n < SETS; n++)
#pragma unroll
                        for (int u = 0; u < kSets; u++)
#pragma unroll
                            for (int d = 0; d < kDims; d++) asm volatile("" : "+a"(acc[n][u][d]));
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
                        for (int u = 0; u < kSets; u++)
#pragma unroll
                            for (int d = 0; d < kDims; d++) acc[n][u][d] *= alpha;
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
        // Cuts values to zero that are of no token (0 * NaN would be NaN) or not
        // finite; whether there are any of those.
        auto cut = [&](mfh_u32 valid) {
            bool odd = false;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const bool keep = valid >> (16 * (j >> 2) + 4 * quad + (j & 3)) & 1;
#pragma unroll
                for (int u = 0; u < kSets; u++) {
                    constexpr int kWords = sizeof(VPiece) / 4;
                    typedef mfh_u32 Words __attribute__((ext_vector_type(kWords)));
                    Words w = __builtin_bit_cast(Words, v[u][j]);
#pragma unroll
                    for (int i = 0; i < kWords; i++) {
                        mfh_u32 whole;
                        if constexpr (FP8) {
                            const mfh_u32 tops = ((w[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                            whole = tops | (tops - (tops >> 7));
                        } else {
                            const mfh_u32 tops = not_finite<DT>(w[i]);
                            whole = tops | (tops - (tops >> 15));
                        }
                        odd |= keep && whole != 0;
                        w[i] &= keep ? ~whole : 0u;
                    }
                    v[u][j] = __builtin_bit_cast(VPiece, w);
                }
            }
            return __any(odd);
        };
        auto add = [&](const u32x4 (&p)[SETS]) {
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
                    const u32x4 other = {high_halves(t[0][i], t[1][i]), high_halves(t[2][i], t[3][i]),
                                         high_halves(t[4][i], t[5][i]), high_halves(t[6][i], t[7][i])};
#pragma unroll
                    for (int n = 0; n < SETS; n++) {
                        acc[n][u][d] = mfma16<DT>(even, p[n], acc[n][u][d]);
                        acc[n][u][d + 1] = mfma16<DT>(other, p[n], acc[n][u][d + 1]);
                    }
                }
            }
        };

        auto page_of = [&](mfh_u32 t) { return (mfh_u32)table[a.pages.by_page.quotient(t)]; };

        mfh_u32 tile = begin + wave;
        bool odd = false;  // some tile had values that are not finite, and columns that do not see it
        if (tile < end) {
            pages.ask(a.pages, table, seen, tile * kTile, lane);
            TileAt<FAST> at = pages.place(a.pages, seen, tile * kTile, lane, true);
            load_k(at);
            pages.ask(a.pages, table, seen, (tile + kWaves) * kTile, lane);
            load_v(at);
            const bool simple = a.cap == kNone && !a.slopes && a.scale > 0.0f;
            // A tile that is seen whole by every column, and whose scores only need
            // their scale, goes without the other questions.  Loads of a tile past
            // the last one are made too, and move nothing: behind loads that only some
            // iterations make, the compiler waits for all that are on their way.
            auto open = [&]() {
                return at.valid == 0xffffffffu && tile * kTile >= all_first && tile * kTile + kTile <= all_length;
            };
            auto turn = [&](auto plain) {
                const mfh_u32 t0 = tile * kTile, valid = at.valid;
                const bool whole = plain.value || open();
                float x[SETS][8];
                u32x4 p[SETS];
                asm volatile("" : "+v"(q_lane));  // else all of Q is read ahead of the loop, into registers
#pragma unroll
                for (int n = 0; n < SETS; n++) scores(n, x[n]);
                at = pages.place(a.pages, seen, t0 + kWaves * kTile, lane, tile + kWaves < end);
                load_k(at);
                pages.ask(a.pages, table, seen, t0 + 2 * kWaves * kTile, lane);
                if constexpr (plain.value) {
                    soften(x, a.scale, p);
                } else {
#pragma unroll
                    for (int n = 0; n < SETS; n++) shape(n, x[n], t0, valid, whole);
                    soften(x, 1.0f, p);
                    if (!whole) odd |= cut(valid);
                }
                add(p);
                load_v(at);
                tile += kWaves;
            };
            while (tile < end) {
                while (simple && tile < end && open()) turn(std::true_type{});
                if (tile < end) turn(std::false_type{});
            }
        }
        // Those values, added to the columns that see them (here, and not in their
        // tile: what the loop holds beside the sums leaves no registers for it).
        for (tile = odd ? begin + wave : end; tile < end; tile += kWaves) {
            const mfh_u32 t0 = tile * kTile;
            const bool open = t0 >= max(all_first, seen.first) && t0 + kTile <= min(all_length, seen.length);
            bool whole = open;  // such a tile was not cut
            for (mfh_u32 i = 0; i < kTile && whole; i++) whole = page_of(t0 + i) < a.pages.pages;
            for (mfh_u32 t = max(t0, seen.first); t < min(t0 + kTile, seen.length) && !whole; t++) {
                const mfh_u32 page = page_of(t);
                if (page >= a.pages.pages) continue;
                const char* row = v_base + (mfh_u64)page * a.pages.page_bytes +
                                  (t - a.pages.by_page.quotient(t) * a.pages.by_page.d) * token_bytes;
#pragma unroll
                for (int u = 0; u < kSets; u++)
#pragma unroll
                    for (int d = 0; d < kDims; d++)
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            const int dim = u * kSetDims + kDims * (4 * quad + x) + d;
                            if (dim >= a.dim) continue;
                            mfh_u32 code;
                            if constexpr (FP8) code = e4m3_pair<DT, false>(*reinterpret_cast<const uint8_t*>(row + dim)) & 0xffffu;
                            else code = load2(row + dim * 2);
                            const float value = dec16<DT>(code);
                            if (__builtin_isfinite(value)) continue;
#pragma unroll
                            for (int n = 0; n < SETS; n++)
                                if (t >= its_first[n] && t < its_length[n]) acc[n][u][d][x] += value;
                        }
            }
        }

        // The waves' results meet, as in decode.hip.
#pragma unroll
        for (int n = 0; n < SETS; n++) {
            sum[n] += __shfl_xor(sum[n], 16);
            sum[n] += __shfl_xor(sum[n], 32);
            const float wave_ref = limit[n] == -INFINITY ? -INFINITY : ref[n];
            __syncthreads();
            if (quad == 0) lds.ref[wave][col] = wave_ref, lds.sum[wave][col] = sum[n];
            __syncthreads();
            float top = lds.ref[0][col];
#pragma unroll
            for (int w = 1; w < kWaves; w++) top = fmaxf(top, lds.ref[w][col]);
            const float weight = wave_ref == -INFINITY ? 0.0f : exp2_fast(wave_ref - top);
            const mfh_u32 first_column = column0 + 16 * n;
            const int heads = first_column < columns ? (int)min((mfh_u32)kHeads, columns - first_column) : 0;
#pragma unroll
            for (int u = 0; u < kSets; u++) {
                if (u) __syncthreads();
#pragma unroll
                for (int d = 0; d < kDims; d++)
#pragma unroll
                    for (int i = 0; i < 4; i++) lds.out[wave][col][kDims * (4 * quad + i) + d] = weight * acc[n][u][d][i];
                __syncthreads();
                const int dims = min(kSetDims, a.dim - u * kSetDims);
                for (int i = threadIdx.x; i < heads * (kSetDims / 2); i += kThreads) {
                    const int h = i / (kSetDims / 2), d = 2 * (i % (kSetDims / 2)), dim = u * kSetDims + d;
                    if (d >= dims) continue;
                    float o0 = 0.0f, o1 = 0.0f;
#pragma unroll
                    for (int w = 0; w < kWaves; w++) o0 += lds.out[w][h][d], o1 += lds.out[w][h][d + 1];
                    const mfh_u32 c = first_column + h, member = a.by_group.quotient(c);
                    const int64_t at = ((int64_t)(request0 + member) * a.q_heads + kv * a.group + (c - member * a.group)) * a.parts + slot;
                    *reinterpret_cast<float2*>(a.part_out + at * a.dim + dim) = make_float2(o0, o1);
                    if (dim == 0) {
                        float all = lds.ref[0][h], total = 0.0f;
#pragma unroll
                        for (int w = 1; w < kWaves; w++) all = fmaxf(all, lds.ref[w][h]);
#pragma unroll
                        for (int w = 0; w < kWaves; w++)
                            total += lds.ref[w][h] == -INFINITY ? lds.sum[w][h] : exp2_fast(lds.ref[w][h] - all) * lds.sum[w][h];  // 0, or NaN
                        a.part_sum[at] = make_float2(all, total);
                    }
                }
            }
        }
    }
};

// DP: head_dim rounded up to 64, 128 or 256.  SETS: of 16 columns, of the shared tokens.
template <int DT, bool FP8, int DP, bool FAST, int SETS>
__global__ __launch_bounds__(kThreads, SETS > 1 ? 1 : DP == 64 ? 3 : DP == 128 ? 2 : 1) void k_shared(SharedArgs a)
{
    typedef Part<DT, FP8, DP, FAST, SETS> Common;
    typedef Part<DT, FP8, DP, FAST, 1> Own;
    __shared__ union {
        typename Common::Lds common;
        typename Own::Lds own;
    } lds;
    const int lane = threadIdx.x & 63;
    if (blockIdx.x < a.shared_blocks) {
        // Workgroups of one head and part, which read the same keys if they are of
        // one group, are on one XCD (every eighth is), one after the other.
        const mfh_u32 eighth = blockIdx.x >> 3, high = a.by_lines.quotient(eighth), line = eighth - high * a.lines;
        const mfh_u32 kv_part = high * 8 + (blockIdx.x & 7);
        const mfh_u32 kv = a.by_shared_parts.quotient(kv_part), part = kv_part - kv * a.shared_parts;
        if (kv >= (mfh_u32)a.kv_heads) return;
        constexpr mfh_u32 kColumns = kHeads * SETS;
        mfh_u32 before = 0, g = ~0u, tile_of = 0;
        for (mfh_u32 base = 0; base < a.groups; base += 64) {
            mfh_u32 its = 0;
            if (base + lane < a.groups) {
                const int from = min(max(a.starts[base + lane], 0), (int)a.requests);
                its = ((mfh_u32)(min(max(a.starts[base + lane + 1], from), (int)a.requests) - from) * a.group + kColumns - 1) / kColumns;
            }
            const mfh_u32 upto = before + lanes_upto(its);
            const mfh_u64 past = __ballot(upto > line);
            if (past) {
                const int at = __ffsll((unsigned long long)past) - 1;
                g = base + at;
                tile_of = line - ((mfh_u32)__builtin_amdgcn_readlane((int)upto, at) - (mfh_u32)__builtin_amdgcn_readlane((int)its, at));
                break;
            }
            before = last_lane(upto);
        }
        if (g == ~0u) return;
        g = uniform(g), tile_of = uniform(tile_of);
        Group group;
        group.of(a, g, lane);
        const Tiles tiles(group, a.by_shared_piece, a.shared_parts);
        if (part >= tiles.parts) return;
        const mfh_u32 share = uniform((tiles.count + tiles.parts - 1) / tiles.parts);
        Common::run(a, lds.common, group.begin, group.members, tile_of * kColumns, kv, group, group.begin,
                    tiles.first + min(part * share, tiles.count), tiles.first + min((part + 1) * share, tiles.count), part);
        return;
    }
    const mfh_u32 block = blockIdx.x - a.shared_blocks;
    mfh_u32 rest = a.by_own_parts.quotient(block);
    const mfh_u32 part = block - rest * a.own_parts;
    const mfh_u32 line = a.by_head_groups.quotient(rest), head_group = rest - line * a.head_groups;
    const mfh_u32 r = a.by_kv_heads.quotient(line), kv = line - r * a.kv_heads;
    Group group;
    group.with(a, r, lane);
    Seen own;
    own.length = uniform(length_of(a, r));
    own.first = max(first_of(a, own.length), group.length);
    const Tiles tiles(own, a.by_own_piece, a.own_parts);
    if (part >= tiles.parts) return;
    const mfh_u32 share = uniform((tiles.count + tiles.parts - 1) / tiles.parts);
    Own::run(a, lds.own, r, 1, head_group * kHeads, kv, own, r,
             tiles.first + min(part * share, tiles.count), tiles.first + min((part + 1) * share, tiles.count),
             a.shared_parts + part);
}

// Joins a row's parts, of the shared tokens and of its own.  A workgroup takes
// 128 dims of a query head, a quarter of the parts in each wave; lanes take two
// dims each.
constexpr int kJoinWaves = 4;

template <int DT>
__global__ __launch_bounds__(64 * kJoinWaves) void k_shared_join(SharedArgs a)
{
    __shared__ float s_all[kJoinWaves];
    __shared__ float2 s_out[kJoinWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int chunks = (a.dim + 127) / 128;
    const mfh_u32 row = blockIdx.x / chunks, chunk = blockIdx.x - row * chunks;
    const mfh_u32 r = a.by_q_heads.quotient(row), head = row - r * a.q_heads;
    Group group;
    group.with(a, r, lane);
    Seen own;
    own.length = length_of(a, r);
    own.first = max(first_of(a, own.length), group.length);
    const mfh_u32 common = group.members > 0 ? Tiles(group, a.by_shared_piece, a.shared_parts).parts : 0;
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
#pragma unroll 4
    for (mfh_u32 n = wave; n < parts; n += kJoinWaves) {
        const float2 s = sums[slot(n)];
        const float2 w = *reinterpret_cast<const float2*>(from + (int64_t)slot(n) * a.dim);
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
    if (d == 0 && a.lse) a.lse[row] = all == 0.0f ? -INFINITY : top * kLn2 + logf(all);
}

struct Layout {
    int sets;
    int64_t lines, shared_blocks, own_blocks;
    mfh_u32 shared_parts, own_parts, shared_piece, own_piece;
    size_t bytes;
};

Layout layout(const Device* dev, const mfh_attention_shape& sh, const mfh_kv_cache& c, int32_t requests, int32_t groups,
              int64_t most_shared, int64_t most_own)
{
    Layout l{};
    const int group = sh.q_heads / c.kv_heads;
    const int64_t columns = (int64_t)requests * group, each = groups > 0 ? columns / groups : 0;
    l.sets = each <= 16 ? 1 : c.head_dim > 128 ? 2 : 4;
    l.lines = columns / (kHeads * l.sets) + groups;
    auto split = [&](int64_t rows, int64_t tokens, mfh_u32& piece, mfh_u32& parts) {
        const int64_t tiles = (std::min<int64_t>(std::max<int64_t>(tokens, 1), kLongest) + kTile - 1) / kTile + 1;
        const int64_t wanted = std::max<int64_t>(1, 2 * dev->compute_units / std::max<int64_t>(rows, 1));
        piece = (mfh_u32)std::max<int64_t>(8, (tiles + wanted - 1) / wanted);
        parts = (mfh_u32)((tiles + piece - 1) / piece);
    };
    split(std::max<int64_t>(groups, columns / (kHeads * l.sets)) * c.kv_heads, most_shared, l.shared_piece, l.shared_parts);
    split((int64_t)requests * c.kv_heads, most_own, l.own_piece, l.own_parts);
    if (groups == 0) l.shared_parts = 0;
    l.shared_blocks = ((int64_t)c.kv_heads * l.shared_parts + 7) / 8 * 8 * l.lines;
    l.own_blocks = (int64_t)requests * c.kv_heads * ((group + kHeads - 1) / kHeads) * l.own_parts;
    l.bytes = (size_t)requests * sh.q_heads * (l.shared_parts + l.own_parts) * (c.head_dim + 2) * sizeof(float);
    return l;
}

template <int DT, bool FP8, int DP, bool FAST>
void launch_sets(int sets, unsigned grid, hipStream_t s, const SharedArgs& a)
{
    if (sets == 1) k_shared<DT, FP8, DP, FAST, 1><<<grid, kThreads, 0, s>>>(a);
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
    *l = layout(dev, *shape, *cache, requests, groups, most_shared, most_own);
    if ((int64_t)requests * shape->q_heads > (1 << 22) || l->shared_blocks + l->own_blocks >= (int64_t(1) << 32) / kThreads)
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
    a.lines = (mfh_u32)l.lines, a.shared_blocks = (mfh_u32)l.shared_blocks;
    a.shared_parts = l.shared_parts, a.own_parts = l.own_parts, a.parts = l.shared_parts + l.own_parts;
    a.part_out = (float*)workspace;
    a.part_sum = (float2*)(a.part_out + (int64_t)requests * a.q_heads * a.parts * a.dim);
    a.by_group = Divider((mfh_u32)a.group), a.by_lines = Divider(std::max(a.lines, 1u));
    a.by_shared_parts = Divider(std::max(a.shared_parts, 1u)), a.by_own_parts = Divider(a.own_parts);
    a.by_kv_heads = Divider((mfh_u32)a.kv_heads), a.by_head_groups = Divider((mfh_u32)a.head_groups);
    a.by_shared_piece = Divider(l.shared_piece), a.by_own_piece = Divider(l.own_piece), a.by_q_heads = Divider((mfh_u32)a.q_heads);
    hipStream_t s = (hipStream_t)stream;
    // whole groups of 16 tokens, and dwords for buffer loads
    const bool fast = cache->page_size % 16 == 0 &&
                      ((uintptr_t)k_cache | (uintptr_t)v_cache | a.pages.page_bytes | a.pages.head_bytes | a.pages.token_bytes) % 4 == 0;
    const bool fp8 = cache->dtype == kF8E4M3;
    const unsigned grid = (unsigned)(l.shared_blocks + l.own_blocks);
    if (shape->dtype == kBFloat16) {
        if (fp8) launch_dims<kBFloat16, true>(fast, l.sets, grid, s, a);
        else launch_dims<kBFloat16, false>(fast, l.sets, grid, s, a);
    } else {
        if (fp8) launch_dims<kFloat16, true>(fast, l.sets, grid, s, a);
        else launch_dims<kFloat16, false>(fast, l.sets, grid, s, a);
    }
    MFH_TRY(launch_status("k_shared"));
    const unsigned joins = (unsigned)((int64_t)requests * a.q_heads * ((a.dim + 127) / 128));
    if (shape->dtype == kBFloat16) k_shared_join<kBFloat16><<<joins, 64 * kJoinWaves, 0, s>>>(a);
    else k_shared_join<kFloat16><<<joins, 64 * kJoinWaves, 0, s>>>(a);
    return launch_status("k_shared_join");
}

}  // extern "C"
