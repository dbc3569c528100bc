// prefill.hip — attention of each request's new tokens over a paged cache
// (mfh_paged_prefill): causal, with an optional window, prefix, cap and bias.
//
// 4 * pairs * q_heads * head_dim operations over keys and values that stay in
// the caches near the cores: the matrix units bound it, and beside them the
// exponentials and what else is done to each score.  The rows of one key-value
// head are its query heads of all new tokens (row = token * group + head of the
// group), so that heads which share keys share a workgroup's key tiles too.  A
// wave has 32 rows and walks over tiles of 64 keys (32 for heads wider than
// 128) in LDS:
//
//   scores^T [keys][rows] = K Q^T      Q stays in registers, K as it stands in LDS
//   out^T [dims][rows] += V^T P^T      V^T by LDS reads that transpose
//
// A lane holds the scores of row lane % 32 for keys 8 * (i / 4) + 4 * (lane / 32)
// + i % 4; eight of them, in that order, are the second product's P^T operand,
// so weights never leave their lane, and a row's maximum is one exchange between
// two lanes.  The running reference is decode.hip's.
//
// A workgroup has eight waves in two groups of four, one of each group on a
// SIMD, a barrier apart: while one wave multiplies, the other one turns its
// scores into weights and puts the next tile into LDS.  The tile's pieces wait
// in registers meanwhile, and 8-bit caches become 16-bit on the way.
//
// One prompt of 8192 tokens, 32 heads over 8 of 128, bf16: 575 to 650 us from card
// to card (mostly 590, 932 TFLOP/s), 850 to 956 TFLOP/s of the 1360 that a large
// matrix product reaches; by workgroups of four waves 890 us.
#include "paged.hpp"

#include <cfloat>

namespace mfh {
namespace {

// Waves of a workgroup, 32 rows each, where rows fill the card: two a SIMD if their registers allow it.
constexpr int waves_of(int dim) { return dim <= 128 ? 8 : 4; }
constexpr int keys_of(int dim) { return dim <= 128 ? 64 : 32; }  // of a tile

struct PrefillArgs {
    PageArgs pages;
    const char* q;
    char* out;
    float* lse;
    const int32_t* starts;
    const int32_t* lengths;
    const int32_t* prefix;
    const float* slopes;
    int64_t q_t, q_h, out_t, out_h;  // elements
    int64_t tokens, most_fresh;
    float scale, cap_factor, cap_scaled, v_scale;  // cap_factor: `twice` with the scale in it, or `scaled_inverse`
    float* part_out;   // [tokens * q_heads][parts][head_dim]
    float2* part_sum;  // [tokens * q_heads][parts]: reference and sum
    int32_t window, kv_heads, q_heads, group, dim;
    mfh_u32 row_tiles;  // of a request and head at most
    mfh_u32 parts;      // of a row's keys
    mfh_u32 part_slots; // of a row in part_out: `parts`, or more
    mfh_u32 step_entries, step_bytes;  // a tile's keys in whole pages, and in bytes of a page
    Divider by_group, by_kv_heads, by_row_tiles, by_parts, by_q_heads;
};

// Where 16 bytes of a row stand among the row's pieces in LDS.  Rows have no gaps
// (with them two workgroups of heads of 64 would not fit a CU's LDS), so pieces
// change places by row: 16 rows of one piece, as K is read, lie in 16 different
// places, and four rows of four pieces, as V is, too.  Counted: no bank conflicts.
template <int PIECES>
MFH_DEV int place(int row, int piece)
{
    return piece ^ (((row & 3) << 2 | (row >> 2 & 3)) & (PIECES - 1));
}

// DP: head_dim rounded up to 64, 128 or 256.  WAVES: 4 (one group) or 8.  WIDE:
// scores have a wide cap; as a branch its code takes registers and time from calls
// without one (heads of 256 13% slower, a prompt of 512 3%).
// SHARED: a "request" is a group of requests with one new token each, whose keys are
// the tokens that they have in common (mfh_paged_decode_shared): starts are those of
// the groups, `prefix` holds the shared tokens, lengths are those of the requests;
// the pages are the first request's, and results are parts.
template <int DT, bool FP8, int DP, int WAVES, bool WIDE, bool SHARED>
__global__ __launch_bounds__(64 * WAVES, WAVES / 4) void k_prefill(PrefillArgs a)
{
    constexpr int kWaves = WAVES, kThreads = 64 * kWaves, kRows = 32 * kWaves;
    constexpr int kBytes = FP8 ? 1 : 2;
    constexpr int kSteps = DP / 16;
    constexpr int kDimTiles = DP / 32;
    constexpr int kKeys = keys_of(DP);
    constexpr int kBlocks = kKeys / 32;
    constexpr int kPitch = 2 * DP;
    constexpr int kPieces = DP / 8;                      // of a key, eight values each
    constexpr int kLoads = kKeys * kPieces / kThreads;   // of a thread
    constexpr int kKeyStep = kThreads / kPieces;         // keys between a thread's pieces
    typedef typename std::conditional<FP8, u32x2, u32x4>::type Raw;
    __shared__ __align__(16) char s_k[3][kKeys * kPitch], s_v[3][kKeys * kPitch];
    __shared__ __align__(16) char s_raw[3][kKeys * kPitch];  // V as it was, where some of it is not finite
    __shared__ int s_odd[3];                                 // the round whose V that is

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int group = wave / 4;  // of waves that multiply while the other one does the rest
    mfh_u32 at_block = blockIdx.x;
    mfh_u32 rest = a.by_parts.quotient(at_block);
    const mfh_u32 part = at_block - rest * a.parts;
    at_block = rest;
    rest = a.by_kv_heads.quotient(at_block);
    const mfh_u32 kv = at_block - rest * a.kv_heads;
    const mfh_u32 r = a.by_row_tiles.quotient(rest);
    const mfh_u32 row_tile = a.row_tiles - 1 - (rest - r * a.row_tiles);  // the longest rows first

    const int64_t begin = min(max((int64_t)a.starts[r], (int64_t)0), a.tokens);
    const int64_t end = min(max((int64_t)a.starts[r + 1], begin), a.tokens);
    const mfh_u32 fresh = (mfh_u32)(end - begin), computed = (mfh_u32)min((int64_t)fresh, a.most_fresh);
    const mfh_u32 rows = computed * a.group, row0 = row_tile * kRows;
    if (row0 >= rows) return;
    const mfh_u64 most = min((mfh_u64)a.pages.width * a.pages.by_page.d, (mfh_u64)kLongest);
    const int length = (int)min((mfh_u64)max(SHARED ? a.prefix[r] : a.lengths[r], 0), most);
    const int prefix = !SHARED && a.prefix ? min(max(a.prefix[r], 0), length) : 0;
    const int first_position = length - (int)fresh;  // of the request's new tokens; may be negative
    // Where a token of the group stands in its request, -1 without one; and the least
    // and the greatest of some.  Returns the least of those that there are.
    auto stands = [&](mfh_u32 token) {
        if constexpr (SHARED) return (int)min((mfh_u64)max(a.lengths[begin + token], 0), most) - 1;
        else return first_position + (int)token;
    };
    auto range = [&](mfh_u32 first_row, mfh_u32 last_row, int& low, int& high) {
        const mfh_u32 first = a.by_group.quotient(first_row), last = a.by_group.quotient(last_row);
        if constexpr (SHARED) {
            mfh_u32 least = kLongest;  // (-1 is the greatest number)
            high = -1;
            bool ended = false;
            for (mfh_u32 t = first + lane; t <= last; t += 64) {
                const int at = stands(t);
                least = min(least, (mfh_u32)at), high = max(high, at), ended |= at < 0;
            }
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) least = min(least, (mfh_u32)__shfl_xor((int)least, x)), high = max(high, __shfl_xor(high, x));
            high = (int)uniform((mfh_u32)high);
            low = __any(ended) ? -1 : (int)uniform(least);
            return (int)uniform(least);
        } else {
            low = stands(first), high = stands(last);
            return low;
        }
    };

    const int32_t* table = a.pages.table + (SHARED ? begin : (int64_t)r) * a.pages.table_stride;
    const char* k_base = a.pages.k + kv * a.pages.head_bytes;
    const char* v_base = a.pages.v + kv * a.pages.head_bytes;

    // Positions of the workgroup's rows, and the keys any of them sees.
    int low_position, high_position;
    const int least_position = range(row0, min(row0 + kRows, rows) - 1, low_position, high_position);
    const int key_end = min(max(high_position + 1, prefix), length);
    const int window_first = a.window > 0 ? max(least_position - a.window + 1, 0) : 0;  // below: the prefix only
    // The next tile at or after `tile` that has a key for some row: between the
    // prefix and the window there is none.
    auto next_tile = [&](int tile) {
        return tile * kKeys >= prefix ? max(tile, window_first / kKeys) : tile;
    };
    // this part's tiles
    const int all_tiles = key_end > 0 ? (key_end + kKeys - 1) / kKeys : 0, first_tile = min(next_tile(0), all_tiles);
    const int share = (int)a.by_parts.quotient((mfh_u32)(all_tiles - first_tile) + a.parts - 1);
    const int tile_end = min(first_tile + (int)(part + 1) * share, all_tiles);

    // This lane's row, and its wave's.
    const mfh_u32 row = row0 + 32 * wave + col;
    const bool real = row < rows;
    const mfh_u32 token = a.by_group.quotient(min(row, rows - 1));
    const mfh_u32 head = kv * a.group + (min(row, rows - 1) - token * a.group);
    const int position = stands(token);
    int wave_low, wave_high;
    range(min(row0 + 32 * wave, rows - 1), min(row0 + 32 * wave + 31, rows - 1), wave_low, wave_high);

    u32x4 q[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; s++) {
        const int d = 16 * s + 8 * half;
        q[s] = u32x4{0, 0, 0, 0};
        if (real && d < a.dim) q[s] = load16<false>(a.q + ((begin + token) * a.q_t + head * a.q_h + d) * 2);
    }
    float slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
    // Q is waited for here: at its first use in the loop the compiler would wait for
    // all loads on its account, those of the next tiles among them, in every round.
#pragma unroll
    for (int s = 0; s < kSteps; s++) asm volatile("" : "+v"(q[s]));
    asm volatile("" : "+v"(slope));

    f32x16 acc[kDimTiles];
#pragma unroll
    for (int d = 0; d < kDimTiles; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[d][i] = 0.0f;
    float ref = 0.0f, limit = -INFINITY;
    // Of the tiles' sums: in f32 a thousand small ones beside a large weight were off by
    // 2^-15 together (their roundings can all go one way); in f64 0.3% of the time.
    double total = 0.0;

    // ---- staging: thread t takes the piece that belongs in place t % kPieces of
    // keys t / kPieces + i * kKeyStep, and follows these keys from tile to tile:
    // their places in the table and, in bytes, in their pages.
    const int key0 = threadIdx.x / kPieces, slot = threadIdx.x % kPieces;
    struct Tile {
        int index;
        bool open;   // every row of the workgroup sees every key
    };
    struct Keys {
        mfh_u32 entry[kLoads], in_page[kLoads];
        int32_t page[kLoads];
    };
    const mfh_u32 last_entry = length > 0 ? a.pages.by_page.quotient((mfh_u32)length - 1) : 0;
    const mfh_u32 page_size_bytes = a.pages.by_page.d * a.pages.token_bytes;
    auto ask = [&](Keys& keys) {  // past the length its last page again
#pragma unroll
        for (int i = 0; i < kLoads; i++) keys.page[i] = table[min(keys.entry[i], last_entry)];
    };
    auto go_to = [&](Keys& keys, int tile) {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const mfh_u32 t = (mfh_u32)(tile * kKeys) + key0 + i * kKeyStep;
            keys.entry[i] = a.pages.by_page.quotient(t);
            keys.in_page[i] = (t - keys.entry[i] * a.pages.by_page.d) * a.pages.token_bytes;
        }
    };
    auto go_on = [&](Keys& keys) {  // by a tile
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const mfh_u32 in_page = keys.in_page[i] + a.step_bytes;
            // (a page of one token has no bytes to go on by, and no use for them)
            const bool over = a.pages.token_bytes > 0 && in_page >= page_size_bytes;
            keys.in_page[i] = over ? in_page - page_size_bytes : in_page;
            keys.entry[i] += a.step_entries + (over ? 1 : 0);
        }
    };
    bool clean = true;  // every page of the request is one of the cache's
    auto there = [&](int key) {
        bool is = key < length;
        if (!clean) is &= (mfh_u32)table[min(a.pages.by_page.quotient((mfh_u32)key), last_entry)] < a.pages.pages;
        return is;
    };
    auto describe = [&](int tile) {
        const int first = tile * kKeys;
        const bool past = first + kKeys <= low_position + 1 && (a.window <= 0 || first > high_position - a.window);
        return Tile{tile, clean && first + kKeys <= length && (past || first + kKeys <= prefix)};
    };
    // This thread's pieces of the tile.
    auto locate = [&](const Keys& keys, int64_t (&from)[kLoads]) {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const mfh_u32 page = (mfh_u32)keys.page[i] < a.pages.pages ? (mfh_u32)keys.page[i] : 0u;
            const int piece = place<kPieces>(key0 + i * kKeyStep, slot);
            from[i] = (int64_t)((mfh_u64)page * (mfh_u64)a.pages.page_bytes) +
                      (keys.in_page[i] + (piece * 8 < a.dim ? piece * 8 * kBytes : 0));
        }
    };

    // Pieces wait in registers while the vector units are busy with the scores,
    // and go to LDS from there, 8-bit ones widened on the way.  (Loads straight
    // into LDS took longer: a wave stands still for 200 cycles at each of them.)
    auto fetch = [&](const int64_t (&from)[kLoads], const char* base, Raw (&raw)[kLoads]) {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            if constexpr (FP8) raw[i] = load8<false>(base + from[i]);
            else raw[i] = load16<false>(base + from[i]);
        }
    };
    // A masked weight of 0 times a value that is not finite would be NaN.  Where
    // a mask cuts a tile that has such values, they are zeros in the product
    // and are kept aside for the rows that see them.
    auto put = [&](const Tile& w, auto plain, char* to, char* aside, const Raw (&raw)[kLoads]) {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const int key = key0 + i * kKeyStep;
            u32x4 x;
            if constexpr (FP8)
                x = u32x4{e4m3_pair<DT, false>(raw[i][0]), e4m3_pair<DT, true>(raw[i][0]),
                          e4m3_pair<DT, false>(raw[i][1]), e4m3_pair<DT, true>(raw[i][1])};
            else x = raw[i];
            if (!plain.value && (!w.open || a.dim != DP)) {
                bool keep = place<kPieces>(key, slot) * 8 < a.dim;
                keep &= there(w.index * kKeys + key);
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] &= keep ? ~0u : 0u;
            }
            if (!plain.value && aside && !w.open) {
                *reinterpret_cast<u32x4*>(aside + key * kPitch + slot * 16) = x;
                mfh_u32 tops[4];
#pragma unroll
                for (int j = 0; j < 4; j++) tops[j] = not_finite<DT>(x[j]);
                if ((tops[0] | tops[1] | tops[2] | tops[3]) != 0) {
                    odd = true;
#pragma unroll
                    for (int j = 0; j < 4; j++) x[j] &= ~(tops[j] | (tops[j] - (tops[j] >> 15)));  // whole halves
                }
            }
            *reinterpret_cast<u32x4*>(to + key * kPitch + slot * 16) = x;
        }
        return odd;
    };
    // ---- what a row sees
    // Score i of block b is of key 32 b + 4 half + 8 (i / 4) + i % 4; whether this lane's row sees it:
    struct Seen {
        mfh_u32 there;
        int back, oldest, in_prefix;
        __device__ bool operator()(int c) const  // (no short cuts: branches cost more than the comparisons)
        {
            return ((there >> c & 1) != 0) & (((c <= back) & (c > oldest)) | (c < in_prefix));
        }
    };
    auto seen_from = [&](int key, mfh_u32 there) {
        return Seen{there, position - key, a.window > 0 ? position - key - a.window : -kKeys, prefix - key};
    };
    auto add_odd = [&](const char* aside, const Tile& w) {
        const Seen seen = seen_from(w.index * kKeys, 0);
        for (int key = 0; key < kKeys; key++) {
            const bool see = there(w.index * kKeys + key) &
                             (((key <= seen.back) & (key > seen.oldest)) | (key < seen.in_prefix));
#pragma unroll
            for (int d = 0; d < kDimTiles; d++) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int dim = 32 * d + 8 * (i / 4) + 4 * half + i % 4;
                    const mfh_u32 v = *reinterpret_cast<const mfh_u16*>(
                        aside + key * kPitch + place<kPieces>(key, dim / 8) * 16 + dim % 8 * 2);
                    if (see & (not_finite<DT>(v) != 0)) acc[d][i] += dec16<DT>(v);
                }
            }
        }
    };

    // ---- the products and what lies between them
    f32x16 s[kBlocks];
    u32x4 p[2 * kBlocks];
    // K of step d (16 dims) for the tile's blocks of 32 keys, and V^T of 16 keys
    // and 32 dims: in 16 lanes row lane % 16 / 4 of four keys, columns 4 (lane % 4) ..
    auto k_piece = [&](const char* k_from, int d, int b) {
        const int key = 32 * b + col;
        return *reinterpret_cast<const u32x4*>(k_from + key * kPitch + place<kPieces>(key, 2 * d + half) * 16);
    };
    auto v_piece = [&](const char* v_from, int n) {
        const int j = n / kDimTiles, d = n % kDimTiles;
        auto column = [&](int key) {
            const int at_key = key + 4 * half + (lane & 15) / 4, piece = 4 * d + 2 * (lane >> 4 & 1) + (lane & 3) / 2;
            return read_column(v_from + at_key * kPitch + place<kPieces>(at_key, piece) * 16 + 8 * (lane & 1));
        };
        const u32x2 lo = column(16 * j), hi = column(16 * j + 8);
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    // Scores of a tile and the weights of the one before times its V.  Reads of
    // LDS run kAhead products ahead of their use, in this order: left to itself
    // the compiler reads right ahead of each product and waits there.
    constexpr int kScores = kSteps * kBlocks, kWeights = kDimTiles * 2 * kBlocks, kAhead = 5;
    auto products = [&](const char* __restrict__ k_from, const char* __restrict__ v_from, auto with_scores) {
        constexpr int kFirst = with_scores.value ? 0 : kScores;
        u32x4 piece[kScores + kWeights];
        auto read = [&](int n) {
            if (n < kScores) piece[n] = k_piece(k_from, n / kBlocks, n % kBlocks);
            else if (n < kScores + kWeights) piece[n] = v_piece(v_from, n - kScores);
        };
        if constexpr (with_scores.value) {
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) s[b][i] = 0.0f;
        }
#pragma unroll
        for (int n = kFirst; n < kFirst + kAhead; n++) read(n);
#pragma unroll
        for (int n = kFirst; n < kScores + kWeights; n++) {
            read(n + kAhead);
            __builtin_amdgcn_sched_barrier(0);
            if (n < kScores) s[n % kBlocks] = mfma32<DT>(piece[n], q[n / kBlocks], s[n % kBlocks]);
            else acc[(n - kScores) % kDimTiles] =
                mfma32<DT>(piece[n], p[(n - kScores) / kDimTiles], acc[(n - kScores) % kDimTiles]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    const bool whole = a.slopes || !(a.scale > 0.0f), optional = a.cap_scaled != 0.0f || whole;
    auto soften = [&](const Tile& w, auto plain) {
        const int key_first = w.index * kKeys;
        const int key_behind = key_first + kKeys;
        const bool past = key_behind <= wave_low + 1 && (a.window <= 0 || key_first > wave_high - a.window);
        const bool all = w.open || (clean && key_behind <= length && (past || key_behind <= prefix));
        // What makes the scores of what s holds: s * scale + offset.  With a cap, s
        // becomes -1 / (1 + e^2y), whose double and 1 are tanh y: two operations for a
        // score fewer than tanh and the scale one after the other (a prompt of 8192,
        // capped: 786 us, so 858).
        float scale = a.scale, offset = 0.0f;
        if (!plain.value || optional) {
            // past the prefix a band of positions, for a row's own is below the length (of shared
            // tokens it may be behind): one comparison a score (a window of 512 over 4096: 119
            // us, so 130)
            const bool band = clean && key_first >= prefix && (!SHARED || key_behind <= length);
            const mfh_u32 width = a.window > 0 ? (mfh_u32)a.window : 1u << 31;
            mfh_u64 mask = 0;   // bit i: key i is there
            if (!plain.value && !all && !band) mask = __ballot(there(key_first + lane));
            if constexpr (WIDE) {
#pragma unroll
                for (int b = 0; b < kBlocks; b++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        s[b][i] = wide_capped(s[b][i] * a.scale, a.cap_factor, a.cap_scaled);
                        asm volatile("" : "+v"(s[b][i]));  // one after the other: registers are short
                    }
                scale = 1.0f;
            } else if (a.cap_scaled != 0.0f) {
#pragma unroll
                for (int b = 0; b < kBlocks; b++)
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        s[b][i] = -__builtin_amdgcn_rcpf(1.0f + exp2_fast(s[b][i] * a.cap_factor));
                scale = 2.0f * a.cap_scaled, offset = a.cap_scaled;
            }
            if (whole) {
#pragma unroll
                for (int b = 0; b < kBlocks; b++)
#pragma unroll
                    for (int i = 0; i < 16; i++) s[b][i] = __builtin_fmaf(s[b][i], scale, offset);
                scale = 1.0f, offset = 0.0f;
            }
#pragma unroll
            for (int b = 0; b < kBlocks; b++) {
                const Seen seen = seen_from(key_first + 32 * b + 4 * half, (mfh_u32)(mask >> (32 * b)) >> (4 * half));
                if (a.slopes) {
                    const float back = (float)seen.back;
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        s[b][i] = __builtin_fmaf(-slope, fabsf(back - (float)(8 * (i / 4) + i % 4)), s[b][i]);
                }
                if (!plain.value && !all) {
                    if (band) {
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const mfh_u32 distance = (mfh_u32)(seen.back - (8 * (i / 4) + i % 4));
                            s[b][i] = distance < width ? s[b][i] : -INFINITY;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; i++) s[b][i] = seen(8 * (i / 4) + i % 4) ? s[b][i] : -INFINITY;
                    }
                }
            }
        }
        float tops[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};  // (four chains, here and for the sum)
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) tops[i / 4] = fmaxf(tops[i / 4], s[b][i]);
        float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        top = __builtin_fmaf(top, scale, offset);
        if (__any(top > limit)) {
            top = fmaxf(top, __shfl_xor(top, 32));
            if (top > limit) {
                // (at first there is nothing to scale but what add_odd put there)
                const float next = top - kBelow<DT, FP8>;
                const float alpha = limit == -INFINITY ? 1.0f : exp2_fast(ref - next);
                ref = next;
                limit = top + kStep;
                total *= alpha;
#pragma unroll
                for (int d = 0; d < kDimTiles; d++) acc[d] *= alpha;
            }
        }
        const float base = offset - ref;
        float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < kBlocks; b++) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                s[b][i] = exp2_fast(__builtin_fmaf(s[b][i], scale, base));
                sums[i % 4] += s[b][i];
            }
#pragma unroll
            for (int i = 0; i < 16; i += 2) p[2 * b + i / 8][i / 2 % 4] = enc16x2<DT>(s[b][i], s[b][i + 1]);
        }
        total += (sums[0] + sums[1]) + (sums[2] + sums[3]);
    };
    auto barrier = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };

    // Round i of a wave multiplies tile i with Q and the weights of tile i - 1
    // with V, and then softens the scores of tile i, each between two barriers.
    // The second four waves run one barrier behind the first four: of the two
    // waves of a SIMD one has the matrix units while the other one has the vector
    // units.  Tiles are three deep in LDS: K of tile i + 2 and V of tile i + 1 are
    // loaded ahead of the softening and put into LDS behind it, where every wave
    // has left round i - 1's products.
    const int tile0 = next_tile(first_tile + (int)part * share);
    if (tile0 < tile_end) {
        Raw k_raw[kLoads], v_raw[kLoads];
        Keys keys;  // of the next tile whose K sets out
        int64_t from[kLoads];  // of the last tile whose K set out
        auto follow = [&](int tile) { return tile < tile_end ? next_tile(tile + 1) : tile; };
        // Tokens that are one row (a stride of 0) have no bytes to go on by either.
        const bool steady = a.pages.token_bytes > 0 || a.pages.by_page.d == 1;
        auto move = [&](int from, int to) {
            if (steady && to == from + 1) go_on(keys);
            else go_to(keys, to);
            ask(keys);
        };
        // (the second tile's K sets out with the first tile)
        const int second = follow(tile0);
        Raw second_raw[kLoads];
        Keys first_keys;
        go_to(first_keys, tile0);
        go_to(keys, second);
        ask(first_keys);
        ask(keys);
        locate(first_keys, from);
        fetch(from, k_base, k_raw);
        fetch(from, v_base, v_raw);
        locate(keys, from);
        if (second < tile_end) fetch(from, k_base, second_raw);
        // Keys of a page that is not one of the cache's are masked, and nothing
        // takes the short ways then.
        bool bad = false;
        for (mfh_u32 i = threadIdx.x; i <= last_entry; i += kThreads) bad |= (mfh_u32)table[i] >= a.pages.pages;
        clean = !__syncthreads_or(bad);
        Tile now = describe(tile0), next = describe(second), after = describe(follow(next.index)), before = now;
        if (threadIdx.x < 3) s_odd[threadIdx.x] = -1;
        for (int i = threadIdx.x * 16; i < kKeys * kPitch; i += kThreads * 16)
            *reinterpret_cast<u32x4*>(s_v[2] + i) = u32x4{0, 0, 0, 0};
        put(now, std::false_type{}, s_k[0], nullptr, k_raw);
        const bool odd0 = put(now, std::false_type{}, s_v[0], s_raw[0], v_raw);
        if (second < tile_end) put(next, std::false_type{}, s_k[1], nullptr, second_raw);
        move(next.index, after.index);
#pragma unroll
        for (int j = 0; j < 2 * kBlocks; j++) p[j] = u32x4{0, 0, 0, 0};
        int third = 0, round = 0;  // third of LDS of tile i
        __syncthreads();
        if (odd0) s_odd[0] = 0;
        __syncthreads();
        if (group == 1) barrier();
        // Rounds whose tiles follow one another and are seen whole go without the
        // questions that the others have to ask: their branches took as long as
        // the products.
        const int plain_begin = a.window > 0 ? max(high_position - a.window + kKeys, 0) / kKeys : 0;
        const int plain_end = clean && steady && a.dim == DP ? min(min(length, low_position + 1) / kKeys, tile_end) : 0;
        auto turn = [&](auto plain) {
            const int ahead = third == 2 ? 0 : third + 1, behind = third == 0 ? 2 : third - 1;
            if (!plain.value && round > 0 && !before.open && s_odd[behind] == round - 1) add_odd(s_raw[behind], before);
            __builtin_amdgcn_s_setprio(1);
            products(s_k[third], s_v[behind], std::true_type{});
            __builtin_amdgcn_s_setprio(0);
            barrier();
            const bool put_v = plain.value || next.index < tile_end, put_k = plain.value || after.index < tile_end;
            if (put_v) fetch(from, v_base, v_raw);
            if (put_k) {
                locate(keys, from);
                fetch(from, k_base, k_raw);
            }
            before = now, now = next, next = after;
            if constexpr (plain.value) {
                after.index++;
                go_on(keys);
                ask(keys);
            } else {
                after = describe(follow(after.index));
                move(next.index, after.index);
            }
            soften(before, plain);
#pragma unroll
            for (int j = 0; j < 2 * kBlocks; j++) asm volatile("" : "+v"(p[j]));  // here, not behind the barrier
            asm volatile("" : "+v"(total));
            if (put_k) put(next, plain, s_k[behind], nullptr, k_raw);
            if (put_v && put(now, plain, s_v[ahead], s_raw[ahead], v_raw)) s_odd[ahead] = round + 1;
            __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): it is in LDS
            barrier();
            third = ahead;
            round++;
        };
        while (now.index < tile_end) {
            // the tile before is whole too, or there is none
            while (now.index > plain_begin && after.index + 1 < plain_end) turn(std::true_type{});
            turn(std::false_type{});
        }
        if (group == 0) barrier();
        const int behind = third == 0 ? 2 : third - 1;
        if (!before.open && s_odd[behind] == round - 1) add_odd(s_raw[behind], before);
        products(s_k[0], s_v[behind], std::false_type{});
    }

    float sum = (float)total;
    sum += __shfl_xor(sum, 32);
    // the row's place anew: kept through the loop it costs registers there
    mfh_u32 out_at = row0 + 32 * wave + col;
    asm volatile("" : "+v"(out_at));
    if (out_at >= rows) return;
    const mfh_u32 out_token = a.by_group.quotient(out_at), out_head = kv * a.group + (out_at - out_token * a.group);
    const int64_t out_row = (begin + out_token) * a.q_heads + out_head;
    if (SHARED || a.parts > 1) {
        const int64_t at_part = out_row * a.part_slots + part;
        if (tile0 < tile_end)
#pragma unroll
        for (int d = 0; d < kDimTiles; d++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int dim = 32 * d + 8 * i + 4 * half;
                if (dim < a.dim)
                    *reinterpret_cast<f32x4*>(a.part_out + at_part * a.dim + dim) =
                        f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
            }
        }
        if (half == 0) a.part_sum[at_part] = make_float2(limit == -INFINITY ? -INFINITY : ref, sum);
        return;
    }
    const float f = sum == 0.0f ? 0.0f : a.v_scale / sum;
    char* to = a.out + ((begin + out_token) * a.out_t + out_head * a.out_h) * 2;
#pragma unroll
    for (int d = 0; d < kDimTiles; d++) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int dim = 32 * d + 8 * i + 4 * half;
            if (dim < a.dim)
                store8(to + dim * 2, u32x2{enc16x2<DT>(acc[d][4 * i] * f, acc[d][4 * i + 1] * f),
                                           enc16x2<DT>(acc[d][4 * i + 2] * f, acc[d][4 * i + 3] * f)});
        }
    }
    if (half == 0 && a.lse) a.lse[out_row] = sum == 0.0f ? -INFINITY : ref * kLn2 + logf(sum);
}

int join_lanes(int dim) { return dim <= 64 ? 16 : dim <= 128 ? 32 : 64; }

// Joins the parts of the rows that were computed.  A row takes the lanes that
// its dims need, four dims each, and the wave as many rows as fit.
template <int DT, int LANES>
__global__ __launch_bounds__(256) void k_prefill_join(PrefillArgs a, int requests)
{
    const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES;  // token * q_heads + head
    const int dim = 4 * (threadIdx.x % LANES);
    if (row >= a.tokens * a.q_heads) return;
    const mfh_u32 token = a.by_q_heads.quotient((mfh_u32)row);
    // the last request that starts at or before the token
    int lo = 0, hi = requests;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.starts[mid] <= (int64_t)token) lo = mid;
        else hi = mid;
    }
    const int64_t begin = min(max((int64_t)a.starts[lo], (int64_t)0), a.tokens);
    const int64_t end = min(max((int64_t)a.starts[lo + 1], begin), a.tokens);
    if (token < begin || token >= end || token - begin >= a.most_fresh || dim >= a.dim) return;
    const float2* sums = a.part_sum + row * a.parts;
    float top = -INFINITY;
    for (mfh_u32 n = 0; n < a.parts; n++) top = fmaxf(top, sums[n].x);
    float all = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (mfh_u32 n = 0; n < a.parts; n++) {
        const float2 s = sums[n];
        if (s.x == -INFINITY && s.y == 0.0f) continue;  // a part that saw nothing has written nothing else
        const float f = s.x == -INFINITY ? 1.0f : exp2_fast(s.x - top);
        all += f * s.y;
        o += f * *reinterpret_cast<const f32x4*>(a.part_out + (row * a.parts + n) * a.dim + dim);
    }
    const float f = all == 0.0f ? 0.0f : a.v_scale / all;
    char* to = a.out + ((int64_t)token * a.out_t + (row - (int64_t)token * a.q_heads) * a.out_h + dim) * 2;
    store8(to, u32x2{enc16x2<DT>(o[0] * f, o[1] * f), enc16x2<DT>(o[2] * f, o[3] * f)});
    if (dim == 0 && a.lse) a.lse[row] = all == 0.0f ? -INFINITY : top * kLn2 + logf(all);
}

// Workgroups of a call at most, their waves, and the parts that a row's keys are
// split into.
//
// A CU holds one workgroup (of heads of 64 two).  Rows that do not fill the card
// are split into as many parts as fit it at once: 4 tokens over 32000 keys, 8
// heads of 128 with 4 queries each, 32 parts 62 us, 48 parts 93 us, for half of
// them have to wait.  A part has eight tiles at least, or four where the join has
// little to do, at most 48 rows a CU: 8 requests, 4 tokens over 1000, whole 36.6
// us, in three parts 25.9; a prompt of 512, which is 64 rows a CU, whole 25.3 us,
// in two parts 29.4.  Rows that nearly fill the card stay whole: 3 requests of 512
// tokens over 2000 (192 workgroups) 103 us, in two parts 131.  Where workgroups
// differ in their work, for requests differ in their new tokens or a request's
// first rows see much less than its last, half as many parts again even it out: 4
// requests of up to 512 tokens over up to 7000 in two parts 171 us, whole 280; a
// prompt of 3000, 4 heads of 64, 60 and 74.
//
// Workgroups of four waves have no second group to work beside them, load every
// tile for half the rows, and are more in number.  8 heads of 128, 4 queries
// each, bf16, four waves and eight:
//   rows of a request's head that four waves hold   8 requests, 16 tokens over 2000      36 us  39 us
//   a few tiles, most of it beginning and end       64 requests of 128 tokens           154    163
//   under 25 tiles and no eight waves for every CU  1 request of 512 tokens              26     31
// and where none of this holds                      1 request of 2048 tokens             92     81
//                                                   2 requests of 1500 tokens           117     81
//                                                   2 requests, 512 tokens over 16000   413    331
struct Layout {
    int waves;
    int64_t row_tiles;
    __int128 blocks;  // of one part
    mfh_u32 parts;
    size_t bytes;
};

Layout layout(const Device* dev, const mfh_attention_shape& sh, const mfh_kv_cache& c, int32_t requests, int64_t tokens,
              int64_t most_fresh, int64_t longest)
{
    Layout l{};
    const int group = sh.q_heads / c.kv_heads;
    most_fresh = std::min(most_fresh, tokens);
    auto with_waves = [&](int waves) {
        l.waves = waves;
        l.row_tiles = (most_fresh * group + 32 * waves - 1) / (32 * waves);
        l.blocks = (__int128)l.row_tiles * c.kv_heads * requests;
    };
    // those that find rows, whatever the requests' sizes
    auto busy = [&]() {
        return std::min<__int128>(l.blocks, ((__int128)tokens * group / (32 * l.waves) + requests) * c.kv_heads);
    };
    const int64_t tiles = std::min<int64_t>(std::max<int64_t>(longest, 1), kLongest) / keys_of(c.head_dim);
    with_waves(waves_of(c.head_dim));
    const int cus = dev->compute_units;
    if (most_fresh * group <= 128 || tiles <= 4 || (tiles <= 24 && busy() < cus)) with_waves(4);
    const bool uneven = 4 * (__int128)tokens < 3 * (__int128)most_fresh * requests || most_fresh > longest / 2;
    const int64_t wanted = busy() > 0 ? (int64_t)((uneven ? 3 * cus : 2 * cus) / (2 * busy())) : 1;
    const int64_t least = tokens * sh.q_heads <= 48 * cus ? 4 : 8;  // tiles of a part
    l.parts = (mfh_u32)std::max<int64_t>(1, std::min<int64_t>({wanted, tiles / least, 64}));
    // few rows may be computed of many: the join's launch holds fewer than 2^32 threads
    if (tokens * sh.q_heads * join_lanes(c.head_dim) > (int64_t(1) << 32) - 256) l.parts = 1;
    l.bytes = l.parts > 1 ? (size_t)tokens * sh.q_heads * l.parts * (c.head_dim + 2) * sizeof(float) : 0;
    return l;
}

template <int DT, bool FP8, bool WIDE, bool SHARED>
void launch_dims(int dim, int waves, unsigned grid, hipStream_t s, const PrefillArgs& a)
{
    if (dim > 128) k_prefill<DT, FP8, 256, 4, WIDE, SHARED><<<grid, 256, 0, s>>>(a);
    else if (waves == 4 && dim <= 64) k_prefill<DT, FP8, 64, 4, WIDE, SHARED><<<grid, 256, 0, s>>>(a);
    else if (waves == 4) k_prefill<DT, FP8, 128, 4, WIDE, SHARED><<<grid, 256, 0, s>>>(a);
    else if (dim <= 64) k_prefill<DT, FP8, 64, 8, WIDE, SHARED><<<grid, 512, 0, s>>>(a);
    else k_prefill<DT, FP8, 128, 8, WIDE, SHARED><<<grid, 512, 0, s>>>(a);
}

template <int DT, bool SHARED>
void launch_form(bool fp8, bool wide, int dim, int waves, unsigned grid, hipStream_t s, const PrefillArgs& a)
{
    if (fp8 && wide) launch_dims<DT, true, true, SHARED>(dim, waves, grid, s, a);
    else if (fp8) launch_dims<DT, true, false, SHARED>(dim, waves, grid, s, a);
    else if (wide) launch_dims<DT, false, true, SHARED>(dim, waves, grid, s, a);
    else launch_dims<DT, false, false, SHARED>(dim, waves, grid, s, a);
}

// What a call's shape says, and its scores' scale and cap.
void describe(PrefillArgs& a, const mfh_attention_shape& shape, const mfh_kv_cache& cache)
{
    a.scale = shape.scale * cache.k_scale * kLog2e;
    if (shape.softcap > 0.0f) {
        a.cap_scaled = shape.softcap * kLog2e;
        a.cap_factor = shape.softcap > kWideCap ? 1.0f / a.cap_scaled : 2.0f / shape.softcap * a.scale;
        if (!__builtin_isfinite(a.cap_factor)) a.cap_factor = __builtin_copysignf(FLT_MAX, a.cap_factor);  // a score of 0 is capped at 0
    }
    a.v_scale = cache.v_scale;
    a.window = shape.window < kLongest ? shape.window : 0, a.kv_heads = cache.kv_heads, a.q_heads = shape.q_heads;
    a.group = shape.q_heads / cache.kv_heads;
    a.dim = cache.head_dim;
    const Strides qs(shape.q_token_stride, shape.q_head_stride, shape.q_heads, cache.head_dim);
    const Strides os(shape.out_token_stride, shape.out_head_stride, shape.q_heads, cache.head_dim);
    a.q_t = qs.token, a.q_h = qs.head, a.out_t = os.token, a.out_h = os.head;
    const int keys = keys_of(a.dim);
    a.step_entries = (mfh_u32)(keys / cache.page_size);
    a.step_bytes = (mfh_u32)(keys % cache.page_size) * a.pages.token_bytes;
    a.by_group = Divider((mfh_u32)a.group), a.by_kv_heads = Divider((mfh_u32)a.kv_heads);
    a.by_q_heads = Divider((mfh_u32)a.q_heads);
}

template <int DT>
void launch_join(const PrefillArgs& a, int requests, hipStream_t s)
{
    const int lanes = join_lanes(a.dim);
    const unsigned blocks = (unsigned)((a.tokens * a.q_heads * lanes + 255) / 256);
    if (lanes == 16) k_prefill_join<DT, 16><<<blocks, 256, 0, s>>>(a, requests);
    else if (lanes == 32) k_prefill_join<DT, 32><<<blocks, 256, 0, s>>>(a, requests);
    else k_prefill_join<DT, 64><<<blocks, 256, 0, s>>>(a, requests);
}

}  // namespace

int prefill_rows(int dim) { return 32 * waves_of(dim); }

int prefill_shared(const mfh_attention_shape& shape, const mfh_kv_cache& cache, const PageArgs& pages, int32_t requests,
                   int32_t groups, const void* q, const int32_t* starts, const int32_t* shared, const int32_t* lengths,
                   const float* slopes, mfh_u32 parts, mfh_u32 part_slots, float* part_out, float2* part_sum,
                   hipStream_t s)
{
    PrefillArgs a{};
    a.pages = pages;
    a.q = (const char*)q, a.starts = starts, a.prefix = shared, a.lengths = lengths, a.slopes = slopes;
    describe(a, shape, cache);
    a.tokens = a.most_fresh = requests;
    a.row_tiles = (mfh_u32)(((int64_t)requests * a.group + prefill_rows(a.dim) - 1) / prefill_rows(a.dim));
    a.parts = parts, a.part_slots = part_slots, a.part_out = part_out, a.part_sum = part_sum;
    a.by_parts = Divider(parts), a.by_row_tiles = Divider(a.row_tiles);
    const unsigned grid = (unsigned)groups * a.row_tiles * a.kv_heads * parts;
    const bool fp8 = cache.dtype == kF8E4M3, wide = shape.softcap > kWideCap;
    if (shape.dtype == kBFloat16) launch_form<kBFloat16, true>(fp8, wide, a.dim, waves_of(a.dim), grid, s, a);
    else launch_form<kFloat16, true>(fp8, wide, a.dim, waves_of(a.dim), grid, s, a);
    return launch_status("k_prefill");
}

}  // namespace mfh

using namespace mfh;

extern "C" {

int mfh_paged_prefill_workspace(const mfh_attention_shape* shape, const mfh_kv_cache* cache, int32_t requests,
                                int64_t tokens, int64_t most_fresh, int64_t longest, size_t* bytes)
{
    const char* what = "mfh_paged_prefill_workspace";
    const Device* dev;
    MFH_TRY(bind_device(&dev));
    MFH_TRY(check_attention(shape, cache, what));
    if (requests < 0 || tokens < 0 || most_fresh < 0 || tokens > kLongest)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d requests, %lld tokens, %lld of one at most", what, requests,
                    (long long)tokens, (long long)most_fresh);
    if (!bytes) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL result", what);
    *bytes = layout(dev, *shape, *cache, requests, tokens, most_fresh, longest).bytes;
    return MFH_OK;
}

int mfh_paged_prefill(const mfh_attention_shape* shape, const mfh_kv_cache* cache, int32_t requests, int64_t tokens,
                      int64_t most_fresh, const void* q, const void* k_cache, const void* v_cache,
                      const int32_t* table, int64_t table_stride, int32_t table_width, const int32_t* starts,
                      const int32_t* lengths, int64_t longest, const int32_t* prefix, const float* slopes, void* out,
                      float* lse, void* workspace, size_t workspace_bytes, void* stream)
{
    const char* what = "mfh_paged_prefill";
    const Device* dev;
    MFH_TRY(bind_device(&dev));
    MFH_TRY(check_attention(shape, cache, what));
    if (requests < 0 || tokens < 0 || most_fresh < 0 || tokens > kLongest)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d requests, %lld tokens, %lld of one at most", what, requests,
                    (long long)tokens, (long long)most_fresh);
    if (table_width < 0 || table_stride < table_width)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: table width %d does not fit its stride %lld", what, table_width,
                    (long long)table_stride);
    if (requests == 0 || tokens == 0 || most_fresh == 0) return MFH_OK;
    if (!q || !out || !k_cache || !v_cache || !starts || !lengths || (table_width > 0 && !table))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL buffer", what);
    if (workspace_bytes > 0 && (!workspace || (uintptr_t)workspace % 16))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: the workspace is NULL or not 16-byte aligned", what);
    PrefillArgs a{};
    a.pages = PageArgs(*cache, k_cache, v_cache, table, table_stride, table_width);
    a.q = (const char*)q, a.out = (char*)out, a.lse = lse;
    a.starts = starts, a.lengths = lengths, a.prefix = prefix, a.slopes = slopes;
    describe(a, *shape, *cache);
    a.tokens = tokens, a.most_fresh = std::min(most_fresh, tokens);
    Layout l = layout(dev, *shape, *cache, requests, tokens, most_fresh,
                      std::min<int64_t>(longest, (int64_t)table_width * cache->page_size));
    if (l.parts > 1) {  // as many as there is room for
        const size_t room = workspace_bytes / (l.bytes / l.parts);
        l.parts = (mfh_u32)std::max<size_t>(1, std::min<size_t>(l.parts, room));
    }
    const __int128 grid = l.blocks * l.parts;
    if (a.most_fresh * a.group > kLongest || grid >= ((int64_t)1 << 32) / (64 * l.waves))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d requests of %lld tokens and %d heads are too many for one call",
                    what, requests, (long long)a.most_fresh, shape->q_heads);
    a.row_tiles = (mfh_u32)l.row_tiles;
    a.parts = a.part_slots = l.parts, a.by_parts = Divider(l.parts);
    if (l.parts > 1) {
        a.part_out = (float*)workspace;
        a.part_sum = (float2*)(a.part_out + tokens * shape->q_heads * l.parts * a.dim);
    }
    a.by_row_tiles = Divider(a.row_tiles);
    hipStream_t s = (hipStream_t)stream;
    const bool fp8 = cache->dtype == kF8E4M3, wide = shape->softcap > kWideCap;
    if (shape->dtype == kBFloat16) launch_form<kBFloat16, false>(fp8, wide, a.dim, l.waves, (unsigned)grid, s, a);
    else launch_form<kFloat16, false>(fp8, wide, a.dim, l.waves, (unsigned)grid, s, a);
    MFH_TRY(launch_status("k_prefill"));
    if (l.parts > 1) {
        if (shape->dtype == kBFloat16) launch_join<kBFloat16>(a, requests, s);
        else launch_join<kFloat16>(a, requests, s);
        MFH_TRY(launch_status("k_prefill_join"));
    }
    return MFH_OK;
}

}  // extern "C"
