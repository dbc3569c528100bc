// prefill.hip — attention of each request's new tokens over a paged cache
// (mfh_paged_prefill): causal, with an optional window, prefix, cap and bias.
//
// 4 * pairs * q_heads * head_dim operations over keys and values that stay in
// the caches near the cores: the matrix cores bound it.  The rows of one
// key-value head are its query heads of all new tokens (row = token * group +
// head of the group), so that heads which share keys share a workgroup's key
// tiles too.  A workgroup is four waves of 32 rows each and walks over tiles of
// 64 keys, staged through LDS: the next tile's pieces are loaded into registers
// while the present one is computed, and 8-bit caches become 16-bit on the way.
//
//   scores^T [keys][rows] = K Q^T      Q stays in registers, K as it stands in LDS
//   out^T [dims][rows] += V^T P^T      V^T by LDS reads that transpose
//
// A lane holds the scores of row lane % 32 for keys 8 * (i / 4) + 4 * (lane / 32)
// + i % 4; eight of them, in that order, are the second product's P^T operand,
// so weights never leave their lane, and a row's maximum is one exchange between
// two lanes.  The running reference is decode.hip's.
#include "paged.hpp"

namespace mfh {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kRows = 32 * kWaves;  // of a workgroup
constexpr float kStep = 8.0f;       // the reference moves where a score passes it by 2^kStep

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
    float scale, cap_twice, cap_scaled, v_scale;
    int32_t window, kv_heads, q_heads, group, dim;
    mfh_u32 row_tiles;  // of a request and head at most
    Divider by_group, by_kv_heads, by_row_tiles;
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Four 16-bit values of one column: in each 16 lanes, lane i gives the address
// of four values of row i / 4, columns 4 (i % 4) .., and gets column i's.
MFH_DEV u32x2 read_column(const char* at)
{
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at)));
}

// Whether a dword's halves are infinite or NaN.
template <int DT>
MFH_DEV bool not_finite(mfh_u32 pair)
{
    constexpr mfh_u32 kExp = DT == kBFloat16 ? 0x7f80u : 0x7c00u;
    return ((pair & kExp) == kExp) | ((pair & kExp << 16) == kExp << 16);
}

// Where 16 bytes of a row stand among the row's pieces in LDS.  Rows have no
// gaps (a load into LDS writes 64 lanes' pieces one after the other), so pieces
// change places by row: 16 rows of one piece, as K is read, lie in 16 different
// places, and four rows of four pieces, as V is, too.
template <int PIECES>
MFH_DEV int place(int row, int piece)
{
    return piece ^ (((row & 3) << 2 | (row >> 2 & 3)) & (PIECES - 1));
}

// DP: head_dim rounded up to 64, 128 or 256.
template <int DT, bool FP8, int DP>
__global__ __launch_bounds__(kThreads, DP <= 128 ? 2 : 1) void k_prefill(PrefillArgs a)
{
    constexpr int kBytes = FP8 ? 1 : 2;
    constexpr int kSteps = DP / 16;
    constexpr int kDimTiles = DP / 32;
    constexpr int kKeys = DP <= 128 ? 64 : 32;           // of a tile
    constexpr int kBlocks = kKeys / 32;
    constexpr int kPitch = 2 * DP;
    constexpr int kPieces = DP / 8;                      // of a key, eight values each
    constexpr int kLoads = kKeys * kPieces / kThreads;   // of a thread
    constexpr int kKeyStep = kThreads / kPieces;         // keys between a thread's pieces
    __shared__ __align__(16) char s_tiles[2][2][kKeys * kPitch];  // K and V of two tiles

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    mfh_u32 rest = a.by_kv_heads.quotient(blockIdx.x);
    const mfh_u32 kv = blockIdx.x - rest * a.kv_heads;
    const mfh_u32 r = a.by_row_tiles.quotient(rest);
    const mfh_u32 row_tile = a.row_tiles - 1 - (rest - r * a.row_tiles);  // the longest rows first

    const int64_t begin = min(max((int64_t)a.starts[r], (int64_t)0), a.tokens);
    const int64_t end = min(max((int64_t)a.starts[r + 1], begin), a.tokens);
    const mfh_u32 fresh = (mfh_u32)(end - begin), computed = (mfh_u32)min((int64_t)fresh, a.most_fresh);
    const mfh_u32 rows = computed * a.group, row0 = row_tile * kRows;
    if (row0 >= rows) return;
    const int length = (int)min((mfh_u64)max(a.lengths[r], 0), min((mfh_u64)a.pages.width * a.pages.by_page.d, (mfh_u64)kLongest));
    const int prefix = a.prefix ? min(max(a.prefix[r], 0), length) : 0;
    const int first_position = length - (int)fresh;  // of the request's new tokens; may be negative

    const int32_t* table = a.pages.table + (int64_t)r * a.pages.table_stride;
    const char* k_base = a.pages.k + kv * a.pages.head_bytes;
    const char* v_base = a.pages.v + kv * a.pages.head_bytes;

    // Positions of the workgroup's rows, and the keys any of them sees.
    const int low_position = first_position + (int)a.by_group.quotient(row0);
    const int high_position = first_position + (int)a.by_group.quotient(min(row0 + kRows, rows) - 1);
    const int key_end = min(max(high_position + 1, prefix), length);
    const int window_first = a.window > 0 ? max(low_position - a.window + 1, 0) : 0;  // below: the prefix only
    const int tile_end = key_end > 0 ? (key_end + kKeys - 1) / kKeys : 0;
    // The next tile at or after `tile` that has a key for some row: between the
    // prefix and the window there is none.
    auto next_tile = [&](int tile) {
        return tile * kKeys >= prefix ? max(tile, window_first / kKeys) : tile;
    };

    // This lane's row, and its wave's.
    const mfh_u32 row = row0 + 32 * wave + col;
    const bool real = row < rows;
    const mfh_u32 token = a.by_group.quotient(min(row, rows - 1)), head = kv * a.group + (min(row, rows - 1) - token * a.group);
    const int position = first_position + (int)token;
    const mfh_u32 wave_row0 = min(row0 + 32 * wave, rows - 1), wave_row1 = min(row0 + 32 * wave + 31, rows - 1);
    const int wave_low = first_position + (int)a.by_group.quotient(wave_row0);
    const int wave_high = first_position + (int)a.by_group.quotient(wave_row1);

    u32x4 q[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; s++) {
        const int d = 16 * s + 8 * half;
        q[s] = u32x4{0, 0, 0, 0};
        if (real && d < a.dim) q[s] = load16<false>(a.q + ((begin + token) * a.q_t + head * a.q_h + d) * 2);
    }
    const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;

    f32x16 acc[kDimTiles];
#pragma unroll
    for (int d = 0; d < kDimTiles; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[d][i] = 0.0f;
    float ref = 0.0f, limit = -INFINITY, sum = 0.0f;

    // Staging: lane l looks up key l of a tile; thread t takes the piece that
    // belongs in place t % kPieces of keys t / kPieces + i * kKeyStep.
    const int key0 = threadIdx.x / kPieces, slot = threadIdx.x % kPieces;
    int64_t at = 0;
    mfh_u64 valid = 0;  // bit i: key i has a page
    auto locate = [&](int tile) {
        const mfh_u32 t = (mfh_u32)(tile * kKeys + (lane & (kKeys - 1)));
        const mfh_u32 in_table = a.pages.by_page.quotient(t), in_page = t - in_table * a.pages.by_page.d;
        const int32_t page = (int)t < length ? table[in_table] : -1;
        const bool ok = (mfh_u32)page < a.pages.pages;
        at = ok ? (mfh_u32)page * a.pages.page_bytes + in_page * a.pages.token_bytes : 0;
        valid = __ballot(ok) << (64 - kKeys);
    };
    constexpr mfh_u64 kAll = ~mfh_u64(0) << (64 - kKeys);
    auto is_valid = [&](mfh_u64 mask, int key) { return (mask >> (64 - kKeys + key) & 1) != 0; };
    // whether every row of the workgroup sees every key
    auto is_open = [&](int tile, mfh_u64 mask) {
        const int key = tile * kKeys;
        return mask == kAll && ((key + kKeys <= low_position + 1 && (a.window <= 0 || key > high_position - a.window)) || key + kKeys <= prefix);
    };
    auto piece_at = [&](int i, bool* in_dim) {  // of this thread's i-th piece
        const int key = key0 + i * kKeyStep, piece = place<kPieces>(key, slot);
        *in_dim = piece * 8 < a.dim;
        return shuffle64(at, key) + (*in_dim ? piece * 8 * kBytes : 0);
    };
    // Eight-bit pieces wait in registers while the tile before is computed, and
    // are widened on the way to LDS; so are those of tiles that a mask cuts.
    u32x2 k_codes[kLoads], v_codes[kLoads];
    auto fetch = [&]() {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            bool in_dim;
            const int64_t from = piece_at(i, &in_dim);
            k_codes[i] = load8<false>(k_base + from);
            v_codes[i] = load8<false>(v_base + from);
        }
    };
    // True if a mask cuts the tile and this thread's part has values that are not finite.
    auto put = [&](char* s_k, char* s_v, mfh_u64 mask, bool open, int i, u32x4 kw, u32x4 vw, bool in_dim) {
        const int key = key0 + i * kKeyStep;
        const u32x4 zero = {0, 0, 0, 0};
        const bool keep = in_dim & is_valid(mask, key);
        kw = keep ? kw : zero, vw = keep ? vw : zero;
        *reinterpret_cast<u32x4*>(s_k + key * kPitch + slot * 16) = kw;
        *reinterpret_cast<u32x4*>(s_v + key * kPitch + slot * 16) = vw;
        return !open & (not_finite<DT>(vw[0]) | not_finite<DT>(vw[1]) | not_finite<DT>(vw[2]) | not_finite<DT>(vw[3]));
    };
    auto put_codes = [&](char* s_k, char* s_v, mfh_u64 mask, bool open) {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const int key = key0 + i * kKeyStep;
            const u32x2 k = k_codes[i], v = v_codes[i];
            odd |= put(s_k, s_v, mask, open, i,
                       u32x4{e4m3_pair<DT, false>(k[0]), e4m3_pair<DT, true>(k[0]), e4m3_pair<DT, false>(k[1]), e4m3_pair<DT, true>(k[1])},
                       u32x4{e4m3_pair<DT, false>(v[0]), e4m3_pair<DT, true>(v[0]), e4m3_pair<DT, false>(v[1]), e4m3_pair<DT, true>(v[1])},
                       place<kPieces>(key, slot) * 8 < a.dim);
        }
        return odd;
    };
    // 16-bit pieces of a tile that is whole go to LDS directly.
    auto stage = [&](char* s_k, char* s_v, mfh_u64 mask, bool open) {
        bool odd = false;
        if (open && a.dim == DP) {
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                bool in_dim;
                const int64_t from = piece_at(i, &in_dim);
                const int to = (i * kThreads + wave * 64) * 16;
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(k_base + from),
                                                 (__attribute__((address_space(3))) void*)(s_k + to), 16, 0, 0);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(v_base + from),
                                                 (__attribute__((address_space(3))) void*)(s_v + to), 16, 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                bool in_dim;
                const int64_t from = piece_at(i, &in_dim);
                const u32x4 k = load16<false>(k_base + from), v = load16<false>(v_base + from);
                odd |= put(s_k, s_v, mask, open, i, k, v, in_dim);
            }
        }
        return odd;
    };

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

    // A masked weight of 0 times a value that is not finite would be NaN.  Where
    // a mask cuts a tile that has such values, they are added to the rows that
    // see them, and are zeros in the product.
    auto add_odd = [&](const char* s_v, int tile, mfh_u64 mask) {
        const Seen seen = seen_from(tile * kKeys, 0);
        for (int key = 0; key < kKeys; key++) {
            const bool see = is_valid(mask, key) & (((key <= seen.back) & (key > seen.oldest)) | (key < seen.in_prefix));
#pragma unroll
            for (int d = 0; d < kDimTiles; d++) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int dim = 32 * d + 8 * (i / 4) + 4 * half + i % 4;
                    const mfh_u32 v = *reinterpret_cast<const mfh_u16*>(s_v + key * kPitch + place<kPieces>(key, dim / 8) * 16 + dim % 8 * 2);
                    if (see & not_finite<DT>(v)) acc[d][i] += dec16<DT>(v);
                }
            }
        }
    };
    auto clear_odd = [&](char* s_v) {
        for (int i = 0; i < kLoads; i++) {
            u32x4& w = *reinterpret_cast<u32x4*>(s_v + (key0 + i * kKeyStep) * kPitch + slot * 16);
            u32x4 v = w;
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] &= (not_finite<DT>(v[j] & 0xffffu) ? 0u : 0xffffu) | (not_finite<DT>(v[j] >> 16) ? 0u : 0xffff0000u);
            w = v;
        }
    };

    auto compute = [&](const char* s_k, const char* s_v, int tile, mfh_u64 mask) {
        const int key_first = tile * kKeys;
        // Rows of this wave that see something here, and whether all of it.
        const bool some = key_first < max(wave_high + 1, prefix) &&
                          (a.window <= 0 || key_first < prefix || key_first + kKeys > wave_low - a.window + 1);
        if (!some) return;
        f32x16 s[kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; b++) {
#pragma unroll
            for (int i = 0; i < 16; i++) s[b][i] = 0.0f;
#pragma unroll
            for (int d = 0; d < kSteps; d++) {
                const int key = 32 * b + col;
                const u32x4 kf = *reinterpret_cast<const u32x4*>(s_k + key * kPitch + place<kPieces>(key, 2 * d + half) * 16);
                s[b] = mfma32<DT>(kf, q[d], s[b]);
            }
        }
        const bool all = mask == kAll && ((key_first + kKeys <= wave_low + 1 && (a.window <= 0 || key_first > wave_high - a.window)) ||
                                          key_first + kKeys <= prefix);
        float scale = a.scale;  // what is left to multiply by
        if (a.cap_scaled != 0.0f || a.slopes || !all || !(scale > 0.0f)) {
            scale = 1.0f;
#pragma unroll
            for (int b = 0; b < kBlocks; b++) {
#pragma unroll
                for (int i = 0; i < 16; i++) s[b][i] *= a.scale;
                if (a.cap_scaled != 0.0f) {
#pragma unroll
                    for (int i = 0; i < 16; i++) s[b][i] = capped(s[b][i], a.cap_twice, a.cap_scaled);
                }
                const Seen seen = seen_from(key_first + 32 * b + 4 * half, (mfh_u32)(mask >> (64 - kKeys + 32 * b)) >> (4 * half));
                if (a.slopes) {
#pragma unroll
                    for (int i = 0; i < 16; i++) s[b][i] -= slope * fabsf((float)(seen.back - (8 * (i / 4) + i % 4)));
                }
                if (!all) {
#pragma unroll
                    for (int i = 0; i < 16; i++) s[b][i] = seen(8 * (i / 4) + i % 4) ? s[b][i] : -INFINITY;
                }
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, s[b][i]);
        top *= scale;
        if (__any(top > limit)) {
            top = fmaxf(top, __shfl_xor(top, 32));
            if (top > limit) {
                // (at first there is nothing to scale but what add_odd put there)
                const float alpha = limit == -INFINITY ? 1.0f : exp2_fast(ref - top);
                ref = top;
                limit = top + kStep;
                sum *= alpha;
#pragma unroll
                for (int d = 0; d < kDimTiles; d++) acc[d] *= alpha;
            }
        }
        u32x4 p[2 * kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; b++) {
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                s[b][i] = exp2_fast(__builtin_fmaf(s[b][i], scale, -ref));
                part += s[b][i];
            }
            sum += part;
#pragma unroll
            for (int i = 0; i < 16; i += 2) p[2 * b + i / 8][i / 2 % 4] = enc16x2<DT>(s[b][i], s[b][i + 1]);
        }
        // V^T: in 16 lanes row lane % 16 / 4 of four keys, columns 4 (lane % 4) ..
        auto column = [&](int key, int d) {
            const int at_key = key + 4 * half + (lane & 15) / 4, piece = 4 * d + 2 * (lane >> 4 & 1) + (lane & 3) / 2;
            return read_column(s_v + at_key * kPitch + place<kPieces>(at_key, piece) * 16 + 8 * (lane & 1));
        };
#pragma unroll
        for (int d = 0; d < kDimTiles; d++) {
#pragma unroll
            for (int j = 0; j < 2 * kBlocks; j++) {
                const u32x2 lo = column(16 * j, d), hi = column(16 * j + 8, d);
                acc[d] = mfma32<DT>(u32x4{lo[0], lo[1], hi[0], hi[1]}, p[j], acc[d]);
            }
        }
    };

    // One tile is computed while the next one is on its way to the other half
    // of LDS.
    int tile = next_tile(0), now = 0;
    mfh_u64 mask = 0;
    bool odd = false, open = true;
    auto meet = [&]() {  // all of the staged tile is in LDS
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): loads into LDS are no one's registers
        odd = open ? (__syncthreads(), false) : __syncthreads_or(odd) != 0;
    };
    if (tile < tile_end) {
        locate(tile);
        mask = valid, open = is_open(tile, mask);
        if constexpr (FP8) {
            fetch();
            odd = put_codes(s_tiles[0][0], s_tiles[0][1], mask, open);
        } else {
            odd = stage(s_tiles[0][0], s_tiles[0][1], mask, open);
        }
        meet();
    }
    while (tile < tile_end) {
        const char* s_k = s_tiles[now][0];
        char* s_v = s_tiles[now][1];
        const int following = next_tile(tile + 1);
        const mfh_u64 mask_now = mask;
        if (odd) {
            add_odd(s_v, tile, mask);
            __syncthreads();
            clear_odd(s_v);
            __syncthreads();
            odd = false;
        }
        if (following < tile_end) {
            locate(following);
            mask = valid, open = is_open(following, mask);
            if constexpr (FP8) fetch();
            else odd = stage(s_tiles[now ^ 1][0], s_tiles[now ^ 1][1], mask, open);
        }
        compute(s_k, s_v, tile, mask_now);
        tile = following;
        if (following < tile_end) {
            if constexpr (FP8) odd = put_codes(s_tiles[now ^ 1][0], s_tiles[now ^ 1][1], mask, open);
            meet();
        }
        now ^= 1;
    }

    sum += __shfl_xor(sum, 32);
    if (!real) return;
    const float f = sum == 0.0f ? 0.0f : a.v_scale / sum;
    char* to = a.out + ((begin + token) * a.out_t + head * a.out_h) * 2;
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
    if (half == 0 && a.lse)
        a.lse[(begin + token) * a.q_heads + head] = sum == 0.0f ? -INFINITY : ref * kLn2 + logf(sum);
}

template <int DT, bool FP8>
void launch_dims(int dim, unsigned grid, hipStream_t s, const PrefillArgs& a)
{
    if (dim <= 64) k_prefill<DT, FP8, 64><<<grid, kThreads, 0, s>>>(a);
    else if (dim <= 128) k_prefill<DT, FP8, 128><<<grid, kThreads, 0, s>>>(a);
    else k_prefill<DT, FP8, 256><<<grid, kThreads, 0, s>>>(a);
}

}  // namespace
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
    if (requests < 0 || tokens < 0 || most_fresh < 0)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: negative number of requests or tokens", what);
    if (!bytes) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL result", what);
    *bytes = 0;
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
    const Strides qs(shape->q_token_stride, shape->q_head_stride, shape->q_heads, cache->head_dim);
    const Strides os(shape->out_token_stride, shape->out_head_stride, shape->q_heads, cache->head_dim);
    a.q_t = qs.token, a.q_h = qs.head, a.out_t = os.token, a.out_h = os.head;
    a.tokens = tokens, a.most_fresh = std::min(most_fresh, tokens);
    a.scale = shape->scale * cache->k_scale;
    if (shape->softcap > 0.0f) {
        a.cap_twice = 2.0f * kLog2e / shape->softcap;
        a.cap_scaled = shape->softcap * kLog2e;
    } else {
        a.scale *= kLog2e;
    }
    a.v_scale = cache->v_scale;
    a.window = shape->window < kLongest ? shape->window : 0, a.kv_heads = cache->kv_heads, a.q_heads = shape->q_heads;
    a.group = shape->q_heads / cache->kv_heads;
    a.dim = cache->head_dim;
    const int64_t row_tiles = (a.most_fresh * a.group + kRows - 1) / kRows;
    const __int128 grid = (__int128)row_tiles * cache->kv_heads * requests;
    if (a.most_fresh * a.group > 0x7fffffff || grid >= ((int64_t)1 << 32) / kThreads)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d requests of %lld tokens and %d heads are too many for one call",
                    what, requests, (long long)a.most_fresh, shape->q_heads);
    a.row_tiles = (mfh_u32)row_tiles;
    a.by_group = Divider((mfh_u32)a.group), a.by_kv_heads = Divider((mfh_u32)a.kv_heads), a.by_row_tiles = Divider(a.row_tiles);
    hipStream_t s = (hipStream_t)stream;
    const bool fp8 = cache->dtype == kF8E4M3;
    if (shape->dtype == kBFloat16) {
        if (fp8) launch_dims<kBFloat16, true>(a.dim, (unsigned)grid, s, a);
        else launch_dims<kBFloat16, false>(a.dim, (unsigned)grid, s, a);
    } else {
        if (fp8) launch_dims<kFloat16, true>(a.dim, (unsigned)grid, s, a);
        else launch_dims<kFloat16, false>(a.dim, (unsigned)grid, s, a);
    }
    return launch_status("k_prefill");
}

}  // extern "C"
