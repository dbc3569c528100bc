// decode.hpp — what the kernels share that attend for one new token per request
// (decode.hip, shared.hip): a wave's tile of 32 tokens, its loads from pages
// into the matrix operands' layouts.
#ifndef MFH_DECODE_HPP
#define MFH_DECODE_HPP

#include "paged.hpp"

namespace mfh {
namespace decode {

constexpr int kTile = 32;    // tokens of a wave's step
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kHeads = 16;   // columns of a product: query heads

enum Cap { kNone, kNarrow, kWide };

MFH_DEV mfh_u32 low_halves(mfh_u32 a, mfh_u32 b) { return __builtin_amdgcn_perm(b, a, 0x05040100); }
MFH_DEV mfh_u32 high_halves(mfh_u32 a, mfh_u32 b) { return __builtin_amdgcn_perm(b, a, 0x07060302); }

// The tokens that are seen: [first, length).
struct Seen {
    mfh_u32 length, first;
};

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
    template <typename Table>
    __device__ void ask(const PageArgs& p, Table table, const Seen& c, mfh_u32 t0, int lane)
    {
        // past the length its last page again
#pragma unroll
        for (int h = 0; h < (FAST ? 2 : 1); h++)
            page[h] = table[p.by_page.quotient(min(t0 + (FAST ? 16 * h : lane & 31), c.length - 1))];
    }
    // `real`: the tile is one of the wave's; else nothing of it is valid.
    __device__ TileAt<FAST> place(const PageArgs& p, const Seen& c, mfh_u32 t0, int lane, bool real) const
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

template <typename T, int POLICY = kStreamed>
MFH_DEV T buffer_piece(__amdgpu_buffer_rsrc_t r, mfh_u32 lane_at, mfh_u32 at)
{
    if constexpr (sizeof(T) == 16) return __builtin_amdgcn_raw_buffer_load_b128(r, (int)lane_at, (int)at, POLICY);
    else if constexpr (sizeof(T) == 8) return __builtin_amdgcn_raw_buffer_load_b64(r, (int)lane_at, (int)at, POLICY);
    else return __builtin_amdgcn_raw_buffer_load_b32(r, (int)lane_at, (int)at, POLICY);
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

template <typename T, bool STREAMED = true>
MFH_DEV T load_piece(const char* p)
{
    if constexpr (sizeof(T) == 16) return load16<STREAMED>(p);
    else if constexpr (sizeof(T) == 8) return load8<STREAMED>(p);
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

}  // namespace decode
}  // namespace mfh

#endif  // MFH_DECODE_HPP
