// pages.hip — block tables and slot maps of a paged key-value cache from the
// requests' lengths (mfh_page_plan), on the device.
//
// With P tokens a page, request r holds have = ceil(before/P) pages and wants
// ceil(after/P).  Three running sums over the requests place everything: new
// tokens (where a request's tokens start), pages needed (which of the ring's
// pages a request takes) and pages returned (where they go at the ring's
// tail).  A token's slot then follows from its request, its position and
// either the table or the ring, with no other thread's result: one launch.
//
// Every workgroup runs the sums over all requests again, 512 at a time, and
// writes its own 512 tokens; workgroup 0 writes what exists once per request.
// Sums again cost each workgroup about a microsecond per 512 requests, a second
// launch behind the first more than that.  A few kilobytes to a few megabytes:
// latency bounds it, of the launch, the sums, a token's search for its request
// and its page's load.  In a row of launches 64 requests with one token each take
// 3.8 us, 1021 requests with 260,000 tokens 10.3 us.  With 1024 threads the
// first takes 6.1 us (twice the waves at each barrier), the second 9.4; with 256
// they take 3.5 and 14.4; with two tokens a thread one after the other 3.8 and
// 9.5, but 300 requests with 77,000 tokens 6.3 instead of 5.4.
//
// The sums saturate at a limit above anything that is granted, so 32 bits
// hold them: min(a + b, limit) is associative, and whatever has reached the
// limit is refused.
#include "common.hpp"
#include "launch.hpp"
#include "paged.hpp"
#include "../../include/mfh_attention.h"

namespace mfh {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr mfh_u32 kMost = 1u << 30;  // tokens, ring entries

struct PlanArgs {
    const int32_t* before;
    const int32_t* after;
    int32_t* table;
    int64_t table_stride;
    int32_t* ring;
    const int64_t* ring_state;
    int64_t* ring_state_out;
    int64_t* slots;
    int32_t* positions;
    int32_t* starts;
    int32_t* lengths;
    int32_t* status;
    mfh_u32 requests, page_size, width, ring_size, tokens;
    Divider by_page;
};

MFH_DEV mfh_u32 sat(mfh_u32 a, mfh_u32 b, mfh_u32 limit) { return min(a + b, limit); }

// Saturating sum of the wave's lanes up to and with this one, by moves between
// lanes of a row of 16 and then from the rows before.  Values and limit are at
// most 2^30 + 1, so a + b fits.
MFH_DEV mfh_u32 lanes_upto(mfh_u32 v, mfh_u32 limit)
{
    v = sat(v, (mfh_u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, true), limit);  // row_shr 1, 2, 4, 8
    v = sat(v, (mfh_u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, true), limit);
    v = sat(v, (mfh_u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, true), limit);
    v = sat(v, (mfh_u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, true), limit);
    v = sat(v, (mfh_u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false), limit);  // row_bcast 15, 31
    v = sat(v, (mfh_u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false), limit);
    return v;
}

// One running sum: a wave leaves the sum of its lanes in by_wave and, behind a
// barrier, `before` is the sum of what came ahead of the thread and `total`
// that with the whole workgroup.
struct Sum {
    mfh_u32 upto, before, total;
    MFH_DEV void lanes(mfh_u32 v, mfh_u32 limit, mfh_u32* by_wave)
    {
        upto = lanes_upto(min(v, limit), limit);
        if ((threadIdx.x & 63) == 63) by_wave[threadIdx.x >> 6] = upto;
    }
    MFH_DEV void join(mfh_u32 ahead, mfh_u32 limit, const mfh_u32* by_wave)
    {
        before = total = ahead;
#pragma unroll
        for (mfh_u32 w = 0; w < kWaves; w++) {
            const mfh_u32 s = by_wave[w];
            if (w < threadIdx.x >> 6) before = sat(before, s, limit);
            total = sat(total, s, limit);
        }
        const mfh_u32 left = (mfh_u32)__builtin_amdgcn_update_dpp(0, (int)upto, 0x138, 0xf, 0xf, false);  // wave_shr 1
        before = sat(before, left, limit);
    }
};

MFH_DEV mfh_u32 wrap(mfh_u32 at, mfh_u32 size) { return at >= size ? at - size : at; }

__global__ __launch_bounds__(kThreads) void k_page_plan(PlanArgs a)
{
    __shared__ mfh_u32 s_start[kThreads];   // first token
    __shared__ mfh_u32 s_before[kThreads];
    __shared__ mfh_u32 s_have[kThreads];    // pages held before
    __shared__ mfh_u32 s_first[kThreads];   // ring index of the first page taken; kNone: refused
    __shared__ mfh_u32 s_give[kThreads];    // pages returned
    __shared__ mfh_u32 s_give_at[kThreads];
    __shared__ mfh_u32 s_sum[3][kWaves];
    __shared__ mfh_u32 s_taken;
    constexpr mfh_u32 kNone = 0xffffffffu;

    const mfh_u32 tid = threadIdx.x;
    const mfh_u32 P = a.page_size;
    const mfh_u32 token_limit = a.tokens + 1, page_limit = kMost + 1;
    const int64_t head = a.ring_state[0], tail = a.ring_state[1];
    const mfh_u32 free_pages = (mfh_u32)min(max(tail - head, (int64_t)0), (int64_t)a.ring_size);
    const mfh_u32 head_at = (mfh_u32)((uint64_t)head % a.ring_size);
    const mfh_u32 tail_at = (mfh_u32)((uint64_t)tail % a.ring_size);
    if (tid == 0) s_taken = 0;

    auto pages_of = [&](mfh_u32 tokens) {
        const mfh_u32 whole = a.by_page.quotient(tokens);
        return whole + (whole * P != tokens);
    };

    // this workgroup's tokens
    const mfh_u32 t_begin = blockIdx.x * kThreads;
    const mfh_u32 t_end = min(t_begin + kThreads, a.tokens);

    mfh_u32 tokens_ahead = 0, need_ahead = 0, give_ahead = 0;
    for (mfh_u32 base = 0; base < a.requests; base += kThreads) {
        const mfh_u32 r = base + tid;
        const bool real = r < a.requests;
        const int32_t b0 = real ? a.before[r] : 0, a0 = real ? a.after[r] : 0;
        const mfh_u32 b = (mfh_u32)max(b0, 0), e = (mfh_u32)max(a0, 0);
        const mfh_u32 have = pages_of(b), want = pages_of(e);
        const mfh_u32 fresh = e > b ? e - b : 0;
        Sum tokens, needed, given;
        tokens.lanes(fresh, token_limit, s_sum[0]);
        __syncthreads();
        tokens.join(tokens_ahead, token_limit, s_sum[0]);
        const mfh_u32 start = tokens.before;
        const mfh_u32 end = sat(start, min(fresh, token_limit), token_limit);
        const bool wide = have > a.width || want > a.width || b0 < 0 || a0 < 0;
        const bool late = end > a.tokens && fresh > 0;
        const bool may = !wide && !late;
        const mfh_u32 need = may && want > have ? want - have : 0;
        const mfh_u32 give = may && have > want ? have - want : 0;
        needed.lanes(need, page_limit, s_sum[1]);
        given.lanes(give, page_limit, s_sum[2]);
        __syncthreads();
        needed.join(need_ahead, page_limit, s_sum[1]);
        given.join(give_ahead, page_limit, s_sum[2]);
        const mfh_u32 first = needed.before, need_end = sat(first, min(need, page_limit), page_limit);
        const bool granted = may && (need == 0 || need_end <= free_pages);
        s_start[tid] = real ? start : kNone;
        s_before[tid] = b;
        s_have[tid] = have;
        s_first[tid] = granted ? first : kNone;
        s_give[tid] = give;
        s_give_at[tid] = given.before;
        if (granted && need > 0) atomicMax(&s_taken, need_end);  // an integer maximum: any order gives it
        if (blockIdx.x == 0 && real) {
            a.starts[r] = (int32_t)min(start, a.tokens);
            a.lengths[r] = (int32_t)(granted ? e : b);
            a.status[r] = wide ? 2 : late ? 3 : granted ? 0 : 1;
        }
        __syncthreads();

        const mfh_u32 chunk = min(a.requests - base, (mfh_u32)kThreads);
        const mfh_u32 chunk_begin = tokens_ahead, chunk_end = tokens.total;
        for (mfh_u32 t = max(t_begin, chunk_begin) + tid; t < min(t_end, chunk_end); t += kThreads) {
            // the last request that starts at or before t (those without tokens start where the next one does)
            mfh_u32 lo = 0, hi = chunk;
            while (hi - lo > 1) {
                const mfh_u32 mid = (lo + hi) >> 1;
                if (s_start[mid] <= t) lo = mid;
                else hi = mid;
            }
            const mfh_u32 position = s_before[lo] + (t - s_start[lo]);
            const mfh_u32 row = a.by_page.quotient(position), in_page = position - row * P;
            int64_t slot = -1;
            if (s_first[lo] != kNone) {
                int32_t* entry = a.table + (int64_t)(base + lo) * a.table_stride + row;
                int32_t page;
                if (row < s_have[lo]) {
                    page = *entry;
                } else {
                    page = a.ring[wrap(head_at + s_first[lo] + (row - s_have[lo]), a.ring_size)];
                    if (in_page == 0) *entry = page;
                }
                if (page >= 0) slot = (int64_t)page * P + in_page;
            }
            a.slots[t] = slot;
            a.positions[t] = (int32_t)position;
        }

        // returned pages: a wave per request that has any
        const mfh_u32 wave = blockIdx.x * kWaves + (tid >> 6), waves = gridDim.x * kWaves;
        for (mfh_u32 i = wave; i < chunk && given.total > give_ahead; i += waves) {
            const mfh_u32 n = s_give[i];
            const int32_t* row = a.table + (int64_t)(base + i) * a.table_stride + (s_have[i] - n);
            for (mfh_u32 k = tid & 63; k < n; k += 64) {
                const mfh_u32 at = s_give_at[i] + k;
                if (at < a.ring_size) a.ring[wrap(tail_at + at, a.ring_size)] = row[k];
            }
        }
        tokens_ahead = tokens.total;
        need_ahead = needed.total;
        give_ahead = given.total;
        __syncthreads();
    }
    // padding behind the last token
    for (mfh_u32 t = max(t_begin, tokens_ahead) + tid; t < t_end; t += kThreads) {
        a.slots[t] = -1;
        a.positions[t] = -1;
    }
    if (blockIdx.x == 0 && tid == 0) {
        a.starts[a.requests] = (int32_t)min(tokens_ahead, a.tokens);
        a.ring_state_out[0] = head + s_taken;
        a.ring_state_out[1] = tail + give_ahead;
    }
}

bool overlap(const int32_t* a, const int32_t* b, int64_t n)
{
    return (uintptr_t)a < (uintptr_t)(b + n) && (uintptr_t)b < (uintptr_t)(a + n);
}

}  // namespace
}  // namespace mfh

using namespace mfh;

extern "C" {

int mfh_page_plan(const int32_t* before, const int32_t* after, int32_t requests, int32_t page_size, int32_t* table,
                  int64_t table_stride, int32_t table_width, int32_t* ring, int64_t ring_size,
                  const int64_t* ring_state, int64_t* ring_state_out, int64_t* slots, int32_t* positions,
                  int64_t tokens, int32_t* starts, int32_t* lengths, int32_t* status, void* stream)
{
    const char* what = "mfh_page_plan";
    const Device* dev;
    MFH_TRY(bind_device(&dev));
    if (requests < 0) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: negative number of requests %d", what, requests);
    if (page_size < 1) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: page size %d is not positive", what, page_size);
    if (tokens < 0 || tokens > (int64_t)kMost)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %lld tokens are not within 0..2^30", what, (long long)tokens);
    if (ring_size < 1 || ring_size > (int64_t)kMost)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: a ring of %lld pages is not within 1..2^30", what,
                    (long long)ring_size);
    if (table_width < 0 || table_stride < table_width)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: table width %d does not fit its stride %lld", what, table_width,
                    (long long)table_stride);
    if (!ring || !ring_state || !ring_state_out || !starts || (tokens > 0 && (!slots || !positions)) ||
        (requests > 0 && (!before || !after || !lengths || !status || (table_width > 0 && !table))))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL buffer", what);
    if (ring_state == ring_state_out)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: ring_state_out is ring_state, which other workgroups still read",
                    what);
    PlanArgs args{before, after, table, table_stride, ring, ring_state, ring_state_out, slots, positions, starts,
                  lengths, status, (mfh_u32)requests, (mfh_u32)page_size, (mfh_u32)table_width, (mfh_u32)ring_size,
                  (mfh_u32)tokens, Divider((mfh_u32)page_size)};
    const unsigned grid = (unsigned)std::max<int64_t>(1, (tokens + kThreads - 1) / kThreads);
    if (grid > 1 && requests > 0 && (overlap(lengths, before, requests) || overlap(lengths, after, requests)))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: lengths is before or after, which other workgroups still read (%lld tokens, %d at most)",
                    what, (long long)tokens, kThreads);
    k_page_plan<<<grid, kThreads, 0, (hipStream_t)stream>>>(args);
    return launch_status("k_page_plan");
}

}  // extern "C"
