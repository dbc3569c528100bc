// fork.hip — requests of a paged cache that grow out of one another
// (mfh_page_fork), and the copies of pages that this asks for (mfh_page_copy).
//
// A page's count of holders changes by what the new requests hold and the old
// ones held.  Both are nearly the same, so only differences are counted: of a
// parent's children the first that is not empty is its heir, and what both hold
// cancels out.  A parent without heir, what an heir does not take over, and
// every other child's pages cost an atomic on an integer each, whose order does
// not matter.  In a beam search's step, where a third of the beams have no
// child, that is two thirds of the tables' entries instead of twice all of them.
//
// Pages that fall to no holder go to the ring in the order of their numbers, so
// that the ring does not depend on which request let go of a page first.  Their
// places are a running sum over the pages' counts.
//
// Where pages and requests are few one workgroup does all of it, with the counts in
// LDS: latency bounds it, 9 us.  Else there are four launches: what concerns each
// request once (one workgroup) beside the counts' copy, the tables, the number of
// pages that go back in each piece of the counts, and those pages.  For 1021
// requests of up to 512 pages they take 5, 9, 3 and 4 us: the chain of loads, the
// atomics, and the starts of launches bound them, not the 3 MB that move.  (Numbers
// kept by the second launch, as pages fall below zero, are a launch less, but
// atomics on a few words: 1021 requests that return 28800 pages, 58 us.)
#include "common.hpp"
#include "launch.hpp"
#include "paged.hpp"

namespace mfh {
namespace {

constexpr int kThreads = 1024;  // of a workgroup that plans
constexpr int kWaves = kThreads / 64;
constexpr mfh_u32 kMostRequests = 8192;
// The form in one workgroup: 9 us for 64 requests of up to 125 pages, in four launches
// 17; from some 14000 table entries on those are faster (25000: 26 and 17 us).
constexpr mfh_u32 kFewRequests = 1024, kFewPages = 16384, kFewEntries = 12288;
constexpr mfh_u32 kChunk = 4 * kThreads;                   // pages of a workgroup that returns them
constexpr mfh_u32 kNone = 0xffffffffu;

struct ForkArgs {
    const int32_t* parents;
    const int32_t* before;
    const int32_t* keep;
    const int32_t* table;
    int32_t* table_out;
    int64_t table_stride;
    const int32_t* shares;
    int32_t* shares_out;
    int32_t* ring;
    const int64_t* ring_state;
    int64_t* ring_state_out;
    int32_t* lengths;
    int32_t* status;
    int32_t* copy_from;
    int32_t* copy_to;
    int32_t* copy_tokens;
    u32x4* rows;      // Row, in workspace
    mfh_u32* freed;   // pages per chunk that go back, and behind them the pages taken
    mfh_u32 requests, width, pages, ring_size, chunks, longest;
    Divider by_page, by_width;
};

// What the tables need to know of a request.
struct Row {
    mfh_u32 parent;  // kNone: the request is empty
    mfh_u32 take;    // tokens
    mfh_u32 fresh;   // page that its last tokens are copied to, or kNone
    mfh_u32 heir;    // of its own old pages, or kNone
};

MFH_DEV mfh_u32 pages_of(const ForkArgs& a, mfh_u32 tokens)
{
    const mfh_u32 whole = a.by_page.quotient(tokens);
    return whole + (whole * a.by_page.d != tokens);
}

// Tokens that a request had; none where its length cannot be.
MFH_DEV mfh_u32 had(const ForkArgs& a, mfh_u32 r)
{
    const int32_t b = a.before[r];
    return b < 0 || (mfh_u32)b > a.longest ? 0 : (mfh_u32)b;
}

struct FreePages {
    mfh_u32 count, head_at, tail_at;
    int64_t head, tail;
    __device__ FreePages(const ForkArgs& a) : head(a.ring_state[0]), tail(a.ring_state[1])
    {
        count = (mfh_u32)min(max(tail - head, (int64_t)0), (int64_t)a.ring_size);
        head_at = (mfh_u32)((uint64_t)head % a.ring_size);
        tail_at = (mfh_u32)((uint64_t)tail % a.ring_size);
    }
};

MFH_DEV mfh_u32 wrap(mfh_u32 at, mfh_u32 size) { return at >= size ? at - size : at; }

// Sum of v over the workgroup's threads before this one; `all` is that with every
// thread.  by_wave is free again behind the next barrier.
MFH_DEV mfh_u32 threads_before(mfh_u32 v, mfh_u32* by_wave, mfh_u32& all)
{
    const mfh_u32 upto = lanes_upto(v);
    if ((threadIdx.x & 63) == 63) by_wave[threadIdx.x >> 6] = upto;
    __syncthreads();
    mfh_u32 before = upto - v;
    all = 0;
#pragma unroll
    for (mfh_u32 w = 0; w < kWaves; w++) {
        const mfh_u32 s = by_wave[w];
        if (w < threadIdx.x >> 6) before += s;
        all += s;
    }
    return before;
}

// Everything that is there once per request: its results, and to(r, row) for the
// tables but for the heirs, which are in s_heir behind the next barrier.  Returns
// the number of pages taken.
template <int MOST, typename To>
MFH_DEV mfh_u32 plan(const ForkArgs& a, mfh_u32* s_first, mfh_u32* s_heir, mfh_u32* s_sum, To to)
{
    constexpr int kEach = MOST / kThreads;
    const FreePages free(a);
    mfh_u32 parent[kEach], take[kEach];
    bool part[kEach], bad[kEach], reaches[kEach];
    for (mfh_u32 r = threadIdx.x; r < a.requests; r += kThreads) s_first[r] = s_heir[r] = kNone;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        const mfh_u32 r = i * kThreads + threadIdx.x;
        parent[i] = kNone, take[i] = 0, part[i] = bad[i] = reaches[i] = false;
        if (i * kThreads >= a.requests || r >= a.requests) continue;
        const int32_t p = a.parents[r], most = a.keep ? max(a.keep[r], 0) : 0x7fffffff;
        if (p < 0) continue;
        const int32_t b = (mfh_u32)p < a.requests ? a.before[p] : -1;
        bad[i] = b < 0 || (mfh_u32)b > a.longest;
        if (bad[i]) continue;
        parent[i] = (mfh_u32)p;
        take[i] = (mfh_u32)min(b, most);
        const mfh_u32 row = a.by_page.quotient(take[i]);
        part[i] = row * a.by_page.d != take[i];
        reaches[i] = part[i] && row == a.by_page.quotient((mfh_u32)b);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; i++)
        if (reaches[i]) atomicMin(&s_first[parent[i]], i * kThreads + threadIdx.x);
    __syncthreads();
    mfh_u32 ahead = 0;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        if (i * kThreads >= a.requests) break;
        const mfh_u32 r = i * kThreads + threadIdx.x;
        const bool need = part[i] && !(reaches[i] && s_first[parent[i]] == r);
        mfh_u32 all;
        const mfh_u32 at = ahead + threads_before(need, s_sum, all);
        ahead += all;
        if (r < a.requests) {
            const bool refused = need && at >= free.count, copies = need && !refused;
            Row row{parent[i], take[i], kNone, kNone};
            if (refused) row.parent = kNone, row.take = 0;
            if (row.take == 0) row.parent = kNone;
            if (copies) row.fresh = (mfh_u32)a.ring[wrap(free.head_at + at, a.ring_size)];
            if (row.parent != kNone) atomicMin(&s_heir[row.parent], r);
            const mfh_u32 last = a.by_page.quotient(row.take);
            a.lengths[r] = (int32_t)row.take;
            a.status[r] = bad[i] ? 2 : refused ? 1 : 0;
            a.copy_from[r] = copies ? a.table[(int64_t)row.parent * a.table_stride + last] : -1;
            a.copy_to[r] = copies ? (int32_t)row.fresh : -1;
            a.copy_tokens[r] = copies ? (int32_t)(row.take - last * a.by_page.d) : 0;
            to(r, row, copies);
        }
        __syncthreads();
    }
    return min(ahead, free.count);
}

// Row r's new entry c, and what of the old one nobody takes over: page numbers
// are asked for in `load`, for several entries at a time, and dealt with in `finish`.
struct Entry {
    mfh_u32 r, c;
    bool write, drop, adds;
    int32_t from, old, fresh;
    // row: of r; heir: of r's heir, if it has one; first: whether r is its parent's heir
    MFH_DEV void load(const ForkArgs& a, mfh_u32 request, mfh_u32 entry, const Row& row, const Row& heir, bool first,
                      bool copies, bool heir_copies, mfh_u32 tokens_had)
    {
        r = request, c = entry;
        write = row.parent != kNone && c < pages_of(a, row.take);
        const bool is_copy = copies && c == a.by_page.quotient(row.take);
        adds = write && !first && !is_copy;
        drop = c < pages_of(a, tokens_had) &&
               (row.heir == kNone || c >= pages_of(a, heir.take) || (heir_copies && c == a.by_page.quotient(heir.take)));
        from = is_copy ? (int32_t)row.fresh : write ? a.table[(int64_t)row.parent * a.table_stride + c] : -1;
        old = drop ? a.table[(int64_t)r * a.table_stride + c] : -1;
    }
    template <typename Add>
    MFH_DEV void finish(const ForkArgs& a, Add add) const
    {
        if (write) a.table_out[(int64_t)r * a.table_stride + c] = from;
        if (adds && (mfh_u32)from < a.pages) add((mfh_u32)from, 1);
        if (drop && (mfh_u32)old < a.pages) add((mfh_u32)old, -1);
    }
};

constexpr int kEntries = 4;  // of a thread at a time

// One workgroup, counts in LDS.
__global__ __launch_bounds__(kThreads) void k_fork_few(ForkArgs a)
{
    __shared__ int32_t s_shares[kFewPages];
    __shared__ mfh_u32 s_parent[kFewRequests], s_take[kFewRequests], s_fresh[kFewRequests], s_had[kFewRequests];
    __shared__ mfh_u32 s_first[kFewRequests], s_heir[kFewRequests], s_sum[kWaves];
    __shared__ bool s_copies[kFewRequests];
    const mfh_u32 tid = threadIdx.x;
    for (mfh_u32 g = tid; g < a.pages; g += kThreads) s_shares[g] = max(a.shares[g], 0);
    for (mfh_u32 r = tid; r < a.requests; r += kThreads) s_had[r] = had(a, r);
    const mfh_u32 taken = plan<kFewRequests>(a, s_first, s_heir, s_sum, [&](mfh_u32 r, const Row& row, bool copies) {
        s_parent[r] = row.parent, s_take[r] = row.take, s_fresh[r] = row.fresh, s_copies[r] = copies;
    });
    __syncthreads();

    const mfh_u32 all = a.requests * a.width;
    for (mfh_u32 base = 0; base < all; base += kEntries * kThreads) {
        Entry e[kEntries];
#pragma unroll
        for (int k = 0; k < kEntries; k++) {
            const mfh_u32 at = base + k * kThreads + tid;
            const mfh_u32 r = at < all ? a.by_width.quotient(at) : 0, c = at < all ? at - r * a.width : kNone;
            const mfh_u32 heir = s_heir[r], h = heir == kNone ? r : heir;
            const Row row{s_parent[r], s_take[r], s_fresh[r], heir};
            const bool first = row.parent != kNone && s_heir[row.parent] == r;
            e[k].load(a, r, c, row, Row{0, s_take[h], 0, 0}, first, s_copies[r], s_copies[h], s_had[r]);
        }
#pragma unroll
        for (int k = 0; k < kEntries; k++) e[k].finish(a, [&](mfh_u32 page, int by) { atomicAdd(&s_shares[page], by); });
    }
    __syncthreads();

    // Pages that go back: a wave has a run of pages.
    const FreePages free(a);
    const int lane = tid & 63;
    const mfh_u32 run = ((a.pages + kWaves - 1) / kWaves + 63) & ~63u;
    const mfh_u32 begin = min((tid >> 6) * run, a.pages), end = min(begin + run, a.pages);
    mfh_u32 count = 0;
    for (mfh_u32 g = begin; g < end; g += 64)
        count += (mfh_u32)__popcll(__ballot(g + lane < end && s_shares[min(g + lane, end - 1)] < 0));
    mfh_u32 freed;
    mfh_u32 at = threads_before(lane == 63 ? count : 0, s_sum, freed);
    at = (mfh_u32)__builtin_amdgcn_readlane((int)at, 63);
    for (mfh_u32 g = begin; g < end; g += 64) {
        const bool in = g + lane < end;
        const int32_t left = s_shares[min(g + lane, end - 1)];
        const mfh_u64 gone = __ballot(in && left < 0);
        if (in) {
            a.shares_out[g + lane] = max(left, 0);
            const mfh_u32 place = at + (mfh_u32)__popcll(gone & (((mfh_u64)1 << lane) - 1));
            if (left < 0 && place < a.ring_size) a.ring[wrap(free.tail_at + place, a.ring_size)] = (int32_t)(g + lane);
        }
        at += (mfh_u32)__popcll(gone);
    }
    if (tid == 0) a.ring_state_out[0] = free.head + taken, a.ring_state_out[1] = free.tail + freed;
}

// Of many: the requests (workgroup 0), and the counts as they were.
__global__ __launch_bounds__(kThreads) void k_fork_plan(ForkArgs a)
{
    __shared__ mfh_u32 s_first[kMostRequests], s_heir[kMostRequests], s_sum[kWaves];
    if (blockIdx.x > 0) {
        const mfh_u32 g = (blockIdx.x - 1) * kChunk + 4 * threadIdx.x;
        for (mfh_u32 k = 0; k < 4 && g + k < a.pages; k++) a.shares_out[g + k] = max(a.shares[g + k], 0);
        return;
    }
    // (whether it copies is the sign of `take`)
    const mfh_u32 taken = plan<kMostRequests>(a, s_first, s_heir, s_sum, [&](mfh_u32 r, const Row& row, bool copies) {
        a.rows[r] = u32x4{row.parent, row.take | (copies ? 1u << 31 : 0u), row.fresh, kNone};
    });
    __syncthreads();
    for (mfh_u32 r = threadIdx.x; r < a.requests; r += kThreads) reinterpret_cast<mfh_u32*>(a.rows + r)[3] = s_heir[r];
    if (threadIdx.x == 0) a.freed[a.chunks] = taken;
}

constexpr int kRowThreads = 256;

__global__ __launch_bounds__(kRowThreads) void k_fork_rows(ForkArgs a, Divider by_parts)
{
    const mfh_u32 r = by_parts.quotient(blockIdx.x), part = blockIdx.x - r * by_parts.d;
    const u32x4 mine = a.rows[r];
    const mfh_u32 heir = mine[3], parent = mine[0];
    const mfh_u32 heir_take = heir != kNone ? a.rows[heir][1] : 0;
    const bool first = parent != kNone && a.rows[parent][3] == r;
    const mfh_u32 tokens_had = had(a, r);
    const Row row{parent, mine[1] & 0x7fffffffu, mine[2], heir};
    Entry e[kEntries];
#pragma unroll
    for (int k = 0; k < kEntries; k++)
        e[k].load(a, r, (part * kEntries + k) * kRowThreads + threadIdx.x, row, Row{0, heir_take & 0x7fffffffu, 0, 0}, first,
                  mine[1] >> 31, heir_take >> 31, tokens_had);
#pragma unroll
    for (int k = 0; k < kEntries; k++) e[k].finish(a, [&](mfh_u32 page, int by) { atomicAdd(&a.shares_out[page], by); });
}

// Which of a thread's four pages go back, and how many.
struct Gone {
    bool page[4];
    mfh_u32 count;
    MFH_DEV explicit Gone(const ForkArgs& a) : count(0)
    {
        const mfh_u32 g = blockIdx.x * kChunk + 4 * threadIdx.x;
        u32x4 left = {0, 0, 0, 0};
        if (g + 4 <= a.pages) {
            left = load16<false>(a.shares_out + g);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (g + k < a.pages) left[k] = (mfh_u32)a.shares_out[g + k];
        }
#pragma unroll
        for (int k = 0; k < 4; k++) page[k] = (int32_t)left[k] < 0, count += page[k];
    }
};

__global__ __launch_bounds__(kThreads) void k_fork_count(ForkArgs a)
{
    __shared__ mfh_u32 s_sum[kWaves];
    mfh_u32 all;
    threads_before(Gone(a).count, s_sum, all);
    if (threadIdx.x == 0) a.freed[blockIdx.x] = all;
}

__global__ __launch_bounds__(kThreads) void k_fork_return(ForkArgs a)
{
    __shared__ mfh_u32 s_sum[kWaves], s_more[kWaves];
    const mfh_u32 mine = a.freed[blockIdx.x];
    if (mine == 0 && blockIdx.x > 0) return;
    const FreePages free(a);
    mfh_u32 before = 0, total;
    for (mfh_u32 c = threadIdx.x; c < (blockIdx.x > 0 ? blockIdx.x : a.chunks); c += kThreads) before += a.freed[c];
    threads_before(before, s_sum, total);  // all chunks' in workgroup 0, else those of the chunks before
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.ring_state_out[0] = free.head + a.freed[a.chunks];
        a.ring_state_out[1] = free.tail + total;
    }
    if (mine == 0) return;
    const mfh_u32 g = blockIdx.x * kChunk + 4 * threadIdx.x;
    const Gone gone(a);
    mfh_u32 all;
    mfh_u32 at = (blockIdx.x > 0 ? total : 0) + threads_before(gone.count, s_more, all);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (!gone.page[k]) continue;
        a.shares_out[g + k] = 0;
        if (at < a.ring_size) a.ring[wrap(free.tail_at + at, a.ring_size)] = (int32_t)(g + k);
        at++;
    }
}

size_t fork_workspace(int32_t requests, int64_t pages)
{
    return (size_t)requests * sizeof(u32x4) + ((size_t)(pages + kChunk - 1) / kChunk + 1) * sizeof(mfh_u32);
}

// ---- copies of pages ------------------------------------------------------------

// A page's rows (one token of one head) in pieces of 16 bytes, in the order in
// which they stand in memory; a workgroup takes kPieces * kCopyThreads of them.
// Memory bounds it: 1000 pages of 64 tokens, 8 heads of 128 e4m3 (262 MB read and
// written) take 52 us, 5.0 TB/s, what a large copy reaches; a step's 64 pages 3.5 us.
constexpr int kCopyThreads = 256;
constexpr int kPieces = 4;

struct CopyArgs {
    char* cache[2];
    const int32_t* from;
    const int32_t* to;
    const int32_t* tokens;
    int64_t page_bytes, head_bytes, token_bytes;
    mfh_u32 pages, page_size, items;  // items: pieces of a page
    mfh_u32 row_pieces;
    bool heads_outside;
    Divider by_outer, by_row, by_parts, by_sides;
};

__global__ __launch_bounds__(kCopyThreads) void k_page_copy(CopyArgs a)
{
    const mfh_u32 unit = a.by_parts.quotient(blockIdx.x), part = blockIdx.x - unit * a.by_parts.d;
    const mfh_u32 pair = a.by_sides.quotient(unit), side = unit - pair * a.by_sides.d;
    const mfh_u32 from = (mfh_u32)a.from[pair], to = (mfh_u32)a.to[pair];
    if (from >= a.pages || to >= a.pages || from == to) return;
    const mfh_u32 tokens = a.tokens ? (mfh_u32)min(max(a.tokens[pair], 0), (int)a.page_size) : a.page_size;
    char* cache = a.cache[side];
    const char* source = cache + (int64_t)from * a.page_bytes;
    char* target = cache + (int64_t)to * a.page_bytes;
    u32x4 piece[kPieces];
    int64_t at[kPieces];
#pragma unroll
    for (int k = 0; k < kPieces; k++) {
        const mfh_u32 item = (part * kPieces + k) * kCopyThreads + threadIdx.x;
        const mfh_u32 outer = a.by_outer.quotient(item), inner = item - outer * a.by_outer.d;
        const mfh_u32 row = a.by_row.quotient(inner), in_row = inner - row * a.row_pieces;
        const mfh_u32 token = a.heads_outside ? row : outer, head = a.heads_outside ? outer : row;
        at[k] = item < a.items && token < tokens ? token * a.token_bytes + head * a.head_bytes + in_row * 16 : -1;
        if (at[k] >= 0) piece[k] = load16<true>(source + at[k]);
    }
#pragma unroll
    for (int k = 0; k < kPieces; k++)
        if (at[k] >= 0) store16(target + at[k], piece[k]);
}

}  // namespace
}  // namespace mfh

using namespace mfh;

extern "C" {

int mfh_page_fork_workspace(int32_t requests, int64_t pages, size_t* bytes)
{
    const char* what = "mfh_page_fork_workspace";
    if (requests < 0 || requests > (int32_t)kMostRequests)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d requests are not within 0..%u", what, requests, kMostRequests);
    if (pages < 1 || pages > kLongest)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %lld pages are not within 1..2^30", what, (long long)pages);
    if (!bytes) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL result", what);
    *bytes = fork_workspace(requests, pages);
    return MFH_OK;
}

int mfh_page_fork(const int32_t* parents, const int32_t* before, const int32_t* keep, int32_t requests,
                  int32_t page_size, const int32_t* table, int32_t* table_out, int64_t table_stride,
                  int32_t table_width, const int32_t* shares, int32_t* shares_out, int64_t pages, int32_t* ring,
                  int64_t ring_size, const int64_t* ring_state, int64_t* ring_state_out, int32_t* lengths,
                  int32_t* status, int32_t* copy_from, int32_t* copy_to, int32_t* copy_tokens, void* workspace,
                  size_t workspace_bytes, void* stream)
{
    const char* what = "mfh_page_fork";
    const Device* dev;
    MFH_TRY(bind_device(&dev));
    size_t need;
    MFH_TRY(mfh_page_fork_workspace(requests, pages, &need));
    if (page_size < 1) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: page size %d is not positive", what, page_size);
    if (table_width < 0 || table_stride < table_width)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: table width %d does not fit its stride %lld", what, table_width,
                    (long long)table_stride);
    if (ring_size < pages || ring_size > kLongest)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: a ring of %lld pages is not within the cache's %lld..2^30", what,
                    (long long)ring_size, (long long)pages);
    if (!shares || !shares_out || !ring || !ring_state || !ring_state_out ||
        (requests > 0 && (!parents || !before || !lengths || !status || !copy_from || !copy_to || !copy_tokens ||
                          (table_width > 0 && (!table || !table_out)))))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL buffer", what);
    auto overlap = [](const void* p, int64_t p_bytes, const void* q, int64_t q_bytes) {
        return (uintptr_t)p < (uintptr_t)q + q_bytes && (uintptr_t)q < (uintptr_t)p + p_bytes;
    };
    if (overlap(ring_state, 16, ring_state_out, 16))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: ring_state_out overlaps ring_state, which other workgroups still read",
                    what);
    const int64_t row_bytes = (int64_t)requests * 4;
    const int64_t table_bytes = requests > 0 && table_width > 0 ? ((requests - 1) * table_stride + table_width) * 4 : 0;
    if (table_bytes && overlap(table, table_bytes, table_out, table_bytes))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: table_out overlaps table, which is still read", what);
    const struct { const char* name; const int32_t* at; } results[] = {
        {"lengths", lengths}, {"status", status}, {"copy_from", copy_from}, {"copy_to", copy_to}, {"copy_tokens", copy_tokens}};
    for (const auto& r : results) {
        if (requests > 0 && overlap(r.at, row_bytes, before, row_bytes))
            return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %s overlaps before, which is still read", what, r.name);
        if (table_bytes && overlap(r.at, row_bytes, table, table_bytes))
            return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %s overlaps table, which is still read", what, r.name);
    }
    if (shares != shares_out && overlap(shares, pages * 4, shares_out, pages * 4))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: shares_out overlaps shares without being it", what);
    if (workspace_bytes < need || !workspace || (uintptr_t)workspace % 16)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: a workspace of %zu bytes is NULL, not 16-byte aligned or less than %zu",
                    what, workspace_bytes, need);
    ForkArgs a{parents, before, keep, table, table_out, table_stride, shares, shares_out, ring, ring_state,
               ring_state_out, lengths, status, copy_from, copy_to, copy_tokens};
    a.requests = (mfh_u32)requests, a.width = (mfh_u32)table_width, a.pages = (mfh_u32)pages;
    a.ring_size = (mfh_u32)ring_size, a.chunks = (mfh_u32)((pages + kChunk - 1) / kChunk);
    a.longest = (mfh_u32)std::min<int64_t>((int64_t)table_width * page_size, 0x7fffffff);
    a.rows = (u32x4*)workspace, a.freed = (mfh_u32*)(a.rows + requests);
    a.by_page = Divider((mfh_u32)page_size), a.by_width = Divider((mfh_u32)std::max(table_width, 1));
    hipStream_t s = (hipStream_t)stream;
    if (requests <= (int32_t)kFewRequests && pages <= (int64_t)kFewPages && (int64_t)requests * table_width <= kFewEntries) {
        k_fork_few<<<1, kThreads, 0, s>>>(a);
        return launch_status("k_fork_few");
    }
    const Divider parts((mfh_u32)std::max<int64_t>(1, ((int64_t)table_width + kEntries * kRowThreads - 1) / (kEntries * kRowThreads)));
    if ((int64_t)requests * parts.d >= (int64_t(1) << 32) / kRowThreads)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d requests of %d pages are too many for one call", what, requests,
                    table_width);
    k_fork_plan<<<1 + a.chunks, kThreads, 0, s>>>(a);
    MFH_TRY(launch_status("k_fork_plan"));
    if (requests > 0) {
        k_fork_rows<<<(unsigned)requests * parts.d, kRowThreads, 0, s>>>(a, parts);
        MFH_TRY(launch_status("k_fork_rows"));
    }
    k_fork_count<<<a.chunks, kThreads, 0, s>>>(a);
    MFH_TRY(launch_status("k_fork_count"));
    k_fork_return<<<a.chunks, kThreads, 0, s>>>(a);
    return launch_status("k_fork_return");
}

int mfh_page_copy(const mfh_kv_cache* cache, int32_t pairs, const int32_t* from, const int32_t* to,
                  const int32_t* tokens, void* k_cache, void* v_cache, void* stream)
{
    const char* what = "mfh_page_copy";
    const Device* dev;
    MFH_TRY(bind_device(&dev));
    MFH_TRY(check_cache(cache, what));
    if (pairs < 0) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: negative number of pairs %d", what, pairs);
    if (pairs == 0) return MFH_OK;
    if (!from || !to || (!k_cache && !v_cache)) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL buffer", what);
    const int bytes = cache->dtype == kF8E4M3 ? 1 : 2;
    CopyArgs a{};
    a.cache[0] = (char*)(k_cache ? k_cache : v_cache), a.cache[1] = (char*)v_cache;
    a.from = from, a.to = to, a.tokens = tokens;
    a.page_bytes = cache->page_stride * bytes, a.head_bytes = cache->head_stride * bytes;
    a.token_bytes = cache->token_stride * bytes;
    a.pages = (mfh_u32)cache->pages, a.page_size = (mfh_u32)cache->page_size;
    a.row_pieces = (mfh_u32)(cache->head_dim * bytes / 16);
    a.heads_outside = cache->head_stride >= cache->token_stride;
    const int64_t items = (int64_t)cache->kv_heads * cache->page_size * a.row_pieces;
    const int64_t parts = (items + kPieces * kCopyThreads - 1) / (kPieces * kCopyThreads);
    const int sides = k_cache && v_cache ? 2 : 1;
    if (items > kLongest || (__int128)parts * sides * pairs >= (int64_t(1) << 32) / kCopyThreads)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d pairs of %lld pieces of 16 bytes are too many for one call", what,
                    pairs, (long long)items);
    a.items = (mfh_u32)items;
    a.by_outer = Divider((mfh_u32)(a.heads_outside ? cache->page_size : cache->kv_heads) * a.row_pieces);
    a.by_row = Divider(a.row_pieces), a.by_parts = Divider((mfh_u32)parts), a.by_sides = Divider((mfh_u32)sides);
    k_page_copy<<<(unsigned)(parts * sides * pairs), kCopyThreads, 0, (hipStream_t)stream>>>(a);
    return launch_status("k_page_copy");
}

}  // extern "C"
