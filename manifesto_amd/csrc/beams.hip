// beams.hip — beam search's selection (mfh_beam_select): the best continuations
// of a group's beams over the vocabulary.
//
// score(b, t) = s_b + l_bt - log sum_u exp(l_bu).  The logits are read once, and
// bytes bound it: 2 or 4 a logit, beside some nine vector operations, one of
// them an exponential.
//
// k_beam_rows: a workgroup keeps a piece of a row in registers, packed as it
// was read, and leaves the piece's largest logit, the sum of the exponentials
// below it and its `picks` largest logits.  These are found without sorting:
// each thread's largest, then the largest of each of 64 columns of threads, and
// the picks-th largest of those is a bound that `picks` elements reach and that
// few others do.  What reaches it is listed in LDS and ranked there by counting.
// Logits are compared together with their tokens, so no two are equal and rows
// of one value (masked ones) list no more than others.  An order that puts very
// many large logits into few columns overflows the list; then the largest is
// taken `picks` times.
//
// k_beam_merge: a group's pieces meet.  Scores of different beams can be closer
// than f32 tells apart, so that sums of a row's pieces, logarithms and scores
// are in f64; inside a piece an exponential's error is that of its argument's
// rounding, 2^-25 of |l - max| log2(e), which the sum averages to about 1e-8.
// The histories' rows are cut over several workgroups, each of which merges
// again: that costs less than one more launch.
//
// A step of few rows is two launches' latency: 4 rows of 32003 f32 6.2 and 5.7 us.
// 256 rows of 131072 bf16 (67 MB, 13 us at a copy's rate) take 20.4 and 7.1: their
// 1024 workgroups are what the card holds at once, all of which load and then all
// compute the exponentials, the bound and the list.  With a quarter of the beams
// ended (50 MB) they take 20.0 and 7.2, for the others' pieces are no faster.
#include "common.hpp"
#include "launch.hpp"
#include "paged.hpp"
#include "../../include/mfh_beams.h"

namespace mfh {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kMostPicks = 64;   // columns of threads
constexpr int kMostBeams = 256;
constexpr int kTokenBits = 24;
constexpr int kList = 1024;

struct BeamArgs {
    const char* logits;
    const float* scores;
    const uint8_t* ended;
    float* scores_out;
    int32_t* tokens;
    int32_t* parents;
    uint8_t* ended_out;
    const int32_t* history;
    const int32_t* known;
    int32_t* history_out;
    mfh_u64* best;    // [rows][pieces][picks], Keys of logits, largest first; 0: none
    double* sums;     // [rows][pieces]
    float* tops;      // [rows][pieces]
    int64_t row_bytes, history_stride;
    mfh_u32 beams, picks, vocab, pieces, slices;
    int32_t end_token;
    Divider by_pieces, by_picks, by_slices, by_piece;  // by_piece: tokens of a piece
};

// A float as a whole number of the same order; -0 is 0.
MFH_DEV mfh_u32 ordered(float x)
{
    const mfh_u32 bits = mfh_bits(x + 0.0f);
    return bits ^ ((mfh_u32)((mfh_i32)bits >> 31) | 0x80000000u);
}

MFH_DEV float unordered(mfh_u32 o) { return mfh_f32(o ^ ((mfh_u32)((mfh_i32)~o >> 31) | 0x80000000u)); }

MFH_DEV mfh_u64 ordered(double x)
{
    const mfh_u64 bits = __builtin_bit_cast(mfh_u64, x + 0.0);
    return bits ^ ((mfh_u64)((mfh_i64)bits >> 63) | (mfh_u64)1 << 63);
}

MFH_DEV double unordered(mfh_u64 o) { return __builtin_bit_cast(double, o ^ ((mfh_u64)((mfh_i64)~o >> 63) | (mfh_u64)1 << 63)); }

// A logit with its token: larger is better, and no two are equal.
MFH_DEV mfh_u64 logit_key(float x, mfh_u32 token) { return (mfh_u64)ordered(x) << 32 | (mfh_u32)~token; }

// A continuation in its order; `low` holds beam, logit and token.
struct Key {
    mfh_u64 high, low;
    MFH_DEV bool operator>(const Key& o) const { return high > o.high || (high == o.high && low > o.low); }
    MFH_DEV bool operator>=(const Key& o) const { return !(o > *this); }
    MFH_DEV bool some() const { return low != 0; }
    // (member by member: a choice between two keys as such goes through memory)
    static MFH_DEV Key choose(bool first, const Key& a, const Key& b) { return Key{first ? a.high : b.high, first ? a.low : b.low}; }
    static MFH_DEV Key none() { return Key{0, 0}; }
    static MFH_DEV Key all() { return Key{~(mfh_u64)0, ~(mfh_u64)0}; }
    MFH_DEV Key from_lane(int mask) const
    {
        return Key{(mfh_u64)__shfl_xor((unsigned long long)high, mask), (mfh_u64)__shfl_xor((unsigned long long)low, mask)};
    }
};

// The same interface for a logit's key.
struct Logit {
    mfh_u64 key;
    MFH_DEV bool operator>(const Logit& o) const { return key > o.key; }
    MFH_DEV bool operator>=(const Logit& o) const { return key >= o.key; }
    MFH_DEV bool some() const { return key != 0; }
    static MFH_DEV Logit none() { return Logit{0}; }
    static MFH_DEV Logit all() { return Logit{~(mfh_u64)0}; }
    MFH_DEV Logit from_lane(int mask) const { return Logit{(mfh_u64)__shfl_xor((unsigned long long)key, mask)}; }
};

// The `picks` largest of a workgroup's elements, in order, into `best` behind a
// barrier.  each(least, f) calls f for every element of the thread, but may leave out
// lower ones than `least`, and all others once f has returned false; top is the
// largest.  `attempt` is false, with nothing done, where no bound is found or
// more than the list holds reach it.
template <typename K>
struct Selection {
    K by_wave[kWaves][64];
    K column[64];
    K list[kList];
    mfh_u32 rank[64];
    K bound;
    mfh_u32 count;

    template <typename Each>
    MFH_DEV bool attempt(mfh_u32 picks, K top, K* best, Each each, bool needs_bound = true)
    {
        const mfh_u32 tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        by_wave[wave][lane] = top;
        if (tid < 64) rank[tid] = 0;
        if (tid == 0) bound = K::none(), count = 0;
        for (mfh_u32 i = tid; i < picks; i += kThreads) best[i] = K::none();
        __syncthreads();
        if (wave == 0) {
            K most = top;
#pragma unroll
            for (int w = 1; w < kWaves; w++)
                if (by_wave[w][lane] > most) most = by_wave[w][lane];
            column[lane] = most;
        }
        __syncthreads();
        const K mine = column[lane];
        mfh_u32 above = 0;
#pragma unroll
        for (int i = 0; i < 64 / kWaves; i++) above += column[wave * (64 / kWaves) + i] > mine;
        atomicAdd(&rank[lane], above);
        __syncthreads();
        if (wave == 0 && rank[lane] == picks - 1) bound = mine;  // with fewer columns than picks none: everything is listed
        __syncthreads();
        const K least = bound;
        if (needs_bound && !least.some()) return false;
        if (top.some() && top >= least)
            each(least, [&](K k) {
                if (!k.some() || !(k >= least)) return true;
                const mfh_u32 at = atomicAdd(&count, 1u);
                if (at < kList) list[at] = k;
                return at < kList;
            });
        __syncthreads();
        const mfh_u32 n = count;
        if (n > kList) return false;
        for (mfh_u32 i = tid; i < n; i += kThreads) {
            const K k = list[i];
            mfh_u32 before = 0;
            for (mfh_u32 j = 0; j < n; j++) before += list[j] > k;
            if (before < picks) best[before] = k;
        }
        return true;
    }

    // One after the other where the attempt fails.
    template <typename Each>
    MFH_DEV void run(mfh_u32 picks, K top, K* best, Each each)
    {
        if (attempt(picks, top, best, each, false)) return;
        const mfh_u32 tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        K last = K::all();
        for (mfh_u32 i = 0; i < picks; i++) {
            K most = K::none();
            each(K::none(), [&](K k) {
                if (last > k && k > most) most = k;
                return true;
            });
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) {
                const K other = most.from_lane(x);
                if (other > most) most = other;
            }
            __syncthreads();
            if (lane == 0) column[wave] = most;
            __syncthreads();
            last = column[0];
#pragma unroll
            for (int w = 1; w < kWaves; w++)
                if (column[w] > last) last = column[w];
            if (tid == 0) best[i] = last;
            if (!last.some()) break;
        }
    }
};

template <int DT>
constexpr int kPacket = DT == kFloat32 ? 4 : 8;  // logits of 16 bytes

template <int DT>
MFH_DEV float logit_of(const u32x4& p, int e)
{
    if constexpr (DT == kFloat32) return mfh_f32(p[e]);
    else return dec16<DT>(e & 1 ? p[e / 2] >> 16 : p[e / 2] & 0xffffu);
}

// PACKETS: of 16 bytes in a thread's registers.
template <int DT, int PACKETS>
__global__ __launch_bounds__(kThreads, 8) void k_beam_rows(BeamArgs a)
{
    constexpr int P = kPacket<DT>, kBytes = 16 / P;
    __shared__ Selection<Logit> s;
    __shared__ Logit s_best[kMostPicks];
    __shared__ float s_top[kWaves];
    __shared__ double s_sum[kWaves];

    const mfh_u32 row = a.by_pieces.quotient(blockIdx.x), piece = blockIdx.x - row * a.pieces;
    if (a.ended && a.ended[row]) return;  // its logits do not matter
    const char* from = a.logits + (int64_t)row * a.row_bytes;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    auto token_of = [&](int i) { return ((piece * PACKETS + i) * kThreads + threadIdx.x) * P; };

    u32x4 packet[PACKETS];
    if ((mfh_u64)(piece + 1) * (PACKETS * kThreads * P) <= a.vocab) {
#pragma unroll
        for (int i = 0; i < PACKETS; i++) packet[i] = load16<true>(from + (int64_t)token_of(i) * kBytes);
    } else {  // a row's last piece: -inf past its end
        constexpr mfh_u32 kLowest = DT == kFloat32 ? 0xff800000u : DT == kBFloat16 ? 0xff80ff80u : 0xfc00fc00u;
#pragma unroll
        for (int i = 0; i < PACKETS; i++) {
            const mfh_u32 t = token_of(i);
            packet[i] = u32x4{kLowest, kLowest, kLowest, kLowest};
            if (t + P <= a.vocab) {
                packet[i] = load16<true>(from + (int64_t)t * kBytes);
            } else if (t < a.vocab) {
#pragma unroll
                for (int e = 0; e < P; e++) {
                    if (t + e >= a.vocab) continue;
                    if constexpr (DT == kFloat32) packet[i][e] = load4(from + (int64_t)(t + e) * 4);
                    else packet[i][e / 2] = e & 1 ? (packet[i][e / 2] & 0xffffu) | load2(from + (int64_t)(t + e) * 2) << 16
                                                  : (packet[i][e / 2] & 0xffff0000u) | load2(from + (int64_t)(t + e) * 2);
                }
            }
        }
    }

    // the thread's largest logit, and the first packet that has it
    float top = -INFINITY;
    int at = 0;
#pragma unroll
    for (int i = 0; i < PACKETS; i++) {
        float most = logit_of<DT>(packet[i], 0);
#pragma unroll
        for (int e = 1; e < P; e++) most = fmaxf(most, logit_of<DT>(packet[i], e));
        if (most > top) top = most, at = i;
    }
    // (unpacked anew for each of its uses: kept unpacked, a workgroup's registers would
    // leave room for no other one)
    auto packed = [&]() {
#pragma unroll
        for (int i = 0; i < PACKETS; i++) asm volatile("" : "+v"(packet[i]));
    };
    packed();
    // sum of exponentials below the wave's largest; NaN and +inf make it NaN
    float wave_top = top;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) wave_top = fmaxf(wave_top, __shfl_xor(wave_top, x));
    const float base = wave_top == -INFINITY ? 0.0f : wave_top;
    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < PACKETS; i++) {
#pragma unroll
        for (int e = 0; e < P; e++) part[e % 4] += exp2_fast((logit_of<DT>(packet[i], e) - base) * kLog2e);
    }
    packed();
    double sum = (double)(part[0] + part[1]) + (double)(part[2] + part[3]);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
    if (lane == 0) s_top[wave] = wave_top, s_sum[wave] = sum;

    u32x4 with_top = packet[0];
#pragma unroll
    for (int i = 1; i < PACKETS; i++) with_top = at == i ? packet[i] : with_top;
    int in_packet = 0;
#pragma unroll
    for (int e = P - 1; e >= 0; e--) in_packet = logit_of<DT>(with_top, e) == top ? e : in_packet;
    const Logit best{top > -INFINITY ? logit_key(top, token_of(at) + in_packet) : 0};
    s.run(a.picks, best, s_best, [&](const Logit& least, auto f) {
        const float above = least.some() ? unordered((mfh_u32)(least.key >> 32)) : -INFINITY;
#pragma unroll
        for (int i = 0; i < PACKETS; i++) {
            float most = logit_of<DT>(packet[i], 0);
#pragma unroll
            for (int e = 1; e < P; e++) most = fmaxf(most, logit_of<DT>(packet[i], e));
            if (!(most >= above)) continue;
            mfh_u32 token = token_of(i);
            asm volatile("" : "+v"(packet[i]), "+v"(token));  // nothing of it ahead of the question
#pragma unroll
            for (int e = 0; e < P; e++) {
                const float x = logit_of<DT>(packet[i], e);
                if (x > -INFINITY) f(Logit{logit_key(x, token + e)});
            }
        }
    });
    __syncthreads();
    if (threadIdx.x < a.picks) a.best[(int64_t)blockIdx.x * a.picks + threadIdx.x] = s_best[threadIdx.x].key;
    if (threadIdx.x == 0) {
        float most = s_top[0];
#pragma unroll
        for (int w = 1; w < kWaves; w++) most = fmaxf(most, s_top[w]);
        double all = 0.0;
#pragma unroll
        for (int w = 0; w < kWaves; w++)
            all += s_top[w] == -INFINITY ? s_sum[w] : exp((double)s_top[w] - (double)most) * s_sum[w];  // 0, or NaN
        a.tops[blockIdx.x] = most;
        a.sums[blockIdx.x] = all;
    }
}

// FLAT: a group's candidates are two a thread at most.
template <bool FLAT>
__global__ __launch_bounds__(kThreads) void k_beam_merge(BeamArgs a)
{
    __shared__ Selection<Key> s;
    __shared__ Key s_best[kMostPicks];
    __shared__ double s_score[kMostBeams], s_norm[kMostBeams];
    __shared__ bool s_ended[kMostBeams];
    const mfh_u32 group = a.by_slices.quotient(blockIdx.x), slice = blockIdx.x - group * a.slices;
    const mfh_u32 row0 = group * a.beams;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

    // Up to two candidates a thread are taken at once.  Of more the heads come first: a
    // piece's list is in order, and its head says whether the rest matters (2 groups of 8
    // beams, 16 picks from 42 pieces each: 8.4 us, all at once 22; 3 groups of 16
    // beams, 32 picks from one piece: 11 us, by the heads 35).  The first ones are
    // on their way during the logarithms.
    const mfh_u32 lists = a.beams * a.pieces;
    const mfh_u64* keys = a.best + (int64_t)row0 * a.pieces * a.picks;
    const mfh_u32 firsts = FLAT ? lists * a.picks : lists;
    mfh_u64 first[2];
#pragma unroll
    for (mfh_u32 i = 0; i < 2; i++) {
        const mfh_u32 n = threadIdx.x + i * kThreads;
        first[i] = n < firsts ? keys[FLAT ? n : (int64_t)n * a.picks] : 0;
    }
    // the logarithm of each beam's sum, a wave each
    for (mfh_u32 b = wave; b < a.beams; b += kWaves) {
        const mfh_u32 row = row0 + b;
        const bool ended = a.ended && a.ended[row];
        const float* tops = a.tops + (int64_t)row * a.pieces;
        const double* sums = a.sums + (int64_t)row * a.pieces;
        float top = -INFINITY;
        double sum = 0.0;
        if (!ended) {
            const bool some = (mfh_u32)lane < a.pieces;
            const float mine = some ? tops[lane] : -INFINITY;
            const double its = some ? sums[lane] : 0.0;
            top = mine;
            for (mfh_u32 n = lane + 64; n < a.pieces; n += 64) top = fmaxf(top, tops[n]);
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
            auto add = [&](float t, double s) { sum += t == -INFINITY ? s : exp((double)t - (double)top) * s; };
            add(mine, its);
            for (mfh_u32 n = lane + 64; n < a.pieces; n += 64) add(tops[n], sums[n]);
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
        }
        if (lane == 0) {
            s_ended[b] = ended;
            s_score[b] = (double)a.scores[row];
            s_norm[b] = (double)top + log(sum);
        }
    }
    __syncthreads();

    auto candidate = [&](mfh_u32 list, mfh_u32 i, mfh_u64 key) {
        const mfh_u32 b = a.by_pieces.quotient(list), piece = list - b * a.pieces;
        double score;
        if (s_ended[b]) {
            if (piece > 0 || i > 0) return Key::none();
            key = (mfh_u64)0xffffffffu << 32 | (mfh_u32)~a.end_token;
            score = s_score[b];
        } else {
            if (key == 0) return Key::none();
            score = s_score[b] + ((double)unordered((mfh_u32)(key >> 32)) - s_norm[b]);
        }
        if (!(score > -INFINITY && score < INFINITY)) return Key::none();
        const mfh_u64 low = (mfh_u64)(kMostBeams - 1 - b) << 56 | (key >> 32) << kTokenBits | (key & ((1u << kTokenBits) - 1));
        return Key{ordered(score), low};
    };
    Key mine[2], top = Key::none();
#pragma unroll
    for (mfh_u32 i = 0; i < 2; i++) {
        const mfh_u32 n = threadIdx.x + i * kThreads, list = FLAT ? a.by_picks.quotient(n) : n;
        mine[i] = Key::none();
        if (n < firsts) mine[i] = candidate(list, FLAT ? n - list * a.picks : 0, first[i]);
        top = Key::choose(mine[i] > top, mine[i], top);
    }
    if constexpr (FLAT) {
        s.run(a.picks, top, s_best, [&](const Key&, auto f) {
#pragma unroll
            for (mfh_u32 i = 0; i < 2; i++)
                if (mine[i].some()) f(mine[i]);
        });
    } else {
        for (mfh_u32 list = threadIdx.x + 2 * kThreads; list < lists; list += kThreads) {
            const Key k = candidate(list, 0, keys[(int64_t)list * a.picks]);
            top = Key::choose(k > top, k, top);
        }
        // From the heads on, each list as far as the bound goes.
        const bool done = s.attempt(a.picks, top, s_best, [&](const Key& least, auto f) {
            for (mfh_u32 list = threadIdx.x; list < lists; list += kThreads) {
                Key k = Key::choose(list < kThreads, mine[0], mine[1]);
                if (list >= 2 * kThreads) k = candidate(list, 0, keys[(int64_t)list * a.picks]);
                for (mfh_u32 i = 1; k.some() && !(least > k); i++) {
                    if (!f(k)) return;
                    if (i == a.picks) break;
                    k = candidate(list, i, keys[(int64_t)list * a.picks + i]);
                }
            }
        });
        if (!done) {
            // Fewer lists than picks, or heads far apart, give no bound that leaves few.  Then
            // the best heads, and of what is behind them what can be among the best: entry i
            // behind the j-th head has i + j others before it (3 groups of 31 beams, 62 picks
            // of 68 tokens: 27 us, one pick after the other 1030; 256 beams, 64 picks of 32000
            // f16: 114 and 960; asked first of every call, 4 us more where the heads suffice).
            __syncthreads();
            s.run(a.picks, top, s_best, [&](const Key&, auto f) {
                for (mfh_u32 list = threadIdx.x; list < lists; list += kThreads) {
                    Key k = Key::choose(list < kThreads, mine[0], mine[1]);
                    if (list >= 2 * kThreads) k = candidate(list, 0, keys[(int64_t)list * a.picks]);
                    f(k);
                }
            });
            __syncthreads();
            // (another i in a lane for each head: a column of threads has some of every rank)
            constexpr int kEach = kMostPicks / kWaves;
            auto place = [&](int e) { return (mfh_u32)(lane - 29 * (wave + e * kWaves)) & (kMostPicks - 1); };
            mfh_u64 entry[kEach];
            mfh_u32 from[kEach];
            Key some[kEach];
#pragma unroll
            for (int e = 0; e < kEach; e++) {
                const mfh_u32 j = wave + e * kWaves, i = place(e);
                some[e] = Key::none(), entry[e] = 0, from[e] = 0;
                if (i + j >= a.picks) continue;
                const Key head = s_best[j];
                if (i == 0) some[e] = head;
                const mfh_u32 b = kMostBeams - 1 - (mfh_u32)(head.low >> 56);
                if (i == 0 || !head.some() || s_ended[b]) continue;
                from[e] = b * a.pieces + a.by_piece.quotient(~(mfh_u32)head.low & ((1u << kTokenBits) - 1));
                entry[e] = keys[(int64_t)from[e] * a.picks + i];
            }
            top = Key::none();
#pragma unroll
            for (int e = 0; e < kEach; e++) {
                if (entry[e] != 0) some[e] = candidate(from[e], place(e), entry[e]);
                top = Key::choose(some[e] > top, some[e], top);
            }
            __syncthreads();
            s.run(a.picks, top, s_best, [&](const Key&, auto f) {
#pragma unroll
                for (int e = 0; e < kEach; e++)
                    if (some[e].some()) f(some[e]);
            });
        }
    }
    __syncthreads();

    auto token_of = [](const Key& k) { return k.some() ? (int32_t)(~k.low & ((1u << kTokenBits) - 1)) : -1; };
    auto parent_of = [&](const Key& k) { return k.some() ? (int32_t)(row0 + (kMostBeams - 1 - (mfh_u32)(k.low >> 56))) : -1; };
    if (slice == 0 && threadIdx.x < a.picks) {
        const Key k = s_best[threadIdx.x];
        const mfh_u32 at = group * a.picks + threadIdx.x;
        const int32_t token = token_of(k), parent = parent_of(k);
        a.scores_out[at] = k.some() ? (float)unordered(k.high) : -INFINITY;
        a.tokens[at] = token;
        a.parents[at] = parent;
        if (a.ended_out) a.ended_out[at] = k.some() && (s_ended[parent - (int32_t)row0] || token == a.end_token);
    }
    if (!a.history) return;
    const int64_t known = min((int64_t)max(a.known[group], 0), a.history_stride);
    const int64_t share = (known + 1 + a.slices - 1) / a.slices, begin = slice * share;
    const int64_t end = min(begin + share, min(known + 1, a.history_stride));
    for (mfh_u32 i = wave; i < a.picks; i += kWaves) {
        const Key k = s_best[i];
        if (!k.some()) continue;
        const int32_t* old = a.history + (int64_t)parent_of(k) * a.history_stride;
        int32_t* to = a.history_out + (int64_t)(group * a.picks + i) * a.history_stride;
#pragma unroll 4
        for (int64_t c = begin + lane; c < end; c += 64) to[c] = c < known ? old[c] : token_of(k);
    }
}

// Packets of a thread: as many as leave every CU two workgroups, for what a
// workgroup does once (the bound, the list) costs the same whatever its piece.
// 256 rows of 131072 bf16: by 8 packets 27 us, by 1 47; 256 of 32000: by 4 as here
// 18.0, by 8 18.7, by 2 18.5; 35 rows of 50001 f16: by 1 12.8 us, by 8 16.  In between
// one more doubling can be 5% faster: 64 rows of 32003 f32 by 2 as here 14.2, by 4 13.6.
struct Layout {
    int packets;
    int64_t pieces;
    size_t bytes;
};

Layout layout(const Device* dev, const mfh_beam_shape& sh, int32_t groups)
{
    Layout l{};
    const int64_t rows = (int64_t)groups * sh.beams;
    auto pieces_by = [&](int packets) {
        const int64_t piece = (int64_t)kThreads * packets * (sh.dtype == kFloat32 ? 4 : 8);
        return (sh.vocab + piece - 1) / piece;
    };
    l.packets = 8;
    while (l.packets > 1 && rows * pieces_by(l.packets) < 2 * dev->compute_units) l.packets /= 2;
    l.pieces = pieces_by(l.packets);
    // Room for all smaller calls too, whose rows may be in more pieces: less than 2 * cus
    // of twice the packets are less than 4 * cus.
    const int64_t most = std::min(rows * pieces_by(1), std::max<int64_t>(rows * pieces_by(8), 4 * dev->compute_units));
    l.bytes = (size_t)most * (sh.picks * sizeof(mfh_u64) + sizeof(double) + sizeof(float));
    return l;
}

template <int DT>
void launch_rows(const Layout& l, unsigned grid, hipStream_t s, const BeamArgs& a)
{
    if (l.packets == 1) k_beam_rows<DT, 1><<<grid, kThreads, 0, s>>>(a);
    else if (l.packets == 2) k_beam_rows<DT, 2><<<grid, kThreads, 0, s>>>(a);
    else if (l.packets == 4) k_beam_rows<DT, 4><<<grid, kThreads, 0, s>>>(a);
    else k_beam_rows<DT, 8><<<grid, kThreads, 0, s>>>(a);
}

int check_beams(const Device* dev, const mfh_beam_shape* sh, int32_t groups, const char* what, Layout* l)
{
    if (!sh) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL shape", what);
    if (sh->dtype != kFloat32 && sh->dtype != kFloat16 && sh->dtype != kBFloat16)
        return fail(MFH_ERR_DTYPE_UNSUPPORTED, "%s: logits of %s are not f32/f16/bf16", what, dtype_name(sh->dtype));
    if (sh->beams < 1 || sh->beams > kMostBeams)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d beams are not within 1..%d", what, sh->beams, kMostBeams);
    if (sh->picks < 1 || sh->picks > kMostPicks)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d picks are not within 1..%d", what, sh->picks, kMostPicks);
    if (sh->vocab < 1 || sh->vocab > 1 << kTokenBits)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d tokens are not within 1..2^%d", what, sh->vocab, kTokenBits);
    if (sh->end_token < -1 || sh->end_token >= sh->vocab)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: end token %d is not -1 or a token", what, sh->end_token);
    if (sh->logits_stride != 0 && sh->logits_stride < sh->vocab)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: rows of %d logits overlap at a stride of %lld", what, sh->vocab,
                    (long long)sh->logits_stride);
    if (sh->history_stride < 0 || sh->history_stride > kLongest)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: a history of %lld tokens is not within 0..2^30", what,
                    (long long)sh->history_stride);
    if (groups < 0) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: negative number of groups %d", what, groups);
    *l = layout(dev, *sh, groups);
    // a group's candidates, and the launch's threads, are counted in 32 bits
    if ((int64_t)sh->beams * l->pieces * sh->picks > kLongest || (int64_t)groups * sh->picks > kLongest ||
        (__int128)groups * sh->beams * l->pieces >= (int64_t(1) << 32) / kThreads)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: %d groups of %d beams over %d tokens are too many for one call", what,
                    groups, sh->beams, sh->vocab);
    return MFH_OK;
}

}  // namespace
}  // namespace mfh

using namespace mfh;

extern "C" {

int mfh_beam_select_workspace(const mfh_beam_shape* shape, int32_t groups, size_t* bytes)
{
    const char* what = "mfh_beam_select_workspace";
    const Device* dev;
    MFH_TRY(bind_device(&dev));
    Layout l;
    MFH_TRY(check_beams(dev, shape, groups, what, &l));
    if (!bytes) return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL result", what);
    *bytes = l.bytes;
    return MFH_OK;
}

int mfh_beam_select(const mfh_beam_shape* shape, int32_t groups, const void* logits, const float* scores,
                    const uint8_t* ended, float* scores_out, int32_t* tokens, int32_t* parents, uint8_t* ended_out,
                    const int32_t* history, const int32_t* known, int32_t* history_out, void* workspace,
                    size_t workspace_bytes, void* stream)
{
    const char* what = "mfh_beam_select";
    const Device* dev;
    MFH_TRY(bind_device(&dev));
    Layout l;
    MFH_TRY(check_beams(dev, shape, groups, what, &l));
    if (groups == 0) return MFH_OK;
    if (!logits || !scores || !scores_out || !tokens || !parents || (history && (!known || !history_out)))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: NULL buffer", what);
    if (ended && shape->end_token < 0)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: beams that have ended, and no end token", what);
    const int64_t rows = (int64_t)groups * shape->beams, results = (int64_t)groups * shape->picks;
    auto overlap = [](const void* p, int64_t p_bytes, const void* q, int64_t q_bytes) {
        return (uintptr_t)p < (uintptr_t)q + q_bytes && (uintptr_t)q < (uintptr_t)p + p_bytes;
    };
    if (overlap(scores, rows * 4, scores_out, results * 4))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: scores_out overlaps scores, which other workgroups still read", what);
    if (ended && ended_out && overlap(ended, rows, ended_out, results))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: ended_out overlaps ended, which other workgroups still read", what);
    if (history && overlap(history, rows * shape->history_stride * 4, history_out, results * shape->history_stride * 4))
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: history_out overlaps history, which other workgroups still read", what);
    if (workspace_bytes < l.bytes || !workspace || (uintptr_t)workspace % 16)
        return fail(MFH_ERR_INVALID_ARGUMENT, "%s: a workspace of %zu bytes is NULL, not 16-byte aligned or less than %zu",
                    what, workspace_bytes, l.bytes);
    BeamArgs a{};
    a.logits = (const char*)logits, a.scores = scores, a.ended = ended;
    a.scores_out = scores_out, a.tokens = tokens, a.parents = parents, a.ended_out = ended_out;
    a.history = history, a.known = known, a.history_out = history_out, a.history_stride = shape->history_stride;
    const int bytes = shape->dtype == kFloat32 ? 4 : 2;
    a.row_bytes = (shape->logits_stride ? shape->logits_stride : shape->vocab) * bytes;
    a.beams = (mfh_u32)shape->beams, a.picks = (mfh_u32)shape->picks, a.vocab = (mfh_u32)shape->vocab;
    a.pieces = (mfh_u32)l.pieces, a.end_token = shape->end_token;
    const int64_t cells = (int64_t)groups * shape->beams * l.pieces;
    a.best = (mfh_u64*)workspace, a.sums = (double*)(a.best + cells * shape->picks), a.tops = (float*)(a.sums + cells);
    // a slice of 16 KiB at least, and a workgroup per CU at most
    const int64_t history_bytes = history ? shape->history_stride * shape->picks * 4 : 0;
    a.slices = (mfh_u32)std::max<int64_t>(1, std::min<int64_t>(history_bytes >> 14, dev->compute_units / groups));
    a.by_pieces = Divider(a.pieces), a.by_picks = Divider(a.picks), a.by_slices = Divider(a.slices);
    a.by_piece = Divider((mfh_u32)(kThreads * l.packets * (16 / bytes)));
    hipStream_t s = (hipStream_t)stream;
    if (shape->dtype == kFloat32) launch_rows<kFloat32>(l, (unsigned)cells, s, a);
    else if (shape->dtype == kFloat16) launch_rows<kFloat16>(l, (unsigned)cells, s, a);
    else launch_rows<kBFloat16>(l, (unsigned)cells, s, a);
    MFH_TRY(launch_status("k_beam_rows"));
    const unsigned grid = (unsigned)groups * a.slices;
    if (a.beams * a.pieces * a.picks <= 2 * kThreads) k_beam_merge<true><<<grid, kThreads, 0, s>>>(a);
    else k_beam_merge<false><<<grid, kThreads, 0, s>>>(a);
    return launch_status("k_beam_merge");
}

}  // extern "C"
