// One choice for each row of logits, 1 to 4,096 wide (a flat head over the 324 packed moves, legal under the same 19 mask bytes,
// for one), with temperature, top-k, top-p and min-p; the definition of a draw stands in heads.cuh. What a row costs is its
// instructions, not its bytes (8,192 rows of 324 bf16 read 5.6 MB, 0.9 us, and take 10 us with no truncation, most of it exp and
// the sums, and 17 us with top-p): a row stays in a warp's registers (in a block's from 1,025 choices on), and a truncation
// is found without sorting.
#include "heads.cuh"

using namespace heads;

namespace {

constexpr int kMaxWidth = 4096;   // 2^12 weights of 2^27 and a u of 2^24 fit 63 bits

// ------------------------------------------------------------------ rows of any width

struct RowArgs {
    const void* logits;
    long long stride;
    int width;
    const uint8_t* legal;   // [rows, legal_width], or null: all
    long long legal_stride;
    int legal_width;        // the row's width, or 19 (the move parts' bytes; the row has 324 packed moves)
    const float* u;
    Cut cut;
    long long* choice;
    float* logp;
    long long rows;
};

// Whole numbers that order floats as the floats do, and back. No NaN comes here; -0 lies below 0, as its neighbour.
__device__ __forceinline__ unsigned key_of(float l) {
    const unsigned b = __float_as_uint(l);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

using u64 = unsigned long long;

// The sum of v < 2^43 over a warp, 16 bits at a time.
__device__ __forceinline__ u64 warp_total(u64 v) {
    return static_cast<u64>(__reduce_add_sync(~0u, static_cast<unsigned>(v) & 0xFFFFu)) +
           (static_cast<u64>(__reduce_add_sync(~0u, static_cast<unsigned>(v >> 16))) << 16);
}

// The sum of v over the lanes of the warp before this one.
template <class V>
__device__ __forceinline__ V lanes_before(V v) {
    V run = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V up = __shfl_up_sync(~0u, run, o);
        if ((threadIdx.x & 31) >= o) run += up;
    }
    return run - v;
}

// Sums and the like over the TPR threads of a row: one warp's by its reduction instructions, more warps' (one row per
// block) through shared memory, in two places that take turns, so that one barrier per call is enough (integer atomics on
// one word per call took longer: 80 us against 74 for 2,049 rows of 4,001 with every truncation).
template <int TPR>
struct Team {
    static constexpr int kWarps = TPR / 32;
    struct Shared {
        u64 word[2][2][kWarps], warp[2][kWarps], part[32];
    };
    Shared* s;
    int turn = 0, side = 0;

    __device__ explicit Team(Shared* shared) : s(shared) {}
    // a: added up, or (MAX) the largest; b (if PAIR): added up. One warp's values already.
    template <bool MAX, bool PAIR>
    __device__ void join(u64& a, u64& b) {
        if constexpr (kWarps > 1) {
            auto& w = s->word[turn];
            turn ^= 1;
            if ((threadIdx.x & 31) == 0) {
                w[0][threadIdx.x >> 5] = a;
                if (PAIR) w[1][threadIdx.x >> 5] = b;
            }
            __syncthreads();
            a = w[0][0];
            if (PAIR) b = w[1][0];
#pragma unroll
            for (int q = 1; q < kWarps; ++q) {
                a = MAX ? (w[0][q] > a ? w[0][q] : a) : a + w[0][q];
                if (PAIR) b += w[1][q];
            }
        }
    }
    // The sums of v and of n, as one word: 2^12 weights of 2^27, and a count of 2^12.
    __device__ void sums(u64 v, unsigned n, u64& total, unsigned& count) {
        u64 a = warp_total(v) | static_cast<u64>(__reduce_add_sync(~0u, n)) << 44, b = 0;
        join<false, false>(a, b);
        total = a & ((1ull << 44) - 1);
        count = static_cast<unsigned>(a >> 44);
    }
    __device__ unsigned count(unsigned n) {
        u64 a = __reduce_add_sync(~0u, n), b = 0;
        join<false, false>(a, b);
        return static_cast<unsigned>(a);
    }
    __device__ unsigned largest(unsigned v) {
        u64 a = __reduce_max_sync(~0u, v), b = 0;
        join<true, false>(a, b);
        return static_cast<unsigned>(a);
    }
    // The largest v, and the sum of n.
    __device__ unsigned largest(unsigned v, unsigned n, unsigned& count) {
        u64 a = __reduce_max_sync(~0u, v), b = __reduce_add_sync(~0u, n);
        join<true, true>(a, b);
        count = static_cast<unsigned>(b);
        return static_cast<unsigned>(a);
    }
    // 32 words, one use per row.
    __device__ u64* parts() { return s->part; }
    // The sum of v over the threads before this one.
    template <class V>
    __device__ V before(V v) {
        V run = lanes_before(v) + v;
        if constexpr (kWarps > 1) {
            u64* p = s->warp[side];
            side ^= 1;
            if ((threadIdx.x & 31) == 31) p[threadIdx.x >> 5] = run;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
                if (w < static_cast<int>(threadIdx.x >> 5)) run += static_cast<V>(p[w]);
        }
        return run - v;
    }
};

// A row's choices in a thread: four neighbours of each stretch of 4 TPR, so that their order is stretch, thread, place.
template <int TPR, int EPT>
struct RowTile {
    float l[EPT];        // -inf: not legal, or cut off
    unsigned wgt[EPT];
    __device__ static int at(int e) { return (e >> 2) * 4 * TPR + 4 * (static_cast<int>(threadIdx.x) & (TPR - 1)) + (e & 3); }
};

// Cuts the row to the shortest run of its ranked choices whose amounts (their weights, or 1 each) reach `reach` >= 1. The
// lowest value that stays is the lowest whose amount above it does not reach yet; choices of that value stay by their index.
// It is looked for by bisection between low (amounts above it reach) and high (they do not) until at most 32 choices lie
// between; a warp then has each of its lanes add up what ranks above one of them. m: the largest value; floor: amounts
// above it reach; n: how many choices lie above floor; guess: where to look first; few: 64 words of shared memory of the team.
// (8,192 rows of 324 at top_p 0.95, device time: 26 us by bisection of 16-bit keys to the end, 20 us this way.)
template <bool WEIGHTS, int TPR, int EPT>
__device__ __forceinline__ void cut_row(RowTile<TPR, EPT>& r, Team<TPR>& team, uint4* few, u64 reach, float m, float floor,
                                        float guess, unsigned n) {
    float low = floor, high = m, at = guess;
    unsigned n_low = n, n_high = 0;   // choices above low, above high
    u64 above = 0;                    // the amount above high
    for (int turn = 0; n_low - n_high > 32; ++turn) {
        if (turn > 0 || !(at > low && at < high)) at = 0.5f * low + 0.5f * high;   // the choices fill a row by value
        if (turn > 24 || !(at > low && at < high)) {   // no value between, an infinite end, or many equal choices: by key
            const unsigned lo = key_of(low), hi = key_of(high);
            if (hi - lo <= 1) break;
            at = value_of(lo + (hi - lo) / 2);
        }
        unsigned v[2] = {0, 0}, c = 0;   // 16 weights of 2^27 each
#pragma unroll
        for (int e = 0; e < EPT; ++e)
            if (r.l[e] > at) {
                if (WEIGHTS) v[e / 16] += r.wgt[e];
                ++c;
            }
        u64 total;
        if (WEIGHTS) {
            team.sums(EPT > 16 ? static_cast<u64>(v[0]) + v[1] : v[0], c, total, c);
        } else {
            c = team.count(c);
            total = c;
        }
        if (total < reach) {
            high = at;
            n_high = c;
            above = total;
        } else {
            low = at;
            n_low = c;
        }
    }
    unsigned group = n_low - n_high;   // the choices in (low, high] that have the lowest value that stays
    if (group > 1 && group <= 32) {
        float* l_s = reinterpret_cast<float*>(few);
        unsigned* w_s = reinterpret_cast<unsigned*>(few + 8);
        if constexpr (TPR == 32) __syncwarp();
        if (threadIdx.x % TPR < 32) l_s[threadIdx.x & 31] = -INFINITY;
        unsigned mine = 0;
#pragma unroll
        for (int e = 0; e < EPT; ++e) mine += r.l[e] > low && r.l[e] <= high;
        unsigned place = team.before(mine);   // (a barrier of the block)
        if constexpr (TPR == 32) __syncwarp();
#pragma unroll
        for (int e = 0; e < EPT; ++e)
            if (r.l[e] > low && r.l[e] <= high) {
                l_s[place] = r.l[e];
                w_s[place++] = r.wgt[e];
            }
        if constexpr (TPR == 32) __syncwarp();
        else __syncthreads();
        const float l = l_s[threadIdx.x & 31];
        const bool has = (threadIdx.x & 31) < group;
        unsigned over = 0;   // at most 31 weights of 2^27
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (4 * j >= static_cast<int>(group)) break;
            const float4 lj = reinterpret_cast<const float4*>(few)[j];
            const uint4 wj = WEIGHTS ? few[8 + j] : make_uint4(1, 1, 1, 1);
            if (lj.x > l) over += wj.x;
            if (lj.y > l) over += wj.y;
            if (lj.z > l) over += wj.z;
            if (lj.w > l) over += wj.w;
        }
        const bool stays = has && above + over < reach;
        const unsigned lowest = __reduce_min_sync(~0u, stays ? key_of(l == 0.f ? -0.f : l) : ~0u);
        high = value_of(lowest);
        low = value_of(lowest - 1);
        const unsigned same = __ballot_sync(~0u, has && l == high);
        group = __popc(same);
        above += __shfl_sync(~0u, over, __ffs(static_cast<int>(same)) - 1);
    }
    if (group > 1) {
        u64 each = 1;
        if (WEIGHTS) {
            unsigned w = 0;
#pragma unroll
            for (int e = 0; e < EPT; ++e)
                if (r.l[e] > low && r.l[e] <= high) w = r.wgt[e];
            each = team.largest(w);
        }
        const u64 left = reach - above, want = each == 0 ? group : (left + each - 1) / each;
        if (want < group) {   // the first of the group by index
            unsigned rank = 0;
#pragma unroll
            for (int s = 0; s < EPT / 4; ++s) {
                unsigned here = 0;
#pragma unroll
                for (int q = 0; q < 4; ++q) here += r.l[4 * s + q] > low && r.l[4 * s + q] <= high;
                unsigned mine = rank + team.before(here);
                rank += team.count(here);
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (r.l[4 * s + q] > low && r.l[4 * s + q] <= high && mine++ >= want) r.l[4 * s + q] = -INFINITY;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < EPT; ++e)
        if (!(r.l[e] > low)) {
            r.l[e] = -INFINITY;
            r.wgt[e] = 0;
        }
}

// A value that at least k of the row's choices reach: k / warps of each warp's threads have a choice that reaches the warp's
// own bound, the lowest of which holds for all. -inf where k is too large for that.
template <int TPR, int EPT>
__device__ __forceinline__ float kth_bound(const RowTile<TPR, EPT>& r, Team<TPR>& team, unsigned k) {
    const unsigned each = (k + Team<TPR>::kWarps - 1) / Team<TPR>::kWarps;
    if (each > 32) return -INFINITY;
    float best = r.l[0];
#pragma unroll
    for (int e = 1; e < EPT; ++e) best = fmaxf(best, r.l[e]);
    const unsigned key = key_of(best);
    unsigned t = 0;
    for (unsigned bit = 1u << 31; bit > 1u << 12; bit >>= 1) {   // coarse: a bound, not the value
        const unsigned n = __popc(__ballot_sync(~0u, key >= (t | bit)));
        if (n >= each) t |= bit;
        if (n == each) break;
    }
    t = ~team.largest(~t);
    const unsigned floor = key_of(-INFINITY);
    return t > floor + 1 ? value_of(t - 1) : -INFINITY;
}

constexpr int kFew = 128;   // choices that one warp takes on from a block

// Shared memory of a team: the choices between a cut's ends (32 values, 32 weights), and the ones that top-k left.
struct Few {
    uint4 ranked[16];
    float l[kFew];
    unsigned wgt[kFew];
    unsigned short at[kFew];
    unsigned count[32];   // of each stretch and warp
};

// Lays the row's choices above -inf, at most kFew, end to end in index order.
template <int TPR, int EPT>
__device__ __forceinline__ void gather(const RowTile<TPR, EPT>& r, Team<TPR>&, Few& few) {
    constexpr int kStretches = EPT / 4, kWarps = TPR / 32;
    static_assert(kStretches * kWarps <= 32, "a count per lane");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned before = (1u << lane) - 1u;
    unsigned rank[kStretches];   // of the thread's first choice among its warp's in the stretch
#pragma unroll
    for (int s = 0; s < kStretches; ++s) {
        unsigned all = 0;
        rank[s] = 0;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const unsigned in = __ballot_sync(~0u, r.l[4 * s + p] > -INFINITY);
            rank[s] += __popc(in & before);
            all += __popc(in);
        }
        if (lane == 0) few.count[s * kWarps + warp] = all;
    }
    __syncthreads();
    const unsigned mine = lane < kStretches * kWarps ? few.count[lane] : 0u;
    unsigned run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned up = __shfl_up_sync(~0u, run, o);
        if (lane >= o) run += up;
    }
    run -= mine;
#pragma unroll
    for (int s = 0; s < kStretches; ++s) {
        unsigned place = __shfl_sync(~0u, run, s * kWarps + warp) + rank[s];
#pragma unroll
        for (int p = 0; p < 4; ++p)
            if (r.l[4 * s + p] > -INFINITY) {
                few.l[place] = r.l[4 * s + p];
                few.wgt[place] = r.wgt[4 * s + p];
                few.at[place++] = static_cast<unsigned short>(r.at(4 * s + p));
            }
    }
    __syncthreads();
}

// The rest of a draw from a row whose top-k is done: top-p, min-p, the choice and its log-probability. index(i): which of the
// row's choices is the i-th here.
template <int TPR, int EPT, class I>
__device__ __forceinline__ void finish(RowTile<TPR, EPT>& r, Team<TPR>& team, uint4* few, const RowCut& q, float m, float u, bool nan,
                                       I index, long long* choice, float* logp) {
    if (q.top_p < 1.f) {
        // what weighs nothing lies at floor or below, since exp(-20) 2^27 rounds to 0; one value below m - 20 T as fp32 has it,
        // which may round up as far as m itself: floor < m always, so the best choice is above it, and so is every weight
        const float floor = nextafterf(m - 20.f / q.scale, -INFINITY);
        unsigned w[2] = {0, 0}, count = 0;
#pragma unroll
        for (int e = 0; e < EPT; ++e) {
            w[e / 16] += r.wgt[e];
            count += r.l[e] > floor;
        }
        u64 total;
        team.sums(EPT > 16 ? static_cast<u64>(w[0]) + w[1] : w[0], count, total, count);
        const double p = ceil(static_cast<double>(q.top_p) * static_cast<double>(total));
        const u64 reach = p < 1.0 ? 1ull : static_cast<u64>(p);
        // choices that could all go together lie below the lowest value that stays: look there first
        const float least = static_cast<float>(total - reach) * kUnit / static_cast<float>(count);
        cut_row<true>(r, team, few, reach, m, floor, m + __logf(least) / q.scale, count);
    }
    if (q.least > 0) {
#pragma unroll
        for (int e = 0; e < EPT; ++e)
            if (r.wgt[e] < q.least) r.wgt[e] = 0;
    }
    // the stretch of the row, then the thread, then the place in which the running sum passes the target
    u64 part[EPT / 4], total = 0;
#pragma unroll
    for (int s = 0; s < EPT / 4; ++s) part[s] = warp_total(static_cast<u64>(r.wgt[4 * s] + r.wgt[4 * s + 1] + r.wgt[4 * s + 2] + r.wgt[4 * s + 3]));
    u64 target, skipped = 0;   // skipped: the sum before this warp's part of the stretch
    int stretch = 0;
    bool ours = true;          // whether it is this warp's part that the target lies in
    if constexpr (TPR == 32) {
#pragma unroll
        for (int s = 0; s < EPT / 4; ++s) total += part[s];
        target = (bits24(u) * total) >> 24;
#pragma unroll
        for (int s = 0; s + 1 < EPT / 4; ++s)
            if (stretch == s && target >= skipped + part[s]) {
                skipped += part[s];
                stretch = s + 1;
            }
    } else {   // a lane per stretch and warp, in index order
        constexpr int kWarps = TPR / 32, kParts = EPT / 4 * kWarps;
        static_assert(kParts <= 32, "a part per lane");
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        u64* parts = team.parts();
        if (lane == 0) {
#pragma unroll
            for (int s = 0; s < EPT / 4; ++s) parts[s * kWarps + warp] = part[s];
        }
        __syncthreads();
        u64 run = lane < kParts ? parts[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 up = __shfl_up_sync(~0u, run, o);
            if (lane >= o) run += up;
        }
        total = __shfl_sync(~0u, run, 31);
        target = (bits24(u) * total) >> 24;
        const int at = __ffs(static_cast<int>(__ballot_sync(~0u, run > target))) - 1;   // the first part that passes the target
        skipped = at > 0 ? __shfl_sync(~0u, run, at - 1) : 0;
        stretch = at / kWarps;
        ours = at % kWarps == warp;
    }
    if (!ours) return;
    target -= skipped;
    unsigned w[4] = {0, 0, 0, 0};
    float l[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < EPT / 4; ++s)
        if (stretch == s) {
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                w[p] = r.wgt[4 * s + p];
                l[p] = r.l[4 * s + p];
            }
        }
    const u64 own = static_cast<u64>(w[0]) + w[1] + w[2] + w[3], run = lanes_before(own);
    if (run <= target && target < run + own) {
        unsigned left = static_cast<unsigned>(target - run);
        int c = 0;
        float lc = l[0];
#pragma unroll
        for (int p = 0; p < 3; ++p)
            if (c == p && left >= w[p]) {
                left -= w[p];
                c = p + 1;
                lc = l[p + 1];
            }
        *choice = index(r.at(4 * stretch) + c);
        *logp = nan ? NAN : (lc - m) * q.scale - logf(static_cast<float>(total) * kUnit);
    }
}

// Warps per SM that the registers of EPT choices per thread leave room for.
template <int EPT>
constexpr int kRowWarps = EPT <= 4 ? 48 : EPT <= 12 ? 32 : EPT <= 16 ? 24 : 16;

// A warp, or a block of TPR threads, per row; the row's values and weights stay in registers. VEC: rows whose four
// neighbours can be loaded at once.
template <class T, int TPR, int EPT, bool VEC>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, TPR == 32 ? kRowWarps<EPT> / 8 : kRowWarps<EPT> * 32 / TPR)
k_rows_sample(RowArgs a) {
    constexpr int kTeams = TPR == 32 ? 8 : 1;
    __shared__ typename Team<TPR>::Shared team_s;
    Team<TPR> team(&team_s);
    __shared__ Few few_s[kTeams];
    uint4* few = few_s[TPR == 32 ? threadIdx.x >> 5 : 0].ranked;
    const int n = a.width, lane = threadIdx.x & 31;
    const bool parts = a.legal && a.legal_width != n;
    __shared__ uint4 need_s[TPR == 32 && EPT == 12 ? kMoves / 4 : 1];   // the five mask bytes that a packed move needs, as bits
    if constexpr (TPR == 32 && EPT == 12) {   // the tile of rows of 324
        if (parts) {
            for (int i = threadIdx.x; i < kMoves; i += 256)
                reinterpret_cast<unsigned*>(need_s)[i] =
                    1u << i % 9 | 1u << (9 + i / 9 % 3) | 1u << (12 + i / 27 % 3) | 1u << (15 + i / 81 % 2) | 1u << (17 + i / 162);
            __syncthreads();
        }
    }
    for (long long row = static_cast<long long>(blockIdx.x) * kTeams + (TPR == 32 ? threadIdx.x >> 5 : 0); row < a.rows;
         row += static_cast<long long>(gridDim.x) * kTeams) {
        const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
        const uint8_t* legal = a.legal ? a.legal + row * a.legal_stride : nullptr;
        const float u = a.u[row];
        const RowCut q = row_cut(a.cut, row);
        unsigned bits = ~0u;
        if (parts) bits = __ballot_sync(~0u, lane < kBytes && legal[min(lane, kBytes - 1)] != 0);
        RowTile<TPR, EPT> r;
        float m = 0.f;
        // Loads the row and returns this thread's largest value, a NaN if there is one. CAREFUL: where the row's largest legal
        // value m (NaNs aside) is not finite, what equals it becomes 0 and the rest -inf; NaNs become -inf.
        auto load = [&](auto careful) {
            float best = -INFINITY;
#pragma unroll
            for (int s = 0; s < EPT / 4; ++s) {
                const int i = r.at(4 * s);
                float l[4];
                bool ok[4] = {i < n, i + 1 < n, i + 2 < n, i + 3 < n};
                if constexpr (VEC) {
                    if (i < n) {
                        struct alignas(4 * sizeof(T)) Four { T v[4]; };
                        const Four f = *reinterpret_cast<const Four*>(logits + i);
#pragma unroll
                        for (int p = 0; p < 4; ++p) l[p] = to_f(f.v[p]);
                        if (legal && !parts) {
                            const uchar4 k = *reinterpret_cast<const uchar4*>(legal + i);
                            ok[0] = k.x;
                            ok[1] = k.y;
                            ok[2] = k.z;
                            ok[3] = k.w;
                        }
                    }
                } else {
#pragma unroll
                    for (int p = 0; p < 4; ++p)
                        if (i + p < n) {
                            l[p] = to_f(logits[i + p]);
                            if (legal && !parts) ok[p] = legal[i + p];
                        }
                }
                if constexpr (TPR == 32 && EPT == 12) {
                    if (parts && i < n) {
                        const uint4 v = need_s[i >> 2];
                        ok[0] = (bits & v.x) == v.x;
                        ok[1] = (bits & v.y) == v.y;
                        ok[2] = (bits & v.z) == v.z;
                        ok[3] = (bits & v.w) == v.w;
                    }
                }
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    float v = ok[p] ? l[p] : -INFINITY;
                    if constexpr (decltype(careful)::value) {
                        if (fabsf(m) < INFINITY) v = v == v ? v : -INFINITY;
                        else v = ok[p] && (m < 0.f ? !(v > m) : v == m) ? 0.f : -INFINITY;
                    }
                    r.l[4 * s + p] = v;
                    best = max_nan(best, v);
                }
            }
            return best;
        };
        float best = load(std::false_type{});
        const bool bad = best != best;
        if (bad) {
            best = -INFINITY;
#pragma unroll
            for (int e = 0; e < EPT; ++e) best = fmaxf(best, r.l[e]);
        }
        unsigned nans;
        m = value_of(team.largest(key_of(best), bad, nans));
        if (nans || !(fabsf(m) < INFINITY)) {   // rare
            best = load(std::true_type{});
            m = value_of(team.largest(key_of(best)));
        }
        if (m == -INFINITY) {   // nothing legal
            if ((threadIdx.x & (TPR - 1)) == 0) {
                a.choice[row] = 0;
                a.logp[row] = 0.f;
            }
            continue;
        }
#pragma unroll
        for (int e = 0; e < EPT; ++e) r.wgt[e] = weight_of((r.l[e] - m) * q.scale);
        unsigned kept = 0;   // choices before top-k
        if (q.top_k > 0) {
#pragma unroll
            for (int e = 0; e < EPT; ++e) kept += r.l[e] > -INFINITY;
            kept = team.count(kept);
            const unsigned k = static_cast<unsigned>(q.top_k);
            if (k < kept) cut_row<false>(r, team, few, k, m, -INFINITY, kth_bound(r, team, k), kept);
        }
        // what a small k left of a wide row is one warp's work (2,049 rows, top-p 0.9, without and with it: at top-k 50 31 and 28 us
        // for 1,500 choices, 59 and 53 for 2,049, 70 and 64 for 4,001; at top-k 128 31 and 29 for 1,025, 74 and 66 for 4,001; at
        // top-k 2 23.9 and 24.2 for 1,025, 57 and 55 for 4,001; without a top-p to follow it does not pay)
        if constexpr (TPR > 32) {
            if (q.top_p < 1.f && q.top_k > 0 && q.top_k <= kFew && kept > static_cast<unsigned>(q.top_k)) {
                gather(r, team, few_s[0]);
                if (threadIdx.x < 32) {
                    RowTile<32, kFew / 32> f;
#pragma unroll
                    for (int e = 0; e < kFew / 32; ++e) {
                        const bool in = f.at(e) < q.top_k;
                        f.l[e] = in ? few_s[0].l[f.at(e)] : -INFINITY;
                        f.wgt[e] = in ? few_s[0].wgt[f.at(e)] : 0u;
                    }
                    __syncwarp();   // the gathered values are free, their places are not
                    Team<32> warp(nullptr);
                    finish(f, warp, few, q, m, u, nans != 0, [&](int i) { return static_cast<int>(few_s[0].at[i]); }, a.choice + row, a.logp + row);
                }
                __syncthreads();
                continue;
            }
        }
        finish(r, team, few, q, m, u, nans != 0, [](int i) { return i; }, a.choice + row, a.logp + row);
    }
}

// f of the row's tile (threads per row, choices per thread): the smallest that holds it.
template <class F>
void with_row_tile(int width, F f) {
    using std::integral_constant;
    if (width <= 128) f(integral_constant<int, 32>{}, integral_constant<int, 4>{});
    else if (width <= 256) f(integral_constant<int, 32>{}, integral_constant<int, 8>{});
    else if (width <= 384) f(integral_constant<int, 32>{}, integral_constant<int, 12>{});
    else if (width <= 512) f(integral_constant<int, 32>{}, integral_constant<int, 16>{});
    else if (width <= 1024) f(integral_constant<int, 32>{}, integral_constant<int, 32>{});
    else if (width <= 2048) f(integral_constant<int, 64>{}, integral_constant<int, 32>{});
    else f(integral_constant<int, 128>{}, integral_constant<int, 32>{});
}

}  // namespace

extern "C" {

int rl_sample(const void* logits, long long stride, int type, int width, const void* legal, long long legal_stride,
              int legal_width, const void* u, float temperature, int top_k, float top_p, float min_p,
              const void* temperatures, const void* top_ks, const void* top_ps, const void* min_ps, void* choice,
              void* logp, long long rows, void* stream) {
    if (rows < 0) return failed("rows must not be negative");
    if (width < 1 || width > kMaxWidth) return failed("width must be 1 .. 4096");
    if (legal && legal_width != width && !(legal_width == kBytes && width == kMoves))
        return failed("legal must have a byte for each choice, or the 19 mask bytes of the 324 moves");
    if (const char* e = bad_cut(temperature, temperatures, top_p, top_ps, min_p, min_ps, top_ks)) return failed(e);
    if (type < 0 || type > 2) return failed("unknown type of the logits");
    if (rows == 0) return 0;
    if (!logits || !u || !choice || !logp) return failed("logits, u, choice and logp must be given");
    if (!fits(logits, size_of(type)) || !fits(u, 4) || !fits(choice, 8) || !fits(logp, 4)) return failed("misaligned pointer");
    RowArgs a;
    a.logits = logits;
    a.stride = stride;
    a.width = width;
    a.legal = static_cast<const uint8_t*>(legal);
    a.legal_stride = legal_stride;
    a.legal_width = legal_width;
    a.u = static_cast<const float*>(u);
    a.cut = Cut{temperature, top_p, min_p, top_k, static_cast<const float*>(temperatures), static_cast<const float*>(top_ps),
                static_cast<const float*>(min_ps), static_cast<const int*>(top_ks)};
    a.choice = static_cast<long long*>(choice);
    a.logp = static_cast<float*>(logp);
    a.rows = rows;
    const size_t e4 = type == 0 ? 16 : 8;   // bytes of four values
    const bool vec = width % 4 == 0 && stride % 4 == 0 && reinterpret_cast<uintptr_t>(logits) % e4 == 0 &&
                     (!legal || legal_width != width || (legal_stride % 4 == 0 && reinterpret_cast<uintptr_t>(legal) % 4 == 0));
    with_type(type, [&](auto t) {
        using T = decltype(t);
        with_row_tile(width, [&](auto tpr, auto ept) {
            // more blocks than fit at once: the last ones even out (8,192 x 324: 1.4 us less than with as many as fit)
            const unsigned grid = tpr() == 32 ? blocks_for(rows, 8, 2 * kRowWarps<ept()> / 8ll * sm_count())
                                              : blocks_for(rows, 1, 16 * kRowWarps<ept()> * 32ll / tpr() * sm_count());
            const unsigned block = tpr() == 32 ? 256 : tpr();
            if (vec) k_rows_sample<T, tpr(), ept(), true><<<grid, block, 0, static_cast<cudaStream_t>(stream)>>>(a);
            else k_rows_sample<T, tpr(), ept(), false><<<grid, block, 0, static_cast<cudaStream_t>(stream)>>>(a);
        });
    });
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : failed(cudaGetErrorString(e));
}

}  // extern "C"
