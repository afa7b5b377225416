// The policy's ordered action heads (rl/model.py:176-194): moves sampled from given random numbers, with temperature, top-k,
// top-p and min-p; rows of any width sampled the same way (a flat head over the 324 packed moves, for one); and the
// log-probability and entropy of given moves, with their gradients.
//
// A move has five parts (d-pad 9, A 3, B 3, Start 2, Select 2 choices). Part k's logits are the head's own plus one row of
// cond[k][j] for each earlier part j, the row of the choice c_j; its legal choices A are the mask bytes that are not 0.
//
// Sampling of a row l: m = max over A, d = (l - m) / T, W = round(exp(d) 2^27), a whole number of 28 bits. Choices are
// ranked by l, equal ones by their index; the first k stay, of those the shortest run from the top whose W sum reaches p
// of theirs, of those the ones with W >= min_p 2^27. With u in [0, 1) as 24 bits, the choice is the first that stayed, in
// index order, whose running sum of W exceeds floor(u total), and its log-probability (of the distribution that was drawn
// from) d - log(total 2^-27). Whole numbers make every sum the same in any order, so a result depends on no tile, lane or
// launch shape; 2^-27 of the best choice is finer than u's own 2^-24.
//
// Log-probability and entropy, per part: w = exp(l - m) over A, S = sum w, p = w / S, log p = l - m - log S,
// H = log S - sum w (l - m) / S. With incoming gradients a (of the log-probability) and b (of the entropy):
//   dl_i = a (1[i = c] - p_i) - b p_i (log p_i + H), dcond[k][j][c_j][i] = the sum of dl_i over the rows with that c_j.
// A part with nothing legal answers its choice 0 (neutral, off), and adds 0 to the log-probability, the entropy and the
// gradients. Masked logits are never used, whatever they hold.
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>
#include "../../include/rlenv_api.h"   // rl_sample, rl_moves_* compiled against their C-ABI declarations

namespace {

constexpr int kParts = 5, kBytes = 19, kMoves = 324, kTables = 10, kCond = 127;
constexpr float kScale = 134217728.f;   // 2^27
constexpr float kUnit = 1.f / kScale;
constexpr int kThreads = 128;           // and rows of a block's batch
constexpr int kDevices = 64;            // whose properties are kept
constexpr int kMaxWidth = 4096;         // 2^12 weights of 2^27 and a u of 2^24 fit 63 bits

thread_local std::string g_heads_error;

__host__ __device__ constexpr int part_at(int k) { return k == 0 ? 0 : k == 1 ? 9 : k == 2 ? 12 : k == 3 ? 15 : 17; }
__host__ __device__ constexpr int part_n(int k) { return k == 0 ? 9 : k < 3 ? 3 : 2; }
__host__ __device__ constexpr int table_of(int k, int j) { return k * (k - 1) / 2 + j; }
// Where table cond[k][j] ([choices of j][choices of k]) starts in the ten laid end to end.
__host__ __device__ constexpr int table_at(int t) {
    int at = 0, i = 0;
    for (int k = 1; k < kParts; ++k)
        for (int j = 0; j < k; ++j, ++i)
            if (i < t) at += part_n(j) * part_n(k);
    return at;
}
static_assert(table_at(kTables) == kCond, "the ten tables' sizes");

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

struct Cond {
    const void* table[kTables];
    int type;   // 0 fp32, 1 bf16, 2 fp16; -1: no tables
};

// The sampling parameters: one number for all rows, or (pointer not null) one for each.
struct Cut {
    float temperature, top_p, min_p;
    int top_k;
    const float *temperatures, *top_ps, *min_ps;
    const int* top_ks;
};

struct RowCut {
    float scale;   // 1 / T
    float top_p, min_p;
    int top_k;     // 0: all
    bool cut;      // whether any of the three takes something off
};

__device__ __forceinline__ RowCut row_cut(const Cut& c, long long row) {
    RowCut r;
    const float t = c.temperatures ? c.temperatures[row] : c.temperature;
    r.top_p = c.top_ps ? c.top_ps[row] : c.top_p;
    r.min_p = c.min_ps ? c.min_ps[row] : c.min_p;
    r.top_k = c.top_ks ? c.top_ks[row] : c.top_k;
    r.top_p = r.top_p < 1.f ? fmaxf(r.top_p, 0.f) : 1.f;   // a NaN takes nothing off
    r.min_p = r.min_p > 0.f ? fminf(r.min_p, 1.f) : 0.f;
    if (r.top_k < 0) r.top_k = 0;
    r.scale = __fdiv_rn(1.f, t);
    if (!(t > 0.f) || r.scale == INFINITY) {   // 0 (or nothing a temperature can be): the best choice alone
        r.top_k = 1;
        r.scale = 1.f;
    }
    r.cut = r.top_k > 0 || r.top_p < 1.f || r.min_p > 0.f;
    return r;
}

// W of a scaled logit d <= 0 (-inf, and the NaN of -inf at an infinite temperature, weigh nothing).
__device__ __forceinline__ unsigned weight_of(float d) { return __float2uint_rn(expf(d) * kScale); }

// The larger of two; a NaN if either is one.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ unsigned bits24(float u) {
    const int v = static_cast<int>(u * 16777216.f);   // a NaN is 0
    return static_cast<unsigned>(min(max(v, 0), 0xFFFFFF));
}

// All ten tables, in fp32, into shared memory: an entry per thread (or two), so that they arrive together.
__device__ __forceinline__ void load_cond(float* tab, const Cond& c) {
    if (c.type < 0) return;
#pragma unroll 2
    for (int e = threadIdx.x; e < kCond; e += blockDim.x) {
        int t = 0, at = 0;
#pragma unroll
        for (int i = 1; i < kTables; ++i)
            if (e >= table_at(i)) {
                t = i;
                at = table_at(i);
            }
        const int i = e - at;
        tab[e] = c.type == 0 ? static_cast<const float*>(c.table[t])[i]
                 : c.type == 1 ? to_f(static_cast<const __nv_bfloat16*>(c.table[t])[i])
                               : to_f(static_cast<const __half*>(c.table[t])[i]);
    }
}

// ------------------------------------------------------------------ batches of rows in shared memory
//
// A block takes kThreads rows at a time, a thread each. A row's 19 logits and 19 mask bytes are no place to start a wide
// load, but kThreads rows of them are: a block's rows come as one stretch of 16-byte asynchronous copies, one batch ahead.
// Rows that do not lie end to end from a 16-byte boundary are fetched value by value.

__device__ __forceinline__ void copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Rows [first, first + n) of COLS values each into shared memory, end to end.
template <int COLS, int THREADS, class T>
__device__ __forceinline__ void stage(T* dst, const void* base, long long first, int n, long long stride, bool dense) {
    const T* src = static_cast<const T*>(base) + first * stride;
    if (dense) {
        constexpr int kPer = 16 / static_cast<int>(sizeof(T));
        const int all = n * COLS, whole = all & ~(kPer - 1);
        for (int i = threadIdx.x * kPer; i < whole; i += THREADS * kPer) copy16(dst + i, src + i);
        for (int i = whole + threadIdx.x; i < all; i += THREADS) dst[i] = src[i];
    } else {
        for (int i = threadIdx.x; i < n * COLS; i += THREADS) {
            const int row = i / COLS;
            dst[i] = src[row * stride + (i - row * COLS)];
        }
    }
}

// Logits of a part whose largest legal one is not finite, brought to the case where it is: what equals it (or, for -inf, what
// is legal at all) becomes 0, the rest -inf. A NaN is taken as -inf. False where nothing is legal.
__device__ __noinline__ bool settle(float* l, int n, const uint8_t* mask, float& m) {
    m = -INFINITY;
    bool any = false;
    for (int i = 0; i < n; ++i) {
        m = fmaxf(m, l[i]);
        any |= mask[i] != 0;
    }
    if (fabsf(m) < INFINITY) {   // there was a NaN
        for (int i = 0; i < n; ++i)
            if (l[i] != l[i]) l[i] = -INFINITY;
        return any;
    }
    for (int i = 0; i < n; ++i) l[i] = mask[i] != 0 && (m < 0.f ? !(l[i] > m) : l[i] == m) ? 0.f : -INFINITY;
    m = 0.f;
    return any;
}

// One choice of N logits (-inf: not legal); its d is added to d_sum, its total multiplied into totals (d_sum - log totals is
// the move's log-probability: one logarithm for the five parts).
template <int N>
__device__ __forceinline__ int choose(float (&l)[N], const uint8_t* mask, float u, const RowCut& q, float& d_sum, float& totals) {
    float m = l[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = max_nan(m, l[i]);
    bool nan = false;
    if (!(fabsf(m) < INFINITY)) {
        nan = m != m;
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = l[i];
        if (!settle(v, N, mask, m)) return 0;
#pragma unroll
        for (int i = 0; i < N; ++i) l[i] = v[i];
    }
    float d[N];
    unsigned w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        d[i] = (l[i] - m) * q.scale;
        w[i] = weight_of(d[i]);
    }
    if (q.cut) {
        int rank[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            rank[i] = 0;
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (j != i) rank[i] += j < i ? l[j] >= l[i] : l[j] > l[i];
        }
        const int top = q.top_k > 0 ? q.top_k : N;
        unsigned total = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (rank[i] >= top) w[i] = 0;
            total += w[i];
        }
        const unsigned reach = static_cast<unsigned>(ceil(static_cast<double>(q.top_p) * static_cast<double>(total)));
        const unsigned least = static_cast<unsigned>(ceil(static_cast<double>(q.min_p) * static_cast<double>(kScale)));
        unsigned kept = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            unsigned before = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) before += rank[j] < rank[i] ? w[j] : 0u;
            const bool keep = rank[i] == 0 || (before < reach && w[i] >= least);
            kept |= static_cast<unsigned>(keep) << i;
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (!(kept >> i & 1)) w[i] = 0;
    }
    unsigned total = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) total += w[i];
    const unsigned target = static_cast<unsigned>((static_cast<unsigned long long>(bits24(u)) * total) >> 24);
    int c = 0;
    float dc = 0.f;
    unsigned run = total;
#pragma unroll
    for (int i = N - 1; i >= 0; --i) {   // the last to match is the first in index order
        if (run > target) {
            c = i;
            dc = d[i];
        }
        run -= w[i];
    }
    d_sum += nan ? NAN : dc;
    totals *= static_cast<float>(total) * kUnit;
    return c;
}

// Part K's logits of a row whose earlier choices are c[0..K); -inf where the mask says so.
template <int K, class T>
__device__ __forceinline__ void part_logits(float (&l)[part_n(K)], const T* logits, const uint8_t* mask, const float* tab,
                                            const int* c) {
#pragma unroll
    for (int i = 0; i < part_n(K); ++i) l[i] = to_f(logits[part_at(K) + i]);
    if (tab) {
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int i = 0; i < part_n(K); ++i) l[i] += tab[table_at(table_of(K, j)) + c[j] * part_n(K) + i];
    }
#pragma unroll
    for (int i = 0; i < part_n(K); ++i) l[i] = mask[part_at(K) + i] != 0 ? l[i] : -INFINITY;
}

struct MoveArgs {
    const void* logits;
    long long stride;
    Cond cond;
    const uint8_t* masks;
    long long mask_stride;
    const float* u;
    bool dense_logits, dense_masks, dense_u;
    Cut cut;
    int16_t* ids;
    float* logp;
    long long rows;
};

template <class T>
struct MoveBatch {
    T logits[kThreads * kBytes];
    alignas(16) uint8_t masks[kThreads * kBytes];
    alignas(16) float u[kThreads * kParts];
};

template <int K, class T>
__device__ __forceinline__ void draw_part(const T* logits, const uint8_t* mask, const float* u, const RowCut& q, const float* tab,
                                          int* c, float& d_sum, float& totals) {
    float l[part_n(K)];
    part_logits<K>(l, logits, mask, tab, c);
    c[K] = choose<part_n(K)>(l, mask + part_at(K), u[K], q, d_sum, totals);
}

// A thread per row.
template <class T>
__global__ void __launch_bounds__(kThreads) k_moves_sample(MoveArgs a) {
    extern __shared__ __align__(16) unsigned char batches[];
    __shared__ float tab_s[kCond];
    auto* batch = reinterpret_cast<MoveBatch<T>*>(batches);
    auto fetch = [&](long long first, MoveBatch<T>& to) {
        if (first < a.rows) {
            const int n = static_cast<int>(min(static_cast<long long>(kThreads), a.rows - first));
            stage<kBytes, kThreads>(to.logits, a.logits, first, n, a.stride, a.dense_logits);
            stage<kBytes, kThreads>(to.masks, a.masks, first, n, a.mask_stride, a.dense_masks);
            stage<kParts, kThreads>(to.u, a.u, first, n, kParts, a.dense_u);
        }
        copies_commit();
    };
    const long long step = static_cast<long long>(gridDim.x) * kThreads;
    long long first = static_cast<long long>(blockIdx.x) * kThreads;
    fetch(first, batch[0]);
    load_cond(tab_s, a.cond);
    const float* tab = a.cond.type < 0 ? nullptr : tab_s;
    for (int b = 0; first < a.rows; first += step, b ^= 1) {
        fetch(first + step, batch[b ^ 1]);
        copies_wait<1>();
        __syncthreads();
        const long long row = first + threadIdx.x;
        if (row < a.rows) {
            const T* logits = batch[b].logits + threadIdx.x * kBytes;
            const uint8_t* mask = batch[b].masks + threadIdx.x * kBytes;
            const float* u = batch[b].u + threadIdx.x * kParts;
            const RowCut q = row_cut(a.cut, row);
            int c[kParts];
            float d_sum = 0.f, totals = 1.f;
            draw_part<0>(logits, mask, u, q, tab, c, d_sum, totals);
            draw_part<1>(logits, mask, u, q, tab, c, d_sum, totals);
            draw_part<2>(logits, mask, u, q, tab, c, d_sum, totals);
            draw_part<3>(logits, mask, u, q, tab, c, d_sum, totals);
            draw_part<4>(logits, mask, u, q, tab, c, d_sum, totals);
            a.ids[row] = static_cast<int16_t>(c[0] + 9 * c[1] + 27 * c[2] + 81 * c[3] + 162 * c[4]);
            a.logp[row] = d_sum - logf(totals);
        }
        __syncthreads();   // the batch may be written again
    }
}

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

// Sums and the like over the TPR threads of a row: one warp's by its reduction instructions, more warps' (one row per
// block) through shared memory, in two places that take turns, so that one barrier per call is enough (integer atomics on
// one word per call took longer: 80 us against 74 for 2,049 rows of 4,001 with every truncation).
template <int TPR>
struct Team {
    static constexpr int kWarps = TPR / 32;
    struct Shared {
        u64 word[2][2][kWarps], warp[2][kWarps];
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
    __device__ u64 sum(u64 v) {
        u64 a = warp_total(v), b = 0;
        join<false, false>(a, b);
        return a;
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
    // The sum of v over the threads before this one.
    template <class V>
    __device__ V before(V v) {
        V run = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const V up = __shfl_up_sync(~0u, run, o);
            if ((threadIdx.x & 31) >= o) run += up;
        }
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
    __shared__ uint4 few_s[kTeams][16];
    uint4* few = few_s[TPR == 32 ? threadIdx.x >> 5 : 0];
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
        if (q.top_k > 0) {
            unsigned count = 0;
#pragma unroll
            for (int e = 0; e < EPT; ++e) count += r.l[e] > -INFINITY;
            count = team.count(count);
            const unsigned k = static_cast<unsigned>(q.top_k);
            if (k < count) cut_row<false>(r, team, few, k, m, -INFINITY, kth_bound(r, team, k), count);
        }
        if (q.top_p < 1.f) {
            const float floor = m - 20.f / q.scale;   // exp(-20) 2^27 rounds to nothing
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
        if (q.min_p > 0.f) {
            const unsigned least = static_cast<unsigned>(ceil(static_cast<double>(q.min_p) * static_cast<double>(kScale)));
#pragma unroll
            for (int e = 0; e < EPT; ++e)
                if (r.wgt[e] < least) r.wgt[e] = 0;
        }
        // the stretch of the row, then the thread, then the place in which the running sum passes the target
        u64 part[EPT / 4], total = 0;
#pragma unroll
        for (int s = 0; s < EPT / 4; ++s) {
            part[s] = team.sum(r.wgt[4 * s] + r.wgt[4 * s + 1] + r.wgt[4 * s + 2] + r.wgt[4 * s + 3]);
            total += part[s];
        }
        u64 target = (bits24(u) * total) >> 24;
        int stretch = 0;
        unsigned w[4] = {r.wgt[0], r.wgt[1], r.wgt[2], r.wgt[3]};
        float l[4] = {r.l[0], r.l[1], r.l[2], r.l[3]};
#pragma unroll
        for (int s = 1; s < EPT / 4; ++s)
            if (stretch == s - 1 && target >= part[s - 1]) {
                target -= part[s - 1];
                stretch = s;
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    w[p] = r.wgt[4 * s + p];
                    l[p] = r.l[4 * s + p];
                }
            }
        const u64 own = static_cast<u64>(w[0]) + w[1] + w[2] + w[3], run = team.before(own);
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
            a.choice[row] = r.at(4 * stretch) + c;
            a.logp[row] = nans ? NAN : (lc - m) * q.scale - logf(static_cast<float>(total) * kUnit);
        }
    }
}

// ------------------------------------------------------------------ log-probability and entropy of given moves

struct LogpArgs {
    const void* logits;
    long long stride;
    Cond cond;
    const uint8_t* masks;
    long long mask_stride;
    bool dense_logits, dense_masks, dense_out;
    const int16_t* ids;
    float *logp, *entropy;               // forward
    const float *glp, *gent;             // backward: incoming gradients, either may be null
    long long glp_stride, gent_stride;
    void* dlogits;                       // [rows, 19] of the logits' type, or null
    float* part;                         // [blocks][127] partial sums of the tables' gradient, or null
    long long rows;
};

template <class T, int ROWS>
struct LogpBatch {
    T logits[ROWS * kBytes];
    alignas(16) uint8_t masks[ROWS * kBytes];
};

template <int THREADS, class T, int ROWS>
__device__ __forceinline__ void fetch_batch(const LogpArgs& a, long long first, LogpBatch<T, ROWS>& to) {
    if (first < a.rows) {
        const int n = static_cast<int>(min(static_cast<long long>(ROWS), a.rows - first));
        stage<kBytes, THREADS>(to.logits, a.logits, first, n, a.stride, a.dense_logits);
        stage<kBytes, THREADS>(to.masks, a.masks, first, n, a.mask_stride, a.dense_masks);
    }
    copies_commit();
}

// The five parts' softmaxes over their legal choices: d = l - m (-200 where that is lower: such weights are 0 either way),
// w = exp(d), S = sum w, 1 / S, and mean_d = sum w d / S: log p = d - log S and the entropy is log S - mean_d, so log p + H =
// d - mean_d needs no logarithm. exp as 2^(d log2 e) by the hardware's instruction, 2 ulp: the rounding of d itself costs as
// much. The choices are known, so the parts do not wait for one another: all 19 logits go side by side.
struct SoftRow {
    float d[kBytes], w[kBytes], sum[kParts], inv[kParts], mean_d[kParts];
    float choice_d[kParts];   // the choice's d; -inf where it is not legal
    unsigned some;            // bit k: part k has a legal choice
};

template <int R, class P>
__device__ __forceinline__ void soft_rows(SoftRow (&s)[R], P const (&logits)[R], const uint8_t* const (&mask)[R], const float* tab,
                                          const int (&c)[R][kParts]) {
    float m[R][kParts];
    bool odd = false;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
#pragma unroll
            for (int i = 0; i < part_n(k); ++i) {
                const int e = part_at(k) + i;
                float l = to_f(logits[r][e]);
                if (tab) {
#pragma unroll
                    for (int j = 0; j < k; ++j) l += tab[table_at(table_of(k, j)) + c[r][j] * part_n(k) + i];
                }
                s[r].d[e] = mask[r][e] != 0 ? l : -INFINITY;
                m[r][k] = i == 0 ? s[r].d[e] : max_nan(m[r][k], s[r].d[e]);
            }
            odd |= fabsf(m[r][k]) == INFINITY;
        }
#pragma unroll
    for (int r = 0; r < R; ++r) s[r].some = 31;
    if (odd) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float v[kBytes];
#pragma unroll
            for (int e = 0; e < kBytes; ++e) v[e] = s[r].d[e];
#pragma unroll
            for (int k = 0; k < kParts; ++k)
                if (fabsf(m[r][k]) == INFINITY && !settle(v + part_at(k), part_n(k), mask[r] + part_at(k), m[r][k])) s[r].some &= ~(1u << k);
#pragma unroll
            for (int e = 0; e < kBytes; ++e) s[r].d[e] = v[e];
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
            float sum = 0.f, t = 0.f;
            s[r].choice_d[k] = 0.f;
#pragma unroll
            for (int i = 0; i < part_n(k); ++i) {
                const int e = part_at(k) + i;
                const float d = s[r].d[e] - m[r][k];
                if (i == c[r][k]) s[r].choice_d[k] = d;
                s[r].d[e] = max_nan(d, -200.f);
                s[r].w[e] = __expf(s[r].d[e]);
                sum += s[r].w[e];
                t = fmaf(s[r].w[e], s[r].d[e], t);
            }
            s[r].sum[k] = sum;
            s[r].inv[k] = __fdividef(1.f, sum);   // the hardware's reciprocal, 1 ulp; S is between 1 and 9
            s[r].mean_d[k] = t * s[r].inv[k];
        }
}

__device__ __forceinline__ bool parts_of(int id, int* c) {
    const bool known = id >= 0 && id < kMoves;
    if (!known) id = 0;
    c[0] = id % 9;
    c[1] = id / 9 % 3;
    c[2] = id / 27 % 3;
    c[3] = id / 81 % 2;
    c[4] = id / 162;
    return known;
}

template <class T>
__global__ void __launch_bounds__(kThreads) k_moves_logp(LogpArgs a) {
    extern __shared__ __align__(16) unsigned char batches[];
    __shared__ float tab_s[kCond];
    auto* batch = reinterpret_cast<LogpBatch<T, kThreads>*>(batches);
    const long long step = static_cast<long long>(gridDim.x) * kThreads;
    long long first = static_cast<long long>(blockIdx.x) * kThreads;
    fetch_batch<kThreads>(a, first, batch[0]);
    load_cond(tab_s, a.cond);
    const float* tab = a.cond.type < 0 ? nullptr : tab_s;
    for (int b = 0; first < a.rows; first += step, b ^= 1) {
        fetch_batch<kThreads>(a, first + step, batch[b ^ 1]);
        const long long row = first + threadIdx.x;
        const int id = row < a.rows ? a.ids[row] : 0;
        copies_wait<1>();
        __syncthreads();
        if (row < a.rows) {
            int c[1][kParts];
            const bool known = parts_of(id, c[0]);   // else no move has this id
            const T* const logits[1] = {batch[b].logits + threadIdx.x * kBytes};
            const uint8_t* const mask[1] = {batch[b].masks + threadIdx.x * kBytes};
            SoftRow rows[1];
            soft_rows<1>(rows, logits, mask, tab, c);
            const SoftRow& s = rows[0];
            float d_sum = 0.f, mean_sum = 0.f, sums = 1.f;   // one logarithm for the five parts
#pragma unroll
            for (int k = 0; k < kParts; ++k)
                if (s.some >> k & 1) {
                    d_sum += s.choice_d[k];
                    mean_sum += s.mean_d[k];
                    sums *= s.sum[k];
                }
            const float log_sums = logf(sums);
            a.logp[row] = known ? d_sum - log_sums : NAN;
            a.entropy[row] = known ? log_sums - mean_sum : NAN;
        }
        __syncthreads();   // the batch may be written again
    }
}

// dl = ga 1[i = c] - p (ga + gb (d - mean_d)), in the logits' place in shared memory and from there to memory as one stretch.
// Every thread sums the tables' gradient in a column of its own of shared memory, so that no two add to one place and the
// order of the additions is the launch's alone; the 23 additions of a row go to 23 places, so they are read together and
// written together. The columns' 508 bytes per thread leave 8 to 10 warps per SM, so a thread takes R = 2 rows side by side
// where there are rows for it (8,192 x 128 rows: 76 us with one row per thread and the next batch on its way, 80 us with two
// and 256 threads, 70 us with two and 128, 59 us with two and blocks of 64); one row each where every block has one batch
// at most.
template <class T, int THREADS, int R>
__global__ void __launch_bounds__(THREADS) k_moves_grad(LogpArgs a) {
    extern __shared__ __align__(16) unsigned char batches[];   // a batch, then [127][THREADS] sums
    __shared__ float tab_s[kCond];
    __shared__ uint8_t none_s[kBytes];
    constexpr int kRows = R * THREADS;
    auto& batch = *reinterpret_cast<LogpBatch<T, kRows>*>(batches);
    float* acc_s = reinterpret_cast<float*>(batches + sizeof(batch));
    const long long step = static_cast<long long>(gridDim.x) * kRows;
    long long first = static_cast<long long>(blockIdx.x) * kRows;
    fetch_batch<THREADS>(a, first, batch);
    if (threadIdx.x < kBytes) none_s[threadIdx.x] = 0;
    load_cond(tab_s, a.cond);
    float* acc = a.part ? acc_s + threadIdx.x : nullptr;
    if (acc)
        for (int e = 0; e < kCond; ++e) acc[e * THREADS] = 0.f;
    const float* tab = a.cond.type < 0 ? nullptr : tab_s;
    for (; first < a.rows; first += step) {
        float ga[R], gb[R];
        int id[R], c[R][kParts];
        T* logits[R];
        const uint8_t* mask[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int at = threadIdx.x + r * THREADS;
            const long long row = first + at;
            ga[r] = gb[r] = 0.f;
            id[r] = -1;
            if (row < a.rows) {
                id[r] = a.ids[row];
                if (a.glp) ga[r] = a.glp[row * a.glp_stride];
                if (a.gent) gb[r] = a.gent[row * a.gent_stride];
            }
            logits[r] = batch.logits + at * kBytes;
            // behind the last row, or no move's id: nothing is legal, nothing is added
            mask[r] = parts_of(id[r], c[r]) ? batch.masks + at * kBytes : none_s;
        }
        copies_wait<0>();
        __syncthreads();
        SoftRow s[R];
        soft_rows<R>(s, logits, mask, tab, c);
        float g[R][kBytes];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int k = 0; k < kParts; ++k) {
                const bool some = s[r].some >> k & 1;
                const int hit = some && mask[r][part_at(k) + c[r][k]] != 0 ? c[r][k] : -1;
                const float gk = some ? ga[r] : 0.f, bk = some ? gb[r] : 0.f, inv = some ? s[r].inv[k] : 0.f;
                const float mean = some ? s[r].mean_d[k] : 0.f;
#pragma unroll
                for (int i = 0; i < part_n(k); ++i) {
                    const int e = part_at(k) + i;
                    g[r][e] = fmaf(-s[r].w[e] * inv, fmaf(bk, s[r].d[e] - mean, gk), i == hit ? gk : 0.f);
                }
            }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (acc) {
                float sum[23];
                int n = 0;
#pragma unroll
                for (int k = 1; k < kParts; ++k)
#pragma unroll
                    for (int j = 0; j < k; ++j)
#pragma unroll
                        for (int i = 0; i < part_n(k); ++i)
                            sum[n++] = acc[(table_at(table_of(k, j)) + c[r][j] * part_n(k) + i) * THREADS] + g[r][part_at(k) + i];
                n = 0;
#pragma unroll
                for (int k = 1; k < kParts; ++k)
#pragma unroll
                    for (int j = 0; j < k; ++j)
#pragma unroll
                        for (int i = 0; i < part_n(k); ++i)
                            acc[(table_at(table_of(k, j)) + c[r][j] * part_n(k) + i) * THREADS] = sum[n++];
            }
#pragma unroll
            for (int e = 0; e < kBytes; ++e) logits[r][e] = from_f<T>(g[r][e]);
        }
        __syncthreads();
        if (a.dlogits) {
            const int n = static_cast<int>(min(static_cast<long long>(kRows), a.rows - first)) * kBytes;
            T* out = static_cast<T*>(a.dlogits) + first * kBytes;
            constexpr int kPer = 16 / static_cast<int>(sizeof(T));
            const int whole = a.dense_out ? n & ~(kPer - 1) : 0;
            for (int i = threadIdx.x * kPer; i < whole; i += THREADS * kPer)
                *reinterpret_cast<uint4*>(out + i) = *reinterpret_cast<const uint4*>(batch.logits + i);
            for (int i = whole + threadIdx.x; i < n; i += THREADS) out[i] = batch.logits[i];
        }
        __syncthreads();   // the batch may be written again
        fetch_batch<THREADS>(a, first + step, batch);
    }
    copies_wait<0>();
    if (!a.part) return;
    for (int e = threadIdx.x; e < kCond; e += THREADS) {   // each reader starts at a bank of its own
        float t = 0.f;
        for (int j = 0; j < THREADS; ++j) t += acc_s[e * THREADS + (j + e) % THREADS];
        a.part[static_cast<long long>(blockIdx.x) * kCond + e] = t;
    }
}

// A warp per table entry adds the blocks' partial sums, in a fixed order.
__global__ void __launch_bounds__(32) k_moves_grad_sum(const float* part, int blocks, float* dcond) {
    float t = 0.f;
    for (int b = threadIdx.x; b < blocks; b += 32) t += part[static_cast<long long>(b) * kCond + blockIdx.x];
#pragma unroll
    for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(~0u, t, o);
    if (threadIdx.x == 0) dcond[blockIdx.x] = t;
}

constexpr int kGradThreads = 64, kGradBlocks = 5;   // of the backward, and per SM: 32 KB of table sums and 12 KB of rows each

int current_device() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess ? dev : -1;
}

// The current device's SM count, asked once per device.
int sm_count() {
    static std::atomic<int> known[kDevices];
    const int dev = current_device();
    const bool kept = dev >= 0 && dev < kDevices;
    int sms = kept ? known[dev].load(std::memory_order_relaxed) : 0;
    if (sms > 0) return sms;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 1) return 148;
    if (kept) known[dev].store(sms, std::memory_order_relaxed);
    return sms;
}

// Launches a kernel that may need more shared memory than the 48 KB it has unasked; `most`, the most that it is ever
// launched with, is asked for once per device.
template <auto KERNEL, class A>
cudaError_t launch(unsigned grid, int block, size_t smem, size_t most, cudaStream_t stream, const A& a) {
    static std::atomic<bool> asked[kDevices];
    if (most > 48 * 1024) {
        const int dev = current_device();
        if (dev < 0 || dev >= kDevices || !asked[dev].load(std::memory_order_acquire)) {
            const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most));
            if (e != cudaSuccess) return e;
            if (dev >= 0 && dev < kDevices) asked[dev].store(true, std::memory_order_release);
        }
    }
    KERNEL<<<grid, static_cast<unsigned>(block), smem, stream>>>(a);
    return cudaSuccess;
}

bool dense(const void* p, bool end_to_end) { return end_to_end && reinterpret_cast<uintptr_t>(p) % 16 == 0; }

unsigned blocks_for(long long rows, long long per_block, long long most) {
    const long long n = (rows + per_block - 1) / per_block;
    return static_cast<unsigned>(n < most ? n : most);
}

int failed(const char* msg) {
    g_heads_error = msg;
    return 1;
}

bool fill_cond(Cond& c, const void* const* tables, int type) {
    c.type = tables ? type : -1;
    for (int t = 0; t < kTables; ++t) {
        c.table[t] = tables ? tables[t] : nullptr;
        if (tables && !tables[t]) return false;
    }
    return !tables || (type >= 0 && type <= 2);
}

template <class F>
bool with_type(int type, F f) {
    if (type == 0) f(float{});
    else if (type == 1) f(__nv_bfloat16{});
    else if (type == 2) f(__half{});
    else return false;
    return true;
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

const char* bad_cut(float temperature, const void* temperatures, float top_p, const void* top_ps, float min_p,
                    const void* min_ps) {
    if (!temperatures && !(temperature >= 0.f)) return "temperature must be 0 or more";
    if (!top_ps && !(top_p >= 0.f)) return "top_p must be 0 or more";
    if (!min_ps && !(min_p <= 1.f)) return "min_p must be at most 1";
    return nullptr;
}

}  // namespace

extern "C" {

const char* rl_heads_error(void) { return g_heads_error.c_str(); }

int rl_moves_sample(const void* logits, long long stride, int type, const void* const* cond, int cond_type,
                    const void* masks, long long mask_stride, const void* u, float temperature, int top_k, float top_p,
                    float min_p, const void* temperatures, const void* top_ks, const void* top_ps, const void* min_ps,
                    void* ids, void* logp, long long rows, void* stream) {
    if (rows < 0) return failed("rows must not be negative");
    if (const char* e = bad_cut(temperature, temperatures, top_p, top_ps, min_p, min_ps)) return failed(e);
    MoveArgs a;
    if (!fill_cond(a.cond, cond, cond_type)) return failed("cond must be ten tables of fp32, bf16 or fp16");
    if (type < 0 || type > 2) return failed("unknown type of the logits");
    if (rows == 0) return 0;
    if (!logits || !masks || !u || !ids || !logp) return failed("logits, masks, u, ids and logp must be given");
    a.logits = logits;
    a.stride = stride;
    a.masks = static_cast<const uint8_t*>(masks);
    a.mask_stride = mask_stride;
    a.u = static_cast<const float*>(u);
    a.cut = Cut{temperature, top_p, min_p, top_k, static_cast<const float*>(temperatures), static_cast<const float*>(top_ps),
                static_cast<const float*>(min_ps), static_cast<const int*>(top_ks)};
    a.ids = static_cast<int16_t*>(ids);
    a.logp = static_cast<float*>(logp);
    a.rows = rows;
    a.dense_logits = dense(logits, stride == kBytes);
    a.dense_masks = dense(masks, mask_stride == kBytes);
    a.dense_u = dense(u, true);
    const unsigned grid = blocks_for(rows, kThreads, 24ll * sm_count());
    with_type(type, [&](auto t) {
        using T = decltype(t);
        k_moves_sample<T><<<grid, kThreads, 2 * sizeof(MoveBatch<T>), static_cast<cudaStream_t>(stream)>>>(a);
    });
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : failed(cudaGetErrorString(e));
}

int rl_sample(const void* logits, long long stride, int type, int width, const void* legal, long long legal_stride,
              int legal_width, const void* u, float temperature, int top_k, float top_p, float min_p,
              const void* temperatures, const void* top_ks, const void* top_ps, const void* min_ps, void* choice,
              void* logp, long long rows, void* stream) {
    if (rows < 0) return failed("rows must not be negative");
    if (width < 1 || width > kMaxWidth) return failed("width must be 1 .. 4096");
    if (legal && legal_width != width && !(legal_width == kBytes && width == kMoves))
        return failed("legal must have a byte for each choice, or the 19 mask bytes of the 324 moves");
    if (const char* e = bad_cut(temperature, temperatures, top_p, top_ps, min_p, min_ps)) return failed(e);
    if (type < 0 || type > 2) return failed("unknown type of the logits");
    if (rows == 0) return 0;
    if (!logits || !u || !choice || !logp) return failed("logits, u, choice and logp must be given");
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
            const unsigned grid = tpr() == 32 ? blocks_for(rows, 8, kRowWarps<ept()> / 8ll * sm_count())
                                              : blocks_for(rows, 1, kRowWarps<ept()> * 32ll / tpr() * sm_count());
            const unsigned block = tpr() == 32 ? 256 : tpr();
            if (vec) k_rows_sample<T, tpr(), ept(), true><<<grid, block, 0, static_cast<cudaStream_t>(stream)>>>(a);
            else k_rows_sample<T, tpr(), ept(), false><<<grid, block, 0, static_cast<cudaStream_t>(stream)>>>(a);
        });
    });
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : failed(cudaGetErrorString(e));
}

int rl_moves_logp(const void* logits, long long stride, int type, const void* const* cond, int cond_type,
                  const void* masks, long long mask_stride, const void* ids, void* logp, void* entropy, long long rows,
                  void* stream) {
    if (rows < 0) return failed("rows must not be negative");
    LogpArgs a{};
    if (!fill_cond(a.cond, cond, cond_type)) return failed("cond must be ten tables of fp32, bf16 or fp16");
    if (type < 0 || type > 2) return failed("unknown type of the logits");
    if (rows == 0) return 0;
    if (!logits || !masks || !ids || !logp || !entropy) return failed("logits, masks, ids, logp and entropy must be given");
    a.logits = logits;
    a.stride = stride;
    a.masks = static_cast<const uint8_t*>(masks);
    a.mask_stride = mask_stride;
    a.ids = static_cast<const int16_t*>(ids);
    a.logp = static_cast<float*>(logp);
    a.entropy = static_cast<float*>(entropy);
    a.rows = rows;
    a.dense_logits = dense(logits, stride == kBytes);
    a.dense_masks = dense(masks, mask_stride == kBytes);
    const unsigned grid = blocks_for(rows, kThreads, 24ll * sm_count());
    with_type(type, [&](auto t) {
        using T = decltype(t);
        k_moves_logp<T><<<grid, kThreads, 2 * sizeof(LogpBatch<T, kThreads>), static_cast<cudaStream_t>(stream)>>>(a);
    });
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : failed(cudaGetErrorString(e));
}

size_t rl_moves_logp_bwd_work_bytes(void) { return static_cast<size_t>(kGradBlocks) * sm_count() * kCond * sizeof(float); }

int rl_moves_logp_bwd(const void* glp, long long glp_stride, const void* gent, long long gent_stride, const void* logits,
                      long long stride, int type, const void* const* cond, int cond_type, const void* masks,
                      long long mask_stride, const void* ids, void* dlogits, void* dcond, long long rows, void* work,
                      size_t work_bytes, void* stream) {
    if (rows < 1) return failed("rows must be positive");
    LogpArgs a{};
    if (!fill_cond(a.cond, cond, cond_type)) return failed("cond must be ten tables of fp32, bf16 or fp16");
    if (type < 0 || type > 2) return failed("unknown type of the logits");
    if (!logits || !masks || !ids) return failed("logits, masks and ids must be given");
    if (dcond && !cond) return failed("dcond needs the tables");
    if (dcond && (!work || work_bytes < rl_moves_logp_bwd_work_bytes()))
        return failed("work space smaller than rl_moves_logp_bwd_work_bytes()");
    a.logits = logits;
    a.stride = stride;
    a.masks = static_cast<const uint8_t*>(masks);
    a.mask_stride = mask_stride;
    a.ids = static_cast<const int16_t*>(ids);
    a.glp = static_cast<const float*>(glp);
    a.gent = static_cast<const float*>(gent);
    a.glp_stride = glp_stride;
    a.gent_stride = gent_stride;
    a.dlogits = dlogits;
    a.part = dcond ? static_cast<float*>(work) : nullptr;
    a.rows = rows;
    a.dense_logits = dense(logits, stride == kBytes);
    a.dense_masks = dense(masks, mask_stride == kBytes);
    a.dense_out = dense(dlogits, true);
    auto s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    unsigned grid = 0;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        auto run = [&](auto per_thread) {
            constexpr int R = per_thread();
            constexpr size_t kBatch = sizeof(LogpBatch<T, R * kGradThreads>);
            constexpr size_t kSums = static_cast<size_t>(kCond) * kGradThreads * sizeof(float);
            grid = blocks_for(rows, R * kGradThreads, static_cast<long long>(kGradBlocks) * sm_count());
            e = launch<k_moves_grad<T, kGradThreads, R>>(grid, kGradThreads, dcond ? kBatch + kSums : kBatch, kBatch + kSums, s, a);
        };
        if (rows <= static_cast<long long>(kGradBlocks) * kGradThreads * sm_count()) run(std::integral_constant<int, 1>{});
        else run(std::integral_constant<int, 2>{});
    });
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e == cudaSuccess && dcond) {
        k_moves_grad_sum<<<kCond, 32, 0, s>>>(a.part, static_cast<int>(grid), static_cast<float*>(dcond));
        e = cudaGetLastError();
    }
    return e == cudaSuccess ? 0 : failed(cudaGetErrorString(e));
}

}  // extern "C"
