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

#include <cmath>
#include <cstdint>
#include <string>
#include "../../include/rlenv_api.h"   // rl_sample, rl_moves_* compiled against their C-ABI declarations

namespace {

constexpr int kParts = 5, kBytes = 19, kMoves = 324, kTables = 10, kCond = 127;
constexpr float kScale = 134217728.f;   // 2^27
constexpr float kUnit = 1.f / kScale;
constexpr int kThreads = 128;
constexpr int kRowThreads = 256;
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
    if (!(t > 0.f)) {   // 0 (or nothing a temperature can be): the best choice alone
        r.top_k = 1;
        r.scale = 1.f;
    }
    r.cut = r.top_k > 0 || r.top_p < 1.f || r.min_p > 0.f;
    return r;
}

// W of a scaled logit d <= 0 (a NaN, -inf at an infinite temperature, weighs nothing).
__device__ __forceinline__ unsigned weight_of(float d) { return d <= 0.f ? __float2uint_rn(expf(d) * kScale) : 0u; }

__device__ __forceinline__ unsigned bits24(float u) {
    const int v = static_cast<int>(u * 16777216.f);   // a NaN is 0
    return static_cast<unsigned>(min(max(v, 0), 0xFFFFFF));
}

// All ten tables, in fp32, into shared memory.
__device__ __forceinline__ void load_cond(float* tab, const Cond& c) {
    if (c.type < 0) return;
#pragma unroll
    for (int k = 1; k < kParts; ++k)
#pragma unroll
        for (int j = 0; j < k; ++j) {
            const int t = table_of(k, j), n = part_n(j) * part_n(k);
            for (int i = threadIdx.x; i < n; i += blockDim.x) {
                const float v = c.type == 0 ? static_cast<const float*>(c.table[t])[i]
                                : c.type == 1 ? to_f(static_cast<const __nv_bfloat16*>(c.table[t])[i])
                                              : to_f(static_cast<const __half*>(c.table[t])[i]);
                tab[table_at(t) + i] = v;
            }
        }
}

// One choice among the legal ones of N logits; adds its log-probability to lp.
template <int N>
__device__ __forceinline__ int choose(float (&l)[N], unsigned legal, float u, const RowCut& q, float& lp) {
    if (!legal) return 0;
    float m = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (l[i] != l[i]) {   // a NaN is chosen as -inf is, and shows in the log-probability
            nan |= legal >> i & 1;
            l[i] = -INFINITY;
        }
        if (legal >> i & 1) m = fmaxf(m, l[i]);
    }
    float d[N];
    unsigned w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        d[i] = l[i] == m ? 0.f : (l[i] - m) * q.scale;
        w[i] = legal >> i & 1 ? weight_of(d[i]) : 0u;
    }
    if (q.cut) {
        int rank[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            rank[i] = 0;
#pragma unroll
            for (int j = 0; j < N; ++j)
                rank[i] += j != i && (legal >> j & 1) && (l[j] > l[i] || (j < i && !(l[i] > l[j])));
        }
        const int top = q.top_k > 0 ? q.top_k : N;
        unsigned total = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (rank[i] >= top) w[i] = 0;
            total += w[i];
        }
        const double reach = static_cast<double>(q.top_p) * static_cast<double>(total);
        const double least = static_cast<double>(q.min_p) * static_cast<double>(kScale);
        unsigned kept = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            unsigned before = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) before += rank[j] < rank[i] ? w[j] : 0u;
            const bool keep = rank[i] == 0 || (static_cast<double>(before) < reach && static_cast<double>(w[i]) >= least);
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
    lp += nan ? NAN : dc - logf(static_cast<float>(total) * kUnit);
    return c;
}

// Part K's logits of a row whose earlier choices are c[0..K).
template <int K, class T>
__device__ __forceinline__ void part_logits(float (&l)[part_n(K)], const T* logits, const float* tab, const int* c) {
#pragma unroll
    for (int i = 0; i < part_n(K); ++i) l[i] = to_f(logits[part_at(K) + i]);
    if (tab) {
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int i = 0; i < part_n(K); ++i) l[i] += tab[table_at(table_of(K, j)) + c[j] * part_n(K) + i];
    }
}

template <int K>
__device__ __forceinline__ unsigned part_legal(const uint8_t* mask) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < part_n(K); ++i) m |= static_cast<unsigned>(mask[part_at(K) + i] != 0) << i;
    return m;
}

struct MoveArgs {
    const void* logits;
    long long stride;
    Cond cond;
    const uint8_t* masks;
    long long mask_stride;
    const float* u;
    Cut cut;
    int16_t* ids;
    float* logp;
    long long rows;
};

template <int K, class T>
__device__ __forceinline__ void draw_part(const MoveArgs& a, const T* logits, const uint8_t* mask, const float* u,
                                          const RowCut& q, const float* tab, int* c, float& lp) {
    float l[part_n(K)];
    part_logits<K>(l, logits, tab, c);
    c[K] = choose<part_n(K)>(l, part_legal<K>(mask), u[K], q, lp);
}

// A thread per row.
template <class T>
__global__ void __launch_bounds__(kThreads) k_moves_sample(MoveArgs a) {
    __shared__ float tab_s[kCond];
    load_cond(tab_s, a.cond);
    __syncthreads();
    const float* tab = a.cond.type < 0 ? nullptr : tab_s;
    for (long long row = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; row < a.rows;
         row += static_cast<long long>(gridDim.x) * blockDim.x) {
        const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
        const uint8_t* mask = a.masks + row * a.mask_stride;
        const float* u = a.u + row * kParts;
        const RowCut q = row_cut(a.cut, row);
        int c[kParts];
        float lp = 0.f;
        draw_part<0>(a, logits, mask, u, q, tab, c, lp);
        draw_part<1>(a, logits, mask, u, q, tab, c, lp);
        draw_part<2>(a, logits, mask, u, q, tab, c, lp);
        draw_part<3>(a, logits, mask, u, q, tab, c, lp);
        draw_part<4>(a, logits, mask, u, q, tab, c, lp);
        a.ids[row] = static_cast<int16_t>(c[0] + 9 * c[1] + 27 * c[2] + 81 * c[3] + 162 * c[4]);
        a.logp[row] = lp;
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

// A whole number that orders floats as the floats do (-0 as 0; a NaN as -inf); 0 is below all of them.
__device__ __forceinline__ unsigned key_of(float l) {
    if (l != l) l = -INFINITY;
    const unsigned b = __float_as_uint(l + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct BlockSums {
    unsigned long long part[kRowThreads / 32];
};

__device__ __forceinline__ unsigned long long block_sum(unsigned long long v, BlockSums& s) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.part[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned long long t = 0;
    for (int w = 0; w < kRowThreads / 32; ++w) t += s.part[w];
    return t;
}

__device__ __forceinline__ bool move_legal(const uint8_t* m, int i) {
    bool ok = m[i % 9] != 0;
    i /= 9;
    ok &= m[9 + i % 3] != 0;
    i /= 3;
    ok &= m[12 + i % 3] != 0;
    i /= 3;
    return ok && m[15 + i % 2] != 0 && m[17 + i / 2] != 0;
}

// A block per row. The row's keys and weights lie in shared memory; what top-k and top-p keep is a run of the ranked
// choices, so its lowest key is found by bisection over the key's 32 bits, and the last group of equal keys is cut by index.
template <class T>
__global__ void __launch_bounds__(kRowThreads) k_rows_sample(RowArgs a) {
    extern __shared__ unsigned smem[];
    __shared__ BlockSums sums;
    __shared__ unsigned long long scan[kRowThreads];
    __shared__ int found;
    unsigned* key = smem;
    unsigned* wgt = smem + a.width;
    const int n = a.width, tid = threadIdx.x;
    const int each = (n + kRowThreads - 1) / kRowThreads;
    const int lo = min(n, tid * each), hi = min(n, lo + each);   // this thread's stretch in index order
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
        const uint8_t* legal = a.legal ? a.legal + row * a.legal_stride : nullptr;
        const RowCut q = row_cut(a.cut, row);
        __syncthreads();   // the previous row's shared memory is free
        if (tid == 0) found = 0;
        unsigned top = 0;
        int any = 0, nan = 0;
        for (int i = tid; i < n; i += kRowThreads) {
            const float l = to_f(logits[i]);
            const bool ok = !legal || (a.legal_width == n ? legal[i] != 0 : move_legal(legal, i));
            const unsigned k = ok ? key_of(l) : 0u;
            key[i] = k;
            top = max(top, k);
            any |= ok;
            nan |= ok && l != l;   // chosen as -inf is, and shown in the log-probability
        }
        top = __reduce_max_sync(~0u, top);
        if ((tid & 31) == 0) scan[tid >> 5] = top;
        any = __syncthreads_or(any);
        nan = __syncthreads_or(nan);
        for (int w = 0; w < kRowThreads / 32; ++w) top = max(top, static_cast<unsigned>(scan[w]));
        const float m = top & 0x80000000u ? __uint_as_float(top & 0x7FFFFFFFu) : __uint_as_float(~top);
        for (int i = tid; i < n; i += kRowThreads) {
            float l = to_f(logits[i]);
            if (l != l) l = -INFINITY;
            wgt[i] = key[i] ? weight_of(l == m ? 0.f : (l - m) * q.scale) : 0u;
        }
        __syncthreads();
        if (any && q.cut) {
            if (q.top_k > 0 && q.top_k < n) {
                // the largest key t with at least k keys >= t, then its group's first by index
                unsigned t = 0;
                for (int b = 31; b >= 0; --b) {
                    const unsigned cand = t | 1u << b;
                    unsigned long long c = 0;
                    for (int i = tid; i < n; i += kRowThreads) c += key[i] >= cand;
                    if (block_sum(c, sums) >= static_cast<unsigned>(q.top_k)) t = cand;
                }
                if (t) {
                    unsigned long long above = 0, mine = 0;
                    for (int i = lo; i < hi; ++i) {
                        above += key[i] > t;
                        mine += key[i] == t;
                    }
                    above = block_sum(above, sums);
                    scan[tid] = mine;
                    __syncthreads();
                    unsigned long long rank = above;
                    for (int w = 0; w < tid; ++w) rank += scan[w];
                    for (int i = lo; i < hi; ++i) {
                        bool drop = key[i] < t;
                        if (key[i] == t) drop = rank++ >= static_cast<unsigned>(q.top_k);
                        if (drop) key[i] = wgt[i] = 0;
                    }
                    __syncthreads();
                }
            }
            unsigned long long s = 0;
            for (int i = tid; i < n; i += kRowThreads) s += wgt[i];
            const double reach = static_cast<double>(q.top_p) * static_cast<double>(block_sum(s, sums));
            // the smallest t for which the weights above t do not reach: what is ranked below the keys >= t goes
            unsigned t = 0;
            if (q.top_p < 1.f) {
                for (int b = 31; b >= 0; --b) {
                    const unsigned cand = t | ((1u << b) - 1u);   // the largest value with t's upper bits and this one 0
                    unsigned long long v = 0;
                    for (int i = tid; i < n; i += kRowThreads) v += key[i] > cand ? wgt[i] : 0u;
                    if (!(static_cast<double>(block_sum(v, sums)) < reach)) t |= 1u << b;
                }
                if (t > top) t = top;   // p <= 0: the best choice alone
            }
            // the lowest key that stays, its group and the weight above it
            unsigned low = ~0u;
            for (int i = tid; i < n; i += kRowThreads)
                if (key[i] && key[i] >= t) low = min(low, key[i]);
            low = __reduce_min_sync(~0u, low);
            __syncthreads();
            if ((tid & 31) == 0) scan[tid >> 5] = low;
            __syncthreads();
            for (int w = 0; w < kRowThreads / 32; ++w) low = min(low, static_cast<unsigned>(scan[w]));
            __syncthreads();
            unsigned long long above = 0, mine = 0;
            for (int i = lo; i < hi; ++i) {
                above += key[i] > low ? wgt[i] : 0u;
                mine += key[i] == low ? wgt[i] : 0u;
            }
            above = block_sum(above, sums);
            scan[tid] = mine;
            __syncthreads();
            unsigned long long run = above;
            bool first = low == top;   // whether the best choice of all is in this group: the first by index is it
            for (int w = 0; w < tid; ++w) {
                run += scan[w];
                first &= scan[w] == 0;
            }
            const double least = static_cast<double>(q.min_p) * static_cast<double>(kScale);
            for (int i = lo; i < hi; ++i) {
                bool keep = key[i] >= low;
                if (key[i] == low) {
                    if (q.top_p < 1.f) keep = first || static_cast<double>(run) < reach;
                    first = false;
                    run += wgt[i];
                }
                if (!keep || (key[i] != top && static_cast<double>(wgt[i]) < least)) wgt[i] = 0;
            }
            __syncthreads();
        }
        unsigned long long mine = 0;
        for (int i = lo; i < hi; ++i) mine += wgt[i];
        const unsigned long long total = block_sum(mine, sums);
        const unsigned long long target = (bits24(a.u[row]) * total) >> 24;
        scan[tid] = mine;
        __syncthreads();
        unsigned long long run = 0;
        for (int w = 0; w < tid; ++w) run += scan[w];
        if (run <= target && target < run + mine)
            for (int i = lo; i < hi; ++i) {
                run += wgt[i];
                if (run > target) {
                    found = i;
                    break;
                }
            }
        __syncthreads();
        if (tid == 0) {
            const int c = any ? found : 0;
            float lp = 0.f;
            if (any) {
                const float l = to_f(logits[c]);
                lp = nan ? NAN : (l == m ? 0.f : (l - m) * q.scale) - logf(static_cast<float>(total) * kUnit);
            }
            a.choice[row] = c;
            a.logp[row] = lp;
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
    const int16_t* ids;
    float *logp, *entropy;               // forward
    const float *glp, *gent;             // backward: incoming gradients, either may be null
    long long glp_stride, gent_stride;
    void* dlogits;                       // [rows, 19] of the logits' type, or null
    float* part;                         // [blocks][127] partial sums of the tables' gradient, or null
    long long rows;
};

// A part's softmax over its legal choices: weights exp(l - m), their sum, l - m.
template <int N>
struct Soft {
    float d[N], w[N], sum, log_sum;
    unsigned legal;
};

template <int K, class T>
__device__ __forceinline__ void soft_part(Soft<part_n(K)>& s, const T* logits, const uint8_t* mask, const float* tab,
                                          const int* c) {
    constexpr int N = part_n(K);
    part_logits<K>(s.d, logits, tab, c);
    s.legal = part_legal<K>(mask);
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (s.legal >> i & 1) m = fmaxf(m, s.d[i]);
    s.sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        s.d[i] = s.d[i] == m ? 0.f : s.d[i] - m;
        s.w[i] = s.legal >> i & 1 ? expf(s.d[i]) : 0.f;
        s.sum += s.w[i];
    }
    s.log_sum = logf(s.sum);
}

template <int N>
__device__ __forceinline__ float entropy_of(const Soft<N>& s) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (s.w[i] != 0.f) t = fmaf(s.w[i], s.d[i], t);
    return s.log_sum - __fdiv_rn(t, s.sum);
}

template <int K, class T>
__device__ __forceinline__ void logp_part(const T* logits, const uint8_t* mask, const float* tab, const int* c, float& lp,
                                          float& ent) {
    constexpr int N = part_n(K);
    Soft<N> s;
    soft_part<K>(s, logits, mask, tab, c);
    if (!s.legal) return;
    float dc = -INFINITY;   // a choice that is not legal
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i == c[K] && (s.legal >> i & 1)) dc = s.d[i];
    lp += dc - s.log_sum;
    ent += entropy_of<N>(s);
}

__device__ __forceinline__ bool parts_of(int id, int* c) {
    c[0] = id % 9;
    c[1] = id / 9 % 3;
    c[2] = id / 27 % 3;
    c[3] = id / 81 % 2;
    c[4] = id / 162;
    return id >= 0 && id < kMoves;
}

template <class T>
__global__ void __launch_bounds__(kThreads) k_moves_logp(LogpArgs a) {
    __shared__ float tab_s[kCond];
    load_cond(tab_s, a.cond);
    __syncthreads();
    const float* tab = a.cond.type < 0 ? nullptr : tab_s;
    for (long long row = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; row < a.rows;
         row += static_cast<long long>(gridDim.x) * blockDim.x) {
        int c[kParts];
        float lp = 0.f, ent = 0.f;
        if (parts_of(a.ids[row], c)) {
            const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
            const uint8_t* mask = a.masks + row * a.mask_stride;
            logp_part<0>(logits, mask, tab, c, lp, ent);
            logp_part<1>(logits, mask, tab, c, lp, ent);
            logp_part<2>(logits, mask, tab, c, lp, ent);
            logp_part<3>(logits, mask, tab, c, lp, ent);
            logp_part<4>(logits, mask, tab, c, lp, ent);
        } else {
            lp = ent = NAN;   // no move has this id
        }
        a.logp[row] = lp;
        a.entropy[row] = ent;
    }
}

// acc: this thread's own column of the block's table sums, kThreads apart.
template <int K, class T>
__device__ __forceinline__ void grad_part(const T* logits, const uint8_t* mask, const float* tab, const int* c, float ga,
                                          float gb, T* dl, float* acc) {
    constexpr int N = part_n(K);
    Soft<N> s;
    soft_part<K>(s, logits, mask, tab, c);
    const float h = s.legal ? entropy_of<N>(s) : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float g = 0.f;
        if (s.legal >> i & 1) {
            const float p = __fdiv_rn(s.w[i], s.sum);
            g = ga * ((i == c[K] ? 1.f : 0.f) - p);
            if (p != 0.f) g -= gb * p * (s.d[i] - s.log_sum + h);
        }
        if (dl) dl[part_at(K) + i] = from_f<T>(g);
        if (acc) {
#pragma unroll
            for (int j = 0; j < K; ++j) acc[(table_at(table_of(K, j)) + c[j] * N + i) * kThreads] += g;
        }
    }
}

// A thread per row; every thread sums the tables' gradient in a column of its own of shared memory, so that no two add
// to one place and the order of the additions is the launch's alone.
template <class T>
__global__ void __launch_bounds__(kThreads) k_moves_grad(LogpArgs a) {
    extern __shared__ float acc_s[];
    __shared__ float tab_s[kCond];
    load_cond(tab_s, a.cond);
    float* acc = a.part ? acc_s + threadIdx.x : nullptr;
    if (acc)
        for (int e = 0; e < kCond; ++e) acc[e * kThreads] = 0.f;
    __syncthreads();
    const float* tab = a.cond.type < 0 ? nullptr : tab_s;
    for (long long row = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; row < a.rows;
         row += static_cast<long long>(gridDim.x) * blockDim.x) {
        int c[kParts];
        T* dl = a.dlogits ? static_cast<T*>(a.dlogits) + row * kBytes : nullptr;
        if (parts_of(a.ids[row], c)) {
            const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
            const uint8_t* mask = a.masks + row * a.mask_stride;
            const float ga = a.glp ? a.glp[row * a.glp_stride] : 0.f, gb = a.gent ? a.gent[row * a.gent_stride] : 0.f;
            grad_part<0>(logits, mask, tab, c, ga, gb, dl, acc);
            grad_part<1>(logits, mask, tab, c, ga, gb, dl, acc);
            grad_part<2>(logits, mask, tab, c, ga, gb, dl, acc);
            grad_part<3>(logits, mask, tab, c, ga, gb, dl, acc);
            grad_part<4>(logits, mask, tab, c, ga, gb, dl, acc);
        } else if (dl) {
            for (int i = 0; i < kBytes; ++i) dl[i] = from_f<T>(0.f);
        }
    }
    if (!a.part) return;
    __syncthreads();
    if (threadIdx.x < kCond) {
        float t = 0.f;
        for (int j = 0; j < kThreads; ++j) t += acc_s[threadIdx.x * kThreads + (j + threadIdx.x) % kThreads];
        a.part[static_cast<long long>(blockIdx.x) * kCond + threadIdx.x] = t;
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

constexpr size_t kGradSmem = static_cast<size_t>(kCond) * kThreads * sizeof(float);

int sm_count() {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

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
    const unsigned grid = blocks_for(rows, kThreads, 16ll * sm_count());
    with_type(type, [&](auto t) { k_moves_sample<decltype(t)><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a); });
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
    const unsigned grid = blocks_for(rows, 1, 8ll * sm_count());
    const size_t smem = 2 * sizeof(unsigned) * static_cast<size_t>(width);
    with_type(type, [&](auto t) {
        k_rows_sample<decltype(t)><<<grid, kRowThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
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
    const unsigned grid = blocks_for(rows, kThreads, 16ll * sm_count());
    with_type(type, [&](auto t) { k_moves_logp<decltype(t)><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a); });
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : failed(cudaGetErrorString(e));
}

size_t rl_moves_logp_bwd_work_bytes(void) { return static_cast<size_t>(3) * sm_count() * kCond * sizeof(float); }

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
    const unsigned grid = blocks_for(rows, kThreads, 3ll * sm_count());
    const size_t smem = dcond ? kGradSmem : 0;
    auto s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    with_type(type, [&](auto t) {
        auto k = k_moves_grad<decltype(t)>;
        e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kGradSmem));
        if (e == cudaSuccess) k<<<grid, kThreads, smem, s>>>(a);
    });
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e == cudaSuccess && dcond) {
        k_moves_grad_sum<<<kCond, 32, 0, s>>>(a.part, static_cast<int>(grid), static_cast<float*>(dcond));
        e = cudaGetLastError();
    }
    return e == cudaSuccess ? 0 : failed(cudaGetErrorString(e));
}

}  // extern "C"
