// The policy's ordered action heads (rl/model.py:176-194): moves sampled from given random numbers, and the log-probability and
// entropy of given moves, with their gradients.
//
// A move has five parts (d-pad 9, A 3, B 3, Start 2, Select 2 choices). Part k's logits are the head's own plus one row of
// cond[k][j] for each earlier part j, the row of the choice c_j; its legal choices A are the mask bytes that are not 0. Each
// part is drawn as heads.cuh says.
//
// Log-probability and entropy, per part: w = exp(l - m) over A, S = sum w, p = w / S, log p = l - m - log S,
// H = log S - sum w (l - m) / S. With incoming gradients a (of the log-probability) and b (of the entropy):
//   dl_i = a (1[i = c] - p_i) - b p_i (log p_i + H), dcond[k][j][c_j][i] = the sum of dl_i over the rows with that c_j.
// A part with nothing legal answers its choice 0 (neutral, off), and adds 0 to the log-probability, the entropy and the
// gradients. Masked logits are never used, whatever they hold.
//
// A row is 19 logits and some 50 bytes more, and some 970 (a draw), 780 (log-probabilities) or 920 (gradients) instructions: on
// 8,192 x 128 rows the kernels issue in 81 %, 76 % and 50 % of their cycles, and take 37, 34 and 60 us where the bytes alone
// would take 13, 17 and 29. A draw with every truncation takes 66 us there: the ranks and the sums before each choice.
#include "heads.cuh"

using namespace heads;

namespace {

constexpr int kParts = 5, kTables = 10, kCond = 127;
constexpr int kThreads = 128;   // and rows of a block's batch

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

struct Cond {
    const void* table[kTables];
    int type;   // 0 fp32, 1 bf16, 2 fp16; -1: no tables
};

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
    if (q.cut) {   // (each pair compared once for both its ranks and sums: no faster, and 72 registers instead of 56)
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
        unsigned kept = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            unsigned before = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) before += rank[j] < rank[i] ? w[j] : 0u;
            const bool keep = rank[i] == 0 || (before < reach && w[i] >= q.least);
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
// and 256 threads, 70 us with two and 128, 60 us with two and blocks of 64); one row each where every block has one batch
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

bool fill_cond(Cond& c, const void* const* tables, int type) {
    c.type = tables ? type : -1;
    for (int t = 0; t < kTables; ++t) {
        c.table[t] = tables ? tables[t] : nullptr;
        if (tables && (!tables[t] || !fits(tables[t], size_of(type)))) return false;
    }
    return !tables || (type >= 0 && type <= 2);
}

}  // namespace

extern "C" {

const char* rl_heads_error(void) { return g_error.c_str(); }

int rl_moves_sample(const void* logits, long long stride, int type, const void* const* cond, int cond_type,
                    const void* masks, long long mask_stride, const void* u, float temperature, int top_k, float top_p,
                    float min_p, const void* temperatures, const void* top_ks, const void* top_ps, const void* min_ps,
                    void* ids, void* logp, long long rows, void* stream) {
    if (rows < 0) return failed("rows must not be negative");
    if (const char* e = bad_cut(temperature, temperatures, top_p, top_ps, min_p, min_ps, top_ks)) return failed(e);
    MoveArgs a;
    if (!fill_cond(a.cond, cond, cond_type)) return failed("cond must be ten tables of fp32, bf16 or fp16");
    if (type < 0 || type > 2) return failed("unknown type of the logits");
    if (rows == 0) return 0;
    if (!logits || !masks || !u || !ids || !logp) return failed("logits, masks, u, ids and logp must be given");
    if (!fits(logits, size_of(type)) || !fits(u, 4) || !fits(ids, 2) || !fits(logp, 4)) return failed("misaligned pointer");
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

int rl_moves_logp(const void* logits, long long stride, int type, const void* const* cond, int cond_type,
                  const void* masks, long long mask_stride, const void* ids, void* logp, void* entropy, long long rows,
                  void* stream) {
    if (rows < 0) return failed("rows must not be negative");
    LogpArgs a{};
    if (!fill_cond(a.cond, cond, cond_type)) return failed("cond must be ten tables of fp32, bf16 or fp16");
    if (type < 0 || type > 2) return failed("unknown type of the logits");
    if (rows == 0) return 0;
    if (!logits || !masks || !ids || !logp || !entropy) return failed("logits, masks, ids, logp and entropy must be given");
    if (!fits(logits, size_of(type)) || !fits(ids, 2) || !fits(logp, 4) || !fits(entropy, 4)) return failed("misaligned pointer");
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
    if (!fits(logits, size_of(type)) || !fits(dlogits, size_of(type)) || !fits(ids, 2) || !fits(glp, 4) || !fits(gent, 4) ||
        !fits(dcond, 4) || !fits(work, 4))
        return failed("misaligned pointer");
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
