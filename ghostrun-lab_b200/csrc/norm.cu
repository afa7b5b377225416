// Layer norm of the policy's blocks (rl/model.py:64-72 SimBa: x + mlp(norm(x))), with the residual sum before it and its
// gradients. A row s of D values (s = x, or x + residual rounded to x's type: the stream that is kept is the one that
// is normalised):
//   mu = sum s / D, v = sum (s - mu)^2 / D, r = 1 / sqrt(v + eps), xh = (s - mu) r, y = xh w + b
//   h = gy w, dx = r (h - mean(h) - xh mean(h xh)) + gsum, dw = sum over rows of gy xh, db = sum over rows of gy
// All of it in fp32 from the inputs' types, rounded once into the outputs'. The variance is summed from the centred
// values (a second pass), so that a large mean costs no digits.
//
// Bound by memory: every value is read once and written once (1,048,576 x 512 bf16 with residuals: forward 4.3 GB in 703 us,
// 6.1 TB/s; backward 4.3 GB in 609 us, 7.1 TB/s; a plain copy 6.5). A warp or a block therefore keeps a row in registers,
// and the copies of coming rows are under way all the time.
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cstdint>
#include <string>
#include <type_traits>
#include "../../include/rlenv_api.h"   // rl_norm_* compiled against their C-ABI declarations

namespace {

constexpr int kThreads = 256;
constexpr int kWideThreads = 512;
constexpr int kDevices = 64;                               // whose properties are kept
constexpr int kMaxRow = 8192;                              // values of a row that a block's registers hold
constexpr int kCols = 64, kColRows = kThreads / kCols;
// Warps per SM that share the rows (524,288 x 512 bf16 with residuals: 24 warps forward 375 us against 360; 24 backward
// spill, 418 against 279).
constexpr int kFwdWarps = 16, kBwdWarps = 16;
// Rows read value by value have their loads in flight in registers, so 8 values per thread go with more warps (1,048,576 x 201
// bf16 forward: 452 us with 16, 350 with 24).
constexpr int kFwdWarpsOne = 24;

thread_local std::string g_norm_error;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// Element i of the weight or bias, whose type (0 fp32, 1 bf16, 2 fp16) is looked at here: it is read once per block.
__device__ __forceinline__ float load_param(const void* p, int type, long long i) {
    if (type == 0) return static_cast<const float*>(p)[i];
    if (type == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}
// N neighbouring elements from i on (0 behind `width`), 16 bytes at a time where `wide` says that they start there.
template <int N>
__device__ __forceinline__ void load_params(float* out, const void* p, int type, int i, int width, bool wide, float missing) {
    if (p && N > 1 && wide && i < width) {   // whole vectors: the width is a multiple of N
        if (type == 0) {
#pragma unroll
            for (int q = 0; q < N / 4; ++q) {
                const float4 v = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i)[q];
                out[4 * q] = v.x;
                out[4 * q + 1] = v.y;
                out[4 * q + 2] = v.z;
                out[4 * q + 3] = v.w;
            }
            return;
        }
    }
#pragma unroll
    for (int q = 0; q < N; ++q) out[q] = p && i + q < width ? load_param(p, type, i + q) : missing;
}
__device__ __forceinline__ void store_param(void* p, int type, long long i, float v) {
    if (type == 0) static_cast<float*>(p)[i] = v;
    else if (type == 1) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

struct FwdArgs {
    const void *x, *res, *weight, *bias;
    void *y, *sum;
    float2* stats;   // mean and 1 / sqrt(v + eps) of each row, or null
    long long rows, width, x_stride, r_stride;
    int w_type;
    bool w_wide;     // weight and bias start at 16 bytes
    float eps;
};

struct BwdArgs {
    const void *gy, *gsum, *s, *weight;
    const float2* stats;
    void *dx, *dweight, *dbias;
    float* part;     // [splits][2][width]
    long long rows, width, gy_stride, gsum_stride, s_stride;
    int w_type;
    bool w_wide;
    int splits;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

// ------------------------------------------------------------------ rows that fit registers (width <= 8192)
//
// TPR threads share a row, EPT values each, in vectors of 16 bytes (VEC) or one by one: vector v of thread t starts at
// value (v TPR + t) VE. A block of 256 threads (512 for the widest rows) takes 256 / TPR rows at a time and goes on to the
// next ones, whose values are on their way to shared memory meanwhile; the weights stay in registers. Rows that are not
// 16-byte aligned are read one value at a time, the next row's into registers.

__host__ __device__ constexpr int block_of(int tpr) { return tpr > kThreads ? tpr : kThreads; }

// How a row is read: one value at a time; in vectors, some of them behind its end; in vectors that it fills to the last
// (524,288 x 512 bf16 with residuals backward: 278 us with the checks of its end, 244 without).
enum Mode { kOne, kVectors, kFull };

template <class TX, Mode MODE, int TPR, int EPT>
struct Tile {
    static constexpr bool VEC = MODE != kOne;
    static constexpr int kVe = VEC ? 16 / static_cast<int>(sizeof(TX)) : 1;   // values of a vector
    static constexpr int kNv = EPT / kVe;                                     // vectors of a thread
    static constexpr int kBlock = block_of(TPR);
    static constexpr int kRows = kBlock / TPR;                                // rows of a block
    static_assert(kNv * kVe == EPT && kRows * TPR == kBlock, "whole vectors, whole rows");
    __device__ static int at(int v, int t) { return (v * TPR + t) * kVe; }
    __device__ static bool in(int v, int t, int width) { return MODE == kFull || at(v, t) < width; }
};

template <class T, int N>
struct alignas(N * sizeof(T) >= 16 ? 16 : N * sizeof(T)) Pack {
    T v[N];
};

template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, N>*>(p);
}
// Values rounded to T, two at a time where T has an instruction for two.
template <class T, int N>
__device__ __forceinline__ Pack<T, N> rounded(const float* v) {
    Pack<T, N> q;
    if constexpr (N % 2 == 0 && sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            if constexpr (std::is_same_v<T, __nv_bfloat16>) *reinterpret_cast<__nv_bfloat162*>(q.v + i) = __floats2bfloat162_rn(v[i], v[i + 1]);
            else *reinterpret_cast<__half2*>(q.v + i) = __floats2half2_rn(v[i], v[i + 1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) q.v[i] = from_f<T>(v[i]);
    }
    return q;
}
template <class T, int N>
__device__ __forceinline__ void store_pack(T* p, const float* v) {
    *reinterpret_cast<Pack<T, N>*>(p) = rounded<T, N>(v);
}

// The sum over the TPR <= 32 lanes that share a row, in each of them.
template <int TPR>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

// The sums of one or two values over a row's TPR threads, in each of them. `red` has a place for each warp of the block, and
// is free again at the next but one call: the calls alternate between its two halves.
template <int TPR>
__device__ __forceinline__ float2 row_sums(float x, float y, float2* red) {
    x = lanes_sum<TPR>(x);
    y = lanes_sum<TPR>(y);
    if constexpr (TPR > 32) {
        const int warp = threadIdx.x >> 5, first = warp & ~(TPR / 32 - 1);
        if ((threadIdx.x & 31) == 0) red[warp] = make_float2(x, y);
        __syncthreads();
        x = y = 0.f;
#pragma unroll
        for (int w = 0; w < TPR / 32; ++w) {
            x += red[first + w].x;
            y += red[first + w].y;
        }
    }
    return make_float2(x, y);
}

template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* red) {
    x = lanes_sum<TPR>(x);
    if constexpr (TPR > 32) {
        const int warp = threadIdx.x >> 5, first = warp & ~(TPR / 32 - 1);
        if ((threadIdx.x & 31) == 0) red[warp] = x;
        __syncthreads();
        x = 0.f;
#pragma unroll
        for (int w = 0; w < TPR / 32; ++w) x += red[first + w];
    }
    return x;
}

// A thread's own values of coming rows in shared memory, S rows deep: each thread copies (cp.async, 16 bytes at a time)
// and reads back only its own slots, so the copies need no barrier and no registers. A slot of N vectors per row lies
// `kBlock` threads apart: neighbours' 16-byte accesses touch neighbouring banks.
__device__ __forceinline__ void copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <class T, int N, int BLOCK>
__device__ __forceinline__ void copy_pack(uint4* slot, const T* p) {
    constexpr int kWords = static_cast<int>(sizeof(Pack<T, N>) / 16);
#pragma unroll
    for (int q = 0; q < kWords; ++q) copy16(slot + q * BLOCK, reinterpret_cast<const uint4*>(p) + q);
}
template <class T, int N, int BLOCK>
__device__ __forceinline__ Pack<T, N> slot_pack(const uint4* slot) {
    constexpr int kWords = static_cast<int>(sizeof(Pack<T, N>) / 16);
    union { Pack<T, N> p; uint4 u[kWords]; } q;
#pragma unroll
    for (int i = 0; i < kWords; ++i) q.u[i] = slot[i * BLOCK];
    return q.p;
}

// Words of 16 bytes that a thread keeps per row of a tensor of T (0: rows are read as they are needed).
template <class T, bool VEC, int EPT>
constexpr int kWords = VEC ? EPT * static_cast<int>(sizeof(T)) / 16 : 0;
// How many rows ahead fit beside `warps` warps per SM in 208 KB, at most 4 (measured: deeper gains nothing).
template <int WORDS>
constexpr int depth_of(int warps) {
    return WORDS == 0 ? 1 : 208 * 1024 / (warps * 32 * 16 * WORDS) < 4 ? 208 * 1024 / (warps * 32 * 16 * WORDS) : 4;
}

template <class TX, class TY, Mode MODE, int TPR, int EPT>
struct Fwd : Tile<TX, MODE, TPR, EPT> {
    static constexpr int kW = kWords<TX, MODE != kOne, EPT>;
    static constexpr int kBlocks = (MODE != kOne || EPT > 8 ? kFwdWarps : kFwdWarpsOne) * 32 / Fwd::kBlock;   // per SM
    static constexpr int kDepth = depth_of<2 * kW>(kFwdWarps);
    static constexpr size_t kSmem = static_cast<size_t>(kDepth) * 2 * kW * 16 * Fwd::kBlock;
};

template <class TX, class TY, Mode MODE, int TPR, int EPT>
struct Bwd : Tile<TX, MODE, TPR, EPT> {
    static constexpr int kW = kWords<TX, MODE != kOne, EPT>, kG = kWords<TY, MODE != kOne, EPT>;
    static constexpr int kBlocks = kBwdWarps * 32 / Bwd::kBlock;   // per SM
    static constexpr int kDepth = depth_of<2 * kW + kG>(kBwdWarps);
    static constexpr size_t kRing = static_cast<size_t>(kDepth) * (2 * kW + kG) * 16 * Bwd::kBlock;
    static constexpr size_t kCols = 2 * sizeof(float) * EPT * Bwd::kBlock;   // at the end, in the ring's place
    static constexpr size_t kSmem = kRing > kCols ? kRing : kCols;
};

// Rows go to teams of TPR threads; the lanes of a warp (teams within one) and the warps of a block (teams of several) take
// the same number of turns. A team behind the last row works on that row again, and writes nothing.
template <class TX, class TY, Mode MODE, int TPR, int EPT>
__global__ void __launch_bounds__(Fwd<TX, TY, MODE, TPR, EPT>::kBlock, Fwd<TX, TY, MODE, TPR, EPT>::kBlocks)
k_norm_fwd(FwdArgs a) {
    using L = Fwd<TX, TY, MODE, TPR, EPT>;
    constexpr bool VEC = L::VEC;
    using P = Pack<TX, L::kVe>;
    constexpr int B = L::kBlock, S = L::kDepth, W = L::kW, E = L::kVe, NV = L::kNv;
    extern __shared__ uint4 ring[];   // [S][x, residual][W][B]
    __shared__ float red[2][B / 32];
    const int t = threadIdx.x % TPR, width = static_cast<int>(a.width);
    const float inv = 1.f / static_cast<float>(width);
    const long long step = static_cast<long long>(gridDim.x) * L::kRows;
    long long row = static_cast<long long>(blockIdx.x) * L::kRows + threadIdx.x / TPR;   // this team's
    long long first = row - (TPR < 32 ? (threadIdx.x & 31) / TPR : TPR == 32 ? 0 : threadIdx.x / TPR);
    auto fetch = [&](long long at_row, int slot) {   // one group of copies, empty behind the last row
        if constexpr (VEC) {
            if (at_row < a.rows) {
                const TX* px = static_cast<const TX*>(a.x) + at_row * a.x_stride;
                const TX* pr = static_cast<const TX*>(a.res) + at_row * a.r_stride;
                uint4* at = ring + slot * 2 * W * B + threadIdx.x;
#pragma unroll
                for (int v = 0; v < NV; ++v)
                    if (L::in(v, t, width)) {
                        copy_pack<TX, E, B>(at + v * (W / NV) * B, px + L::at(v, t));
                        if (a.res) copy_pack<TX, E, B>(at + (W + v * (W / NV)) * B, pr + L::at(v, t));
                    }
            }
            copies_commit();
        }
    };
    P next_x[VEC ? 1 : NV], next_r[VEC ? 1 : NV];
    auto load_next = [&](long long at_row) {   // value by value: the next row's loads are under way in registers
        if constexpr (!VEC) {
            const long long from = at_row < a.rows ? at_row : a.rows - 1;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                next_x[v] = P{};
                if (L::in(v, t, width)) next_x[v] = load_pack<TX, E>(static_cast<const TX*>(a.x) + from * a.x_stride + L::at(v, t));
            }
            if (a.res) {
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    next_r[v] = P{};
                    if (L::in(v, t, width)) next_r[v] = load_pack<TX, E>(static_cast<const TX*>(a.res) + from * a.r_stride + L::at(v, t));
                }
            }
        }
    };
#pragma unroll
    for (int q = 0; q < S; ++q) fetch(row + q * step, q);
    load_next(row);
    float w[EPT], b[EPT];   // behind the first rows' copies, which take as long
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        load_params<E>(w + v * E, a.weight, a.w_type, L::at(v, t), width, a.w_wide, 1.f);
        load_params<E>(b + v * E, a.bias, a.w_type, L::at(v, t), width, a.w_wide, 0.f);
    }
    for (int slot = 0; first < a.rows; first += step, row += step) {
        const bool live = row < a.rows;
        if constexpr (VEC) copies_wait<S - 1>();
        P x[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if constexpr (VEC) {
                x[v] = P{};
                if (L::in(v, t, width)) x[v] = slot_pack<TX, E, B>(ring + (slot * 2 * W + v * (W / NV)) * B + threadIdx.x);
            } else {
                x[v] = next_x[v];
            }
        }
        if (a.res) {
            P r[NV];
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if constexpr (VEC) {
                    r[v] = P{};
                    if (L::in(v, t, width)) r[v] = slot_pack<TX, E, B>(ring + (slot * 2 * W + W + v * (W / NV)) * B + threadIdx.x);
                } else {
                    r[v] = next_r[v];
                }
            }
            TX* ps = static_cast<TX*>(a.sum) + row * width;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float q[E];
#pragma unroll
                for (int i = 0; i < E; ++i) q[i] = to_f(x[v].v[i]) + to_f(r[v].v[i]);
                x[v] = rounded<TX, E>(q);
                if (live && L::in(v, t, width)) *reinterpret_cast<P*>(ps + L::at(v, t)) = x[v];
            }
        }
        if constexpr (VEC) {
            fetch(row + S * step, slot);
            slot = slot + 1 == S ? 0 : slot + 1;
        } else {
            load_next(row + step);
        }
        float s[EPT];
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < E; ++i) sum += s[v * E + i] = to_f(x[v].v[i]);
        const float mu = row_sum<TPR>(sum, red[0]) * inv;
        float sq = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (L::in(v, t, width)) {
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    s[v * E + i] -= mu;
                    sq = fmaf(s[v * E + i], s[v * E + i], sq);
                }
            }
        const float rs = rsqrtf(fmaf(row_sum<TPR>(sq, red[1]), inv, a.eps));
        if (!live) continue;
        TY* py = static_cast<TY*>(a.y) + row * width;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (L::in(v, t, width)) {
                float y[E];
#pragma unroll
                for (int i = 0; i < E; ++i) y[i] = fmaf(s[v * E + i] * rs, w[v * E + i], b[v * E + i]);
                store_pack<TY, E>(py + L::at(v, t), y);
            }
        if (a.stats && t == 0) a.stats[row] = make_float2(mu, rs);
    }
}

// Both gradients in one pass over gy and s: each thread also sums its columns' gy xh and gy over the rows that it sees, and
// the block writes their sums once, a.splits blocks in all. The row's values are read a second time, from shared memory (or
// L1), when their means are known, not kept in registers.
template <class TX, class TY, Mode MODE, int TPR, int EPT>
__global__ void __launch_bounds__(Bwd<TX, TY, MODE, TPR, EPT>::kBlock, Bwd<TX, TY, MODE, TPR, EPT>::kBlocks)
k_norm_bwd(BwdArgs a) {
    using L = Bwd<TX, TY, MODE, TPR, EPT>;
    constexpr bool VEC = L::VEC;
    using PX = Pack<TX, L::kVe>;
    using PY = Pack<TY, L::kVe>;
    constexpr int B = L::kBlock, S = L::kDepth, W = L::kW, G = L::kG, E = L::kVe, NV = L::kNv, R = 2 * W + G;
    extern __shared__ uint4 ring[];   // [S][s, gsum, gy][W, W, G][B]
    __shared__ float2 red[2][B / 32];
    int half = 0;
    const int t = threadIdx.x % TPR, width = static_cast<int>(a.width);
    const float inv = 1.f / static_cast<float>(width);
    const long long step = static_cast<long long>(gridDim.x) * L::kRows;
    long long row = static_cast<long long>(blockIdx.x) * L::kRows + threadIdx.x / TPR;
    long long first = row - (TPR < 32 ? (threadIdx.x & 31) / TPR : TPR == 32 ? 0 : threadIdx.x / TPR);
    auto fetch = [&](long long at_row, int slot) {
        if constexpr (VEC) {
            if (at_row < a.rows) {
                const TX* ps = static_cast<const TX*>(a.s) + at_row * a.s_stride;
                const TX* pq = static_cast<const TX*>(a.gsum) + at_row * a.gsum_stride;
                const TY* pg = static_cast<const TY*>(a.gy) + at_row * a.gy_stride;
                uint4* at = ring + slot * R * B + threadIdx.x;
#pragma unroll
                for (int v = 0; v < NV; ++v)
                    if (L::in(v, t, width)) {
                        copy_pack<TX, E, B>(at + v * (W / NV) * B, ps + L::at(v, t));
                        if (a.gsum) copy_pack<TX, E, B>(at + (W + v * (W / NV)) * B, pq + L::at(v, t));
                        copy_pack<TY, E, B>(at + (2 * W + v * (G / NV)) * B, pg + L::at(v, t));
                    }
            }
            copies_commit();
        }
    };
#pragma unroll
    for (int q = 0; q < S; ++q) fetch(row + q * step, q);
    float w[EPT], dw[EPT], db[EPT];
#pragma unroll
    for (int v = 0; v < NV; ++v) load_params<E>(w + v * E, a.weight, a.w_type, L::at(v, t), width, a.w_wide, 1.f);
#pragma unroll
    for (int e = 0; e < EPT; ++e) dw[e] = db[e] = 0.f;
    PX next_s[VEC ? 1 : NV];
    PY next_g[VEC ? 1 : NV];
    auto load_next = [&](long long at_row) {
        if constexpr (!VEC) {
            const long long from = at_row < a.rows ? at_row : a.rows - 1;
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (L::in(v, t, width)) {
                    next_s[v] = load_pack<TX, E>(static_cast<const TX*>(a.s) + from * a.s_stride + L::at(v, t));
                    next_g[v] = load_pack<TY, E>(static_cast<const TY*>(a.gy) + from * a.gy_stride + L::at(v, t));
                }
        }
    };
    load_next(row);
    float2 st = a.stats[row < a.rows ? row : a.rows - 1];
    for (int slot = 0; first < a.rows; first += step, row += step) {
        const bool live = row < a.rows;
        const uint4* at = ring + slot * R * B + threadIdx.x;
        PX now_s[VEC ? 1 : NV];
        PY now_g[VEC ? 1 : NV];
        if constexpr (VEC) {
            copies_wait<S - 1>();
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                now_s[v] = next_s[v];
                now_g[v] = next_g[v];
            }
            load_next(row + step);
        }
        auto value_s = [&](int v) -> PX {
            if constexpr (VEC) return slot_pack<TX, E, B>(at + v * (W / NV) * B);
            else return now_s[v];
        };
        auto value_g = [&](int v) -> PY {
            if constexpr (VEC) return slot_pack<TY, E, B>(at + (2 * W + v * (G / NV)) * B);
            else return now_g[v];
        };
        auto value_q = [&](int v) -> PX {
            if constexpr (VEC) return slot_pack<TX, E, B>(at + (W + v * (W / NV)) * B);
            else return load_pack<TX, E>(static_cast<const TX*>(a.gsum) + row * a.gsum_stride + L::at(v, t));
        };
        const float mu = st.x, rs = st.y;
        if (row + step < a.rows) st = a.stats[row + step];
        float th = 0.f, thx = 0.f;
        if (live) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (L::in(v, t, width)) {
                    const PX s = value_s(v);
                    const PY g = value_g(v);
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        const int e = v * E + i;
                        const float q = to_f(g.v[i]), xh = (to_f(s.v[i]) - mu) * rs, h = q * w[e];
                        dw[e] = fmaf(q, xh, dw[e]);
                        db[e] += q;
                        th += h;
                        thx = fmaf(h, xh, thx);
                    }
                }
        }
        const float2 sums = row_sums<TPR>(th, thx, red[half ^= 1]);
        const float mh = sums.x * inv, mhx = sums.y * inv;
        if (live && a.dx) {
            TX* pd = static_cast<TX*>(a.dx) + row * width;
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (L::in(v, t, width)) {
                    const PX s = value_s(v);
                    const PY g = value_g(v);
                    float d[E];
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        const float xh = (to_f(s.v[i]) - mu) * rs;
                        d[i] = fmaf(-xh, mhx, to_f(g.v[i]) * w[v * E + i] - mh) * rs;
                    }
                    if (a.gsum) {
                        const PX q = value_q(v);
#pragma unroll
                        for (int i = 0; i < E; ++i) d[i] += to_f(q.v[i]);
                    }
                    store_pack<TX, E>(pd + L::at(v, t), d);
                }
        }
        if constexpr (VEC) {
            fetch(row + S * step, slot);
            slot = slot + 1 == S ? 0 : slot + 1;
        }
    }
    if (!a.part) return;
    // the block's rows side by side: their column sums, in the order of the groups
    float* cols = reinterpret_cast<float*>(ring);   // [rows of the block][2][TPR * EPT]; no copy is under way any more
    if constexpr (VEC) copies_wait<0>();
    __syncthreads();
    float* mine = cols + threadIdx.x / TPR * 2 * TPR * EPT;
#pragma unroll
    for (int v = 0; v < L::kNv; ++v)
#pragma unroll
        for (int i = 0; i < E; ++i) {
            mine[L::at(v, t) + i] = dw[v * E + i];
            mine[TPR * EPT + L::at(v, t) + i] = db[v * E + i];
        }
    __syncthreads();
    float* part = a.part + static_cast<long long>(blockIdx.x) * 2 * width;
    for (int c = threadIdx.x; c < 2 * width; c += B) {
        const int at = c < width ? c : c - width + TPR * EPT;
        float sum = cols[at];
#pragma unroll
        for (int q = 1; q < L::kRows; ++q) sum += cols[q * 2 * TPR * EPT + at];
        part[c] = sum;
    }
}

// ------------------------------------------------------------------ wider rows: read again for each pass
//
// A block per row, N neighbouring values per thread and turn (16 bytes, or one where the rows are not aligned).

template <class TX, class TY, int N>
__global__ void __launch_bounds__(kWideThreads) k_norm_fwd_wide(FwdArgs a) {
    __shared__ float red[2][kWideThreads / 32];
    const float inv = 1.f / static_cast<float>(a.width);
    const int width = static_cast<int>(a.width), start = threadIdx.x * N;
    constexpr int kStep = kWideThreads * N;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const TX* x = static_cast<const TX*>(a.x) + row * a.x_stride;
        if (a.res) {
            const TX* r = static_cast<const TX*>(a.res) + row * a.r_stride;
            TX* s = static_cast<TX*>(a.sum) + row * a.width;
#pragma unroll 4
            for (int i = start; i < width; i += kStep) {
                const Pack<TX, N> p = load_pack<TX, N>(x + i), q = load_pack<TX, N>(r + i);
                float v[N];
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] = to_f(p.v[e]) + to_f(q.v[e]);
                store_pack<TX, N>(s + i, v);
            }
            x = s;   // each thread reads back only what it wrote itself
        }
        float t = 0.f;
#pragma unroll 4
        for (int i = start; i < width; i += kStep) {
            const Pack<TX, N> p = load_pack<TX, N>(x + i);
#pragma unroll
            for (int e = 0; e < N; ++e) t += to_f(p.v[e]);
        }
        const float mu = row_sum<kWideThreads>(t, red[0]) * inv;
        t = 0.f;
#pragma unroll 4
        for (int i = start; i < width; i += kStep) {
            const Pack<TX, N> p = load_pack<TX, N>(x + i);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float c = to_f(p.v[e]) - mu;
                t = fmaf(c, c, t);
            }
        }
        const float rs = rsqrtf(fmaf(row_sum<kWideThreads>(t, red[1]), inv, a.eps));
        TY* y = static_cast<TY*>(a.y) + row * a.width;
#pragma unroll 2
        for (int i = start; i < width; i += kStep) {
            const Pack<TX, N> p = load_pack<TX, N>(x + i);
            float w[N], b[N], v[N];
            load_params<N>(w, a.weight, a.w_type, i, width, a.w_wide, 1.f);
            load_params<N>(b, a.bias, a.w_type, i, width, a.w_wide, 0.f);
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = fmaf((to_f(p.v[e]) - mu) * rs, w[e], b[e]);
            store_pack<TY, N>(y + i, v);
        }
        if (a.stats && threadIdx.x == 0) a.stats[row] = make_float2(mu, rs);
    }
}

template <class TX, class TY, int N>
__global__ void __launch_bounds__(kWideThreads) k_norm_dx_wide(BwdArgs a) {
    __shared__ float2 red[2][kWideThreads / 32];
    int half = 0;
    const float inv = 1.f / static_cast<float>(a.width);
    const int width = static_cast<int>(a.width), start = threadIdx.x * N;
    constexpr int kStep = kWideThreads * N;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const TX* s = static_cast<const TX*>(a.s) + row * a.s_stride;
        const TY* g = static_cast<const TY*>(a.gy) + row * a.gy_stride;
        const float2 st = a.stats[row];
        float th = 0.f, thx = 0.f;
#pragma unroll 2
        for (int i = start; i < width; i += kStep) {
            const Pack<TX, N> p = load_pack<TX, N>(s + i);
            const Pack<TY, N> q = load_pack<TY, N>(g + i);
            float w[N];
            load_params<N>(w, a.weight, a.w_type, i, width, a.w_wide, 1.f);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float h = to_f(q.v[e]) * w[e];
                th += h;
                thx = fmaf(h, (to_f(p.v[e]) - st.x) * st.y, thx);
            }
        }
        const float2 sums = row_sums<kWideThreads>(th, thx, red[half ^= 1]);
        const float mh = sums.x * inv, mhx = sums.y * inv;
        TX* dx = static_cast<TX*>(a.dx) + row * a.width;
        const TX* gs = a.gsum ? static_cast<const TX*>(a.gsum) + row * a.gsum_stride : nullptr;
#pragma unroll 2
        for (int i = start; i < width; i += kStep) {
            const Pack<TX, N> p = load_pack<TX, N>(s + i);
            const Pack<TY, N> q = load_pack<TY, N>(g + i);
            float w[N], d[N];
            load_params<N>(w, a.weight, a.w_type, i, width, a.w_wide, 1.f);
#pragma unroll
            for (int e = 0; e < N; ++e)
                d[e] = fmaf(-(to_f(p.v[e]) - st.x) * st.y, mhx, to_f(q.v[e]) * w[e] - mh) * st.y;
            if (gs) {
                const Pack<TX, N> u = load_pack<TX, N>(gs + i);
#pragma unroll
                for (int e = 0; e < N; ++e) d[e] += to_f(u.v[e]);
            }
            store_pack<TX, N>(dx + i, d);
        }
    }
}

// Column sums of gy xh and gy over one split of the rows; a block takes 64 columns, 4 rows at a time.
template <class TX, class TY>
__global__ void __launch_bounds__(kThreads) k_norm_dw_wide(BwdArgs a) {
    __shared__ float red[2][kColRows][kCols];
    const int c = threadIdx.x % kCols, q = threadIdx.x / kCols;
    const long long col = static_cast<long long>(blockIdx.x) * kCols + c;
    float dw = 0.f, db = 0.f;
    if (col < a.width) {
        for (long long row = static_cast<long long>(blockIdx.y) * kColRows + q; row < a.rows;
             row += static_cast<long long>(a.splits) * kColRows) {
            const float2 st = a.stats[row];
            const float g = to_f(static_cast<const TY*>(a.gy)[row * a.gy_stride + col]);
            dw = fmaf(g, (to_f(static_cast<const TX*>(a.s)[row * a.s_stride + col]) - st.x) * st.y, dw);
            db += g;
        }
    }
    red[0][q][c] = dw;
    red[1][q][c] = db;
    __syncthreads();
    if (q == 0 && col < a.width) {
        for (int j = 1; j < kColRows; ++j) {
            dw += red[0][j][c];
            db += red[1][j][c];
        }
        a.part[(static_cast<long long>(blockIdx.y) * 2) * a.width + col] = dw;
        a.part[(static_cast<long long>(blockIdx.y) * 2 + 1) * a.width + col] = db;
    }
}

// The partial sums of 32 columns per block, 32 runs of them side by side and then in order: the result does not depend on
// which block ran when. (8 runs per block took 6.0 us for 296 partial sums of 512 columns, 32 take 3.3 us.)
__global__ void __launch_bounds__(1024) k_norm_dw_sum(BwdArgs a) {
    __shared__ float red[32][33];
    const int c = threadIdx.x & 31, q = threadIdx.x >> 5;
    const long long i = static_cast<long long>(blockIdx.x) * 32 + c;
    float t = 0.f;
    if (i < 2 * a.width) {
#pragma unroll 4
        for (int p = q; p < a.splits; p += 32) t += a.part[static_cast<long long>(p) * 2 * a.width + i];
    }
    red[q][c] = t;
    __syncthreads();
    t = warp_sum(red[c][q]);   // column q of the block
    const long long col = static_cast<long long>(blockIdx.x) * 32 + q;
    if (c == 0 && col < 2 * a.width) {
        void* out = col < a.width ? a.dweight : a.dbias;
        if (out) store_param(out, a.w_type, col < a.width ? col : col - a.width, t);
    }
}

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

// f(threads per row, values per thread) of the tile that holds a row of at most kMaxRow values, the smallest. few: 8 values per
// thread, for the backward of rows read value by value (262,144 x 1,001 bf16: 885 us with 16 read twice, 500 with 8 kept).
template <class F>
void with_tile(long long width, bool few, F f) {
    using std::integral_constant;
    if (width <= 64) f(integral_constant<int, 8>{}, integral_constant<int, 8>{});
    else if (width <= 128) f(integral_constant<int, 16>{}, integral_constant<int, 8>{});
    else if (width <= 256) f(integral_constant<int, 32>{}, integral_constant<int, 8>{});
    else if (width > 4096) f(integral_constant<int, 512>{}, integral_constant<int, 16>{});
    else if (few) {
        if (width <= 512) f(integral_constant<int, 64>{}, integral_constant<int, 8>{});
        else if (width <= 1024) f(integral_constant<int, 128>{}, integral_constant<int, 8>{});
        else if (width <= 2048) f(integral_constant<int, 256>{}, integral_constant<int, 8>{});
        else f(integral_constant<int, 512>{}, integral_constant<int, 8>{});
    } else if (width <= 512) f(integral_constant<int, 32>{}, integral_constant<int, 16>{});
    else if (width <= 1024) f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
    else if (width <= 2048) f(integral_constant<int, 128>{}, integral_constant<int, 16>{});
    else f(integral_constant<int, 256>{}, integral_constant<int, 16>{});
}

template <Mode MODE> using Of = std::integral_constant<Mode, MODE>;

long long ceil_of(long long a, long long b) { return (a + b - 1) / b; }

// Partial sums of the parameters' gradients: blocks of k_norm_bwd, or row splits of k_norm_dw_wide.
int splits_of(long long rows, long long width, bool vec) {
    long long n = 1, most = 1;
    if (width <= kMaxRow) {
        with_tile(width, !vec, [&](auto tpr, auto) {
            n = static_cast<long long>(kBwdWarps * 32 / block_of(tpr())) * sm_count();
            most = ceil_of(rows, block_of(tpr()) / tpr());
        });
    } else {
        n = ceil_of(8ll * sm_count(), ceil_of(width, kCols));
        most = ceil_of(rows, 16 * kColRows);
    }
    if (n > most) n = most;
    return static_cast<int>(n < 1 ? 1 : n);
}

unsigned blocks_of(long long groups, int per_sm) {
    const long long most = static_cast<long long>(per_sm) * sm_count();
    return static_cast<unsigned>(groups < most ? groups : most);
}

// Launches a kernel that may need more shared memory than the 48 KB it has unasked (asked for once per device).
template <auto KERNEL, class A>
cudaError_t launch(unsigned grid, int block, size_t smem, cudaStream_t stream, const A& a) {
    static std::atomic<bool> asked[kDevices];
    if (smem > 48 * 1024) {
        const int dev = current_device();
        if (dev < 0 || dev >= kDevices || !asked[dev].load(std::memory_order_acquire)) {
            const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
            if (e != cudaSuccess) return e;
            if (dev >= 0 && dev < kDevices) asked[dev].store(true, std::memory_order_release);
        }
    }
    KERNEL<<<grid, static_cast<unsigned>(block), smem, stream>>>(a);
    return cudaSuccess;
}

int failed(const char* msg) noexcept {
    try {
        g_norm_error = msg;
    } catch (...) {   // no memory for the message: the code alone
    }
    return 1;
}

// Whether a (non-null) pointer may hold values of a type.
bool fits(const void* p, int type) { return reinterpret_cast<uintptr_t>(p) % (type == 0 ? 4 : 2) == 0; }

bool aligned(const void* p, long long stride, int type) {
    const long long e = type == 0 ? 4 : 2;
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * e % 16 == 0;
}

// f(TX, TY) of the types of x and y: y has x's type or is fp32.
template <class F>
bool with_types(int x_type, int y_type, F f) {
    if (y_type != x_type && y_type != 0) return false;
    if (x_type == 0) f(float{}, float{});
    else if (x_type == 1 && y_type == 1) f(__nv_bfloat16{}, __nv_bfloat16{});
    else if (x_type == 1) f(__nv_bfloat16{}, float{});
    else if (x_type == 2 && y_type == 2) f(__half{}, __half{});
    else if (x_type == 2) f(__half{}, float{});
    else return false;
    return true;
}

const char* bad_shape(long long rows, long long width, int x_type, int y_type, int w_type) {
    if (rows < 0) return "rows must not be negative";
    if (width < 1 || width > (1ll << 30)) return "width must be 1 .. 2^30";
    if (x_type < 0 || x_type > 2 || w_type < 0 || w_type > 2) return "unknown type";
    if (y_type != x_type && y_type != 0) return "y must have x's type or be fp32";
    return nullptr;
}

}  // namespace

extern "C" {

const char* rl_norm_error(void) { return g_norm_error.c_str(); }

int rl_norm_fwd(const void* x, const void* residual, const void* weight, const void* bias, void* y, void* sum, void* stats,
                long long rows, long long width, long long x_stride, long long r_stride, int x_type, int y_type,
                int w_type, float eps, void* stream) {
    if (const char* e = bad_shape(rows, width, x_type, y_type, w_type)) return failed(e);
    if (rows == 0) return 0;
    if (!x || !y || (residual && !sum)) return failed("x, y and (with a residual) sum must be given");
    if (!fits(x, x_type) || !fits(residual, x_type) || !fits(y, y_type) || !fits(sum, x_type) || !fits(weight, w_type) ||
        !fits(bias, w_type) || reinterpret_cast<uintptr_t>(stats) % 8)
        return failed("misaligned pointer");
    FwdArgs a{x, residual, weight, bias, y, sum, static_cast<float2*>(stats), rows, width, x_stride, r_stride, w_type, aligned(weight, 0, w_type) && aligned(bias, 0, w_type), eps};
    auto s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    with_types(x_type, y_type, [&](auto tx, auto ty) {
        using TX = decltype(tx);
        using TY = decltype(ty);
        const bool vec = width * sizeof(TX) % 16 == 0 && aligned(x, x_stride, x_type) && aligned(residual, r_stride, x_type) &&
                         aligned(y, 0, y_type) && aligned(sum, 0, x_type);
        if (width > kMaxRow) {
            constexpr int kN = 16 / static_cast<int>(sizeof(TX));
            if (vec) k_norm_fwd_wide<TX, TY, kN><<<blocks_of(rows, 4), kWideThreads, 0, s>>>(a);
            else k_norm_fwd_wide<TX, TY, 1><<<blocks_of(rows, 4), kWideThreads, 0, s>>>(a);
            return;
        }
        with_tile(width, false, [&](auto tpr, auto ept) {
            auto run = [&](auto mode) {
                using K = Fwd<TX, TY, mode(), tpr(), ept()>;
                e = launch<k_norm_fwd<TX, TY, mode(), tpr(), ept()>>(blocks_of(ceil_of(rows, K::kRows), K::kBlocks), K::kBlock, K::kSmem, s, a);
            };
            if constexpr (ept() == 16 || tpr() <= 32) {
                if (vec && width == tpr() * ept()) run(Of<kFull>{});
                else if (vec) run(Of<kVectors>{});
                else run(Of<kOne>{});
            }
        });
    });
    if (e == cudaSuccess) e = cudaGetLastError();
    return e == cudaSuccess ? 0 : failed(cudaGetErrorString(e));
}

size_t rl_norm_bwd_work_bytes(long long rows, long long width) {
    if (rows < 1 || width < 1) return 0;
    const int one = splits_of(rows, width, false), wide = splits_of(rows, width, true);   // which one depends on the pointers
    return static_cast<size_t>(one > wide ? one : wide) * 2 * static_cast<size_t>(width) * sizeof(float);
}

int rl_norm_bwd(const void* gy, const void* gsum, const void* s, const void* stats, const void* weight, void* dx,
                void* dweight, void* dbias, long long rows, long long width, long long gy_stride, long long gsum_stride,
                long long s_stride, int x_type, int y_type, int w_type, void* work, size_t work_bytes, void* stream) {
    if (const char* e = bad_shape(rows, width, x_type, y_type, w_type)) return failed(e);
    if (rows < 1) return failed("rows must be positive");
    if (!gy || !s || !stats) return failed("gy, s and stats must be given");
    if (!fits(gy, y_type) || !fits(gsum, x_type) || !fits(s, x_type) || !fits(weight, w_type) || !fits(dx, x_type) ||
        !fits(dweight, w_type) || !fits(dbias, w_type) || !fits(work, 0) || reinterpret_cast<uintptr_t>(stats) % 8)
        return failed("misaligned pointer");
    const bool params = dweight || dbias;
    if (params && (!work || work_bytes < rl_norm_bwd_work_bytes(rows, width)))
        return failed("work space smaller than rl_norm_bwd_work_bytes()");
    BwdArgs a{gy, gsum, s, weight, static_cast<const float2*>(stats), dx, dweight, dbias,
              params ? static_cast<float*>(work) : nullptr, rows, width, gy_stride, gsum_stride, s_stride, w_type,
              aligned(weight, 0, w_type), splits_of(rows, width, true)};
    if (!dx && !params) return 0;
    auto q = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    with_types(x_type, y_type, [&](auto tx, auto ty) {
        using TX = decltype(tx);
        using TY = decltype(ty);
        const bool vec = width * sizeof(TX) % 16 == 0 && aligned(s, s_stride, x_type) && aligned(gy, gy_stride, y_type) &&
                         aligned(gsum, gsum_stride, x_type) && aligned(dx, 0, x_type);
        if (width > kMaxRow) {
            constexpr int kN = 16 / static_cast<int>(sizeof(TX));
            if (dx && vec) k_norm_dx_wide<TX, TY, kN><<<blocks_of(rows, 4), kWideThreads, 0, q>>>(a);
            else if (dx) k_norm_dx_wide<TX, TY, 1><<<blocks_of(rows, 4), kWideThreads, 0, q>>>(a);
            if (params) {
                const dim3 grid(static_cast<unsigned>((width + kCols - 1) / kCols), static_cast<unsigned>(a.splits));
                k_norm_dw_wide<TX, TY><<<grid, kThreads, 0, q>>>(a);
            }
            return;
        }
        a.splits = splits_of(rows, width, vec);
        with_tile(width, !vec, [&](auto tpr, auto ept) {
            auto run = [&](auto mode) {
                using K = Bwd<TX, TY, mode(), tpr(), ept()>;
                e = launch<k_norm_bwd<TX, TY, mode(), tpr(), ept()>>(static_cast<unsigned>(a.splits), K::kBlock, K::kSmem, q, a);
            };
            if constexpr (ept() == 16 || tpr() <= 32) {
                if (vec && width == tpr() * ept()) return run(Of<kFull>{});
                if (vec) return run(Of<kVectors>{});
            }
            if constexpr (ept() == 8 || tpr() == 512) run(Of<kOne>{});
        });
    });
    if (e == cudaSuccess && params) k_norm_dw_sum<<<static_cast<unsigned>((2 * width + 31) / 32), 1024, 0, q>>>(a);
    if (e == cudaSuccess) e = cudaGetLastError();
    return e == cudaSuccess ? 0 : failed(cudaGetErrorString(e));
}

}  // extern "C"
