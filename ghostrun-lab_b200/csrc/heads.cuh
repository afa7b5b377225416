// What the ordered heads (heads.cu) and the rows of any width (sample.cu) share: the definition of a draw, and the host side's
// helpers.
//
// Sampling of a row l with legal choices A: m = max over A, d = (l - m) / T, W = round(exp(d) 2^27), a whole number of 28
// bits. Choices are ranked by l, equal ones by their index; the first k stay, of those the shortest run from the top whose W
// sum reaches p of theirs, of those the ones with W >= min_p 2^27. With u in [0, 1) as 24 bits, the choice is the first that
// stayed, in index order, whose running sum of W exceeds floor(u total), and its log-probability (of the distribution that
// was drawn from) d - log(total 2^-27). Whole numbers make every sum the same in any order, so a result depends on no tile,
// lane or launch shape; 2^-27 of the best choice is finer than u's own 2^-24. exp is CUDA's own expf, so that the same W
// come from any fp32 program that calls it.
#pragma once
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>
#include "../../include/rlenv_api.h"   // rl_sample, rl_moves_* compiled against their C-ABI declarations

namespace heads {

constexpr int kBytes = 19, kMoves = 324;   // mask bytes of a move's five parts, and packed moves
constexpr float kScale = 134217728.f;      // 2^27
constexpr float kUnit = 1.f / kScale;
constexpr int kDevices = 64;               // whose properties are kept

inline thread_local std::string g_error;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// The sampling parameters: one number for all rows, or (pointer not null) one for each.
struct Cut {
    float temperature, top_p, min_p;
    int top_k;
    const float *temperatures, *top_ps, *min_ps;
    const int* top_ks;
};

struct RowCut {
    float scale;      // 1 / T
    float top_p;
    unsigned least;   // min_p 2^27: the least weight that stays
    int top_k;        // 0: all
    bool cut;         // whether any of the three takes something off
};

__device__ __forceinline__ RowCut row_cut(const Cut& c, long long row) {
    RowCut r;
    const float t = c.temperatures ? c.temperatures[row] : c.temperature;
    r.top_p = c.top_ps ? c.top_ps[row] : c.top_p;
    const float min_p = c.min_ps ? c.min_ps[row] : c.min_p;
    r.top_k = c.top_ks ? c.top_ks[row] : c.top_k;
    r.top_p = r.top_p < 1.f ? fmaxf(r.top_p, 0.f) : 1.f;   // a NaN takes nothing off
    r.least = min_p > 0.f ? static_cast<unsigned>(ceil(static_cast<double>(fminf(min_p, 1.f)) * static_cast<double>(kScale))) : 0u;
    if (r.top_k < 0) r.top_k = 0;
    r.scale = __fdiv_rn(1.f, t);
    if (!(t > 0.f) || r.scale == INFINITY) {   // 0 (or nothing a temperature can be): the best choice alone
        r.top_k = 1;
        r.scale = 1.f;
    }
    r.cut = r.top_k > 0 || r.top_p < 1.f || r.least > 0;
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

// ------------------------------------------------------------------ host side

inline int current_device() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess ? dev : -1;
}

// The current device's SM count, asked once per device.
inline int sm_count() {
    static std::atomic<int> known[kDevices];
    const int dev = current_device();
    const bool kept = dev >= 0 && dev < kDevices;
    int sms = kept ? known[dev].load(std::memory_order_relaxed) : 0;
    if (sms > 0) return sms;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 1) return 148;
    if (kept) known[dev].store(sms, std::memory_order_relaxed);
    return sms;
}

inline unsigned blocks_for(long long rows, long long per_block, long long most) {
    const long long n = (rows + per_block - 1) / per_block;
    return static_cast<unsigned>(n < most ? n : most);
}

inline int failed(const char* msg) noexcept {
    try {
        g_error = msg;
    } catch (...) {   // no memory for the message: the code alone
    }
    return 1;
}

// Whether a (non-null) pointer may hold values of `bytes` each.
inline bool fits(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline size_t size_of(int type) { return type == 0 ? 4 : 2; }

template <class F>
bool with_type(int type, F f) {
    if (type == 0) f(float{});
    else if (type == 1) f(__nv_bfloat16{});
    else if (type == 2) f(__half{});
    else return false;
    return true;
}

inline const char* bad_cut(float temperature, const void* temperatures, float top_p, const void* top_ps, float min_p,
                    const void* min_ps, const void* top_ks) {
    if (!temperatures && !(temperature >= 0.f)) return "temperature must be 0 or more";
    if (!top_ps && !(top_p >= 0.f)) return "top_p must be 0 or more";
    if (!min_ps && !(min_p <= 1.f)) return "min_p must be at most 1";
    if (!fits(temperatures, 4) || !fits(top_ks, 4) || !fits(top_ps, 4) || !fits(min_ps, 4)) return "misaligned parameters";
    return nullptr;
}

}  // namespace heads
