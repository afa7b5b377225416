// Layer norm of the policy's blocks (rl/model.py:64-72 SimBa: x + mlp(norm(x))), with the residual sum before it and its
// gradients. A row s of D values (s = x, or x + residual rounded to x's type: the stream that is kept is the one that
// is normalised):
//   mu = sum s / D, v = sum (s - mu)^2 / D, r = 1 / sqrt(v + eps), xh = (s - mu) r, y = xh w + b
//   h = gy w, dx = r (h - mean(h) - xh mean(h xh)) + gsum, dw = sum over rows of gy xh, db = sum over rows of gy
// All of it in fp32 from the inputs' types, rounded once into the outputs'. The variance is summed from the centred
// values (a second pass), so that a large mean costs no digits.
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <string>
#include "../../include/rlenv_api.h"   // rl_norm_* compiled against their C-ABI declarations

namespace {

constexpr int kWideThreads = 256;
constexpr int kColThreads = 256, kCols = 64, kColRows = kColThreads / kCols;

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
    float eps;
};

struct BwdArgs {
    const void *gy, *gsum, *s, *weight;
    const float2* stats;
    void *dx, *dweight, *dbias;
    float* part;     // [splits][2][width]
    long long rows, width, gy_stride, gsum_stride, s_stride;
    int w_type;
    int splits;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

// The sum of v over the block's threads, in every thread.
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.f;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) t += red[w];
    return t;
}

// A row per block at a time, any width; the row is read again (from L1 or L2) for each pass.
template <class TX, class TY>
__global__ void __launch_bounds__(kWideThreads) k_norm_fwd_wide(FwdArgs a) {
    __shared__ float red[kWideThreads / 32];
    const float inv = 1.f / static_cast<float>(a.width);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const TX* x = static_cast<const TX*>(a.x) + row * a.x_stride;
        if (a.res) {
            const TX* r = static_cast<const TX*>(a.res) + row * a.r_stride;
            TX* s = static_cast<TX*>(a.sum) + row * a.width;
            for (long long i = threadIdx.x; i < a.width; i += blockDim.x) s[i] = from_f<TX>(to_f(x[i]) + to_f(r[i]));
            x = s;   // each thread reads back only what it wrote itself
        }
        float t = 0.f;
        for (long long i = threadIdx.x; i < a.width; i += blockDim.x) t += to_f(x[i]);
        const float mu = block_sum(t, red) * inv;
        t = 0.f;
        for (long long i = threadIdx.x; i < a.width; i += blockDim.x) {
            const float c = to_f(x[i]) - mu;
            t = fmaf(c, c, t);
        }
        const float rs = rsqrtf(fmaf(block_sum(t, red), inv, a.eps));
        TY* y = static_cast<TY*>(a.y) + row * a.width;
        for (long long i = threadIdx.x; i < a.width; i += blockDim.x) {
            const float w = a.weight ? load_param(a.weight, a.w_type, i) : 1.f;
            const float b = a.bias ? load_param(a.bias, a.w_type, i) : 0.f;
            y[i] = from_f<TY>(fmaf((to_f(x[i]) - mu) * rs, w, b));
        }
        if (a.stats && threadIdx.x == 0) a.stats[row] = make_float2(mu, rs);
    }
}

template <class TX, class TY>
__global__ void __launch_bounds__(kWideThreads) k_norm_dx_wide(BwdArgs a) {
    __shared__ float red[kWideThreads / 32];
    const float inv = 1.f / static_cast<float>(a.width);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const TX* s = static_cast<const TX*>(a.s) + row * a.s_stride;
        const TY* g = static_cast<const TY*>(a.gy) + row * a.gy_stride;
        const float2 st = a.stats[row];
        float th = 0.f, thx = 0.f;
        for (long long i = threadIdx.x; i < a.width; i += blockDim.x) {
            const float h = to_f(g[i]) * (a.weight ? load_param(a.weight, a.w_type, i) : 1.f);
            th += h;
            thx = fmaf(h, (to_f(s[i]) - st.x) * st.y, thx);
        }
        const float mh = block_sum(th, red) * inv, mhx = block_sum(thx, red) * inv;
        TX* dx = static_cast<TX*>(a.dx) + row * a.width;
        const TX* gs = a.gsum ? static_cast<const TX*>(a.gsum) + row * a.gsum_stride : nullptr;
        for (long long i = threadIdx.x; i < a.width; i += blockDim.x) {
            const float h = to_f(g[i]) * (a.weight ? load_param(a.weight, a.w_type, i) : 1.f);
            const float xh = (to_f(s[i]) - st.x) * st.y;
            const float d = (h - mh - xh * mhx) * st.y;
            dx[i] = from_f<TX>(gs ? d + to_f(gs[i]) : d);
        }
    }
}

// Column sums of gy xh and gy over one split of the rows; a block takes 64 columns, 4 rows at a time.
template <class TX, class TY>
__global__ void __launch_bounds__(kColThreads) k_norm_dw_wide(BwdArgs a) {
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

// The splits' partial sums in their order: the result does not depend on which block ran when.
__global__ void __launch_bounds__(256) k_norm_dw_sum(BwdArgs a) {
    const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= 2 * a.width) return;
    float t = 0.f;
    for (int p = 0; p < a.splits; ++p) t += a.part[static_cast<long long>(p) * 2 * a.width + i];
    const long long col = i < a.width ? i : i - a.width;
    void* out = i < a.width ? a.dweight : a.dbias;
    if (out) store_param(out, a.w_type, col, t);
}

int sm_count() {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

int splits_of(long long rows, long long width) {
    const long long blocks = (width + kCols - 1) / kCols;
    long long n = (8ll * sm_count() + blocks - 1) / blocks;
    const long long most = (rows + 16 * kColRows - 1) / (16 * kColRows);
    if (n > most) n = most;
    return static_cast<int>(n < 1 ? 1 : n);
}

unsigned wide_grid(long long rows) {
    const long long most = 8ll * sm_count();
    return static_cast<unsigned>(rows < most ? rows : most);
}

int failed(const char* msg) {
    g_norm_error = msg;
    return 1;
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
    if (width < 1 || width >= (1ll << 31)) return "width must be 1 .. 2^31 - 1";
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
    FwdArgs a{x, residual, weight, bias, y, sum, static_cast<float2*>(stats), rows, width, x_stride, r_stride, w_type, eps};
    auto s = static_cast<cudaStream_t>(stream);
    with_types(x_type, y_type, [&](auto tx, auto ty) {
        k_norm_fwd_wide<decltype(tx), decltype(ty)><<<wide_grid(rows), kWideThreads, 0, s>>>(a);
    });
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : failed(cudaGetErrorString(e));
}

size_t rl_norm_bwd_work_bytes(long long rows, long long width) {
    if (rows < 1 || width < 1) return 0;
    return static_cast<size_t>(splits_of(rows, width)) * 2 * static_cast<size_t>(width) * sizeof(float);
}

int rl_norm_bwd(const void* gy, const void* gsum, const void* s, const void* stats, const void* weight, void* dx,
                void* dweight, void* dbias, long long rows, long long width, long long gy_stride, long long gsum_stride,
                long long s_stride, int x_type, int y_type, int w_type, void* work, size_t work_bytes, void* stream) {
    if (const char* e = bad_shape(rows, width, x_type, y_type, w_type)) return failed(e);
    if (rows < 1) return failed("rows must be positive");
    if (!gy || !s || !stats) return failed("gy, s and stats must be given");
    const bool params = dweight || dbias;
    if (params && (!work || work_bytes < rl_norm_bwd_work_bytes(rows, width)))
        return failed("work space smaller than rl_norm_bwd_work_bytes()");
    BwdArgs a{gy, gsum, s, weight, static_cast<const float2*>(stats), dx, dweight, dbias, static_cast<float*>(work),
              rows, width, gy_stride, gsum_stride, s_stride, w_type, params ? splits_of(rows, width) : 0};
    auto q = static_cast<cudaStream_t>(stream);
    with_types(x_type, y_type, [&](auto tx, auto ty) {
        using TX = decltype(tx);
        using TY = decltype(ty);
        if (dx) k_norm_dx_wide<TX, TY><<<wide_grid(rows), kWideThreads, 0, q>>>(a);
        if (params) {
            const dim3 grid(static_cast<unsigned>((width + kCols - 1) / kCols), static_cast<unsigned>(a.splits));
            k_norm_dw_wide<TX, TY><<<grid, kColThreads, 0, q>>>(a);
        }
    });
    if (params) k_norm_dw_sum<<<static_cast<unsigned>((2 * width + 255) / 256), 256, 0, q>>>(a);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : failed(cudaGetErrorString(e));
}

}  // extern "C"
