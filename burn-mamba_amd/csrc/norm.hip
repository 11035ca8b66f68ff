// Layer norm over the last axis for gfx950, forward and backward (f32 or bf16
// rows, f32 statistics, weight, bias and their gradients).
//
//   xh = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = xh w + b
//   g = dy w:  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum_r dy xh,  db = sum_r dy
//
// The variance is the mean of the squared distances from the mean (a second
// sweep over the row), not a difference of two large sums.
#include <algorithm>

#include "pack.h"

namespace mamba {

struct LnParams {
    int64_t rows;
    int cols;
    float eps;
    const void* x; int64_t x_sr;
    const void* dy; int64_t dy_sr;
    const float* w; const float* b;
    void* out; int64_t out_sr;    // y, or dx (may be NULL)
    float* mean; float* rstd;     // written by the forward (may be NULL), read by the backward
    float* part; int parts;       // [parts][2][cols] partial sums of dw and db
    float* dw; float* db;
};

__device__ __forceinline__ float ln_block_sum(float v, float* red) {
    v = wave_sum_dpp(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = red[0];
    for (int i = 1; i < (int)(blockDim.x >> 6); ++i) s += red[i];
    return s;
}

// Any width: a workgroup per row, the row read once per sweep.
template <typename T>
__global__ __launch_bounds__(256) void ln_fwd_wide(LnParams p) {
    __shared__ float red[4];
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(p.x) + r * p.x_sr;
        T* y = static_cast<T*>(p.out) + r * p.out_sr;
        float s = 0.f;
        for (int c = threadIdx.x; c < p.cols; c += 256) s += load_f32<T>(x + c);
        const float mean = ln_block_sum(s, red) / (float)p.cols;
        s = 0.f;
        for (int c = threadIdx.x; c < p.cols; c += 256) {
            const float d = load_f32<T>(x + c) - mean;
            s += d * d;
        }
        const float rstd = 1.f / sqrtf(ln_block_sum(s, red) / (float)p.cols + p.eps);
        for (int c = threadIdx.x; c < p.cols; c += 256) {
            const float v = (load_f32<T>(x + c) - mean) * rstd;
            store_f32<T>(y + c, v * (p.w ? p.w[c] : 1.f) + (p.b ? p.b[c] : 0.f));
        }
        if (threadIdx.x == 0) {
            if (p.mean) p.mean[r] = mean;
            if (p.rstd) p.rstd[r] = rstd;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_dx_wide(LnParams p) {
    __shared__ float red[4];
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(p.x) + r * p.x_sr;
        const T* dy = static_cast<const T*>(p.dy) + r * p.dy_sr;
        T* dx = static_cast<T*>(p.out) + r * p.out_sr;
        const float mean = p.mean[r], rstd = p.rstd[r];
        float s1 = 0.f, s2 = 0.f;
        for (int c = threadIdx.x; c < p.cols; c += 256) {
            const float g = load_f32<T>(dy + c) * (p.w ? p.w[c] : 1.f);
            s1 += g;
            s2 += g * (load_f32<T>(x + c) - mean) * rstd;
        }
        s1 = ln_block_sum(s1, red) / (float)p.cols;
        s2 = ln_block_sum(s2, red) / (float)p.cols;
        for (int c = threadIdx.x; c < p.cols; c += 256) {
            const float g = load_f32<T>(dy + c) * (p.w ? p.w[c] : 1.f);
            store_f32<T>(dx + c, rstd * (g - s1 - (load_f32<T>(x + c) - mean) * rstd * s2));
        }
    }
}

// dw and db of 64 columns over one part of the rows: thread (c, q) takes every
// fourth row.
template <typename T>
__global__ __launch_bounds__(256) void ln_dw_wide(LnParams p) {
    __shared__ float red[2][4][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
    const int64_t per = (p.rows + p.parts - 1) / p.parts;
    const int64_t r0 = blockIdx.y * per, r1 = min(p.rows, r0 + per);
    float sw = 0.f, sb = 0.f;
    if (c < p.cols)
        for (int64_t r = r0 + q; r < r1; r += 4) {
            const float dy = load_f32<T>(static_cast<const T*>(p.dy) + r * p.dy_sr + c);
            sb += dy;
            sw += dy * (load_f32<T>(static_cast<const T*>(p.x) + r * p.x_sr + c) - p.mean[r]) * p.rstd[r];
        }
    red[0][q][threadIdx.x & 63] = sw;
    red[1][q][threadIdx.x & 63] = sb;
    __syncthreads();
    if (q < 2 && c < p.cols) {
        const int l = threadIdx.x & 63;
        p.part[((int64_t)blockIdx.y * 2 + q) * p.cols + c] = (red[q][0][l] + red[q][1][l]) + (red[q][2][l] + red[q][3][l]);
    }
}

// The parts in order of their number: the same sums every time.
__global__ __launch_bounds__(256) void ln_dw_join(LnParams p) {
    __shared__ float red[2][4][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
    float sw = 0.f, sb = 0.f;
    if (c < p.cols)
        for (int i = q; i < p.parts; i += 4) {
            sw += p.part[(int64_t)(2 * i) * p.cols + c];
            sb += p.part[(int64_t)(2 * i + 1) * p.cols + c];
        }
    red[0][q][threadIdx.x & 63] = sw;
    red[1][q][threadIdx.x & 63] = sb;
    __syncthreads();
    if (q < 2 && c < p.cols) {
        const int l = threadIdx.x & 63;
        float* out = q ? p.db : p.dw;
        if (out) out[c] = (red[q][0][l] + red[q][1][l]) + (red[q][2][l] + red[q][3][l]);
    }
}

// workgroups of a kernel that takes a row each in turn
static uint32_t ln_grid(int64_t rows) { return (uint32_t)std::min<int64_t>(rows, 1 << 20); }
static int ln_parts(int64_t rows) { return (int)std::min<int64_t>(256, (rows + 31) / 32); }

// rows x cols with these row strides: rows overlap nowhere and every element
// offset fits 63 bits
static bool ln_rows_ok(int64_t rows, int cols, int64_t sr) {
    return sr >= cols || rows <= 1;
}

template <typename T>
static void ln_fwd_launch(const LnParams& p, hipStream_t s) {
    hipLaunchKernelGGL(ln_fwd_wide<T>, dim3(ln_grid(p.rows)), dim3(256), 0, s, p);
}

template <typename T>
static void ln_bwd_launch(const LnParams& p, hipStream_t s) {
    if (p.out) hipLaunchKernelGGL(ln_dx_wide<T>, dim3(ln_grid(p.rows)), dim3(256), 0, s, p);
    if (!p.dw && !p.db) return;
    hipLaunchKernelGGL(ln_dw_wide<T>, dim3(ceil_div(p.cols, 64), p.parts), dim3(256), 0, s, p);
    hipLaunchKernelGGL(ln_dw_join, dim3(ceil_div(p.cols, 64)), dim3(256), 0, s, p);
}

}  // namespace mamba

using namespace mamba;

extern "C" int mamba_layernorm_fwd(const mamba_layernorm_args* a, mamba_stream_t stream) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    MAMBA_CHECK_ARG(a->rows >= 0 && a->rows < (1ll << 31), "rows must be in [0, 2^31)");
    MAMBA_CHECK_ARG(a->cols >= 1, "cols must be >= 1");
    MAMBA_CHECK_ARG(a->io_dtype == MAMBA_F32 || a->io_dtype == MAMBA_BF16, "io_dtype must be f32 or bf16");
    MAMBA_CHECK_ARG(a->eps >= 0.f, "eps must be >= 0");
    if (a->rows == 0) return MAMBA_OK;
    MAMBA_CHECK_ARG(a->x && a->y, "x and y are required");
    MAMBA_CHECK_ARG(ln_rows_ok(a->rows, a->cols, a->y_sr), "rows of y overlap");
    LnParams p{};
    p.rows = a->rows; p.cols = a->cols; p.eps = a->eps;
    p.x = a->x; p.x_sr = a->x_sr; p.w = a->weight; p.b = a->bias;
    p.out = a->y; p.out_sr = a->y_sr; p.mean = a->mean; p.rstd = a->rstd;
    if (a->io_dtype == MAMBA_BF16) ln_fwd_launch<bf16_t>(p, (hipStream_t)stream);
    else ln_fwd_launch<float>(p, (hipStream_t)stream);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}

static int ln_bwd_check(const mamba_layernorm_bwd_args* a) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    MAMBA_CHECK_ARG(a->rows >= 0 && a->rows < (1ll << 31), "rows must be in [0, 2^31)");
    MAMBA_CHECK_ARG(a->cols >= 1, "cols must be >= 1");
    MAMBA_CHECK_ARG(a->io_dtype == MAMBA_F32 || a->io_dtype == MAMBA_BF16, "io_dtype must be f32 or bf16");
    return MAMBA_OK;
}

extern "C" size_t mamba_layernorm_bwd_workspace_size(const mamba_layernorm_bwd_args* a) {
    if (ln_bwd_check(a) != MAMBA_OK || (!a->dweight && !a->dbias)) return 0;
    return (size_t)ln_parts(a->rows) * 2 * a->cols * 4;
}

extern "C" int mamba_layernorm_bwd(const mamba_layernorm_bwd_args* a, void* ws, size_t ws_bytes, mamba_stream_t stream) {
    int st = ln_bwd_check(a);
    if (st != MAMBA_OK) return st;
    const size_t need = mamba_layernorm_bwd_workspace_size(a);
    MAMBA_CHECK_ARG(a->rows == 0 || (a->x && a->dy && a->mean && a->rstd), "x, dy, mean and rstd are required");
    MAMBA_CHECK_ARG(!a->dx || ln_rows_ok(a->rows, a->cols, a->dx_sr), "rows of dx overlap");
    if (need && (ws == nullptr || ws_bytes < need)) {
        set_error("mamba_layernorm_bwd: workspace missing or too small");
        return MAMBA_ERR_WORKSPACE;
    }
    LnParams p{};
    p.rows = a->rows; p.cols = a->cols;
    p.x = a->x; p.x_sr = a->x_sr; p.dy = a->dy; p.dy_sr = a->dy_sr; p.w = a->weight;
    p.out = a->rows ? a->dx : nullptr; p.out_sr = a->dx_sr;
    p.mean = const_cast<float*>(a->mean); p.rstd = const_cast<float*>(a->rstd);
    p.part = static_cast<float*>(ws); p.parts = ln_parts(a->rows);
    p.dw = a->dweight; p.db = a->dbias;
    if (a->rows == 0) {  // the sums of no rows: zeros
        if (p.dw || p.db) hipLaunchKernelGGL(ln_dw_join, dim3(ceil_div(p.cols, 64)), dim3(256), 0, (hipStream_t)stream, p);
    } else if (a->io_dtype == MAMBA_BF16) {
        ln_bwd_launch<bf16_t>(p, (hipStream_t)stream);
    } else {
        ln_bwd_launch<float>(p, (hipStream_t)stream);
    }
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}
