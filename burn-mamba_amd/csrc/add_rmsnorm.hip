// RMS norm with the residual's addition for gfx950: forward (rows of f32 or bf16, or of
// 8 bits with a scale each), backward.
//
//   s = residual + x,  rstd = 1 / sqrt(mean(s^2) + eps),  y = s rstd w
//   8 bits: scale = max |y| / top, q = round(y / scale), top = 127 (int8) or 448 (e4m3)
//   g = dy w,  xh = s rstd:  d = ds + rstd (g - xh mean(g xh)),  dw = sum_r dy xh
//
// The sum is normalised as it is in f32, before it is rounded to the stream's type: y
// then has one rounding.  The backward reads the stored s.
#include <algorithm>

#include "pack.h"

namespace mamba {

struct ArnP {
    int64_t rows;
    int cols;
    float eps;
    const void* x; int64_t x_sr;
    const void* res; int64_t res_sr;
    const float* w;
    void* s; int64_t s_sr;        // forward: written (may be NULL); backward: read
    void* y; int64_t y_sr;        // y, or dx
    float* rstd;
    uint8_t* q; int64_t q_sr; float* scale; bool e4m3;
    // backward
    const void* dy; int64_t dy_sr;
    const void* ds; int64_t ds_sr;
    void* dres; int64_t dres_sr;
    float* part; int parts;       // [parts][cols] partial sums of dw
    float* dw;
};

__device__ __forceinline__ float arn_block_sum(float v, float* red) {
    v = wave_sum_dpp(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}
// the largest of the values' bits without their sign: a NaN is above infinity, which is above
// every number
__device__ __forceinline__ uint32_t arn_block_max(uint32_t v, uint32_t* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return max(max(red[0], red[1]), max(red[2], red[3]));
}

// The scale of a row whose largest |y| has these bits, and what y is multiplied by (0: a row
// of zeros).  From 2^-100 on, 1 / scale is a number.
struct ArnScale { float scale, inv; };
__device__ __forceinline__ ArnScale arn_scale(uint32_t amax, bool e4m3) {
    const float top = e4m3 ? 448.f : 127.f;
    if (amax >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.f};
    if (amax < 0x0d800000u) return {0.f, 0.f};
    const float s = __uint_as_float(amax) / top;
    return {s, 1.f / s};
}
__device__ __forceinline__ uint8_t arn_q8(float v, ArnScale s, bool e4m3) {
    if (s.inv == 0.f) return 0;
    const float t = v * s.inv;
    if (e4m3) return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(fminf(fmaxf(t, -448.f), 448.f), 0.f, 0, false);
    return (uint8_t)(int8_t)(int)rintf(fminf(fmaxf(t, -127.f), 127.f));
}

// Any width: a workgroup per row, the row read once per sweep.
template <typename T, typename S>
__global__ __launch_bounds__(256) void arn_fwd_wide(ArnP p) {
    constexpr int E = 4, ST = 256 * E;
    __shared__ float red[4];
    __shared__ uint32_t redu[4];
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(p.x) + r * p.x_sr;
        const S* res = p.res ? static_cast<const S*>(p.res) + r * p.res_sr : nullptr;
        float v[E], b[E], w[E];
        auto sum = [&](int c) __attribute__((always_inline)) {
            ld_run<E, T>(x + c, p.cols - c, v);
            if (res) {
                ld_run<E, S>(res + c, p.cols - c, b);
#pragma unroll
                for (int i = 0; i < E; ++i) v[i] += b[i];
            }
        };
        auto weigh = [&](int c, float rstd) __attribute__((always_inline)) {
            if (p.w) ld_run<E, float>(p.w + c, p.cols - c, w);
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = p.w ? v[i] * rstd * w[i] : v[i] * rstd;
        };
        float ss = 0.f;
        for (int c = threadIdx.x * E; c < p.cols; c += ST) {
            sum(c);
#pragma unroll
            for (int i = 0; i < E; ++i) ss = __builtin_fmaf(v[i], v[i], ss);
        }
        const float rstd = 1.f / sqrtf(arn_block_sum(ss, red) / (float)p.cols + p.eps);
        if (threadIdx.x == 0 && p.rstd) p.rstd[r] = rstd;
        ArnScale sc{};
        if (p.q) {
            uint32_t amax = 0;
            for (int c = threadIdx.x * E; c < p.cols; c += ST) {
                sum(c);
                weigh(c, rstd);
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (c + i < p.cols) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
            }
            sc = arn_scale(arn_block_max(amax, redu), p.e4m3);
            if (threadIdx.x == 0) p.scale[r] = sc.scale;
        }
        for (int c = threadIdx.x * E; c < p.cols; c += ST) {
            sum(c);
            if (p.s) st_run<E, S>(static_cast<S*>(p.s) + r * p.s_sr + c, p.cols - c, v);
            weigh(c, rstd);
            if (p.q) {
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (c + i < p.cols) p.q[r * p.q_sr + c + i] = arn_q8(v[i], sc, p.e4m3);
            } else {
                st_run<E, T>(static_cast<T*>(p.y) + r * p.y_sr + c, p.cols - c, v);
            }
        }
    }
}

template <typename T, typename S>
__global__ __launch_bounds__(256) void arn_dx_wide(ArnP p) {
    constexpr int E = 4, ST = 256 * E;
    __shared__ float red[4];
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const S* s = static_cast<const S*>(p.s) + r * p.s_sr;
        const T* dy = static_cast<const T*>(p.dy) + r * p.dy_sr;
        const float rstd = p.rstd[r];
        float v[E], g[E], w[E];
        auto load = [&](int c) __attribute__((always_inline)) {
            ld_run<E, S>(s + c, p.cols - c, v);
            ld_run<E, T>(dy + c, p.cols - c, g);
            if (p.w) ld_run<E, float>(p.w + c, p.cols - c, w);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                v[i] *= rstd;
                if (p.w) g[i] *= w[i];
            }
        };
        float dot = 0.f;
        for (int c = threadIdx.x * E; c < p.cols; c += ST) {
            load(c);
#pragma unroll
            for (int i = 0; i < E; ++i) dot = __builtin_fmaf(g[i], v[i], dot);
        }
        dot = arn_block_sum(dot, red) / (float)p.cols;
        for (int c = threadIdx.x * E; c < p.cols; c += ST) {
            load(c);
            float d[E];
            if (p.ds) ld_run<E, S>(static_cast<const S*>(p.ds) + r * p.ds_sr + c, p.cols - c, d);
#pragma unroll
            for (int i = 0; i < E; ++i) d[i] = __builtin_fmaf(rstd, __builtin_fmaf(-v[i], dot, g[i]), p.ds ? d[i] : 0.f);
            if (p.y) st_run<E, T>(static_cast<T*>(p.y) + r * p.y_sr + c, p.cols - c, d);
            if (p.dres) st_run<E, S>(static_cast<S*>(p.dres) + r * p.dres_sr + c, p.cols - c, d);
        }
    }
}

// dw of 64 runs of columns over one part of the rows: thread (run, q) takes every fourth row.
template <typename T, typename S>
__global__ __launch_bounds__(256) void arn_dw_wide(ArnP p) {
    constexpr int E = 4;
    __shared__ float red[4][E][64];
    const int l = threadIdx.x & 63, c = (blockIdx.x * 64 + l) * E, q = threadIdx.x >> 6;
    const int64_t per = (p.rows + p.parts - 1) / p.parts;
    const int64_t r0 = blockIdx.y * per, r1 = min(p.rows, r0 + per);
    float sw[E] = {0.f, 0.f, 0.f, 0.f};
    if (c < p.cols)
        for (int64_t r = r0 + q; r < r1; r += 4) {
            float v[E], g[E];
            ld_run<E, S>(static_cast<const S*>(p.s) + r * p.s_sr + c, p.cols - c, v);
            ld_run<E, T>(static_cast<const T*>(p.dy) + r * p.dy_sr + c, p.cols - c, g);
            const float rstd = p.rstd[r];
#pragma unroll
            for (int i = 0; i < E; ++i) sw[i] = __builtin_fmaf(g[i], v[i] * rstd, sw[i]);
        }
#pragma unroll
    for (int i = 0; i < E; ++i) red[q][i][l] = sw[i];
    __syncthreads();
    if (q == 0) {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (c + i < p.cols)
                p.part[(int64_t)blockIdx.y * p.cols + c + i] = (red[0][i][l] + red[1][i][l]) + (red[2][i][l] + red[3][i][l]);
    }
}

// The parts in order of their number: the same sums every time.  16 threads a column,
// four loads in flight each; 16 columns a workgroup and turn.
__global__ __launch_bounds__(256) void arn_dw_join(ArnP p) {
    __shared__ float red[16][17];
    const int x = threadIdx.x & 15, q = threadIdx.x >> 4;
    for (int c0 = blockIdx.x * 16; c0 < p.cols; c0 += gridDim.x * 16) {
        const int c = c0 + x;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        if (c < p.cols) {
            const float* src = p.part + c;
            int i = q;
            for (; i + 48 < p.parts; i += 64) {
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] += src[(int64_t)(i + 16 * j) * p.cols];
            }
            for (; i < p.parts; i += 16) s[0] += src[(int64_t)i * p.cols];
        }
        red[q][x] = (s[0] + s[1]) + (s[2] + s[3]);
        __syncthreads();
        if (q == 0 && c < p.cols) {
            float a = 0.f;
            for (int j = 0; j < 16; ++j) a += red[j][x];
            p.dw[c] = a;
        }
        __syncthreads();
    }
}

static uint32_t arn_grid(int64_t rows) { return (uint32_t)std::min<int64_t>(rows, 1 << 20); }
static int arn_parts(int64_t rows) { return (int)std::min<int64_t>(256, (rows + 31) / 32); }

template <typename T, typename S>
static void arn_fwd_launch(const ArnP& p, hipStream_t s) {
    hipLaunchKernelGGL((arn_fwd_wide<T, S>), dim3(arn_grid(p.rows)), dim3(256), 0, s, p);
}
template <typename T, typename S>
static void arn_bwd_launch(const ArnP& p, hipStream_t s) {
    if (p.rows && (p.y || p.dres)) hipLaunchKernelGGL((arn_dx_wide<T, S>), dim3(arn_grid(p.rows)), dim3(256), 0, s, p);
    if (p.rows && p.dw) hipLaunchKernelGGL((arn_dw_wide<T, S>), dim3(ceil_div(p.cols, 256), p.parts), dim3(256), 0, s, p);
    if (p.dw) hipLaunchKernelGGL(arn_dw_join, dim3((uint32_t)std::min(ceil_div(p.cols, 16), 1 << 20)), dim3(256), 0, s, p);
}

}  // namespace mamba

using namespace mamba;

#define ARN_DISPATCH(fn, io, stream_type, ...)                                       \
    do {                                                                             \
        if ((io) == MAMBA_F32) fn<float, float>(__VA_ARGS__);                        \
        else if ((stream_type) == MAMBA_F32) fn<bf16_t, float>(__VA_ARGS__);         \
        else fn<bf16_t, bf16_t>(__VA_ARGS__);                                        \
    } while (0)

// a and b of e and f bytes an element share no memory; where e = f and same, b may be a itself
static bool arn_clash(const void* a, int64_t a_sr, int e, const void* b, int64_t b_sr, int f, int64_t rows, int cols, bool same) {
    if (e == f) return rows_clash(a, a_sr, b, b_sr, cols, cols, rows, e, same);
    if (a == nullptr || b == nullptr || rows <= 0) return false;
    const char *pa = static_cast<const char*>(a), *pb = static_cast<const char*>(b);
    return !(pa + ((rows - 1) * a_sr + cols) * e <= pb || pb + ((rows - 1) * b_sr + cols) * f <= pa);
}

static int arn_check(int64_t rows, int cols, int io, int st) {
    MAMBA_CHECK_ARG(rows >= 0 && rows < (1ll << 31), "rows must be in [0, 2^31)");
    MAMBA_CHECK_ARG(cols >= 1 && cols <= (1 << 28), "cols must be in [1, 2^28]");
    MAMBA_CHECK_ARG((io == MAMBA_F32 && st == MAMBA_F32) || (io == MAMBA_BF16 && (st == MAMBA_F32 || st == MAMBA_BF16)),
                    "io_dtype must be f32 with an f32 stream, or bf16 with an f32 or bf16 one");
    return MAMBA_OK;
}

extern "C" int mamba_add_rmsnorm_fwd(const mamba_add_rmsnorm_args* a, mamba_stream_t stream) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    int st = arn_check(a->rows, a->cols, a->io_dtype, a->stream_dtype);
    if (st != MAMBA_OK) return st;
    MAMBA_CHECK_ARG(a->eps >= 0.f, "eps must be >= 0");
    MAMBA_CHECK_ARG((a->y != nullptr) != (a->q != nullptr) || a->rows == 0, "one of y and q is required");
    MAMBA_CHECK_ARG(!a->q || a->q_dtype == MAMBA_INT8 || a->q_dtype == MAMBA_E4M3, "q_dtype must be int8 or e4m3");
    if (a->rows == 0) return MAMBA_OK;
    MAMBA_CHECK_ARG(a->x != nullptr, "x is required");
    MAMBA_CHECK_ARG((a->residual != nullptr) == (a->s != nullptr), "s goes with residual");
    MAMBA_CHECK_ARG(!a->q || a->scale, "scale goes with q");
    const int64_t R = a->rows;
    const int C = a->cols, e = a->io_dtype == MAMBA_BF16 ? 2 : 4, f = a->stream_dtype == MAMBA_BF16 ? 2 : 4;
    MAMBA_CHECK_ARG(R == 1 || ((!a->y || a->y_sr >= C) && (!a->s || a->s_sr >= C) && (!a->q || a->q_sr >= C)), "rows of y, s or q overlap");
    MAMBA_CHECK_ARG(!arn_clash(a->y, a->y_sr, e, a->x, a->x_sr, e, R, C, true) &&
                        !arn_clash(a->y, a->y_sr, e, a->residual, a->residual_sr, f, R, C, false) &&
                        !arn_clash(a->y, a->y_sr, e, a->s, a->s_sr, f, R, C, false) &&
                        !arn_clash(a->s, a->s_sr, f, a->x, a->x_sr, e, R, C, true) &&
                        !arn_clash(a->s, a->s_sr, f, a->residual, a->residual_sr, f, R, C, true) &&
                        !arn_clash(a->q, a->q_sr, 1, a->x, a->x_sr, e, R, C, false) &&
                        !arn_clash(a->q, a->q_sr, 1, a->residual, a->residual_sr, f, R, C, false) &&
                        !arn_clash(a->q, a->q_sr, 1, a->s, a->s_sr, f, R, C, false),
                    "an output overlaps an input or another (s may be residual or x itself, y x)");
    ArnP p{};
    p.rows = R; p.cols = C; p.eps = a->eps; p.x = a->x; p.x_sr = a->x_sr; p.res = a->residual; p.res_sr = a->residual_sr;
    p.w = a->weight; p.s = a->s; p.s_sr = a->s_sr; p.y = a->y; p.y_sr = a->y_sr; p.rstd = a->rstd;
    p.q = static_cast<uint8_t*>(a->q); p.q_sr = a->q_sr; p.scale = a->scale; p.e4m3 = a->q_dtype == MAMBA_E4M3;
    ARN_DISPATCH(arn_fwd_launch, a->io_dtype, a->stream_dtype, p, (hipStream_t)stream);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}

extern "C" size_t mamba_add_rmsnorm_bwd_workspace_size(const mamba_add_rmsnorm_bwd_args* a) {
    if (a == nullptr || arn_check(a->rows, a->cols, a->io_dtype, a->stream_dtype) != MAMBA_OK || !a->dweight) return 0;
    return (size_t)arn_parts(a->rows) * a->cols * 4;
}

extern "C" int mamba_add_rmsnorm_bwd(const mamba_add_rmsnorm_bwd_args* a, void* ws, size_t ws_bytes, mamba_stream_t stream) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    int st = arn_check(a->rows, a->cols, a->io_dtype, a->stream_dtype);
    if (st != MAMBA_OK) return st;
    MAMBA_CHECK_ARG(a->rows == 0 || (a->s && a->dy && a->rstd), "s, dy and rstd are required");
    const int64_t R = a->rows;
    const int C = a->cols, e = a->io_dtype == MAMBA_BF16 ? 2 : 4, f = a->stream_dtype == MAMBA_BF16 ? 2 : 4;
    MAMBA_CHECK_ARG(R <= 1 || ((!a->dx || a->dx_sr >= C) && (!a->dresidual || a->dresidual_sr >= C)), "rows of dx or dresidual overlap");
    struct Rows { const void* p; int64_t sr; int e; };
    const Rows ins[] = {{a->s, a->s_sr, f}, {a->dy, a->dy_sr, e}, {a->ds, a->ds_sr, f}}, outs[] = {{a->dx, a->dx_sr, e}, {a->dresidual, a->dresidual_sr, f}};
    for (const Rows& o : outs)
        for (const Rows& i : ins)
            MAMBA_CHECK_ARG(!arn_clash(o.p, o.sr, o.e, i.p, i.sr, i.e, R, C, false), "a gradient overlaps an input");
    MAMBA_CHECK_ARG(!arn_clash(a->dx, a->dx_sr, e, a->dresidual, a->dresidual_sr, f, R, C, false), "dx overlaps dresidual");
    const size_t need = mamba_add_rmsnorm_bwd_workspace_size(a);
    if (need && (ws == nullptr || ws_bytes < need)) {
        set_error("mamba_add_rmsnorm_bwd: workspace missing or too small");
        return MAMBA_ERR_WORKSPACE;
    }
    ArnP p{};
    p.rows = R; p.cols = C; p.s = const_cast<void*>(a->s); p.s_sr = a->s_sr; p.dy = a->dy; p.dy_sr = a->dy_sr; p.ds = a->ds; p.ds_sr = a->ds_sr;
    p.w = a->weight; p.rstd = const_cast<float*>(a->rstd); p.y = a->dx; p.y_sr = a->dx_sr; p.dres = a->dresidual; p.dres_sr = a->dresidual_sr;
    p.part = need ? static_cast<float*>(ws) : nullptr; p.parts = arn_parts(R); p.dw = a->dweight;
    ARN_DISPATCH(arn_bwd_launch, a->io_dtype, a->stream_dtype, p, (hipStream_t)stream);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}
