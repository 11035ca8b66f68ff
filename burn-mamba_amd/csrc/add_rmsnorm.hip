// RMS norm with the residual's addition for gfx950: forward (rows of f32 or bf16, or of
// 8 bits with a scale each), backward.
//
//   s = residual + x,  rstd = 1 / sqrt(mean(s^2) + eps),  y = s rstd w
//   8 bits: scale = max |y| / top, q = round(y / scale), top = 127 (int8) or 448 (e4m3), the quotients
//   rounded to f32 first
//   g = dy w,  xh = s rstd:  d = ds + rstd (g - xh mean(g xh)),  dw = sum_r dy xh
//
// The sum is normalised as it is in f32, before it is rounded to the stream's type: y
// then has one rounding.  The backward reads the stored s, or, where that one was rounded to bf16,
// the two rows that it was the sum of (16384 x 2560 93 us against 77): from the rounded s dw is off
// by 2e-3 of itself, from the sum by 1e-7.
//
// Some ten operations an element against three or four elements moved: HBM-bound.  Rows of up to
// 16384 bf16 or 8192 f32 stream elements stay in registers, so that each element is read
// once: G lanes hold a row, E = 16 bytes of the stream a lane and step, G = 16, 64, 256 or 512 by
// the row's width; the next row's loads are in flight while this one is summed.  The backward's
// workgroups take rows in turn and sum dw of their columns in registers, joined in LDS
// and, over the workgroups, by arn_dw_join, in a fixed order.  16384 x 2560, bf16 rows with an f32
// stream: forward 97 us (5.2 TB/s), backward with the join 127 (5.3), to int8 90 (5.1): what a copy
// reaches.  4096 x 16384 of bf16 in registers / by the wide kernels below: forward 103 / 166, backward
// 128 / 310, int8 106 / 211.  Times: calls back to back in a captured graph on a warm card.
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

// The scale of a row whose largest |y| has these bits (from 2^-100 on), and what the quotients y /
// scale are formed with: y up times inv + lo, which is 1 / (scale up) to 2^-47 of itself (inv = 0: a row of
// zeros).  up, a power of two, keeps lo of large rows above the smallest number.
struct ArnScale { float scale, up, inv, lo; };
__device__ __forceinline__ ArnScale arn_scale(uint32_t amax, bool e4m3) {
    const float top = e4m3 ? 448.f : 127.f;
    if (amax >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 1.f, 0.f, 0.f};
    if (amax < 0x0d800000u) return {0.f, 1.f, 0.f, 0.f};
    const float s = __uint_as_float(amax) / top, up = amax >= 0x5f800000u ? 0x1p-64f : 1.f;  // from 2^64 on
    const float inv = 1.f / (s * up);
    return {s, up, inv, __builtin_fmaf(-inv, s * up, 1.f) * inv};
}
// v / (scale up), v = y up, rounded once: what a division gives, but where the quotient lies within 2^-22
// steps of midway between two f32.  The product with inv alone is up to one and a half steps off, and of
// values at the edge between two codes a sixth fell on its wrong side.  4000 x 2560 to e4m3 15.3 us, with the
// product alone 15.2, with a division 17.7.
__device__ __forceinline__ float arn_quotient(float v, const ArnScale& s) { return __builtin_fmaf(v, s.inv, v * s.lo); }
__device__ __forceinline__ uint8_t arn_q8(float v, const ArnScale& s, bool e4m3) {
    if (s.inv == 0.f) return 0;
    const float t = arn_quotient(v * s.up, s);
    if (e4m3) return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(fminf(fmaxf(t, -448.f), 448.f), 0.f, 0, false);
    return (uint8_t)(int8_t)(int)rintf(fminf(fmaxf(t, -127.f), 127.f));
}

// ---- rows in registers
// Sum, or largest, over aligned groups of G lanes in every lane; over the workgroup for G = 256 and
// 512 (red: 8 places, which no wave may still read from a sum before the last barrier: the callers
// alternate between two sets).
template <int CTRL>
__device__ __forceinline__ uint32_t arn_dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true); }
struct ArnAdd {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }
};
struct ArnMax {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return max(a, b); }
};
template <int G, typename Op>
__device__ __forceinline__ uint32_t arn_all(uint32_t v, uint32_t* red, Op op) {
    v = op(v, arn_dpp<0xB1>(v));   // xor 1
    v = op(v, arn_dpp<0x4E>(v));   // xor 2
    v = op(v, arn_dpp<0x141>(v));  // the other quad of the half row
    v = op(v, arn_dpp<0x140>(v));  // the other half row
    if constexpr (G >= 64) {
        const uint32_t a = op((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16));
        v = op(a, op((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48)));
    }
    if constexpr (G >= 256) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = op(op(red[0], red[1]), op(red[2], red[3]));
        if constexpr (G == 512) v = op(v, op(op(red[4], red[5]), op(red[6], red[7])));
    }
    return v;
}
template <int G>
__device__ __forceinline__ float arn_sum(float v, uint32_t* red) { return __uint_as_float(arn_all<G>(__float_as_uint(v), red, ArnAdd())); }

constexpr int arn_block(int G) { return G > 256 ? G : 256; }
// elements of a lane and step: 16 bytes of the stream
template <typename S>
constexpr int kArnE = 16 / (int)sizeof(S);

// E consecutive results of 8 bits (v: y up), the first n of them
template <int E>
__device__ __forceinline__ void arn_put8(uint8_t* q, int n, const float (&v)[E], const ArnScale& sc, bool e4m3) {
    uint32_t w[E / 4];
#pragma unroll
    for (int i = 0; i < E; i += 4) {
        float t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float top = e4m3 ? 448.f : 127.f;
            t[j] = sc.inv == 0.f ? 0.f : __builtin_amdgcn_fmed3f(arn_quotient(v[i + j], sc), -top, top);
        }
        if (e4m3) {
            const int a = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
            w[i / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], a, true);
        } else {
            uint32_t b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = (uint32_t)(int)rintf(t[j]) & 255u;
            w[i / 4] = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
        }
    }
    if (n >= E) {
        __builtin_memcpy(q, w, E);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i < n) q[i] = (uint8_t)(w[i / 4] >> (8 * (i & 3)));
    }
}

// G lanes a row, V steps: G (V - 1) E < cols <= G V E, so that only the last step can pass the row's
// end.  Q: rows of 8 bits.
template <typename T, typename S, int G, int V, bool Q>
__global__ __launch_bounds__(arn_block(G)) void arn_fwd_rows(ArnP p) {
    constexpr int E = kArnE<S>, RB = arn_block(G) / G;
    __shared__ uint32_t red[32];
    const int l = threadIdx.x % G, sub = threadIdx.x / G;
    Elems<T, E> rx[V];
    Elems<S, E> rr[V];
    auto fetch = [&](int64_t r) __attribute__((always_inline)) {
        if (r >= p.rows) return;
        const T* x = static_cast<const T*>(p.x) + r * p.x_sr;
        const S* res = static_cast<const S*>(p.res) + r * p.res_sr;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int c = (k * G + l) * E, n = p.cols - c;
            if (k < V - 1 || n >= E) {
                rx[k].load(x + c);
                if (p.res) rr[k].load(res + c);
            } else {
                rx[k].load_part(x + c, n);
                if (p.res) rr[k].load_part(res + c, n);
            }
        }
    };
    fetch(blockIdx.x * (int64_t)RB + sub);
    float w[V][E];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int c = (k * G + l) * E;
        if (p.w) ld_run<E, float>(p.w + c, k < V - 1 ? E : p.cols - c, w[k]);
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (!p.w) w[k][i] = 1.f;
    }
    const float inv = 1.f / (float)p.cols;
    const int64_t step = (int64_t)gridDim.x * RB;
    int odd = 0;
    // every group of a workgroup makes the same number of turns (the sums of G >= 256 meet at a barrier)
    for (int64_t r0 = blockIdx.x * (int64_t)RB; r0 < p.rows; r0 += step) {
        const int64_t r = r0 + sub;
        float v[V][E], ss = 0.f;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            rx[k].get(v[k]);
            if (p.res) {
                float b[E];
                rr[k].get(b);
#pragma unroll
                for (int i = 0; i < E; ++i) v[k][i] += b[i];
            }
        }
        fetch(r + step);
        if (p.s && r < p.rows) {
            S* s = static_cast<S*>(p.s) + r * p.s_sr;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int c = (k * G + l) * E, n = k < V - 1 ? E : p.cols - c;
                if (n > 0) st_run<E, S>(s + c, n, v[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int i = 0; i < E; ++i) ss = __builtin_fmaf(v[k][i], v[k][i], ss);  // zeros past the row's end
        const float rstd = 1.f / sqrtf(__builtin_fmaf(arn_sum<G>(ss, red + 16 * odd), inv, p.eps));
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int i = 0; i < E; ++i) v[k][i] = v[k][i] * rstd * w[k][i];
        ArnScale sc{};
        if constexpr (Q) {
            uint32_t amax = 0;
#pragma unroll
            for (int k = 0; k < V; ++k)
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (k < V - 1 || (k * G + l) * E + i < p.cols) amax = max(amax, __float_as_uint(v[k][i]) & 0x7fffffffu);
            sc = arn_scale(arn_all<G>(amax, red + 16 * odd + 8, ArnMax()), p.e4m3);
            if (sc.up != 1.f) {
#pragma unroll
                for (int k = 0; k < V; ++k)
#pragma unroll
                    for (int i = 0; i < E; ++i) v[k][i] *= sc.up;
            }
        }
        odd ^= 1;
        if (r >= p.rows) continue;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int c = (k * G + l) * E, n = k < V - 1 ? E : p.cols - c;
            if (n <= 0) break;
            if constexpr (Q) arn_put8<E>(p.q + r * p.q_sr + c, n, v[k], sc, p.e4m3);
            else st_run<E, T>(static_cast<T*>(p.y) + r * p.y_sr + c, n, v[k]);
        }
        if (l == 0) {
            if (p.rstd) p.rstd[r] = rstd;
            if constexpr (Q) p.scale[r] = sc.scale;
        }
    }
}

// The workgroups take their rows in turn; part[blockIdx.x] gets the workgroup's dw.  SUM: s + x in
// the place of s.
template <typename T, typename S, int G, int V, bool SUM>
__global__ __launch_bounds__(arn_block(G)) void arn_bwd_rows(ArnP p) {
    constexpr int E = kArnE<S>, RB = arn_block(G) / G;
    __shared__ uint32_t red[16];
    __shared__ float s_w[G < 256 ? G * V * E : 1];  // after the rows, the groups' sums
    const int l = threadIdx.x % G, sub = threadIdx.x / G;
    Elems<S, E> rs[V], rd[V];
    Elems<T, E> rg[V], rx[SUM ? V : 1];
    float rstd = 0.f, dw[V][E], w[V][E];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int c = (k * G + l) * E;
        if (p.w) ld_run<E, float>(p.w + c, k < V - 1 ? E : p.cols - c, w[k]);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            if (!p.w) w[k][i] = 1.f;
            dw[k][i] = 0.f;
        }
    }
    auto fetch = [&](int64_t r) __attribute__((always_inline)) {
        if (r >= p.rows) return;
        const S* s = static_cast<const S*>(p.s) + r * p.s_sr;
        const S* d = static_cast<const S*>(p.ds) + r * p.ds_sr;
        const T* g = static_cast<const T*>(p.dy) + r * p.dy_sr;
        const T* x = static_cast<const T*>(p.x) + r * p.x_sr;
        rstd = p.rstd[r];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int c = (k * G + l) * E, n = p.cols - c;
            if (k < V - 1 || n >= E) {
                rs[k].load(s + c);
                rg[k].load(g + c);
                if (p.ds) rd[k].load(d + c);
                if constexpr (SUM) rx[k].load(x + c);
            } else {
                rs[k].load_part(s + c, n);
                rg[k].load_part(g + c, n);
                if (p.ds) rd[k].load_part(d + c, n);
                if constexpr (SUM) rx[k].load_part(x + c, n);
            }
        }
    };
    const float inv = 1.f / (float)p.cols;
    const int64_t step = (int64_t)gridDim.x * RB;
    int odd = 0;
    fetch(blockIdx.x * (int64_t)RB + sub);
    for (int64_t r0 = blockIdx.x * (int64_t)RB; r0 < p.rows; r0 += step) {
        const int64_t r = r0 + sub;
        const bool live = r < p.rows;
        float xh[V][E], g[V][E], d[V][E], dot = 0.f;
        const float rsd = rstd;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            rs[k].get(xh[k]);
            rg[k].get(g[k]);
            if (p.ds) rd[k].get(d[k]);
            if constexpr (SUM) {
                float x[E];
                rx[k].get(x);
#pragma unroll
                for (int i = 0; i < E; ++i) xh[k][i] += x[i];
            }
        }
        fetch(r + step);
        if (live) {
#pragma unroll
            for (int k = 0; k < V; ++k)
#pragma unroll
                for (int i = 0; i < E; ++i) {  // zeros past the row's end
                    xh[k][i] *= rsd;
                    dw[k][i] = __builtin_fmaf(g[k][i], xh[k][i], dw[k][i]);
                    g[k][i] *= w[k][i];
                    dot = __builtin_fmaf(g[k][i], xh[k][i], dot);
                }
        }
        dot = arn_sum<G>(dot, red + 8 * odd) * inv;
        odd ^= 1;
        if (!live) continue;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int c = (k * G + l) * E, n = k < V - 1 ? E : p.cols - c;
            if (n <= 0) break;
            float o[E];
#pragma unroll
            for (int i = 0; i < E; ++i) o[i] = __builtin_fmaf(rsd, __builtin_fmaf(-xh[k][i], dot, g[k][i]), p.ds ? d[k][i] : 0.f);
            if (p.y) st_run<E, T>(static_cast<T*>(p.y) + r * p.y_sr + c, n, o);
            if (p.dres) st_run<E, S>(static_cast<S*>(p.dres) + r * p.dres_sr + c, n, o);
        }
    }
    if (!p.part) return;
    float* part = p.part + (int64_t)blockIdx.x * p.cols;
    if constexpr (G < 256) {  // the workgroup's groups, one behind the other
        for (int q = 0; q < RB; ++q) {
            if (sub == q) {
#pragma unroll
                for (int k = 0; k < V; ++k)
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        const int at = (k * E + i) * G + l;
                        s_w[at] = q ? s_w[at] + dw[k][i] : dw[k][i];
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < p.cols; c += 256) part[c] = s_w[(c / (G * E) * E + c % E) * G + c / E % G];
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int c = (k * G + l) * E, n = p.cols - c;
            if (n > 0) st_run<E, float>(part + c, n, dw[k]);
        }
    }
}

// Any width: a workgroup per row, the row read once per sweep (two forward, three to 8 bits; two and
// one more for dw backward): 2048 x 20000, bf16 with an f32 stream: 167 us, 203 and 257.
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

// the backward's s from column c of a row on
template <typename T, typename S, int E>
__device__ __forceinline__ void arn_sum_row(const ArnP& p, const S* s, int64_t r, int c, float (&v)[E]) {
    ld_run<E, S>(s + c, p.cols - c, v);
    if constexpr (sizeof(S) == 2) {
        if (p.x) {
            float x[E];
            ld_run<E, T>(static_cast<const T*>(p.x) + r * p.x_sr + c, p.cols - c, x);
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] += x[i];
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
            arn_sum_row<T, S, E>(p, s, r, c, v);
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
            arn_sum_row<T, S, E>(p, static_cast<const S*>(p.s) + r * p.s_sr, r, c, v);
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
// steps of 16 stream bytes a lane that the columns take with G lanes a row
static int arn_steps(int cols, int E, int G) { return ceil_div(cols, G * E); }
// Lanes a row, 0: the row is not held in registers.
static int arn_lanes(int cols, int E) {
    return arn_steps(cols, E, 16) <= 2 ? 16 : arn_steps(cols, E, 64) <= 3 ? 64 : arn_steps(cols, E, 256) <= 5 ? 256 : arn_steps(cols, E, 512) <= 4 ? 512 : 0;
}
// Workgroups of the forward, which take rows in turn.  us at 1024 / 2048 / 16384: 16384 x 2560 with an f32
// stream 93 / 97 / 87, 4000 x 2560 of bf16 14.3 / 14.5 / 15.3, 65536 x 256 30.6 / 31.2 / 30.8, 8192 x 5120
// 97 / 95 / 88.
static uint32_t arn_fwd_grid(int64_t rows, int G) {
    const int rb = arn_block(G) / G;
    return (uint32_t)std::min<int64_t>((rows + rb - 1) / rb, 2048);
}
// Workgroups of the backward: two a CU, and some eight rows a group at least, so that the parts
// stay few beside the rows.  us at 512 / 1024 with the join: 16384 x 2560 with an f32 stream 127 /
// 137, bf16 77 / 88, 65536 x 256 52 / 50.
static int arn_parts(int64_t rows, int cols, int E) {
    const int G = arn_lanes(cols, E);
    if (G == 0) return (int)std::min<int64_t>(256, (rows + 31) / 32);
    const int rb = arn_block(G) / G;
    return (int)std::min<int64_t>(512, (rows + 8 * rb - 1) / (8 * rb));
}

template <typename T, typename S, int G, int V>
static void arn_rows_launch(const ArnP& p, bool back, hipStream_t s) {
    if (back) {
        if constexpr (sizeof(S) == 2) {
            if (p.x) {
                hipLaunchKernelGGL((arn_bwd_rows<T, S, G, V, true>), dim3(p.parts), dim3(arn_block(G)), 0, s, p);
                return;
            }
        }
        hipLaunchKernelGGL((arn_bwd_rows<T, S, G, V, false>), dim3(p.parts), dim3(arn_block(G)), 0, s, p);
    } else if (p.q) hipLaunchKernelGGL((arn_fwd_rows<T, S, G, V, true>), dim3(arn_fwd_grid(p.rows, G)), dim3(arn_block(G)), 0, s, p);
    else hipLaunchKernelGGL((arn_fwd_rows<T, S, G, V, false>), dim3(arn_fwd_grid(p.rows, G)), dim3(arn_block(G)), 0, s, p);
}
// rows in registers; false where they are too wide
template <typename T, typename S>
static bool arn_rows(const ArnP& p, bool back, hipStream_t s) {
    const int G = arn_lanes(p.cols, kArnE<S>);
    if (G == 0) return false;
    switch (G * 8 + arn_steps(p.cols, kArnE<S>, G)) {
        case 16 * 8 + 1: arn_rows_launch<T, S, 16, 1>(p, back, s); break;
        case 16 * 8 + 2: arn_rows_launch<T, S, 16, 2>(p, back, s); break;
        case 64 * 8 + 1: arn_rows_launch<T, S, 64, 1>(p, back, s); break;
        case 64 * 8 + 2: arn_rows_launch<T, S, 64, 2>(p, back, s); break;
        case 64 * 8 + 3: arn_rows_launch<T, S, 64, 3>(p, back, s); break;
        case 256 * 8 + 1: arn_rows_launch<T, S, 256, 1>(p, back, s); break;
        case 256 * 8 + 2: arn_rows_launch<T, S, 256, 2>(p, back, s); break;
        case 256 * 8 + 3: arn_rows_launch<T, S, 256, 3>(p, back, s); break;
        case 256 * 8 + 4: arn_rows_launch<T, S, 256, 4>(p, back, s); break;
        case 256 * 8 + 5: arn_rows_launch<T, S, 256, 5>(p, back, s); break;
        case 512 * 8 + 3: arn_rows_launch<T, S, 512, 3>(p, back, s); break;
        default: arn_rows_launch<T, S, 512, 4>(p, back, s);
    }
    return true;
}

template <typename T, typename S>
static void arn_fwd_launch(const ArnP& p, hipStream_t s) {
    if (!arn_rows<T, S>(p, false, s)) hipLaunchKernelGGL((arn_fwd_wide<T, S>), dim3(arn_grid(p.rows)), dim3(256), 0, s, p);
}
template <typename T, typename S>
static void arn_bwd_launch(const ArnP& p, hipStream_t s) {
    if (p.rows && !arn_rows<T, S>(p, true, s)) {
        if (p.y || p.dres) hipLaunchKernelGGL((arn_dx_wide<T, S>), dim3(arn_grid(p.rows)), dim3(256), 0, s, p);
        if (p.dw) hipLaunchKernelGGL((arn_dw_wide<T, S>), dim3(ceil_div(p.cols, 256), p.parts), dim3(256), 0, s, p);
    }
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
    return (size_t)arn_parts(a->rows, a->cols, a->stream_dtype == MAMBA_BF16 ? 8 : 4) * a->cols * 4;
}

extern "C" int mamba_add_rmsnorm_bwd(const mamba_add_rmsnorm_bwd_args* a, void* ws, size_t ws_bytes, mamba_stream_t stream) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    int st = arn_check(a->rows, a->cols, a->io_dtype, a->stream_dtype);
    if (st != MAMBA_OK) return st;
    MAMBA_CHECK_ARG(a->rows == 0 || (a->s && a->dy && a->rstd), "s, dy and rstd are required");
    MAMBA_CHECK_ARG(!a->x || a->stream_dtype == MAMBA_BF16, "x goes with a bf16 stream");
    const int64_t R = a->rows;
    const int C = a->cols, e = a->io_dtype == MAMBA_BF16 ? 2 : 4, f = a->stream_dtype == MAMBA_BF16 ? 2 : 4;
    MAMBA_CHECK_ARG(R <= 1 || ((!a->dx || a->dx_sr >= C) && (!a->dresidual || a->dresidual_sr >= C)), "rows of dx or dresidual overlap");
    struct Rows { const void* p; int64_t sr; int e; };
    const Rows ins[] = {{a->s, a->s_sr, f}, {a->dy, a->dy_sr, e}, {a->ds, a->ds_sr, f}, {a->x, a->x_sr, e}}, outs[] = {{a->dx, a->dx_sr, e}, {a->dresidual, a->dresidual_sr, f}};
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
    p.w = a->weight; p.rstd = const_cast<float*>(a->rstd); p.x = a->x; p.x_sr = a->x_sr; p.y = a->dx; p.y_sr = a->dx_sr; p.dres = a->dresidual; p.dres_sr = a->dresidual_sr;
    p.part = need ? static_cast<float*>(ws) : nullptr; p.parts = arn_parts(R, C, 16 / f); p.dw = a->dweight;
    ARN_DISPATCH(arn_bwd_launch, a->io_dtype, a->stream_dtype, p, (hipStream_t)stream);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}
