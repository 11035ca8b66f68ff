// Layer norm over the last axis for gfx950, forward and backward (f32 or bf16
// rows, f32 statistics, weight, bias and their gradients).
//
//   xh = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = xh w + b
//   g = dy w:  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum_r dy xh,  db = sum_r dy
//
// The variance is the mean of the squared distances from the mean, not a
// difference of two large sums.
//
// About ten operations an element against two elements moved (forward) or three
// (backward): HBM-bound.  Rows of up to 10240 bf16 or 5120 f32 elements stay in
// registers (each element is read once): G lanes hold a row, 8 (bf16) or 4 (f32) consecutive
// elements a lane and step, G = 16, 64 or 256 by the row's width.  The backward's
// workgroups take rows in turn and sum dw and db of their columns in registers,
// joined in LDS and, over the workgroups, by ln_dw_join, in a fixed order.
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

// elements of a lane and step: 16 bytes
template <typename T>
constexpr int kLnE = 16 / (int)sizeof(T);

// E weights from column c of those up to cols, 1 where there are none
template <int E>
__device__ __forceinline__ void ln_weights(const float* w, int c, int cols, float (&v)[E]) {
    if (w) {
        ld_run<E, float>(w + c, cols - c, v);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = 1.f;
    }
}

// Any width: a workgroup per row, the row read once per sweep.  4096 x 16384 bf16 138 us,
// f32 201: the three sweeps and the store at 3.9 TB/s (512 or 768 workgroups, whose
// rows the L2 would hold, take longer).
template <typename T>
__global__ __launch_bounds__(256) void ln_fwd_wide(LnParams p) {
    constexpr int E = kLnE<T>, S = 256 * E;
    __shared__ float red[4];
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(p.x) + r * p.x_sr;
        T* y = static_cast<T*>(p.out) + r * p.out_sr;
        float s = 0.f, v[E];
        for (int c = threadIdx.x * E; c < p.cols; c += S) {
            ld_run<E, T>(x + c, p.cols - c, v);
#pragma unroll
            for (int i = 0; i < E; ++i) s += v[i];
        }
        const float mean = ln_block_sum(s, red) / (float)p.cols;
        s = 0.f;
        for (int c = threadIdx.x * E; c < p.cols; c += S) {
            ld_run<E, T>(x + c, p.cols - c, v);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float d = c + i < p.cols ? v[i] - mean : 0.f;
                s = __builtin_fmaf(d, d, s);
            }
        }
        const float rstd = 1.f / sqrtf(ln_block_sum(s, red) / (float)p.cols + p.eps);
        for (int c = threadIdx.x * E; c < p.cols; c += S) {
            float w[E], b[E];
            ld_run<E, T>(x + c, p.cols - c, v);
            ln_weights<E>(p.w, c, p.cols, w);
            if (p.b) ld_run<E, float>(p.b + c, p.cols - c, b);
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = __builtin_fmaf((v[i] - mean) * rstd, w[i], p.b ? b[i] : 0.f);
            st_run<E, T>(y + c, p.cols - c, v);
        }
        if (threadIdx.x == 0) {
            if (p.mean) p.mean[r] = mean;
            if (p.rstd) p.rstd[r] = rstd;
        }
    }
}

// 4096 x 16384 with ln_dw_wide and the join: bf16 260 us, f32 369
template <typename T>
__global__ __launch_bounds__(256) void ln_dx_wide(LnParams p) {
    constexpr int E = kLnE<T>, S = 256 * E;
    __shared__ float red[4];
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(p.x) + r * p.x_sr;
        const T* dy = static_cast<const T*>(p.dy) + r * p.dy_sr;
        T* dx = static_cast<T*>(p.out) + r * p.out_sr;
        const float mean = p.mean[r], rstd = p.rstd[r];
        float s1 = 0.f, s2 = 0.f, v[E], g[E], w[E];
        auto load = [&](int c) __attribute__((always_inline)) {  // dy is 0 past the row's end
            ld_run<E, T>(x + c, p.cols - c, v);
            ld_run<E, T>(dy + c, p.cols - c, g);
            ln_weights<E>(p.w, c, p.cols, w);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                g[i] *= w[i];
                v[i] = c + i < p.cols ? (v[i] - mean) * rstd : 0.f;
            }
        };
        for (int c = threadIdx.x * E; c < p.cols; c += S) {
            load(c);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                s1 += g[i];
                s2 = __builtin_fmaf(g[i], v[i], s2);
            }
        }
        s1 = ln_block_sum(s1, red) / (float)p.cols;
        s2 = ln_block_sum(s2, red) / (float)p.cols;
        for (int c = threadIdx.x * E; c < p.cols; c += S) {
            load(c);
#pragma unroll
            for (int i = 0; i < E; ++i) g[i] = rstd * (g[i] - s1 - v[i] * s2);
            st_run<E, T>(dx + c, p.cols - c, g);
        }
    }
}

// dw and db of 64 runs of columns over one part of the rows: thread (run, q) takes
// every fourth row.
template <typename T>
__global__ __launch_bounds__(256) void ln_dw_wide(LnParams p) {
    constexpr int E = kLnE<T>;
    __shared__ float red[2][4][E][64];
    const int l = threadIdx.x & 63, c = (blockIdx.x * 64 + l) * E, q = threadIdx.x >> 6;
    const int64_t per = (p.rows + p.parts - 1) / p.parts;
    const int64_t r0 = blockIdx.y * per, r1 = min(p.rows, r0 + per);
    float sw[E], sb[E];
#pragma unroll
    for (int i = 0; i < E; ++i) sw[i] = sb[i] = 0.f;
    if (c < p.cols)
        for (int64_t r = r0 + q; r < r1; r += 4) {
            float v[E], g[E];
            ld_run<E, T>(static_cast<const T*>(p.x) + r * p.x_sr + c, p.cols - c, v);
            ld_run<E, T>(static_cast<const T*>(p.dy) + r * p.dy_sr + c, p.cols - c, g);
            const float mean = p.mean[r], rstd = p.rstd[r];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                sb[i] += g[i];
                sw[i] = __builtin_fmaf(g[i], (v[i] - mean) * rstd, sw[i]);
            }
        }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        red[0][q][i][l] = sw[i];
        red[1][q][i][l] = sb[i];
    }
    __syncthreads();
    if (q < 2) {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (c + i < p.cols)
                p.part[((int64_t)blockIdx.y * 2 + q) * p.cols + c + i] = (red[q][0][i][l] + red[q][1][i][l]) + (red[q][2][i][l] + red[q][3][i][l]);
    }
}

// ---- rows in registers
// Sum over aligned groups of G lanes in every lane; over the workgroup for G = 256
// (red: 4 floats, which no wave may still read from a sum before
// the last barrier: the callers alternate between four places).
template <int CTRL>
__device__ __forceinline__ float ln_dpp(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int G>
__device__ __forceinline__ float ln_sum(float v, float* red) {
    if constexpr (G == 16) {
        v += ln_dpp<0xB1>(v);   // xor 1
        v += ln_dpp<0x4E>(v);   // xor 2
        v += ln_dpp<0x141>(v);  // the other quad of the half row
        v += ln_dpp<0x140>(v);  // the other half row
        return v;
    } else if constexpr (G == 64) {
        return wave_sum_dpp(v);
    } else {
        v = wave_sum_dpp(v);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        return (red[0] + red[1]) + (red[2] + red[3]);
    }
}

// G lanes a row, V steps: G (V - 1) kLnE < cols <= G V kLnE, so that only the last
// step can pass the row's end.  The workgroups take their rows in
// turn, the next row's loads in flight while this one is summed; weight and bias
// stay in registers.  16384 x 2560 bf16: 27 us, 168 MB (6 TB/s, part of it out of the
// last-level cache).
template <typename T, int G, int V>
__global__ __launch_bounds__(256) void ln_fwd_rows(LnParams p) {
    constexpr int E = kLnE<T>, RB = 256 / G;
    __shared__ float red[16];
    const int l = threadIdx.x % G, sub = threadIdx.x / G;
    Elems<T, E> rx[V];
    auto fetch = [&](int64_t r) {
        if (r >= p.rows) return;
        const T* x = static_cast<const T*>(p.x) + r * p.x_sr;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int c = (k * G + l) * E, n = p.cols - c;
            if (k < V - 1 || n >= E) rx[k].load(x + c);
            else rx[k].load_part(x + c, n);
        }
    };
    fetch(blockIdx.x * (int64_t)RB + sub);
    float w[V][E], b[V][E];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int c = (k * G + l) * E;
        if (p.w) ld_run<E, float>(p.w + c, k < V - 1 ? E : p.cols - c, w[k]);
        if (p.b) ld_run<E, float>(p.b + c, k < V - 1 ? E : p.cols - c, b[k]);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            if (!p.w) w[k][i] = 1.f;
            if (!p.b) b[k][i] = 0.f;
        }
    }
    const float inv = 1.f / (float)p.cols;
    const int64_t step = (int64_t)gridDim.x * RB;
    int odd = 0;
    // every group of a workgroup makes the same number of turns (the sums of G = 256 meet at a barrier)
    for (int64_t r0 = blockIdx.x * (int64_t)RB; r0 < p.rows; r0 += step) {
        const int64_t r = r0 + sub;
        float v[V][E], s = 0.f;
#pragma unroll
        for (int k = 0; k < V; ++k) rx[k].get(v[k]);
        fetch(r + step);
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int i = 0; i < E; ++i) s += v[k][i];  // zeros past the row's end
        const float mean = ln_sum<G>(s, red + 8 * odd) * inv;
        s = 0.f;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int c = (k * G + l) * E;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                v[k][i] = k < V - 1 || c + i < p.cols ? v[k][i] - mean : 0.f;
                s = __builtin_fmaf(v[k][i], v[k][i], s);
            }
        }
        const float rstd = 1.f / sqrtf(ln_sum<G>(s, red + 8 * odd + 4) * inv + p.eps);
        odd ^= 1;
        if (r >= p.rows) continue;
        T* y = static_cast<T*>(p.out) + r * p.out_sr;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int c = (k * G + l) * E, n = k < V - 1 ? E : p.cols - c;
            if (n <= 0) break;
#pragma unroll
            for (int i = 0; i < E; ++i) v[k][i] = __builtin_fmaf(v[k][i] * rstd, w[k][i], b[k][i]);
            st_run<E, T>(y + c, n, v[k]);
        }
        if (l == 0) {
            if (p.mean) p.mean[r] = mean;
            if (p.rstd) p.rstd[r] = rstd;
        }
    }
}

// The workgroups take their rows in turn, the next row's loads issued before this
// one's sums; part[blockIdx.x] gets the workgroup's dw and db.  16384 x 2560 bf16: 51
// us, 252 MB and 10 of parts (5.1 TB/s), the join 5.
template <typename T, int G, int V>
__global__ __launch_bounds__(256) void ln_bwd_rows(LnParams p) {
    constexpr int E = kLnE<T>, RB = 256 / G;  // rows at a time
    __shared__ float red[16];
    // the weights, place (k E + i) G + l for element i of lane l's step k (they would take
    // the registers that a second wave needs); after the rows, the groups' sums
    __shared__ float s_w[G * V * E], s_b[G < 256 ? G * V * E : 1];
    const int l = threadIdx.x % G, sub = threadIdx.x / G;
    float dw[V][E], db[V][E];
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
        for (int i = 0; i < E; ++i) dw[k][i] = db[k][i] = 0.f;
    for (int c = threadIdx.x; c < G * V * E; c += 256)
        s_w[(c / (G * E) * E + c % E) * G + c / E % G] = c < p.cols ? (p.w ? p.w[c] : 1.f) : 0.f;
    __syncthreads();
    const float inv = 1.f / (float)p.cols;
    Elems<T, E> rx[V], rg[V];
    float mean = 0.f, rstd = 0.f;
    auto fetch = [&](int64_t r) {
        if (r >= p.rows) return;
        const T* x = static_cast<const T*>(p.x) + r * p.x_sr;
        const T* dy = static_cast<const T*>(p.dy) + r * p.dy_sr;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int c = (k * G + l) * E, n = p.cols - c;
            if (k < V - 1 || n >= E) {
                rx[k].load(x + c);
                rg[k].load(dy + c);
            } else {
                rx[k].load_part(x + c, n);
                rg[k].load_part(dy + c, n);
            }
        }
        mean = p.mean[r];
        rstd = p.rstd[r];
    };
    const int64_t step = (int64_t)gridDim.x * RB;
    int odd = 0;
    fetch(blockIdx.x * (int64_t)RB + sub);
    // every group of a workgroup makes the same number of turns (the sums of G = 256 meet at a barrier)
    for (int64_t r0 = blockIdx.x * (int64_t)RB; r0 < p.rows; r0 += step) {
        const int64_t r = r0 + sub;
        const bool live = r < p.rows;
        asm volatile("" ::: "memory");  // the weights stay in LDS: in registers they would cost a wave
        Elems<T, E> cx[V], cg[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            cx[k] = rx[k];
            cg[k] = rg[k];
        }
        const float mu = mean, rs = rstd;
        fetch(r + step);
        // xh and dy of step k, from the row as it was loaded (kept in f32 between the two
        // sweeps they would take twice the registers)
        auto values = [&](int k, float (&xh)[E], float (&g)[E]) __attribute__((always_inline)) {
            cx[k].get(xh);
            cg[k].get(g);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                xh[i] = (xh[i] - mu) * rs;
                if (k == V - 1 && (k * G + l) * E + i >= p.cols) xh[i] = 0.f;  // g is 0 there
            }
        };
        float s1 = 0.f, s2 = 0.f;
        if (live) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float xh[E], g[E];
                values(k, xh, g);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    dw[k][i] = __builtin_fmaf(g[i], xh[i], dw[k][i]);
                    db[k][i] += g[i];
                    g[i] *= s_w[(k * E + i) * G + l];
                    s1 += g[i];
                    s2 = __builtin_fmaf(g[i], xh[i], s2);
                }
            }
        }
        if (!p.out) continue;
        s1 = ln_sum<G>(s1, red + 8 * odd) * inv;
        s2 = ln_sum<G>(s2, red + 8 * odd + 4) * inv;
        odd ^= 1;
        if (!live) continue;
        T* dx = static_cast<T*>(p.out) + r * p.out_sr;
        asm volatile("" ::: "memory");
#pragma unroll
        for (int k = 0; k < V; ++k) {
#pragma unroll
            for (int j = 0; j < Elems<T, E>::W; ++j) asm volatile("" : "+v"(cx[k].w[j]), "+v"(cg[k].w[j]));
            const int c = (k * G + l) * E, n = k < V - 1 ? E : p.cols - c;
            if (n <= 0) break;
            float xh[E], g[E];
            values(k, xh, g);
#pragma unroll
            for (int i = 0; i < E; ++i) g[i] = rs * (g[i] * s_w[(k * E + i) * G + l] - s1 - xh[i] * s2);
            st_run<E, T>(dx + c, n, g);
        }
    }
    if (!p.part) return;
    float* part = p.part + (int64_t)blockIdx.x * 2 * p.cols;
    // the workgroup's groups, one behind the other
    if constexpr (G < 256) {
        __syncthreads();
        for (int q = 0; q < RB; ++q) {
            if (sub == q) {
#pragma unroll
                for (int k = 0; k < V; ++k)
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        const int at = (k * E + i) * G + l;
                        s_w[at] = q ? s_w[at] + dw[k][i] : dw[k][i];
                        s_b[at] = q ? s_b[at] + db[k][i] : db[k][i];
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < p.cols; c += 256) {
            const int k = c / (G * E), at = (k * E + c % E) * G + c / E % G;
            part[c] = s_w[at];
            part[p.cols + c] = s_b[at];
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int c = (k * G + l) * E, n = p.cols - c;
            if (n <= 0) break;
            st_run<E, float>(part + c, n, dw[k]);
            st_run<E, float>(part + p.cols + c, n, db[k]);
        }
    }
}

// The parts in order of their number: the same sums every time.  16 threads a
// column, four loads in flight each; 16 columns a workgroup and turn.
__global__ __launch_bounds__(256) void ln_dw_join(LnParams p) {
    __shared__ float red[16][17];
    const int x = threadIdx.x & 15, q = threadIdx.x >> 4;
    const int64_t pitch = 2ll * p.cols;
    // columns 0 .. cols - 1: dw, cols .. 2 cols - 1: db
    for (int c0 = blockIdx.x * 16; c0 < 2 * p.cols; c0 += gridDim.x * 16) {
        const int c = c0 + x;
        const bool live = c < 2 * p.cols;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        if (live) {
            const float* src = p.part + c;
            int i = q;
            for (; i + 48 < p.parts; i += 64) {
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] += src[(i + 16 * j) * pitch];
            }
            for (; i < p.parts; i += 16) s[0] += src[i * pitch];
        }
        red[q][x] = (s[0] + s[1]) + (s[2] + s[3]);
        __syncthreads();
        if (q == 0 && live) {
            float a = 0.f;
            for (int j = 0; j < 16; ++j) a += red[j][x];
            float* out = c < p.cols ? p.dw : p.db;
            if (out) out[c < p.cols ? c : c - p.cols] = a;
        }
        __syncthreads();
    }
}
// one turn up to 2^20 workgroups (a grid of 2^32 threads, reached at 2^27 columns, is none)
static uint32_t ln_join_grid(int cols) { return (uint32_t)std::min(ceil_div(2 * cols, 16), 1 << 20); }

// workgroups of a kernel that takes a row each in turn
static uint32_t ln_grid(int64_t rows) { return (uint32_t)std::min<int64_t>(rows, 1 << 20); }
// steps of 16 bytes a lane that the columns take with G lanes a row
template <typename T>
static int ln_steps(int cols, int G) { return ceil_div(cols, G * kLnE<T>); }
// Lanes a row, 0: the row is not held in registers.  16 lanes where four steps of them
// are enough (backward: one, for sixteen groups' sums meet at its end), a wave for
// five steps of it (2560 bf16 elements), then a workgroup.  us with 16 lanes / a wave, bf16,
// forward: 65536 x 192 11 / 21, x 384 17 / 22, x 512 23 / 24; backward: 65536 x 256
// 30 / 36, but 16384 x 256 21 / 17 and 16384 x 512 32 / 19.
template <typename T>
static int ln_lanes(int cols, bool back) {
    return ln_steps<T>(cols, 16) <= (back ? 1 : 4) ? 16 : ln_steps<T>(cols, 64) <= 5 ? 64 : ln_steps<T>(cols, 256) <= 5 ? 256 : 0;
}
// Workgroups of the forward: four a CU (16384 x 2560 bf16: 27.6 us; 29.5 with three, 31.5
// with sixteen), or one for each group of rows.
static uint32_t ln_fwd_grid(int64_t rows, int G) { return (uint32_t)std::min<int64_t>((rows + 256 / G - 1) / (256 / G), 1024); }
// Workgroups of the backward: two a CU where the rows are enough for it, which is what
// the registers of wide rows leave room for (four for up to 256 columns), and some eight
// rows a group at least, so that the parts stay few beside the rows.  us at 512 / 1024:
// 16384 x 5120 bf16 123 / 145, 65536 x 2560 202 / 216, f32 103 / 111 at 16384 x 2560,
// 65536 x 256 bf16 41 / 36.
static int ln_parts(int64_t rows, int cols, bool bf16) {
    const int G = bf16 ? ln_lanes<bf16_t>(cols, true) : ln_lanes<float>(cols, true);
    if (G == 0) return (int)std::min<int64_t>(256, (rows + 31) / 32);
    return (int)std::min<int64_t>(cols > 256 ? 512 : 1024, (rows + 8 * (256 / G) - 1) / (8 * (256 / G)));
}

// rows of cols elements with this row stride overlap nowhere
static bool ln_rows_ok(int64_t rows, int cols, int64_t sr) {
    return sr >= cols || rows <= 1;
}

template <typename T, int G, int V>
static void ln_rows_launch(const LnParams& p, bool back, hipStream_t s) {
    if constexpr (G > 16 || V == 1) {
        if (back) {
            hipLaunchKernelGGL((ln_bwd_rows<T, G, V>), dim3(p.parts), dim3(256), 0, s, p);
            return;
        }
    }
    hipLaunchKernelGGL((ln_fwd_rows<T, G, V>), dim3(ln_fwd_grid(p.rows, G)), dim3(256), 0, s, p);
}

// rows in registers; false where they are too wide
template <typename T>
static bool ln_rows(const LnParams& p, bool back, hipStream_t s) {
    const int G = ln_lanes<T>(p.cols, back);
    if (G == 0) return false;
    switch (G * 8 + ln_steps<T>(p.cols, G)) {
        case 16 * 8 + 1: ln_rows_launch<T, 16, 1>(p, back, s); break;
        case 16 * 8 + 2: ln_rows_launch<T, 16, 2>(p, back, s); break;
        case 16 * 8 + 3: ln_rows_launch<T, 16, 3>(p, back, s); break;
        case 16 * 8 + 4: ln_rows_launch<T, 16, 4>(p, back, s); break;
        case 64 * 8 + 1: ln_rows_launch<T, 64, 1>(p, back, s); break;
        case 64 * 8 + 2: ln_rows_launch<T, 64, 2>(p, back, s); break;
        case 64 * 8 + 3: ln_rows_launch<T, 64, 3>(p, back, s); break;
        case 64 * 8 + 4: ln_rows_launch<T, 64, 4>(p, back, s); break;
        case 64 * 8 + 5: ln_rows_launch<T, 64, 5>(p, back, s); break;
        case 256 * 8 + 2: ln_rows_launch<T, 256, 2>(p, back, s); break;
        case 256 * 8 + 3: ln_rows_launch<T, 256, 3>(p, back, s); break;
        case 256 * 8 + 4: ln_rows_launch<T, 256, 4>(p, back, s); break;
        default: ln_rows_launch<T, 256, 5>(p, back, s);
    }
    return true;
}

template <typename T>
static void ln_fwd_launch(const LnParams& p, hipStream_t s) {
    if (!ln_rows<T>(p, false, s)) hipLaunchKernelGGL(ln_fwd_wide<T>, dim3(ln_grid(p.rows)), dim3(256), 0, s, p);
}

template <typename T>
static void ln_bwd_launch(const LnParams& p, hipStream_t s) {
    const bool sums = p.dw || p.db;
    if (!ln_rows<T>(p, true, s)) {
        if (p.out) hipLaunchKernelGGL(ln_dx_wide<T>, dim3(ln_grid(p.rows)), dim3(256), 0, s, p);
        if (sums) hipLaunchKernelGGL(ln_dw_wide<T>, dim3(ceil_div(p.cols, 64 * kLnE<T>), p.parts), dim3(256), 0, s, p);
    }
    if (sums) hipLaunchKernelGGL(ln_dw_join, dim3(ln_join_grid(p.cols)), dim3(256), 0, s, p);
}

}  // namespace mamba

using namespace mamba;

extern "C" int mamba_layernorm_fwd(const mamba_layernorm_args* a, mamba_stream_t stream) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    MAMBA_CHECK_ARG(a->rows >= 0 && a->rows < (1ll << 31), "rows must be in [0, 2^31)");
    MAMBA_CHECK_ARG(a->cols >= 1 && a->cols <= (1 << 28), "cols must be in [1, 2^28]");
    MAMBA_CHECK_ARG(a->io_dtype == MAMBA_F32 || a->io_dtype == MAMBA_BF16, "io_dtype must be f32 or bf16");
    MAMBA_CHECK_ARG(a->eps >= 0.f, "eps must be >= 0");
    if (a->rows == 0) return MAMBA_OK;
    MAMBA_CHECK_ARG(a->x && a->y, "x and y are required");
    MAMBA_CHECK_ARG(ln_rows_ok(a->rows, a->cols, a->y_sr), "rows of y overlap");
    MAMBA_CHECK_ARG(!rows_clash(a->y, a->y_sr, a->x, a->x_sr, a->cols, a->cols, a->rows, a->io_dtype == MAMBA_BF16 ? 2 : 4, true),
                    "y overlaps x (it may be x itself)");
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
    MAMBA_CHECK_ARG(a->cols >= 1 && a->cols <= (1 << 28), "cols must be in [1, 2^28]");
    MAMBA_CHECK_ARG(a->io_dtype == MAMBA_F32 || a->io_dtype == MAMBA_BF16, "io_dtype must be f32 or bf16");
    return MAMBA_OK;
}

extern "C" size_t mamba_layernorm_bwd_workspace_size(const mamba_layernorm_bwd_args* a) {
    if (ln_bwd_check(a) != MAMBA_OK || (!a->dweight && !a->dbias)) return 0;
    return (size_t)ln_parts(a->rows, a->cols, a->io_dtype == MAMBA_BF16) * 2 * a->cols * 4;
}

extern "C" int mamba_layernorm_bwd(const mamba_layernorm_bwd_args* a, void* ws, size_t ws_bytes, mamba_stream_t stream) {
    int st = ln_bwd_check(a);
    if (st != MAMBA_OK) return st;
    const size_t need = mamba_layernorm_bwd_workspace_size(a);
    MAMBA_CHECK_ARG(a->rows == 0 || (a->x && a->dy && a->mean && a->rstd), "x, dy, mean and rstd are required");
    MAMBA_CHECK_ARG(!a->dx || ln_rows_ok(a->rows, a->cols, a->dx_sr), "rows of dx overlap");
    const size_t e = a->io_dtype == MAMBA_BF16 ? 2 : 4;
    MAMBA_CHECK_ARG(!rows_clash(a->dx, a->dx_sr, a->x, a->x_sr, a->cols, a->cols, a->rows, e, false) &&
                        !rows_clash(a->dx, a->dx_sr, a->dy, a->dy_sr, a->cols, a->cols, a->rows, e, false),
                    "dx overlaps x or dy");
    if (need && (ws == nullptr || ws_bytes < need)) {
        set_error("mamba_layernorm_bwd: workspace missing or too small");
        return MAMBA_ERR_WORKSPACE;
    }
    LnParams p{};
    p.rows = a->rows; p.cols = a->cols;
    p.x = a->x; p.x_sr = a->x_sr; p.dy = a->dy; p.dy_sr = a->dy_sr; p.w = a->weight;
    p.out = a->rows ? a->dx : nullptr; p.out_sr = a->dx_sr;
    p.mean = const_cast<float*>(a->mean); p.rstd = const_cast<float*>(a->rstd);
    p.part = need ? static_cast<float*>(ws) : nullptr; p.parts = ln_parts(a->rows, a->cols, a->io_dtype == MAMBA_BF16);
    p.dw = a->dweight; p.db = a->dbias;
    if (a->rows == 0) {  // the sums of no rows: zeros
        if (p.dw || p.db) hipLaunchKernelGGL(ln_dw_join, dim3(ln_join_grid(p.cols)), dim3(256), 0, (hipStream_t)stream, p);
    } else if (a->io_dtype == MAMBA_BF16) {
        ln_bwd_launch<bf16_t>(p, (hipStream_t)stream);
    } else {
        ln_bwd_launch<float>(p, (hipStream_t)stream);
    }
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}
