// Depthwise causal convolution with SiLU over packed sequences, forward and
// backward, and its single-token form on a cache addressed by slot, for gfx950.
//
//   pre[t, c] = b[c] + sum_k w[c, k] x[t - K + 1 + k, c],   out = silu(pre)
// with the taps before a sequence's first row taken from its window (the last K
// inputs it has seen, in the cache's slot) or zero.  Backward, g = dout silu'(pre):
//   dx[t] = sum_k w[k] g[t + K - 1 - k] inside the sequence,
//   dw[c, k] = sum_t g[t] x[t - K + 1 + k],  db[c] = sum_t g[t].
//
// About 2 K + 10 operations an element against two elements moved: HBM-bound.
// A wave owns 64 V channels of one chunk of rows and walks down them with the
// taps in registers, so each row is read once but for the K - 1 rows before a
// chunk (and behind one, in the backward pass).  Where V does not divide the
// channels the last lane's run begins earlier, over channels that its neighbour has
// too: both compute and store the same values, and no load or store is in parts.
#include <algorithm>
#include <type_traits>

#include "pack.h"

namespace mamba {

struct ConvPk {
    Seqs q;
    int64_t rows;
    int C, K;
    bool silu, fill;
    const void* x; int64_t x_st;
    const void* dout; int64_t dout_st;
    const float* w; const float* b;
    void* out; int64_t out_st;      // out, or dx
    float* state; int64_t nslots; const int32_t* slots;
    int64_t chunk, nchunk;
    float* part;                    // [nchunk][K + 1][C]
    float* dw; float* db;
};

// the hardware's exp2 and reciprocal (a float below the normal ones adds 0 to 1)
__device__ __forceinline__ float conv_sigmoid(float v) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f));
}

// KT = K as a constant, or 0: any K up to kMaxTaps (and fewer than 4 channels), the taps in
// scratch memory, because registers cannot be indexed by a tap that the compiler does not know,
// and shifted by one each row (16384 x 5120 bf16: forward 75 us with K = 7 as a
// constant, 1074 without; backward 137, 3276).
constexpr int kMaxTaps = 64;
constexpr int kConvRows = 4;  // rows whose loads are in flight while four others are computed

// V channels' weights and bias; taps[k] = the input of row t - (K - 1) + k, k < K - 1
template <int V, int KM>
__device__ __forceinline__ void conv_weights(const ConvPk& p, int K, int c, float (&w)[KM][V], float (&bias)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bias[v] = p.b ? p.b[c + v] : 0.f;
        for (int k = 0; k < K; ++k) w[k][v] = p.w[(int64_t)(c + v) * K + k];
    }
}
template <typename T, int V, int KM>
__device__ __forceinline__ void conv_taps(const ConvPk& p, int K, int s, int st, int t, int c, float (&tap)[KM][V]) {
    const int64_t slot = p.state ? slot_of(p.slots, s, p.nslots) : -1;
    for (int k = 0; k < K - 1; ++k) {
        const int at = t - (K - 1) + k;
        if (at >= st) {
            ld_run<V, T>(static_cast<const T*>(p.x) + (int64_t)at * p.x_st + c, V, tap[k]);
        } else {
            const int col = K + at - st;
#pragma unroll
            for (int v = 0; v < V; ++v) tap[k][v] = slot >= 0 ? p.state[(slot * p.C + c + v) * K + col] : 0.f;
        }
    }
}
// A row of V channels from c.  The row's base is in scalar registers, the lane's place
// 32 bits.
template <typename T, int V>
__device__ __forceinline__ void conv_load(const void* src, int64_t st, int t, int c, Elems<T, V>& e) {
    e.load(static_cast<const T*>(src) + t * st + (uint32_t)c);
}
template <typename T, int V>
__device__ __forceinline__ void conv_store(void* dst, int64_t st, int t, int c, const float (&o)[V]) {
    st_run<V, T>(static_cast<T*>(dst) + t * st + (uint32_t)c, V, o);
}

// 16384 x 5120 bf16, K = 4: 61 us, 344 MB (5.6 TB/s).
template <typename T, int KT, int V>
__global__ __launch_bounds__(256) void conv_pk_fwd(ConvPk p) {
    constexpr int KM = KT ? KT : kMaxTaps, R = KT ? kConvRows : 1;
    const int K = KT ? KT : p.K;
    const int lane = threadIdx.x & 63;
    const int nblk = (p.C + 64 * V - 1) / (64 * V);
    const int64_t item = blockIdx.x * 4ll + wave_id();
    const int64_t ck = item / nblk;
    if (ck >= p.nchunk) return;
    const int at_c = ((int)(item - ck * nblk) * 64 + lane) * V, c = min(at_c, p.C - V);
    if (at_c >= p.C) return;
    float w[KM][V], bias[V], tap[KM + R - 1][V];
    conv_weights<V, KM>(p, K, c, w, bias);
    const int c0 = (int)(ck * p.chunk), c1 = (int)min(p.rows, ck * p.chunk + p.chunk);
    int t = c0;
    const float zero[V] = {};
    Elems<T, V> raw[R];
    auto fetch = [&](int t0, int stop) {  // rows t0 .. of those before stop
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (t0 + i < stop) conv_load<T, V>(p.x, p.x_st, t0 + i, c, raw[i]);
    };
    for (int s = p.q.after(c0); s < p.q.n && t < c1; ++s) {
        const int st = p.q.begin(s), en = p.q.end(s);
        if (en <= t) {
            s = p.q.skip(s, t);
            continue;
        }
        for (; p.fill && t < min(st, c1); ++t) conv_store<T, V>(p.out, p.out_st, t, c, zero);
        t = max(t, st);
        if (t >= c1) break;
        const int stop = min(en, c1);
        fetch(t, stop);
        conv_taps<T, V, KM + R - 1>(p, K, s, st, t, c, tap);
        for (; t < stop; t += R) {
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (t + i < stop) raw[i].get(tap[K - 1 + i]);
            fetch(t + R, stop);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                if (t + i >= stop) break;
                float o[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    o[v] = bias[v];
                    for (int k = 0; k < K; ++k) o[v] = __builtin_fmaf(w[k][v], tap[i + k][v], o[v]);
                }
                if (p.silu) {
#pragma unroll
                    for (int v = 0; v < V; ++v) o[v] *= conv_sigmoid(o[v]);
                }
                conv_store<T, V>(p.out, p.out_st, t + i, c, o);
            }
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) tap[k][v] = tap[k + R][v];
        }
        t = stop;
    }
    for (; p.fill && t < c1; ++t) conv_store<T, V>(p.out, p.out_st, t, c, zero);
}

// an offset of a sequence that differs between the lanes
__device__ __forceinline__ int seq_at(const Seqs& q, int s) { return min(max(q.cu[s], 0), q.rows); }

// The windows after the call: window[k] = old window[k + length], then the last
// inputs.  After the forward kernel, which reads the old ones.
template <typename T>
__global__ __launch_bounds__(256) void conv_pk_window(ConvPk p) {
    const int64_t total = (int64_t)p.q.n * p.C;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const int s = (int)(i / p.C), c = (int)(i - (int64_t)s * p.C);
        const int64_t slot = slot_of(p.slots, s, p.nslots);
        const int st = seq_at(p.q, s), en = max(st, seq_at(p.q, s + 1)), len = en - st;
        if (slot < 0 || len == 0) continue;
        float* win = p.state + (slot * p.C + c) * p.K;
        const T* x = static_cast<const T*>(p.x) + c;
        for (int k = 0; k < p.K; ++k)
            win[k] = k + len < p.K ? win[k + len] : load_f32<T>(x + (int64_t)(en - p.K + k) * p.x_st);
    }
}

// dx, and a chunk's share of dw and db in registers.  16384 x 5120 bf16, K = 4: 111 us, 519
// MB and 16 of parts (4.8 TB/s; the vector units issue 0.7 of the time), the join 6.6.
template <typename T, int KT, int V>
__global__ __launch_bounds__(256) void conv_pk_bwd(ConvPk p) {
    constexpr int KM = KT ? KT : kMaxTaps, R = KT ? kConvRows : 1;
    const int K = KT ? KT : p.K;
    const int lane = threadIdx.x & 63;
    const int nblk = (p.C + 64 * V - 1) / (64 * V);
    const int64_t item = blockIdx.x * 4ll + wave_id();
    const int64_t ck = item / nblk;
    if (ck >= p.nchunk) return;
    const int at_c = ((int)(item - ck * nblk) * 64 + lane) * V, c = min(at_c, p.C - V);
    if (at_c >= p.C) return;
    // tap[K - 1 + i]: row r + i of x; g[i + k]: of row r + i - (K - 1) + k
    float w[KM][V], bias[V], tap[KM + R - 1][V], g[KM + R - 1][V], dw[KM][V], db[V];
    conv_weights<V, KM>(p, K, c, w, bias);
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) dw[k][v] = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) db[v] = 0.f;
    const int c0 = (int)(ck * p.chunk), c1 = (int)min(p.rows, ck * p.chunk + p.chunk);
    int t = c0;
    const float zero[V] = {};
    Elems<T, V> rx[R], rg[R];
    auto fetch = [&](int r, int last) {  // rows r .. of those before last
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (r + i >= last) break;
            conv_load<T, V>(p.x, p.x_st, r + i, c, rx[i]);
            conv_load<T, V>(p.dout, p.dout_st, r + i, c, rg[i]);
        }
    };
    for (int s = p.q.after(c0); s < p.q.n && t < c1; ++s) {
        const int st = p.q.begin(s), en = p.q.end(s);
        if (en <= t) {
            s = p.q.skip(s, t);
            continue;
        }
        for (; p.out && p.fill && t < min(st, c1); ++t) conv_store<T, V>(p.out, p.out_st, t, c, zero);
        t = max(t, st);
        if (t >= c1) break;
        // rows of this part give dw; the K - 1 behind it, where the sequence goes on, dx only
        const int stop = min(en, c1), last = min(en, stop + K - 1);
        fetch(t, last);
        conv_taps<T, V, KM + R - 1>(p, K, s, st, t, c, tap);
        for (int k = 0; k < K - 1; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) g[k][v] = 0.f;
        // R rows from r: g of them, and dx of the rows K - 1 before.  W: all of these are
        // in the part, and nothing is asked row by row (which would part the rows in the
        // schedule).
        int r = t;
        auto rows = [&](auto whole) __attribute__((always_inline)) {
            constexpr bool W = decltype(whole)::value;
#pragma unroll
            for (int i = 0; i < R; ++i) {
                if (W || r + i < last) {
                    rx[i].get(tap[K - 1 + i]);
                    rg[i].get(g[K - 1 + i]);
                } else {
#pragma unroll
                    for (int v = 0; v < V; ++v) g[K - 1 + i][v] = 0.f;
                }
            }
            fetch(r + R, last);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                if (p.silu && (W || r + i < last)) {
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        float acc = bias[v];
                        for (int k = 0; k < K; ++k) acc = __builtin_fmaf(w[k][v], tap[i + k][v], acc);
                        const float sg = conv_sigmoid(acc);
                        g[K - 1 + i][v] *= sg * __builtin_fmaf(acc, 1.f - sg, 1.f);
                    }
                }
                if (W || r + i < stop) {
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        db[v] += g[K - 1 + i][v];
                        for (int k = 0; k < K; ++k) dw[k][v] = __builtin_fmaf(g[K - 1 + i][v], tap[i + k][v], dw[k][v]);
                    }
                }
                const int at = r + i - (K - 1);
                if (p.out && (W || (at >= t && at < stop))) {
                    float o[V];
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        o[v] = 0.f;
                        for (int k = 0; k < K; ++k) o[v] = __builtin_fmaf(w[K - 1 - k][v], g[i + k][v], o[v]);
                    }
                    conv_store<T, V>(p.out, p.out_st, at, c, o);
                }
            }
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    tap[k][v] = tap[k + R][v];
                    g[k][v] = g[k + R][v];
                }
            r += R;
        };
        while (r < min(t + K - 1, stop + K - 1)) rows(std::false_type{});
        while (r + R <= stop) rows(std::true_type{});
        while (r < stop + K - 1) rows(std::false_type{});
        t = stop;
    }
    for (; p.out && p.fill && t < c1; ++t) conv_store<T, V>(p.out, p.out_st, t, c, zero);
    if (!p.part) return;
    float* part = p.part + (ck * (K + 1)) * (int64_t)p.C + c;
    for (int k = 0; k < K; ++k) st_run<V, float>(part + (int64_t)k * p.C, V, dw[k]);
    st_run<V, float>(part + (int64_t)K * p.C, V, db);
}

// The chunks' sums in order: the same result every time.  16 threads a column,
// four loads in flight each.
__global__ __launch_bounds__(256) void conv_pk_join(ConvPk p) {
    __shared__ float red[16][17];
    const int x = threadIdx.x & 15, q = threadIdx.x >> 4, c = blockIdx.x * 16 + x, k = blockIdx.y;
    const int64_t pitch = (int64_t)(p.K + 1) * p.C;
    const float* src = p.part + (int64_t)k * p.C + c;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < p.C) {
        int64_t i = q;
        for (; i + 48 < p.nchunk; i += 64) {
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += src[(i + 16 * j) * pitch];
        }
        for (; i < p.nchunk; i += 16) s[0] += src[i * pitch];
    }
    red[q][x] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (q == 0 && c < p.C) {
        float a = 0.f;
        for (int j = 0; j < 16; ++j) a += red[j][x];
        if (k < p.K) {
            if (p.dw) p.dw[(int64_t)c * p.K + k] = a;
        } else if (p.db) {
            p.db[c] = a;
        }
    }
}

// One token per row: the window of the row's slot moves on by it.
struct ConvSlotParams {
    int nb, C, K;
    bool silu;
    const void* x; int64_t x_sb;
    float* state; int64_t nslots; const int32_t* slots;
    const float* w; const float* b;
    void* out; int64_t out_sb;
};

// KT = K up to 8 (4 and 2 with windows of 16 and 8 aligned bytes), or 0 for any width.  HBM-bound (8 K bytes
// of window an element), so the arithmetic may be the plain composition's: each
// product rounded, pairs of them summed first, then the bias, and SiLU with a
// correctly rounded division (silu_f32).  A bf16 output then rounds the way the
// composition's does, and the state that the scan keeps from it in f32 does not
// differ by bf16 steps.  256 tokens x 5120, K = 4, bf16: 8.7 us, 47 MB (5.4 TB/s).
template <typename T, int KT>
__global__ __launch_bounds__(256) void conv_slot_step(ConvSlotParams p) {
#pragma clang fp contract(off)
    const int b = blockIdx.y, c = blockIdx.x * 256 + threadIdx.x;
    if (c >= p.C) return;
    const int64_t slot = slot_of(p.slots, b, p.nslots);
    T* out = static_cast<T*>(p.out) + b * p.out_sb + c;
    if (slot < 0) {
        store_f32<T>(out, 0.f);
        return;
    }
    const int K = KT ? KT : p.K;
    float* win = p.state + (slot * p.C + c) * K;
    const float* w = p.w + (int64_t)c * K;
    const float xv = load_f32<T>(static_cast<const T*>(p.x) + b * p.x_sb + c);
    float acc;
    if constexpr (KT != 0) {
        constexpr int kAlign = KT == 4 || KT == 2 ? 4 * KT : 4;
        float v[KT], wv[KT];
        __builtin_memcpy(v, __builtin_assume_aligned(win, kAlign), 4 * KT);
        __builtin_memcpy(wv, __builtin_assume_aligned(w, kAlign), 4 * KT);
#pragma unroll
        for (int k = 0; k < KT; ++k) v[k] = k + 1 < KT ? v[k + 1] : xv;
        if constexpr (KT == 4) {
            acc = (v[0] * wv[0] + v[1] * wv[1]) + (v[2] * wv[2] + v[3] * wv[3]);
        } else {  // even taps and odd ones
            float s[2] = {0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KT; ++k) s[k & 1] = s[k & 1] + v[k] * wv[k];
            acc = s[0] + s[1];
        }
        __builtin_memcpy(__builtin_assume_aligned(win, kAlign), v, 4 * KT);
    } else {
        float s[2] = {0.f, 0.f};
        for (int k = 0; k < K; ++k) {
            const float v = k + 1 < K ? win[k + 1] : xv;
            win[k] = v;
            s[k & 1] = s[k & 1] + v * w[k];
        }
        acc = s[0] + s[1];
    }
    if (p.b) acc = acc + p.b[c];
    store_f32<T>(out, p.silu ? silu_f32(acc) : acc);
}

template <typename T>
static void conv_slot_launch(const ConvSlotParams& p, hipStream_t s) {
    const dim3 grid(ceil_div(p.C, 256), p.nb);
    const uintptr_t at = (uintptr_t)p.state | (uintptr_t)p.w;
    const int kt = (p.K == 4 && (at & 15u)) || (p.K == 2 && (at & 7u)) ? 0 : p.K;
    switch (kt) {
        case 2: hipLaunchKernelGGL((conv_slot_step<T, 2>), grid, dim3(256), 0, s, p); break;
        case 3: hipLaunchKernelGGL((conv_slot_step<T, 3>), grid, dim3(256), 0, s, p); break;
        case 4: hipLaunchKernelGGL((conv_slot_step<T, 4>), grid, dim3(256), 0, s, p); break;
        case 5: hipLaunchKernelGGL((conv_slot_step<T, 5>), grid, dim3(256), 0, s, p); break;
        case 6: hipLaunchKernelGGL((conv_slot_step<T, 6>), grid, dim3(256), 0, s, p); break;
        case 7: hipLaunchKernelGGL((conv_slot_step<T, 7>), grid, dim3(256), 0, s, p); break;
        case 8: hipLaunchKernelGGL((conv_slot_step<T, 8>), grid, dim3(256), 0, s, p); break;
        default: hipLaunchKernelGGL((conv_slot_step<T, 0>), grid, dim3(256), 0, s, p);
    }
}

static int conv_pk_make(const mamba_conv1d_packed_args* a, bool back, ConvPk* o) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    MAMBA_CHECK_ARG(a->rows >= 0 && a->rows < kMaxRows, "rows must be in [0, 2^31 - 2^20)");
    MAMBA_CHECK_ARG(a->channels >= 1 && a->channels <= (1 << 20), "channels must be in [1, 2^20]");
    MAMBA_CHECK_ARG(a->kernel >= 1 && a->kernel <= kMaxTaps, "kernel must be in [1, 64]");
    MAMBA_CHECK_ARG(a->nseq >= 0, "nseq must be >= 0");
    MAMBA_CHECK_ARG(a->io_dtype == MAMBA_F32 || a->io_dtype == MAMBA_BF16, "io_dtype must be f32 or bf16");
    MAMBA_CHECK_ARG(a->w != nullptr, "w is required");
    MAMBA_CHECK_ARG(a->cu_seqlens != nullptr, "cu_seqlens is required");
    ConvPk& p = *o;
    p = ConvPk{};
    p.q = Seqs{a->cu_seqlens, a->nseq, (int)a->rows};
    p.rows = a->rows; p.C = a->channels; p.K = a->kernel;
    p.silu = a->silu != 0; p.fill = a->fill_outside != 0;
    p.x = a->x; p.x_st = a->x_st; p.w = a->w; p.b = a->bias;
    // Rows of a chunk, and at most 2^20 items of 64 channels, which keeps the grid small.
    // Forward: four waves a SIMD where the rows are enough for it; 8 to 64 (long chunks
    // read fewer rows twice at their edges; 16384 x 5120 60 us with 64, 70 with 32).
    // Backward: rounds of three waves a SIMD, of at most 128 rows, so that the last round is a
    // whole one (16384 x 5120 bf16, 4 taps, with the join: 108 rows, one round, 126 us; 64
    // rows, 1.7 rounds, 136; 36 rows, 3 rounds, 145).  Three is what the registers of bf16 with
    // 4 taps (136) and of f32 with 2, 3 and 8 allow; bf16 with 2, 3, 7 and 8 and f32 with 5 to 7
    // have room for four, bf16 with 5 and 6 for five, f32 with 4 (178 registers) for two.  us at
    // 16384 x 5120 with the join: bf16 2, 3, 4, 6, 8 taps 112, 112, 115, 132, 136; f32 208,
    // 210, 228, 219, 227 (4.8 to 4.4 TB/s).
    if (back) {
        const int64_t fill = std::max<int64_t>(1, a->rows * ceil_div(p.C, 256) / (3 * 1024)), rounds = (fill + 127) / 128;
        p.chunk = std::max<int64_t>(8, (fill / rounds + 4) / 4 * 4);
    } else {
        const int64_t fill = a->rows * ceil_div(p.C, 256) / 4096;
        p.chunk = std::min<int64_t>(64, std::max<int64_t>(8, fill / 4 * 4));
    }
    while ((a->rows + p.chunk - 1) / p.chunk * ceil_div(p.C, 64) > (1ll << 20)) p.chunk *= 2;
    p.nchunk = (a->rows + p.chunk - 1) / p.chunk;
    return MAMBA_OK;
}

static uint32_t conv_pk_grid(const ConvPk& p, int V) {
    return (uint32_t)((p.nchunk * ((p.C + 64 * V - 1) / (64 * V)) + 3) / 4);
}

template <typename T, int KT, int V>
static void conv_pk_launch(const ConvPk& p, bool back, hipStream_t s) {
    const dim3 grid(conv_pk_grid(p, V));
    if (back) hipLaunchKernelGGL((conv_pk_bwd<T, KT, V>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((conv_pk_fwd<T, KT, V>), grid, dim3(256), 0, s, p);
}

template <typename T>
static void conv_pk_dispatch(const ConvPk& p, bool back, hipStream_t s) {
    switch (p.C >= 4 ? p.K : 0) {
        case 2: conv_pk_launch<T, 2, 4>(p, back, s); break;
        case 3: conv_pk_launch<T, 3, 4>(p, back, s); break;
        case 4: conv_pk_launch<T, 4, 4>(p, back, s); break;
        case 5: conv_pk_launch<T, 5, 2>(p, back, s); break;
        case 6: conv_pk_launch<T, 6, 2>(p, back, s); break;
        case 7: conv_pk_launch<T, 7, 2>(p, back, s); break;
        case 8: conv_pk_launch<T, 8, 2>(p, back, s); break;
        default: conv_pk_launch<T, 0, 1>(p, back, s);
    }
}

}  // namespace mamba

using namespace mamba;

extern "C" int mamba_conv1d_packed_fwd(const mamba_conv1d_packed_args* a, mamba_stream_t stream) {
    ConvPk p;
    int st = conv_pk_make(a, false, &p);
    if (st != MAMBA_OK) return st;
    if (p.rows == 0) return MAMBA_OK;
    MAMBA_CHECK_ARG(a->x && a->out, "x and out are required");
    MAMBA_CHECK_ARG(a->out_st >= p.C || p.rows == 1, "rows of out overlap");
    MAMBA_CHECK_ARG(a->state == nullptr || a->slots != nullptr || a->nslots >= a->nseq,
                    "without slots the state needs a row per sequence");
    MAMBA_CHECK_ARG(!rows_clash(a->out, a->out_st, a->x, a->x_st, p.C, p.C, p.rows, a->io_dtype == MAMBA_BF16 ? 2 : 4, false),
                    "out overlaps x, whose rows are read by their successors");
    p.out = a->out; p.out_st = a->out_st;
    p.state = a->state; p.nslots = a->nslots; p.slots = a->slots;
    hipStream_t s = (hipStream_t)stream;
    const bool bf16 = a->io_dtype == MAMBA_BF16;
    if (bf16) conv_pk_dispatch<bf16_t>(p, false, s);
    else conv_pk_dispatch<float>(p, false, s);
    MAMBA_CHECK_LAUNCH();
    if (p.state && p.q.n) {
        const dim3 grid((uint32_t)std::min<int64_t>(((int64_t)p.q.n * p.C + 255) / 256, 1 << 16));
        if (bf16) hipLaunchKernelGGL(conv_pk_window<bf16_t>, grid, dim3(256), 0, s, p);
        else hipLaunchKernelGGL(conv_pk_window<float>, grid, dim3(256), 0, s, p);
        MAMBA_CHECK_LAUNCH();
    }
    return MAMBA_OK;
}

extern "C" size_t mamba_conv1d_packed_bwd_workspace_size(const mamba_conv1d_packed_args* a) {
    ConvPk p;
    if (conv_pk_make(a, true, &p) != MAMBA_OK || (!a->dw && !a->dbias)) return 0;
    return (size_t)p.nchunk * (p.K + 1) * p.C * 4;
}

extern "C" int mamba_conv1d_packed_bwd(const mamba_conv1d_packed_args* a, void* ws, size_t ws_bytes, mamba_stream_t stream) {
    ConvPk p;
    int st = conv_pk_make(a, true, &p);
    if (st != MAMBA_OK) return st;
    MAMBA_CHECK_ARG(a->state == nullptr, "the gradient is of sequences without a window");
    MAMBA_CHECK_ARG(p.rows == 0 || (a->x && a->dout), "x and dout are required");
    MAMBA_CHECK_ARG(a->dx == nullptr || a->dx_st >= p.C || p.rows <= 1, "rows of dx overlap");
    const size_t e = a->io_dtype == MAMBA_BF16 ? 2 : 4;
    MAMBA_CHECK_ARG(!rows_clash(a->dx, a->dx_st, a->x, a->x_st, p.C, p.C, p.rows, e, false) &&
                        !rows_clash(a->dx, a->dx_st, a->dout, a->dout_st, p.C, p.C, p.rows, e, false),
                    "dx overlaps x or dout");
    const size_t need = mamba_conv1d_packed_bwd_workspace_size(a);
    if (need && (ws == nullptr || ws_bytes < need)) {
        set_error("mamba_conv1d_packed_bwd: workspace missing or too small");
        return MAMBA_ERR_WORKSPACE;
    }
    p.dout = a->dout; p.dout_st = a->dout_st; p.out = a->dx; p.out_st = a->dx_st;
    p.part = need ? static_cast<float*>(ws) : nullptr; p.dw = a->dw; p.db = a->dbias;
    hipStream_t s = (hipStream_t)stream;
    if (p.rows) {
        if (a->io_dtype == MAMBA_BF16) conv_pk_dispatch<bf16_t>(p, true, s);
        else conv_pk_dispatch<float>(p, true, s);
    }
    if (p.dw || p.db) hipLaunchKernelGGL(conv_pk_join, dim3(ceil_div(p.C, 16), p.K + 1), dim3(256), 0, s, p);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}

extern "C" int mamba_conv1d_step_slots(const mamba_conv1d_step_slots_args* a, mamba_stream_t stream) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    MAMBA_CHECK_ARG(a->batch >= 0 && a->batch <= 65535, "batch must be in [0, 65535]");
    MAMBA_CHECK_ARG(a->channels >= 1, "channels must be >= 1");
    MAMBA_CHECK_ARG(a->kernel >= 1 && a->kernel <= kMaxTaps, "kernel must be in [1, 64]");
    MAMBA_CHECK_ARG(a->io_dtype == MAMBA_F32 || a->io_dtype == MAMBA_BF16, "io_dtype must be f32 or bf16");
    if (a->batch == 0) return MAMBA_OK;
    MAMBA_CHECK_ARG(a->x && a->state && a->w && a->out, "x, state, w and out are required");
    MAMBA_CHECK_ARG(a->slots != nullptr || a->nslots >= a->batch, "without slots the state needs a row per token");
    MAMBA_CHECK_ARG(a->out_sb >= a->channels || a->batch == 1, "rows of out overlap");
    MAMBA_CHECK_ARG(!rows_clash(a->out, a->out_sb, a->x, a->x_sb, a->channels, a->channels, a->batch,
                                a->io_dtype == MAMBA_BF16 ? 2 : 4, true),
                    "out overlaps x (it may be x itself)");
    ConvSlotParams p{};
    p.nb = a->batch; p.C = a->channels; p.K = a->kernel; p.silu = a->silu != 0;
    p.x = a->x; p.x_sb = a->x_sb; p.state = a->state; p.nslots = a->nslots; p.slots = a->slots;
    p.w = a->w; p.b = a->bias; p.out = a->out; p.out_sb = a->out_sb;
    if (a->io_dtype == MAMBA_BF16) conv_slot_launch<bf16_t>(p, (hipStream_t)stream);
    else conv_slot_launch<float>(p, (hipStream_t)stream);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}
