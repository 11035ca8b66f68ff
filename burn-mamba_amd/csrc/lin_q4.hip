// Products of few rows with weights of 4 bits for gfx950.
//
//   y[m, n] = xs[m] sum_g scale[g, n] (sum_{k in g} x[m, k] c[k, n] - zero[g, n] sum_{k in g} x[m, k]) + bias[n]
//
// Packed weight: tiles of 16 columns x 128 rows of k (a block: 1 KB, 16 bytes a lane), a
// column tile's blocks one behind the other along k.  Lane l of a block holds column l % 16;
// dword st of its four the codes of k = 32 st + 8 (l / 16) + e, e = 0..7: nibble e / 2 for even
// e, 4 + e / 2 for odd, so that two consecutive k lie 16 bits apart.  Behind the blocks the
// scales [tile][group][16], then the zero points [tile][group][16] bytes.  What k and columns
// are padded with has code 0, scale 0 and zero point 0.
#include <algorithm>

#include "pack.h"

namespace mamba {

constexpr int kQ4N = 16, kQ4K = 128;  // columns and k of a block

struct Q4W {
    int K, N, G;            // group: k of a group
    int KB, NT, NG;         // blocks along k, column tiles, groups along k (padded to whole blocks)
    bool zeros, sbf16;
    const uint4* codes;     // [NT][KB][64]
    const void* scale;      // [NT][NG][16]
    const uint8_t* zero;    // [NT][NG][16]
};

static bool q4_make(const mamba_q4_weight* w, Q4W* o, size_t* bytes) {
    if (w == nullptr || w->d_in < 1 || w->d_out < 1 || w->d_in > (1 << 24) || w->d_out > (1 << 24)) return false;
    if (w->group != 32 && w->group != 64 && w->group != 128) return false;
    if (w->scale_dtype != MAMBA_F32 && w->scale_dtype != MAMBA_BF16) return false;
    Q4W q{};
    q.K = w->d_in; q.N = w->d_out; q.G = w->group;
    q.KB = ceil_div(q.K, kQ4K); q.NT = ceil_div(q.N, kQ4N); q.NG = q.KB * (kQ4K / q.G);
    q.zeros = w->has_zero != 0; q.sbf16 = w->scale_dtype == MAMBA_BF16;
    const size_t codes = (size_t)q.NT * q.KB * 1024, scales = align_up((size_t)q.NT * q.NG * kQ4N * (q.sbf16 ? 2 : 4), 256);
    const char* base = static_cast<const char*>(w->packed);
    q.codes = reinterpret_cast<const uint4*>(base);
    q.scale = base + codes;
    q.zero = reinterpret_cast<const uint8_t*>(base + codes + scales);
    *o = q;
    *bytes = codes + scales + (q.zeros ? (size_t)q.NT * q.NG * kQ4N : 0);
    return true;
}

__global__ __launch_bounds__(256) void q4_pack(Q4W w, const uint8_t* codes, const void* scale, const uint8_t* zero, uint32_t* out, void* oscale,
                                               uint8_t* ozero) {
    const int64_t step = (int64_t)gridDim.x * 256, at0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
    // column-major in the threads, so that neighbours read neighbouring codes
    for (int64_t i = at0; i < (int64_t)w.NT * w.KB * 256; i += step) {
        const int col = (int)(i % 16);
        int64_t t = i / 16;
        const int j = (int)(t % w.NT);
        t /= w.NT;
        const int k8 = (int)(t % 16);  // the run of 8 k inside the block
        const int64_t kb = t / 16;
        const int n = j * kQ4N + col;
        uint32_t v = 0;
        for (int e = 0; e < 8; ++e) {
            const int64_t k = kb * kQ4K + k8 * 8 + e;
            const uint32_t c = k < w.K && n < w.N ? codes[k * w.N + n] & 15u : 0u;
            v |= c << (4 * (e / 2 + 4 * (e & 1)));
        }
        out[((j * (int64_t)w.KB + kb) * 64 + (k8 & 3) * 16 + col) * 4 + k8 / 4] = v;
    }
    const int groups = (w.K + w.G - 1) / w.G;
    for (int64_t i = at0; i < (int64_t)w.NT * w.NG * kQ4N; i += step) {
        const int col = (int)(i % 16), g = (int)(i / 16 % w.NG), n = (int)(i / 16 / w.NG) * kQ4N + col;
        const bool in = g < groups && n < w.N;
        const int64_t src = (int64_t)g * w.N + n;
        if (w.sbf16) static_cast<bf16_t*>(oscale)[i] = in ? static_cast<const bf16_t*>(scale)[src] : (bf16_t)0;
        else static_cast<float*>(oscale)[i] = in ? static_cast<const float*>(scale)[src] : 0.f;
        if (ozero) ozero[i] = in ? zero[src] & 15 : 0;
    }
}

struct Q4P {
    Q4W w;
    int64_t rows;
    const void* x; int64_t x_ld;
    const float* xs;
    const float* bias;
    void* y; int64_t y_ld; bool ybf16;
};

template <typename T>
__device__ __forceinline__ float q4_x(const T* x) { return load_f32<T>(x); }
template <>
__device__ __forceinline__ float q4_x<int8_t>(const int8_t* x) { return (float)*x; }

// A wave per row and column tile.
template <typename T>
__global__ __launch_bounds__(64) void q4_rows(Q4P p) {
    const int l = threadIdx.x, col = l & 15, kq = l >> 4, n = blockIdx.x * kQ4N + col;
    for (int64_t m = blockIdx.y; m < p.rows; m += gridDim.y) {
        const T* x = static_cast<const T*>(p.x) + m * p.x_ld;
        float total = 0.f;
        for (int kb = 0; kb < p.w.KB; ++kb) {
            const uint4 c4 = p.w.codes[((int64_t)blockIdx.x * p.w.KB + kb) * 64 + l];
            const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                const int g = (kb * kQ4K + 32 * st) / p.w.G;
                const int64_t at = ((int64_t)blockIdx.x * p.w.NG + g) * kQ4N + col;
                const float s = p.w.sbf16 ? bf16_to_f32(static_cast<const bf16_t*>(p.w.scale)[at]) : static_cast<const float*>(p.w.scale)[at];
                const float z = p.w.zeros ? (float)p.w.zero[at] : 8.f;
                float sum = 0.f, sx = 0.f;
                for (int e = 0; e < 8; ++e) {
                    const int k = kb * kQ4K + 32 * st + 8 * kq + e;
                    const float v = k < p.w.K ? q4_x<T>(x + k) : 0.f;
                    sum = __builtin_fmaf(v, (float)((c[st] >> (4 * (e / 2 + 4 * (e & 1)))) & 15u), sum);
                    sx += v;
                }
                total = __builtin_fmaf(s, __builtin_fmaf(-z, sx, sum), total);
            }
        }
        total += __shfl_xor(total, 16, 64);
        total += __shfl_xor(total, 32, 64);
        if (kq == 0 && n < p.w.N) {
            if (p.xs) total *= p.xs[m];
            if (p.bias) total += p.bias[n];
            if (p.ybf16) store_f32<bf16_t>(static_cast<bf16_t*>(p.y) + m * p.y_ld + n, total);
            else static_cast<float*>(p.y)[m * p.y_ld + n] = total;
        }
    }
}

}  // namespace mamba

using namespace mamba;

#define Q4_SHAPE "d_in and d_out in [1, 2^24], group 32, 64 or 128 and scales of f32 or bf16 required"

extern "C" size_t mamba_linear_q4_packed_size(const mamba_q4_weight* w) {
    Q4W q;
    size_t bytes;
    return q4_make(w, &q, &bytes) ? bytes : 0;
}

extern "C" int mamba_linear_q4_pack(const mamba_q4_weight* w, const void* codes, const void* scale, const void* zero, void* packed,
                                    mamba_stream_t stream) {
    Q4W q;
    size_t bytes;
    MAMBA_CHECK_ARG(w != nullptr, "weight is NULL");
    mamba_q4_weight at = *w;
    at.packed = packed;
    MAMBA_CHECK_ARG(q4_make(&at, &q, &bytes), Q4_SHAPE);
    MAMBA_CHECK_ARG(codes && scale && packed && (zero || !q.zeros), "codes, scale, packed and, with has_zero, zero are required");
    MAMBA_CHECK_ARG(((uintptr_t)packed & 15u) == 0, "packed must be 16-byte aligned");
    const int64_t items = (int64_t)q.NT * q.KB * 256;
    hipLaunchKernelGGL(q4_pack, dim3((uint32_t)std::min<int64_t>((items + 255) / 256, 1 << 16)), dim3(256), 0, (hipStream_t)stream, q, (const uint8_t*)codes,
                       scale, (const uint8_t*)zero, (uint32_t*)packed, const_cast<void*>(q.scale), q.zeros ? const_cast<uint8_t*>(q.zero) : nullptr);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}

static int q4_check(const mamba_linear_q4_args* a, Q4P* out) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    size_t bytes;
    Q4P p{};
    MAMBA_CHECK_ARG(q4_make(&a->w, &p.w, &bytes), Q4_SHAPE);
    MAMBA_CHECK_ARG(a->rows >= 0 && a->rows < (1ll << 31), "rows must be in [0, 2^31)");
    MAMBA_CHECK_ARG(a->x_dtype == MAMBA_F32 || a->x_dtype == MAMBA_BF16 || a->x_dtype == MAMBA_INT8, "x_dtype must be f32, bf16 or int8");
    MAMBA_CHECK_ARG(a->y_dtype == MAMBA_F32 || a->y_dtype == MAMBA_BF16, "y_dtype must be f32 or bf16");
    MAMBA_CHECK_ARG((a->x_dtype == MAMBA_INT8) == (a->x_scale != nullptr) || a->rows == 0, "x_scale goes with rows of int8");
    p.rows = a->rows; p.x = a->x; p.x_ld = a->x_ld; p.xs = a->x_scale; p.bias = a->bias;
    p.y = a->y; p.y_ld = a->y_ld; p.ybf16 = a->y_dtype == MAMBA_BF16;
    *out = p;
    return MAMBA_OK;
}

extern "C" size_t mamba_linear_q4_workspace_size(const mamba_linear_q4_args* a) {
    Q4P p;
    if (q4_check(a, &p) != MAMBA_OK) return 0;
    return 0;
}

extern "C" int mamba_linear_q4_fwd(const mamba_linear_q4_args* a, void* ws, size_t ws_bytes, mamba_stream_t stream) {
    Q4P p;
    int st = q4_check(a, &p);
    if (st != MAMBA_OK) return st;
    if (p.rows == 0) return MAMBA_OK;
    MAMBA_CHECK_ARG(a->w.packed && p.x && p.y, "packed, x and y are required");
    MAMBA_CHECK_ARG(((uintptr_t)a->w.packed & 15u) == 0, "packed must be 16-byte aligned");
    MAMBA_CHECK_ARG(p.y_ld >= p.w.N || p.rows == 1, "rows of y overlap");
    const size_t ex = a->x_dtype == MAMBA_F32 ? 4 : a->x_dtype == MAMBA_BF16 ? 2 : 1, ey = p.ybf16 ? 2 : 4;
    const char *px = static_cast<const char*>(p.x), *py = static_cast<const char*>(p.y);
    MAMBA_CHECK_ARG(py + ((p.rows - 1) * p.y_ld + p.w.N) * ey <= px || px + ((p.rows - 1) * p.x_ld + p.w.K) * ex <= py, "y overlaps x");
    const dim3 grid(p.w.NT, (uint32_t)std::min<int64_t>(p.rows, 1024));
    if (a->x_dtype == MAMBA_F32) hipLaunchKernelGGL(q4_rows<float>, grid, dim3(64), 0, (hipStream_t)stream, p);
    else if (a->x_dtype == MAMBA_BF16) hipLaunchKernelGGL(q4_rows<bf16_t>, grid, dim3(64), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(q4_rows<int8_t>, grid, dim3(64), 0, (hipStream_t)stream, p);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}
