// Dropout with an optional residual sum for gfx950, its mask computed where it
// is used and never stored.
//
//   out[i] = residual[i] + (word(i) >= p 2^32 ? x[i] / (1 - p) : 0)
//
// word(i) is word i % 4 of Philox 4x32 with ten rounds (Salmon, Moraes, Dror and
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) at counter
// (i / 4, call), i the element's place in row-major order and call = rng[1] +
// offset, under the key rng[0].  The gradient is the same function of dy, so
// the backward pass is this kernel again.  rng is read on the device: a captured
// graph draws new masks when the program advances it between replays.
#include "pack.h"

namespace mamba {

struct DropoutParams {
    int64_t rows, cols;
    const void* x; int64_t x_sr;
    const void* res; int64_t res_sr;
    void* out; int64_t out_sr;
    const int64_t* rng;
    uint64_t offset;
    uint64_t threshold;  // of 2^32: kept from here up
    float scale;
};

// The ten rounds: per round two 32 x 32 -> 64 bit products.
__device__ __forceinline__ void philox4x32(uint64_t block, uint64_t call, uint64_t seed, uint32_t (&c)[4]) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)call, c3 = (uint32_t)(call >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    c[0] = c0; c[1] = c1; c[2] = c2; c[3] = c3;
}

// A thread per block of four elements, which may span rows: strided rows of a width
// that 16 bytes do not divide (16384 x 5117 bf16: 163 us; 67 where they do).
template <typename T>
__global__ __launch_bounds__(256) void dropout_any(DropoutParams p) {
    const int64_t n = p.rows * p.cols, blocks = (n + 3) / 4;
    const uint64_t seed = (uint64_t)p.rng[0], call = (uint64_t)p.rng[1] + p.offset;
    for (int64_t k = blockIdx.x * 256ll + threadIdx.x; k < blocks; k += gridDim.x * 256ll) {
        uint32_t w[4];
        philox4x32((uint64_t)k, call, seed, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t i = 4 * k + e;
            if (i >= n) break;
            const int64_t r = i / p.cols, c = i - r * p.cols;
            // a dropped element's value is not looked at: an infinity there is dropped too
            float v = w[e] >= p.threshold ? load_f32<T>(static_cast<const T*>(p.x) + r * p.x_sr + c) * p.scale : 0.f;
            if (p.res) v += load_f32<T>(static_cast<const T*>(p.res) + r * p.res_sr + c);
            store_f32<T>(static_cast<T*>(p.out) + r * p.out_sr + c, v);
        }
    }
}

// Rows one behind the other (rows = 1), or of a multiple of V columns: V = 8
// (bf16) or 4 (f32) elements, 16 bytes, a thread and turn, two turns' loads in
// flight.  The generator takes about 30 32-bit operations an element (a 32 x 32
// -> 64 product counts four), which bf16's 4 to 6 bytes an element only just
// cover: HBM-bound, with little to spare.  16384 x 2560 bf16: 51 us with a residual (252
// MB, 4.9 TB/s), 38 without (168 MB, 4.5 TB/s, the vector units issuing 0.86 of the time).
template <typename T, int V, bool RES>
__global__ __launch_bounds__(256) void dropout_vec(DropoutParams p) {
    const int64_t n = p.rows * p.cols, units = (n + V - 1) / V, per = (p.cols + V - 1) / V;
    const uint64_t seed = (uint64_t)p.rng[0], call = (uint64_t)p.rng[1] + p.offset;
    const int64_t stride = gridDim.x * 256ll;
    constexpr int U = 2;
    for (int64_t k0 = blockIdx.x * 256ll + threadIdx.x; k0 < units; k0 += U * stride) {
        Elems<T, V> x[U], r[U];
        int64_t row[U], c[U];
        int left[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = k0 + u * stride;
            row[u] = p.rows > 1 ? k / per : 0;
            c[u] = (k - row[u] * per) * V;
            left[u] = k < units ? (int)min((int64_t)V, p.cols - c[u]) : 0;
            const T* xs = static_cast<const T*>(p.x) + row[u] * p.x_sr + c[u];
            const T* rs = static_cast<const T*>(p.res) + row[u] * p.res_sr + c[u];
            if (left[u] >= V) {
                x[u].load(xs);
                if (RES) r[u].load(rs);
            } else {
                x[u].load_part(xs, left[u]);
                if (RES) r[u].load_part(rs, left[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (left[u] <= 0) break;
            const int64_t first = (k0 + u * stride) * (V / 4);  // its first block of the generator
            float xv[V], rv[V];
            x[u].get(xv);
            if (RES) r[u].get(rv);
#pragma unroll
            for (int b = 0; b < V / 4; ++b) {
                uint32_t w[4];
                philox4x32((uint64_t)(first + b), call, seed, w);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = w[e] >= p.threshold ? xv[4 * b + e] * p.scale : 0.f;
                    if (RES) v += rv[4 * b + e];
                    xv[4 * b + e] = v;
                }
            }
            st_run<V, T>(static_cast<T*>(p.out) + row[u] * p.out_sr + c[u], left[u], xv);
        }
    }
}

template <typename T>
static void dropout_launch(const DropoutParams& p, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    auto grid = [](int64_t threads) { return dim3((uint32_t)std::min<int64_t>((threads + 255) / 256, 16384)); };
    if (p.rows == 1 || p.cols % V == 0) {
        const int64_t units = (p.rows * p.cols + V - 1) / V;
        if (p.res) hipLaunchKernelGGL((dropout_vec<T, V, true>), grid((units + 1) / 2), dim3(256), 0, s, p);
        else hipLaunchKernelGGL((dropout_vec<T, V, false>), grid((units + 1) / 2), dim3(256), 0, s, p);
    } else {
        hipLaunchKernelGGL(dropout_any<T>, grid((p.rows * p.cols + 3) / 4), dim3(256), 0, s, p);
    }
}

}  // namespace mamba

using namespace mamba;

extern "C" int mamba_dropout(const mamba_dropout_args* a, mamba_stream_t stream) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    MAMBA_CHECK_ARG(a->rows >= 0 && a->cols >= 0, "rows and cols must be >= 0");
    MAMBA_CHECK_ARG(a->io_dtype == MAMBA_F32 || a->io_dtype == MAMBA_BF16, "io_dtype must be f32 or bf16");
    MAMBA_CHECK_ARG(a->p >= 0.0 && a->p <= 1.0, "p must be in [0, 1]");
    if (a->rows == 0 || a->cols == 0) return MAMBA_OK;
    MAMBA_CHECK_ARG(a->cols < (1ll << 46) / a->rows, "rows * cols must be below 2^46");
    MAMBA_CHECK_ARG(a->x && a->out && a->rng, "x, out and rng are required");
    MAMBA_CHECK_ARG(a->rows == 1 || a->out_sr >= a->cols, "rows of out overlap");
    const size_t e = a->io_dtype == MAMBA_BF16 ? 2 : 4;
    MAMBA_CHECK_ARG(!rows_clash(a->out, a->out_sr, a->x, a->x_sr, a->cols, a->cols, a->rows, e, true) &&
                        !rows_clash(a->out, a->out_sr, a->residual, a->residual_sr, a->cols, a->cols, a->rows, e, true),
                    "out overlaps x or residual (it may be either itself)");
    DropoutParams p{};
    p.rows = a->rows; p.cols = a->cols;
    p.x = a->x; p.x_sr = a->x_sr; p.res = a->residual; p.res_sr = a->residual_sr;
    p.out = a->out; p.out_sr = a->out_sr; p.rng = a->rng; p.offset = (uint64_t)a->offset;
    // to the nearest 2^-32, so 2^32 (none is kept) is reached
    p.threshold = (uint64_t)(a->p * 4294967296.0 + 0.5);
    p.scale = a->p < 1.0 ? (float)(1.0 / (1.0 - a->p)) : 0.f;
    if (a->io_dtype == MAMBA_BF16) dropout_launch<bf16_t>(p, (hipStream_t)stream);
    else dropout_launch<float>(p, (hipStream_t)stream);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}
