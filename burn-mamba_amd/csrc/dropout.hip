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

// A thread per block of four elements, which may span rows.
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

template <typename T>
static void dropout_launch(const DropoutParams& p, hipStream_t s) {
    const int64_t blocks = (p.rows * p.cols + 3) / 4;
    hipLaunchKernelGGL(dropout_any<T>, dim3((uint32_t)std::min<int64_t>((blocks + 255) / 256, 8192)), dim3(256), 0, s, p);
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
