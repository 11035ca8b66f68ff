// Products of few rows with weights of 4 bits for gfx950.
//
//   y[m, n] = xs[m] sum_g scale[g, n] (sum_{k in g} x[m, k] c[k, n] - zero[g, n] sum_{k in g} x[m, k]) + bias[n]
//
// Packed weight: tiles of 16 columns x 128 rows of k (a block: 1 KB, 16 bytes a lane), a
// column tile's blocks one behind the other along k.  Lane l of a block holds column l % 16;
// dword st of its four the codes of k = 32 st + 8 (l / 16) + e, e = 0..7: nibble e / 2 for even
// e, 4 + e / 2 for odd, so that two consecutive k lie 16 bits apart.  Behind the blocks, for
// [tile][group][16], the scale and -(16 + zero point): two bf16 in a word, or with f32 scales two
// floats.  What k and columns are padded with has scale 0, a group with a zero point above 16 a NaN.
//
// A code goes into the matrix instruction as 16 + c, which its bits give in one or two instructions,
// and -(16 + zero) as a second operand with the same rows: no weight is formed, and no rounding but
// that of f32 sums.  Those are sums of up to 31 x, of which the second operand takes most off again:
// a step of theirs is up to 16 times one of the result's terms.  f32 rows go in as three bf16 parts.
// int8 rows take the codes as bytes, and their sums are whole numbers up to the scale.
//
// Few rows are bound by the weight's bytes and a kernel's trips to memory: 1 x 2560 x 10240 5.3 us
// (13.9 MB; at a copy's rate 2.8; of its 640 column tiles 128 are a second turn of 512 workgroups), 7 x
// 2560 x 50001 15.8 (67 MB, 4.2 TB/s).  More rows are loaded into registers before the first block is
// used, 16 in 2.5 us, and a turn of a workgroup (four waves of five blocks, then a barrier) takes 1.3: 64
// rows of int8 13.7 us, in which two waves a SIMD issue two thirds of the time.  A prompt's rows go the
// same way, 16 or 32 a workgroup and every code taken apart for each: 4000 x 2560 x 10240 of bf16 378 us,
// 555 TFLOP/s.  Times: calls back to back in a captured graph on a warm card.
#include <algorithm>

#include "pack.h"

namespace mamba {

constexpr int kQ4N = 16, kQ4K = 128;  // columns and k of a block
constexpr int kQ4Waves = 12;           // of a workgroup that holds the rows, at most

struct Q4W {
    int K, N, G;            // group: k of a group
    int KB, NT, NG;         // blocks along k, column tiles, groups along k (padded to whole blocks)
    bool zeros, sbf16;
    const uint4* codes;     // [NT][KB][64]
    const void* scale;      // [NT][NG][16] words of 4 (bf16 scales) or 8 bytes
};

static bool q4_make(const mamba_q4_weight* w, Q4W* o, size_t* bytes) {
    if (w == nullptr || w->d_in < 1 || w->d_out < 1 || w->d_in > (1 << 22) || w->d_out > (1 << 24)) return false;
    if (w->group != 32 && w->group != 64 && w->group != 128) return false;
    if (w->scale_dtype != MAMBA_F32 && w->scale_dtype != MAMBA_BF16) return false;
    Q4W q{};
    q.K = w->d_in; q.N = w->d_out; q.G = w->group;
    q.KB = ceil_div(q.K, kQ4K); q.NT = ceil_div(q.N, kQ4N); q.NG = q.KB * (kQ4K / q.G);
    q.zeros = w->has_zero != 0; q.sbf16 = w->scale_dtype == MAMBA_BF16;
    const size_t codes = (size_t)q.NT * q.KB * 1024;
    const char* base = static_cast<const char*>(w->packed);
    q.codes = reinterpret_cast<const uint4*>(base);
    q.scale = base + codes;
    *o = q;
    *bytes = codes + (size_t)q.NT * q.NG * kQ4N * (q.sbf16 ? 4 : 8);
    return true;
}

// A thread forms what four lanes of a block hold (run q of 8 k in each 32, four columns): a dword of
// codes a row, 16 bytes out a lane.  2560 x 50001 (196 MB) 44 us with its scales.
__global__ __launch_bounds__(256) void q4_pack(Q4W w, const uint8_t* codes, const void* scale, const uint8_t* zero, uint4* out, void* oscale) {
    const int64_t step = (int64_t)gridDim.x * 256, at0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int n4 = w.NT * (kQ4N / 4);
    for (int64_t i = at0; i < (int64_t)w.KB * 4 * n4; i += step) {
        const int n = (int)(i % n4) * 4, q = (int)(i / n4 & 3), here = w.N - n;
        const int64_t kb = i / n4 / 4;
        uint32_t v[4][4] = {};  // [column][dword]
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int64_t k = kb * kQ4K + 32 * st + 8 * q + e;
                uint32_t c = 0;
                if (k < w.K) {
                    const uint8_t* at = codes + k * w.N + n;
                    if (here >= 4) {
                        __builtin_memcpy(&c, at, 4);
                    } else {
                        for (int m = 0; m < here; ++m) c |= (uint32_t)at[m] << (8 * m);
                    }
                }
#pragma unroll
                for (int m = 0; m < 4; ++m) v[m][st] |= (c >> (8 * m) & 15u) << (4 * (e / 2 + 4 * (e & 1)));
            }
        uint4* to = out + (((int64_t)(n / kQ4N) * w.KB + kb) * 64 + q * 16 + n % kQ4N);
#pragma unroll
        for (int m = 0; m < 4; ++m) to[m] = make_uint4(v[m][0], v[m][1], v[m][2], v[m][3]);
    }
    const int groups = (w.K + w.G - 1) / w.G;
    for (int64_t i = at0; i < (int64_t)w.NT * w.NG * kQ4N; i += step) {
        const int col = (int)(i % 16), g = (int)(i / 16 % w.NG), n = (int)(i / 16 / w.NG) * kQ4N + col;
        const bool in = g < groups && n < w.N;
        const int64_t src = (int64_t)g * w.N + n;
        const int zp = in ? (zero ? zero[src] : 8) : 0;
        const float z = -16.f - (float)min(zp, 16);  // whole numbers to 32: bf16 holds them
        uint32_t sc = 0;
        if (in) sc = w.sbf16 ? (uint32_t)static_cast<const bf16_t*>(scale)[src] << 16 : __float_as_uint(static_cast<const float*>(scale)[src]);
        if (zp > 16) sc = 0x7fc00000u;
        if (w.sbf16) static_cast<uint32_t*>(oscale)[i] = sc | __float_as_uint(z) >> 16;
        else static_cast<float2*>(oscale)[i] = make_float2(__uint_as_float(sc), z);
    }
}

struct Q4P {
    Q4W w;
    int64_t rows;
    const void* x; int64_t x_ld;
    int K8;                 // elements of a row of x: a multiple of 8
    const float* xs;
    const float* bias;
    void* y; int64_t y_ld; bool ybf16;
};

typedef __bf16 q4_bf16x8 __attribute__((ext_vector_type(8)));
typedef float q4_f32x4 __attribute__((ext_vector_type(4)));
typedef int q4_i32x4 __attribute__((ext_vector_type(4)));

enum Q4X { Q4_BF16 = 0, Q4_F32 = 1, Q4_I8 = 2 };
// What lies beside the codes: bf16 scales alone, with zero points, f32 scales (with or without).
enum Q4S { Q4_S16 = 0, Q4_S16Z = 1, Q4_S32 = 2 };
constexpr uint32_t kQ4Out = 0x80000000u;  // a byte offset past every buffer's extent

// Lane l's operand of 32 k of 16 rows: row l % 16, k 8 (l / 16) .. + 7, loaded through a buffer
// resource (an offset past its extent reads zeros).  f32 rows are three bf16 parts, each the
// upper half of what the ones before leave (8 bits of the 24).
template <int X> struct Q4A;
template <> struct Q4A<Q4_BF16> {
    static constexpr int kParts = 1, kSize = 2;
    uint4 v;
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t soff) { v = buf_ld16(r, off, soff); }
    __device__ __forceinline__ q4_bf16x8 part(int) const { return __builtin_bit_cast(q4_bf16x8, v); }
};
template <> struct Q4A<Q4_F32> {
    static constexpr int kParts = 3, kSize = 4;
    uint4 v[2];
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t soff) {
        v[0] = buf_ld16(r, off, soff);
        v[1] = buf_ld16(r, off + 16, soff);
    }
    __device__ __forceinline__ q4_bf16x8 part(int k) const {
        const uint32_t u[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
        uint32_t d[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float r = __uint_as_float(u[i]);
#pragma unroll
            for (int j = 0; j < k; ++j) r -= __uint_as_float(__float_as_uint(r) & 0xffff0000u);
            const uint32_t h = __float_as_uint(r) >> 16;
            d[i / 2] = i & 1 ? d[i / 2] | h << 16 : h;
        }
        return __builtin_bit_cast(q4_bf16x8, d);
    }
};
template <> struct Q4A<Q4_I8> {
    static constexpr int kParts = 1, kSize = 1;
    uint2 v;
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t soff) {
        v = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(r, off, (int)__builtin_amdgcn_readfirstlane(soff), 0));
    }
    // in the order in which the codes' bytes come: 0 4 1 5 2 6 3 7
    __device__ __forceinline__ long part(int) const {
        return (long)((uint64_t)__builtin_amdgcn_perm(v.y, v.x, 0x07030602u) << 32 | __builtin_amdgcn_perm(v.y, v.x, 0x05010400u));
    }
};

// The codes of a dword, as operands.  A bf16 whose upper four bits of mantissa are the code
// is 16 + code: a shift and an and-or a pair (the mask in a vector register, for an instruction takes
// one scalar).  A byte whose upper four bits are code ^ 8 is 16 (code - 8).
__device__ __forceinline__ q4_bf16x8 q4_codes_bf16(uint32_t w) {
    uint32_t mask = 0x00780078u;
    asm("" : "+v"(mask));
    const uint32_t d[4] = {(w << 3 & mask) | 0x41804180u, (w >> 1 & mask) | 0x41804180u, (w >> 5 & mask) | 0x41804180u, (w >> 9 & mask) | 0x41804180u};
    return __builtin_bit_cast(q4_bf16x8, d);
}
__device__ __forceinline__ long q4_codes_i8x16(uint32_t w) {
    return (long)((uint64_t)((w & 0xf0f0f0f0u) ^ 0x80808080u) << 32 | ((w << 4 & 0xf0f0f0f0u) ^ 0x80808080u));
}
__device__ __forceinline__ long q4_codes_i8(uint32_t w) { return (long)((uint64_t)(w >> 4 & 0x0f0f0f0fu) << 32 | (w & 0x0f0f0f0fu)); }

// The rows' operands as the products take them, kept in registers: NP parts.
template <int X>
struct Q4Op {
    static constexpr int kParts = Q4A<X>::kParts;
    q4_bf16x8 v[kParts];
    __device__ __forceinline__ void make(const Q4A<X>& a) {
#pragma unroll
        for (int k = 0; k < kParts; ++k) v[k] = a.part(k);
    }
};
template <>
struct Q4Op<Q4_I8> {
    static constexpr int kParts = 1;
    long v[1];
    __device__ __forceinline__ void make(const Q4A<Q4_I8>& a) { v[0] = a.part(0); }
};

// Column tile j through buffer resources (scalar bases, 32-bit offsets).  A tile behind the last
// has no extent; whatever of the first tile's its loads bring, no result of it is stored.
struct Q4Tile {
    __amdgpu_buffer_rsrc_t codes, scale;
    __device__ __forceinline__ Q4Tile(const Q4W& q, int j) {
        const int64_t at = j < q.NT ? j : 0;
        const uint32_t kb = j < q.NT ? q.KB : 0, words = q.NG * kQ4N * (q.sbf16 ? 4 : 8);
        codes = buf_rsrc(q.codes + at * q.KB * 64, kb * 1024u);
        scale = buf_rsrc(static_cast<const char*>(q.scale) + at * words, kb ? words : 0u);
    }
};
// Block kb of KB, as the loads take it.  One behind the last reads zeros: that is told by the lane's own
// offset, past the extent, while the scalar one stays inside (how far that one is checked is not relied on).
struct Q4At {
    int kb;
    uint32_t out;
    __device__ __forceinline__ Q4At(int k, int KB) : kb(k < KB ? k : 0), out(k < KB ? 0u : kQ4Out) {}
};
// A block of a column tile: its codes, and its groups' scales and zero points.
template <int GB, int S>
struct Q4Block {
    uint4 w;
    uint32_t s[GB];
    uint32_t z[S == Q4_S32 ? GB : 1];
    __device__ __forceinline__ void load(const Q4Tile& t, const Q4At& at, int l) {
        constexpr int word = S == Q4_S32 ? 8 : 4;
        w = buf_ld16(t.codes, l * 16 + at.out, at.kb * 1024);
#pragma unroll
        for (int g = 0; g < GB; ++g) {
            const uint32_t off = (l & 15) * word + at.out + g * kQ4N * word;
            const int soff = at.kb * GB * kQ4N * word;
            if constexpr (S == Q4_S32) {
                const uint2 v = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(t.scale, off, soff, 0));
                s[g] = v.x;
                z[g] = v.y;
            } else {
                s[g] = __builtin_amdgcn_raw_buffer_load_b32(t.scale, off, soff, 0);
            }
        }
    }
    __device__ __forceinline__ float scale(int g) const { return __uint_as_float(S == Q4_S32 ? s[g] : s[g] & 0xffff0000u); }
    // -(16 + zero point), as two bf16
    __device__ __forceinline__ uint32_t minus2(int g) const {
        if constexpr (S == Q4_S16) return 0xc1c0c1c0u;  // -24
        else if constexpr (S == Q4_S16Z) return __builtin_amdgcn_perm(s[g], s[g], 0x01000100u);
        else return __builtin_amdgcn_perm(z[S == Q4_S32 ? g : 0], z[S == Q4_S32 ? g : 0], 0x03020302u);
    }
    // - zero point, as eight bytes
    __device__ __forceinline__ long minus8(int g) const {
        const uint32_t v = 16 + (int)__uint_as_float(S == Q4_S32 ? z[S == Q4_S32 ? g : 0] : s[g] << 16);
        const uint32_t b = __builtin_amdgcn_perm(v, v, 0u);
        return (long)((uint64_t)b << 32 | b);
    }
    __device__ __forceinline__ uint32_t dword(int st) const { return st == 0 ? w.x : st == 1 ? w.y : st == 2 ? w.z : w.w; }
};

// Group g of a block against RT row tiles, scaled and added to tot.
template <int X, int RT, int GB, int S>
__device__ __forceinline__ void q4_group(const Q4Block<GB, S>& b, int g, const Q4Op<X> (&x)[RT][4], q4_f32x4 (&tot)[RT]) {
    const float scale = b.scale(g);
    if constexpr (X == Q4_I8) {
        const long off = S == Q4_S16 ? 0 : b.minus8(g);
        q4_i32x4 acc[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) acc[i] = q4_i32x4{0, 0, 0, 0};
#pragma unroll
        for (int st = g * 4 / GB; st < (g + 1) * 4 / GB; ++st) {
            const long c = S == Q4_S16 ? q4_codes_i8x16(b.dword(st)) : q4_codes_i8(b.dword(st));
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                acc[i] = __builtin_amdgcn_mfma_i32_16x16x32_i8(x[i][st].v[0], c, acc[i], 0, 0, 0);
                if constexpr (S != Q4_S16) acc[i] = __builtin_amdgcn_mfma_i32_16x16x32_i8(x[i][st].v[0], off, acc[i], 0, 0, 0);
            }
        }
        // whole numbers of at most 128 x 128 x 128 < 2^24: exact up to the scale (a sixteenth of them is
        // taken with the row's scale)
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) tot[i][e] = __builtin_fmaf(scale, (float)acc[i][e], tot[i][e]);
    } else {
        const uint32_t z2 = b.minus2(g);
        const q4_bf16x8 off = __builtin_bit_cast(q4_bf16x8, make_uint4(z2, z2, z2, z2));
        q4_f32x4 acc[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) acc[i] = q4_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = g * 4 / GB; st < (g + 1) * 4 / GB; ++st) {
            const q4_bf16x8 c = q4_codes_bf16(b.dword(st));
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int k = Q4Op<X>::kParts - 1; k >= 0; --k) {  // the lowest part first
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i][st].v[k], c, acc[i], 0, 0, 0);
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i][st].v[k], off, acc[i], 0, 0, 0);
                }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) tot[i][e] = __builtin_fmaf(scale, acc[i][e], tot[i][e]);
    }
}

// The rows of a workgroup and where a lane's operands of them lie.
template <int X, int RT>
struct Q4Src {
    static constexpr int e = Q4A<X>::kSize;
    __amdgpu_buffer_rsrc_t r;
    uint32_t off[RT];
    int K8, KB, k8;
    __device__ __forceinline__ Q4Src(const Q4P& p, int64_t m0, int l) : K8(p.K8), KB(p.w.KB), k8(8 * (l >> 4)) {
        const int here = (int)min((int64_t)16 * RT, p.rows - m0), col = l & 15;  // an operand's row is the lane's low four bits, as a weight's column is
        r = buf_rsrc(static_cast<const char*>(p.x) + m0 * p.x_ld * e, (uint32_t)(((here - 1) * p.x_ld + p.K8) * e));
#pragma unroll
        for (int i = 0; i < RT; ++i) off[i] = 16 * i + col < here ? ((uint32_t)(16 * i + col) * (uint32_t)p.x_ld + k8) * e : kQ4Out;
    }
    // block kb; runs of 8 behind the rows' end, and blocks behind the last, read zeros
    __device__ __forceinline__ void load(Q4A<X> (&a)[RT][4], int kb) const {
        const int left = K8 - kb * kQ4K, soff = min(kb, KB - 1) * kQ4K * e;
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int i = 0; i < RT; ++i) a[i][st].load(r, (k8 + 32 * st < left ? off[i] : kQ4Out) + 32 * st * e, soff);
    }
};

// A column's bias, and the scales of a lane's four rows of each row tile (1 but for int8 rows): through
// buffer resources, 0 where there is none.
struct Q4Bias {
    __amdgpu_buffer_rsrc_t r;
    __device__ __forceinline__ explicit Q4Bias(const Q4P& p) : r(buf_rsrc(p.bias, p.bias ? (uint32_t)p.w.N * 4u : 0u)) {}
    __device__ __forceinline__ float at(int n) const { return buf_ld4(r, (uint32_t)n * 4u); }
};
template <int X, int RT>
struct Q4Scales {
    float v[RT][4];
    __device__ __forceinline__ Q4Scales(const Q4P& p, int64_t m0, int l, float by) {  // by a power of two
        const int here = (int)min((int64_t)16 * RT, p.rows - m0);
        const __amdgpu_buffer_rsrc_t r = buf_rsrc(p.xs + (X == Q4_I8 ? m0 : 0), X == Q4_I8 ? here * 4u : 0u);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = X == Q4_I8 ? buf_ld4(r, (16 * i + 4 * (l >> 4) + e) * 4) * by : 1.f;
    }
};

// The sums of a row tile (the lane's column and four of its rows) as results.
template <int X>
__device__ __forceinline__ void q4_store(const Q4P& p, int64_t m0, int n, const q4_f32x4& s, const float (&xs)[4], float bias) {
    if (n >= p.w.N) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int64_t m = m0 + e;
        if (m >= p.rows) continue;
        const float v = X == Q4_I8 ? __builtin_fmaf(s[e], xs[e], bias) : s[e] + bias;
        if (p.ybf16) store_f32<bf16_t>(static_cast<bf16_t*>(p.y) + m * p.y_ld + n, v);
        else static_cast<float*>(p.y)[m * p.y_ld + n] = v;
    }
}

// The rows in registers: wave w holds the operands of RT row tiles of 16 for NK blocks of k, and
// the workgroup's waves all of k.  It takes column tiles in turn; a block's registers are loaded for
// the next tile as soon as this one's are used.  The waves' sums meet in LDS, in the order of k, in
// two places by turns, so that a tile has one barrier.
template <int X, int RT, int NK, int GB, int S>
__global__ __launch_bounds__(64 * (RT > 1 ? 8 : kQ4Waves)) void q4_held(Q4P p) {
    extern __shared__ __align__(16) q4_f32x4 q4_red[];  // [2][RT][waves][64]
    const int nw = blockDim.x >> 6, w = wave_id(), l = threadIdx.x & 63;
    const int64_t m0 = (int64_t)blockIdx.y * (16 * RT);
    const int kb0 = w * NK;
    // No load has a branch of its own, behind which the compiler would wait for every load in
    // flight; for the same reason the rows are waited for before the tiles' loop, and the blocks are
    // loaded in the order of their use before it as in it.
    const Q4Src<X, RT> src(p, m0, l);
    Q4A<X> a[NK][RT][4];
#pragma unroll
    for (int k = 0; k < NK; ++k) src.load(a[k], kb0 + k);
    __builtin_amdgcn_sched_barrier(0);
    Q4Block<GB, S> b[NK];
    {
        const Q4Tile t(p.w, blockIdx.x);
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            b[k].load(t, Q4At(kb0 + k, p.w.KB), l);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    Q4Op<X> x[NK][RT][4];
#pragma unroll
    for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                x[k][i][st].make(a[k][i][st]);
#pragma unroll
                for (int e = 0; e < Q4Op<X>::kParts; ++e) asm volatile("" : "+v"(x[k][i][st].v[e]));
            }
    const Q4Bias bias(p);
    Q4Scales<X, RT> xs(p, m0, l, S == Q4_S16 ? 0.0625f : 1.f);
    if constexpr (X == Q4_I8) {
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) asm volatile("" : "+v"(xs.v[i][e]));
    }
    int turn = 0;
    for (int j = blockIdx.x; j < p.w.NT; j += gridDim.x, ++turn) {
        const Q4Tile next(p.w, j + gridDim.x);
        const float add = bias.at(j * kQ4N + (l & 15));
        q4_f32x4 tot[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) tot[i] = q4_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NK; ++k) {
#pragma unroll
            for (int g = 0; g < GB; ++g) q4_group<X, RT, GB, S>(b[k], g, x[k], tot);
            // behind the block's last use, so that its registers are these
            __builtin_amdgcn_sched_barrier(0);
            b[k].load(next, Q4At(kb0 + k, p.w.KB), l);
            __builtin_amdgcn_sched_barrier(0);
        }
        q4_f32x4* red = q4_red + (turn & 1) * RT * nw * 64;
#pragma unroll
        for (int i = 0; i < RT; ++i) red[(i * nw + w) * 64 + l] = tot[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            if (w != (turn * RT + i) % nw) continue;
            q4_f32x4 s = red[i * nw * 64 + l];
            for (int k = 1; k < nw; ++k) s += red[(i * nw + k) * 64 + l];
            q4_store<X>(p, m0 + 16 * i + 4 * (l >> 4), j * kQ4N + (l & 15), s, xs.v[i], add);
        }
    }
}

// Any k: RT row tiles with C column tiles, a wave walks a stretch of k with two blocks of codes and
// one of rows in flight.
template <int X, int RT, int C, int GB, int S>
__global__ __launch_bounds__(512) void q4_walk(Q4P p) {
    extern __shared__ __align__(16) q4_f32x4 q4_red[];  // [waves][RT][C][64]
    const int nw = blockDim.x >> 6, w = wave_id(), l = threadIdx.x & 63;
    const int j0 = blockIdx.x * C;
    const int64_t m0 = (int64_t)blockIdx.y * (16 * RT);
    const int per = (p.w.KB + nw - 1) / nw, kb0 = min(p.w.KB, w * per), kb1 = min(p.w.KB, kb0 + per);
    const Q4Src<X, RT> src(p, m0, l);
    q4_f32x4 tot[C][RT];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < RT; ++i) tot[c][i] = q4_f32x4{0.f, 0.f, 0.f, 0.f};
    Q4Block<GB, S> b[2][C];
    Q4A<X> a[RT][4];
    Q4Tile tile[C] = {Q4Tile(p.w, j0), Q4Tile(p.w, j0 + 1)};
    static_assert(C == 2, "two tiles");
    auto codes = [&](int q, int kb) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < C; ++c) b[q][c].load(tile[c], Q4At(kb, p.w.KB), l);
    };
    const int stop = p.w.KB;
    codes(0, kb0);
    src.load(a, kb0 < kb1 ? kb0 : stop);
    codes(1, kb0 + 1);
    for (int kb = kb0; kb < kb1; kb += 2) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            Q4Op<X> x[RT][4];
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int st = 0; st < 4; ++st) x[i][st].make(a[i][st]);
            src.load(a, kb + q + 1 < kb1 ? kb + q + 1 : stop);
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int g = 0; g < GB; ++g) q4_group<X, RT, GB, S>(b[q][c], g, x, tot[c]);
            __builtin_amdgcn_sched_barrier(0);
            codes(q, kb + q + 2);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int c = 0; c < C; ++c) q4_red[((w * RT + i) * C + c) * 64 + l] = tot[c][i];
    __syncthreads();
    const Q4Bias bias(p);
    const Q4Scales<X, RT> xs(p, m0, l, S == Q4_S16 ? 0.0625f : 1.f);
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if ((i * C + c) % nw != w) continue;  // one wave a tile
            q4_f32x4 s = q4_red[(i * C + c) * 64 + l];
            for (int k = 1; k < nw; ++k) s += q4_red[((k * RT + i) * C + c) * 64 + l];
            const int n = (j0 + c) * kQ4N + (l & 15);
            q4_store<X>(p, m0 + 16 * i + 4 * (l >> 4), n, s, xs.v[i], bias.at(n));
        }
}

// Rows of a width that is no multiple of 8 (or too far apart for the buffer's offsets), copied with
// zeros behind them.
template <typename T>
__global__ __launch_bounds__(256) void q4_pad(const T* x, int64_t ld, int64_t rows, int K, int K8, T* out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * K8; i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / K8;
        const int k = (int)(i - m * K8);
        out[i] = k < K ? x[m * ld + k] : T(0);
    }
}

template <int X, int RT, int NK, int GB>
static void q4_held_launch(const Q4P& p, int nw, hipStream_t s) {
    const int by = (int)((p.rows + 16 * RT - 1) / (16 * RT));
    // the chip full once: two workgroups of four waves a CU, or one
    const dim3 grid(std::min(p.w.NT, std::max(8, (nw == 4 ? 512 : 256) / by)), by), block(64 * nw);
    const size_t lds = (size_t)2 * RT * nw * 64 * 16;
    if (!p.w.sbf16) hipLaunchKernelGGL((q4_held<X, RT, NK, GB, Q4_S32>), grid, block, lds, s, p);
    else if (p.w.zeros) hipLaunchKernelGGL((q4_held<X, RT, NK, GB, Q4_S16Z>), grid, block, lds, s, p);
    else hipLaunchKernelGGL((q4_held<X, RT, NK, GB, Q4_S16>), grid, block, lds, s, p);
}
template <int X, int RT, int C, int GB>
static void q4_walk_launch(const Q4P& p, hipStream_t s) {
    // Some 2048 waves in all, each with two blocks at least.  us at 1024 / 2048 / 4096: one bf16 row of 10240 x
    // 10240 22.2 / 23.8 / 23.8, x 20480 28.8 / 28.6 / 34.4; one f32 row of 5120 x 10240 31.0 / 37.7 / 37.8, x 20480
    // 44.5 / 44.4 / 55; four bf16 rows of 10240 x 2560 13.0.
    int nw = 4;
    while (nw < 8 && (int64_t)p.w.NT * nw < 2048 * C && p.w.KB >= 4 * nw) nw *= 2;
    const dim3 grid(ceil_div(p.w.NT, C), (uint32_t)((p.rows + 16 * RT - 1) / (16 * RT))), block(64 * nw);
    const size_t lds = (size_t)nw * RT * C * 64 * 16;
    if (!p.w.sbf16) hipLaunchKernelGGL((q4_walk<X, RT, C, GB, Q4_S32>), grid, block, lds, s, p);
    else if (p.w.zeros) hipLaunchKernelGGL((q4_walk<X, RT, C, GB, Q4_S16Z>), grid, block, lds, s, p);
    else hipLaunchKernelGGL((q4_walk<X, RT, C, GB, Q4_S16>), grid, block, lds, s, p);
}
// The rows in registers wherever twelve waves hold them (60 blocks of k, f32 24), as four, eight or
// twelve waves, which load the four SIMDs evenly; else the walk.  us held / walked, bf16 at 2560 x 10240:
// one row 5.3 / 11.1, 32 rows 11.4 / 17.5, 64 rows 14.8 / 24.8, 256 rows 34 / 78; int8 64 rows 13.7 / 22.8,
// at 5120 x 2560 11.0 / 14.9; f32 one row 9.0 / 26.3.
// Two row tiles a wave take apart a block once for both, but start with twice the rows to load: where
// a workgroup has ten tiles or more to go through.  us with one / two at 2560 x 10240: bf16 64 rows
// (5 tiles) 14.8 / 17.2, 128 rows (10) 23.2 / 22.4, 256 rows (20) 39.3 / 34.2, int8 33.5 / 29.0; bf16
// 64 rows at 2560 x 50001 (24) 46.7 / 40.6.
template <int X, int GB>
static void q4_shape(const Q4P& p, hipStream_t s) {
    constexpr int most = X == Q4_F32 ? 2 : 5;  // blocks of k whose operands a wave's registers hold
    const int nw = p.w.KB <= 4 * most ? 4 : p.w.KB <= 8 * most ? 8 : 12, NK = ceil_div(p.w.KB, nw);
    if (NK > most) return q4_walk_launch<X, 2, 2, GB>(p, s);
    if constexpr (X == Q4_F32) {
        q4_held_launch<X, 1, 2, GB>(p, nw, s);
    } else if (nw < kQ4Waves && p.rows > 16 && ((p.rows + 15) / 16) * p.w.NT >= 5120) {
        if (NK <= 2) q4_held_launch<X, 2, 2, GB>(p, nw, s);
        else if (NK == 3) q4_held_launch<X, 2, 3, GB>(p, nw, s);
        else if (NK == 4) q4_held_launch<X, 2, 4, GB>(p, nw, s);
        else q4_held_launch<X, 2, 5, GB>(p, nw, s);
    } else {
        if (NK <= 2) q4_held_launch<X, 1, 2, GB>(p, nw, s);
        else if (NK == 3) q4_held_launch<X, 1, 3, GB>(p, nw, s);
        else if (NK == 4) q4_held_launch<X, 1, 4, GB>(p, nw, s);
        else q4_held_launch<X, 1, 5, GB>(p, nw, s);
    }
}
template <int X>
static void q4_dispatch(const Q4P& p, hipStream_t s) {
    if (p.w.G == 128) q4_shape<X, 1>(p, s);
    else if (p.w.G == 64) q4_shape<X, 2>(p, s);
    else q4_shape<X, 4>(p, s);
}
// Rows that are read in place: whole runs of 8, and 64 of them within a buffer's offsets.
static bool q4_in_place(const Q4P& p, int size) { return p.K8 == p.w.K && p.x_ld >= 0 && (63 * p.x_ld + p.K8) * size < (1ll << 31); }

}  // namespace mamba

using namespace mamba;

#define Q4_SHAPE "d_in in [1, 2^22], d_out in [1, 2^24], group 32, 64 or 128 and scales of f32 or bf16 required"

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
    const int64_t items = (int64_t)q.NT * q.KB * 16;
    hipLaunchKernelGGL(q4_pack, dim3((uint32_t)std::min<int64_t>((items + 255) / 256, 1 << 16)), dim3(256), 0, (hipStream_t)stream, q, (const uint8_t*)codes,
                       scale, (const uint8_t*)zero, (uint4*)packed, const_cast<void*>(q.scale));
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
    p.K8 = (p.w.K + 7) / 8 * 8;
    MAMBA_CHECK_ARG((p.rows + 15) / 16 <= 65535, "rows must be at most 1048560");
    *out = p;
    return MAMBA_OK;
}
static int q4_xsize(int x_dtype) { return x_dtype == MAMBA_F32 ? 4 : x_dtype == MAMBA_BF16 ? 2 : 1; }

extern "C" size_t mamba_linear_q4_workspace_size(const mamba_linear_q4_args* a) {
    Q4P p;
    if (q4_check(a, &p) != MAMBA_OK) return 0;
    return q4_in_place(p, q4_xsize(a->x_dtype)) ? 0 : (size_t)p.rows * p.K8 * q4_xsize(a->x_dtype);
}

extern "C" int mamba_linear_q4_fwd(const mamba_linear_q4_args* a, void* ws, size_t ws_bytes, mamba_stream_t stream) {
    Q4P p;
    int st = q4_check(a, &p);
    if (st != MAMBA_OK) return st;
    if (p.rows == 0) return MAMBA_OK;
    MAMBA_CHECK_ARG(a->w.packed && p.x && p.y, "packed, x and y are required");
    MAMBA_CHECK_ARG(((uintptr_t)a->w.packed & 15u) == 0, "packed must be 16-byte aligned");
    MAMBA_CHECK_ARG(p.y_ld >= p.w.N || p.rows == 1, "rows of y overlap");
    const size_t ex = q4_xsize(a->x_dtype), ey = p.ybf16 ? 2 : 4;
    const char *px = static_cast<const char*>(p.x), *py = static_cast<const char*>(p.y);
    const bool apart = py + ((p.rows - 1) * p.y_ld + p.w.N) * ey <= px || px + ((p.rows - 1) * p.x_ld + p.w.K) * ex <= py;
    MAMBA_CHECK_ARG(apart || (ex == ey && !rows_clash(p.y, p.y_ld, p.x, p.x_ld, p.w.N, p.w.K, p.rows, ex, false)), "y overlaps x");
    hipStream_t s = (hipStream_t)stream;
    const size_t need = mamba_linear_q4_workspace_size(a);
    MAMBA_CHECK_ARG(((uintptr_t)ws & 15u) == 0, "the workspace must be 16-byte aligned");
    if (need && (ws == nullptr || ws_bytes < need)) {
        set_error("mamba_linear_q4_fwd: workspace missing or too small");
        return MAMBA_ERR_WORKSPACE;
    }
    if (need) {
        const dim3 grid((uint32_t)std::min<int64_t>((p.rows * p.K8 + 255) / 256, 4096));
        if (ex == 4) hipLaunchKernelGGL(q4_pad<uint32_t>, grid, dim3(256), 0, s, (const uint32_t*)p.x, p.x_ld, p.rows, p.w.K, p.K8, (uint32_t*)ws);
        else if (ex == 2) hipLaunchKernelGGL(q4_pad<uint16_t>, grid, dim3(256), 0, s, (const uint16_t*)p.x, p.x_ld, p.rows, p.w.K, p.K8, (uint16_t*)ws);
        else hipLaunchKernelGGL(q4_pad<uint8_t>, grid, dim3(256), 0, s, (const uint8_t*)p.x, p.x_ld, p.rows, p.w.K, p.K8, (uint8_t*)ws);
        MAMBA_CHECK_LAUNCH();
        p.x = ws;
        p.x_ld = p.K8;
    }
    if (a->x_dtype == MAMBA_F32) q4_dispatch<Q4_F32>(p, s);
    else if (a->x_dtype == MAMBA_BF16) q4_dispatch<Q4_BF16>(p, s);
    else q4_dispatch<Q4_I8>(p, s);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}
