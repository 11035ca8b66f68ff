// Mamba-1 selective scan over packed sequences for gfx950: forward, backward, and
// single tokens on a cache addressed by slot.  f32 or bf16 rows (channels
// contiguous), f32 states, A, D, bias and their gradients.
//
//   d = softplus(delta + bias),  a_t = exp(d_t A),  h_t = a_t h_{t-1} + d_t u_t B_t,
//   pre_t = sum_n C_t h_t + D u_t,  y_t = pre_t silu(z_t)
// Backward, with e_t = dy_t silu(z_t) and g_t = C_t e_t + a_{t+1} g_{t+1}:
//   s_t = sum_n g B,  du = d s + D e,  dd = sum_n g a h_{t-1} A + u s,  ddelta = dd sigmoid(delta + bias),
//   dz = dy pre silu'(z),  dB_n = sum_d g d u,  dC_n = sum_d h e,  dA = sum_t g a h_{t-1} d,
//   dD = sum_t e u,  dbias = sum_t ddelta,  dh_0 = a_1 g_1
//
// Each (channel, state) pair decays at its own rate, so there is no matrix
// product: one exp (a quarter-rate instruction) and four multiplies and fmas per
// state and token bound the forward, about four times that the backward.
//
// Rows are cut into chunks of equal length without regard to the sequences, so
// that a batch of unequal ones loads the chip evenly.  A sequence that crosses a
// chunk's end is carried: scan_pk_state finds the state a chunk leaves behind
// when it starts from zero (or from the sequence's own start) and the sum of d
// over it, a walk over the chunks, h <- exp(A sum d) h + own, finds what comes into each
// (in scan_pk_out, or for many chunks in scan_pk_carry), and scan_pk_out scans again
// from there.  Where the sequences are many and the longest
// is known to be short, scan_pk_out takes whole sequences instead and nothing is
// carried.
//
// Backward: scan_pk_state_bwd finds both carries of a chunk on one set of exps
// (the gradient of the state that enters it is sum_t P_t C_t e_t, P_t the product
// of the decays up to row t, so it walks forwards too) and keeps the state at
// every 8th row; scan_pk_bwd then takes 8 rows at a time from the last (fewer than 8
// at a part's end one by one) to the first, finds their states and decays again in registers and walks back over
// them.  dB and dC are sums over channels: over a wave's by lane exchanges, over
// the workgroup's in LDS, over the workgroups in scan_pk_join; every sum is in a
// fixed order.
//
// A workgroup of 256 threads holds CPB = 1024 / NP channels, NP = the states
// padded to 8, 16, 32 or 64; a channel is spread over NS = NP / 4 lanes with 4 states
// each.  Tiles of 16 rows (8 for NP = 8) are staged through LDS as f32 with the element-wise
// work (softplus, d u, the gate) done once per element; rows past a tile's end
// and channels past D are staged as zeros, which are steps that change nothing.
// The next tile's rows are loaded while a tile is scanned.
//
// Measured at 8192 rows x 5120 channels, 16 states, bf16, six sequences (us, then
// the share of cycles that the vector units issue in; HBM moves what each reads and
// writes in a fraction of its time): state pass 114, all of them; out 183, 0.98;
// backward state pass 212, all; backward 596, 0.85; the join 20.6.  Their bytes alone
// would take 32, 71, 139 and 213 us at the rate of a copy.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "pack.h"

namespace mamba {

constexpr float kLog2e = 1.4426950408889634f;

struct ScanPk {
    Seqs q;
    int64_t rows;
    int D, N;
    bool softplus, fill;
    const void* u; int64_t u_st;
    const void* dl; int64_t dl_st;
    const void* z; int64_t z_st;
    const void* B; int64_t B_st;
    const void* C; int64_t C_st;
    const float* A; const float* Dv; const float* bias;
    void* y; int64_t y_st;
    float* state; int64_t nslots; const int32_t* slots;
    int chunk, nchunk;
    bool walk;                      // chunks find what comes into them by themselves
    bool whole;                     // a workgroup takes a sequence: nchunk = the sequences
    // per chunk: what it leaves behind [nchunk][D][NP] (then, carried, what
    // leaves it), the sum of d [nchunk][D], and the state that its last sequence
    // began from [nchunk][D][NP] (the cache's slot may be written meanwhile)
    float* E; float* sumd; float* h0c;
    int32_t* ends;                  // per chunk: kIn | kOut | kThrough
    // backward
    const void* dy; int64_t dy_st;
    const float* h0; const float* dhT;
    float* G;                       // [nchunk][D][NP]: gradient of the state that enters a chunk
    float* ckh; float* ckd;         // [rows / kSub + 1][D][NP], [rows / kSub + 1][D]: the state at every
                                    // kSub rows of a sequence's part of a chunk, from zero, and sum of d
    float* pA; float* pD; float* pb;  // [nchunk][D][NP], [nchunk][D] x 2: partial dA, dD, dbias
    float* pBC;                     // [channel blocks][rows][2][NP]: partial dB, dC
    void* du; int64_t du_st;
    void* ddl; int64_t ddl_st;
    void* dz; int64_t dz_st;
    void* dB; int64_t dB_st;
    void* dC; int64_t dC_st;
    float* dA; float* dD; float* db; float* dh0;
};

// softplus(x) = log(1 + e^x), x itself above 20 (equal in f32); log1p through the
// hardware log with Goldberg's correction, log(v) e / (v - 1) for v = 1 + e.  The
// hardware's exp2, log2 and reciprocal as they are (1 <= v, and an e below the normal
// floats is 0): the library's cases for the smallest floats cost as much again.
// Without a branch, which would part the elements in the schedule.  The minimum of a
// NaN and 20 is 20, so the last select asks for x <= 20: what fails it is x itself.
__device__ __forceinline__ float pk_softplus(float x) {
    const float e = __builtin_amdgcn_exp2f(fminf(x, 20.f) * kLog2e);
    const float v = 1.f + e;
    const float l = __builtin_amdgcn_logf(v) * (1.f / kLog2e) * (e * __builtin_amdgcn_rcpf(v - 1.f));
    return x <= 20.f ? (v == 1.f ? e : l) : x;
}
__device__ __forceinline__ float pk_sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -kLog2e));
}

template <int CTRL>
__device__ __forceinline__ float pk_dpp(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
// Sum over aligned groups of NS lanes, in every lane: xor 1, xor 2 inside quads,
// then the mirrors of half rows and rows.
template <int NS>
__device__ __forceinline__ float group_sum_all(float v) {
    static_assert(NS == 2 || NS == 4 || NS == 8 || NS == 16, "2, 4, 8 or 16 lanes");
    v += pk_dpp<0xB1>(v);
    if (NS >= 4) v += pk_dpp<0x4E>(v);
    if (NS >= 8) v += pk_dpp<0x141>(v);
    if (NS >= 16) v += pk_dpp<0x140>(v);
    return v;
}

constexpr int kTile = 16;  // rows of a chunk come in multiples of this

// NS lanes a channel, CPB channels a workgroup, tiles of TT rows, EV elements a thread
template <int NP>
struct ScanShape {
    static constexpr int NS = NP / 4, CPB = 256 / NS, TT = NP == 8 ? 8 : kTile, EV = TT * CPB / 256;
};

// The element-wise mapping: row tid / (CPB / EV) of the tile, EV channels from
// EV (tid % (CPB / EV)); with A, u and e = 0 the states of channels past D stay 0
// (and B and C, in scan_pk_bwd), so that sums over a wave's channels need no mask.
template <int NP>
struct ElemMap {
    int row, ch;
    __device__ __forceinline__ ElemMap() {
        constexpr int W = ScanShape<NP>::CPB / ScanShape<NP>::EV;
        row = threadIdx.x / W;
        ch = ScanShape<NP>::EV * (threadIdx.x % W);
    }
};

// B or C of a tile: element i = tid + 256 k of [TT rows][NP states]
template <typename T, int NP>
struct BcTile {
    static constexpr int TT = ScanShape<NP>::TT, K = (TT * NP + 255) / 256;
    T v[K];
    __device__ __forceinline__ void load(const void* src, int64_t st, int t0, int n, int N) {
        const T* base = static_cast<const T*>(src) + t0 * st;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = threadIdx.x + 256 * k, r = i / NP, c = i % NP;
            v[k] = r < n && c < N ? base[(uint32_t)(r * (int)st + c)] : (T)0;
        }
    }
    __device__ __forceinline__ void stage(float (*dst)[NP]) const {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = threadIdx.x + 256 * k;
            if (TT * NP % 256 == 0 || i < TT * NP) dst[i / NP][i % NP] = load_f32<T>(&v[k]);
        }
    }
};

enum { kIn = 1, kOut = 2, kThrough = 4 };

// What chunk ck does at its two ends: the sequence that crosses into it and the
// one that crosses out of it (-1: none).
struct ChunkEnds {
    int c0, c1;
    int first, last;   // first sequence with rows in the chunk, and the one that crosses c1
    bool in, through;  // the first one began before c0; it fills the chunk and goes on
    __device__ __forceinline__ ChunkEnds(const ScanPk& p, int64_t ck) {
        if (p.whole) {
            first = (int)ck;
            c0 = p.q.begin(first);
            c1 = p.q.end(first);
            in = through = false;
            last = -1;
            return;
        }
        c0 = (int)(ck * p.chunk);
        c1 = min((int)p.rows, c0 + p.chunk);
        first = p.q.after(c0);
        in = first < p.q.n && p.q.begin(first) < c0;
        last = -1;
        if (c1 < p.rows) {
            const int s = p.q.after(c1);
            if (s < p.q.n && p.q.begin(s) < c1) last = s;
        }
        through = in && last == first;
    }
    __device__ __forceinline__ int flags() const { return (in ? kIn : 0) | (last >= 0 ? kOut : 0) | (through ? kThrough : 0); }
};

template <int NP>
__device__ __forceinline__ void load_A2(const ScanPk& p, int d, int ng, float (&A2)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int n = 4 * ng + k;
        A2[k] = d < p.D && n < p.N ? p.A[(int64_t)d * p.N + n] * kLog2e : 0.f;
    }
}

// 4 states of a [., D, N] tensor's row
__device__ __forceinline__ void load_state(const float* base, int64_t row, const ScanPk& p, int d, int ng, float (&h)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int n = 4 * ng + k;
        h[k] = base && row >= 0 && d < p.D && n < p.N ? base[(row * p.D + d) * p.N + n] : 0.f;
    }
}
__device__ __forceinline__ void store_state(float* base, int64_t row, const ScanPk& p, int d, int ng, const float (&h)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int n = 4 * ng + k;
        if (base && row >= 0 && d < p.D && n < p.N) base[(row * p.D + d) * p.N + n] = h[k];
    }
}
template <int NP>
__device__ __forceinline__ float4* plane(float* base, int64_t ck, const ScanPk& p, int d, int ng) {
    return reinterpret_cast<float4*>(base + ((ck * p.D + d) * (int64_t)NP + 4 * ng));
}
template <int NP>
__device__ __forceinline__ void load_plane(float* base, int64_t ck, const ScanPk& p, int d, int ng, float (&h)[4]) {
    const float4 v = d < p.D ? *plane<NP>(base, ck, p, d, ng) : make_float4(0.f, 0.f, 0.f, 0.f);
    h[0] = v.x; h[1] = v.y; h[2] = v.z; h[3] = v.w;
}
template <int NP>
__device__ __forceinline__ void store_plane(float* base, int64_t ck, const ScanPk& p, int d, int ng, const float (&h)[4]) {
    if (d < p.D) *plane<NP>(base, ck, p, d, ng) = make_float4(h[0], h[1], h[2], h[3]);
}

// What comes into a chunk over the chunks of its sequence before it (or, for a
// gradient, behind it): X[from], then X[j] + exp(A sum d of j) times what came so far,
// to chunk `to`.  With the carries already walked (p.walk false), X[to] itself.
template <int NP>
__device__ __forceinline__ void load_carry(float* X, int from, int to, const ScanPk& p, int d, int ng, const float (&A2)[4], float (&h)[4]) {
    constexpr int kAhead = 4;
    if (!p.walk) from = to;
    const int step = to >= from ? 1 : -1, count = (to - from) * step;
    load_plane<NP>(X, from, p, d, ng, h);
    for (int j = 1; j <= count; j += kAhead) {
        float own[kAhead][4], sd[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int ck = from + min(j + i, count) * step;
            load_plane<NP>(X, ck, p, d, ng, own[i]);
            sd[i] = d < p.D ? p.sumd[(int64_t)ck * p.D + d] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (j + i > count) break;
#pragma unroll
            for (int k = 0; k < 4; ++k) h[k] = __builtin_fmaf(__builtin_amdgcn_exp2f(sd[i] * A2[k]), h[k], own[i][k]);
        }
    }
}

// The state that chunk ck leaves to the next, from zero or from its last sequence's own
// start, and the sum of d.  Four rows' operands are read from LDS before the four
// dependent steps.  114 us at 8192 x 5120 bf16: 52 M wave instructions, of which 10.5 M
// exps at about four times a multiply's time, leave the vector units no idle cycle.
template <typename T, int NP>
__global__ __launch_bounds__(256) void scan_pk_state(ScanPk p) {
    constexpr int NS = ScanShape<NP>::NS, CPB = ScanShape<NP>::CPB, EV = ScanShape<NP>::EV, TT = ScanShape<NP>::TT;
    __shared__ float2 s_dd[TT][CPB];
    __shared__ __align__(16) float s_B[TT][NP];
    const int nblk = (p.D + CPB - 1) / CPB;
    const int ck = (int)(blockIdx.x / (uint32_t)nblk);
    const int d0 = (int)(blockIdx.x % (uint32_t)nblk) * CPB;
    const ChunkEnds e(p, ck);
    if (d0 == 0 && threadIdx.x == 0) p.ends[ck] = e.flags();
    if (e.last < 0) return;  // nothing crosses its end
    const ElemMap<NP> m;
    // this thread's place in a tile (32 bits, beside a scalar base)
    auto at = [&](int64_t st) { return (uint32_t)(m.row * (int)st + m.ch); };
    const int c = threadIdx.x / NS, ng = threadIdx.x % NS, d = d0 + c;
    const int nc = p.D - (d0 + m.ch);
    float A2[4], h[4] = {0.f, 0.f, 0.f, 0.f}, sumd = 0.f, bias[EV];
    load_A2<NP>(p, d, ng, A2);
#pragma unroll
    for (int k = 0; k < EV; ++k) bias[k] = p.bias && k < nc ? p.bias[d0 + m.ch + k] : 0.f;
    const int st = p.q.begin(e.last), a = max(st, e.c0);
    if (st >= e.c0 && p.state) {
        load_state(p.state, slot_of(p.slots, e.last, p.nslots), p, d, ng, h);
        store_plane<NP>(p.h0c, ck, p, d, ng, h);
    }
    Elems<T, EV> ru, rd;
    BcTile<T, NP> rB;
    auto fetch = [&](int t0) {
        const int n = min(TT, e.c1 - t0);
        if (m.row < n && nc >= EV) {
            ru.load(static_cast<const T*>(p.u) + (t0 * p.u_st + d0) + at(p.u_st));
            rd.load(static_cast<const T*>(p.dl) + (t0 * p.dl_st + d0) + at(p.dl_st));
        } else {
            const int q = m.row < n ? nc : 0;
            ru.load_part(static_cast<const T*>(p.u) + (t0 * p.u_st + d0) + at(p.u_st), q);
            rd.load_part(static_cast<const T*>(p.dl) + (t0 * p.dl_st + d0) + at(p.dl_st), q);
        }
        rB.load(p.B, p.B_st, t0, n, p.N);
    };
    fetch(a);
    for (int t0 = a; t0 < e.c1; t0 += TT) {
        const int n = min(TT, e.c1 - t0);
        float uv[EV], dv[EV];
        ru.get(uv);
        rd.get(dv);
#pragma unroll
        for (int k = 0; k < EV; ++k) dv[k] += bias[k];
        if (p.softplus) {
#pragma unroll
            for (int k = 0; k < EV; ++k) dv[k] = pk_softplus(dv[k]);
        }
#pragma unroll
        for (int k = 0; k < EV; ++k) {
            if (m.row >= n) dv[k] = 0.f;
            s_dd[m.row][m.ch + k] = make_float2(dv[k], dv[k] * uv[k]);
        }
        rB.stage(s_B);
        __syncthreads();
        if (t0 + TT < e.c1) fetch(t0 + TT);
#pragma unroll 1
        for (int t = 0; t < n; t += 4) {
            float2 dd[4];
            float4 bv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                dd[i] = s_dd[t + i][c];
                bv[i] = *(const float4*)&s_B[t + i][4 * ng];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sumd += dd[i].x;
                h[0] = __builtin_fmaf(h[0], __builtin_amdgcn_exp2f(dd[i].x * A2[0]), dd[i].y * bv[i].x);
                h[1] = __builtin_fmaf(h[1], __builtin_amdgcn_exp2f(dd[i].x * A2[1]), dd[i].y * bv[i].y);
                h[2] = __builtin_fmaf(h[2], __builtin_amdgcn_exp2f(dd[i].x * A2[2]), dd[i].y * bv[i].z);
                h[3] = __builtin_fmaf(h[3], __builtin_amdgcn_exp2f(dd[i].x * A2[3]), dd[i].y * bv[i].w);
            }
        }
        __syncthreads();
    }
    store_plane<NP>(p.E, ck, p, d, ng, h);
    if (d < p.D && ng == 0) p.sumd[(int64_t)ck * p.D + d] = sumd;
}

// A thread per (channel, state) walks the chunks: E[ck] <- the state that leaves
// chunk ck, or (BACK, from the last) G[ck] <- the gradient of the state that
// enters it.  kAhead chunks' values are loaded at a time: the walk is one round of
// memory latency per 16 chunks (11 us for 32 chunks x 5120 x 16, 14 backward).
template <int NP, bool BACK>
__device__ __forceinline__ void carry_walk(const ScanPk& p, int i) {
    constexpr int kAhead = 16;
    const int d = i / NP, n = i % NP;
    if (d >= p.D) return;
    const float A2 = n < p.N ? p.A[(int64_t)d * p.N + n] * kLog2e : 0.f;
    float* X = (BACK ? p.G : p.E) + (int64_t)d * NP + n;
    const int64_t pitch = (int64_t)p.D * NP, steps = p.nchunk - 1;
    const int have = BACK ? kIn : kOut;
    float v = 0.f;
    for (int64_t j = 0; j < steps; j += kAhead) {
        float own[kAhead], sd[kAhead];
        int f[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int64_t ck = BACK ? p.nchunk - 1 - (j + k) : j + k;
            f[k] = j + k < steps ? p.ends[ck] : 0;
            own[k] = f[k] & have ? X[ck * pitch] : 0.f;
            sd[k] = f[k] & kThrough ? p.sumd[ck * p.D + d] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int64_t ck = BACK ? p.nchunk - 1 - (j + k) : j + k;
            if (!(f[k] & have)) continue;
            v = f[k] & kThrough ? __builtin_fmaf(__builtin_amdgcn_exp2f(sd[k] * A2), v, own[k]) : own[k];
            X[ck * pitch] = v;
        }
    }
}

template <int NP>
__global__ __launch_bounds__(64) void scan_pk_carry(ScanPk p) {
    carry_walk<NP, false>(p, blockIdx.x * 64 + threadIdx.x);
}

// The outputs of a chunk (or of a whole sequence) from the state that enters it.  A
// row's sum over the states stays inside NS lanes (DPP); it goes through LDS to the
// element-wise mapping for D u, the gate and a wide store.  183 us at 8192 x 5120
// bf16: 0.98 of the vector units' cycles.  PAD: fewer states than NP.  Those past N are
// held at 0: their B and C are 0 already, but an infinite d or d u times 0 is not a number.
template <typename T, int NP, bool PAD>
__global__ __launch_bounds__(256) void scan_pk_out(ScanPk p) {
    constexpr int NS = ScanShape<NP>::NS, CPB = ScanShape<NP>::CPB, EV = ScanShape<NP>::EV, TT = ScanShape<NP>::TT;
    __shared__ float2 s_dd[TT][CPB];
    __shared__ __align__(16) float s_y[TT][CPB];
    __shared__ __align__(16) float s_B[TT][NP];
    __shared__ __align__(16) float s_C[TT][NP];
    const int nblk = (p.D + CPB - 1) / CPB;
    const int ck = (int)(blockIdx.x / (uint32_t)nblk);
    const int d0 = (int)(blockIdx.x % (uint32_t)nblk) * CPB;
    const ChunkEnds e(p, ck);
    const ElemMap<NP> m;
    // this thread's place in a tile (32 bits, beside a scalar base)
    auto at = [&](int64_t st) { return (uint32_t)(m.row * (int)st + m.ch); };
    const int c = threadIdx.x / NS, ng = threadIdx.x % NS, d = d0 + c;
    const int nc = p.D - (d0 + m.ch);
    float A2[4], h[4], bias[EV], Dv[EV];
    load_A2<NP>(p, d, ng, A2);
#pragma unroll
    for (int k = 0; k < EV; ++k) {
        bias[k] = p.bias && k < nc ? p.bias[d0 + m.ch + k] : 0.f;
        Dv[k] = p.Dv && k < nc ? p.Dv[d0 + m.ch + k] : 0.f;
    }
    const float zero[EV] = {};
    auto outside = [&](int a, int b) {  // rows of no sequence
        for (int t = a + m.row; p.fill && t < b; t += TT)
            st_run<EV, T>(static_cast<T*>(p.y) + (int64_t)t * p.y_st + d0 + m.ch, nc, zero);
    };
    Elems<T, EV> ru, rd, rz;
    BcTile<T, NP> rB, rC;
    auto fetch = [&](int t0, int b) {
        const int n = min(TT, b - t0);
        if (m.row < n && nc >= EV) {
            ru.load(static_cast<const T*>(p.u) + (t0 * p.u_st + d0) + at(p.u_st));
            rd.load(static_cast<const T*>(p.dl) + (t0 * p.dl_st + d0) + at(p.dl_st));
            if (p.z) rz.load(static_cast<const T*>(p.z) + (t0 * p.z_st + d0) + at(p.z_st));
        } else {
            const int q = m.row < n ? nc : 0;
            ru.load_part(static_cast<const T*>(p.u) + (t0 * p.u_st + d0) + at(p.u_st), q);
            rd.load_part(static_cast<const T*>(p.dl) + (t0 * p.dl_st + d0) + at(p.dl_st), q);
            if (p.z) rz.load_part(static_cast<const T*>(p.z) + (t0 * p.z_st + d0) + at(p.z_st), q);
        }
        rB.load(p.B, p.B_st, t0, n, p.N);
        rC.load(p.C, p.C_st, t0, n, p.N);
    };
    int t = e.c0;
    for (int s = e.first; s < p.q.n && t < e.c1; ++s) {
        const int st = p.q.begin(s), en = p.q.end(s);
        if (en <= t) {
            s = p.q.skip(s, t);
            continue;
        }
        if (st > t) {
            outside(t, min(st, e.c1));
            t = min(st, e.c1);
            if (t >= e.c1) break;
        }
        const int b = min(en, e.c1);
        const int64_t slot = p.state ? slot_of(p.slots, s, p.nslots) : -1;
        fetch(t, b);
        if (e.in && t == e.c0) {  // goes on from the chunk before
            load_carry<NP>(p.E, min(st / p.chunk, ck - 1), ck - 1, p, d, ng, A2, h);
        } else if (en > e.c1 && p.state) {
            load_plane<NP>(p.h0c, ck, p, d, ng, h);
        } else {
            load_state(p.state, slot, p, d, ng, h);
        }
        for (int t0 = t; t0 < b; t0 += TT) {
            const int n = min(TT, b - t0);
            float Du[EV], gate[EV], uv[EV], dv[EV];
            ru.get(uv);
            rd.get(dv);
            if (p.z) rz.get(gate);
#pragma unroll
            for (int k = 0; k < EV; ++k) dv[k] += bias[k];
            if (p.softplus) {
#pragma unroll
                for (int k = 0; k < EV; ++k) dv[k] = pk_softplus(dv[k]);
            }
#pragma unroll
            for (int k = 0; k < EV; ++k) {
                if (m.row >= n) dv[k] = 0.f;
                s_dd[m.row][m.ch + k] = make_float2(dv[k], dv[k] * uv[k]);
                Du[k] = Dv[k] * uv[k];
            }
            if (p.z) {
#pragma unroll
                for (int k = 0; k < EV; ++k) gate[k] *= pk_sigmoid(gate[k]);
            } else {
#pragma unroll
                for (int k = 0; k < EV; ++k) gate[k] = 1.f;
            }
            rB.stage(s_B);
            rC.stage(s_C);
            __syncthreads();
            if (t0 + TT < b) fetch(t0 + TT, b);
#pragma unroll 1
            for (int r = 0; r < n; r += 4) {
                float2 dd[4];
                float4 bv[4], cv[4];
                float yq[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    dd[i] = s_dd[r + i][c];
                    bv[i] = *(const float4*)&s_B[r + i][4 * ng];
                    cv[i] = *(const float4*)&s_C[r + i][4 * ng];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    h[0] = __builtin_fmaf(h[0], __builtin_amdgcn_exp2f(dd[i].x * A2[0]), dd[i].y * bv[i].x);
                    h[1] = __builtin_fmaf(h[1], __builtin_amdgcn_exp2f(dd[i].x * A2[1]), dd[i].y * bv[i].y);
                    h[2] = __builtin_fmaf(h[2], __builtin_amdgcn_exp2f(dd[i].x * A2[2]), dd[i].y * bv[i].z);
                    h[3] = __builtin_fmaf(h[3], __builtin_amdgcn_exp2f(dd[i].x * A2[3]), dd[i].y * bv[i].w);
                    if (PAD) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) h[k] = 4 * ng + k < p.N ? h[k] : 0.f;
                    }
                    yq[i] = __builtin_fmaf(cv[i].w, h[3], __builtin_fmaf(cv[i].z, h[2], __builtin_fmaf(cv[i].y, h[1], cv[i].x * h[0])));
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) yq[i] = group_sum_all<NS>(yq[i]);
#pragma unroll
                for (int i = 0; i < 4; ++i) s_y[r + i][c] = yq[i];  // the same value from each of the channel's lanes
            }
            __syncthreads();
            if (m.row < n) {
                float o[EV];
#pragma unroll
                for (int k = 0; k < EV; ++k) o[k] = (s_y[m.row][m.ch + k] + Du[k]) * gate[k];
                st_run<EV, T>(static_cast<T*>(p.y) + (t0 * p.y_st + d0) + at(p.y_st), nc, o);
            }
        }
        if (b == en) store_state(p.state, slot, p, d, ng, h);
        t = b;
    }
    if (p.whole) {  // the rows between this sequence and the next, and before the first
        outside(e.c1, ck + 1 < p.nchunk ? p.q.begin(ck + 1) : (int)p.rows);
        if (ck == 0) outside(0, e.c0);
    } else {
        outside(t, e.c1);
    }
}

// ---------------------------------------------------------------- backward ---

constexpr int kSub = 8;  // rows whose states and decays wait in registers

// Both carries of a chunk, each from zero: E as in the forward, G the gradient of
// the state that enters it; and the state before every kSub-th row of each
// sequence's part (from zero where the sequence came in, with the sum of d up to
// there: scan_pk_bwd adds what came in).  Row a + kSub i, i >= 1, of a part that
// begins at a is kept at place (a + kSub i) / kSub: no two parts share one.
// 212 us at 8192 x 5120 bf16, the vector units busy throughout; 357 MB written, 8 rows'
// states apart (every 4th row's would be 690 MB, every 16th's would not fit the
// registers of scan_pk_bwd).
template <typename T, int NP>
__global__ __launch_bounds__(256) void scan_pk_state_bwd(ScanPk p) {
    constexpr int NS = ScanShape<NP>::NS, CPB = ScanShape<NP>::CPB, EV = ScanShape<NP>::EV, TT = ScanShape<NP>::TT;
    __shared__ float2 s_dd[TT][CPB];
    __shared__ float s_e[TT][CPB];
    __shared__ __align__(16) float s_B[TT][NP];
    __shared__ __align__(16) float s_C[TT][NP];
    const int nblk = (p.D + CPB - 1) / CPB;
    const int ck = (int)(blockIdx.x / (uint32_t)nblk);
    const int d0 = (int)(blockIdx.x % (uint32_t)nblk) * CPB;
    const ChunkEnds e(p, ck);
    if (d0 == 0 && threadIdx.x == 0) p.ends[ck] = e.flags();
    const ElemMap<NP> m;
    // this thread's place in a tile (32 bits, beside a scalar base)
    auto at = [&](int64_t st) { return (uint32_t)(m.row * (int)st + m.ch); };
    const int c = threadIdx.x / NS, ng = threadIdx.x % NS, d = d0 + c;
    const int nc = p.D - (d0 + m.ch);
    float A2[4], h[4], P[4], G[4], sumd, bias[EV];
    load_A2<NP>(p, d, ng, A2);
#pragma unroll
    for (int k = 0; k < EV; ++k) bias[k] = p.bias && k < nc ? p.bias[d0 + m.ch + k] : 0.f;
    Elems<T, EV> ru, rd, re, rz;
    BcTile<T, NP> rB, rC;
    auto fetch = [&](int t0, int b) {
        const int n = min(TT, b - t0);
        if (m.row < n && nc >= EV) {
            ru.load(static_cast<const T*>(p.u) + (t0 * p.u_st + d0) + at(p.u_st));
            rd.load(static_cast<const T*>(p.dl) + (t0 * p.dl_st + d0) + at(p.dl_st));
            re.load(static_cast<const T*>(p.dy) + (t0 * p.dy_st + d0) + at(p.dy_st));
            if (p.z) rz.load(static_cast<const T*>(p.z) + (t0 * p.z_st + d0) + at(p.z_st));
        } else {
            const int q = m.row < n ? nc : 0;
            ru.load_part(static_cast<const T*>(p.u) + (t0 * p.u_st + d0) + at(p.u_st), q);
            rd.load_part(static_cast<const T*>(p.dl) + (t0 * p.dl_st + d0) + at(p.dl_st), q);
            re.load_part(static_cast<const T*>(p.dy) + (t0 * p.dy_st + d0) + at(p.dy_st), q);
            if (p.z) rz.load_part(static_cast<const T*>(p.z) + (t0 * p.z_st + d0) + at(p.z_st), q);
        }
        rB.load(p.B, p.B_st, t0, n, p.N);
        rC.load(p.C, p.C_st, t0, n, p.N);
    };
    int t = e.c0;
    for (int s = e.first; s < p.q.n && t < e.c1; ++s) {
        const int st = p.q.begin(s), en = p.q.end(s);
        if (en <= t) {
            s = p.q.skip(s, t);
            continue;
        }
        t = max(t, st);
        if (t >= e.c1) break;
        const int b = min(en, e.c1);
        const bool in = e.in && t == e.c0;
        fetch(t, b);
        if (in) h[0] = h[1] = h[2] = h[3] = 0.f;
        else load_state(p.h0, s, p, d, ng, h);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            P[k] = 1.f;
            G[k] = 0.f;
        }
        sumd = 0.f;
        for (int t0 = t; t0 < b; t0 += TT) {
            const int n = min(TT, b - t0);
            float uv[EV], dv[EV], ev[EV], zv[EV];
            ru.get(uv);
            rd.get(dv);
            re.get(ev);
            if (p.z) rz.get(zv);
#pragma unroll
            for (int k = 0; k < EV; ++k) dv[k] += bias[k];
            if (p.softplus) {
#pragma unroll
                for (int k = 0; k < EV; ++k) dv[k] = pk_softplus(dv[k]);
            }
            if (p.z) {
#pragma unroll
                for (int k = 0; k < EV; ++k) ev[k] *= zv[k] * pk_sigmoid(zv[k]);
            }
#pragma unroll
            for (int k = 0; k < EV; ++k) {
                if (m.row >= n) dv[k] = ev[k] = 0.f;
                s_dd[m.row][m.ch + k] = make_float2(dv[k], dv[k] * uv[k]);
                s_e[m.row][m.ch + k] = ev[k];
            }
            rB.stage(s_B);
            rC.stage(s_C);
            __syncthreads();
            if (t0 + TT < b) fetch(t0 + TT, b);
#pragma unroll 1
            for (int r0 = 0; r0 < n; r0 += 4) {
                if (r0 % kSub == 0 && t0 + r0 > t) {
                    const int place = (t0 + r0) / kSub;
                    store_plane<NP>(p.ckh, place, p, d, ng, h);
                    if (ng == 0 && d < p.D) p.ckd[(int64_t)place * p.D + d] = sumd;
                }
                float2 dd[4];
                float ee[4];
                float4 bq[4], cq[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    dd[i] = s_dd[r0 + i][c];
                    ee[i] = s_e[r0 + i][c];
                    bq[i] = *(const float4*)&s_B[r0 + i][4 * ng];
                    cq[i] = *(const float4*)&s_C[r0 + i][4 * ng];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float bv[4] = {bq[i].x, bq[i].y, bq[i].z, bq[i].w}, cv[4] = {cq[i].x, cq[i].y, cq[i].z, cq[i].w};
                    sumd += dd[i].x;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float a = __builtin_amdgcn_exp2f(dd[i].x * A2[k]);
                        h[k] = __builtin_fmaf(h[k], a, dd[i].y * bv[k]);
                        P[k] *= a;
                        G[k] = __builtin_fmaf(P[k], cv[k] * ee[i], G[k]);
                    }
                }
            }
            __syncthreads();
        }
        if (in) {
            if (b == en && p.dhT) {  // the sequence ends here: its own gradient comes in
                float g[4];
                load_state(p.dhT, s, p, d, ng, g);
#pragma unroll
                for (int k = 0; k < 4; ++k) G[k] = __builtin_fmaf(P[k], g[k], G[k]);
            }
            store_plane<NP>(p.G, ck, p, d, ng, G);
        }
        if (s == e.last) {
            store_plane<NP>(p.E, ck, p, d, ng, h);
            if (ng == 0 && d < p.D) p.sumd[(int64_t)ck * p.D + d] = sumd;
        }
        t = b;
    }
}

template <int NP>
__global__ __launch_bounds__(64) void scan_pk_carry_bwd(ScanPk p) {
    const int i = blockIdx.x * 64 + threadIdx.x;
    if (blockIdx.y == 0) carry_walk<NP, false>(p, i);
    else carry_walk<NP, true>(p, i);
}

// Sums over the wave's channels (lanes ng, ng + NS, ...) of v[0..3] and w[0..3].
// The halves and then the rows of 16 lanes are exchanged with half of the values
// each (a swap and an add for two of them), so that row R of lanes ends with
// element R % 2 of v (R < 2) or w in x0, and 2 + R % 2 in x1.
template <int NS>
__device__ __forceinline__ void channel_sums(const float (&v)[4], const float (&w)[4], float& x0, float& x1) {
    float y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[k]), __float_as_uint(w[k]), false, false);
        y[k] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(y[0]), __float_as_uint(y[1]), false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(y[2]), __float_as_uint(y[3]), false, false);
    x0 = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    x1 = __uint_as_float(b[0]) + __uint_as_float(b[1]);
    if (NS <= 8) {
        x0 += pk_dpp<0x128>(x0);  // row_ror:8
        x1 += pk_dpp<0x128>(x1);
    }
    if (NS <= 4) {
        x0 += pk_dpp<0x124>(x0);  // row_ror:4
        x1 += pk_dpp<0x124>(x1);
    }
    if (NS <= 2) {
        x0 += pk_dpp<0x122>(x0);  // row_ror:2
        x1 += pk_dpp<0x122>(x1);
    }
}

// The gradients of a chunk's rows, from the last to the first, kSub at a time.  596 us at
// 8192 x 5120 bf16: 256 M wave instructions at two waves a SIMD (230 registers), 0.85
// of the vector units' cycles; three waves (161 registers, the rows' operands read
// from LDS again) took 4 % longer.  PAD: fewer states than NP, those past N
// held at 0 with their gradients, as in scan_pk_out.
template <typename T, int NP, bool PAD>
__global__ __launch_bounds__(256) void scan_pk_bwd(ScanPk p) {
    constexpr int NS = ScanShape<NP>::NS, CPB = ScanShape<NP>::CPB, EV = ScanShape<NP>::EV, TT = ScanShape<NP>::TT;
    __shared__ __align__(16) float2 s_dd[TT][CPB];
    __shared__ __align__(16) float s_e[TT][CPB];
    __shared__ __align__(16) float s_sB[TT][CPB], s_sA[TT][CPB], s_sC[TT][CPB];
    __shared__ __align__(16) float s_BC[4][TT][NP];  // B, C, and zeros twice
    __shared__ __align__(16) float s_bc[4][TT][2 * NP];
    const int nblk = (p.D + CPB - 1) / CPB;
    const int ck = (int)(blockIdx.x / (uint32_t)nblk);
    const int blk = (int)(blockIdx.x % (uint32_t)nblk), d0 = blk * CPB;
    const ChunkEnds e(p, ck);
    const ElemMap<NP> m;
    // this thread's place in a tile (32 bits, beside a scalar base)
    auto at = [&](int64_t st) { return (uint32_t)(m.row * (int)st + m.ch); };
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int c = threadIdx.x / NS, ng = threadIdx.x % NS, d = d0 + c;
    const int nc = p.D - (d0 + m.ch);
    // Channels past D read zeros for B and C: an infinite one times their d u or e of 0 is not a
    // number, and dB and dC are sums over a wave's channels.
    const float (*const BC)[TT][NP] = s_BC + (d < p.D ? 0 : 2);
    for (int i = threadIdx.x; i < 2 * TT * NP; i += 256) (&s_BC[2][0][0])[i] = 0.f;
    // where this lane's channel sums go: element lane / 16 % 2 (and + 2) of B's (C's) four states
    const int bc_at = (lane >> 5) * NP + 4 * ng + ((lane >> 4) & 1);
    float A2[4], dA[4] = {0.f, 0.f, 0.f, 0.f};
    load_A2<NP>(p, d, ng, A2);
    float Dv[EV], bias[EV], dD[EV], db[EV];
#pragma unroll
    for (int k = 0; k < EV; ++k) {
        Dv[k] = p.Dv && k < nc ? p.Dv[d0 + m.ch + k] : 0.f;
        bias[k] = p.bias && k < nc ? p.bias[d0 + m.ch + k] : 0.f;
        dD[k] = db[k] = 0.f;
    }
    const float zero[EV] = {};
    float* pBC = p.pBC + (int64_t)blk * p.rows * 2 * NP;
    auto outside = [&](int a, int b) {
        for (int t = a + m.row; t < b; t += TT) {
            st_run<EV, T>(static_cast<T*>(p.du) + (int64_t)t * p.du_st + d0 + m.ch, nc, zero);
            st_run<EV, T>(static_cast<T*>(p.ddl) + (int64_t)t * p.ddl_st + d0 + m.ch, nc, zero);
            if (p.z) st_run<EV, T>(static_cast<T*>(p.dz) + (int64_t)t * p.dz_st + d0 + m.ch, nc, zero);
        }
        for (int64_t i = (int64_t)a * 2 * NP + threadIdx.x; i < (int64_t)b * 2 * NP; i += 256) pBC[i] = 0.f;
    };
    Elems<T, EV> ru, rd, re, rz;
    BcTile<T, NP> rB, rC;
    auto fetch = [&](int t0, int b) {
        const int n = min(TT, b - t0);
        if (m.row < n && nc >= EV) {
            ru.load(static_cast<const T*>(p.u) + (t0 * p.u_st + d0) + at(p.u_st));
            rd.load(static_cast<const T*>(p.dl) + (t0 * p.dl_st + d0) + at(p.dl_st));
            re.load(static_cast<const T*>(p.dy) + (t0 * p.dy_st + d0) + at(p.dy_st));
            if (p.z) rz.load(static_cast<const T*>(p.z) + (t0 * p.z_st + d0) + at(p.z_st));
        } else {
            const int q = m.row < n ? nc : 0;
            ru.load_part(static_cast<const T*>(p.u) + (t0 * p.u_st + d0) + at(p.u_st), q);
            rd.load_part(static_cast<const T*>(p.dl) + (t0 * p.dl_st + d0) + at(p.dl_st), q);
            re.load_part(static_cast<const T*>(p.dy) + (t0 * p.dy_st + d0) + at(p.dy_st), q);
            if (p.z) rz.load_part(static_cast<const T*>(p.z) + (t0 * p.z_st + d0) + at(p.z_st), q);
        }
        rB.load(p.B, p.B_st, t0, n, p.N);
        rC.load(p.C, p.C_st, t0, n, p.N);
    };
    int t = e.c0;
    for (int s = e.first; s < p.q.n && t < e.c1; ++s) {
        const int st = p.q.begin(s), en = p.q.end(s);
        if (en <= t) {
            s = p.q.skip(s, t);
            continue;
        }
        if (st > t) {
            outside(t, min(st, e.c1));
            t = min(st, e.c1);
            if (t >= e.c1) break;
        }
        const int b = min(en, e.c1);
        const bool in = e.in && t == e.c0;
        const int len = b - t, tiles = (len + TT - 1) / TT;
        fetch(t + (tiles - 1) * TT, b);
        float h0[4], g[4], hn[4], dn = 0.f;  // hn, dn: the next part's kept state and sum of d
        if (in) load_carry<NP>(p.E, min(st / p.chunk, ck - 1), ck - 1, p, d, ng, A2, h0);
        else load_state(p.h0, s, p, d, ng, h0);
        if (en > e.c1) load_carry<NP>(p.G, (en - 1) / p.chunk, ck + 1, p, d, ng, A2, g);
        else load_state(p.dhT, s, p, d, ng, g);
        auto kept = [&](int q) {  // before row kSub q of the run
            if (q <= 0) return;
            const int place = (t + q * kSub) / kSub;
            load_plane<NP>(p.ckh, place, p, d, ng, hn);
            if (in) dn = d < p.D ? p.ckd[(int64_t)place * p.D + d] : 0.f;
        };
        kept(len / kSub - 1);
        for (int tl = tiles - 1; tl >= 0; --tl) {
            const int t0 = t + tl * TT;
            const int n = min(TT, b - t0);
            float uv[EV], dv[EV], yv[EV], zv[EV];
            ru.get(uv);
            rd.get(dv);
            re.get(yv);
            if (p.z) rz.get(zv);
#pragma unroll
            for (int k = 0; k < EV; ++k) dv[k] += bias[k];
            float dt[EV], ev[EV], sz[EV];  // sz: sigmoid(z)
            if (p.softplus) {
#pragma unroll
                for (int k = 0; k < EV; ++k) dt[k] = pk_softplus(dv[k]);
            } else {
#pragma unroll
                for (int k = 0; k < EV; ++k) dt[k] = dv[k];
            }
            if (p.z) {
#pragma unroll
                for (int k = 0; k < EV; ++k) {
                    sz[k] = pk_sigmoid(zv[k]);
                    ev[k] = yv[k] * (zv[k] * sz[k]);
                }
            } else {
#pragma unroll
                for (int k = 0; k < EV; ++k) ev[k] = yv[k];
            }
#pragma unroll
            for (int k = 0; k < EV; ++k) {
                if (m.row >= n) dt[k] = ev[k] = 0.f;
                s_dd[m.row][m.ch + k] = make_float2(dt[k], dt[k] * uv[k]);
                s_e[m.row][m.ch + k] = ev[k];
            }
            rB.stage(s_BC[0]);
            rC.stage(s_BC[1]);
            __syncthreads();
            if (tl > 0) fetch(t0 - TT, b);
            auto held = [&](float v, int k) __attribute__((always_inline)) { return !PAD || 4 * ng + k < p.N ? v : 0.f; };
            auto step = [&](int r, const float (&h)[4], float (&a)[4], float (&after)[4]) __attribute__((always_inline)) {
                const float2 dd = s_dd[r][c];
                const float4 bq = *(const float4*)&BC[0][r][4 * ng];
                const float bv[4] = {bq.x, bq.y, bq.z, bq.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    a[k] = __builtin_amdgcn_exp2f(dd.x * A2[k]);
                    after[k] = held(__builtin_fmaf(h[k], a[k], dd.y * bv[k]), k);
                }
            };
            auto back = [&](int r, const float (&h)[4], const float (&a)[4], const float (&after)[4]) __attribute__((always_inline)) {
                const float2 dd = s_dd[r][c];
                const float ev = s_e[r][c];
                const float4 bq = *(const float4*)&BC[0][r][4 * ng], cq = *(const float4*)&BC[1][r][4 * ng];
                const float bv[4] = {bq.x, bq.y, bq.z, bq.w}, cv[4] = {cq.x, cq.y, cq.z, cq.w};
                float sB = 0.f, sA = 0.f, sC = 0.f, vb[4], vc[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float gk = held(__builtin_fmaf(cv[k], ev, g[k]), k);
                    vb[k] = gk * dd.y;
                    vc[k] = after[k] * ev;
                    sB = __builtin_fmaf(gk, bv[k], sB);
                    sC = __builtin_fmaf(cv[k], after[k], sC);
                    g[k] = held(gk * a[k], k);
                    const float x = g[k] * h[k];
                    sA = __builtin_fmaf(x, A2[k], sA);
                    dA[k] = __builtin_fmaf(x, dd.x, dA[k]);
                }
                sB = group_sum_all<NS>(sB);
                sA = group_sum_all<NS>(sA);
                sC = group_sum_all<NS>(sC);
                float x0, x1;
                channel_sums<NS>(vb, vc, x0, x1);
                // every lane that holds a sum writes it (the same value to the same
                // place): a branch here would keep the rows apart in the schedule
                s_sB[r][c] = sB;
                s_sA[r][c] = sA;
                s_sC[r][c] = sC;
                s_bc[wave][r][bc_at] = x0;
                s_bc[wave][r][bc_at + 2] = x1;
            };
            const int whole = n / kSub * kSub;
            if (n > whole) {
                // The last rows of a part, fewer than kSub: each finds its state again from the
                // start.  (Made up to kSub by steps that change nothing, they would add an infinite
                // state times a gradient of 0 to dA.  Their kept state is not hn: did that come from
                // two places, the loop below would wait for the next tile's rows before its first:
                // 826 us for 8192 x 5120 bf16 with all kernels, 792 so.)
                float h0r[4] = {h0[0], h0[1], h0[2], h0[3]};
                if (len > kSub) {
                    const int place = (t0 + whole) / kSub;
                    const float sum = in && d < p.D ? p.ckd[(int64_t)place * p.D + d] : 0.f;
                    load_plane<NP>(p.ckh, place, p, d, ng, h0r);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (in) h0r[k] = __builtin_fmaf(__builtin_amdgcn_exp2f(sum * A2[k]), h0[k], h0r[k]);
                }
                if (PAD) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) h0r[k] = held(h0r[k], k);
                }
#pragma unroll 1
                for (int r = n - 1; r >= whole; --r) {
                    float h[4], a[4], after[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) h[k] = h0r[k];
#pragma unroll 1
                    for (int j = whole; j < r; ++j) step(j, h, a, h);
                    step(r, h, a, after);
                    back(r, h, a, after);
                }
            }
#pragma unroll 1
            for (int r0 = whole - kSub; r0 >= 0; r0 -= kSub) {
                float hs[kSub + 1][4], as[kSub][4];
                const int q = tl * (TT / kSub) + r0 / kSub;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    hs[0][k] = held(q == 0 ? h0[k] : in ? __builtin_fmaf(__builtin_amdgcn_exp2f(dn * A2[k]), h0[k], hn[k]) : hn[k], k);
                kept(q - 1);
#pragma unroll
                for (int i = 0; i < kSub; ++i) step(r0 + i, hs[i], as[i], hs[i + 1]);
#pragma unroll
                for (int i = kSub - 1; i >= 0; --i) back(r0 + i, hs[i], as[i], hs[i + 1]);
            }
            __syncthreads();
            // ---- the tile's dB and dC over the workgroup, and the gradients of its elements
            for (int i = threadIdx.x; i < n * 2 * NP; i += 256) {
                const int r = i / (2 * NP), k = i % (2 * NP);
                pBC[(int64_t)t0 * 2 * NP + i] = (s_bc[0][r][k] + s_bc[1][r][k]) + (s_bc[2][r][k] + s_bc[3][r][k]);
            }
            if (m.row < n) {
                float o1[EV], o2[EV], o3[EV];
#pragma unroll
                for (int k = 0; k < EV; ++k) {
                    const float sB = s_sB[m.row][m.ch + k], sA = s_sA[m.row][m.ch + k] * (1.f / kLog2e);
                    const float dt = s_dd[m.row][m.ch + k].x, ev = s_e[m.row][m.ch + k];
                    o1[k] = __builtin_fmaf(sB, dt, Dv[k] * ev);
                    o2[k] = __builtin_fmaf(sB, uv[k], sA);
                    dD[k] = __builtin_fmaf(ev, uv[k], dD[k]);
                }
                if (p.softplus) {
#pragma unroll
                    for (int k = 0; k < EV; ++k) o2[k] *= pk_sigmoid(dv[k]);
                }
                if (p.z) {
#pragma unroll
                    for (int k = 0; k < EV; ++k) {
                        o3[k] = yv[k] * __builtin_fmaf(Dv[k], uv[k], s_sC[m.row][m.ch + k]) *
                                (sz[k] * __builtin_fmaf(zv[k], 1.f - sz[k], 1.f));
                    }
                }
#pragma unroll
                for (int k = 0; k < EV; ++k) db[k] += o2[k];
                st_run<EV, T>(static_cast<T*>(p.du) + (t0 * p.du_st + d0) + at(p.du_st), nc, o1);
                st_run<EV, T>(static_cast<T*>(p.ddl) + (t0 * p.ddl_st + d0) + at(p.ddl_st), nc, o2);
                if (p.z) st_run<EV, T>(static_cast<T*>(p.dz) + (t0 * p.dz_st + d0) + at(p.dz_st), nc, o3);
            }
        }
        if (t == st) store_state(p.dh0, s, p, d, ng, g);
        t = b;
    }
    outside(t, e.c1);
    // ---- the chunk's share of dA, dD and dbias
    store_plane<NP>(p.pA, ck, p, d, ng, dA);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EV; ++k) {
        s_sB[m.row][m.ch + k] = dD[k];
        s_sA[m.row][m.ch + k] = db[k];
    }
    __syncthreads();
    if (threadIdx.x < CPB && d0 + (int)threadIdx.x < p.D) {
        float x = 0.f, y = 0.f;
        for (int r = 0; r < TT; ++r) {
            x += s_sB[r][threadIdx.x];
            y += s_sA[r][threadIdx.x];
        }
        p.pD[(int64_t)ck * p.D + d0 + threadIdx.x] = x;
        p.pb[(int64_t)ck * p.D + d0 + threadIdx.x] = y;
    }
}

// The joins, each in a fixed order, 64 values a workgroup and a quarter of their terms
// each of its waves: workgroups 0 .. par - 1 dA, dD and dbias over the chunks, column j
// of [D][NP] | [D] | [D]; those behind them dB and dC over the channel blocks.  Their
// bytes are read once, as they were written (8192 x 5120 x 16: 84 + 12 MB, 20.5 us).
template <typename T, int NP>
__global__ __launch_bounds__(256) void scan_pk_join(ScanPk p, int nblk, uint32_t par) {
    __shared__ float red[4][64];
    const int q = wave_id(), l = threadIdx.x & 63;
    const bool params = blockIdx.x < par;
    const int64_t i = (params ? blockIdx.x : blockIdx.x - par) * 64ll + l, nA = (int64_t)p.D * NP;
    const int64_t total = params ? nA + 2 * p.D : p.rows * 2 * NP;
    const float* src = !params ? p.pBC + i : i < nA ? p.pA + i : i < nA + p.D ? p.pD + (i - nA) : p.pb + (i - nA - p.D);
    const int64_t pitch = !params ? total : i < nA ? nA : p.D;
    const int count = params ? p.nchunk : nblk;
    float s = 0.f;
    if (i < total) {
#pragma unroll 8
        for (int k = q; k < count; k += 4) s += src[k * pitch];
    }
    red[q][l] = s;
    __syncthreads();
    if (q || i >= total) return;
    s = (red[0][l] + red[1][l]) + (red[2][l] + red[3][l]);
    if (!params) {
        const int64_t t = i / (2 * NP);
        const int k = (int)(i - t * 2 * NP), n = k % NP;
        if (n >= p.N) return;
        if (k < NP) store_f32<T>(static_cast<T*>(p.dB) + t * p.dB_st + n, s);
        else store_f32<T>(static_cast<T*>(p.dC) + t * p.dC_st + n, s);
    } else if (i < nA) {
        const int n = (int)(i % NP);
        if (n < p.N) p.dA[i / NP * p.N + n] = s;
    } else if (i < nA + p.D) {
        if (p.dD) p.dD[i - nA] = s;
    } else if (p.db) {
        p.db[i - nA - p.D] = s;
    }
}

// ------------------------------------------------------------ single tokens ---

struct ScanSlotParams {
    int nb, D, N;
    bool softplus;
    const void* u; int64_t u_sb;
    const void* dl; int64_t dl_sb;
    const void* z; int64_t z_sb;
    const void* B; int64_t B_sb;
    const void* C; int64_t C_sb;
    const float* A; const float* Dv; const float* bias;
    float* state; int64_t nslots; const int32_t* slots;
    void* y; int64_t y_sb;
};

// Any dstate up to 1024: the states of CH = 1024 / N channels lie one behind the other, so
// the workgroup takes them four a thread whatever N is, and adds h C up by channel
// in LDS, Q lanes each.  256 tokens x 5120, bf16: 12 states 43 us, 20 states 68 (3.2 TB/s; a
// thread per channel 90 and 211).
constexpr int kSlotRun = 1024;
template <typename T>
__global__ __launch_bounds__(256) void scan_slot_any(ScanSlotParams p) {
    __shared__ float2 s_dd[kSlotRun];
    __shared__ float s_u[kSlotRun], s_p[kSlotRun], s_B[kSlotRun], s_C[kSlotRun];
    const int N = p.N, CH = kSlotRun / N, d0 = blockIdx.x * CH, nc = min(CH, p.D - d0), b = blockIdx.y;
    T* y = static_cast<T*>(p.y) + b * p.y_sb + d0;
    const int64_t slot = slot_of(p.slots, b, p.nslots);
    if (slot < 0) {
        for (int c = threadIdx.x; c < nc; c += 256) store_f32<T>(y + c, 0.f);
        return;
    }
    const int e0 = 4 * threadIdx.x, left = nc * N - e0;
    float* state = p.state + (slot * p.D + d0) * N + e0;
    float h[4], A[4];
    ld_run<4, float>(state, left, h);
    ld_run<4, float>(p.A + (int64_t)d0 * N + e0, left, A);
    for (int c = threadIdx.x; c < nc; c += 256) {
        const float u = load_f32<T>(static_cast<const T*>(p.u) + b * p.u_sb + d0 + c);
        float dv = load_f32<T>(static_cast<const T*>(p.dl) + b * p.dl_sb + d0 + c);
        if (p.bias) dv += p.bias[d0 + c];
        if (p.softplus) dv = pk_softplus(dv);
        s_dd[c] = make_float2(dv, dv * u);
        s_u[c] = u;
    }
    for (int n = threadIdx.x; n < N; n += 256) {
        s_B[n] = load_f32<T>(static_cast<const T*>(p.B) + b * p.B_sb + n);
        s_C[n] = load_f32<T>(static_cast<const T*>(p.C) + b * p.C_sb + n);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (k >= left) break;
        const int c = (e0 + k) / N, n = e0 + k - c * N;
        const float2 dd = s_dd[c];
        h[k] = __builtin_fmaf(h[k], __builtin_amdgcn_exp2f(dd.x * (A[k] * kLog2e)), dd.y * s_B[n]);
        s_p[e0 + k] = h[k] * s_C[n];
    }
    if (left > 0) st_run<4, float>(state, left, h);
    __syncthreads();
    int Q = 1;
    while (Q < 64 && 2 * Q * CH <= 256) Q *= 2;
    for (int i0 = 0; i0 < nc * Q; i0 += 256) {
        const int c = (i0 + (int)threadIdx.x) / Q, q = threadIdx.x % Q;
        float acc = 0.f;
        for (int n = q; c < nc && n < N; n += Q) acc += s_p[c * N + n];
        for (int o = Q / 2; o > 0; o >>= 1) acc += __shfl_xor(acc, o);
        if (q || c >= nc) continue;
        if (p.Dv) acc = __builtin_fmaf(p.Dv[d0 + c], s_u[c], acc);
        if (p.z) {
            const float zv = load_f32<T>(static_cast<const T*>(p.z) + b * p.z_sb + d0 + c);
            acc *= zv * pk_sigmoid(zv);
        }
        store_f32<T>(y + c, acc);
    }
}

// dstate 8, 16, 32 or 64: a channel over N / 4 lanes with 16 bytes of its state
// each, CPT channels a thread.  The state is read and written once (HBM-bound:
// 8 N bytes a channel against some 12 of everything else), so its loads are
// issued first and none waits under a branch: what is optional is read through a
// pointer to something that is there, and dropped.  256 tokens x 5120 x 16, bf16: 35.6
// us, 178 MB, 5.0 TB/s.
template <typename T, int N, int CPT>
__global__ __launch_bounds__(256) void scan_slot_step(ScanSlotParams p) {
    constexpr int LPC = N / 4, CPB = 256 / LPC;
    const int b = blockIdx.y, q = threadIdx.x % LPC;
    const int64_t slot = slot_of(p.slots, b, p.nslots);
    const int base = blockIdx.x * CPB * CPT + threadIdx.x / LPC;
    T* y = static_cast<T*>(p.y) + b * p.y_sb;
    if (slot < 0) {
#pragma unroll
        for (int k = 0; k < CPT; ++k)
            if (q == 0 && base + k * CPB < p.D) store_f32<T>(y + base + k * CPB, 0.f);
        return;
    }
    const T* u = static_cast<const T*>(p.u) + b * p.u_sb;
    const T* dl = static_cast<const T*>(p.dl) + b * p.dl_sb;
    const T* z = p.z ? static_cast<const T*>(p.z) + b * p.z_sb : dl;
    float4* state = reinterpret_cast<float4*>(p.state + slot * p.D * N) + q;
    float4 h[CPT], A[CPT];
    float uv[CPT], dv[CPT], zv[CPT], Dv[CPT], bias[CPT];
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        const int d = min(base + k * CPB, p.D - 1);
        h[k] = ld_nt4(state + (int64_t)d * LPC);
        A[k] = *(reinterpret_cast<const float4*>(p.A + (int64_t)d * N) + q);
        dv[k] = load_f32<T>(dl + d);
        uv[k] = load_f32<T>(u + d);
        zv[k] = load_f32<T>(z + d);
        Dv[k] = *(p.Dv ? p.Dv + d : p.A);
        bias[k] = *(p.bias ? p.bias + d : p.A);
    }
    float bv[4], cv[4];
    ld_run<4, T>(static_cast<const T*>(p.B) + b * p.B_sb + 4 * q, 4, bv);
    ld_run<4, T>(static_cast<const T*>(p.C) + b * p.C_sb + 4 * q, 4, cv);
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        if (p.bias) dv[k] += bias[k];
        if (p.softplus) dv[k] = pk_softplus(dv[k]);
        const float du = dv[k] * uv[k], d2 = dv[k] * kLog2e;
        h[k].x = __builtin_fmaf(h[k].x, __builtin_amdgcn_exp2f(d2 * A[k].x), du * bv[0]);
        h[k].y = __builtin_fmaf(h[k].y, __builtin_amdgcn_exp2f(d2 * A[k].y), du * bv[1]);
        h[k].z = __builtin_fmaf(h[k].z, __builtin_amdgcn_exp2f(d2 * A[k].z), du * bv[2]);
        h[k].w = __builtin_fmaf(h[k].w, __builtin_amdgcn_exp2f(d2 * A[k].w), du * bv[3]);
        float acc = __builtin_fmaf(h[k].w, cv[3], __builtin_fmaf(h[k].z, cv[2], __builtin_fmaf(h[k].y, cv[1], h[k].x * cv[0])));
        acc = group_sum_last<LPC>(acc);
        const int d = base + k * CPB;
        if (d >= p.D) continue;
        st_nt4(state + (int64_t)d * LPC, h[k]);
        if (q == LPC - 1) {
            if (p.Dv) acc = __builtin_fmaf(Dv[k], uv[k], acc);
            if (p.z) acc *= zv[k] * pk_sigmoid(zv[k]);
            store_f32<T>(y + d, acc);
        }
    }
}

template <typename T, int N>
static void scan_slot_launch(const ScanSlotParams& p, hipStream_t s) {
    // four channels a thread while that leaves two workgroups a CU, else one
    constexpr int CPB = 256 / (N / 4);
    if ((int64_t)ceil_div(p.D, 4 * CPB) * p.nb >= 512)
        hipLaunchKernelGGL((scan_slot_step<T, N, 4>), dim3(ceil_div(p.D, 4 * CPB), p.nb), dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((scan_slot_step<T, N, 1>), dim3(ceil_div(p.D, CPB), p.nb), dim3(256), 0, s, p);
}

template <typename T>
static void scan_slot_dispatch(const ScanSlotParams& p, hipStream_t s) {
    const bool aligned = (((uintptr_t)p.state | (uintptr_t)p.A) & 15u) == 0;
    switch (aligned ? p.N : 0) {
        case 8: scan_slot_launch<T, 8>(p, s); break;
        case 16: scan_slot_launch<T, 16>(p, s); break;
        case 32: scan_slot_launch<T, 32>(p, s); break;
        case 64: scan_slot_launch<T, 64>(p, s); break;
        default: hipLaunchKernelGGL(scan_slot_any<T>, dim3(ceil_div(p.D, kSlotRun / p.N), p.nb), dim3(256), 0, s, p);
    }
}

// ---------------------------------------------------------------- dispatch ---

// (8192 x 5120 bf16 with 8 states: 224 us forward and 537 backward, 312 and 835 padded to 16)
static int scan_np(int N) { return N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }

static int scan_pk_make(const mamba1_scan_packed_args* a, ScanPk* o) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    MAMBA_CHECK_ARG(a->rows >= 0 && a->rows < kMaxRows, "rows must be in [0, 2^31 - 2^20)");
    MAMBA_CHECK_ARG(a->dim >= 1 && a->dim <= (1 << 20), "dim must be in [1, 2^20]");
    MAMBA_CHECK_ARG(a->dstate >= 1, "dstate must be >= 1");
    MAMBA_CHECK_ARG(a->nseq >= 0, "nseq must be >= 0");
    MAMBA_CHECK_ARG(a->io_dtype == MAMBA_F32 || a->io_dtype == MAMBA_BF16, "io_dtype must be f32 or bf16");
    if (a->dstate > 64) {
        set_error(std::string(__func__) + ": dstate above 64 is not implemented for packed sequences");
        return MAMBA_ERR_UNSUPPORTED;
    }
    MAMBA_CHECK_ARG(a->cu_seqlens != nullptr && a->A != nullptr, "cu_seqlens and A are required");
    MAMBA_CHECK_ARG(a->rows == 0 || (a->u && a->delta && a->B && a->C), "u, delta, B and C are required");
    for (int64_t st : {a->u_st, a->delta_st, a->z_st, a->B_st, a->C_st})
        MAMBA_CHECK_ARG(a->rows <= 1 || (st >= 0 && st < kMaxStride), "row strides must be in [0, 2^25)");
    ScanPk& p = *o;
    p = ScanPk{};
    p.q = Seqs{a->cu_seqlens, a->nseq, (int)a->rows};
    p.rows = a->rows; p.D = a->dim; p.N = a->dstate;
    p.softplus = a->delta_softplus != 0; p.fill = a->fill_outside != 0;
    p.u = a->u; p.u_st = a->u_st; p.dl = a->delta; p.dl_st = a->delta_st; p.z = a->z; p.z_st = a->z_st;
    p.B = a->B; p.B_st = a->B_st; p.C = a->C; p.C_st = a->C_st;
    p.A = a->A; p.Dv = a->D; p.bias = a->delta_bias;
    return MAMBA_OK;
}

// Rows of a chunk: four workgroups a CU where the rows are enough for it, at most
// 256 rows (longer ones gain nothing), and at least about 0.6 sqrt(rows), where a
// chunk's walk over those before it and its own scan (0.2 us a row and pass) weigh alike.
// us, forward, at 1024 / 2048 / 4096 workgroups: 8192 x 5120 325 / 328 / 323, 4000 x
// 2560 103 / 107 / 114, 2000 x 2560 63 / 67 / 72; at 0.3 / 0.45 / 0.6 / 0.85 sqrt(rows):
// 8192 x 256 89 / 72 / 50 / 48, with the backward 218 / 185 / 137 / 139, 1023 x 777 31 / 31 / 25 / 25.
// Up to 128 chunks find what comes into them by themselves; the walk of all of them in a
// kernel of its own takes 10 to 14 us more where they are few (forward and backward,
// 1023 x 777 84 against 71; 4000 x 2560 340 against 325; 8192 x 256, 128 chunks, 158
// against 137), but each walks over half of them on average.
static void scan_pk_plan(ScanPk& p) {
    const int64_t nblk = ceil_div(p.D, 1024 / scan_np(p.N));
    const int64_t fill = (p.rows * nblk + 1023) / 1024, least = (int64_t)(0.6 * std::sqrt((double)p.rows));
    const int64_t rows = std::max<int64_t>(1, std::max(fill, least));
    p.chunk = (int)std::min<int64_t>(256, (rows + kTile - 1) / kTile * kTile);
    p.nchunk = (int)((p.rows + p.chunk - 1) / p.chunk);
    p.walk = p.nchunk <= 128;
}
constexpr int64_t kMaxGroups = 1ll << 24;  // a grid's threads stay below 2^32
// Whole sequences, a workgroup of CPB channels each, where the longest is known to
// be short beside all the rows' work: its rows take some 0.15 us one behind the
// other, and in chunks most rows are scanned twice.  Up to 96 rows in any case: the
// chunks' second launch and workspace cost a call more than they save: one call among
// others takes 13 us whole and 17 in chunks to 64 rows, 16.5 and 17.3 at 96.  (Its time on the
// GPU alone, which a captured graph has, turns at some 48 rows: 9.1 and 9.5 us at 40 x 512,
// 13.8 and 10.3 at 77, 16.2 and 10.5 at 96 x 2560; a caller that knows no bound gets chunks.)
// Longer ones, whole / in chunks: 8 sequences of 2048 x 5120 466 / 558, 4 of them 352 /
// 285, 16 of 512 190 / 259, 16 of 256 x 2560 64 / 91, 8 of 512 95 / 95, 16 of 128 x 1024
// 23 / 31, 8 of them 22 / 21.
static void scan_pk_fwd_plan(ScanPk& p, int max_seqlen) {
    scan_pk_plan(p);
    const int64_t nblk = ceil_div(p.D, 1024 / scan_np(p.N));
    if (p.nchunk > 1 && max_seqlen > 0 && p.q.n > 0 && p.q.n * nblk < kMaxGroups && max_seqlen <= std::max<int64_t>(96, 64 + p.rows * nblk / 384)) {
        p.whole = true;
        p.nchunk = p.q.n;
    }
}
static int scan_pk_grid_ok(const ScanPk& p, bool back) {
    const int64_t nblk = ceil_div(p.D, 1024 / scan_np(p.N));
    const int64_t np = scan_np(p.N), joined = back ? p.rows * 2 * np + p.D * (np + 2) + 128 : 0;
    if (p.nchunk * nblk >= kMaxGroups || joined > 64 * kMaxGroups) {  // the join: 64 values a workgroup
        set_error("mamba1_scan_packed: rows * dim is too large for one call");
        return MAMBA_ERR_UNSUPPORTED;
    }
    return MAMBA_OK;
}

template <typename T, int NP>
static void scan_pk_fwd_launch(const ScanPk& p, hipStream_t s) {
    const uint32_t nblk = ceil_div(p.D, ScanShape<NP>::CPB);
    if (p.nchunk > 1 && !p.whole) {
        hipLaunchKernelGGL((scan_pk_state<T, NP>), dim3(nblk * (uint32_t)(p.nchunk - 1)), dim3(256), 0, s, p);
        if (!p.walk) hipLaunchKernelGGL((scan_pk_carry<NP>), dim3(ceil_div(p.D * NP, 64)), dim3(64), 0, s, p);
    }
    const dim3 grid(nblk * (uint32_t)p.nchunk);
    if (p.N == NP) hipLaunchKernelGGL((scan_pk_out<T, NP, false>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((scan_pk_out<T, NP, true>), grid, dim3(256), 0, s, p);
}

template <typename T, int NP>
static void scan_pk_bwd_launch(const ScanPk& p, hipStream_t s) {
    const uint32_t nblk = ceil_div(p.D, ScanShape<NP>::CPB);
    if (p.rows) {
        const dim3 grid(nblk * (uint32_t)p.nchunk);
        hipLaunchKernelGGL((scan_pk_state_bwd<T, NP>), grid, dim3(256), 0, s, p);
        if (!p.walk) hipLaunchKernelGGL((scan_pk_carry_bwd<NP>), dim3(ceil_div(p.D * NP, 64), 2), dim3(64), 0, s, p);
        if (p.N == NP) hipLaunchKernelGGL((scan_pk_bwd<T, NP, false>), grid, dim3(256), 0, s, p);
        else hipLaunchKernelGGL((scan_pk_bwd<T, NP, true>), grid, dim3(256), 0, s, p);
    }
    const uint32_t par = (uint32_t)(((int64_t)p.D * (NP + 2) + 63) / 64);
    hipLaunchKernelGGL((scan_pk_join<T, NP>), dim3(par + (uint32_t)((p.rows * 2 * NP + 63) / 64)), dim3(256), 0, s, p, (int)nblk, par);
}

#define SCAN_PK_DISPATCH(fn, np, bf16, ...)              \
    do {                                                 \
        if ((np) == 8) {                                 \
            if (bf16) fn<bf16_t, 8>(__VA_ARGS__);        \
            else fn<float, 8>(__VA_ARGS__);              \
        } else if ((np) == 16) {                         \
            if (bf16) fn<bf16_t, 16>(__VA_ARGS__);       \
            else fn<float, 16>(__VA_ARGS__);             \
        } else if ((np) == 32) {                         \
            if (bf16) fn<bf16_t, 32>(__VA_ARGS__);       \
            else fn<float, 32>(__VA_ARGS__);             \
        } else {                                         \
            if (bf16) fn<bf16_t, 64>(__VA_ARGS__);       \
            else fn<float, 64>(__VA_ARGS__);             \
        }                                                \
    } while (0)

// Workspaces: planes of floats, each of a multiple of four (16 bytes).
struct ScanPlanes {
    float* base; size_t used = 0;
    explicit ScanPlanes(void* ws) : base(static_cast<float*>(ws)) {}
    float* take(size_t n) {
        float* at = base ? base + used : nullptr;
        used += (n + 3) / 4 * 4;
        return at;
    }
};
static size_t scan_pk_fwd_planes(ScanPk& p, void* ws) {
    if (p.nchunk <= 1 || p.whole) return 0;
    ScanPlanes w(ws);
    const size_t nd = (size_t)p.nchunk * p.D, np = scan_np(p.N);
    p.E = w.take(nd * np);
    p.h0c = w.take(nd * np);
    p.sumd = w.take(nd);
    p.ends = reinterpret_cast<int32_t*>(w.take(p.nchunk));
    return w.used * 4;
}
static size_t scan_pk_bwd_planes(ScanPk& p, void* ws) {
    ScanPlanes w(ws);
    const size_t nd = (size_t)p.nchunk * p.D, np = scan_np(p.N), nk = (size_t)p.rows / kSub + 1;
    p.E = w.take(nd * np);
    p.G = w.take(nd * np);
    p.pA = w.take(nd * np);
    p.sumd = w.take(nd);
    p.pD = w.take(nd);
    p.pb = w.take(nd);
    p.ends = reinterpret_cast<int32_t*>(w.take(p.nchunk));
    p.ckh = w.take(nk * p.D * np);
    p.ckd = w.take(nk * p.D);
    p.pBC = w.take((size_t)ceil_div(p.D, 1024 / (int)np) * p.rows * 2 * np);
    return w.used * 4;
}

}  // namespace mamba

using namespace mamba;

extern "C" size_t mamba1_scan_packed_workspace_size(const mamba1_scan_packed_args* a) {
    ScanPk p;
    if (scan_pk_make(a, &p) != MAMBA_OK) return 0;
    scan_pk_fwd_plan(p, a->max_seqlen);
    return scan_pk_fwd_planes(p, nullptr);
}

extern "C" int mamba1_scan_packed_fwd(const mamba1_scan_packed_args* a, void* ws, size_t ws_bytes, mamba_stream_t stream) {
    ScanPk p;
    int st = scan_pk_make(a, &p);
    if (st != MAMBA_OK) return st;
    if (p.rows == 0) return MAMBA_OK;
    MAMBA_CHECK_ARG(a->y != nullptr, "y is required");
    MAMBA_CHECK_ARG((a->y_st >= p.D && a->y_st < kMaxStride) || p.rows == 1, "rows of y overlap (or lie 2^25 elements apart)");
    MAMBA_CHECK_ARG(a->state == nullptr || a->slots != nullptr || a->nslots >= a->nseq,
                    "without slots the state needs a row per sequence");
    const size_t e = a->io_dtype == MAMBA_BF16 ? 2 : 4;
    MAMBA_CHECK_ARG(!rows_clash(a->y, a->y_st, a->u, a->u_st, p.D, p.D, p.rows, e, true) &&
                        !rows_clash(a->y, a->y_st, a->delta, a->delta_st, p.D, p.D, p.rows, e, true) &&
                        !rows_clash(a->y, a->y_st, a->z, a->z_st, p.D, p.D, p.rows, e, true) &&
                        !rows_clash(a->y, a->y_st, a->B, a->B_st, p.D, p.N, p.rows, e, false) &&
                        !rows_clash(a->y, a->y_st, a->C, a->C_st, p.D, p.N, p.rows, e, false),
                    "y overlaps an input (it may be u, delta or z itself)");
    p.y = a->y; p.y_st = a->y_st;
    p.state = a->state; p.nslots = a->nslots; p.slots = a->slots;
    scan_pk_fwd_plan(p, a->max_seqlen);
    if ((st = scan_pk_grid_ok(p, false)) != MAMBA_OK) return st;
    const size_t need = scan_pk_fwd_planes(p, ws);
    MAMBA_CHECK_ARG(((uintptr_t)ws & 15u) == 0, "the workspace must be 16-byte aligned");
    if (need && (ws == nullptr || ws_bytes < need)) {
        set_error("mamba1_scan_packed_fwd: workspace missing or too small");
        return MAMBA_ERR_WORKSPACE;
    }
    SCAN_PK_DISPATCH(scan_pk_fwd_launch, scan_np(p.N), a->io_dtype == MAMBA_BF16, p, (hipStream_t)stream);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}

extern "C" size_t mamba1_scan_packed_bwd_workspace_size(const mamba1_scan_packed_bwd_args* a) {
    ScanPk p;
    if (a == nullptr || scan_pk_make(&a->fwd, &p) != MAMBA_OK) return 0;
    scan_pk_plan(p);
    return scan_pk_bwd_planes(p, nullptr);
}

extern "C" int mamba1_scan_packed_bwd(const mamba1_scan_packed_bwd_args* a, void* ws, size_t ws_bytes, mamba_stream_t stream) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    ScanPk p;
    int st = scan_pk_make(&a->fwd, &p);
    if (st != MAMBA_OK) return st;
    MAMBA_CHECK_ARG(a->fwd.state == nullptr && a->fwd.slots == nullptr,
                    "the gradient takes initial_state, a row per sequence, and no slots");
    MAMBA_CHECK_ARG(a->dA != nullptr, "dA is required");
    MAMBA_CHECK_ARG(p.rows == 0 || (a->dy && a->du && a->ddelta && a->dB && a->dC), "dy, du, ddelta, dB and dC are required");
    MAMBA_CHECK_ARG(p.rows == 0 || (p.z != nullptr) == (a->dz != nullptr), "dz goes with z");
    MAMBA_CHECK_ARG(p.rows <= 1 || (a->du_st >= p.D && a->ddelta_st >= p.D && (!a->dz || a->dz_st >= p.D)),
                    "rows of du, ddelta or dz overlap");
    MAMBA_CHECK_ARG(p.rows <= 1 || (a->dB_st >= p.N && a->dC_st >= p.N), "rows of dB or dC overlap");
    for (int64_t st : {a->dy_st, a->du_st, a->ddelta_st, a->dz_st, a->dB_st, a->dC_st})
        MAMBA_CHECK_ARG(p.rows <= 1 || (st >= 0 && st < kMaxStride), "row strides must be in [0, 2^25)");
    struct Rows { const void* p; int64_t st; int cols; };
    const Rows ins[] = {{a->fwd.u, a->fwd.u_st, p.D}, {a->fwd.delta, a->fwd.delta_st, p.D}, {a->fwd.z, a->fwd.z_st, p.D},
                        {a->dy, a->dy_st, p.D}, {a->fwd.B, a->fwd.B_st, p.N}, {a->fwd.C, a->fwd.C_st, p.N}};
    const Rows outs[] = {{a->du, a->du_st, p.D}, {a->ddelta, a->ddelta_st, p.D}, {a->dz, a->dz_st, p.D},
                         {a->dB, a->dB_st, p.N}, {a->dC, a->dC_st, p.N}};
    const size_t es = a->fwd.io_dtype == MAMBA_BF16 ? 2 : 4;
    for (const Rows& o : outs) {
        for (const Rows& i : ins)
            MAMBA_CHECK_ARG(!rows_clash(o.p, o.st, i.p, i.st, o.cols, i.cols, p.rows, es, false), "a gradient overlaps an input");
        for (const Rows* q = outs; q != &o; ++q)
            MAMBA_CHECK_ARG(!rows_clash(o.p, o.st, q->p, q->st, o.cols, q->cols, p.rows, es, false), "two gradients overlap");
    }
    p.dy = a->dy; p.dy_st = a->dy_st; p.h0 = a->initial_state; p.dhT = a->d_final_state;
    p.du = a->du; p.du_st = a->du_st; p.ddl = a->ddelta; p.ddl_st = a->ddelta_st; p.dz = a->dz; p.dz_st = a->dz_st;
    p.dB = a->dB; p.dB_st = a->dB_st; p.dC = a->dC; p.dC_st = a->dC_st;
    p.dA = a->dA; p.dD = a->dD; p.db = a->d_delta_bias; p.dh0 = a->d_initial_state;
    scan_pk_plan(p);
    if ((st = scan_pk_grid_ok(p, true)) != MAMBA_OK) return st;
    const size_t need = scan_pk_bwd_planes(p, ws);
    MAMBA_CHECK_ARG(((uintptr_t)ws & 15u) == 0, "the workspace must be 16-byte aligned");
    if (need && (ws == nullptr || ws_bytes < need)) {
        set_error("mamba1_scan_packed_bwd: workspace missing or too small");
        return MAMBA_ERR_WORKSPACE;
    }
    SCAN_PK_DISPATCH(scan_pk_bwd_launch, scan_np(p.N), a->fwd.io_dtype == MAMBA_BF16, p, (hipStream_t)stream);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}

extern "C" int mamba1_scan_step_slots(const mamba1_scan_step_slots_args* a, mamba_stream_t stream) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    MAMBA_CHECK_ARG(a->batch >= 0 && a->batch <= 65535, "batch must be in [0, 65535]");
    MAMBA_CHECK_ARG(a->dim >= 1 && a->dim <= (1 << 20), "dim must be in [1, 2^20]");
    MAMBA_CHECK_ARG(a->dstate >= 1 && a->dstate <= 1024, "dstate must be in [1, 1024]");
    MAMBA_CHECK_ARG(a->io_dtype == MAMBA_F32 || a->io_dtype == MAMBA_BF16, "io_dtype must be f32 or bf16");
    if (a->batch == 0) return MAMBA_OK;
    MAMBA_CHECK_ARG(a->u && a->delta && a->A && a->B && a->C && a->state && a->y,
                    "u, delta, A, B, C, state and y are required");
    MAMBA_CHECK_ARG(a->slots != nullptr || a->nslots >= a->batch, "without slots the state needs a row per token");
    MAMBA_CHECK_ARG(a->y_sb >= a->dim || a->batch == 1, "rows of y overlap");
    const size_t e = a->io_dtype == MAMBA_BF16 ? 2 : 4;
    MAMBA_CHECK_ARG(!rows_clash(a->y, a->y_sb, a->u, a->u_sb, a->dim, a->dim, a->batch, e, true) &&
                        !rows_clash(a->y, a->y_sb, a->delta, a->delta_sb, a->dim, a->dim, a->batch, e, true) &&
                        !rows_clash(a->y, a->y_sb, a->z, a->z_sb, a->dim, a->dim, a->batch, e, true) &&
                        !rows_clash(a->y, a->y_sb, a->B, a->B_sb, a->dim, a->dstate, a->batch, e, false) &&
                        !rows_clash(a->y, a->y_sb, a->C, a->C_sb, a->dim, a->dstate, a->batch, e, false),
                    "y overlaps an input (it may be u, delta or z itself)");
    ScanSlotParams p{};
    p.nb = a->batch; p.D = a->dim; p.N = a->dstate; p.softplus = a->delta_softplus != 0;
    p.u = a->u; p.u_sb = a->u_sb; p.dl = a->delta; p.dl_sb = a->delta_sb; p.z = a->z; p.z_sb = a->z_sb;
    p.B = a->B; p.B_sb = a->B_sb; p.C = a->C; p.C_sb = a->C_sb;
    p.A = a->A; p.Dv = a->D; p.bias = a->delta_bias;
    p.state = a->state; p.nslots = a->nslots; p.slots = a->slots; p.y = a->y; p.y_sb = a->y_sb;
    if (a->io_dtype == MAMBA_BF16) scan_slot_dispatch<bf16_t>(p, (hipStream_t)stream);
    else scan_slot_dispatch<float>(p, (hipStream_t)stream);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}
