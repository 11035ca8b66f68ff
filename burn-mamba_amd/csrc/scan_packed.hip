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
// over it, scan_pk_carry walks the chunks, h <- exp(A sum d) h + own, and
// scan_pk_out scans again from there.  In the backward the gradient of the state
// is carried the same way from the last chunk to the first.
//
// A workgroup of 256 threads holds CPB = 1024 / NP channels, NP = the states
// padded to 16, 32 or 64; a channel is spread over NS = NP / 4 lanes with 4 states
// each.  Tiles of NP rows are staged through LDS as f32 with the element-wise
// work (softplus, d u) done once per element.
#include <algorithm>

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
    int chunk; int64_t nchunk;
    // per chunk: what it leaves behind [nchunk][D][NP] (then, carried, what
    // leaves it), the sum of d [nchunk][D], and the state that its last sequence
    // began from [nchunk][D][NP] (the cache's slot may be written meanwhile)
    float* E; float* sumd; float* h0c;
    // backward
    const void* dy; int64_t dy_st;
    const float* h0; const float* dhT;
    float* G;                       // [nchunk][D][NP]: gradient of the state that enters a chunk
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
// hardware log with Goldberg's correction, log(v) e / (v - 1) for v = 1 + e
__device__ __forceinline__ float pk_softplus(float x) {
    if (x > 20.f) return x;
    const float e = __expf(x);
    const float v = 1.f + e;
    return v == 1.f ? e : __logf(v) * (e * __builtin_amdgcn_rcpf(v - 1.f));
}
__device__ __forceinline__ float pk_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + __expf(-x)); }

template <int CTRL>
__device__ __forceinline__ float pk_dpp(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
// Sum over aligned groups of NS lanes, in every lane: xor 1, xor 2 inside quads,
// then the mirrors of half rows and rows.
template <int NS>
__device__ __forceinline__ float group_sum_all(float v) {
    static_assert(NS == 4 || NS == 8 || NS == 16, "4, 8 or 16 lanes");
    v += pk_dpp<0xB1>(v);
    v += pk_dpp<0x4E>(v);
    if (NS >= 8) v += pk_dpp<0x141>(v);
    if (NS >= 16) v += pk_dpp<0x140>(v);
    return v;
}

template <int NP>
struct ScanShape {
    static constexpr int NS = NP / 4, CPB = 256 / NS, TT = NP;  // TT CPB = 1024: four elements a thread
};

// The element-wise mapping: row tid / (CPB / 4) of the tile, 4 channels from
// 4 (tid % (CPB / 4)).  Channels past D are staged as zeros (with A = 0 their
// states stay 0), so that sums over a wave's channels need no mask.
template <int NP>
struct ElemMap {
    int row, c4;
    __device__ __forceinline__ ElemMap() {
        constexpr int W = ScanShape<NP>::CPB / 4;
        row = threadIdx.x / W;
        c4 = 4 * (threadIdx.x % W);
    }
};

// B or C of rows t0 .. into [row][NP] (zero past n rows and N states)
template <typename T, int NP>
__device__ __forceinline__ void stage_bc(const void* src, int64_t st, int64_t t0, int n, int N, float (*dst)[NP]) {
    for (int i = threadIdx.x; i < n * NP; i += 256) {
        const int r = i / NP, k = i % NP;
        dst[r][k] = k < N ? load_f32<T>(static_cast<const T*>(src) + (t0 + r) * st + k) : 0.f;
    }
}

// What chunk ck does at its two ends: the sequence that crosses into it and the
// one that crosses out of it (-1: none).
struct ChunkEnds {
    int64_t c0, c1;
    int first, last;   // first sequence with rows in the chunk, and the one that crosses c1
    bool in, through;  // the first one began before c0; it fills the chunk and goes on
    __device__ __forceinline__ ChunkEnds(const ScanPk& p, int64_t ck) {
        c0 = ck * p.chunk;
        c1 = min(p.rows, c0 + p.chunk);
        first = p.q.after(c0);
        in = first < p.q.n && p.q.begin(first) < c0;
        last = -1;
        if (c1 < p.rows) {
            const int s = p.q.after(c1);
            if (s < p.q.n && p.q.begin(s) < c1) last = s;
        }
        through = in && last == first;
    }
};

// Rows [a, b) of one sequence from state h: the state behind them, and sum of d.
template <typename T, int NP>
__device__ __forceinline__ void scan_state_run(const ScanPk& p, int64_t a, int64_t b, int d0, const float (&A2)[4],
                                               float (&h)[4], float& sumd, float2 (*s_dd)[ScanShape<NP>::CPB],
                                               float (*s_B)[NP]) {
    constexpr int NS = ScanShape<NP>::NS, TT = ScanShape<NP>::TT;
    const ElemMap<NP> m;
    const int c = threadIdx.x / NS, ng = threadIdx.x % NS;
    const int nc = p.D - (d0 + m.c4);
    for (int64_t t0 = a; t0 < b; t0 += TT) {
        const int n = (int)min((int64_t)TT, b - t0);
        if (m.row < n) {
            float uv[4], dv[4];
            ld_run<4, T>(static_cast<const T*>(p.u) + (t0 + m.row) * p.u_st + d0 + m.c4, nc, uv);
            ld_run<4, T>(static_cast<const T*>(p.dl) + (t0 + m.row) * p.dl_st + d0 + m.c4, nc, dv);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (p.bias && e < nc) dv[e] += p.bias[d0 + m.c4 + e];
                if (p.softplus) dv[e] = pk_softplus(dv[e]);
                s_dd[m.row][m.c4 + e] = make_float2(dv[e], dv[e] * uv[e]);
            }
        }
        stage_bc<T, NP>(p.B, p.B_st, t0, n, p.N, s_B);
        __syncthreads();
        for (int t = 0; t < n; ++t) {
            const float2 dd = s_dd[t][c];
            const float4 bv = *(const float4*)&s_B[t][4 * ng];
            sumd += dd.x;
            h[0] = __builtin_fmaf(h[0], __builtin_amdgcn_exp2f(dd.x * A2[0]), dd.y * bv.x);
            h[1] = __builtin_fmaf(h[1], __builtin_amdgcn_exp2f(dd.x * A2[1]), dd.y * bv.y);
            h[2] = __builtin_fmaf(h[2], __builtin_amdgcn_exp2f(dd.x * A2[2]), dd.y * bv.z);
            h[3] = __builtin_fmaf(h[3], __builtin_amdgcn_exp2f(dd.x * A2[3]), dd.y * bv.w);
        }
        __syncthreads();
    }
}

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
    return reinterpret_cast<float4*>(base + ((ck * p.D + d) * NP + 4 * ng));
}

template <typename T, int NP>
__global__ __launch_bounds__(256) void scan_pk_state(ScanPk p) {
    constexpr int NS = ScanShape<NP>::NS, CPB = ScanShape<NP>::CPB, TT = ScanShape<NP>::TT;
    __shared__ float2 s_dd[TT][CPB];
    __shared__ __align__(16) float s_B[TT][NP];
    const int nblk = (p.D + CPB - 1) / CPB;
    const int64_t ck = blockIdx.x / nblk;
    const int d0 = (int)(blockIdx.x % nblk) * CPB;
    const ChunkEnds e(p, ck);
    if (e.last < 0) return;  // nothing crosses its end
    const int c = threadIdx.x / NS, ng = threadIdx.x % NS, d = d0 + c;
    float A2[4], h[4] = {0.f, 0.f, 0.f, 0.f}, sumd = 0.f;
    load_A2<NP>(p, d, ng, A2);
    const int64_t st = p.q.begin(e.last);
    if (st >= e.c0 && p.state) {
        load_state(p.state, slot_of(p.slots, e.last, p.nslots), p, d, ng, h);
        if (d < p.D) *plane<NP>(p.h0c, ck, p, d, ng) = make_float4(h[0], h[1], h[2], h[3]);
    }
    scan_state_run<T, NP>(p, max(st, e.c0), e.c1, d0, A2, h, sumd, s_dd, s_B);
    if (d < p.D) {
        *plane<NP>(p.E, ck, p, d, ng) = make_float4(h[0], h[1], h[2], h[3]);
        if (ng == 0) p.sumd[ck * p.D + d] = sumd;
    }
}

// E[ck] <- the state that leaves chunk ck.  A thread per (channel, state).
template <int NP>
__global__ __launch_bounds__(256) void scan_pk_carry(ScanPk p) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    const int d = i / NP, n = i % NP;
    const bool live = d < p.D;
    const float A2 = live && n < p.N ? p.A[(int64_t)d * p.N + n] * kLog2e : 0.f;
    float h = 0.f;
    for (int64_t ck = 0; ck + 1 < p.nchunk; ++ck) {
        const ChunkEnds e(p, ck);
        if (e.last < 0) continue;
        if (!live) continue;
        float* E = p.E + (ck * p.D + d) * NP + n;
        float own = *E;
        if (e.through) own = __builtin_fmaf(__builtin_amdgcn_exp2f(p.sumd[ck * p.D + d] * A2), h, own);
        h = own;
        *E = h;
    }
}

template <typename T, int NP>
__global__ __launch_bounds__(256) void scan_pk_out(ScanPk p) {
    constexpr int NS = ScanShape<NP>::NS, CPB = ScanShape<NP>::CPB, TT = ScanShape<NP>::TT;
    __shared__ float2 s_dd[TT][CPB];
    __shared__ __align__(16) float s_y[TT][CPB];
    __shared__ __align__(16) float s_B[TT][NP];
    __shared__ __align__(16) float s_C[TT][NP];
    const int nblk = (p.D + CPB - 1) / CPB;
    const int64_t ck = blockIdx.x / nblk;
    const int d0 = (int)(blockIdx.x % nblk) * CPB;
    const ChunkEnds e(p, ck);
    const ElemMap<NP> m;
    const int c = threadIdx.x / NS, ng = threadIdx.x % NS, d = d0 + c;
    const int nc = p.D - (d0 + m.c4);
    float A2[4], h[4];
    load_A2<NP>(p, d, ng, A2);
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    auto outside = [&](int64_t a, int64_t b) {  // rows of no sequence
        for (int64_t t = a + m.row; p.fill && t < b; t += TT)
            st_run<4, T>(static_cast<T*>(p.y) + t * p.y_st + d0 + m.c4, nc, zero);
    };
    int64_t t = e.c0;
    for (int s = e.first; s < p.q.n && t < e.c1; ++s) {
        const int64_t st = p.q.begin(s), en = p.q.end(s);
        if (en <= t) continue;
        if (st > t) {
            outside(t, min(st, e.c1));
            t = min(st, e.c1);
            if (t >= e.c1) break;
        }
        const int64_t b = min(en, e.c1), slot = p.state ? slot_of(p.slots, s, p.nslots) : -1;
        if (e.in && t == e.c0) {  // goes on from the chunk before
            const float4 v = d < p.D ? *plane<NP>(p.E, ck - 1, p, d, ng) : make_float4(0.f, 0.f, 0.f, 0.f);
            h[0] = v.x; h[1] = v.y; h[2] = v.z; h[3] = v.w;
        } else if (en > e.c1 && p.state) {
            const float4 v = d < p.D ? *plane<NP>(p.h0c, ck, p, d, ng) : make_float4(0.f, 0.f, 0.f, 0.f);
            h[0] = v.x; h[1] = v.y; h[2] = v.z; h[3] = v.w;
        } else {
            load_state(p.state, slot, p, d, ng, h);
        }
        for (int64_t t0 = t; t0 < b; t0 += TT) {
            const int n = (int)min((int64_t)TT, b - t0);
            float Du[4], gate[4];
            if (m.row < n) {
                float uv[4], dv[4];
                ld_run<4, T>(static_cast<const T*>(p.u) + (t0 + m.row) * p.u_st + d0 + m.c4, nc, uv);
                ld_run<4, T>(static_cast<const T*>(p.dl) + (t0 + m.row) * p.dl_st + d0 + m.c4, nc, dv);
                if (p.z) ld_run<4, T>(static_cast<const T*>(p.z) + (t0 + m.row) * p.z_st + d0 + m.c4, nc, gate);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (p.bias && k < nc) dv[k] += p.bias[d0 + m.c4 + k];
                    if (p.softplus) dv[k] = pk_softplus(dv[k]);
                    s_dd[m.row][m.c4 + k] = make_float2(dv[k], dv[k] * uv[k]);
                    Du[k] = p.Dv && k < nc ? p.Dv[d0 + m.c4 + k] * uv[k] : 0.f;
                    gate[k] = p.z ? gate[k] * pk_sigmoid(gate[k]) : 1.f;
                }
            }
            stage_bc<T, NP>(p.B, p.B_st, t0, n, p.N, s_B);
            stage_bc<T, NP>(p.C, p.C_st, t0, n, p.N, s_C);
            __syncthreads();
            for (int r = 0; r < n; ++r) {
                const float2 dd = s_dd[r][c];
                const float4 bv = *(const float4*)&s_B[r][4 * ng], cv = *(const float4*)&s_C[r][4 * ng];
                h[0] = __builtin_fmaf(h[0], __builtin_amdgcn_exp2f(dd.x * A2[0]), dd.y * bv.x);
                h[1] = __builtin_fmaf(h[1], __builtin_amdgcn_exp2f(dd.x * A2[1]), dd.y * bv.y);
                h[2] = __builtin_fmaf(h[2], __builtin_amdgcn_exp2f(dd.x * A2[2]), dd.y * bv.z);
                h[3] = __builtin_fmaf(h[3], __builtin_amdgcn_exp2f(dd.x * A2[3]), dd.y * bv.w);
                const float part = __builtin_fmaf(cv.w, h[3], __builtin_fmaf(cv.z, h[2], __builtin_fmaf(cv.y, h[1], cv.x * h[0])));
                s_y[r][c] = group_sum_all<NS>(part);
            }
            __syncthreads();
            if (m.row < n) {
                const float4 yv = *(const float4*)&s_y[m.row][m.c4];
                const float o[4] = {(yv.x + Du[0]) * gate[0], (yv.y + Du[1]) * gate[1], (yv.z + Du[2]) * gate[2],
                                    (yv.w + Du[3]) * gate[3]};
                st_run<4, T>(static_cast<T*>(p.y) + (t0 + m.row) * p.y_st + d0 + m.c4, nc, o);
            }
        }
        if (b == en) store_state(p.state, slot, p, d, ng, h);
        t = b;
    }
    outside(t, e.c1);
}

// ---------------------------------------------------------------- backward ---

// Both carries of a chunk, each from zero: E (forward, rows of the sequence that
// crosses its end) and G (the gradient of the state that enters it, from the rows
// of the sequence that crosses its start): with P_t the product of the decays from
// the chunk's start, G = sum_t P_t C_t e_t, so both walk forwards on the same exp.
template <typename T, int NP>
__global__ __launch_bounds__(256) void scan_pk_state_bwd(ScanPk p) {
    constexpr int NS = ScanShape<NP>::NS, CPB = ScanShape<NP>::CPB, TT = ScanShape<NP>::TT;
    __shared__ float s_d[TT][CPB], s_du[TT][CPB], s_e[TT][CPB];
    __shared__ __align__(16) float s_B[TT][NP];
    __shared__ __align__(16) float s_C[TT][NP];
    const int nblk = (p.D + CPB - 1) / CPB;
    const int64_t ck = blockIdx.x / nblk;
    const int d0 = (int)(blockIdx.x % nblk) * CPB;
    const ChunkEnds e(p, ck);
    const ElemMap<NP> m;
    const int c = threadIdx.x / NS, ng = threadIdx.x % NS, d = d0 + c;
    const int nc = p.D - (d0 + m.c4);
    float A2[4], h[4], P[4], G[4], sumd;
    load_A2<NP>(p, d, ng, A2);
    auto run = [&](int64_t a, int64_t b) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            P[k] = 1.f;
            G[k] = 0.f;
        }
        sumd = 0.f;
        for (int64_t t0 = a; t0 < b; t0 += TT) {
            const int n = (int)min((int64_t)TT, b - t0);
            if (m.row < n) {
                float uv[4], dv[4], ev[4], zv[4];
                ld_run<4, T>(static_cast<const T*>(p.u) + (t0 + m.row) * p.u_st + d0 + m.c4, nc, uv);
                ld_run<4, T>(static_cast<const T*>(p.dl) + (t0 + m.row) * p.dl_st + d0 + m.c4, nc, dv);
                ld_run<4, T>(static_cast<const T*>(p.dy) + (t0 + m.row) * p.dy_st + d0 + m.c4, nc, ev);
                if (p.z) ld_run<4, T>(static_cast<const T*>(p.z) + (t0 + m.row) * p.z_st + d0 + m.c4, nc, zv);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (p.bias && k < nc) dv[k] += p.bias[d0 + m.c4 + k];
                    if (p.softplus) dv[k] = pk_softplus(dv[k]);
                    if (p.z) ev[k] *= zv[k] * pk_sigmoid(zv[k]);
                    s_d[m.row][m.c4 + k] = dv[k];
                    s_du[m.row][m.c4 + k] = dv[k] * uv[k];
                    s_e[m.row][m.c4 + k] = ev[k];
                }
            }
            stage_bc<T, NP>(p.B, p.B_st, t0, n, p.N, s_B);
            stage_bc<T, NP>(p.C, p.C_st, t0, n, p.N, s_C);
            __syncthreads();
            for (int t = 0; t < n; ++t) {
                const float dv = s_d[t][c], du = s_du[t][c], ev = s_e[t][c];
                const float4 bq = *(const float4*)&s_B[t][4 * ng], cq = *(const float4*)&s_C[t][4 * ng];
                const float bv[4] = {bq.x, bq.y, bq.z, bq.w}, cv[4] = {cq.x, cq.y, cq.z, cq.w};
                sumd += dv;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float a = __builtin_amdgcn_exp2f(dv * A2[k]);
                    h[k] = __builtin_fmaf(h[k], a, du * bv[k]);
                    P[k] *= a;
                    G[k] = __builtin_fmaf(P[k], cv[k] * ev, G[k]);
                }
            }
            __syncthreads();
        }
    };
    if (e.in) {
        const int64_t en = p.q.end(e.first);
        h[0] = h[1] = h[2] = h[3] = 0.f;
        run(e.c0, min(en, e.c1));
        if (en <= e.c1 && p.dhT) {  // the sequence ends here: its own gradient comes in
            float g[4];
            load_state(p.dhT, e.first, p, d, ng, g);
#pragma unroll
            for (int k = 0; k < 4; ++k) G[k] = __builtin_fmaf(P[k], g[k], G[k]);
        }
        if (d < p.D) *plane<NP>(p.G, ck, p, d, ng) = make_float4(G[0], G[1], G[2], G[3]);
    }
    if (e.last >= 0) {
        if (!e.through) {
            load_state(p.h0, e.last, p, d, ng, h);
            run(p.q.begin(e.last), e.c1);
        }
        if (d < p.D) *plane<NP>(p.E, ck, p, d, ng) = make_float4(h[0], h[1], h[2], h[3]);
    }
    if (e.through && d < p.D && ng == 0) p.sumd[ck * p.D + d] = sumd;
}

// blockIdx.y 0: E as in the forward; 1: G from the last chunk to the first.
template <int NP>
__global__ __launch_bounds__(256) void scan_pk_carry_bwd(ScanPk p) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    const int d = i / NP, n = i % NP;
    if (d >= p.D) return;
    const float A2 = n < p.N ? p.A[(int64_t)d * p.N + n] * kLog2e : 0.f;
    float v = 0.f;
    for (int64_t j = 0; j + 1 < p.nchunk; ++j) {
        const bool fwd = blockIdx.y == 0;
        const int64_t ck = fwd ? j : p.nchunk - 1 - j;
        const ChunkEnds e(p, ck);
        if (fwd ? e.last < 0 : !e.in) continue;
        float* X = (fwd ? p.E : p.G) + (ck * p.D + d) * NP + n;
        float own = *X;
        if (e.through) own = __builtin_fmaf(__builtin_amdgcn_exp2f(p.sumd[ck * p.D + d] * A2), v, own);
        v = own;
        *X = v;
    }
}

constexpr int kSub = 8;    // rows whose states and decays wait in registers
constexpr int kBwdChunk = 64;

// The chunk itself: forwards over its rows once for the state at every kSub rows,
// then backwards, kSub rows at a time, the states in between found again.  The
// staged d, d u and e of a row are overwritten by its s, sum_n g a h A and sum_n C h.
template <typename T, int NP>
__global__ __launch_bounds__(256) void scan_pk_bwd(ScanPk p) {
    constexpr int NS = ScanShape<NP>::NS, CPB = ScanShape<NP>::CPB, TT = ScanShape<NP>::TT, Q = kBwdChunk;
    constexpr int NK = Q / kSub;
    __shared__ __align__(16) float s_d[Q][CPB], s_du[Q][CPB], s_e[Q][CPB];
    __shared__ __align__(16) float s_B[Q][NP];
    __shared__ __align__(16) float s_C[Q][NP];
    __shared__ __align__(16) float s_bc[4][kSub][2 * NP];
    const int nblk = (p.D + CPB - 1) / CPB;
    const int64_t ck = blockIdx.x / nblk;
    const int blk = (int)(blockIdx.x % nblk), d0 = blk * CPB;
    const ChunkEnds e(p, ck);
    const ElemMap<NP> m;
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int c = threadIdx.x / NS, ng = threadIdx.x % NS, d = d0 + c;
    const int nc = p.D - (d0 + m.c4);
    float A2[4], dA[4] = {0.f, 0.f, 0.f, 0.f};
    load_A2<NP>(p, d, ng, A2);
    float Dv[4], bias[4], dD[4], db[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        Dv[k] = p.Dv && k < nc ? p.Dv[d0 + m.c4 + k] : 0.f;
        bias[k] = p.bias && k < nc ? p.bias[d0 + m.c4 + k] : 0.f;
        dD[k] = db[k] = 0.f;
    }
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    float* pBC = p.pBC + (int64_t)blk * p.rows * 2 * NP;
    auto outside = [&](int64_t a, int64_t b) {
        for (int64_t t = a + m.row; t < b; t += TT) {
            st_run<4, T>(static_cast<T*>(p.du) + t * p.du_st + d0 + m.c4, nc, zero);
            st_run<4, T>(static_cast<T*>(p.ddl) + t * p.ddl_st + d0 + m.c4, nc, zero);
            if (p.z) st_run<4, T>(static_cast<T*>(p.dz) + t * p.dz_st + d0 + m.c4, nc, zero);
        }
        for (int64_t i = a * 2 * NP + threadIdx.x; i < b * 2 * NP; i += 256) pBC[i] = 0.f;
    };
    int64_t t = e.c0;
    for (int s = e.first; s < p.q.n && t < e.c1; ++s) {
        const int64_t st = p.q.begin(s), en = p.q.end(s);
        if (en <= t) continue;
        if (st > t) {
            outside(t, min(st, e.c1));
            t = min(st, e.c1);
            if (t >= e.c1) break;
        }
        const int64_t b = min(en, e.c1);
        const int n = (int)(b - t);
        // ---- the run's elements
        for (int r = m.row; r < n; r += TT) {
            float uv[4], dv[4], ev[4], zv[4];
            ld_run<4, T>(static_cast<const T*>(p.u) + (t + r) * p.u_st + d0 + m.c4, nc, uv);
            ld_run<4, T>(static_cast<const T*>(p.dl) + (t + r) * p.dl_st + d0 + m.c4, nc, dv);
            ld_run<4, T>(static_cast<const T*>(p.dy) + (t + r) * p.dy_st + d0 + m.c4, nc, ev);
            if (p.z) ld_run<4, T>(static_cast<const T*>(p.z) + (t + r) * p.z_st + d0 + m.c4, nc, zv);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                dv[k] += bias[k];
                if (p.softplus) dv[k] = pk_softplus(dv[k]);
                if (p.z) ev[k] *= zv[k] * pk_sigmoid(zv[k]);
                s_d[r][m.c4 + k] = dv[k];
                s_du[r][m.c4 + k] = dv[k] * uv[k];
                s_e[r][m.c4 + k] = ev[k];
            }
        }
        stage_bc<T, NP>(p.B, p.B_st, t, n, p.N, s_B);
        stage_bc<T, NP>(p.C, p.C_st, t, n, p.N, s_C);
        float h[4], g[4];
        if (e.in && t == e.c0) {  // goes on from the chunk before
            const float4 v = d < p.D ? *plane<NP>(p.E, ck - 1, p, d, ng) : make_float4(0.f, 0.f, 0.f, 0.f);
            h[0] = v.x; h[1] = v.y; h[2] = v.z; h[3] = v.w;
        } else {
            load_state(p.h0, s, p, d, ng, h);
        }
        if (en > e.c1) {
            const float4 v = d < p.D ? *plane<NP>(p.G, ck + 1, p, d, ng) : make_float4(0.f, 0.f, 0.f, 0.f);
            g[0] = v.x; g[1] = v.y; g[2] = v.z; g[3] = v.w;
        } else {
            load_state(p.dhT, s, p, d, ng, g);
        }
        __syncthreads();
        // ---- forwards: the state at every kSub rows
        float ck_h[NK][4];
#pragma unroll
        for (int j = 0; j < NK; ++j) {
#pragma unroll
            for (int k = 0; k < 4; ++k) ck_h[j][k] = h[k];
            if ((j + 1) * kSub < n)
                for (int r = j * kSub; r < (j + 1) * kSub; ++r) {
                    const float dv = s_d[r][c], du = s_du[r][c];
                    const float4 bq = *(const float4*)&s_B[r][4 * ng];
                    const float bv[4] = {bq.x, bq.y, bq.z, bq.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) h[k] = __builtin_fmaf(h[k], __builtin_amdgcn_exp2f(dv * A2[k]), du * bv[k]);
                }
        }
        // ---- backwards
#pragma unroll
        for (int j = NK - 1; j >= 0; --j) {
            if (j * kSub >= n) continue;
            float hs[kSub + 1][4], as[kSub][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) hs[0][k] = ck_h[j][k];
#pragma unroll
            for (int i = 0; i < kSub; ++i) {
                const int r = j * kSub + i;
                const bool in = r < n;
                const float dv = in ? s_d[r][c] : 0.f, du = in ? s_du[r][c] : 0.f;
                const float4 bq = *(const float4*)&s_B[r][4 * ng];
                const float bv[4] = {bq.x, bq.y, bq.z, bq.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    as[i][k] = __builtin_amdgcn_exp2f(dv * A2[k]);
                    hs[i + 1][k] = __builtin_fmaf(hs[i][k], as[i][k], in ? du * bv[k] : 0.f);
                }
            }
#pragma unroll
            for (int i = kSub - 1; i >= 0; --i) {
                const int r = j * kSub + i;
                if (r >= n) continue;
                const float dv = s_d[r][c], du = s_du[r][c], ev = s_e[r][c];
                const float4 bq = *(const float4*)&s_B[r][4 * ng], cq = *(const float4*)&s_C[r][4 * ng];
                const float bv[4] = {bq.x, bq.y, bq.z, bq.w}, cv[4] = {cq.x, cq.y, cq.z, cq.w};
                float sB = 0.f, sA = 0.f, sC = 0.f, vb[4], vc[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float gk = __builtin_fmaf(cv[k], ev, g[k]);
                    vb[k] = gk * du;
                    vc[k] = hs[i + 1][k] * ev;
                    sB = __builtin_fmaf(gk, bv[k], sB);
                    sC = __builtin_fmaf(cv[k], hs[i + 1][k], sC);
                    g[k] = gk * as[i][k];
                    const float x = g[k] * hs[i][k];
                    sA = __builtin_fmaf(x, A2[k], sA);
                    dA[k] = __builtin_fmaf(x, dv, dA[k]);
                }
                sB = group_sum_all<NS>(sB);
                sA = group_sum_all<NS>(sA);
                sC = group_sum_all<NS>(sC);
                if (ng == 0) {
                    s_d[r][c] = sB;
                    s_du[r][c] = sA * (1.f / kLog2e);
                    s_e[r][c] = sC;
                }
                // over the wave's channels: lanes ng, ng + NS, ...
#pragma unroll
                for (int k = 0; k < 4; ++k) {
#pragma unroll
                    for (int o = NS; o < 64; o <<= 1) {
                        vb[k] += __shfl_xor(vb[k], o, 64);
                        vc[k] += __shfl_xor(vc[k], o, 64);
                    }
                }
                if (lane < NS) {
                    *(float4*)&s_bc[wave][i][4 * ng] = make_float4(vb[0], vb[1], vb[2], vb[3]);
                    *(float4*)&s_bc[wave][i][NP + 4 * ng] = make_float4(vc[0], vc[1], vc[2], vc[3]);
                }
            }
            __syncthreads();
            for (int i = threadIdx.x; i < kSub * 2 * NP; i += 256) {
                const int r = i / (2 * NP), k = i % (2 * NP);
                if (j * kSub + r < n)
                    pBC[(t + j * kSub + r) * 2 * NP + k] =
                        (s_bc[0][r][k] + s_bc[1][r][k]) + (s_bc[2][r][k] + s_bc[3][r][k]);
            }
            __syncthreads();
        }
        // ---- the gradients of the elements
        for (int r = m.row; r < n; r += TT) {
            float uv[4], dv[4], yv[4], zv[4], o1[4], o2[4], o3[4];
            ld_run<4, T>(static_cast<const T*>(p.u) + (t + r) * p.u_st + d0 + m.c4, nc, uv);
            ld_run<4, T>(static_cast<const T*>(p.dl) + (t + r) * p.dl_st + d0 + m.c4, nc, dv);
            ld_run<4, T>(static_cast<const T*>(p.dy) + (t + r) * p.dy_st + d0 + m.c4, nc, yv);
            if (p.z) ld_run<4, T>(static_cast<const T*>(p.z) + (t + r) * p.z_st + d0 + m.c4, nc, zv);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float raw = dv[k] + bias[k];
                const float dt = p.softplus ? pk_softplus(raw) : raw;
                const float sB = s_d[r][m.c4 + k], sA = s_du[r][m.c4 + k], sC = s_e[r][m.c4 + k];
                float ev = yv[k];
                if (p.z) {
                    const float sg = pk_sigmoid(zv[k]);
                    ev *= zv[k] * sg;
                    o3[k] = yv[k] * __builtin_fmaf(Dv[k], uv[k], sC) * (sg * (1.f + zv[k] * (1.f - sg)));
                }
                o1[k] = __builtin_fmaf(sB, dt, Dv[k] * ev);
                o2[k] = __builtin_fmaf(sB, uv[k], sA);
                if (p.softplus) o2[k] *= pk_sigmoid(raw);
                dD[k] = __builtin_fmaf(ev, uv[k], dD[k]);
                db[k] += o2[k];
            }
            st_run<4, T>(static_cast<T*>(p.du) + (t + r) * p.du_st + d0 + m.c4, nc, o1);
            st_run<4, T>(static_cast<T*>(p.ddl) + (t + r) * p.ddl_st + d0 + m.c4, nc, o2);
            if (p.z) st_run<4, T>(static_cast<T*>(p.dz) + (t + r) * p.dz_st + d0 + m.c4, nc, o3);
        }
        if (t == st) store_state(p.dh0, s, p, d, ng, g);
        t = b;
        __syncthreads();
    }
    outside(t, e.c1);
    // ---- the chunk's share of dA, dD and dbias
    if (d < p.D) *plane<NP>(p.pA, ck, p, d, ng) = make_float4(dA[0], dA[1], dA[2], dA[3]);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        s_d[m.row][m.c4 + k] = dD[k];
        s_du[m.row][m.c4 + k] = db[k];
    }
    __syncthreads();
    if (threadIdx.x < CPB && d0 + (int)threadIdx.x < p.D) {
        float x = 0.f, y = 0.f;
        for (int r = 0; r < TT; ++r) {
            x += s_d[r][threadIdx.x];
            y += s_du[r][threadIdx.x];
        }
        p.pD[ck * p.D + d0 + threadIdx.x] = x;
        p.pb[ck * p.D + d0 + threadIdx.x] = y;
    }
}

// The joins, each in a fixed order: dB and dC over the channel blocks (a thread
// per row and state) ...
template <typename T, int NP>
__global__ __launch_bounds__(256) void scan_pk_join_bc(ScanPk p, int nblk) {
    const int64_t total = p.rows * 2 * NP;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        float s = 0.f;
        for (int b = 0; b < nblk; ++b) s += p.pBC[b * total + i];
        const int64_t t = i / (2 * NP);
        const int k = (int)(i - t * 2 * NP), n = k % NP;
        if (n >= p.N) continue;
        if (k < NP) store_f32<T>(static_cast<T*>(p.dB) + t * p.dB_st + n, s);
        else store_f32<T>(static_cast<T*>(p.dC) + t * p.dC_st + n, s);
    }
}

// ... and dA, dD, dbias over the chunks: column j of [D][NP] | [D] | [D].
template <int NP>
__global__ __launch_bounds__(256) void scan_pk_join_par(ScanPk p) {
    __shared__ float red[4][64];
    const int64_t j = blockIdx.x * 64ll + (threadIdx.x & 63), nA = (int64_t)p.D * NP;
    const int q = threadIdx.x >> 6;
    const float* src = j < nA ? p.pA + j : j < nA + p.D ? p.pD + (j - nA) : p.pb + (j - nA - p.D);
    const int64_t pitch = j < nA ? nA : p.D;
    const bool live = j < nA + 2 * p.D;
    float s = 0.f;
    if (live)
        for (int64_t ck = q; ck < p.nchunk; ck += 4) s += src[ck * pitch];
    red[q][threadIdx.x & 63] = s;
    __syncthreads();
    if (q || !live) return;
    s = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
    if (j < nA) {
        const int64_t d = j / NP;
        const int n = (int)(j % NP);
        if (n < p.N) p.dA[d * p.N + n] = s;
    } else if (j < nA + p.D) {
        if (p.dD) p.dD[j - nA] = s;
    } else if (p.db) {
        p.db[j - nA - p.D] = s;
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

template <typename T>
__global__ __launch_bounds__(256) void scan_slot_step(ScanSlotParams p) {
    const int b = blockIdx.y, d = blockIdx.x * 256 + threadIdx.x;
    if (d >= p.D) return;
    T* y = static_cast<T*>(p.y) + b * p.y_sb + d;
    const int64_t slot = slot_of(p.slots, b, p.nslots);
    if (slot < 0) {
        store_f32<T>(y, 0.f);
        return;
    }
    const float u = load_f32<T>(static_cast<const T*>(p.u) + b * p.u_sb + d);
    float dv = load_f32<T>(static_cast<const T*>(p.dl) + b * p.dl_sb + d);
    if (p.bias) dv += p.bias[d];
    if (p.softplus) dv = pk_softplus(dv);
    float* h = p.state + (slot * p.D + d) * p.N;
    float acc = 0.f;
    for (int n = 0; n < p.N; ++n) {
        const float bv = load_f32<T>(static_cast<const T*>(p.B) + b * p.B_sb + n);
        const float cv = load_f32<T>(static_cast<const T*>(p.C) + b * p.C_sb + n);
        const float hn = __builtin_fmaf(h[n], __builtin_amdgcn_exp2f(dv * (p.A[(int64_t)d * p.N + n] * kLog2e)), dv * u * bv);
        h[n] = hn;
        acc = __builtin_fmaf(hn, cv, acc);
    }
    if (p.Dv) acc = __builtin_fmaf(p.Dv[d], u, acc);
    if (p.z) {
        const float zv = load_f32<T>(static_cast<const T*>(p.z) + b * p.z_sb + d);
        acc *= zv * pk_sigmoid(zv);
    }
    store_f32<T>(y, acc);
}

// ---------------------------------------------------------------- dispatch ---

static int scan_np(int N) { return N <= 16 ? 16 : N <= 32 ? 32 : 64; }

static int scan_pk_make(const mamba1_scan_packed_args* a, ScanPk* o) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    MAMBA_CHECK_ARG(a->rows >= 0 && a->rows < (1ll << 31), "rows must be in [0, 2^31)");
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
    ScanPk& p = *o;
    p = ScanPk{};
    p.q = Seqs{a->cu_seqlens, a->nseq, a->rows};
    p.rows = a->rows; p.D = a->dim; p.N = a->dstate;
    p.softplus = a->delta_softplus != 0; p.fill = a->fill_outside != 0;
    p.u = a->u; p.u_st = a->u_st; p.dl = a->delta; p.dl_st = a->delta_st; p.z = a->z; p.z_st = a->z_st;
    p.B = a->B; p.B_st = a->B_st; p.C = a->C; p.C_st = a->C_st;
    p.A = a->A; p.Dv = a->D; p.bias = a->delta_bias;
    return MAMBA_OK;
}

static void scan_pk_fwd_plan(ScanPk& p) {
    p.chunk = 128;
    p.nchunk = (p.rows + p.chunk - 1) / p.chunk;
}
static void scan_pk_bwd_plan(ScanPk& p) {
    p.chunk = kBwdChunk;
    p.nchunk = (p.rows + p.chunk - 1) / p.chunk;
}
// a grid's threads stay below 2^32
static int scan_pk_grid_ok(const ScanPk& p) {
    const int64_t nblk = ceil_div(p.D, 1024 / scan_np(p.N));
    if (p.nchunk * nblk >= (1ll << 24)) {
        set_error("mamba1_scan_packed: rows * dim is too large for one call");
        return MAMBA_ERR_UNSUPPORTED;
    }
    return MAMBA_OK;
}

template <typename T, int NP>
static void scan_pk_fwd_launch(const ScanPk& p, hipStream_t s) {
    const uint32_t nblk = ceil_div(p.D, ScanShape<NP>::CPB);
    if (p.nchunk > 1) {
        hipLaunchKernelGGL((scan_pk_state<T, NP>), dim3(nblk * (uint32_t)(p.nchunk - 1)), dim3(256), 0, s, p);
        hipLaunchKernelGGL((scan_pk_carry<NP>), dim3(ceil_div(p.D * NP, 256)), dim3(256), 0, s, p);
    }
    hipLaunchKernelGGL((scan_pk_out<T, NP>), dim3(nblk * (uint32_t)p.nchunk), dim3(256), 0, s, p);
}

template <typename T, int NP>
static void scan_pk_bwd_launch(const ScanPk& p, hipStream_t s) {
    const uint32_t nblk = ceil_div(p.D, ScanShape<NP>::CPB);
    if (p.nchunk > 1) {
        hipLaunchKernelGGL((scan_pk_state_bwd<T, NP>), dim3(nblk * (uint32_t)p.nchunk), dim3(256), 0, s, p);
        hipLaunchKernelGGL((scan_pk_carry_bwd<NP>), dim3(ceil_div(p.D * NP, 256), 2), dim3(256), 0, s, p);
    }
    if (p.rows) {
        hipLaunchKernelGGL((scan_pk_bwd<T, NP>), dim3(nblk * (uint32_t)p.nchunk), dim3(256), 0, s, p);
        const int64_t n = p.rows * 2 * NP;
        hipLaunchKernelGGL((scan_pk_join_bc<T, NP>), dim3((uint32_t)std::min<int64_t>((n + 255) / 256, 8192)), dim3(256), 0, s, p,
                           (int)nblk);
    }
    hipLaunchKernelGGL((scan_pk_join_par<NP>), dim3((uint32_t)(((int64_t)p.D * (NP + 2) + 63) / 64)), dim3(256), 0, s, p);
}

#define SCAN_PK_DISPATCH(fn, np, bf16, ...)              \
    do {                                                 \
        if ((np) == 16) {                                \
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

// floats of the forward's planes
static size_t scan_pk_fwd_floats(const ScanPk& p) {
    return p.nchunk > 1 ? (size_t)p.nchunk * p.D * (2 * scan_np(p.N) + 1) : 0;
}
static size_t scan_pk_bwd_floats(const ScanPk& p) {
    const size_t np = scan_np(p.N), nblk = ceil_div(p.D, 1024 / (int)np);
    return (size_t)p.nchunk * p.D * (3 * np + 3) + nblk * (size_t)p.rows * 2 * np;
}

}  // namespace mamba

using namespace mamba;

extern "C" size_t mamba1_scan_packed_workspace_size(const mamba1_scan_packed_args* a) {
    ScanPk p;
    if (scan_pk_make(a, &p) != MAMBA_OK) return 0;
    scan_pk_fwd_plan(p);
    return scan_pk_fwd_floats(p) * 4;
}

extern "C" int mamba1_scan_packed_fwd(const mamba1_scan_packed_args* a, void* ws, size_t ws_bytes, mamba_stream_t stream) {
    ScanPk p;
    int st = scan_pk_make(a, &p);
    if (st != MAMBA_OK) return st;
    if (p.rows == 0) return MAMBA_OK;
    MAMBA_CHECK_ARG(a->y != nullptr, "y is required");
    MAMBA_CHECK_ARG(a->y_st >= p.D || p.rows == 1, "rows of y overlap");
    MAMBA_CHECK_ARG(a->state == nullptr || a->slots != nullptr || a->nslots >= a->nseq,
                    "without slots the state needs a row per sequence");
    p.y = a->y; p.y_st = a->y_st;
    p.state = a->state; p.nslots = a->nslots; p.slots = a->slots;
    scan_pk_fwd_plan(p);
    if ((st = scan_pk_grid_ok(p)) != MAMBA_OK) return st;
    const size_t need = scan_pk_fwd_floats(p) * 4;
    MAMBA_CHECK_ARG(((uintptr_t)ws & 15u) == 0, "the workspace must be 16-byte aligned");
    if (need && (ws == nullptr || ws_bytes < need)) {
        set_error("mamba1_scan_packed_fwd: workspace missing or too small");
        return MAMBA_ERR_WORKSPACE;
    }
    const size_t pl = (size_t)p.nchunk * p.D * scan_np(p.N);
    p.E = static_cast<float*>(ws);
    p.h0c = p.E + pl;
    p.sumd = p.h0c + pl;
    SCAN_PK_DISPATCH(scan_pk_fwd_launch, scan_np(p.N), a->io_dtype == MAMBA_BF16, p, (hipStream_t)stream);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}

extern "C" size_t mamba1_scan_packed_bwd_workspace_size(const mamba1_scan_packed_bwd_args* a) {
    ScanPk p;
    if (a == nullptr || scan_pk_make(&a->fwd, &p) != MAMBA_OK) return 0;
    scan_pk_bwd_plan(p);
    return scan_pk_bwd_floats(p) * 4;
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
    p.dy = a->dy; p.dy_st = a->dy_st; p.h0 = a->initial_state; p.dhT = a->d_final_state;
    p.du = a->du; p.du_st = a->du_st; p.ddl = a->ddelta; p.ddl_st = a->ddelta_st; p.dz = a->dz; p.dz_st = a->dz_st;
    p.dB = a->dB; p.dB_st = a->dB_st; p.dC = a->dC; p.dC_st = a->dC_st;
    p.dA = a->dA; p.dD = a->dD; p.db = a->d_delta_bias; p.dh0 = a->d_initial_state;
    scan_pk_bwd_plan(p);
    if ((st = scan_pk_grid_ok(p)) != MAMBA_OK) return st;
    const size_t need = scan_pk_bwd_floats(p) * 4;
    MAMBA_CHECK_ARG(((uintptr_t)ws & 15u) == 0, "the workspace must be 16-byte aligned");
    if (need && (ws == nullptr || ws_bytes < need)) {
        set_error("mamba1_scan_packed_bwd: workspace missing or too small");
        return MAMBA_ERR_WORKSPACE;
    }
    const size_t np = scan_np(p.N), nd = (size_t)p.nchunk * p.D;
    p.E = static_cast<float*>(ws);
    p.G = p.E + nd * np;
    p.pA = p.G + nd * np;
    p.pBC = p.pA + nd * np;
    p.sumd = p.pBC + (size_t)ceil_div(p.D, 1024 / (int)np) * p.rows * 2 * np;
    p.pD = p.sumd + nd;
    p.pb = p.pD + nd;
    SCAN_PK_DISPATCH(scan_pk_bwd_launch, (int)np, a->fwd.io_dtype == MAMBA_BF16, p, (hipStream_t)stream);
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
    ScanSlotParams p{};
    p.nb = a->batch; p.D = a->dim; p.N = a->dstate; p.softplus = a->delta_softplus != 0;
    p.u = a->u; p.u_sb = a->u_sb; p.dl = a->delta; p.dl_sb = a->delta_sb; p.z = a->z; p.z_sb = a->z_sb;
    p.B = a->B; p.B_sb = a->B_sb; p.C = a->C; p.C_sb = a->C_sb;
    p.A = a->A; p.Dv = a->D; p.bias = a->delta_bias;
    p.state = a->state; p.nslots = a->nslots; p.slots = a->slots; p.y = a->y; p.y_sb = a->y_sb;
    const dim3 grid(ceil_div(p.D, 256), p.nb);
    if (a->io_dtype == MAMBA_BF16) hipLaunchKernelGGL(scan_slot_step<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(scan_slot_step<float>, grid, dim3(256), 0, (hipStream_t)stream, p);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}
