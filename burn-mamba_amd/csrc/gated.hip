// Gated linear recurrence over packed sequences for gfx950, one state a channel:
// forward, backward, and single tokens on a cache addressed by slot.  f32 or bf16 rows
// (channels contiguous), f32 states, A and its gradient.
//
//   a_t = exp(A s(r_t)),  m_t = sqrt(1 - a_t^2),  u_t = s(i_t) x_t
//   h_t = a_t h_{t-1} + m_t u_t,  y_t = h_t silu(z_t) (or h_t)
// Backward, with g_t = dy_t silu(z_t) (dhT added at a sequence's last row):
//   dh_t = g_t + q_{t+1},  q_t = a_t dh_t,  e_t = dh_t (a_t h_{t-1} - u_t a_t^2 / m_t)
//   dx = dh m s(i),  di = dh m u s(-i),  dr = e A s(r) s(-r),  dA = sum_t e s(r)
//   dz = dy h silu'(z),  dh0 = q at a sequence's first row
//
// With one state a channel some 30 (forward) to 90 (backward) operations stand against 8 to
// 18 bytes an element of bf16, so memory bounds it, and every row is read once: the rows are
// cut into tiles (of 64; the forward of bf16: 128) without regard to the sequences, a workgroup
// takes one tile of 128 channels, keeps it in registers, and finds the state that enters it while the tile is there.
// A stretch of rows maps the state that enters it, h -> P h + H; P is the product of its
// decays and H what it leaves from zero.  A lane holds R rows of two channels; its map and
// the maps of the eight waves are joined in LDS to the tile's, which is published to the
// other workgroups before the tile's own state is waited for.  That state is joined from the
// published maps of the tiles before it, back to the one in which the tile's first sequence
// begins, or to the last group of 32 tiles, whose final state its last tile publishes.  The
// joins follow a fixed order: the same inputs give the same bits.  The backward walks the other way
// with q in the state's place, and finds h again from the states that the forward kept.
//
// A map is published as one 64-bit word (P, H) and read with relaxed atomics of the whole card:
// the word is its own flag, all ones until it is written (P of a NaN is made the usual one, so
// that no map has that value).  A workgroup takes its tile by ticket, so the tiles that it waits
// for belong to workgroups that run already, and those publish before they wait: every wait ends.
#include <algorithm>

#include "pack.h"

namespace mamba {

struct GatedP {
    Seqs q;
    int64_t rows;
    int D;
    bool fill;
    const void* x; int64_t x_st;
    const void* r; int64_t r_st;
    const void* i; int64_t i_st;
    const void* z; int64_t z_st;
    const float* A;
    float* state; int64_t nslots; const int32_t* slots;
    float* carry;                       // [ceil(rows / kCarryRows), D]
    void* y; int64_t y_st;
    // backward
    const float* h0;
    const void* dy; int64_t dy_st;
    const float* dhT;
    void* dx; int64_t dx_st;
    void* dr; int64_t dr_st;
    void* di; int64_t di_st;
    void* dz; int64_t dz_st;
    float* dA; float* dh0;
    // tiles of rows and of channels; the workspace
    int ntile, nct;
    uint32_t* ticket;
    uint64_t* map;                      // [ntile][nct kGC] published maps
    uint64_t* ends;                     // [ntile / kGGroup][nct kGC] states at the ends of groups
    float* part;                        // [ntile][D] partial sums of dA
};

constexpr int kCarryRows = 64;  // rows between the states that the forward keeps for the backward
constexpr int kGW = 8, kGV = 2, kGC = 64 * kGV;  // waves of a workgroup, channels of a lane and of a tile
constexpr int kGGroup = 32;                      // tiles of a group
constexpr uint64_t kGNone = ~0ull;               // nothing published yet
// rows of a lane: a tile of the backward has kCarryRows, one of the forward as many or twice that
constexpr int kGRows = kCarryRows / kGW;
template <typename T>
constexpr int kGFwdRows = sizeof(T) == 2 ? 2 * kGRows : kGRows;

// s(v) = 1 / (1 + exp(-v)) and s(-v) = 1 - s(v), by the hardware's exp2 and reciprocal (one
// step each); 0 and 1 at the ends.  s(-v) of a large v is exp(-v) s(v): the difference from 1
// would lose its size.
__device__ __forceinline__ float g_sigmoid(float v) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.44269504088896341f));
}
struct Logistic { float s, c; };
__device__ __forceinline__ Logistic g_logistic(float v) {
    const float e = __builtin_amdgcn_exp2f(v * -1.44269504088896341f), s = __builtin_amdgcn_rcpf(1.f + e);
    return {s, v > 0.f ? e * s : 1.f - s};
}

// a = exp(v) and q = 1 - a^2 for v <= 0, both to a few steps of their own size.  From -1/8 up by
// e = exp(v) - 1, the series to v^5 / 5! (its next term is 2^-24 of the sum there): a = 1 + e,
// 1 - a^2 = -e (2 + e) keep what a difference from 1 would lose as a nears 1.  The exponential,
// for what lies below, is passed over where no lane needs it.
struct Decay { float a, q; };
__device__ __forceinline__ Decay g_decay(float v) {
    float e = 1.f / 120.f;
    e = __builtin_fmaf(e, v, 1.f / 24.f);
    e = __builtin_fmaf(e, v, 1.f / 6.f);
    e = __builtin_fmaf(e, v, 0.5f);
    e = __builtin_fmaf(e, v, 1.f) * v;
    Decay d = {1.f + e, -e * (2.f + e)};
    const bool near = v >= -0.125f;  // not of a NaN
    if (__ballot(!near)) {
        const float far = __builtin_amdgcn_exp2f(v * 1.44269504088896341f);
        d.a = near ? d.a : far;
        d.q = near ? d.q : __builtin_fmaf(-far, far, 1.f);
    }
    return d;
}

// What the R rows from t0 are (R <= 64, t0 uniform over the wave): bit j of a mask for row
// t0 + j, whether it is in a sequence, its first, its last; lane j holds the row's sequence and
// that one's first row and end.  The offsets are clamped: a wrong one gives a wrong result and
// no access out of range.
struct GRows {
    uint64_t live, first, last;
    int s, b, e;
};
__device__ __forceinline__ GRows g_rows(const Seqs& q, int t0, int R) {
    const int j = threadIdx.x & 63, t = t0 + j;
    int lo = 0, hi = q.n;
    while (lo < hi) {  // the first sequence that ends behind row t
        const int mid = (lo + hi) >> 1;
        if (q.cu[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    GRows o;
    o.s = lo;
    o.b = o.e = 0;
    const bool in = j < R && t < q.rows && lo < q.n;
    if (in) {
        o.b = min(max(q.cu[lo], 0), q.rows);
        o.e = min(max(q.cu[lo + 1], o.b), q.rows);
    }
    const bool live = in && t >= o.b && t < o.e;
    o.live = __ballot(live);
    o.first = __ballot(live && t == o.b);
    o.last = __ballot(live && t == o.e - 1);
    return o;
}
__device__ __forceinline__ int g_lane(int v, int j) { return __builtin_amdgcn_readlane(v, j); }
__device__ __forceinline__ bool g_bit(uint64_t m, int j) { return (m >> j) & 1; }

__device__ __forceinline__ uint64_t g_word(float P, float H) {
    uint32_t p = __float_as_uint(P);
    if ((p & 0x7fffffffu) > 0x7f800000u) p = 0x7fc00000u;  // never kGNone
    return (uint64_t)__float_as_uint(H) << 32 | p;
}
__device__ __forceinline__ void g_publish(uint64_t* at, uint64_t v) {
    __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t g_peek(const uint64_t* at) {
    return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// The word at `at`, waited for.  The wait is bounded (seconds: no run comes near) so that a card on
// which it could not end would give a NaN and no hang.
__device__ __forceinline__ uint64_t g_wait(const uint64_t* at, uint64_t v) {
    for (int i = 0; v == kGNone && i < (1 << 22); ++i) {
        __builtin_amdgcn_s_sleep(1);
        v = g_peek(at);
    }
    return v;
}

__global__ __launch_bounds__(256) void gated_clear(uint32_t* ticket, uint4* words, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i == 0) *ticket = 0;
    for (int64_t k = i; k < n; k += (int64_t)gridDim.x * 256) words[k] = make_uint4(~0u, ~0u, ~0u, ~0u);
}

struct GMap { float P[kGV], H[kGV]; };
struct GShared {
    float P[kGW][kGV][64], H[kGW][kGV][64];    // the waves' maps
    float P2[kGW][kGV][64], H2[kGW][kGV][64];  // joined runs of tiles; the backward's sums
    float in[kGV][64];                         // the group's entry
    int cut[kGW];                              // whether a wave's rows cut the state that enters them off
    int tile, far;
};

// The tile of this workgroup (in the order in which the tiles wait for one another) and its channels.
__device__ __forceinline__ void g_tile(const GatedP& p, GShared& s, int& o, int& ct) {
    if (p.ntile > 1) {
        if (threadIdx.x == 0) s.tile = (int)atomicAdd(p.ticket, 1u);
        __syncthreads();
        const int k = __builtin_amdgcn_readfirstlane(s.tile);
        o = k / p.nct;
        ct = k - o * p.nct;
    } else {
        o = 0;
        ct = blockIdx.x;
    }
}

// The state that enters tile o: joined from the maps of tiles far .. o - 1, tile `far` being cut, or
// from the end of the group before o's.  Called by the whole workgroup (o > far >= 0).
__device__ __forceinline__ void g_enter(const GatedP& p, GShared& s, int o, int ct, int far, float (&h)[kGV]) {
    const int w = wave_id(), l = threadIdx.x & 63;
    const int64_t Dp = (int64_t)p.nct * kGC, at = (int64_t)ct * kGC + l;
    const int base = o / kGGroup * kGGroup, from = max(far, base);
    const bool group = far < base;
    const int per = (o - from + kGW - 1) / kGW, k0 = min(o, from + w * per), k1 = min(o, k0 + per);
    GMap m;
#pragma unroll
    for (int v = 0; v < kGV; ++v) m.P[v] = 1.f, m.H[v] = 0.f;
    uint64_t word[kGGroup / kGW][kGV], end[kGV];
#pragma unroll
    for (int i = 0; i < kGGroup / kGW; ++i)
#pragma unroll
        for (int v = 0; v < kGV; ++v) word[i][v] = k0 + i < k1 ? g_peek(p.map + (int64_t)(k0 + i) * Dp + at + 64 * v) : 0;
    const uint64_t* ends = p.ends + (int64_t)(base / kGGroup - 1) * Dp + at;
    if (group && w == 0) {
#pragma unroll
        for (int v = 0; v < kGV; ++v) end[v] = g_peek(ends + 64 * v);
    }
#pragma unroll
    for (int i = 0; i < kGGroup / kGW; ++i) {
        if (k0 + i >= k1) break;
#pragma unroll
        for (int v = 0; v < kGV; ++v) {
            const uint64_t x = g_wait(p.map + (int64_t)(k0 + i) * Dp + at + 64 * v, word[i][v]);
            const float P = __uint_as_float((uint32_t)x), H = __uint_as_float((uint32_t)(x >> 32));
            m.H[v] = i ? __builtin_fmaf(P, m.H[v], H) : H;
            m.P[v] = i ? P * m.P[v] : P;
        }
    }
    if (group && w == 0) {
#pragma unroll
        for (int v = 0; v < kGV; ++v) s.in[v][l] = __uint_as_float((uint32_t)(g_wait(ends + 64 * v, end[v]) >> 32));
    }
#pragma unroll
    for (int v = 0; v < kGV; ++v) s.P2[w][v][l] = m.P[v], s.H2[w][v][l] = m.H[v];
    __syncthreads();
#pragma unroll
    for (int v = 0; v < kGV; ++v) {
        h[v] = group ? __builtin_fmaf(s.P2[0][v][l], s.in[v][l], s.H2[0][v][l]) : s.H2[0][v][l];  // a cut tile's P is no factor
        for (int k = 1; k < kGW && from + k * per < o; ++k) h[v] = __builtin_fmaf(s.P2[k][v][l], h[v], s.H2[k][v][l]);
    }
}

// Two channels of a row from column c: loaded whole by every lane, those past the row's end from
// its last two channels, so that no load has a branch of its own.  MODE 0: an even number of
// channels; 1: an odd one, whose last lane takes the second of the two; 2: a single channel.
template <int MODE>
__device__ __forceinline__ int g_column(int c, int D) { return MODE == 2 ? c : min(c, D - kGV); }
// (row: uniform; an unsigned offset keeps the address a scalar base and one register)
template <typename T, int MODE>
__device__ __forceinline__ void g_load(Elems<T, kGV>& e, const T* row, int cl, int n) {
    const T* at = reinterpret_cast<const T*>(reinterpret_cast<const char*>(row) + (uint32_t)cl * (uint32_t)sizeof(T));
    if constexpr (MODE == 2) e.load_part(at, n);
    else e.load(at);
}
template <typename T>
__device__ __forceinline__ void g_store(T* row, int c, int n, const float (&v)[kGV]) {
    st_run<kGV, T>(reinterpret_cast<T*>(reinterpret_cast<char*>(row) + (uint32_t)c * (uint32_t)sizeof(T)), n, v);
}

template <typename T, int MODE>
__global__ __launch_bounds__(64 * kGW, 4) void gated_fwd(GatedP p) {
    constexpr int R = kGFwdRows<T>;
    __shared__ GShared s;
    int o, ct;
    g_tile(p, s, o, ct);
    const int w = wave_id(), l = threadIdx.x & 63;
    const int row0 = o * (kGW * R), t0 = row0 + w * R, c = ct * kGC + l * kGV, n = p.D - c;
    const int rows = min(R, max(0, (int)p.rows - t0));  // of this wave
    Elems<T, kGV> ex[R], er[R], ei[R], ez[R];
    const int cl = g_column<MODE>(c, p.D);
    auto fetch = [&](Elems<T, kGV> (&e)[R], const void* q, int64_t st) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < R; ++j) g_load<T, MODE>(e[j], static_cast<const T*>(q) + (int64_t)min(t0 + j, (int)p.rows - 1) * st, cl, n);
    };
    auto get = [&](const Elems<T, kGV>& e, float (&v)[kGV]) __attribute__((always_inline)) {
        e.get(v);
        if (MODE == 1 && n == 1) v[0] = v[1];
    };
    fetch(er, p.r, p.r_st);
    fetch(ei, p.i, p.i_st);
    fetch(ex, p.x, p.x_st);
    const GRows g = g_rows(p.q, t0, R);
    float A[kGV];
#pragma unroll
    for (int v = 0; v < kGV; ++v) A[v] = v < n ? p.A[c + v] : 0.f;
    constexpr uint64_t full = (1ull << R) - 1;
    const bool plain = g.live == full && (g.first | g.last) == 0;
    float a[R][kGV], b[R][kGV];
#pragma unroll
    for (int j = 0; j < R; ++j) {
        float r[kGV], i[kGV], x[kGV];
        get(er[j], r);
        get(ei[j], i);
        get(ex[j], x);
#pragma unroll
        for (int v = 0; v < kGV; ++v) {
            const Decay d = g_decay(A[v] * g_sigmoid(r[v]));
            a[j][v] = d.a;
            b[j][v] = __builtin_amdgcn_sqrtf(d.q) * (g_sigmoid(i[v]) * x[v]);
        }
    }
    GMap m;
#pragma unroll
    for (int v = 0; v < kGV; ++v) m.P[v] = 1.f, m.H[v] = 0.f;
    if (plain) {
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int v = 0; v < kGV; ++v) {
                m.H[v] = __builtin_fmaf(a[j][v], m.H[v], b[j][v]);
                m.P[v] *= a[j][v];
            }
    } else {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (g_bit(g.first, j)) {  // from the sequence's state on; b holds the new one
                const int64_t slot = p.state ? slot_of(p.slots, g_lane(g.s, j), p.nslots) : -1;
#pragma unroll
                for (int v = 0; v < kGV; ++v) {
                    const float h0 = slot >= 0 && v < n ? p.state[slot * p.D + c + v] : 0.f;
                    m.H[v] = b[j][v] = __builtin_fmaf(a[j][v], h0, b[j][v]);
                }
            } else if (g_bit(g.live, j)) {
#pragma unroll
                for (int v = 0; v < kGV; ++v) {
                    m.H[v] = __builtin_fmaf(a[j][v], m.H[v], b[j][v]);
                    m.P[v] *= a[j][v];
                }
            } else {
#pragma unroll
                for (int v = 0; v < kGV; ++v) m.H[v] = 0.f;
            }
        }
    }
#pragma unroll
    for (int v = 0; v < kGV; ++v) s.P[w][v][l] = m.P[v], s.H[w][v][l] = m.H[v];
    if (l == 0) s.cut[w] = g.live != full || g.first != 0;
    if (w == 0 && l == 0) s.far = (g.live & ~g.first & 1) ? g.b / (kGW * R) : -1;
    if (p.z) fetch(ez, p.z, p.z_st);
    __syncthreads();
    float h[kGV] = {0.f, 0.f};
    const int64_t at = ((int64_t)o * p.nct + ct) * kGC + l;
    const bool ends = (o + 1) % kGGroup == 0 && o + 1 < p.ntile;
    GMap whole;
    bool cut = false;
    if (w == kGW - 1 && p.ntile > 1) {
#pragma unroll
        for (int v = 0; v < kGV; ++v) whole.P[v] = 1.f, whole.H[v] = 0.f;
        for (int k = 0; k < kGW; ++k) {
            const bool here = s.cut[k] != 0;
            cut |= here;
#pragma unroll
            for (int v = 0; v < kGV; ++v) {
                whole.H[v] = here ? s.H[k][v][l] : __builtin_fmaf(s.P[k][v][l], whole.H[v], s.H[k][v][l]);
                whole.P[v] *= s.P[k][v][l];
            }
        }
#pragma unroll
        for (int v = 0; v < kGV; ++v) g_publish(p.map + at + 64 * v, g_word(whole.P[v], whole.H[v]));
    }
    const int far = __builtin_amdgcn_readfirstlane(s.far);
    if (far >= 0) g_enter(p, s, o, ct, far, h);
    if (w == kGW - 1 && ends) {
#pragma unroll
        for (int v = 0; v < kGV; ++v)
            g_publish(p.ends + ((int64_t)(o / kGGroup) * p.nct + ct) * kGC + l + 64 * v, g_word(0.f, cut ? whole.H[v] : __builtin_fmaf(whole.P[v], h[v], whole.H[v])));
    }
    for (int k = 0; k < w; ++k) {
        const bool here = s.cut[k] != 0;
#pragma unroll
        for (int v = 0; v < kGV; ++v) h[v] = here ? s.H[k][v][l] : __builtin_fmaf(s.P[k][v][l], h[v], s.H[k][v][l]);
    }
    if (p.carry && t0 % kCarryRows == 0 && rows > 0) st_run<kGV, float>(p.carry + (int64_t)(t0 / kCarryRows) * p.D + c, n, h);
    auto put = [&](int j) __attribute__((always_inline)) {
        float y[kGV];
        if (p.z) {
            float z[kGV];
            get(ez[j], z);
#pragma unroll
            for (int v = 0; v < kGV; ++v) y[v] = h[v] * z[v] * g_sigmoid(z[v]);
        } else {
#pragma unroll
            for (int v = 0; v < kGV; ++v) y[v] = h[v];
        }
        g_store<T>(static_cast<T*>(p.y) + (t0 + j) * p.y_st, c, n, y);
    };
    if (plain) {
#pragma unroll
        for (int j = 0; j < R; ++j) {
#pragma unroll
            for (int v = 0; v < kGV; ++v) h[v] = __builtin_fmaf(a[j][v], h[v], b[j][v]);
            put(j);
        }
    } else {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (!g_bit(g.live, j)) {
#pragma unroll
                for (int v = 0; v < kGV; ++v) h[v] = 0.f;
                if (p.fill && j < rows) g_store<T>(static_cast<T*>(p.y) + (t0 + j) * p.y_st, c, n, h);
                continue;
            }
#pragma unroll
            for (int v = 0; v < kGV; ++v) h[v] = g_bit(g.first, j) ? b[j][v] : __builtin_fmaf(a[j][v], h[v], b[j][v]);
            put(j);
            if (g_bit(g.last, j) && p.state) {
                const int64_t slot = slot_of(p.slots, g_lane(g.s, j), p.nslots);
                if (slot >= 0) st_run<kGV, float>(p.state + slot * p.D + c, n, h);
            }
        }
    }
}

template <typename T, int MODE>
__global__ __launch_bounds__(64 * kGW, 2) void gated_bwd(GatedP p) {
    constexpr int R = kGRows;
    __shared__ GShared s;
    int o, ct;
    g_tile(p, s, o, ct);
    const int tile = p.ntile - 1 - o;  // from the last one on
    const int w = wave_id(), l = threadIdx.x & 63;
    const int row0 = tile * kCarryRows, t0 = row0 + w * R, c = ct * kGC + l * kGV, n = p.D - c;
    const int rows = min(R, max(0, (int)p.rows - t0));
    Elems<T, kGV> ex[R], er[R], ei[R], ez[R], ey[R];
    const int cl = g_column<MODE>(c, p.D);
    auto fetch = [&](Elems<T, kGV> (&e)[R], const void* q, int64_t st) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < R; ++j) g_load<T, MODE>(e[j], static_cast<const T*>(q) + (int64_t)min(t0 + j, (int)p.rows - 1) * st, cl, n);
    };
    auto get = [&](const Elems<T, kGV>& e, float (&v)[kGV]) __attribute__((always_inline)) {
        e.get(v);
        if (MODE == 1 && n == 1) v[0] = v[1];
    };
    fetch(er, p.r, p.r_st);
    fetch(ei, p.i, p.i_st);
    fetch(ex, p.x, p.x_st);
    fetch(ey, p.dy, p.dy_st);
    if (p.z) fetch(ez, p.z, p.z_st);
    const GRows g = g_rows(p.q, t0, R);
    float A[kGV], hin[kGV] = {0.f, 0.f};
    ld_run<kGV, float>(p.A + c, n, A);
    ld_run<kGV, float>(p.carry + (int64_t)tile * p.D + c, n, hin);
    constexpr uint64_t full = (1ull << R) - 1;
    const bool plain = g.live == full && (g.first | g.last) == 0;
    float a[R][kGV], m[R][kGV], im[R][kGV], b[R][kGV];  // im: 1 / m; b: m u, and then the state before the row
#pragma unroll
    for (int j = 0; j < R; ++j) {
        float r[kGV], i[kGV], x[kGV];
        get(er[j], r);
        get(ei[j], i);
        get(ex[j], x);
#pragma unroll
        for (int v = 0; v < kGV; ++v) {
            const Decay d = g_decay(A[v] * g_sigmoid(r[v]));
            a[j][v] = d.a;
            const float q = d.q;
            im[j][v] = q > 0.f ? __builtin_amdgcn_rsqf(q) : q * 0.f;  // 0 where a is 1, a NaN of a NaN
            m[j][v] = q * im[j][v];
            b[j][v] = m[j][v] * (g_sigmoid(i[v]) * x[v]);
        }
    }
    auto start = [&](int j, float (&h)[kGV]) __attribute__((always_inline)) {  // what the sequence of row j starts from
#pragma unroll
        for (int v = 0; v < kGV; ++v) h[v] = 0.f;
        if (p.h0) ld_run<kGV, float>(p.h0 + (int64_t)g_lane(g.s, j) * p.D + c, n, h);
    };
    // the waves' maps of h
    GMap f, q;
#pragma unroll
    for (int v = 0; v < kGV; ++v) f.P[v] = 1.f, f.H[v] = 0.f, q.P[v] = 1.f, q.H[v] = 0.f;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        if (!plain && !g_bit(g.live, j)) {
#pragma unroll
            for (int v = 0; v < kGV; ++v) f.H[v] = 0.f;
        } else {
            if (!plain && g_bit(g.first, j)) start(j, f.H);
#pragma unroll
            for (int v = 0; v < kGV; ++v) {
                f.H[v] = __builtin_fmaf(a[j][v], f.H[v], b[j][v]);
                f.P[v] *= a[j][v];
            }
        }
    }
    // g of row j
    auto grad = [&](int j, const Logistic (&sz)[kGV], const float (&z)[kGV], const float (&dy)[kGV], float (&o_)[kGV]) __attribute__((always_inline)) {
#pragma unroll
        for (int v = 0; v < kGV; ++v) o_[v] = p.z ? dy[v] * z[v] * sz[v].s : dy[v];
        if (!plain && g_bit(g.last, j) && p.dhT) {
            float d[kGV];
            ld_run<kGV, float>(p.dhT + (int64_t)g_lane(g.s, j) * p.D + c, n, d);
#pragma unroll
            for (int v = 0; v < kGV; ++v) o_[v] += d[v];
        }
    };
    auto gate = [&](int j, Logistic (&sz)[kGV], float (&z)[kGV]) __attribute__((always_inline)) {
#pragma unroll
        for (int v = 0; v < kGV; ++v) z[v] = 0.f, sz[v] = Logistic{0.f, 0.f};
        if (p.z) {
            get(ez[j], z);
#pragma unroll
            for (int v = 0; v < kGV; ++v) sz[v] = g_logistic(z[v]);
        }
    };
    // and of q
#pragma unroll
    for (int j = R - 1; j >= 0; --j) {
        if (!plain && !g_bit(g.live, j)) {
#pragma unroll
            for (int v = 0; v < kGV; ++v) q.H[v] = 0.f;
            continue;
        }
        Logistic sz[kGV];
        float z[kGV], dy[kGV], gr[kGV];
        gate(j, sz, z);
        get(ey[j], dy);
        grad(j, sz, z, dy, gr);
#pragma unroll
        for (int v = 0; v < kGV; ++v) {
            q.H[v] = a[j][v] * (gr[v] + q.H[v]);
            q.P[v] *= a[j][v];
            if (!plain && g_bit(g.first, j)) q.H[v] = 0.f;
        }
    }
#pragma unroll
    for (int v = 0; v < kGV; ++v) {
        s.P[w][v][l] = q.P[v], s.H[w][v][l] = q.H[v];
        s.P2[w][v][l] = f.P[v], s.H2[w][v][l] = f.H[v];
    }
    const bool cut_here = g.live != full || g.first != 0;
    if (l == 0) s.cut[w] = cut_here;
    // the tile's last row: its sequence's last tile, where that is another
    if (w == 0 && l == 0) s.far = -1;
    __syncthreads();
    const int lastrow = min((int)p.rows, row0 + kCarryRows) - 1 - t0;  // of the tile, counted from this wave's first
    if (lastrow >= 0 && lastrow < R && g_bit(g.live & ~g.last, lastrow) && l == 0)
        s.far = p.ntile - 1 - (g_lane(g.e, lastrow) - 1) / kCarryRows;
    // the state that enters this wave's rows
    float h[kGV] = {hin[0], hin[1]};
    for (int k = 0; k < w; ++k) {
        const bool here = s.cut[k] != 0;
#pragma unroll
        for (int v = 0; v < kGV; ++v) h[v] = here ? s.H2[k][v][l] : __builtin_fmaf(s.P2[k][v][l], h[v], s.H2[k][v][l]);
    }
    const int64_t at = ((int64_t)o * p.nct + ct) * kGC + l;
    const bool ends = (o + 1) % kGGroup == 0 && o + 1 < p.ntile;
    GMap whole;
    bool cut = false;
    if (w == 0 && p.ntile > 1) {
#pragma unroll
        for (int v = 0; v < kGV; ++v) whole.P[v] = 1.f, whole.H[v] = 0.f;
        for (int k = kGW - 1; k >= 0; --k) {
            const bool here = s.cut[k] != 0;
            cut |= here;
#pragma unroll
            for (int v = 0; v < kGV; ++v) {
                whole.H[v] = here ? s.H[k][v][l] : __builtin_fmaf(s.P[k][v][l], whole.H[v], s.H[k][v][l]);
                whole.P[v] *= s.P[k][v][l];
            }
        }
#pragma unroll
        for (int v = 0; v < kGV; ++v) g_publish(p.map + at + 64 * v, g_word(whole.P[v], whole.H[v]));
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {  // b: the state before the row
        if (!plain && !g_bit(g.live, j)) {
#pragma unroll
            for (int v = 0; v < kGV; ++v) h[v] = 0.f;
        } else {
            if (!plain && g_bit(g.first, j)) start(j, h);
#pragma unroll
            for (int v = 0; v < kGV; ++v) {
                const float after = __builtin_fmaf(a[j][v], h[v], b[j][v]);
                b[j][v] = h[v];
                h[v] = after;
            }
        }
    }
    __syncthreads();  // the waves' maps of h have been read, and far is known
    float qin[kGV] = {0.f, 0.f};
    const int far = __builtin_amdgcn_readfirstlane(s.far);
    if (far >= 0) g_enter(p, s, o, ct, far, qin);
    if (w == 0 && ends) {
#pragma unroll
        for (int v = 0; v < kGV; ++v)
            g_publish(p.ends + ((int64_t)(o / kGGroup) * p.nct + ct) * kGC + l + 64 * v, g_word(0.f, cut ? whole.H[v] : __builtin_fmaf(whole.P[v], qin[v], whole.H[v])));
    }
    for (int k = kGW - 1; k > w; --k) {
        const bool here = s.cut[k] != 0;
#pragma unroll
        for (int v = 0; v < kGV; ++v) qin[v] = here ? s.H[k][v][l] : __builtin_fmaf(s.P[k][v][l], qin[v], s.H[k][v][l]);
    }
    float dA[kGV] = {0.f, 0.f};
    auto put = [&](void* to, int64_t st, int j, const float (&v)[kGV]) __attribute__((always_inline)) {
        g_store<T>(static_cast<T*>(to) + (t0 + j) * st, c, n, v);
    };
#pragma unroll
    for (int j = R - 1; j >= 0; --j) {
        if (j >= rows) continue;
        if (!plain && !g_bit(g.live, j)) {
            const float zero[kGV] = {0.f, 0.f};
            put(p.dx, p.dx_st, j, zero);
            put(p.dr, p.dr_st, j, zero);
            put(p.di, p.di_st, j, zero);
            if (p.z) put(p.dz, p.dz_st, j, zero);
#pragma unroll
            for (int v = 0; v < kGV; ++v) qin[v] = 0.f;
            continue;
        }
        Logistic sz[kGV];
        float z[kGV], dy[kGV], gr[kGV], r[kGV], i[kGV], x[kGV], dx[kGV], dr[kGV], di[kGV], dz[kGV];
        gate(j, sz, z);
        get(ey[j], dy);
        grad(j, sz, z, dy, gr);
        get(er[j], r);
        get(ei[j], i);
        get(ex[j], x);
#pragma unroll
        for (int v = 0; v < kGV; ++v) {
            const Logistic sr = g_logistic(r[v]), si = g_logistic(i[v]);
            const float aj = a[j][v], mj = m[j][v], u = si.s * x[v], dh = gr[v] + qin[v], ah = aj * b[j][v], dm = dh * mj;
            const float pull = u * aj * aj * im[j][v];
            const float e = dh * (ah - pull);
            dx[v] = dm * si.s;
            di[v] = dm * u * si.c;
            dr[v] = e * A[v] * sr.s * sr.c;
            dA[v] = __builtin_fmaf(e, sr.s, dA[v]);
            dz[v] = dy[v] * __builtin_fmaf(mj, u, ah) * sz[v].s * __builtin_fmaf(z[v], sz[v].c, 1.f);
            qin[v] = aj * dh;
        }
        put(p.dx, p.dx_st, j, dx);
        put(p.dr, p.dr_st, j, dr);
        put(p.di, p.di_st, j, di);
        if (p.z) put(p.dz, p.dz_st, j, dz);
        if (!plain && g_bit(g.first, j)) {
            if (p.dh0) st_run<kGV, float>(p.dh0 + (int64_t)g_lane(g.s, j) * p.D + c, n, qin);
#pragma unroll
            for (int v = 0; v < kGV; ++v) qin[v] = 0.f;
        }
    }
    __syncthreads();  // P and H have been read
#pragma unroll
    for (int v = 0; v < kGV; ++v) s.P[w][v][l] = dA[v];
    __syncthreads();
    if (w < kGV) {  // wave v: the channels v of the lanes
        float sum = 0.f;
        for (int k = 0; k < kGW; ++k) sum += s.P[k][w][l];
        if (w < n) p.part[(int64_t)tile * p.D + c + w] = sum;
    }
}

// dA from the tiles' sums in order of their number: the same sum every time.  16 threads a channel,
// four loads in flight each; 16 channels a workgroup.
__global__ __launch_bounds__(256) void gated_join(const float* part, int parts, int D, float* dA) {
    __shared__ float red[16][17];
    const int x = threadIdx.x & 15, q = threadIdx.x >> 4, c = blockIdx.x * 16 + x;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < D) {
        const float* src = part + c;
        int i = q;
        for (; i + 48 < parts; i += 64) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += src[(int64_t)(i + 16 * j) * D];
        }
        for (; i < parts; i += 16) v[0] += src[(int64_t)i * D];
    }
    red[q][x] = (v[0] + v[1]) + (v[2] + v[3]);
    __syncthreads();
    if (q == 0 && c < D) {
        float a = 0.f;
        for (int j = 0; j < 16; ++j) a += red[j][x];
        dA[c] = a;
    }
}

struct GatedStepP {
    int nb, D;
    const void* x; int64_t x_sb;
    const void* r; int64_t r_sb;
    const void* i; int64_t i_sb;
    const void* z; int64_t z_sb;
    const float* A;
    float* state; int64_t nslots; const int32_t* slots;
    void* y; int64_t y_sb;
};

template <typename T>
__global__ __launch_bounds__(256) void gated_step(GatedStepP p) {
    const int b = blockIdx.y, c = blockIdx.x * 256 + threadIdx.x;
    if (c >= p.D) return;
    const int64_t slot = slot_of(p.slots, b, p.nslots);
    T* y = static_cast<T*>(p.y) + b * p.y_sb + c;
    if (slot < 0) {
        store_f32<T>(y, 0.f);
        return;
    }
    const Decay g = g_decay(p.A[c] * g_sigmoid(load_f32<T>(static_cast<const T*>(p.r) + b * p.r_sb + c)));
    float* st = p.state + slot * p.D + c;
    const float u = g_sigmoid(load_f32<T>(static_cast<const T*>(p.i) + b * p.i_sb + c)) * load_f32<T>(static_cast<const T*>(p.x) + b * p.x_sb + c);
    const float h = __builtin_fmaf(g.a, *st, __builtin_amdgcn_sqrtf(g.q) * u);
    *st = h;
    const float z = p.z ? load_f32<T>(static_cast<const T*>(p.z) + b * p.z_sb + c) : 0.f;
    store_f32<T>(y, p.z ? h * z * g_sigmoid(z) : h);
}

// The tiles of a call, and its workspace at ws (counted from NULL: its size): the ticket, the maps
// and ends (none for one tile of rows: nothing is waited for), and the backward's sums.
static size_t gated_plan(GatedP& p, bool back, bool bf16, void* ws) {
    const int tile = kGW * (back ? kGRows : bf16 ? kGFwdRows<bf16_t> : kGFwdRows<float>);
    p.ntile = (int)((p.rows + tile - 1) / tile);
    p.nct = ceil_div(p.D, kGC);
    const int64_t Dp = (int64_t)p.nct * kGC, words = p.ntile > 1 ? (p.ntile + p.ntile / kGGroup) * Dp : 0;
    char* at = static_cast<char*>(ws);
    size_t n = 0;
    auto take = [&](size_t bytes) {
        char* q = at + n;
        n += align_up(bytes, 256);
        return q;
    };
    if (words) {
        p.ticket = reinterpret_cast<uint32_t*>(take(4));
        p.map = reinterpret_cast<uint64_t*>(take(8 * words));
        p.ends = p.map + p.ntile * Dp;
    }
    if (back) p.part = reinterpret_cast<float*>(take((size_t)p.ntile * p.D * 4));
    return n;
}
static void gated_clear_launch(const GatedP& p, hipStream_t s) {
    if (p.ntile <= 1) return;
    const int64_t n = (int64_t)(p.ntile + p.ntile / kGGroup) * p.nct * kGC / 2;  // kGC words are whole 16 bytes
    hipLaunchKernelGGL(gated_clear, dim3((uint32_t)std::min<int64_t>((n + 255) / 256, 2048)), dim3(256), 0, s, p.ticket, reinterpret_cast<uint4*>(p.map), n);
}
static int gated_grid_ok(const GatedP& p) {
    MAMBA_CHECK_ARG((int64_t)p.ntile * p.nct * 64 * kGW < (1ll << 32), "rows x dim is too large for one call");
    return MAMBA_OK;
}

static int gated_make(const mamba_gated_scan_args* a, GatedP* out) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    MAMBA_CHECK_ARG(a->rows >= 0 && a->rows < kMaxRows, "rows must be in [0, 2^31 - 2^20)");
    MAMBA_CHECK_ARG(a->nseq >= 0, "nseq must be >= 0");
    MAMBA_CHECK_ARG(a->dim >= 1 && a->dim <= (1 << 20), "dim must be in [1, 2^20]");
    MAMBA_CHECK_ARG(a->io_dtype == MAMBA_F32 || a->io_dtype == MAMBA_BF16, "io_dtype must be f32 or bf16");
    MAMBA_CHECK_ARG(a->A != nullptr && a->cu_seqlens != nullptr, "A and cu_seqlens are required");
    MAMBA_CHECK_ARG(a->rows == 0 || (a->x && a->r && a->i), "x, r and i are required");
    GatedP& p = *out;
    p = GatedP{};
    p.q = Seqs{a->cu_seqlens, a->nseq, (int)a->rows};
    p.rows = a->rows; p.D = a->dim; p.fill = a->fill_outside != 0;
    p.x = a->x; p.x_st = a->x_st; p.r = a->r; p.r_st = a->r_st; p.i = a->i; p.i_st = a->i_st; p.z = a->z; p.z_st = a->z_st;
    p.A = a->A; p.carry = a->carry;
    return MAMBA_OK;
}

}  // namespace mamba

using namespace mamba;

// kernel<..., MODE>, by the number of channels
#define GATED_MODE(kernel, grid, block, stream, p, ...)                                                          \
    do {                                                                                                         \
        if ((p).D % 2 == 0) hipLaunchKernelGGL((kernel<__VA_ARGS__, 0>), grid, block, 0, (hipStream_t)stream, p); \
        else if ((p).D > 1) hipLaunchKernelGGL((kernel<__VA_ARGS__, 1>), grid, block, 0, (hipStream_t)stream, p); \
        else hipLaunchKernelGGL((kernel<__VA_ARGS__, 2>), grid, block, 0, (hipStream_t)stream, p);               \
    } while (0)

extern "C" size_t mamba_gated_scan_workspace_size(const mamba_gated_scan_args* a) {
    GatedP p;
    if (gated_make(a, &p) != MAMBA_OK) return 0;
    return gated_plan(p, false, a->io_dtype == MAMBA_BF16, nullptr);
}

extern "C" int mamba_gated_scan_fwd(const mamba_gated_scan_args* a, void* ws, size_t ws_bytes, mamba_stream_t stream) {
    GatedP p;
    int st = gated_make(a, &p);
    if (st != MAMBA_OK) return st;
    if (p.rows == 0) return MAMBA_OK;
    MAMBA_CHECK_ARG(a->y != nullptr, "y is required");
    MAMBA_CHECK_ARG(a->y_st >= p.D || p.rows == 1, "rows of y overlap");
    MAMBA_CHECK_ARG(a->state == nullptr || a->slots != nullptr || a->nslots >= a->nseq,
                    "without slots the state needs a row per sequence");
    const size_t e = a->io_dtype == MAMBA_BF16 ? 2 : 4;
    MAMBA_CHECK_ARG(!rows_clash(a->y, a->y_st, a->x, a->x_st, p.D, p.D, p.rows, e, true) &&
                        !rows_clash(a->y, a->y_st, a->r, a->r_st, p.D, p.D, p.rows, e, true) &&
                        !rows_clash(a->y, a->y_st, a->i, a->i_st, p.D, p.D, p.rows, e, true) &&
                        !rows_clash(a->y, a->y_st, a->z, a->z_st, p.D, p.D, p.rows, e, true),
                    "y overlaps an input (it may be x, r, i or z itself)");
    p.y = a->y; p.y_st = a->y_st; p.state = a->state; p.nslots = a->nslots; p.slots = a->slots;
    const size_t need = gated_plan(p, false, a->io_dtype == MAMBA_BF16, ws);
    if ((st = gated_grid_ok(p)) != MAMBA_OK) return st;
    MAMBA_CHECK_ARG(((uintptr_t)ws & 15u) == 0, "the workspace must be 16-byte aligned");
    if (need && (ws == nullptr || ws_bytes < need)) {
        set_error("mamba_gated_scan_fwd: workspace missing or too small");
        return MAMBA_ERR_WORKSPACE;
    }
    gated_clear_launch(p, (hipStream_t)stream);
    const dim3 grid(p.ntile * p.nct), block(64 * kGW);
    if (a->io_dtype == MAMBA_BF16) GATED_MODE(gated_fwd, grid, block, stream, p, bf16_t);
    else GATED_MODE(gated_fwd, grid, block, stream, p, float);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}

extern "C" size_t mamba_gated_scan_bwd_workspace_size(const mamba_gated_scan_bwd_args* a) {
    GatedP p;
    if (a == nullptr || gated_make(&a->fwd, &p) != MAMBA_OK) return 0;
    return gated_plan(p, true, a->fwd.io_dtype == MAMBA_BF16, nullptr);
}

extern "C" int mamba_gated_scan_bwd(const mamba_gated_scan_bwd_args* a, void* ws, size_t ws_bytes, mamba_stream_t stream) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    GatedP p;
    int st = gated_make(&a->fwd, &p);
    if (st != MAMBA_OK) return st;
    MAMBA_CHECK_ARG(a->fwd.state == nullptr && a->fwd.slots == nullptr,
                    "the gradient takes initial_state, a row per sequence, and no slots");
    MAMBA_CHECK_ARG(a->dA != nullptr, "dA is required");
    MAMBA_CHECK_ARG(p.rows == 0 || (p.carry && a->dy && a->dx && a->dr && a->di), "carry, dy, dx, dr and di are required");
    MAMBA_CHECK_ARG(p.rows == 0 || (p.z != nullptr) == (a->dz != nullptr), "dz goes with z");
    struct Rows { const void* p; int64_t st; };
    const Rows ins[] = {{p.x, p.x_st}, {p.r, p.r_st}, {p.i, p.i_st}, {p.z, p.z_st}, {a->dy, a->dy_st}};
    const Rows outs[] = {{a->dx, a->dx_st}, {a->dr, a->dr_st}, {a->di, a->di_st}, {a->dz, a->dz_st}};
    const size_t es = a->fwd.io_dtype == MAMBA_BF16 ? 2 : 4;
    for (const Rows& o : outs) {
        MAMBA_CHECK_ARG(p.rows <= 1 || o.p == nullptr || o.st >= p.D, "rows of a gradient overlap");
        for (const Rows& i : ins)
            MAMBA_CHECK_ARG(!rows_clash(o.p, o.st, i.p, i.st, p.D, p.D, p.rows, es, false), "a gradient overlaps an input");
        for (const Rows* q = outs; q != &o; ++q)
            MAMBA_CHECK_ARG(!rows_clash(o.p, o.st, q->p, q->st, p.D, p.D, p.rows, es, false), "two gradients overlap");
    }
    p.h0 = a->initial_state; p.dhT = a->d_final_state; p.dh0 = a->d_initial_state; p.dA = a->dA;
    p.dy = a->dy; p.dy_st = a->dy_st; p.dx = a->dx; p.dx_st = a->dx_st; p.dr = a->dr; p.dr_st = a->dr_st;
    p.di = a->di; p.di_st = a->di_st; p.dz = a->dz; p.dz_st = a->dz_st;
    const size_t need = gated_plan(p, true, a->fwd.io_dtype == MAMBA_BF16, ws);
    if ((st = gated_grid_ok(p)) != MAMBA_OK) return st;
    MAMBA_CHECK_ARG(((uintptr_t)ws & 15u) == 0, "the workspace must be 16-byte aligned");
    if (need && (ws == nullptr || ws_bytes < need)) {
        set_error("mamba_gated_scan_bwd: workspace missing or too small");
        return MAMBA_ERR_WORKSPACE;
    }
    gated_clear_launch(p, (hipStream_t)stream);
    if (p.ntile) {
        const dim3 grid(p.ntile * p.nct), block(64 * kGW);
        if (a->fwd.io_dtype == MAMBA_BF16) GATED_MODE(gated_bwd, grid, block, stream, p, bf16_t);
        else GATED_MODE(gated_bwd, grid, block, stream, p, float);
    }
    hipLaunchKernelGGL(gated_join, dim3(ceil_div(p.D, 16)), dim3(256), 0, (hipStream_t)stream, p.part, p.ntile, p.D, p.dA);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}

extern "C" int mamba_gated_step_slots(const mamba_gated_step_slots_args* a, mamba_stream_t stream) {
    MAMBA_CHECK_ARG(a != nullptr, "args is NULL");
    MAMBA_CHECK_ARG(a->batch >= 0 && a->batch <= 65535, "batch must be in [0, 65535]");
    MAMBA_CHECK_ARG(a->dim >= 1 && a->dim <= (1 << 20), "dim must be in [1, 2^20]");
    MAMBA_CHECK_ARG(a->io_dtype == MAMBA_F32 || a->io_dtype == MAMBA_BF16, "io_dtype must be f32 or bf16");
    if (a->batch == 0) return MAMBA_OK;
    MAMBA_CHECK_ARG(a->x && a->r && a->i && a->A && a->state && a->y, "x, r, i, A, state and y are required");
    MAMBA_CHECK_ARG(a->slots != nullptr || a->nslots >= a->batch, "without slots the state needs a row per token");
    MAMBA_CHECK_ARG(a->y_sb >= a->dim || a->batch == 1, "rows of y overlap");
    const size_t e = a->io_dtype == MAMBA_BF16 ? 2 : 4;
    MAMBA_CHECK_ARG(!rows_clash(a->y, a->y_sb, a->x, a->x_sb, a->dim, a->dim, a->batch, e, true) &&
                        !rows_clash(a->y, a->y_sb, a->r, a->r_sb, a->dim, a->dim, a->batch, e, true) &&
                        !rows_clash(a->y, a->y_sb, a->i, a->i_sb, a->dim, a->dim, a->batch, e, true) &&
                        !rows_clash(a->y, a->y_sb, a->z, a->z_sb, a->dim, a->dim, a->batch, e, true),
                    "y overlaps an input (it may be x, r, i or z itself)");
    GatedStepP p{};
    p.nb = a->batch; p.D = a->dim;
    p.x = a->x; p.x_sb = a->x_sb; p.r = a->r; p.r_sb = a->r_sb; p.i = a->i; p.i_sb = a->i_sb; p.z = a->z; p.z_sb = a->z_sb;
    p.A = a->A; p.state = a->state; p.nslots = a->nslots; p.slots = a->slots; p.y = a->y; p.y_sb = a->y_sb;
    const dim3 grid(ceil_div(p.D, 256), p.nb);
    if (a->io_dtype == MAMBA_BF16) hipLaunchKernelGGL(gated_step<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(gated_step<float>, grid, dim3(256), 0, (hipStream_t)stream, p);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}
