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
// cut into tiles (128 in the forward, 64 in the backward) without regard to the sequences, a
// workgroup takes one tile of 64 channels, keeps it in registers, and finds the state that enters
// it while the tile is there.
// A stretch of rows maps the state that enters it, h -> P h + H; P is the product of its
// decays and H what it leaves from zero.  A lane holds R rows of one channel (two channels would take
// twice the registers and leave the backward one workgroup a CU, which took half as long again).
// The maps of the eight waves are joined in LDS to the tile's, which is published to the other
// workgroups before the tile's own state is waited for.  That state is joined from the published
// maps of the tiles before it, back to the one in which the tile's first sequence begins, or to
// the last group of 16 or 64 tiles, whose final state its last tile publishes.  The joins follow a
// fixed order: the same inputs give the same bits.  The backward walks the other way with q in the
// state's place, and finds h again from the states that the forward kept.
//
// A map is published as one 64-bit word (P, H) and read with relaxed atomics of the whole card:
// the word is its own flag, all ones until it is written (P of a NaN is made the usual one, so
// that no map has that value).  A workgroup takes its tile by ticket, so the tiles that it waits
// for belong to workgroups that run already, and those publish before they wait: every wait ends.
//
// Times below: calls back to back in a captured graph on a warm card, with their clear and join.
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
    int ntile, nct, group;              // group: log2 of the tiles of a group
    uint32_t* ticket;                   // [nct], kGTicket words apart
    uint64_t* map;                      // [ntile][nct kGC] published maps
    uint64_t* ends;                     // [ntile >> group][nct kGC] states at the ends of groups
    float* part;                        // [ntile][D] partial sums of dA
};

constexpr int kCarryRows = 64;  // rows between the states that the forward keeps for the backward
constexpr int kGW = 8, kGC = 64;  // waves of a workgroup; channels of a tile: one a lane
// Log2 of the tiles of a group.  The ends of groups are found one behind the other: with many of them
// in flight that chain is the longer wait, with few the maps of a group are (64 / 16 tiles: 262144 x
// 256 of bf16 forward 185 / 202 us, backward 381 / 410; 65536 x 512 77 / 77 and 160 / 159, 8192 x 5120
// 104 / 99 and 208 / 196).
constexpr int kGGroup = 4, kGGroupLong = 6;
constexpr int kGLong = 2048;                     // tiles of rows from which on groups are long
constexpr uint64_t kGNone = ~0ull;               // nothing published yet
constexpr int kGTicket = 32;                     // words between the tickets of two column tiles
// Rows of a lane.  What a tile costs beside its rows is the same for 8 of them: with 8 the forward
// of 8192 x 5120 takes 1.2 times as long as with 16.  The backward holds nine values of a row where
// the forward holds two, and a tile of it enters with kept states.
constexpr int kGRows = kCarryRows / kGW, kGFwdRows = 2 * kGRows;

// v is formed here: the compiler moves a value to the block of its only use, and what it is
// formed from stays in registers until then.
__device__ __forceinline__ void g_keep(float& v) { asm volatile("" : "+v"(v)); }

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

// a = exp(v) and q = 1 - a^2 for v <= 0, both to a few steps of their own size (below -1/8 a's error
// grows as |v|, by the rounding of the exponent).  From -1/8 up by
// e = exp(v) - 1, the series to v^5 / 5! (its next term is 2^-24 of the sum there): a = 1 + e,
// 1 - a^2 = -e (2 + e) keep what a difference from 1 would lose as a nears 1.  FAR: with the
// exponential for what lies below, which a wave takes only where it has such a value.  Forward and
// backward where no wave has one / every wave has one, through one channel in 64: 8192 x 5120 of bf16
// 99 / 102 and 196 / 198 us, 2048 x 2560 22.6 / 23.3 and 38.1 / 38.3, 65536 x 512 77 / 80 and 160 / 162;
// in f32, bound by memory, no different.
struct Decay { float a, q; };
__device__ __forceinline__ bool g_near(float v) { return v >= -0.125f; }  // not of a NaN
template <bool FAR>
__device__ __forceinline__ Decay g_decay(float v) {
    float e = 1.f / 120.f;
    e = __builtin_fmaf(e, v, 1.f / 24.f);
    e = __builtin_fmaf(e, v, 1.f / 6.f);
    e = __builtin_fmaf(e, v, 0.5f);
    e = __builtin_fmaf(e, v, 1.f) * v;
    Decay d = {1.f + e, -e * (2.f + e)};
    if constexpr (FAR) {
        float far = __builtin_amdgcn_exp2f(v * 1.44269504088896341f);
        g_keep(far);  // for every lane: a branch of its own would cost more
        const float q = __builtin_fmaf(-far, far, 1.f);
        d.a = g_near(v) ? d.a : far;
        d.q = g_near(v) ? d.q : q;
    }
    return d;
}
// The decays of R rows: a holds A s(r).
template <int R>
__device__ __forceinline__ void g_decays(float (&a)[R], float (&q)[R]) {
    bool far = false;
#pragma unroll
    for (int j = 0; j < R; ++j) far |= !g_near(a[j]);
    if (__ballot(far)) {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const Decay d = g_decay<true>(a[j]);
            a[j] = d.a;
            q[j] = d.q;
        }
    } else {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const Decay d = g_decay<false>(a[j]);
            a[j] = d.a;
            q[j] = d.q;
        }
    }
}

// What the R rows from t0 are (R < 64, t0 uniform over the wave): bit j of a mask for row
// t0 + j, whether it is in a sequence, its first, its last; lane j holds the row's sequence and
// that one's first row and end.  The offsets are clamped: a wrong one gives a wrong result and
// no access out of range.  They are searched with scalar loads, which do not queue behind the rows
// in flight (lanes that searched cost 8192 x 5120 a tenth).
struct GRows {
    uint64_t live, first, last;
    int s, b, e;
};
__device__ __forceinline__ int g_offset(const Seqs& q, int s) {  // cu[s], s uniform
    return min(max(((const __attribute__((address_space(4))) int32_t*)q.cu)[s], 0), q.rows);
}
// The first sequence from lo on that ends behind row t.
__device__ __forceinline__ int g_search(const Seqs& q, int lo, int t) {
    int hi = q.n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (g_offset(q, mid + 1) > t) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}
__device__ __forceinline__ GRows g_rows(const Seqs& q, int t0, int R) {
    const int j = threadIdx.x & 63;
    GRows o{0, 0, 0, 0, 0, 0};
    int t = t0, s = g_search(q, 0, t0);
    if (s >= q.n) return o;
    int b = g_offset(q, s), e = g_offset(q, s + 1);
    while (true) {  // sequence s, b .. e, ends behind t, which grows
        const int j0 = max(b, t) - t0, j1 = min(e - t0, R);
        if (j0 < j1) {
            o.live |= (1ull << j1) - (1ull << j0);
            if (b >= t0) o.first |= 1ull << j0;
            if (e - t0 <= R) o.last |= 1ull << (j1 - 1);
            const bool here = j >= j0 && j < j1;
            o.s = here ? s : o.s;
            o.b = here ? b : o.b;
            o.e = here ? e : o.e;
        }
        t = e;
        if (t >= t0 + R || ++s >= q.n) break;
        b = e;
        e = g_offset(q, s + 1);
        if (e <= t) {  // an empty one, or many
            s = g_search(q, s + 1, t);
            if (s >= q.n) break;
            b = g_offset(q, s);
            e = g_offset(q, s + 1);
        }
    }
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

__global__ __launch_bounds__(256) void gated_clear(uint32_t* ticket, int nct, uint4* words, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < nct) ticket[i * kGTicket] = 0;  // nct <= n
    for (int64_t k = i; k < n; k += (int64_t)gridDim.x * 256) words[k] = make_uint4(~0u, ~0u, ~0u, ~0u);
}

struct GMap { float P = 1.f, H = 0.f; };
struct GShared {
    float P[kGW][64], H[kGW][64];    // the waves' maps
    float P2[kGW][64], H2[kGW][64];  // joined runs of tiles; the backward's maps of h
    float in[64];                    // the group's entry
    int cut[kGW];                    // whether a wave's rows cut the state that enters them off
    int tile, far;
};

// The tile of this workgroup (in the order in which the tiles wait for one another) and its channels.
// A ticket for each column tile: one counter for all is asked by 512 workgroups at once when a
// kernel starts (4000 x 2560 of bf16 took 1.14 times as long).  The columns turn against the
// workgroups' numbers from a row of tiles to the next, as the numbers go around the chip's eight
// dies: a die that kept every eighth column would go through a few channels of its L2 (8192 x 5120
// took 1.09 times as long).
__device__ __forceinline__ void g_tile(const GatedP& p, GShared& s, int& o, int& ct) {
    if (p.ntile > 1) {
        ct = (blockIdx.x + blockIdx.x / p.nct) % p.nct;
        if (threadIdx.x == 0) s.tile = (int)atomicAdd(p.ticket + ct * kGTicket, 1u);
        __syncthreads();
        o = __builtin_amdgcn_readfirstlane(s.tile);
    } else {
        o = 0;
        ct = blockIdx.x;
    }
}
__device__ __forceinline__ int64_t g_at(const GatedP& p, int o, int ct, int l) { return ((int64_t)o * p.nct + ct) * kGC + l; }

// The waves' maps, joined onto h: the waves from .. to - 1 in the order of time, or against it.
template <bool BACK>
__device__ __forceinline__ void g_fold(const float (&P)[kGW][64], const float (&H)[kGW][64], const int (&cut)[kGW], int n, int l, float& h) {
    for (int i = 0; i < n; ++i) {
        const int k = BACK ? kGW - 1 - i : i;
        h = cut[k] ? H[k][l] : __builtin_fmaf(P[k][l], h, H[k][l]);
    }
}
// The tile's map, published by one wave; cut: whether its rows cut off what enters.
template <bool BACK>
__device__ __forceinline__ GMap g_publish_map(const GatedP& p, const GShared& s, int o, int ct, int l, bool& cut) {
    GMap m;
    g_fold<BACK>(s.P, s.H, s.cut, kGW, l, m.H);
    cut = false;
#pragma unroll
    for (int k = 0; k < kGW; ++k) {
        m.P *= s.P[k][l];
        cut |= s.cut[k] != 0;
    }
    g_publish(p.map + g_at(p, o, ct, l), g_word(m.P, m.H));
    return m;
}
__device__ __forceinline__ void g_publish_end(const GatedP& p, int o, int ct, int l, const GMap& m, bool cut, float h) {
    if (((o + 1) & ((1 << p.group) - 1)) == 0 && o + 1 < p.ntile)
        g_publish(p.ends + g_at(p, o >> p.group, ct, l), g_word(0.f, cut ? m.H : __builtin_fmaf(m.P, h, m.H)));
}

// The state that enters tile o: joined from the maps of tiles far .. o - 1, tile `far` being cut, or
// from the end of the group before o's.  Called by the whole workgroup (o > far >= 0).
__device__ __forceinline__ float g_enter(const GatedP& p, GShared& s, int o, int ct, int far) {
    const int w = wave_id(), l = threadIdx.x & 63;
    const int base = o >> p.group << p.group, from = max(far, base);
    const bool group = far < base;
    const int per = (o - from + kGW - 1) / kGW, k0 = min(o, from + w * per), k1 = min(o, k0 + per);
    GMap m;
    constexpr int most = (1 << kGGroupLong) / kGW;  // maps of a wave
    uint64_t word[most], end = 0;
#pragma unroll
    for (int i = 0; i < most; ++i) word[i] = k0 + i < k1 ? g_peek(p.map + g_at(p, k0 + i, ct, l)) : 0;
    const uint64_t* ends = p.ends + g_at(p, (base >> p.group) - 1, ct, l);
    if (group && w == 0) end = g_peek(ends);
#pragma unroll
    for (int i = 0; i < most; ++i) {
        if (k0 + i >= k1) break;
        const uint64_t x = g_wait(p.map + g_at(p, k0 + i, ct, l), word[i]);
        const float P = __uint_as_float((uint32_t)x), H = __uint_as_float((uint32_t)(x >> 32));
        m.H = i ? __builtin_fmaf(P, m.H, H) : H;
        m.P = i ? P * m.P : P;
    }
    if (group && w == 0) s.in[l] = __uint_as_float((uint32_t)(g_wait(ends, end) >> 32));
    s.P2[w][l] = m.P;
    s.H2[w][l] = m.H;
    __syncthreads();
    float h = group ? __builtin_fmaf(s.P2[0][l], s.in[l], s.H2[0][l]) : s.H2[0][l];  // a cut tile's P is no factor
    for (int k = 1; k < kGW && from + k * per < o; ++k) h = __builtin_fmaf(s.P2[k][l], h, s.H2[k][l]);
    return h;
}

// A wave's rows of one tensor from row t0 on, a channel a lane, through a buffer resource: a scalar
// offset a row (16 rows' offsets and a column fit 31 bits) and one of the lane, which lies behind the resource's
// end for a lane without a channel.  Such a lane reads 0 and writes nothing, without a branch.
template <typename T>
struct GRow {
    __amdgpu_buffer_rsrc_t r;
    uint32_t st;
    __device__ __forceinline__ GRow(const void* p, int64_t t0, int64_t stride)
        : r(buf_rsrc(static_cast<const T*>(p) + t0 * stride, 0x7fffffffu)), st((uint32_t)stride * (uint32_t)sizeof(T)) {}
    static __device__ __forceinline__ uint32_t column(int c, int D) { return c < D ? (uint32_t)c * (uint32_t)sizeof(T) : 0x80000000u; }
    __device__ __forceinline__ uint32_t load(int j, uint32_t col) const {
        if constexpr (sizeof(T) == 2) return (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, col, j * st, 0);
        else return __builtin_amdgcn_raw_buffer_load_b32(r, col, j * st, 0);
    }
    __device__ __forceinline__ void store(int j, uint32_t col, float v) const {
        if constexpr (sizeof(T) == 2) __builtin_amdgcn_raw_buffer_store_b16((short)pack_bf16x2(v, v), r, col, j * st, 0);
        else __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), r, col, j * st, 0);
    }
};
template <typename T>
__device__ __forceinline__ float g_value(uint32_t w) { return __uint_as_float(sizeof(T) == 2 ? w << 16 : w); }
// rows past the last one are read as the last
template <typename T, int R>
__device__ __forceinline__ void g_fetch(uint32_t (&e)[R], const GatedP& p, const void* q, int64_t st, int t0, uint32_t col) {
    const int t = min(t0, (int)p.rows - 1), k = (int)p.rows - 1 - t;
    const GRow<T> row(q, t, st);
#pragma unroll
    for (int j = 0; j < R; ++j) e[j] = row.load(min(j, k), col);
}

// 8192 x 5120: bf16 with z 99 us (420 MB, 4.2 TB/s), f32 without 125 (671 MB, 5.4: what a copy
// reaches and a little from the last-level cache).  bf16: half the time is issue of vector instructions (44 a row, 7 of them at a quarter
// of the rate), the rest a tile's latencies (ticket, rows, the states that enter), which two
// workgroups a CU hide in part; three (80 registers) spill and take 1.2 times as long.
template <typename T, bool Z>
__global__ __launch_bounds__(64 * kGW, 4) void gated_fwd(GatedP p) {
    constexpr int R = kGFwdRows;
    __shared__ GShared s;
    int o, ct;
    g_tile(p, s, o, ct);
    const int w = wave_id(), l = threadIdx.x & 63;
    const int t0 = (o * kGW + w) * R, c = ct * kGC + l;
    const int rows = min(R, max(0, (int)p.rows - t0));  // of this wave
    const uint32_t col = GRow<T>::column(c, p.D);
    uint32_t ez[Z ? R : 1];
    float a[R], b[R];
    GRows g;
    int j0;    // the first row here that begins a sequence, and
    float h0;  // what that one starts from, on its way with the rows
    {
        uint32_t ex[R], er[R], ei[R];
        const float A = c < p.D ? p.A[c] : 0.f;  // first: loads come back in order
        g_fetch<T, R>(er, p, p.r, p.r_st, t0, col);
        g_fetch<T, R>(ei, p, p.i, p.i_st, t0, col);
        g_fetch<T, R>(ex, p, p.x, p.x_st, t0, col);
        g = g_rows(p.q, t0, R);
        j0 = g.first ? __builtin_ctzll(g.first) : 0;
        const int64_t slot = p.state && g.first ? slot_of(p.slots, g_lane(g.s, j0), p.nslots) : -1;
        h0 = buf_ld4(buf_rsrc(p.state + max(slot, (int64_t)0) * p.D, slot >= 0 ? p.D * 4u : 0u), c * 4u);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            a[j] = A * g_sigmoid(g_value<T>(er[j]));
            g_keep(a[j]);
        }
        g_decays<R>(a, b);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            b[j] = __builtin_amdgcn_sqrtf(b[j]) * (g_sigmoid(g_value<T>(ei[j])) * g_value<T>(ex[j]));
            g_keep(b[j]);
        }
    }
    constexpr uint64_t full = (1ull << R) - 1;
    const bool plain = g.live == full && (g.first | g.last) == 0;
    GMap m;
    if (plain) {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            m.H = __builtin_fmaf(a[j], m.H, b[j]);
            m.P *= a[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (g_bit(g.first, j)) {  // from the sequence's state on; b holds the new one
                if (j != j0) {
                    const int64_t slot = p.state ? slot_of(p.slots, g_lane(g.s, j), p.nslots) : -1;
                    h0 = slot >= 0 && c < p.D ? p.state[slot * p.D + c] : 0.f;
                }
                m.H = b[j] = __builtin_fmaf(a[j], h0, b[j]);
            } else if (g_bit(g.live, j)) {
                m.H = __builtin_fmaf(a[j], m.H, b[j]);
                m.P *= a[j];
            } else {
                m.H = 0.f;
            }
        }
    }
    s.P[w][l] = m.P;
    s.H[w][l] = m.H;
    if (l == 0) s.cut[w] = g.live != full || g.first != 0;
    if (threadIdx.x == 0) s.far = (g.live & ~g.first & 1) ? g.b / (kGW * R) : -1;
    if constexpr (Z) g_fetch<T, R>(ez, p, p.z, p.z_st, t0, col);
    __syncthreads();
    float h = 0.f;
    GMap whole;
    bool cut = false;
    if (w == kGW - 1 && p.ntile > 1) whole = g_publish_map<false>(p, s, o, ct, l, cut);
    const int far = __builtin_amdgcn_readfirstlane(s.far);
    if (far >= 0) h = g_enter(p, s, o, ct, far);
    if (w == kGW - 1) g_publish_end(p, o, ct, l, whole, cut, h);
    g_fold<false>(s.P, s.H, s.cut, w, l, h);
    if (p.carry && t0 % kCarryRows == 0 && rows > 0 && c < p.D) p.carry[(int64_t)(t0 / kCarryRows) * p.D + c] = h;
    const GRow<T> y(p.y, t0, p.y_st);
    auto put = [&](int j) __attribute__((always_inline)) {
        float v = h;
        if constexpr (Z) {
            const float z = g_value<T>(ez[j]);
            v = h * (z * g_sigmoid(z));  // silu first: h z may pass f32 where silu is 0
        }
        y.store(j, col, v);
    };
    if (plain) {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            h = __builtin_fmaf(a[j], h, b[j]);
            put(j);
        }
    } else {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (!g_bit(g.live, j)) {
                h = 0.f;
                if (p.fill && j < rows) y.store(j, col, 0.f);
                continue;
            }
            h = g_bit(g.first, j) ? b[j] : __builtin_fmaf(a[j], h, b[j]);
            put(j);
            if (g_bit(g.last, j) && p.state) {
                const int64_t slot = slot_of(p.slots, g_lane(g.s, j), p.nslots);
                if (slot >= 0 && c < p.D) p.state[slot * p.D + c] = h;
            }
        }
    }
}

// What a row's gradients need is formed once, where its values are read: with u = s(i) x,
//   gr = dy silu(z), zk = dy silu'(z), pull = u a^2 / m, kr = A s(r) s(-r), ui = u s(-i)
// so that dz = h zk, dx = dh m s(i), di = dh m ui, dr = e kr, e = dh (a h_{t-1} - pull).
// 8192 x 5120: bf16 with z 196 us (755 MB, 3.9 TB/s), f32 without 229 (1174 MB, 5.1).
// Bound as the forward is: some 90 vector instructions a row.
template <typename T, bool Z>
__global__ __launch_bounds__(64 * kGW, 4) void gated_bwd(GatedP p) {
    constexpr int R = kGRows;
    __shared__ GShared s;
    int o, ct;
    g_tile(p, s, o, ct);
    const int tile = p.ntile - 1 - o;  // from the last one on
    const int w = wave_id(), l = threadIdx.x & 63;
    const int row0 = tile * kCarryRows, t0 = row0 + w * R, c = ct * kGC + l;
    const int rows = min(R, max(0, (int)p.rows - t0));
    const uint32_t col = GRow<T>::column(c, p.D);
    // sm = m s(i), um = m ui
    float a[R], b[R], pull[R], sr[R], kr[R], sm[R], um[R], gr[R], zk[Z ? R : 1];
    float h = 0.f;
    GRows g;
    {
        uint32_t ex[R], er[R], ei[R], ez[R], ey[R];
        const float A = c < p.D ? p.A[c] : 0.f;
        g_fetch<T, R>(er, p, p.r, p.r_st, t0, col);
        g_fetch<T, R>(ei, p, p.i, p.i_st, t0, col);
        g_fetch<T, R>(ex, p, p.x, p.x_st, t0, col);
        g_fetch<T, R>(ey, p, p.dy, p.dy_st, t0, col);
        if constexpr (Z) g_fetch<T, R>(ez, p, p.z, p.z_st, t0, col);
        g = g_rows(p.q, t0, R);
        if (c < p.D) h = p.carry[(int64_t)tile * p.D + c];
        float q[R];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const Logistic r = g_logistic(g_value<T>(er[j]));
            sr[j] = r.s;
            a[j] = A * r.s;
            kr[j] = a[j] * r.c;
            g_keep(kr[j]);
        }
        g_decays<R>(a, q);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            // 0 where a is 1 (of a q below the normal numbers the hardware's root is 0 and its reciprocal
            // infinity), a NaN of a NaN
            const float im = q[j] >= 0x1p-126f ? __builtin_amdgcn_rsqf(q[j]) : q[j] * 0.f;
            const float m = q[j] * im;
            const Logistic i = g_logistic(g_value<T>(ei[j]));
            const float u = i.s * g_value<T>(ex[j]);
            sm[j] = m * i.s;
            um[j] = m * (u * i.c);
            b[j] = m * u;
            pull[j] = u * a[j] * (a[j] * im);
            g_keep(sm[j]);
            g_keep(um[j]);
            g_keep(pull[j]);
            const float dy = g_value<T>(ey[j]);
            gr[j] = dy;
            if constexpr (Z) {
                const float z = g_value<T>(ez[j]);
                const Logistic k = g_logistic(z);
                gr[j] = dy * k.s * z;
                zk[j] = dy * k.s * __builtin_fmaf(z, k.c, 1.f);
                g_keep(gr[j]);
                g_keep(zk[j]);
            }
        }
    }
    constexpr uint64_t full = (1ull << R) - 1;
    const bool plain = g.live == full && (g.first | g.last) == 0;
    auto start = [&](int j) __attribute__((always_inline)) {  // what the sequence of row j starts from
        return p.h0 && c < p.D ? p.h0[(int64_t)g_lane(g.s, j) * p.D + c] : 0.f;
    };
    // the waves' maps of h and of q
    GMap f, q;
    if (plain) {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            f.H = __builtin_fmaf(a[j], f.H, b[j]);
            f.P *= a[j];
            q.H = a[R - 1 - j] * (gr[R - 1 - j] + q.H);
        }
    } else {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (!g_bit(g.live, j)) {
                f.H = 0.f;
                continue;
            }
            if (g_bit(g.first, j)) f.H = start(j);
            f.H = __builtin_fmaf(a[j], f.H, b[j]);
            f.P *= a[j];
            if (g_bit(g.last, j) && p.dhT && c < p.D) gr[j] += p.dhT[(int64_t)g_lane(g.s, j) * p.D + c];
        }
#pragma unroll
        for (int j = R - 1; j >= 0; --j) q.H = g_bit(g.live & ~g.first, j) ? a[j] * (gr[j] + q.H) : 0.f;
    }
    s.P[w][l] = f.P;  // one product for both
    s.H[w][l] = q.H;
    s.H2[w][l] = f.H;
    if (l == 0) s.cut[w] = g.live != full || g.first != 0;
    if (threadIdx.x == 0) s.far = -1;
    __syncthreads();
    // the tile's last row: its sequence's last tile, where that is another
    const int lastrow = min((int)p.rows, row0 + kCarryRows) - 1 - t0;  // counted from this wave's first
    if (lastrow >= 0 && lastrow < R && g_bit(g.live & ~g.last, lastrow) && l == 0)
        s.far = p.ntile - 1 - (g_lane(g.e, lastrow) - 1) / kCarryRows;
    GMap whole;
    bool cut = false;
    if (w == 0 && p.ntile > 1) whole = g_publish_map<true>(p, s, o, ct, l, cut);
    g_fold<false>(s.P, s.H2, s.cut, w, l, h);  // the state that enters this wave's rows
    const GRow<T> dz(p.dz, t0, p.dz_st);
    // b: a h_{t-1} - pull
    if (plain) {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const float ah = a[j] * h;
            h = ah + b[j];
            b[j] = ah - pull[j];
            if constexpr (Z) dz.store(j, col, h * zk[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const bool live = g_bit(g.live, j);
            if (g_bit(g.first, j)) h = start(j);
            const float ah = a[j] * h;
            h = live ? ah + b[j] : 0.f;
            b[j] = ah - pull[j];
            if constexpr (Z) {
                if (j < rows) dz.store(j, col, live ? h * zk[j] : 0.f);
            }
        }
    }
    __syncthreads();  // the waves' maps of h have been read, and far is known
    float qin = 0.f;
    const int far = __builtin_amdgcn_readfirstlane(s.far);
    if (far >= 0) qin = g_enter(p, s, o, ct, far);
    if (w == 0) g_publish_end(p, o, ct, l, whole, cut, qin);
    g_fold<true>(s.P, s.H, s.cut, kGW - 1 - w, l, qin);
    float dA = 0.f;
    const GRow<T> dx(p.dx, t0, p.dx_st), dr(p.dr, t0, p.dr_st), di(p.di, t0, p.di_st);
    auto put = [&](int j) __attribute__((always_inline)) {
        const float dh = gr[j] + qin, e = dh * b[j];
        dx.store(j, col, dh * sm[j]);
        di.store(j, col, dh * um[j]);
        dr.store(j, col, e * kr[j]);
        dA = __builtin_fmaf(e, sr[j], dA);
        qin = a[j] * dh;
    };
    if (plain) {
#pragma unroll
        for (int j = R - 1; j >= 0; --j) put(j);
    } else {
#pragma unroll
        for (int j = R - 1; j >= 0; --j) {
            if (g_bit(g.live, j)) {
                put(j);
                if (g_bit(g.first, j)) {
                    if (p.dh0 && c < p.D) p.dh0[(int64_t)g_lane(g.s, j) * p.D + c] = qin;
                    qin = 0.f;
                }
            } else {
                qin = 0.f;
                if (j < rows) {
                    dx.store(j, col, 0.f);
                    di.store(j, col, 0.f);
                    dr.store(j, col, 0.f);
                }
            }
        }
    }
    __syncthreads();  // P has been read
    s.P[w][l] = dA;
    __syncthreads();
    if (w == 0 && c < p.D) {
        float sum = 0.f;
        for (int k = 0; k < kGW; ++k) sum += s.P[k][l];
        p.part[(int64_t)tile * p.D + c] = sum;
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

// A token a row, a channel a lane: 256 tokens of 5120 bf16 channels 6.0 us for 23.6 MB, a single one
// 2.4.  Bound by the latency of its loads, which do not wait for the slot.  Two and four channels a lane
// took 1.15 and 0.95 times as long for 256 tokens, 1.08 and 1.25 for one, where latency counts most.
template <typename T>
__global__ __launch_bounds__(256) void gated_step(GatedStepP p) {
    const int b = blockIdx.y, c = blockIdx.x * 256 + threadIdx.x;
    if (c >= p.D) return;
    const float r = load_f32<T>(static_cast<const T*>(p.r) + b * p.r_sb + c);
    const float i = load_f32<T>(static_cast<const T*>(p.i) + b * p.i_sb + c);
    const float x = load_f32<T>(static_cast<const T*>(p.x) + b * p.x_sb + c);
    const float z = p.z ? load_f32<T>(static_cast<const T*>(p.z) + b * p.z_sb + c) : 0.f;
    const float A = p.A[c];
    const int64_t slot = slot_of(p.slots, b, p.nslots);
    float y = 0.f;
    if (slot >= 0) {
        float* st = p.state + slot * p.D + c;
        const float h0 = *st;
        const Decay g = g_decay<true>(A * g_sigmoid(r));
        y = __builtin_fmaf(g.a, h0, __builtin_amdgcn_sqrtf(g.q) * (g_sigmoid(i) * x));
        *st = y;
        if (p.z) y = y * (z * g_sigmoid(z));
    }
    store_f32<T>(static_cast<T*>(p.y) + b * p.y_sb + c, y);
}

// The tiles of a call, and its workspace at ws (counted from NULL: its size): the ticket, the maps
// and ends (none for one tile of rows: nothing is waited for), and the backward's sums.
static size_t gated_plan(GatedP& p, bool back, void* ws) {
    const int tile = kGW * (back ? kGRows : kGFwdRows);
    p.ntile = (int)((p.rows + tile - 1) / tile);
    p.nct = ceil_div(p.D, kGC);
    p.group = p.ntile >= kGLong ? kGGroupLong : kGGroup;
    const int64_t Dp = (int64_t)p.nct * kGC, words = p.ntile > 1 ? (p.ntile + (p.ntile >> p.group)) * Dp : 0;
    char* at = static_cast<char*>(ws);
    size_t n = 0;
    auto take = [&](size_t bytes) {
        char* q = at + n;
        n += align_up(bytes, 256);
        return q;
    };
    if (words) {
        p.ticket = reinterpret_cast<uint32_t*>(take((size_t)p.nct * kGTicket * 4));
        p.map = reinterpret_cast<uint64_t*>(take(8 * words));
        p.ends = p.map + p.ntile * Dp;
    }
    if (back) p.part = reinterpret_cast<float*>(take((size_t)p.ntile * p.D * 4));
    return n;
}
static void gated_clear_launch(const GatedP& p, hipStream_t s) {
    if (p.ntile <= 1) return;
    const int64_t n = (int64_t)(p.ntile + (p.ntile >> p.group)) * p.nct * kGC / 2;  // kGC words are whole 16 bytes
    hipLaunchKernelGGL(gated_clear, dim3((uint32_t)std::min<int64_t>((n + 255) / 256, 2048)), dim3(256), 0, s, p.ticket, p.nct, reinterpret_cast<uint4*>(p.map), n);
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
    for (const int64_t st : {a->x_st, a->r_st, a->i_st, a->z ? a->z_st : 0})
        MAMBA_CHECK_ARG(a->rows <= 1 || (st >= 0 && st < kMaxStride), "row strides must be in [0, 2^25)");
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

#define GATED_LAUNCH(kernel, ...) \
    hipLaunchKernelGGL((kernel<__VA_ARGS__>), dim3(p.ntile * p.nct), dim3(64 * kGW), 0, (hipStream_t)stream, p)
// kernel<T, Z>, by the type and the gate
#define GATED_TILES(kernel, bf16)                             \
    do {                                                      \
        if (bf16 && p.z) GATED_LAUNCH(kernel, bf16_t, true);  \
        else if (bf16) GATED_LAUNCH(kernel, bf16_t, false);   \
        else if (p.z) GATED_LAUNCH(kernel, float, true);      \
        else GATED_LAUNCH(kernel, float, false);              \
    } while (0)

extern "C" size_t mamba_gated_scan_workspace_size(const mamba_gated_scan_args* a) {
    GatedP p;
    if (gated_make(a, &p) != MAMBA_OK) return 0;
    return gated_plan(p, false, nullptr);
}

extern "C" int mamba_gated_scan_fwd(const mamba_gated_scan_args* a, void* ws, size_t ws_bytes, mamba_stream_t stream) {
    GatedP p;
    int st = gated_make(a, &p);
    if (st != MAMBA_OK) return st;
    if (p.rows == 0) return MAMBA_OK;
    MAMBA_CHECK_ARG(a->y != nullptr, "y is required");
    MAMBA_CHECK_ARG((a->y_st >= p.D && a->y_st < kMaxStride) || p.rows == 1, "rows of y overlap (or lie 2^25 elements apart)");
    MAMBA_CHECK_ARG(a->state == nullptr || a->slots != nullptr || a->nslots >= a->nseq,
                    "without slots the state needs a row per sequence");
    const size_t e = a->io_dtype == MAMBA_BF16 ? 2 : 4;
    MAMBA_CHECK_ARG(!rows_clash(a->y, a->y_st, a->x, a->x_st, p.D, p.D, p.rows, e, true) &&
                        !rows_clash(a->y, a->y_st, a->r, a->r_st, p.D, p.D, p.rows, e, true) &&
                        !rows_clash(a->y, a->y_st, a->i, a->i_st, p.D, p.D, p.rows, e, true) &&
                        !rows_clash(a->y, a->y_st, a->z, a->z_st, p.D, p.D, p.rows, e, true),
                    "y overlaps an input (it may be x, r, i or z itself)");
    p.y = a->y; p.y_st = a->y_st; p.state = a->state; p.nslots = a->nslots; p.slots = a->slots;
    const size_t need = gated_plan(p, false, ws);
    if ((st = gated_grid_ok(p)) != MAMBA_OK) return st;
    MAMBA_CHECK_ARG(((uintptr_t)ws & 15u) == 0, "the workspace must be 16-byte aligned");
    if (need && (ws == nullptr || ws_bytes < need)) {
        set_error("mamba_gated_scan_fwd: workspace missing or too small");
        return MAMBA_ERR_WORKSPACE;
    }
    gated_clear_launch(p, (hipStream_t)stream);
    GATED_TILES(gated_fwd, a->io_dtype == MAMBA_BF16);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}

extern "C" size_t mamba_gated_scan_bwd_workspace_size(const mamba_gated_scan_bwd_args* a) {
    GatedP p;
    if (a == nullptr || gated_make(&a->fwd, &p) != MAMBA_OK) return 0;
    return gated_plan(p, true, nullptr);
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
    MAMBA_CHECK_ARG(p.rows <= 1 || (a->dy_st >= 0 && a->dy_st < kMaxStride), "row strides must be in [0, 2^25)");
    struct Rows { const void* p; int64_t st; };
    const Rows ins[] = {{p.x, p.x_st}, {p.r, p.r_st}, {p.i, p.i_st}, {p.z, p.z_st}, {a->dy, a->dy_st}};
    const Rows outs[] = {{a->dx, a->dx_st}, {a->dr, a->dr_st}, {a->di, a->di_st}, {a->dz, a->dz_st}};
    const size_t es = a->fwd.io_dtype == MAMBA_BF16 ? 2 : 4;
    for (const Rows& o : outs) {
        MAMBA_CHECK_ARG(p.rows <= 1 || o.p == nullptr || (o.st >= p.D && o.st < kMaxStride), "rows of a gradient overlap (or lie 2^25 elements apart)");
        for (const Rows& i : ins)
            MAMBA_CHECK_ARG(!rows_clash(o.p, o.st, i.p, i.st, p.D, p.D, p.rows, es, false), "a gradient overlaps an input");
        for (const Rows* q = outs; q != &o; ++q)
            MAMBA_CHECK_ARG(!rows_clash(o.p, o.st, q->p, q->st, p.D, p.D, p.rows, es, false), "two gradients overlap");
    }
    p.h0 = a->initial_state; p.dhT = a->d_final_state; p.dh0 = a->d_initial_state; p.dA = a->dA;
    p.dy = a->dy; p.dy_st = a->dy_st; p.dx = a->dx; p.dx_st = a->dx_st; p.dr = a->dr; p.dr_st = a->dr_st;
    p.di = a->di; p.di_st = a->di_st; p.dz = a->dz; p.dz_st = a->dz_st;
    const size_t need = gated_plan(p, true, ws);
    if ((st = gated_grid_ok(p)) != MAMBA_OK) return st;
    MAMBA_CHECK_ARG(((uintptr_t)ws & 15u) == 0, "the workspace must be 16-byte aligned");
    if (need && (ws == nullptr || ws_bytes < need)) {
        set_error("mamba_gated_scan_bwd: workspace missing or too small");
        return MAMBA_ERR_WORKSPACE;
    }
    gated_clear_launch(p, (hipStream_t)stream);
    if (p.ntile) GATED_TILES(gated_bwd, a->fwd.io_dtype == MAMBA_BF16);
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
