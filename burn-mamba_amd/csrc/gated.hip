// Gated linear recurrence over packed sequences for gfx950, one state a channel:
// forward, backward, and single tokens on a cache addressed by slot.  f32 or bf16 rows
// (channels contiguous), f32 states, A and its gradient.
//
//   a_t = exp(A s(r_t)),  m_t = sqrt(1 - a_t^2),  u_t = s(i_t) x_t
//   h_t = a_t h_{t-1} + m_t u_t,  y_t = h_t silu(z_t) (or h_t)
// Backward, with g_t = dy_t silu(z_t) (dhT added at a sequence's last row):
//   dh_t = g_t + a_{t+1} dh_{t+1},  e_t = dh_t (a_t h_{t-1} - u_t a_t^2 / m_t)
//   dx = dh m s(i),  di = dh m u s(-i),  dr = e A s(r) s(-r),  dA = sum_t e s(r)
//   dz = dy h silu'(z),  dh0 = a dh at a sequence's first row
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
};

constexpr int kCarryRows = 64;  // rows between the states that the forward keeps for the backward

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

// a = exp(v) and m = sqrt(1 - a^2) for v <= 0, both to a few steps of their own size.  Above
// -1/4 from e = exp(v) - 1, the series to v^7 / 7! (its next term is 2^-29 of the sum there):
// a = 1 + e, 1 - a^2 = -e (2 + e) keep what a difference from 1 would lose as a nears 1.
struct Decay { float a, m; };
__device__ __forceinline__ Decay g_decay(float v) {
    float e = 1.f / 5040.f;
    e = __builtin_fmaf(e, v, 1.f / 720.f);
    e = __builtin_fmaf(e, v, 1.f / 120.f);
    e = __builtin_fmaf(e, v, 1.f / 24.f);
    e = __builtin_fmaf(e, v, 1.f / 6.f);
    e = __builtin_fmaf(e, v, 0.5f);
    e = __builtin_fmaf(e, v, 1.f) * v;
    const float far = __builtin_amdgcn_exp2f(v * 1.44269504088896341f);
    const bool near = v >= -0.25f;
    return {near ? 1.f + e : far, __builtin_amdgcn_sqrtf(near ? -e * (2.f + e) : __builtin_fmaf(-far, far, 1.f))};
}

// the row's sequence: s, and whether it is in one, its first, its last (uniform)
struct RowAt {
    int s;
    bool live, first, last;
};
__device__ __forceinline__ RowAt g_row(const Seqs& q, int t) {
    RowAt o;
    o.s = q.after(t);
    o.live = o.s < q.n && t >= q.begin(o.s);
    o.first = o.live && t == q.begin(o.s);
    o.last = o.live && t == q.end(o.s) - 1;
    return o;
}

template <typename T>
__global__ __launch_bounds__(64) void gated_fwd_walk(GatedP p) {
    const int c = blockIdx.x * 64 + threadIdx.x;
    const bool on = c < p.D;
    float h = 0.f;
    const float A = on ? p.A[c] : 0.f;
    for (int t = 0; t < (int)p.rows; ++t) {
        const RowAt w = g_row(p.q, t);
        if (p.carry && t % kCarryRows == 0 && on) p.carry[(int64_t)(t / kCarryRows) * p.D + c] = h;
        T* y = static_cast<T*>(p.y) + t * p.y_st + c;
        if (!w.live) {
            if (p.fill && on) store_f32<T>(y, 0.f);
            h = 0.f;
            continue;
        }
        const int64_t slot = p.state ? slot_of(p.slots, w.s, p.nslots) : -1;
        if (!on) continue;
        if (w.first) h = slot >= 0 ? p.state[slot * p.D + c] : 0.f;
        const Decay g = g_decay(A * g_sigmoid(load_f32<T>(static_cast<const T*>(p.r) + t * p.r_st + c)));
        const float u = g_sigmoid(load_f32<T>(static_cast<const T*>(p.i) + t * p.i_st + c)) * load_f32<T>(static_cast<const T*>(p.x) + t * p.x_st + c);
        h = __builtin_fmaf(g.a, h, g.m * u);
        const float z = p.z ? load_f32<T>(static_cast<const T*>(p.z) + t * p.z_st + c) : 0.f;
        store_f32<T>(y, p.z ? h * z * g_sigmoid(z) : h);
        if (w.last && slot >= 0) p.state[slot * p.D + c] = h;
    }
}

template <typename T>
__global__ __launch_bounds__(64) void gated_bwd_walk(GatedP p) {
    __shared__ float s_h[kCarryRows][64];  // the state before each row of a stretch
    const int c = blockIdx.x * 64 + threadIdx.x, l = threadIdx.x;
    const bool on = c < p.D;
    const float A = on ? p.A[c] : 0.f;
    float e_in = 0.f, dA = 0.f;
    auto at = [&](const void* q, int64_t st, int t) { return on ? load_f32<T>(static_cast<const T*>(q) + t * st + c) : 0.f; };
    auto put = [&](void* q, int64_t st, int t, float v) { if (on) store_f32<T>(static_cast<T*>(q) + t * st + c, v); };
    // no rows: no stretch (and no carry to read), and dA is 0
    for (int t0 = p.rows ? ((int)p.rows - 1) / kCarryRows * kCarryRows : -1; t0 >= 0; t0 -= kCarryRows) {
        const int t1 = min((int)p.rows, t0 + kCarryRows);
        float h = on ? p.carry[(int64_t)(t0 / kCarryRows) * p.D + c] : 0.f;
        for (int t = t0; t < t1; ++t) {
            const RowAt w = g_row(p.q, t);
            if (w.first) h = p.h0 && on ? p.h0[(int64_t)w.s * p.D + c] : 0.f;
            s_h[t - t0][l] = h;
            const Decay g = g_decay(A * g_sigmoid(at(p.r, p.r_st, t)));
            h = w.live ? __builtin_fmaf(g.a, h, g.m * (g_sigmoid(at(p.i, p.i_st, t)) * at(p.x, p.x_st, t))) : 0.f;
        }
        for (int t = t1 - 1; t >= t0; --t) {
            const RowAt w = g_row(p.q, t);
            if (!w.live) {
                put(p.dx, p.dx_st, t, 0.f);
                put(p.dr, p.dr_st, t, 0.f);
                put(p.di, p.di_st, t, 0.f);
                if (p.z) put(p.dz, p.dz_st, t, 0.f);
                e_in = 0.f;
                continue;
            }
            const Logistic r = g_logistic(at(p.r, p.r_st, t)), i = g_logistic(at(p.i, p.i_st, t));
            const Decay g = g_decay(A * r.s);
            const float dy = at(p.dy, p.dy_st, t), u = i.s * at(p.x, p.x_st, t), before = s_h[t - t0][l];
            float gy = dy;
            if (p.z) {
                const float z = at(p.z, p.z_st, t);
                const Logistic sz = g_logistic(z);
                gy = dy * z * sz.s;
                put(p.dz, p.dz_st, t, dy * __builtin_fmaf(g.a, before, g.m * u) * sz.s * __builtin_fmaf(z, sz.c, 1.f));
            }
            if (w.last && p.dhT && on) gy += p.dhT[(int64_t)w.s * p.D + c];
            const float dh = gy + e_in;
            const float pull = g.m > 0.f ? u * g.a * g.a * __builtin_amdgcn_rcpf(g.m) : 0.f;
            const float e = dh * (g.a * before - pull);
            put(p.dx, p.dx_st, t, dh * g.m * i.s);
            put(p.di, p.di_st, t, dh * g.m * u * i.c);
            put(p.dr, p.dr_st, t, e * A * r.s * r.c);
            dA = __builtin_fmaf(e, r.s, dA);
            e_in = g.a * dh;
            if (w.first) {
                if (p.dh0 && on) p.dh0[(int64_t)w.s * p.D + c] = e_in;
                e_in = 0.f;
            }
        }
    }
    if (on) p.dA[c] = dA;
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
    const float h = __builtin_fmaf(g.a, *st, g.m * u);
    *st = h;
    const float z = p.z ? load_f32<T>(static_cast<const T*>(p.z) + b * p.z_sb + c) : 0.f;
    store_f32<T>(y, p.z ? h * z * g_sigmoid(z) : h);
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

extern "C" size_t mamba_gated_scan_workspace_size(const mamba_gated_scan_args* a) {
    GatedP p;
    if (gated_make(a, &p) != MAMBA_OK) return 0;
    return 0;
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
    const dim3 grid(ceil_div(p.D, 64));
    if (a->io_dtype == MAMBA_BF16) hipLaunchKernelGGL(gated_fwd_walk<bf16_t>, grid, dim3(64), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(gated_fwd_walk<float>, grid, dim3(64), 0, (hipStream_t)stream, p);
    MAMBA_CHECK_LAUNCH();
    return MAMBA_OK;
}

extern "C" size_t mamba_gated_scan_bwd_workspace_size(const mamba_gated_scan_bwd_args* a) {
    GatedP p;
    if (a == nullptr || gated_make(&a->fwd, &p) != MAMBA_OK) return 0;
    return 0;
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
    const dim3 grid(ceil_div(p.D, 64));
    if (a->fwd.io_dtype == MAMBA_BF16) hipLaunchKernelGGL(gated_bwd_walk<bf16_t>, grid, dim3(64), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(gated_bwd_walk<float>, grid, dim3(64), 0, (hipStream_t)stream, p);
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
