// Runs of consecutive elements of an f32 or bf16 row as f32 values, and the
// sequences of a packed batch: shared by the norm, dropout, convolution and
// packed scan kernels.
#pragma once

#include "common.h"

namespace mamba {

// V consecutive elements at p (V sizeof(T) = 4, 8, 16 or 32 bytes; any element
// alignment: the memory system takes unaligned vectors), the first n of them
// read (n >= V: one vector), the others 0.
template <int V, typename T>
__device__ __forceinline__ void ld_run(const T* p, int n, float (&v)[V]) {
    if (n >= V) {
        T r[V];
        __builtin_memcpy(r, p, V * sizeof(T));
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = load_f32<T>(&r[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = i < n ? load_f32<T>(p + i) : 0.f;
    }
}

template <int V, typename T>
__device__ __forceinline__ void st_run(T* p, int n, const float (&v)[V]) {
    if (n >= V) {
        T r[V];
        if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const uint32_t w = pack_bf16x2(v[i], v[i + 1]);
                r[i] = (T)w;
                r[i + 1] = (T)(w >> 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) store_f32<T>(&r[i], v[i]);
        }
        __builtin_memcpy(p, r, V * sizeof(T));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) store_f32<T>(p + i, v[i]);
    }
}

// V consecutive elements of a row as they lie in memory, so that a
// load may stay in flight until they are used.
template <typename T, int V>
struct Elems {
    static constexpr int W = (V * (int)sizeof(T) + 3) / 4;
    uint32_t w[W];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (V * sizeof(T) == 2) w[0] = *p;
        else __builtin_memcpy(w, p, V * sizeof(T));
    }
    __device__ __forceinline__ void load_part(const T* p, int n) {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = 0u;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) {
                if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(p[i]);
                else w[i / 2] |= (uint32_t)p[i] << (16 * (i & 1));
            }
    }
    __device__ __forceinline__ void get(float (&o)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if constexpr (sizeof(T) == 4) o[i] = __uint_as_float(w[i]);
            else o[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        }
    }
};

// ------------------------------------------------- packed sequences ---
// Sequence s is rows cu[s] .. cu[s + 1] - 1 of a tensor of `rows` rows; rows
// outside every sequence belong to none.  The offsets live on the device, where
// the host cannot check them: each is clamped, so that a wrong one gives a wrong
// result and no access out of range.
struct Seqs {
    const int32_t* cu;
    int n, rows;
    // in scalar registers: s and t are uniform over a wave
    __device__ __forceinline__ int at(int s) const { return min(max(__builtin_amdgcn_readfirstlane(cu[s]), 0), rows); }
    __device__ __forceinline__ int begin(int s) const { return at(s); }
    __device__ __forceinline__ int end(int s) const { return max(at(s), at(s + 1)); }
    // s + 1 is the next sequence to look at behind an empty one s at row t: many empty
    // ones are passed over at once (and s never goes back, whatever the offsets are)
    __device__ __forceinline__ int skip(int s, int t) const { return max(s, after(t) - 1); }
    // the first sequence that ends behind row t, n if none does
    __device__ __forceinline__ int after(int t) const {
        int lo = 0, hi = n;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (__builtin_amdgcn_readfirstlane(cu[mid + 1]) > t) hi = mid;
            else lo = mid + 1;
        }
        return lo;
    }
};
// What an output may share with an input: nothing, or (same = true) exactly its own
// rows, where each element is read by the thread that writes it.  Rows of a wider
// tensor beside one another (one stride, disjoint columns) share nothing.
inline bool rows_clash(const void* a, int64_t a_st, const void* b, int64_t b_st, int64_t a_cols, int64_t b_cols,
                       int64_t rows, size_t esize, bool same) {
    if (a == nullptr || b == nullptr || rows <= 0) return false;
    const char *pa = static_cast<const char*>(a), *pb = static_cast<const char*>(b);
    const int64_t e = (int64_t)esize;
    if (pa + ((rows - 1) * a_st + a_cols) * e <= pb || pb + ((rows - 1) * b_st + b_cols) * e <= pa) return false;
    if (rows == 1) return !(same && pa == pb);
    if (a_st != b_st || a_st <= 0 || (pa - pb) % e != 0) return true;
    int64_t off = (pb - pa) / e % a_st;  // b's first column behind a's, in a row of a_st
    if (off < 0) off += a_st;
    if (off == 0) return !(same && pa == pb);
    return off < a_cols || a_st - off < b_cols;
}

// rows of a packed tensor: a chunk's last row and one more chunk still fit an int
constexpr int64_t kMaxRows = (1ll << 31) - (1ll << 20);
// elements between rows: 16 rows' offsets fit 32 bits of bytes
constexpr int64_t kMaxStride = 1ll << 25;

// Row of a cache that sequence s keeps its state in, -1: none (a slot out of range).
__device__ __forceinline__ int64_t slot_of(const int32_t* slots, int s, int64_t nslots) {
    const int64_t r = slots ? (int64_t)slots[s] : (int64_t)s;
    return r >= 0 && r < nslots ? r : -1;
}

}  // namespace mamba
