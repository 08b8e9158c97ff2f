// Rows of C elements as 16-byte vectors, for the kernels that take any C: WHOLE rows hold whole
// vectors (C a multiple of Vec::N, so that every vector of a 16-byte aligned array is aligned);
// otherwise the last vector of a row is partial and rows begin at any element.
#pragma once

#include <algorithm>

#include "common.hpp"

namespace clk {

template <typename TR>
struct Vec {
    static constexpr int N = 16 / sizeof(typename TR::elem);
};

// A row's partial last vector is loaded where the row still holds a whole one and moved down by the
// difference: a branch to single elements would wait for its loads before the next load is issued.

// The vector without its first s elements of 2 (4) bytes, zeros behind.
__device__ __forceinline__ u32x4 move_down2(u32x4 r, int s) {
    r = s & 4 ? u32x4{r[2], r[3], 0u, 0u} : r;
    r = s & 2 ? u32x4{r[1], r[2], r[3], 0u} : r;
    return s & 1 ? u32x4{r[0] >> 16 | r[1] << 16, r[1] >> 16 | r[2] << 16, r[2] >> 16 | r[3] << 16,
                         r[3] >> 16}
                 : r;
}
__device__ __forceinline__ u32x4 move_down4(u32x4 r, int s) {
    r = s & 2 ? u32x4{r[2], r[3], 0u, 0u} : r;
    return s & 1 ? u32x4{r[1], r[2], r[3], 0u} : r;
}

// Moves a vector that was loaded at `at` to `col`, up to N elements on: zeros past the row's end.
template <typename TR>
__device__ __forceinline__ u32x4 move_to(u32x4 raw, int at, int col) {
    return Vec<TR>::N == 8 ? move_down2(raw, col - at) : move_down4(raw, col - at);
}

// The N elements from `col` < C on, zero past the row's end. NT: non-temporal where a vector is
// aligned (rows that are read once).
template <typename TR, bool WHOLE, bool NT = false>
__device__ __forceinline__ u32x4 load_vec(const typename TR::elem* row, int col, int C) {
    constexpr int N = Vec<TR>::N;
    if (WHOLE && NT) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(row + col));
    if (WHOLE) return ld16(row + col);
    if (C < N) {  // the same for all rows
        typename TR::elem e[N];
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = col + i < C ? row[col + i] : TR::from_f(0.f);
        u32x4 raw;
        __builtin_memcpy(&raw, e, 16);
        return raw;
    }
    const int at = col < C - N ? col : C - N;
    const u32x4 raw = ld16_a2(row + at);
    return move_to<TR>(raw, at, col);
}

template <typename TR>
__device__ __forceinline__ void unpack_vec(u32x4 raw, float (&out)[Vec<TR>::N]) {
    typename TR::elem e[Vec<TR>::N];
    __builtin_memcpy(e, &raw, 16);
#pragma unroll
    for (int i = 0; i < Vec<TR>::N; ++i) out[i] = TR::to_f(e[i]);
}

template <typename TR>
__device__ __forceinline__ u32x4 pack_vec(const float (&v)[Vec<TR>::N]) {
    typename TR::elem e[Vec<TR>::N];
#pragma unroll
    for (int i = 0; i < Vec<TR>::N; ++i) e[i] = TR::from_f(v[i]);
    u32x4 raw;
    __builtin_memcpy(&raw, e, 16);
    return raw;
}

// Stores, non-temporal with NT where a vector is aligned.
template <typename TR, bool WHOLE, bool NT>
__device__ __forceinline__ void store_vec(typename TR::elem* row, int col, int C, u32x4 raw) {
    constexpr int N = Vec<TR>::N;
    if (WHOLE && NT) {
        __builtin_nontemporal_store(raw, reinterpret_cast<u32x4*>(row + col));
    } else if (WHOLE) {
        st16(row + col, raw);
    } else if (col + N <= C) {
        *reinterpret_cast<u32x4_a2*>(row + col) = raw;
    } else {
        typename TR::elem e[N];
        __builtin_memcpy(e, &raw, 16);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (col + i < C) row[col + i] = e[i];
    }
}

// N floats of a [C] vector from `col` on, at float alignment; `fill` past its end.
template <int N, bool WHOLE>
__device__ __forceinline__ void load_floats(const float* p, int col, int C, float fill,
                                            float (&out)[N]) {
#pragma unroll
    for (int q = 0; q < N; q += 4) {
        if (WHOLE || C >= 4) {
            const int at = WHOLE || col + q < C - 4 ? col + q : C - 4;
            u32x4 raw = __builtin_bit_cast(u32x4, ld4f(p + at));
            if (!WHOLE) raw = move_down4(raw, col + q - at < 4 ? col + q - at : 3);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                out[q + i] = WHOLE || col + q + i < C ? __uint_as_float(raw[i]) : fill;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) out[q + i] = col + q + i < C ? p[col + q + i] : fill;
        }
    }
}

template <int N>
__device__ __forceinline__ void store_floats(float* p, int col, int C, const float (&v)[N]) {
#pragma unroll
    for (int q = 0; q < N; q += 4) {
        if (col + q + 4 <= C) {
            *reinterpret_cast<f32x4_a4*>(p + col + q) = f32x4{v[q], v[q + 1], v[q + 2], v[q + 3]};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (col + q + i < C) p[col + q + i] = v[q + i];
        }
    }
}

// Do two arrays of a and b bytes overlap? Null pointers overlap nothing.
inline bool overlap(const void* p, size_t a, const void* q, size_t b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q);
    return x && y && (x < y ? y - x < a : x - y < b);
}

inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace clk
