// seq_hidden.h -- values that are not finite in places that a row does not see.
//
// In the matrix products a masked weight is 0, and 0 * inf and 0 * NaN are NaN: a key or
// value of a tile reaches every row of the tile, a query every key. With finite inputs no
// sum is ever infinite or NaN, so each kernel looks at its sums once, when they are done (a
// multiply-add for two), and where one is not finite and the cause lies in a hidden place,
// the row's (key's) sums are formed again from their definition, over what it sees alone.
// That takes a wave about 0.4 ms for such a row of a thousand keys, and happens only near
// such values: ten sequences of 1 to 8,191, 32 heads of 128 over 8, take 59 ms with one NaN
// among the values and 1.2 with nothing else. The look costs short sequences 1 %
// (8,192 of 3 to 63 with gradient, 8 heads of 64: 696 and 702 us), long ones nothing that
// shows.
//
// What does so is called, not inlined: the kernels' registers stay as they are. A called
// function gets the kernel's arguments by a pointer to them, the same for the wave.
#ifndef CUSR_SEQ_HIDDEN_H
#define CUSR_SEQ_HIDDEN_H

#include "seq_attn.h"

namespace seq {

// The kernel's first argument in memory. In a kernel alone: a called function has no
// pointer of its own to the kernel's arguments.
template <typename A> using Arguments = const __attribute__((address_space(4))) A *;
template <typename A> __device__ __attribute__((always_inline)) inline Arguments<A> arguments() {
    return (Arguments<A>)__builtin_amdgcn_kernarg_segment_ptr();
}
// Of a called function's arguments, those that are the wave's.
__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
template <typename P> __device__ inline P *uniform(P *p) {
    const uint64_t x = (uint64_t)p;
    const uint32_t lo = uniform((int)(uint32_t)x), hi = uniform((int)(uint32_t)(x >> 32));
    return (P *)((uint64_t)hi << 32 | lo);
}
__device__ inline Place uniform(const Place &p) {
    return {uniform(p.q0), uniform(p.k0), uniform(p.lq), uniform(p.lk)};
}

__device__ inline bool finite(float x) { return fabsf(x) < __builtin_inff(); }

// Lanes' truth values as a bit for each of the wave's 32 rows, in both of its lanes.
__device__ inline uint32_t row_bits(bool x) {
    const uint64_t b = __ballot(x);
    return (uint32_t)b | (uint32_t)(b >> 32);
}

// Adds up what shows whether a lane's sums are finite: a product of two of which one is
// not finite is not finite either, nor a sum with it. Products that overflow show too; a
// look at the hidden places then finds no cause.
template <int DP> __device__ inline void watch(float &t, const float16v *sums) {
#pragma unroll
    for (int dt = 0; dt < DP / 32; dt++)
#pragma unroll
        for (int r = 0; r < 16; r += 2) t = __builtin_fmaf(sums[dt][r], sums[dt][r + 1], t);
}
// Which of the wave's 32 rows (keys) may have a sum that is not finite.
template <int DP> __device__ inline uint32_t not_finite(const float16v *sums) {
    float t = 0.0f;
    watch<DP>(t, sums);
    return row_bits(!finite(t));
}

template <typename T> __device__ inline float value(const uint16_t *x) { return T::lo(*x); }
template <typename T> __device__ inline float dot(const uint16_t *x, const uint16_t *y, int d) {
    float s = 0.0f;
    const uint4v z = {0, 0, 0, 0};
#pragma unroll 1
    for (int c0 = 0; c0 < d; c0 += 32) {     // four pieces of 8 on their way at a time
        uint4v a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bool in = c0 + 8 * i < d;
            a[i] = in ? *(const uint4v *)(x + c0 + 8 * i) : z;
            b[i] = in ? *(const uint4v *)(y + c0 + 8 * i) : z;
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                s += T::lo(a[i][j]) * T::lo(b[i][j]) + T::hi(a[i][j]) * T::hi(b[i][j]);
    }
    return s;
}
// rounded to the type, as the operands of the products are
template <typename T> __device__ inline float rounded(float x) { return T::lo(T::pack(x, 0.0f)); }

// f(which, column) for this lane's columns of a row
template <typename F> __device__ inline void each_column(int d, F f) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int e = 0; e < 2; e++)
        if (lane + 64 * e < d) f(e, lane + 64 * e);
}

// Whether some column has a value that is not finite in a hidden row, j0 <= j < j1, and a
// finite one in the row `seen` (-1: none): else a sum that is not finite is right so. Row
// j is at row(j).
template <typename T, typename R>
__device__ inline bool hidden_cause(R row, int d, int j0, int j1, int seen) {
    bool cause = false;
    each_column(d, [&](int, int col) {
        if (seen >= 0 && !finite(value<T>(row(seen) + col))) return;
#pragma unroll 8
        for (int j = j0; j < j1; j++) cause |= !finite(value<T>(row(j) + col));
    });
    return __any(cause);
}

// sum[e] += sum of weight(j) row(j)[column e] over j0 <= j < j1; weights 64 at a time,
// one to a lane.
template <typename T, typename R, typename W>
__device__ inline void add_seen(R row, int d, int j0, int j1, W weight, float (&sum)[2]) {
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int j = j0; j < j1; j += 64) {
        const float w = j + lane < j1 ? weight(j + lane) : 0.0f;
        const int n = min(64, j1 - j);
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += 8) {  // eight rows on their way at a time
            each_column(d, [&](int e, int col) {
                uint16_t x[8];
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = row(j + min(i0 + i, n - 1))[col];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint32_t wi = __builtin_amdgcn_readlane(__float_as_uint(w), min(i0 + i, 63));
                    if (i0 + i < n) sum[e] += __uint_as_float(wi) * T::lo(x[i]);
                }
            });
        }
    }
}

// Keys of a tile lie at most so far beyond what a row of it sees.
constexpr int kReach = 96;

}  // namespace seq
#endif
