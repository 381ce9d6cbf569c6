// seq_rows.h -- pieces of the row kernels (embedding, norm, log-probabilities).
#ifndef CUSR_SEQ_ROWS_H
#define CUSR_SEQ_ROWS_H

#include "seq_common.h"

namespace seq {

// 8 values of a row side by side, as loaded: one piece of 16 bytes in a 16-bit type,
// two in fp32. Loading and unpacking are apart, so that several are on their way.
template <typename T> struct Eight {
    uint4v a;
    __device__ void load(const T *p) { a = *(const uint4v *)p; }
    __device__ void zero() { a = uint4v{0, 0, 0, 0}; }
    __device__ void get(float *f) const {
        typedef T vec __attribute__((ext_vector_type(8)));
        const vec v = __builtin_bit_cast(vec, a);
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = (float)v[j];
    }
    static __device__ void put(T *p, const float *f) {
        typedef T vec __attribute__((ext_vector_type(8)));
        vec v;
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = (T)f[j];
        *(vec *)p = v;
    }
};
template <> struct Eight<float> {
    float4v a, b;
    __device__ void load(const float *p) { a = *(const float4v *)p; b = *(const float4v *)(p + 4); }
    __device__ void zero() { a = b = float4v{0, 0, 0, 0}; }
    __device__ void get(float *f) const {
#pragma unroll
        for (int j = 0; j < 4; j++) { f[j] = a[j]; f[j + 4] = b[j]; }
    }
    static __device__ void put(float *p, const float *f) {
        *(float4v *)p = float4v{f[0], f[1], f[2], f[3]};
        *(float4v *)(p + 4) = float4v{f[4], f[5], f[6], f[7]};
    }
};

// one value, where the type is known to the call only
__device__ inline float get1(const void *p, int dtype, int64_t at) {
    if (dtype == SEQ_FP32) return ((const float *)p)[at];
    if (dtype == SEQ_BF16) return (float)((const __bf16 *)p)[at];
    return (float)((const _Float16 *)p)[at];
}
__device__ inline void put1(void *p, int dtype, int64_t at, float f) {
    if (dtype == SEQ_FP32) ((float *)p)[at] = f;
    else if (dtype == SEQ_BF16) ((__bf16 *)p)[at] = (__bf16)f;
    else ((_Float16 *)p)[at] = (_Float16)f;
}
__device__ inline int64_t get_id(const void *p, int ids_64, int64_t at) {
    return ids_64 ? ((const int64_t *)p)[at] : ((const int32_t *)p)[at];
}

// Up to 8 values of a row side by side. ANY: at any place, `n` of them (a row's last may be
// fewer), zeros beyond; the memory takes wide loads and stores off their boundaries (the
// norm's gradient of 20,000 rows of 2,047 in bf16: 67 us, value by value 153, of 2,048 44).
// Else all 8 on a boundary of 16 bytes.
template <typename T, bool ANY> struct Cells;
template <typename T> struct Cells<T, false> {
    Eight<T> v;
    __device__ void load(const T *p, int) { v.load(p); }
    __device__ void zero() { v.zero(); }
    __device__ void get(float *f) const { v.get(f); }
    static __device__ void put(T *p, const float *f, int) { Eight<T>::put(p, f); }
};
template <typename T> struct Cells<T, true> {
    typedef T vec __attribute__((ext_vector_type(8)));
    vec v;
    __device__ void load(const T *p, int n) {
        if (n == 8) {
            __builtin_memcpy(&v, p, sizeof(v));
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = j < n ? p[j] : (T)0.0f;
        }
    }
    __device__ void zero() {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = (T)0.0f;
    }
    __device__ void get(float *f) const {
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = (float)v[j];
    }
    static __device__ void put(T *p, const float *f, int n) {
        if (n == 8) {
            vec v;
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = (T)f[j];
            __builtin_memcpy(p, &v, sizeof(v));
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j < n) p[j] = (T)f[j];
        }
    }
};
template <bool ANY, typename T>
__device__ inline void get_typed(const void *p, int64_t at, float *f, int n) {
    Cells<T, ANY> v;
    v.load((const T *)p + at, n);
    v.get(f);
}
// the same where the type is known to the call only: the branch is the wave's
template <bool ANY>
__device__ inline void get_cells(const void *p, int dtype, int64_t at, float *f, int n) {
    if (dtype == SEQ_FP32) get_typed<ANY, float>(p, at, f, n);
    else if (dtype == SEQ_BF16) get_typed<ANY, __bf16>(p, at, f, n);
    else get_typed<ANY, _Float16>(p, at, f, n);
}
template <bool ANY>
__device__ inline void put_cells(void *p, int dtype, int64_t at, const float *f, int n) {
    if (dtype == SEQ_FP32) Cells<float, ANY>::put((float *)p + at, f, n);
    else if (dtype == SEQ_BF16) Cells<__bf16, ANY>::put((__bf16 *)p + at, f, n);
    else Cells<_Float16, ANY>::put((_Float16 *)p + at, f, n);
}
// values of part `at` of a row
template <bool ANY> __device__ inline int cells_of(int64_t width, int at) {
    return ANY && width - at * 8 < 8 ? (int)(width - at * 8) : 8;
}

inline bool float_type(int t) { return t >= SEQ_FP32 && t <= SEQ_FP16; }
inline int type_bytes(int t) { return t == SEQ_FP32 ? 4 : (t == SEQ_INT8 ? 1 : 2); }
// whether rows hold whole pieces of 8 values, each on a boundary of 16 bytes (8 of int8)
inline bool in_eights(const void *p, int64_t row) {
    return !p || (!((uintptr_t)p & 15) && row % 8 == 0);
}

// Reductions over lanes by exchanges that stay in vector registers (a wave's sum by way of
// the LDS crossbar waits for it six times): lanes 1 and 2 apart, mirrored eights and
// sixteens, whose halves are alike by then, and swapped sixteens and halves.
struct Add { static __device__ float of(float a, float b) { return a + b; } };
// keeps a NaN, as fmaxf would not
struct Most { static __device__ float of(float a, float b) { return a > b || a != a ? a : b; } };
// drops a NaN
struct Larger {
    static __device__ float of(float a, float b) { return fmaxf(a, b); }
    static __device__ uint32_t of(uint32_t a, uint32_t b) { return a > b ? a : b; }
};
template <int CTRL, typename T> __device__ inline T moved(T x) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL,
                                                             0xf, 0xf, false));
}
// over G lanes side by side, a power of two up to 64; every lane gets the result
template <typename Op, int G, typename T> __device__ inline T over_lanes(T x) {
    if constexpr (G >= 2) x = Op::of(x, moved<0xb1>(x));
    if constexpr (G >= 4) x = Op::of(x, moved<0x4e>(x));
    if constexpr (G >= 8) x = Op::of(x, moved<0x141>(x));
    if constexpr (G >= 16) x = Op::of(x, moved<0x140>(x));
    if constexpr (G >= 32) {
        const uint32_t u = __builtin_bit_cast(uint32_t, x);
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        x = Op::of(__builtin_bit_cast(T, (uint32_t)r[0]), __builtin_bit_cast(T, (uint32_t)r[1]));
    }
    if constexpr (G >= 64) {
        const uint32_t u = __builtin_bit_cast(uint32_t, x);
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        x = Op::of(__builtin_bit_cast(T, (uint32_t)r[0]), __builtin_bit_cast(T, (uint32_t)r[1]));
    }
    return x;
}
// over G threads, up to the block's 1,024: beyond a wave through LDS, `red` with a float
// for each wave. Every thread gets the result, formed in one order.
template <typename Op, int G> __device__ inline float over_group(float x, float *red) {
    x = over_lanes<Op, (G < 64 ? G : 64)>(x);
    if constexpr (G > 64) {
        __syncthreads();                     // red may still be read from a call before
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
        __syncthreads();
        x = red[0];
#pragma unroll
        for (int i = 1; i < G / 64; i++) x = Op::of(x, red[i]);
    }
    return x;
}

}  // namespace seq
#endif
