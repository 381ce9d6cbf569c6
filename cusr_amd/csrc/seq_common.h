// seq_common.h -- shared by the sequence operators (include/cusr_seq.h).
#ifndef CUSR_SEQ_COMMON_H
#define CUSR_SEQ_COMMON_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cusr_seq.h"

namespace seq {

typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

template <int N> struct Const { static constexpr int value = N; };

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ inline float neg_inf() { return -__builtin_inff(); }

// 2^x: one v_exp_f32 (results below 2^-126 flush to 0)
__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// larger of two, as the middle one of them and infinity: unlike fmaxf it needs no
// instruction before it to quiet a NaN of a matrix product, and unlike assembly it
// waits for the product
__device__ inline float max2(float a, float b) {
    return __builtin_amdgcn_fmed3f(a, b, __builtin_inff());
}

// larger of the two halves' values, in both lanes of (l, l + 32)
__device__ inline float max_halves(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float add_halves(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The 16-bit types: packing of two floats (round to nearest even) and the
// 32x32x16 matrix product. Lane l of A holds row l % 32, of B column l % 32,
// both at k = 8 (l / 32) + 0..7; D's register r is row
// 8 (r / 4) + 4 (l / 32) + r % 4 of column l % 32.
struct Bf16 {
    typedef __bf16 elem;
    static __device__ uint32_t pack(float a, float b) {
        bf16x2 v = {(__bf16)a, (__bf16)b};
        return __builtin_bit_cast(uint32_t, v);
    }
    static __device__ float16v mfma(uint4v a, uint4v b, float16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ float lo(uint32_t x) { return __uint_as_float(x << 16); }
    static __device__ float hi(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
};
struct Fp16 {
    typedef _Float16 elem;
    static __device__ uint32_t pack(float a, float b) {
        f16x2 v = {(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(uint32_t, v);
    }
    static __device__ float16v mfma(uint4v a, uint4v b, float16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ float lo(uint32_t x) {
        return (float)__builtin_bit_cast(_Float16, (uint16_t)(x & 0xffffu));
    }
    static __device__ float hi(uint32_t x) {
        return (float)__builtin_bit_cast(_Float16, (uint16_t)(x >> 16));
    }
};

// Wave-private LDS: writes of this wave's other lanes are visible to what
// follows (LDS operations of one wave complete in order; the compiler must
// not move them across this point).
__device__ inline void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// 4 x 16 block of 16-bit values in LDS, transposed on the way to registers:
// lane i of each group of 16 gives the address of row i / 4, columns
// 4 (i % 4) .. + 3, and gets column i, rows 0..3.
__device__ inline uint2v read_transposed(__attribute__((address_space(3))) const uint16_t *p) {
    typedef __attribute__((address_space(3))) short4v *lds4;
    return __builtin_bit_cast(uint2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p));
}
__device__ inline uint2v read_transposed(const uint16_t *p) {
    return read_transposed((__attribute__((address_space(3))) const uint16_t *)p);
}

// Blocks of a launch. An axis has fewer than 2^32 threads (HIP starts what is left of
// the number modulo 2^32, without an error), so more blocks continue along z, in equal
// parts: the last numbers may be past the end, and a kernel leaves those alone.
inline dim3 grid_of(int64_t blocks, int threads, unsigned y = 1) {
    const int64_t most = 0xffffffffll / threads;
    const int64_t z = (blocks + most - 1) / most;
    return dim3((unsigned)((blocks + z - 1) / z), y, (unsigned)z);
}
__device__ inline int block_number() {
    return (int)(blockIdx.x + (blockIdx.z ? blockIdx.z * gridDim.x : 0));
}

inline int launch_status() {
    return hipGetLastError() == hipSuccess ? CO_OK : CO_ERR_CUDA;
}

}  // namespace seq
#endif
