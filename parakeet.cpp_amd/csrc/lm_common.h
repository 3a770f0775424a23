// lm_common.h -- what the serving kernels share: element types, wave and workgroup sums, the 4-bit cache's layout.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace pklm {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));

__device__ inline float bf16_f32(unsigned short h) { return __uint_as_float((unsigned)h << 16); }
__device__ inline float f16_f32(unsigned short h) { return (float)__builtin_bit_cast(_Float16, h); }
__device__ inline unsigned short f32_bf16(float x) { return __builtin_bit_cast(unsigned short, (__bf16)x); }
__device__ inline unsigned short f32_f16(float x) { return __builtin_bit_cast(unsigned short, (_Float16)x); }

// Element types: f32 and the two 16-bit ones.
struct F32 {
    using Raw = float;
    __device__ static float get(Raw v) { return v; }
    __device__ static Raw put(float v) { return v; }
};
struct F16 {
    using Raw = unsigned short;
    __device__ static float get(Raw v) { return f16_f32(v); }
    __device__ static Raw put(float v) { return f32_f16(v); }
};
struct BF16 {
    using Raw = unsigned short;
    __device__ static float get(Raw v) { return bf16_f32(v); }
    __device__ static Raw put(float v) { return f32_bf16(v); }
};

// 2^e of whole numbers -126 .. 127
__device__ inline float pow2i(int e) { return __int_as_float((e + 127) << 23); }

// Bytes of one (page, kv head) record and where its parts begin.
struct Record {
    int page, dim;
    __host__ __device__ int64_t bytes() const { return (int64_t)page * (dim + dim / 16); }
    __host__ __device__ int v_codes() const { return page * (dim / 2); }
    __host__ __device__ int k_scales() const { return page * dim; }
    __host__ __device__ int v_scales() const { return page * dim + page * (dim / 32); }
};

template <class T>
__device__ inline T wave_scan(T v) {   // inclusive sum over the wave
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const T o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

}  // namespace pklm
