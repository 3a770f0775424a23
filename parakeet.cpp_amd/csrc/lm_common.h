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

// Element types: f32 and the two 16-bit ones.  held: a value of the cache, or a mean of such, as the type is to have it.
struct F32 {
    using Raw = float;
    __device__ static float get(Raw v) { return v; }
    __device__ static Raw put(float v) { return v; }
    __device__ static float held(float v) { return v; }
};
struct F16 {
    using Raw = unsigned short;
    __device__ static float get(Raw v) { return f16_f32(v); }
    __device__ static Raw put(float v) { return f32_f16(v); }
    // The cache holds f16 rows over 57,344 as 65,536, the step past f16's largest value: that, and means of it to their
    // rounding, go back to 65,504, so that finite rows stay finite.  Beyond it there are infinities as in any conversion.
    __device__ static float held(float v) { return fabsf(v) <= 0x1.002p16f ? fminf(fmaxf(v, -65504.0f), 65504.0f) : v; }
};
struct BF16 {
    using Raw = unsigned short;
    __device__ static float get(Raw v) { return bf16_f32(v); }
    __device__ static Raw put(float v) { return f32_bf16(v); }
    __device__ static float held(float v) { return v; }
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

// Whole-wave scans and sums in the vector unit: lanes 1, 2, 4 and 8 before within rows of 16, then the last lanes of
// the rows before (a shuffle through LDS takes several times as long, and there are six in a row).
template <int Ctrl, int RowMask>
__device__ inline unsigned from_lane(unsigned v, unsigned none) {
    return (unsigned)__builtin_amdgcn_update_dpp((int)none, (int)v, Ctrl, RowMask, 0xF, false);
}
template <int Ctrl, int RowMask>
__device__ inline unsigned long long from_lane(unsigned long long v, unsigned long long none) {
    return (unsigned long long)from_lane<Ctrl, RowMask>((unsigned)(v >> 32), (unsigned)(none >> 32)) << 32 |
           from_lane<Ctrl, RowMask>((unsigned)v, (unsigned)none);
}
template <int Ctrl, int RowMask>
__device__ inline int from_lane(int v, int none) { return (int)from_lane<Ctrl, RowMask>((unsigned)v, (unsigned)none); }
template <int Ctrl, int RowMask>
__device__ inline float from_lane(float v, float none) {
    return __uint_as_float(from_lane<Ctrl, RowMask>(__float_as_uint(v), __float_as_uint(none)));
}
template <class V, class F>
__device__ inline V wave_scan(V v, V none, F f) {      // inclusive; lane 63 has all
    v = f(v, from_lane<0x111, 0xF>(v, none));
    v = f(v, from_lane<0x112, 0xF>(v, none));
    v = f(v, from_lane<0x114, 0xF>(v, none));
    v = f(v, from_lane<0x118, 0xF>(v, none));
    v = f(v, from_lane<0x142, 0xA>(v, none));
    v = f(v, from_lane<0x143, 0xC>(v, none));
    return v;
}
template <class V>
__device__ inline V wave_scan(V v) {
    return wave_scan(v, V(0), [](V a, V b) { return a + b; });
}
__device__ inline unsigned lane_value(unsigned v, int lane) { return (unsigned)__builtin_amdgcn_readlane((int)v, lane); }
__device__ inline int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ inline float lane_value(float v, int lane) { return __uint_as_float(lane_value(__float_as_uint(v), lane)); }
__device__ inline unsigned long long lane_value(unsigned long long v, int lane) {
    return (unsigned long long)lane_value((unsigned)(v >> 32), lane) << 32 | lane_value((unsigned)v, lane);
}
template <class V>
__device__ inline V wave_sum(V v) { return lane_value(wave_scan(v), 63); }
__device__ inline float wave_max(float v) {
    return lane_value(wave_scan(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); }), 63);
}

// Values that workgroups on other XCDs read within the launch: written through to, and read from, where all XCDs meet.
// base is the same in the whole wave, at counts 32-bit words from it, below 2^29.
__device__ inline void store_shared4(unsigned *base, unsigned at, u4 v) {
    const auto r = __builtin_amdgcn_make_buffer_rsrc(base, 0, 0x7FFFFFFF, 0x00020000);
    __builtin_amdgcn_raw_buffer_store_b128(v, r, 4 * at, 0, 16);
}
__device__ inline u4 load_shared4(const unsigned *base, unsigned at) {
    const auto r = __builtin_amdgcn_make_buffer_rsrc((unsigned *)base, 0, 0x7FFFFFFF, 0x00020000);
    return __builtin_amdgcn_raw_buffer_load_b128(r, 4 * at, 0, 16);
}

}  // namespace pklm
