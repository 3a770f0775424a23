// lm_cache.h -- rows into the 4-bit paged cache and out of it (pk_kv4_store, pk_kv4_load).
#pragma once

#include "lm_common.h"
#include "parakeet_lm.h"

namespace pklm {

constexpr int kRowThreads = 256;

template <class T>
__device__ inline void load8(const typename T::Raw *p, bool wide, float (&x)[8]) {
    if (sizeof(typename T::Raw) == 2) {
        unsigned short r[8];
        if (wide) {
            *(u4 *)r = *(const u4 *)p;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) r[i] = ((const unsigned short *)p)[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = T::get((typename T::Raw)r[i]);
    } else {
        float r[8];
        if (wide) {
            ((u4 *)r)[0] = ((const u4 *)p)[0];
            ((u4 *)r)[1] = ((const u4 *)p)[1];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) r[i] = ((const float *)p)[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = r[i];
    }
}

template <class T>
__device__ inline void store8(typename T::Raw *p, bool wide, const float (&x)[8]) {
    typename T::Raw r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = T::put(x[i]);
    if (wide) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(r) / 16; ++i) ((u4 *)p)[i] = ((u4 *)r)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = r[i];
    }
}

// Where the 8 channels from 8c of a row lie: K codes are 4 adjacent bytes; V codes are spread over D/16-channel entries.
template <int D>
struct Place {
    uint8_t *rec;
    int page, off;
    __device__ uint8_t *k(int c) const { return rec + off * (D / 2) + 4 * c; }
    __device__ uint8_t *v(int c) const {
        uint8_t *base = rec + page * (D / 2) + (off >> 3) * (8 * D / 2) + (off & 7) * (D / 32);
        if (D == 64) return base + (2 * c) * (8 * D / 32);                     // entries 2c and 2c + 1, 2 bytes each
        if (D == 128) return base + c * (8 * D / 32);                          // entry c
        return base + (c >> 1) * (8 * D / 32) + (c & 1) * 4;                   // half of entry c / 2
    }
    __device__ uint8_t *ks(int g) const { return rec + page * D + off * (D / 32) + g; }
    __device__ uint8_t *vs(int g) const { return rec + page * D + page * (D / 32) + g * page + off; }
};

// One thread takes 8 channels of one row of K or V, four threads a block of 32; the largest magnitude is the integer
// maximum of the f32 patterns (a NaN's is above every other), its exponent the block's scale.
template <class T, int D, bool Store>
__global__ __launch_bounds__(kRowThreads) void rows_kernel(pk_kv4_rows_desc a, int wide) {
    const int64_t unit = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
    const int c = (int)(unit % (D / 8));                 // which 8 channels
    const int64_t rest = unit / (D / 8);
    const int which = (int)(rest & 1);                   // K or V
    const int64_t rh = rest >> 1;
    const int h = (int)(rh % a.heads);
    const int64_t row = rh / a.heads;
    if (row >= a.n_rows) return;                         // whole blocks of 32 channels: four threads leave together
    const int slot = a.slots[row];
    if (slot < 0 || slot >= (int64_t)a.n_pages * a.page) return;
    using Raw = typename T::Raw;
    Raw *x_at = which ? (Raw *)a.v + row * a.v_row + h * a.v_head : (Raw *)a.k + row * a.k_row + h * a.k_head;
    const Record rec{a.page, D};
    const int id = slot / a.page;
    const Place<D> at{(uint8_t *)a.cache + id * a.page_stride + h * rec.bytes(), a.page, slot - id * a.page};
    float x[8];
    if (Store) {
        load8<T>(x_at + 8 * c, wide, x);
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
        top = max(top, (unsigned)__shfl_xor((int)top, 1));
        top = max(top, (unsigned)__shfl_xor((int)top, 2));
        // top = 1.f 2^(ex - 127): the scale 2^(ex - 129) puts it in [4, 8), one step up in [2, 4); up if over 7
        int s = (int)(top >> 23) - 2 + ((top & 0x7FFFFFu) > 0x600000u);
        s = min(max(s, 7), 252);                         // clear of subnormal values; and 6 times the scale is finite
        unsigned code = 0;
        if (top < 0x7F800000u) {
            const float scale = __uint_as_float((unsigned)s << 23);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[0], x[1], scale, 0);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[2], x[3], scale, 1);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[4], x[5], scale, 2);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[6], x[7], scale, 3);
        } else {
            s = 255;
        }
        if (which) {
            uint8_t *v = at.v(c);
            if (D == 64) {
                *(uint16_t *)v = (uint16_t)code;
                *(uint16_t *)(v + 8 * D / 32) = (uint16_t)(code >> 16);
            } else {
                *(unsigned *)v = code;
            }
            if ((c & 3) == 0) *at.vs(c >> 2) = (uint8_t)s;
        } else {
            *(unsigned *)at.k(c) = code;
            if ((c & 3) == 0) *at.ks(c >> 2) = (uint8_t)s;
        }
    } else {
        unsigned code;
        if (which) {
            const uint8_t *v = at.v(c);
            code = D == 64 ? *(const uint16_t *)v | (unsigned)*(const uint16_t *)(v + 8 * D / 32) << 16 : *(const unsigned *)v;
        } else {
            code = *(const unsigned *)at.k(c);
        }
        const unsigned s = which ? *at.vs(c >> 2) : *at.ks(c >> 2);
        const float scale = __uint_as_float(s << 23);
        typedef float v2f __attribute__((ext_vector_type(2)));
        v2f p;
#define PK_TWO(i)                                                            \
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, i);            \
    x[2 * i] = p[0], x[2 * i + 1] = p[1];
        PK_TWO(0) PK_TWO(1) PK_TWO(2) PK_TWO(3)
#undef PK_TWO
        store8<T>(x_at + 8 * c, wide, x);
    }
}

}  // namespace pklm
