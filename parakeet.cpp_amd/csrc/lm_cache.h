// lm_cache.h -- rows into the 4-bit paged cache and out of it (pk_kv4_store, pk_kv4_load).
#pragma once

#include "lm_common.h"
#include "parakeet_lm.h"

namespace pklm {

constexpr int kRowThreads = 256, kRowPasses = 4;

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

// Where the 8 channels from 8c of a row are put from, and read to: f32 in registers.
template <int D, bool V>
__device__ inline void put_codes(const Place<D> &at, int c, unsigned code, unsigned scale) {
    if (V) {
        uint8_t *v = at.v(c);
        if (D == 64) {
            *(uint16_t *)v = (uint16_t)code;
            *(uint16_t *)(v + 8 * D / 32) = (uint16_t)(code >> 16);
        } else {
            *(unsigned *)v = code;
        }
        if ((c & 3) == 0) *at.vs(c >> 2) = (uint8_t)scale;
    } else {
        *(unsigned *)at.k(c) = code;
        if ((c & 3) == 0) *at.ks(c >> 2) = (uint8_t)scale;
    }
}
template <int D, bool V>
__device__ inline void get_codes(const Place<D> &at, int c, unsigned &code, unsigned &scale) {
    if (V) {
        const uint8_t *v = at.v(c);
        code = D == 64 ? *(const uint16_t *)v | (unsigned)*(const uint16_t *)(v + 8 * D / 32) << 16 : *(const unsigned *)v;
        scale = *at.vs(c >> 2);
    } else {
        code = *(const unsigned *)at.k(c);
        scale = *at.ks(c >> 2);
    }
}

// One thread takes 8 channels of one row of K or V at a time, four threads a block of 32; the largest magnitude is the
// integer maximum of the f32 patterns (a NaN's is above every other), its exponent the block's scale.  Eight adjacent
// threads take the same channels of 8 rows of V: where these go to the 8 slots of one group, as a prompt's do, they write
// 32 adjacent bytes, 512 with the channels beside.  A block of workgroups is one head's K or V, so that no thread divides
// by the number of heads; four passes a thread where there are many rows, their loads together.  24,577 rows of 8 x 128
// bf16: 32.8 us in (101 MB read, 27 written: 3.9 TB/s), 21.0 us back out (27 MB read, 101 written: 6.1 TB/s); with threads
// along the channels of V, one pass and 64-bit divisions 52 and 38.  64 rows: 2.7 and 2.5 us, a launch each.
template <class T, int D, bool Store, bool V, int Passes>
__device__ inline void some_rows(const pk_kv4_rows_desc &a, int page_shift, int wide, int h) {
    constexpr int kPer = D / 8, kPass = kRowThreads / kPer;
    constexpr int kNext = V ? 8 : 1;                     // threads from one to the next 8 channels of a row
    using Raw = typename T::Raw;
    const int t = threadIdx.x, c = V ? (t >> 3) % kPer : t % kPer;
    const int first = V ? (t & 7) + 8 * (t / (8 * kPer)) : t / kPer;
    const int64_t row0 = (int64_t)blockIdx.x * kPass * Passes + first;
    const Record rec{a.page, D};
    Raw *x_at = V ? (Raw *)a.v + h * a.v_head + 8 * c : (Raw *)a.k + h * a.k_head + 8 * c;
    const int64_t x_row = V ? a.v_row : a.k_row;
    uint8_t *cache = (uint8_t *)a.cache + h * rec.bytes();
    const int slots = a.n_pages << page_shift;
    int slot[Passes];
    float x[Passes][8];
    unsigned code[Passes], scale[Passes];
#pragma unroll
    for (int p = 0; p < Passes; ++p) {
        const int64_t row = row0 + p * kPass;
        slot[p] = row < a.n_rows ? a.slots[row] : -1;
        if (Store && row < a.n_rows) load8<T>(x_at + row * x_row, wide, x[p]);
    }
    auto place = [&](int s) {
        const int id = s >> page_shift;
        return Place<D>{cache + id * a.page_stride, a.page, s & (a.page - 1)};
    };
    if (!Store)
#pragma unroll
        for (int p = 0; p < Passes; ++p)
            if (slot[p] >= 0 && slot[p] < slots) get_codes<D, V>(place(slot[p]), c, code[p], scale[p]);
#pragma unroll
    for (int p = 0; p < Passes; ++p) {
        if (Store) {
            unsigned top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[p][i]) & 0x7FFFFFFFu);
            top = max(top, (unsigned)__shfl_xor((int)top, kNext));
            top = max(top, (unsigned)__shfl_xor((int)top, 2 * kNext));
            // top = 1.f 2^(ex - 127): the scale 2^(ex - 129) puts it in [4, 8), one step up in [2, 4); up if over 7
            int s = (int)(top >> 23) - 2 + ((top & 0x7FFFFFu) > 0x600000u);
            s = min(max(s, 7), 252);                     // clear of subnormal values; and 6 times the scale is finite
            unsigned w = 0;
            if (top < 0x7F800000u) {
                const float sc = __uint_as_float((unsigned)s << 23);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[p][0], x[p][1], sc, 0);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[p][2], x[p][3], sc, 1);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[p][4], x[p][5], sc, 2);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[p][6], x[p][7], sc, 3);
            } else {
                s = 255;
            }
            if (slot[p] >= 0 && slot[p] < slots) put_codes<D, V>(place(slot[p]), c, w, (unsigned)s);
        } else if (slot[p] >= 0 && slot[p] < slots) {
            const float sc = __uint_as_float(scale[p] << 23);
            typedef float v2f __attribute__((ext_vector_type(2)));
            v2f two;
#define PK_TWO(i)                                                                \
    two = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[p], sc, i);              \
    x[p][2 * i] = two[0], x[p][2 * i + 1] = two[1];
            PK_TWO(0) PK_TWO(1) PK_TWO(2) PK_TWO(3)
#undef PK_TWO
            if (scale[p] >= 127 + 14)                    // 4 x 2^14 is the first value past f16's largest
#pragma unroll
                for (int i = 0; i < 8; ++i) x[p][i] = T::held(x[p][i]);
            store8<T>(x_at + (row0 + p * kPass) * x_row, wide, x[p]);
        }
    }
}

template <class T, int D, bool Store, int Passes>
__global__ __launch_bounds__(kRowThreads) void rows_kernel(pk_kv4_rows_desc a, int page_shift, int wide) {
    const int h = blockIdx.y >> 1;
    if (blockIdx.y & 1) some_rows<T, D, Store, true, Passes>(a, page_shift, wide, h);
    else some_rows<T, D, Store, false, Passes>(a, page_shift, wide, h);
}

}  // namespace pklm
