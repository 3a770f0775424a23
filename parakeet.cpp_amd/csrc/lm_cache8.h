// lm_cache8.h -- rows into the 8-bit paged cache and out of it (pk_kv8_append, pk_kv8_load).
#pragma once

#include "lm_cache.h"
#include "lm_common.h"
#include "lm_rope.h"
#include "parakeet_lm.h"

namespace pklm {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef short v2s __attribute__((ext_vector_type(2)));

constexpr int kBlock = 32;                            // tokens under one scale
constexpr int kScaleMin = 127 - 100, kScaleMax = 127 + 119;     // as f32 exponents; 448 times the largest is finite

// Bytes of one (page, kv head) record and where its parts begin.
struct Record8 {
    int page, dim;
    __host__ __device__ int64_t bytes() const { return (int64_t)page * 2 * dim + page / 2; }
    __host__ __device__ int v_codes() const { return page * dim; }
    __host__ __device__ int scales() const { return page * 2 * dim; }
};

// Four values, none beyond 448 scale, as codes; NaN as NaN.
__device__ inline unsigned encode4(float a, float b, float c, float d, float scale) {
    v2s w = {0, 0};
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, a, b, scale, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, c, d, scale, true);
    return __builtin_bit_cast(unsigned, w);
}
__device__ inline u2 encode8(const float (&x)[8], float scale) {
    return u2{encode4(x[0], x[1], x[2], x[3], scale), encode4(x[4], x[5], x[6], x[7], scale)};
}
__device__ inline void decode8(u2 code, float scale, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const v2f lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(code[i], scale, false);
        const v2f hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(code[i], scale, true);
        x[4 * i] = lo[0], x[4 * i + 1] = lo[1], x[4 * i + 2] = hi[0], x[4 * i + 3] = hi[1];
    }
}

// Codes of the 8 channels from 8c of the row at offset `off` of its page: in K adjacent; in V the D/32 channels of 256 / D
// half entries, which are D/4 bytes, 8 tokens, apart.
template <int D, bool V>
__device__ inline int code_at(const Record8 &rec, int off, int c) {
    if (!V) return off * D + 8 * c;
    return rec.v_codes() + (off >> 3) * (8 * D) + c * 64 + (off & 7) * (D / 32);
}
template <int D, bool V>
__device__ inline void put_codes8(uint8_t *rec, int at, u2 code) {
    if (V && D == 64) {
#pragma unroll
        for (int i = 0; i < 4; ++i) *(uint16_t *)(rec + at + i * (D / 4)) = (uint16_t)(code[i >> 1] >> 16 * (i & 1));
    } else if (V && D == 128) {
        *(unsigned *)(rec + at) = code[0], *(unsigned *)(rec + at + D / 4) = code[1];
    } else {
        *(u2 *)(rec + at) = code;
    }
}
template <int D, bool V>
__device__ inline u2 get_codes8(const uint8_t *rec, int at) {
    if (V && D == 64) {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = *(const uint16_t *)(rec + at + i * (D / 4));
        return u2{w[0] | w[1] << 16, w[2] | w[3] << 16};
    }
    if (V && D == 128) return u2{*(const unsigned *)(rec + at), *(const unsigned *)(rec + at + D / 4)};
    return *(const u2 *)(rec + at);
}

// One head's K or V rows row0 .. row0 + n into one block, from its offset o0 on, on one wave: all values into registers
// (32 D, D/2 a lane), the largest magnitude, the scale, the codes.  Rows before o0 are held already: the block keeps the
// larger of both scales, and where that has grown they are rounded again.  (A power of two more drops at most the last
// bit of subnormal codes, below 2^-9 of the scale.)
template <class T, int D, bool V>
__device__ inline void append_rows(const pk_kv8_append_desc &a, const Turn &turn, const TurnTable<D> &table, int h, int64_t row0, int n, int slot0,
                                   int page_shift, bool wide) {
    using Raw = typename T::Raw;
    constexpr int kLanes = D / 8, kRows = 64 / kLanes, kPasses = kBlock / kRows;
    const int lane = threadIdx.x & 63, o0 = slot0 & (kBlock - 1), page_off = (slot0 & (a.page - 1)) - o0;
    // lanes of V: 8 rows, so that they write runs of bytes; 8 channel groups beside
    auto row_of = [&](int p) { return V ? 8 * (p / (D / 64)) + (lane & 7) : p * kRows + lane / kLanes; };
    auto c_of = [&](int p) { return V ? 8 * (p % (D / 64)) + (lane >> 3) : lane % kLanes; };
    auto begin = [&](int p) { return V ? 8 * (p / (D / 64)) : p * kRows; };
    constexpr int kSpan = V ? 8 : kRows;
    const Record8 rec{a.page, D};
    uint8_t *at = (uint8_t *)a.cache + (int64_t)(slot0 >> page_shift) * a.page_stride + h * rec.bytes();
    unsigned *scale_at = (unsigned *)(at + rec.scales() + (page_off / kBlock) * 16 + (V ? 4 : 0));
    const unsigned before = o0 ? *scale_at : 0;
    const Raw *x_at = V ? (const Raw *)a.v + h * a.v_head : (const Raw *)a.k + h * a.k_head;
    const int64_t x_row = V ? a.v_row : a.k_row;
    float x[kPasses][8], w[8];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[p][i] = 0;
        const int r = row_of(p);
        if (begin(p) < o0 + n && begin(p) + kSpan > o0 && r >= o0 && r < o0 + n) load8<T>(x_at + (row0 + r - o0) * x_row + 8 * c_of(p), wide, x[p]);
    }
    if (!V && (turn.norm || turn.rot)) {
        load_weights(a.k_weight, lane % kLanes, w);
#pragma unroll
        for (int p = 0; p < kPasses; ++p)
            if (begin(p) < o0 + n && begin(p) + kSpan > o0)
                norm_and_turn<D>(x[p], lane % kLanes, turn, table, min(max(row_of(p) - o0, 0), n - 1), w);
    }
    unsigned top = 0, all = 0;
#pragma unroll
    for (int p = 0; p < kPasses; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned m = __float_as_uint(x[p][i]) & 0x7FFFFFFFu;
            all = max(all, m), top = max(top, m < 0x7F800000u ? m : 0u);
        }
    top = __float_as_uint(wave_max(__uint_as_float(top)));
    bool bad = __any(all >= 0x7F800000u);
    if (bad)
#pragma unroll
        for (int p = 0; p < kPasses; ++p)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((__float_as_uint(x[p][i]) & 0x7F800000u) == 0x7F800000u) x[p][i] = __builtin_nanf("");
    // top = 1.f 2^(ex - 127): the scale 2^(ex - 127 - 8) puts it at or below 448 = 1.75 2^8 unless its fraction is over .75
    int s = (int)(top >> 23) - 8 + ((top & 0x7FFFFFu) > 0x600000u);
    s = min(max(s, kScaleMin), kScaleMax);
    if (o0) {
        const int old = min(max((int)(before >> 23 & 255u), kScaleMin), kScaleMax);
        bad |= before >> 31;
        if (s > old) {
            const float from = __uint_as_float((unsigned)old << 23), to = __uint_as_float((unsigned)s << 23);
#pragma unroll
            for (int p = 0; p < kPasses; ++p)
                if (begin(p) < o0 && row_of(p) < o0) {
                    const int place = code_at<D, V>(rec, page_off + row_of(p), c_of(p));
                    float y[8];
                    decode8(get_codes8<D, V>(at, place), from, y);
                    put_codes8<D, V>(at, place, encode8(y, to));
                }
        }
        s = max(s, old);
    }
    const float scale = __uint_as_float((unsigned)s << 23);
    if (s == kScaleMax) {
        const float most = 448.0f * scale;
#pragma unroll
        for (int p = 0; p < kPasses; ++p)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[p][i] = x[p][i] > most ? most : x[p][i] < -most ? -most : x[p][i];
    }
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const int r = row_of(p);
        if (begin(p) < o0 + n && begin(p) + kSpan > o0 && r >= o0 && r < o0 + n)
            put_codes8<D, V>(at, code_at<D, V>(rec, page_off + r, c_of(p)), encode8(x[p], scale));
    }
    if (lane == 0) {
        *scale_at = (unsigned)s << 23 | (bad ? 0x80000000u : 0u);
        if (V) *(u2 *)(scale_at + 1) = u2{0, 0};
    }
}

// A workgroup has `rows` rows of the call (at most kTurnRows) and takes the runs that begin in them: rows one after the other
// whose slots are one after the other in one block, 32 at most, the last of them perhaps behind its own rows.  Its waves go
// over the run's heads: K, V and where they are given the queries.  Rows without a slot are runs of one, for their query.
template <class T, int D>
__global__ __launch_bounds__(kTurnThreads) void append_kernel(pk_kv8_append_desc a, int rows, int page_shift, int wide_q, int wide_kv) {
    using Raw = typename T::Raw;
    __shared__ TurnTable<D> s_table;
    const Turn turn{a.inv_freq, a.pos, a.rot_dim, a.norm, a.interleaved, a.eps};
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // lane 1 has the first row, lane 0 the one before
    const int64_t row = (int64_t)blockIdx.x * rows - 1 + lane;
    const bool in = row >= 0 && row < a.n_rows, live = in && turn.live(row);
    int slot = live ? a.slots[row] : -1;
    if (slot >= a.n_pages << page_shift) slot = -1;
    slot = max(slot, -1);
    const int prior = __shfl_up(slot, 1);
    const bool more = lane > 0 && slot > 0 && prior >= 0 && slot == prior + 1 && (slot & (kBlock - 1)) != 0;
    const unsigned long long going = __ballot(more);
    unsigned long long begins = __ballot(lane > 0 && lane <= rows && live && !more && (slot >= 0 || a.heads > 0));
    const int units = 2 * a.kv_heads + a.heads;
    bool first = true;
    while (begins) {
        const int l = __builtin_ctzll(begins);
        begins &= begins - 1;
        const int slot0 = lane_value(slot, l), n = 1 + __builtin_ctzll(~(going >> (l + 1)));
        const int64_t row0 = (int64_t)blockIdx.x * rows - 1 + l;
        if (a.rot_dim) {
            if (!first) __syncthreads();
            s_table.fill(turn, row0, n);
            __syncthreads();
            first = false;
        }
        for (int u = blockIdx.y * kTurnWaves + wave; u < units; u += gridDim.y * kTurnWaves) {
            if (u < a.kv_heads) {
                if (slot0 >= 0) append_rows<T, D, false>(a, turn, s_table, u, row0, n, slot0, page_shift, wide_kv);
            } else if (u < 2 * a.kv_heads) {
                if (slot0 >= 0) append_rows<T, D, true>(a, turn, s_table, u - a.kv_heads, row0, n, slot0, page_shift, wide_kv);
            } else {
                const int h = u - 2 * a.kv_heads;
                turn_rows<T, D>((const Raw *)a.q + h * a.q_head, a.q_row, wide_q & 1, (Raw *)a.q_out + h * a.q_out_head, a.q_out_row, wide_q & 2,
                                a.q_weight, turn, s_table, row0, n);
            }
        }
    }
}

// Rows out of the cache: 8 channels a thread, of V eight adjacent threads the same channels of 8 rows.
template <class T, int D, bool V>
__device__ inline void load_rows8(const pk_kv4_rows_desc &a, int page_shift, bool wide, int h) {
    constexpr int kLanes = D / 8, kEach = kRowThreads / kLanes;
    const int t = threadIdx.x, c = V ? (t >> 3) % kLanes : t % kLanes;
    const int64_t row = (int64_t)blockIdx.x * kEach + (V ? (t & 7) + 8 * (t / (8 * kLanes)) : t / kLanes);
    if (row >= a.n_rows) return;
    const int slot = a.slots[row];
    if (slot < 0 || slot >= a.n_pages << page_shift) return;
    const Record8 rec{a.page, D};
    const int off = slot & (a.page - 1);
    const uint8_t *at = (const uint8_t *)a.cache + (int64_t)(slot >> page_shift) * a.page_stride + h * rec.bytes();
    const unsigned s = *(const unsigned *)(at + rec.scales() + off / kBlock * 16 + (V ? 4 : 0)) & 0x7F800000u;
    float x[8];
    decode8(get_codes8<D, V>(at, code_at<D, V>(rec, off, c)), __uint_as_float(s), x);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = T::held(x[i]);
    using Raw = typename T::Raw;
    store8<T>(V ? (Raw *)a.v + row * a.v_row + h * a.v_head + 8 * c : (Raw *)a.k + row * a.k_row + h * a.k_head + 8 * c, wide, x);
}

template <class T, int D>
__global__ __launch_bounds__(kRowThreads) void load8_kernel(pk_kv4_rows_desc a, int page_shift, int wide) {
    const int h = blockIdx.y >> 1;
    if (blockIdx.y & 1) load_rows8<T, D, true>(a, page_shift, wide, h);
    else load_rows8<T, D, false>(a, page_shift, wide, h);
}

}  // namespace pklm
