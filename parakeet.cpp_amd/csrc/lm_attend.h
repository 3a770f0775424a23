// lm_attend.h -- attention over the 4-bit paged cache (pk_kv4_attend).
//
// With columns c for the 16 query rows of a tile (a row is a (token, query head of one kv head) pair), S = K Q^T and
// O^T = V^T P both run on v_mfma_f32_16x16x32_bf16.  K's and V's codes become bf16 with their block's scale applied in
// one conversion of two (exact: a level has two significant bits).  A bf16 query is its own operand, an f16 one the sum
// of two bf16 (exact: 11 bits in 8 + 8).  So scores are f32 sums of exact products; P is rounded to bf16, or for an f16
// result to a pair of them (16 bits).  The matrix core could multiply the 4-bit codes as they are
// (v_mfma_scale_f32_16x16x128_f8f6f4, queries as sums of 8-bit floats), at the same rate for exact bf16 queries and with
// no conversion of K, but its sums keep too little: errors of up to 2^-16 of the sum of magnitudes were measured, 2^-22
// for the bf16 products.
//
// The D layout of S (lane g*16 + c holds keys 4g .. 4g+3 of its 16-row tile, column c) is the B layout that O^T wants
// when tile t's row 4g + i stands for key 8g + 4t + i of 32: a lane's 8 probabilities are then its own operand and no
// value crosses lanes.  The cache's V order gives a lane its 8 keys x D/16 channels in one run of bytes; of a K row it
// takes D/4 adjacent channels, the order of channels being free as long as the queries have the same.
#pragma once

#include "lm_common.h"
#include "parakeet_lm.h"

namespace pklm {

constexpr int kAttendThreads = 512, kAttendWaves = 8;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttendParams {
    const void *q;
    void *out;
    float *lse;
    const uint8_t *cache;
    const int *table, *lens, *first;
    int *arrived;       // [tiles][1 + groups] how many groups of a tile are done, how many splits of each group
    float *part;        // [tiles][splits + groups][16][D sums, maximum, total, 2 unused]
    int64_t q_row, q_head, out_row, out_head, page_stride, table_stride;
    int n_rows, requests, heads, kv_heads, page, page_shift, n_pages, width, max_len, window, group;
    int tiles, splits, groups, chunk, vec, vec_out;
    float scale;
};

__device__ inline unsigned pack_bf16(float lo, float hi) {
    const bf2 v = {(__bf16)lo, (__bf16)hi};
    return __builtin_bit_cast(unsigned, v);
}

// The query operands of one 16-column tile: lane g*16 + c has channels g D/4 .. of column c, as one bf16 plane or two.
template <int D, int Planes>
struct Queries {
    u4 b[Planes][D / 32];

    template <class T>
    __device__ void load(const typename T::Raw *row, bool vec, bool negate) {
        const int g = (threadIdx.x & 63) >> 4;
        const typename T::Raw *p = row + g * (D / 4);
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) {
            unsigned short raw[8];
            if (vec) {
                *(u4 *)raw = ((const u4 *)p)[ks];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) raw[i] = p[8 * ks + i];
            }
            if (negate)
#pragma unroll
                for (int i = 0; i < 8; ++i) raw[i] ^= 0x8000;
            if (Planes == 1) {
                b[0][ks] = *(u4 *)raw;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = T::get(raw[2 * j]), y = T::get(raw[2 * j + 1]);
                    const unsigned hi = pack_bf16(x, y);
                    b[0][ks][j] = hi;
                    b[Planes - 1][ks][j] = pack_bf16(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xFFFF0000u));
                }
            }
        }
    }
};

// 8 codes as 8 bf16
__device__ inline u4 unpack8(unsigned w, float scale) {
    u4 r;
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
    return r;
}

__device__ inline v4f mfma(u4 a, u4 b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}

// max and sum over the four lanes g of a column
__device__ inline float column_max(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float column_sum(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ inline void store_shared(float *base, unsigned at, v4f v) {
    store_shared4((unsigned *)base, at, __builtin_bit_cast(u4, v));
}
__device__ inline v4f load_shared(const float *base, unsigned at) {
    return __builtin_bit_cast(v4f, load_shared4((const unsigned *)base, at));
}

// Where a lane's codes of 32 keys lie in their record, which does not change from step to step.  A step's keys are on
// one page, or with pages of 16 (Small) on two; on one page the rest of an address is the same in the whole wave.
template <int D, bool Small>
struct KeyOffsets {
    unsigned k, v;

    __device__ KeyOffsets(const Record &rec) {
        const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
        k = ((8 * (c >> 2) + (c & 3)) & (Small ? 15 : 31)) * (D / 2) + g * (D / 8);
        v = rec.v_codes() + (Small ? g & 1 : g) * (4 * D) + c * (D / 4);
    }
};

// One step's operands of a lane: 32 keys, of K two rows' D/4 channels, of V 8 keys' D/16 channels.
template <int D>
struct KeyTile {
    static constexpr int kKWords = D / 32, kVWords = D == 64 ? 4 : D / 16;
    unsigned k[2][kKWords], v[kVWords];
    unsigned ks[2];
    u2 vs;

    // id0, id1: pages of the tile's two 16-key halves (the same where pages are larger), -1: none
    template <bool Small>
    __device__ void load_k(const AttendParams &a, const Record &rec, const KeyOffsets<D, Small> &at, int64_t head_at, int kb, int id0,
                           int id1) {
        const uint8_t *p = a.cache + head_at + max(id0, 0) * a.page_stride;
        if (Small) p = (threadIdx.x & 8) ? a.cache + head_at + max(id1, 0) * a.page_stride : p;
        const int off = Small ? 0 : kb & (a.page - 1);
        const uint8_t *kp = p + off * (D / 2), *sp = p + off * (D / 32);
        unsigned kat = at.k;
        asm volatile("" : "+v"(kat));       // the scales' offset is worked out anew: registers are scarcer than that
        const unsigned ksat = rec.k_scales() + (kat >> 4);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if (D == 64) *(u2 *)k[t] = *(const u2 *)(kp + kat + 4 * t * (D / 2));
            else
#pragma unroll
                for (int i = 0; i < D / 128; ++i) *(u4 *)&k[t][4 * i] = *(const u4 *)(kp + kat + 4 * t * (D / 2) + 16 * i);
            ks[t] = D == 256 ? *(const uint16_t *)(sp + ksat + 4 * t * (D / 32)) : sp[ksat + 4 * t * (D / 32)];
        }
    }
    template <bool Small>
    __device__ void load_v(const AttendParams &a, const Record &rec, const KeyOffsets<D, Small> &at, int64_t head_at, int kb, int id0,
                           int id1) {
        const uint8_t *p = a.cache + head_at + max(id0, 0) * a.page_stride;
        if (Small) p = (threadIdx.x & 32) ? a.cache + head_at + max(id1, 0) * a.page_stride : p;
        const int off = Small ? 0 : kb & (a.page - 1);
        const uint8_t *vp = p + (off >> 3) * (4 * D), *sp = p + off;
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int g = lane >> 4, c = lane & 15;
        const unsigned vsat = rec.v_scales() + (c * (D / 16) / 32) * a.page + (Small ? g & 1 : g) * 8;
#pragma unroll
        for (int i = 0; i < kVWords / 4; ++i) *(u4 *)&v[4 * i] = *(const u4 *)(vp + at.v + 16 * i);
        vs = *(const u2 *)(sp + vsat);
    }
    // key j's word w of V codes (D = 64: its 16 bits, in the low half)
    __device__ unsigned v_word(int j, int w) const {
        return D == 64 ? (j & 1 ? v[j >> 1] >> 16 : v[j >> 1]) : v[j * (D / 128 > 0 ? D / 128 : 1) + w];
    }
};

// Online softmax of 16 columns over 32 keys a step, on one wave.
template <int D, int Planes>
struct Softmax {
    static constexpr int kTiles = D / 16;
    v4f acc[kTiles];      // O^T: channel (D/16)(4g + i) + n of column c in acc[n][i]
    float m, l;           // largest score so far (before the scale), this lane's share of the sum

    __device__ void clear() {
#pragma unroll
        for (int n = 0; n < kTiles; ++n) acc[n] = v4f{0, 0, 0, 0};
        m = -INFINITY, l = 0;
    }

    __device__ void scores(const KeyTile<D> &x, const Queries<D, Planes> &q, v4f (&s)[2]) const {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            s[t] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < D / 32; ++ks) {
                const unsigned sb = D == 256 ? x.ks[t] >> (8 * (ks / 4)) & 255u : x.ks[t];
                const u4 k8 = unpack8(x.k[t][ks], __uint_as_float(sb << 23));
#pragma unroll
                for (int n = 0; n < Planes; ++n) s[t] = mfma(k8, q.b[n][ks], s[t]);
            }
        }
    }

    // Keys vk .. vk + 7 of this lane: [lo, hi) is what its column sees, [lo_all, hi_all) what any column sees.  Scores
    // of keys not seen become -inf.  What lies at keys that no column sees may be anything: their V scale becomes 1.  A
    // NaN block of V that only some columns see is taken out, and those columns are made NaN.
    __device__ void mask(v4f (&s)[2], u2 &vs, int vk, bool fine, int lo, int hi, int lo_all, int hi_all) {
        unsigned nan_keys = 0, seen = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int key = vk + j, at = 8 * (j & 3);
            if (fine && key < hi && key >= lo) seen |= 1u << j;
            else s[j >> 2][j & 3] = -INFINITY;
            const bool dead = !fine || key >= hi_all || key < lo_all;
            const bool nan = (vs[j >> 2] >> at & 255u) == 255u;
            if (!dead && nan) nan_keys |= 1u << j;
            if (dead || nan) vs[j >> 2] = (vs[j >> 2] & ~(255u << at)) | 127u << at;
        }
        if (__any(nan_keys != 0)) {
            u4 va, pa;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                va[j] = (nan_keys >> (2 * j) & 1 ? 0x3F80u : 0) | (nan_keys >> (2 * j + 1) & 1 ? 0x3F800000u : 0);
                pa[j] = (seen >> (2 * j) & 1 ? 0x3F80u : 0) | (seen >> (2 * j + 1) & 1 ? 0x3F800000u : 0);
            }
            const v4f n = mfma(va, pa, v4f{0, 0, 0, 0});      // how many such keys each column sees, by channel entry
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n[i] > 0)
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) acc[t][i] = __builtin_nanf("");
        }
    }

    __device__ void add(const v4f (&s)[2], const KeyTile<D> &x, u2 vs, float to_log2) {
        float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                          fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        top = column_max(top);
        if (__any(top > m)) {
            const float m2 = fmaxf(m, top);
            const float keep = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - m2) * to_log2);
            m = m2;
            l *= keep;
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[n][i] *= keep;
        }
        const float shift = m == -INFINITY ? 0.0f : m;
        u4 ph, pl;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // subtracted first: s to_log2 - m to_log2 in one rounding is not 0 at s = m, and large scores overflow by it
            const float a = __builtin_amdgcn_exp2f((s[j >> 1][2 * (j & 1)] - shift) * to_log2);
            const float b = __builtin_amdgcn_exp2f((s[j >> 1][2 * (j & 1) + 1] - shift) * to_log2);
            l += a + b;
            ph[j] = pack_bf16(a, b);
            if (Planes == 2)      // an f16 result wants more than bf16's 8 bits of P: the rest of it as a second product
                pl[j] = pack_bf16(a - __uint_as_float(ph[j] << 16), b - __uint_as_float(ph[j] & 0xFFFF0000u));
        }
        float vscale[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) vscale[j] = __uint_as_float((vs[j >> 2] >> (8 * (j & 3)) & 255u) << 23);
        // two channels at a time: a byte of each key's codes
        auto two = [&](auto sel, int word, v4f &even, v4f &odd) {
            constexpr int kSel = decltype(sel)::value;
            u4 ve, vo;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x.v_word(2 * j, word), vscale[2 * j], kSel);
                const bf2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x.v_word(2 * j + 1, word), vscale[2 * j + 1], kSel);
                const unsigned au = __builtin_bit_cast(unsigned, a), bu = __builtin_bit_cast(unsigned, b);
                ve[j] = __builtin_amdgcn_perm(bu, au, 0x05040100u);
                vo[j] = __builtin_amdgcn_perm(bu, au, 0x07060302u);
            }
            even = mfma(ve, ph, even);
            odd = mfma(vo, ph, odd);
            if (Planes == 2) {
                even = mfma(ve, pl, even);
                odd = mfma(vo, pl, odd);
            }
        };
#pragma unroll
        for (int w = 0; w < (D == 64 ? 1 : D / 128); ++w) {
            two(std::integral_constant<int, 0>{}, w, acc[8 * w + 0], acc[8 * w + 1]);
            two(std::integral_constant<int, 1>{}, w, acc[8 * w + 2], acc[8 * w + 3]);
            if constexpr (D > 64) {
                two(std::integral_constant<int, 2>{}, w, acc[8 * w + 4], acc[8 * w + 5]);
                two(std::integral_constant<int, 3>{}, w, acc[8 * w + 6], acc[8 * w + 7]);
            }
        }
    }
};

// Splits meet in memory, sixteen at a time: the last of a group to arrive joins the group's sums, the last group to be
// joined joins those.  (One workgroup joining all of them takes 2 us for every 8: 40 of 63 us for 196 splits.)
constexpr int kJoin = 16;

__device__ inline bool last_to_come(int *counter, int of, int *s_last) {
    __builtin_amdgcn_s_waitcnt(0);        // this thread's sums have landed
    __syncthreads();
    if (threadIdx.x == 0) {
        *s_last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == of - 1;
        if (*s_last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return *s_last;
}

// base: [n][Cols][D sums, maximum, total, 2 unused]; finish(column, quad, sums of its 4 channels, maximum, total)
template <int D, int Cols, class Finish>
__device__ inline void join_some(const float *base, int n, int live, float to_log2, Finish finish) {
    constexpr int kQuads = D / 4, kRow = D + 4;
    for (int u = threadIdx.x; u < live * kQuads; u += kAttendThreads) {
        const int col = u / kQuads, quad = u % kQuads;
        v4f o = {0, 0, 0, 0};
        float top = -INFINITY, total = 0;
        // batches of 8, their loads together
        for (int i0 = 0; i0 < n; i0 += 8) {
            v4f x[8], ml[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned p = (min(i0 + i, n - 1) * Cols + col) * kRow;
                x[i] = load_shared(base, p + 4 * quad), ml[i] = load_shared(base, p + D);
            }
            float t2 = top;
#pragma unroll
            for (int i = 0; i < 8; ++i) t2 = fmaxf(t2, ml[i][0]);
            const float keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((top - t2) * to_log2);
            o *= keep, total *= keep, top = t2;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float w = t2 == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((ml[i][0] - t2) * to_log2);
                if (i0 + i < n) o += x[i] * w, total += ml[i][1] * w;
            }
        }
        finish(col, quad, o, top, total);
    }
}

// This split's sums are in its place of tile `at`; `mine` splits have keys.
template <int D, int Cols = 16, class Finish>
__device__ inline void join(const AttendParams &a, int64_t at, int split, int mine, int live, float to_log2, int *s_last, Finish finish) {
    constexpr int kPlace = Cols * (D + 4);
    float *all = a.part + at * (a.splits + a.groups) * kPlace, *joined = all + (int64_t)a.splits * kPlace;
    int *arrived = a.arrived + at * (1 + a.groups);
    const int group = split / kJoin, groups = (mine + kJoin - 1) / kJoin, n = min(kJoin, mine - group * kJoin);
    if (!last_to_come(arrived + 1 + group, n, s_last)) return;
    const float *base = all + (int64_t)group * kJoin * kPlace;
    if (groups == 1) {
        join_some<D, Cols>(base, n, live, to_log2, finish);
        return;
    }
    join_some<D, Cols>(base, n, live, to_log2, [&](int col, int quad, v4f o, float top, float total) {
        const unsigned p = (group * Cols + col) * (D + 4);
        store_shared(joined, p + 4 * quad, o);
        if (quad == 0) store_shared(joined, p + D, v4f{top, total, 0, 0});
    });
    if (!last_to_come(arrived, groups, s_last)) return;
    join_some<D, Cols>(joined, groups, live, to_log2, finish);
}

// One 16-column tile, its keys dealt to the eight waves 32 at a time; `splits` workgroups share a tile's keys.  Each wave
// keeps its own maximum, sum and O of all columns, in registers, and they meet once at the end: keys are read and unpacked
// once and no step waits for another wave.  What bounds it is memory where sessions are many: 64 of up to 4,097 keys, 32
// heads on 8 of 128 channels, 144 MB in 35 to 39 us (4.1 to 3.7 TB/s, a large copy 4.9).  200,003 and up to 100,001 keys on
// 2 kv heads in f16, 77 MB in 29.4 us (2.6 TB/s): the unpacking, two bf16 planes and the join, and the split, which goes by the
// longest request: up to 336 workgroups have keys, two on some units and one on most.  One session of 733 keys: 7.3 us, a launch,
// two steps of the first of its two splits, and their join.
template <class T, int D, bool Small>
__global__ __launch_bounds__(kAttendThreads, D == 256 ? 2 : 4) void attend_kernel(AttendParams a) {
    constexpr int Planes = __is_same(T, F16) ? 2 : 1;
    constexpr int kTiles = D / 16, kRow = D + 4;
    using Raw = typename T::Raw;
    __shared__ float s_m[kAttendWaves][16], s_l[kAttendWaves][16];
    __shared__ float s_o[4][16][kRow];
    __shared__ int s_last;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    int id = blockIdx.x;
    const int hk = id % a.kv_heads;
    id /= a.kv_heads;
    // Workgroups go round the 8 XCDs and within one round its 4 shader engines, in order: with 8 heads and 4 requests
    // each engine would get one request alone, and a long one would leave the others idle (measured: a quarter of the
    // slots in use).  So the requests are turned on by one from tile to tile.
    const int turn = id / a.requests, b = (id + turn) % a.requests;
    const int tile = turn % a.tiles, split = turn / a.tiles;

    const int f0 = a.first ? a.first[b] : b, f1 = a.first ? a.first[b + 1] : b + 1;
    const int q0 = max(f0, 0), q1 = min(f1, a.n_rows), rows = (q1 - q0) * a.group;
    if (q1 <= q0 || tile * 16 >= rows) return;
    const int held = max(min(min(a.lens[b], a.max_len), a.width * a.page), 0);
    const int row = min(tile * 16 + c, rows - 1), tok = row / a.group, head = hk * a.group + row % a.group;
    // keys [lo, hi) of this column; of the whole tile: tokens rise with the column
    const int place0 = held - (f1 - q0);                    // of the first token
    const int tok_a = tile * 16 / a.group, tok_b = (min(tile * 16 + 16, rows) - 1) / a.group;
    auto begin_of = [&](int p) { return a.window ? max(p + 1 - a.window, 0) : 0; };
    const int hi = max(place0 + tok + 1, 0), lo = begin_of(place0 + tok);
    const int hi_min = max(place0 + tok_a + 1, 0), hi_max = max(place0 + tok_b + 1, 0);
    const int lo_min = begin_of(place0 + tok_a), lo_max = begin_of(place0 + tok_b), start = lo_min & ~31;
    const int mine = max((hi_max - start + a.chunk - 1) / a.chunk, 1);     // splits with keys in them
    if (split >= mine) return;
    const int k0 = start + split * a.chunk, k1 = min(k0 + a.chunk, hi_max);

    Queries<D, Planes> q;
    q.template load<T>((const Raw *)a.q + (q0 + tok) * a.q_row + head * a.q_head, a.vec, a.scale < 0);
    // the scale's sign is in the queries; a scale of zero would make 0 * -inf of a key not seen
    const float to_log2 = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);

    const Record rec{a.page, D};
    const int64_t head_at = hk * rec.bytes();
    const int *table = a.table + b * a.table_stride;
    const int last_page = max(held - 1, 0) >> a.page_shift;
    auto page_of = [&](int key) {
        const int p = table[min(key >> a.page_shift, last_page)];
        return (unsigned)p < (unsigned)a.n_pages ? p : -1;
    };

    Softmax<D, Planes> sm;
    sm.clear();
    constexpr int kStride = 32 * kAttendWaves;
    int kb = k0 + 32 * wave;
    if (kb < k1) {
        // The next step's K is read into this one's registers as soon as the scores are formed, V after the sums; pages are
        // looked up a step ahead.  (A second set of registers, read a whole step ahead, spills where two planes of Q and P
        // are held, and takes longer elsewhere too: 64 sessions of up to 4,097 keys 37.5 us against 35.1, 200,003 and
        // 100,001 keys in f16 48.5 against 29.4.)
        const KeyOffsets<D, Small> at(rec);
        KeyTile<D> x;
        auto second = [&](int first, int key) { return Small ? page_of(key + 16) : first; };
        int id0 = page_of(kb), id1 = second(id0, kb);
        int n0 = page_of(kb + kStride), n1 = second(n0, kb + kStride);
        x.load_k(a, rec, at, head_at, kb, id0, id1);
        x.load_v(a, rec, at, head_at, kb, id0, id1);
        for (;;) {
            const int nb = kb + kStride < k1 ? kb + kStride : kb;
            const int l0 = nb == kb ? id0 : n0, l1 = nb == kb ? id1 : n1;
            n0 = page_of(nb + kStride), n1 = second(n0, nb + kStride);
            v4f s[2];
            sm.scores(x, q, s);
            __builtin_amdgcn_sched_barrier(0);
            x.load_k(a, rec, at, head_at, nb, l0, l1);
            u2 vs = x.vs;
            if (kb + 32 > hi_min || kb < lo_max || id0 < 0 || id1 < 0)
                sm.mask(s, vs, kb + 8 * g, (g < 2 ? id0 : id1) >= 0, lo, hi, lo_min, hi_max);
            sm.add(s, x, vs, to_log2);
            __builtin_amdgcn_sched_barrier(0);
            x.load_v(a, rec, at, head_at, nb, l0, l1);
            if (nb == kb) break;
            kb = nb, id0 = l0, id1 = l1;
        }
    }

    // the eight waves' sums into one, each brought to the common maximum first
    float l = column_sum(sm.l);
    if (g == 0) s_m[wave][c] = sm.m, s_l[wave][c] = l;
    __syncthreads();
    float M = s_m[0][c];
#pragma unroll
    for (int w = 1; w < kAttendWaves; ++w) M = fmaxf(M, s_m[w][c]);
    const float f = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((sm.m - M) * to_log2);
    const int live = min(rows - tile * 16, 16);
    float *mine_o = &s_o[wave & 3][c][kTiles * 4 * g];
#pragma unroll
    for (int round = 0; round < 2; ++round) {
        if (wave >> 2 == round && c < live)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < kTiles; n += 4) {
                    v4f x = {sm.acc[n][i] * f, sm.acc[n + 1][i] * f, sm.acc[n + 2][i] * f, sm.acc[n + 3][i] * f};
                    v4f *at = (v4f *)(mine_o + kTiles * i + n);
                    if (round) x += *at;
                    *at = x;
                }
        __syncthreads();
    }
    constexpr int kQuads = D / 4;       // 4 channels a thread from here on
    const int64_t at = ((int64_t)b * a.kv_heads + hk) * a.tiles + tile;
    float *all = a.part + at * (a.splits + a.groups) * 16 * kRow;      // 32-bit offsets: see attend_shape
    auto finish = [&](int col, int quad, v4f o, float top, float total) {
        const int r = tile * 16 + col, t = r / a.group, h = hk * a.group + r % a.group;
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        Raw *out = (Raw *)a.out + (int64_t)(q0 + t) * a.out_row + h * a.out_head + 4 * quad;
        Raw v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = T::put(T::held(o[i] * inv));
        if (a.vec_out) *(u2 *)out = *(u2 *)v;
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = v[i];
        if (a.lse && quad == 0)
            a.lse[(int64_t)(q0 + t) * a.heads + h] = total == 0.0f ? -INFINITY : top * to_log2 * kLn2 + logf(total);
    };
    for (int u = threadIdx.x; u < live * kQuads; u += kAttendThreads) {
        const int col = u / kQuads, quad = u % kQuads;
        v4f o = *(v4f *)&s_o[0][col][4 * quad];
#pragma unroll
        for (int w = 1; w < 4; ++w) o += *(v4f *)&s_o[w][col][4 * quad];
        float top = s_m[0][col], total = 0;
#pragma unroll
        for (int w = 1; w < kAttendWaves; ++w) top = fmaxf(top, s_m[w][col]);
#pragma unroll
        for (int w = 0; w < kAttendWaves; ++w)      // with no maximum the sums are 0, or NaN
            total += s_l[w][col] * (top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((s_m[w][col] - top) * to_log2));
        if (mine == 1) {
            finish(col, quad, o, top, total);
        } else {
            const unsigned p = (split * 16 + col) * kRow;
            store_shared(all, p + 4 * quad, o);
            if (quad == 0) store_shared(all, p + D, v4f{top, total, 0, 0});
        }
    }
    if (mine > 1) join<D>(a, at, split, mine, live, to_log2, &s_last, finish);
}

// ---- many query rows: prompts ----
//
// A workgroup takes 128 columns, a wave 32 of them, and goes over the keys 64 at a time.  K's and V's values are
// unpacked to bf16 once for the four waves, into LDS, two buffers deep: the next 64 keys' bytes are on their way from
// memory while these are worked on.  v_mfma_f32_32x32x16_bf16: a lane holds 16 scores of 32 keys of its own column, so
// the maximum crosses lanes once per 64 keys; row 8b + 4h + i of a score tile stands for key 16 (b / 2) + 8h + 4 (b % 2) + i,
// which makes a lane's scores its own operand of O^T as above.  V lies transposed, row 16j + r holding channel
// (D/16) r + j: rows that 16 lanes write together are adjacent.
//
// Four prompts of up to 2,047 tokens on up to 4,095 keys, 32 heads on 8 of 128 channels in bf16: 225 us, 162 GFLOP at 0.72
// PFLOP/s, where a large library product of bf16 reaches 1.22.  A wave and 64 keys take 1,024 cycles of matrix instructions
// and about 1,400 of vector ones (the exponentials and the unpacking); of two waves a vector unit the one's seldom run
// beside the other's for long.  LDS is as full as the matrix cores: eight waves a unit read 32 KB of K and V each, 256 KB in
// the 2,048 cycles of their matrix instructions, 128 bytes a cycle, since each operand read serves 32 columns only.  Memory is
// not (54 MB fetched).  Splitting the keys in two to shorten the tail took 342 us.

constexpr int kPromptThreads = 256, kPromptCols = 128, kPromptKeys = 64;

typedef float v16f __attribute__((ext_vector_type(16)));

__device__ inline v16f mfma32(u4 a, u4 b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}

// As KeyOffsets, for a thread's share of 64 keys.  Small: they may be on pages of their own, of 16 or 32 tokens.
template <int D, bool Small>
struct PromptOffsets {
    unsigned k, ks, v, vs;

    __device__ PromptOffsets(const AttendParams &a, const Record &rec) {
        const int t = threadIdx.x, quarter = t & 3, r = (t >> 1) & 15, half = t & 1;
        const int tokens = Small ? min(a.page, 64) : 64, kkey = (t >> 2) & (tokens - 1), vkey = ((t >> 5) * 8) & (tokens - 1);
        k = kkey * (D / 2) + quarter * (D / 8);
        ks = rec.k_scales() + kkey * (D / 32) + quarter * (D / 4) / 32;
        v = rec.v_codes() + (vkey >> 3) * (4 * D) + r * (D / 4) + (D == 256 ? 4 * half : 0);
        vs = rec.v_scales() + (r * (D / 16) / 32) * a.page + vkey;
    }
};

// One thread's share of 64 keys' bytes: of K a quarter of a key's channels, of V half the channels of an entry of 8 keys.
template <int D>
struct PromptBytes {
    unsigned k[D / 32], v[8], ks;
    u2 vs;

    // What is made of the bytes is made after this point, not before (the compiler would).
    __device__ void pin() {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) asm volatile("" : "+v"(k[i]));
#pragma unroll
        for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(v[i]));
        unsigned a = vs[0], b = vs[1];
        asm volatile("" : "+v"(ks), "+v"(a), "+v"(b));
        vs = u2{a, b};
    }

    // kid, vid: pages of this thread's keys, the same for all threads where pages hold 64 tokens or more (not Small)
    template <bool Small>
    __device__ void load(const AttendParams &a, const PromptOffsets<D, Small> &at, int64_t head_at, int kb, int kid, int vid) {
        const int half = threadIdx.x & 1, off = kb & (a.page - 1);
        const uint8_t *krec = a.cache + max(kid, 0) * a.page_stride + head_at;
        const uint8_t *vrec = Small ? a.cache + max(vid, 0) * a.page_stride + head_at : krec;
        const uint8_t *kp = krec + off * (D / 2), *ksp = krec + off * (D / 32), *vp = vrec + (off >> 3) * (4 * D), *vsp = vrec + off;
        if (D == 64) *(u2 *)k = *(const u2 *)(kp + at.k);
        else
#pragma unroll
            for (int i = 0; i < D / 128; ++i) *(u4 *)&k[4 * i] = *(const u4 *)(kp + at.k + 16 * i);
        ks = D == 256 ? *(const uint16_t *)(ksp + at.ks) : ksp[at.ks];
        if (D == 64) {
            const u4 w = *(const u4 *)(vp + at.v);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[2 * i] = w[i] >> (8 * half), v[2 * i + 1] = w[i] >> (16 + 8 * half);
        } else if (D == 128) {
            *(u4 *)&v[0] = *(const u4 *)(vp + at.v), *(u4 *)&v[4] = *(const u4 *)(vp + at.v + 16);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = *(const unsigned *)(vp + at.v + 8 * i);
        }
        vs = *(const u2 *)(vsp + at.vs);
    }
};

template <int D>
struct alignas(16) PromptTile {
    static constexpr int kKRow = D * 2 + 16, kVRow = kPromptKeys * 2 + 16;     // bytes; the pads spread rows over banks
    uint8_t k[kPromptKeys * kKRow], v[D * kVRow];

    uint8_t nan[kPromptKeys][D / 32];       // of an edge tile: blocks of V that are NaN

    // What lies at keys without a page may be anything; so at an edge, where some column does not see some key, at keys
    // outside [lo, hi), which no column sees.  NaN blocks of the others are taken out there and marked; marked becomes kb.
    __device__ void clean(PromptBytes<D> &x, int kb, bool edge, bool vfine, int lo, int hi, int &marked) {
        const int t = threadIdx.x, a8 = t >> 5, r = (t >> 1) & 15;
        if (edge || !vfine) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int at = 8 * (j & 3), kj = kb + 8 * a8 + j;
                const bool dead = !vfine || kj >= hi || kj < lo, bad = (x.vs[j >> 2] >> at & 255u) == 255u;
                if (edge) nan[8 * a8 + j][r * (D / 16) / 32] = bad && !dead;     // by all threads of the block alike
                if (bad && !dead) marked = kb;
                if (bad || dead) x.vs[j >> 2] = (x.vs[j >> 2] & ~(255u << at)) | 127u << at;
            }
        }
    }
    __device__ void stage(const PromptBytes<D> &x) {
        const int t = threadIdx.x, key = t >> 2, quarter = t & 3;
        uint8_t *krow = k + key * kKRow + quarter * (D / 2);
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
            const unsigned sb = D == 256 ? x.ks >> (8 * (w / 4)) & 255u : x.ks;
            *(u4 *)(krow + 16 * w) = unpack8(x.k[w], __uint_as_float(sb << 23));
        }
        const int a8 = t >> 5, r = (t >> 1) & 15, half = t & 1;
        const u2 vs = x.vs;
        float scale[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) scale[j] = __uint_as_float((vs[j >> 2] >> (8 * (j & 3)) & 255u) << 23);
        constexpr int kEach = D / 32;                  // channels of this thread, two a byte
        auto two = [&](auto sel, int shift) {
            constexpr int kSel = decltype(sel)::value;
            u4 even, odd;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bf2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x.v[2 * j] >> shift, scale[2 * j], kSel);
                const bf2 q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x.v[2 * j + 1] >> shift, scale[2 * j + 1], kSel);
                const unsigned pu = __builtin_bit_cast(unsigned, p), qu = __builtin_bit_cast(unsigned, q);
                even[j] = __builtin_amdgcn_perm(qu, pu, 0x05040100u);
                odd[j] = __builtin_amdgcn_perm(qu, pu, 0x07060302u);
            }
            const int n = half * kEach + 2 * kSel;
            *(u4 *)(v + (n * 16 + r) * kVRow + a8 * 16) = even;
            *(u4 *)(v + ((n + 1) * 16 + r) * kVRow + a8 * 16) = odd;
        };
        const int shift = D == 128 ? 16 * half : 0;
        two(std::integral_constant<int, 0>{}, shift);
        if constexpr (D >= 128) two(std::integral_constant<int, 1>{}, shift);
        if constexpr (D == 256) {
            two(std::integral_constant<int, 2>{}, shift);
            two(std::integral_constant<int, 3>{}, shift);
        }
    }
};

template <class T, int D, bool Small>
__global__ __launch_bounds__(kPromptThreads, D == 256 ? 1 : 2) void attend_prompt_kernel(AttendParams a) {
    constexpr int Planes = __is_same(T, F16) ? 2 : 1;
    constexpr int kSteps = D / 16, kTiles = D / 32;
    using Raw = typename T::Raw;
    __shared__ PromptTile<D> s_tile[2];
    __shared__ int s_missing[2], s_marked[2];       // the tile of each buffer that lacks a page, has marked NaN blocks

    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), h = lane >> 5, c = lane & 31;
    // the last tiles of a prompt see the most keys: they go first
    int id = blockIdx.x;
    const int hk = id % a.kv_heads;
    id /= a.kv_heads;
    const int turn = id / a.requests, b = (id + turn) % a.requests;       // turned on: see attend_kernel
    const int tile = a.tiles - 1 - turn;

    const int f0 = a.first ? a.first[b] : b, f1 = a.first ? a.first[b + 1] : b + 1;
    const int q0 = max(f0, 0), q1 = min(f1, a.n_rows), rows = (q1 - q0) * a.group, row0 = tile * kPromptCols;
    if (q1 <= q0 || row0 >= rows) return;
    const int held = max(min(min(a.lens[b], a.max_len), a.width * a.page), 0);
    const int place0 = held - (f1 - q0);
    auto end_of = [&](int r) { return max(place0 + r / a.group + 1, 0); };
    auto begin_of = [&](int r) { return a.window ? max(place0 + r / a.group + 1 - a.window, 0) : 0; };
    const int row_last = min(row0 + kPromptCols, rows) - 1;
    const int hi_min = end_of(row0), hi_max = end_of(row_last), lo_min = begin_of(row0), lo_max = begin_of(row_last);
    const int k0 = lo_min & ~(kPromptKeys - 1), k1 = hi_max;

    // this wave's columns
    const int wrow0 = row0 + wave * 32, row = min(wrow0 + c, rows - 1), tok = row / a.group, head = hk * a.group + row % a.group;
    const int hi = end_of(row), lo = begin_of(row);
    const int whi_min = end_of(min(wrow0, rows - 1)), whi_max = end_of(min(wrow0 + 31, rows - 1));
    const int wlo_min = begin_of(min(wrow0, rows - 1)), wlo_max = begin_of(min(wrow0 + 31, rows - 1));
    u4 q[Planes][kSteps];
    {
        const Raw *p = (const Raw *)a.q + (int64_t)(q0 + tok) * a.q_row + head * a.q_head + 8 * h;
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
            unsigned short raw[8];
            if (a.vec) {
                *(u4 *)raw = *(const u4 *)(p + 16 * ks);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) raw[i] = p[16 * ks + i];
            }
            if (a.scale < 0)
#pragma unroll
                for (int i = 0; i < 8; ++i) raw[i] ^= 0x8000;
            if (Planes == 1) {
                q[0][ks] = *(u4 *)raw;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = T::get(raw[2 * j]), y = T::get(raw[2 * j + 1]);
                    const unsigned top = pack_bf16(x, y);
                    q[0][ks][j] = top;
                    q[Planes - 1][ks][j] = pack_bf16(x - __uint_as_float(top << 16), y - __uint_as_float(top & 0xFFFF0000u));
                }
            }
        }
    }
    const float to_log2 = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);

    const Record rec{a.page, D};
    const int64_t head_at = hk * rec.bytes();
    const int *table = a.table + b * a.table_stride;
    const int last_page = max(held - 1, 0) >> a.page_shift;
    auto page_of = [&](int key) {
        const int p = table[min(key >> a.page_shift, last_page)];
        return (unsigned)p < (unsigned)a.n_pages ? p : -1;
    };

    v16f acc[kTiles];
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n][i] = 0;
    float m = -INFINITY, l = 0;

    const int kkey = t >> 2, vkey = (t >> 5) * 8;        // of 64, in this thread's staging
    auto edge_at = [&](int kb) { return kb + kPromptKeys > hi_min || kb < lo_max; };
    if (k0 < k1) {
        const PromptOffsets<D, Small> offsets(a, rec);
        PromptBytes<D> bytes;
        auto page_k = [&](int key) { return page_of(Small ? key + kkey : key); };
        auto page_v = [&](int key, int k_page) { return Small ? page_of(key + vkey) : k_page; };
        int kid = page_k(k0), vid = page_v(k0, kid);
        bytes.load(a, offsets, head_at, k0, kid, vid);
        if (t < 2) s_missing[t] = s_marked[t] = -1;
        __syncthreads();
        if (kid < 0 || vid < 0) s_missing[0] = k0;
        s_tile[0].clean(bytes, k0, edge_at(k0), vid >= 0, lo_min, hi_max, s_marked[0]);
        s_tile[0].stage(bytes);
        kid = page_k(k0 + kPromptKeys), vid = page_v(k0 + kPromptKeys, kid);
        bytes.load(a, offsets, head_at, k0 + kPromptKeys, kid, vid);
        int kid2 = page_k(k0 + 2 * kPromptKeys), vid2 = page_v(k0 + 2 * kPromptKeys, kid2);
        __syncthreads();
        int buf = 0;
        // While a tile is worked on, the next one is unpacked (between the products of Q and K, which leave the vector
        // unit free) and the one after that is on its way from memory; behind the last one the last page is read again.
        for (int kb = k0; kb < k1; kb += kPromptKeys, buf ^= 1) {
            const int nb = kb + kPromptKeys;
            PromptTile<D> &next = s_tile[buf ^ 1];
            if (D < 256) __builtin_amdgcn_s_setprio(0);
            if (kid < 0 || vid < 0) s_missing[buf ^ 1] = nb;
            next.clean(bytes, nb, edge_at(nb), vid >= 0, lo_min, hi_max, s_marked[buf ^ 1]);
            const bool active = kb < whi_max && nb > wlo_min;
            v16f s[2];
            const PromptTile<D> &x = s_tile[buf];
            {
                // all operands first, so that no product waits for its own; the two halves' products in turn, the next
                // tile's unpacking between them
                const int krow = 16 * (c >> 4) + 8 * ((c >> 2) & 1) + 4 * ((c >> 3) & 1) + (c & 3);
                constexpr int kAhead = kSteps < 8 ? kSteps : 8;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[u][i] = 0;
#pragma unroll
                for (int k8 = 0; k8 < kSteps; k8 += kAhead) {
                    u4 kk[2][kAhead];
#pragma unroll
                    for (int ks = 0; ks < kAhead; ++ks)
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            kk[u][ks] = *(const u4 *)(x.k + (32 * u + krow) * PromptTile<D>::kKRow + 32 * (k8 + ks) + 16 * h);
                    __builtin_amdgcn_sched_barrier(0);
                    if (k8 + kAhead >= kSteps) bytes.pin();
#pragma unroll
                    for (int ks = 0; ks < kAhead; ++ks)
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int n = 0; n < Planes; ++n) s[u] = mfma32(kk[u][ks], q[n][k8 + ks], s[u]);
                    if (k8 + kAhead >= kSteps) {
                        next.stage(bytes);
#pragma unroll
                        for (int i = 0; i < 2 * kAhead * Planes; ++i) {
                            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(0x202, 8 / Planes, 0);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            kid = kid2, vid = vid2;
            bytes.load(a, offsets, head_at, kb + 2 * kPromptKeys, kid, vid);
            kid2 = page_k(kb + 3 * kPromptKeys), vid2 = page_v(kb + 3 * kPromptKeys, kid2);
            if (active) {
                // a tile can be an edge, its NaN blocks marked, for other waves' columns and whole for this one's
                const bool missing = s_missing[buf] == kb, marked = s_marked[buf] == kb;
                if (kb + kPromptKeys > whi_min || kb < wlo_max || missing || marked) {
                    unsigned bad = 0;             // channel blocks whose NaN this column sees
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int at = 32 * (i >> 4) + 16 * (i >> 3 & 1) + 8 * h + (i & 7), key = kb + at;
                        const bool see = key < hi && key >= lo && !(missing && page_of(key) < 0);
                        if (!see) s[i >> 4][i & 15] = -INFINITY;
                        else if (marked)
#pragma unroll
                            for (int j = 0; j < D / 32; ++j) bad |= (unsigned)x.nan[at][j] << j;
                    }
                    bad |= (unsigned)__shfl_xor((int)bad, 32);
                    if (__any(bad != 0))
#pragma unroll
                        for (int n = 0; n < kTiles; ++n)
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const int r = (8 * (i >> 2) + 4 * h + (i & 3)) & 15;
                                if (bad >> (r * (D / 16) / 32) & 1) acc[n][i] = __builtin_nanf("");
                            }
                }
                float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
                for (int i = 1; i < 16; ++i) top = fmaxf(top, fmaxf(s[0][i], s[1][i]));
                {
                    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                    top = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
                }
                // sums are brought to a new maximum only where it has outgrown the old one by 2^6
                if (__any((top - m) * to_log2 > 6.0f)) {
                    const float m2 = fmaxf(m, top);
                    const float keep = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - m2) * to_log2);
                    m = m2;
                    l *= keep;
#pragma unroll
                    for (int n = 0; n < kTiles; ++n)
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[n][i] *= keep;
                }
                const float shift = m == -INFINITY ? 0.0f : m * to_log2;
                if (__any(fabsf(shift) > 0x1p24f)) {
                    // s to_log2 - shift in one rounding is not 0 at s = m: nothing beside what it is beyond such scores
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[u][i] = m == -INFINITY ? s[u][i] * to_log2 : (s[u][i] - m) * to_log2;
                } else {
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[u][i] = __builtin_fmaf(s[u][i], to_log2, -shift);
                }
                // 16 keys at a time: their products with V run beside the next ones' exponentials
                u4 ph[4], pl[4];
                auto exponentials = [&](int g) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float e0 = __builtin_amdgcn_exp2f(s[g >> 1][8 * (g & 1) + 2 * j]);
                        const float e1 = __builtin_amdgcn_exp2f(s[g >> 1][8 * (g & 1) + 2 * j + 1]);
                        l += e0 + e1;
                        ph[g][j] = pack_bf16(e0, e1);
                        if (Planes == 2)
                            pl[g][j] = pack_bf16(e0 - __uint_as_float(ph[g][j] << 16), e1 - __uint_as_float(ph[g][j] & 0xFFFF0000u));
                    }
                };
                u4 vv[2][kTiles];
                auto operands = [&](int g) {
#pragma unroll
                    for (int n = 0; n < kTiles; ++n)
                        vv[g & 1][n] = *(const u4 *)(x.v + (32 * n + c) * PromptTile<D>::kVRow + 32 * g + 16 * h);
                };
                // Waves that sum go before the other workgroup's that unpack: 231 -> 225 us; in f16, 512 tokens x 4 on up to
                // 8,191 keys, 408 -> 383.  (D = 256 is alone on its unit.)
                if (D < 256) __builtin_amdgcn_s_setprio(1);
                operands(0);
                __builtin_amdgcn_sched_barrier(0);
                exponentials(0);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    if (g < 3) operands(g + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    if (g < 3) exponentials(g + 1);
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) {
                        acc[n] = mfma32(vv[g & 1][n], ph[g], acc[n]);
                        if (Planes == 2) acc[n] = mfma32(vv[g & 1][n], pl[g], acc[n]);
                    }
#pragma unroll
                    for (int i = 0; i < kTiles; ++i) {
                        __builtin_amdgcn_sched_group_barrier(0x008, Planes, 1);
                        __builtin_amdgcn_sched_group_barrier(0x400, 8 / kTiles > 0 ? 8 / kTiles : 1, 1);
                        __builtin_amdgcn_sched_group_barrier(0x002, 4, 1);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            __syncthreads();
        }
    }
    {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
        l = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    const bool live = wrow0 + c < rows;
    // entry r of D/16 channels from acc[n][8 b + ..]: this lane has the entries 4h + i and 8 + 4h + i
    auto entry = [&](int half, int i, float (&v)[D / 16]) {
#pragma unroll
        for (int n = 0; n < kTiles; ++n) v[2 * n] = acc[n][4 * half + i], v[2 * n + 1] = acc[n][8 + 4 * half + i];
        return 8 * half + 4 * h + i;
    };
    if (!live) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    Raw *out = (Raw *)a.out + (int64_t)(q0 + tok) * a.out_row + head * a.out_head;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v[D / 16];
            const int r = entry(half, i, v);
            alignas(8) Raw w[D / 16];
#pragma unroll
            for (int j = 0; j < D / 16; ++j) w[j] = T::put(T::held(v[j] * inv));
            Raw *o = out + r * (D / 16);
            if (a.vec_out)
#pragma unroll
                for (int j = 0; j < D / 64; ++j) ((u2 *)o)[j] = ((u2 *)w)[j];
            else
#pragma unroll
                for (int j = 0; j < D / 16; ++j) o[j] = w[j];
        }
    if (a.lse && h == 0) a.lse[(int64_t)(q0 + tok) * a.heads + head] = l == 0.0f ? -INFINITY : m * to_log2 * kLn2 + logf(l);
}

}  // namespace pklm
