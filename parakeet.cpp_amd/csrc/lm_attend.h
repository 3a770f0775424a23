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

constexpr int kAttendThreads = 256, kAttendWaves = 4;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttendParams {
    const void *q;
    void *out;
    float *lse;
    const uint8_t *cache;
    const int *table, *lens, *first;
    int *arrived;       // [tiles] how many splits of a tile are done
    float *part;        // [splits][rows][D + 2]
    int64_t q_row, q_head, out_row, out_head, page_stride, table_stride;
    int n_rows, requests, heads, kv_heads, page, page_shift, n_pages, width, max_len, window, group;
    int tiles, splits, chunk, vec;
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
    __device__ void load(const typename T::Raw *row, bool vec) {
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

// One 16-column tile, its keys dealt to the four waves 32 at a time; `splits` workgroups share a tile's keys.
template <class T, int D>
__global__ __launch_bounds__(kAttendThreads) void attend_kernel(AttendParams a) {
    constexpr int Planes = __is_same(T, F16) ? 2 : 1;
    constexpr int kTiles = D / 16;                          // channel tiles of O^T, and channels of a V entry
    constexpr int kWords = D / 32 >= 4 ? D / 128 : 1;       // 32-bit words of a V entry (D = 64: half of one)
    using Raw = typename T::Raw;
    __shared__ float s_m[kAttendWaves][16], s_l[kAttendWaves][16];
    __shared__ float s_o[kAttendWaves][16][D + 4];
    __shared__ int s_last;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    int id = blockIdx.x;
    const int hk = id % a.kv_heads;
    id /= a.kv_heads;
    const int b = id % a.requests;
    id /= a.requests;
    const int tile = id % a.tiles, split = id / a.tiles;

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
    const int lo_min = begin_of(place0 + tok_a) & ~31, lo_max = begin_of(place0 + tok_b);
    const int mine = max((hi_max - lo_min + a.chunk - 1) / a.chunk, 1);     // splits with keys in them
    if (split >= mine) return;
    const int k0 = lo_min + split * a.chunk, k1 = min(k0 + a.chunk, hi_max);

    Queries<D, Planes> q;
    q.template load<T>((const Raw *)a.q + (q0 + tok) * a.q_row + head * a.q_head, a.vec);

    const Record rec{a.page, D};
    const int64_t head_at = hk * rec.bytes();
    const int *table = a.table + b * a.table_stride;
    const int last_page = max(held - 1, 0) >> a.page_shift;

    v4f acc[kTiles];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) acc[n] = v4f{0, 0, 0, 0};
    float m = -INFINITY, l = 0;
    const float to_log2 = a.scale * kLog2e;

    for (int kb = k0 + 32 * wave; kb < k1; kb += 32 * kAttendWaves) {
        // two 16-row code tiles; row 4x + i of tile t is key kb + 8x + 4t + i
        const int kk = kb + 8 * (c >> 2) + (c & 3);
        const int kp = table[min(kk >> a.page_shift, last_page)];
        const int vk = kb + 8 * g;
        const int vp = table[min(vk >> a.page_shift, last_page)];
        const bool kfine = (unsigned)kp < (unsigned)a.n_pages, vfine = (unsigned)vp < (unsigned)a.n_pages;
        const uint8_t *krec = a.cache + (kfine ? kp : 0) * a.page_stride + head_at;
        const uint8_t *vrec = a.cache + (vfine ? vp : 0) * a.page_stride + head_at;
        const int koff = kk & (a.page - 1), voff = vk & (a.page - 1);

        v4f s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            s[t] = v4f{0, 0, 0, 0};
            const uint8_t *code = krec + (koff + 4 * t) * (D / 2) + g * (D / 8);
            const uint8_t *sc = krec + rec.k_scales() + (koff + 4 * t) * (D / 32) + g * (D / 4) / 32;
            unsigned w[D / 32];
            if (D == 64) *(u2 *)w = *(const u2 *)code;
            else
#pragma unroll
                for (int i = 0; i < D / 128; ++i) *(u4 *)&w[4 * i] = *(const u4 *)(code + 16 * i);
#pragma unroll
            for (int ks = 0; ks < D / 32; ++ks) {
                const u4 k8 = unpack8(w[ks], __uint_as_float((unsigned)sc[ks / 4] << 23));
#pragma unroll
                for (int n = 0; n < Planes; ++n) s[t] = mfma(k8, q.b[n][ks], s[t]);
            }
        }
        // V: 8 keys x D/16 channels, 8 scale bytes
        unsigned vw[8 * kWords];
        const uint8_t *vcode = vrec + rec.v_codes() + (voff >> 3) * (4 * D) + c * (D / 4);
        if (D == 64) {
            const u4 h = *(const u4 *)vcode;
#pragma unroll
            for (int i = 0; i < 4; ++i) vw[2 * i] = h[i] & 0xFFFFu, vw[2 * i + 1] = h[i] >> 16;
        } else {
#pragma unroll
            for (int i = 0; i < 2 * kWords; ++i) *(u4 *)&vw[4 * i] = *(const u4 *)(vcode + 16 * i);
        }
        u2 vs = *(const u2 *)(vrec + rec.v_scales() + (c * (D / 16) / 32) * a.page + voff);

        float p[8];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) p[4 * t + i] = s[t][i] * to_log2;
        unsigned nan_keys = 0;
        if (kb + 32 > hi_min || kb < lo_max || !__all(vfine)) {
            // some key of the 32 is not seen by some column: its score goes, and so does what its V holds.  A NaN block
            // seen by some columns alone is taken out and marked for those.
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = vk + j, at = 8 * (j & 3);
                if (!vfine || key >= hi || key < lo) p[j] = -INFINITY;
                const bool dead = !vfine || key >= hi_max || key < lo_min;     // what lies there may be anything
                const bool nan = (vs[j >> 2] >> at & 255u) == 255u;
                if (!dead && nan) nan_keys |= 1u << j;
                if (dead || nan) vs[j >> 2] = (vs[j >> 2] & ~(255u << at)) | 127u << at;
            }
        }
        if (__any(nan_keys != 0)) {
            u4 va, pa;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                va[j] = (nan_keys >> (2 * j) & 1 ? 0x3F80u : 0) | (nan_keys >> (2 * j + 1) & 1 ? 0x3F800000u : 0);
                const bool see0 = vfine && vk + 2 * j < hi && vk + 2 * j >= lo;
                const bool see1 = vfine && vk + 2 * j + 1 < hi && vk + 2 * j + 1 >= lo;
                pa[j] = (see0 ? 0x3F80u : 0) | (see1 ? 0x3F800000u : 0);
            }
            v4f n = {0, 0, 0, 0};
            n = mfma(va, pa, n);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n[i] > 0)
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) acc[t][i] = __builtin_nanf("");
        }

        float top = p[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, p[j]);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        if (__any(top > m)) {
            const float m2 = fmaxf(m, top), keep = exp2f(m == -INFINITY ? -INFINITY : m - m2);
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
            const float x = __builtin_amdgcn_exp2f(p[2 * j] - shift), y = __builtin_amdgcn_exp2f(p[2 * j + 1] - shift);
            l += x + y;
            ph[j] = pack_bf16(x, y);
            if (Planes == 2)      // an f16 result wants more than bf16's 8 bits of P: the rest of it as a second product
                pl[j] = pack_bf16(x - __uint_as_float(ph[j] << 16), y - __uint_as_float(ph[j] & 0xFFFF0000u));
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
                const bf2 x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(vw[2 * j * kWords + word], vscale[2 * j], kSel);
                const bf2 y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(vw[(2 * j + 1) * kWords + word], vscale[2 * j + 1], kSel);
                const unsigned xu = __builtin_bit_cast(unsigned, x), yu = __builtin_bit_cast(unsigned, y);
                ve[j] = __builtin_amdgcn_perm(yu, xu, 0x05040100u);
                vo[j] = __builtin_amdgcn_perm(yu, xu, 0x07060302u);
            }
            even = mfma(ve, ph, even);
            odd = mfma(vo, ph, odd);
            if (Planes == 2) {
                even = mfma(ve, pl, even);
                odd = mfma(vo, pl, odd);
            }
        };
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            two(std::integral_constant<int, 0>{}, w, acc[8 * w + 0], acc[8 * w + 1]);
            two(std::integral_constant<int, 1>{}, w, acc[8 * w + 2], acc[8 * w + 3]);
            if constexpr (D > 64) {
                two(std::integral_constant<int, 2>{}, w, acc[8 * w + 4], acc[8 * w + 5]);
                two(std::integral_constant<int, 3>{}, w, acc[8 * w + 6], acc[8 * w + 7]);
            }
        }
    }

    // the four waves' sums into one
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) s_m[wave][c] = m, s_l[wave][c] = l;
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_o[wave][c][kTiles * (4 * g + i) + n] = acc[n][i];
    __syncthreads();
    const int live = min(rows - tile * 16, 16);
    const int col = threadIdx.x >> 4, part = threadIdx.x & 15;         // 16 threads a column, D/16 channels each
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kAttendWaves; ++w) M = fmaxf(M, s_m[w][col]);
    const float shift = M == -INFINITY ? 0.0f : M;
    float L = 0, o[kTiles];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) o[n] = 0;
#pragma unroll
    for (int w = 0; w < kAttendWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(s_m[w][col] - shift);
        L += f * s_l[w][col];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) o[n] += f * s_o[w][col][part * kTiles + n];
    }
    const int row2 = tile * 16 + col;
    if (mine > 1) {
        // splits meet in memory; the last to arrive adds them up
        const int64_t at = ((int64_t)b * a.kv_heads + hk) * a.tiles + tile;
        float *p = a.part + ((at * a.splits + split) * 16 + col) * (D + 2);
        if (col < live) {
            if (part == 0) p[D] = M, p[D + 1] = L;
#pragma unroll
            for (int n = 0; n < kTiles; ++n) p[part * kTiles + n] = o[n];
        }
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
            s_last = atomicAdd(&a.arrived[at], 1) == mine - 1;
            if (s_last) atomicExch(&a.arrived[at], 0);
        }
        __syncthreads();
        if (!s_last) return;
        __threadfence();
        if (col >= live) return;
        const float *all = a.part + (at * a.splits * 16 + col) * (D + 2);
        M = -INFINITY;
        for (int i = 0; i < mine; ++i) M = fmaxf(M, all[(int64_t)i * 16 * (D + 2) + D]);
        const float sh = M == -INFINITY ? 0.0f : M;
        L = 0;
#pragma unroll
        for (int n = 0; n < kTiles; ++n) o[n] = 0;
        for (int i = 0; i < mine; ++i) {
            const float *pi = all + (int64_t)i * 16 * (D + 2);
            const float f = __builtin_amdgcn_exp2f(pi[D] - sh);
            L += f * pi[D + 1];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) o[n] += f * pi[part * kTiles + n];
        }
    }
    if (col >= live) return;
    const int tok2 = row2 / a.group, head2 = hk * a.group + row2 % a.group;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    Raw *out = (Raw *)a.out + (int64_t)(q0 + tok2) * a.out_row + head2 * a.out_head + part * kTiles;
#pragma unroll
    for (int n = 0; n < kTiles; ++n) out[n] = T::put(o[n] * inv);
    if (a.lse && part == 0) a.lse[(int64_t)(q0 + tok2) * a.heads + head2] = L == 0.0f ? -INFINITY : (M + log2f(L)) * kLn2;
}

}  // namespace pklm
