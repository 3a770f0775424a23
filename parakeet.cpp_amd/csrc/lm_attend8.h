// lm_attend8.h -- attention over the 8-bit paged cache (pk_kv8_attend).
//
// As in lm_attend.h, S = K Q^T and O^T = V^T P run on 16-bit matrix instructions whose D layout of S is the B layout that
// O^T wants, and tiles' sums meet by its join.  What a code of 8 bits allows:
//   K's codes, four significant bits, are exact in bf16 and in f16 without their scale, so queries of either type are their own
//   operand, products are exact, and the block's scale comes to the f32 scores.
//   V's codes and P go through f16.  A code is taken times 2^(e - r + 7), e its block's exponent and r the largest of any block so far:
//   at most 57,344, exact down to e = r - 22, and below that off by 2^-41 of the largest value of the blocks at r.  Sums are
//   brought to a new r by a power of two.  P is taken times 2^14 (or 2^9 where it may pass 1 by 2^6), so that f16's 11
//   bits hold down to 2^-28; it is what a result's error comes from beside its own rounding: 2^-11 sum p |v|.
// A step of 32 keys, and a wave's share of a prompt's 64, lie in one block: on one page, under one scale of K and one of V.
//
// What lies at keys that no column sees may be anything: their V codes become zeros.  A block that holds a NaN has a
// negative scale of V; where some columns see such a key and others do not its NaNs are taken out and put into the
// channels of the columns that see them.
#pragma once

#include <utility>

#include "lm_attend.h"
#include "lm_cache8.h"

namespace pklm {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// f(0), f(1) .. f(N - 1), each a constant.
template <class F, int... I>
__device__ inline void unrolled(F f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, class F>
__device__ inline void unrolled(F f) { unrolled(f, std::make_integer_sequence<int, N>{}); }

__device__ inline unsigned pack_f16(float lo, float hi) {
    const h2 v = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(unsigned, v);
}
// Two codes, a word's lower or upper half, as T without a scale; as f16 with one.
template <class T>
__device__ inline unsigned codes2(unsigned w, bool high) {
    if (__is_same(T, F16))
        return high ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))
                    : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    return high ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))
                : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
}
__device__ inline unsigned scaled2(unsigned w, bool high, float scale) {
    return high ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true))
                : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
}
template <class T>
__device__ inline u4 codes8(unsigned a, unsigned b) {
    return u4{codes2<T>(a, false), codes2<T>(a, true), codes2<T>(b, false), codes2<T>(b, true)};
}
__device__ inline bool nan_code(unsigned code) { return (code & 0x7Fu) == 0x7Fu; }

template <class T>
__device__ inline v4f mfma16(u4 a, u4 b, v4f c) {
    if (__is_same(T, F16)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    return mfma(a, b, c);
}
template <class T>
__device__ inline v16f mfma32x(u4 a, u4 b, v16f c) {
    if (__is_same(T, F16)) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    return mfma32(a, b, c);
}

// A value that is the same in the whole wave, through the scalar cache: what waits for it does not wait for the keys and values that
// were asked for before it.  (Read as vectors, page ids and scales held up each step of a prompt: 265 us, not 250, for 4
// prompts of up to 2,047 tokens on up to 4,095 keys, 32 heads on 8 x 128 in bf16.)
template <class V>
__device__ inline V scalar(const void *p) { return *(const __attribute__((address_space(4))) V *)(uintptr_t)p; }

// The exponent of a block's scale of V, and the power of two that codes are taken times; -128 stands for no block so far.
constexpr int kNoExponent = -128, kCodeShift = 7;
__device__ inline int exponent_of(float scale) { return __builtin_amdgcn_readfirstlane((int)(__float_as_uint(scale) >> 23 & 255u)) - 127; }
__device__ inline float code_scale(int e, int r) { return __uint_as_float((unsigned)max(e - r + kCodeShift + 127, 1) << 23); }
__device__ inline float power_of_two(int e) { return e < -126 ? 0.0f : __uint_as_float((unsigned)(min(e, 127) + 127) << 23); }

// One step's operands of a lane: 32 keys, of K two rows' D/4 channels, of V 8 keys' D/16 channels.
template <int D>
struct KeyTile8 {
    static constexpr int kKWords = D / 16, kVWords = D / 8;
    unsigned k[2][kKWords], v[kVWords];
    float ks, vs;

    // where the lane's codes lie in a block of a record
    struct Offsets {
        unsigned k, v;
        __device__ Offsets(const Record8 &rec) {
            const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
            k = (8 * (c >> 2) + (c & 3)) * D + g * (D / 4);
            v = rec.v_codes() + g * (8 * D) + c * (D / 2);
        }
    };

    __device__ void load_k(const AttendParams &a, const Record8 &rec, const Offsets &at, int64_t head_at, int kb, int id) {
        const uint8_t *p = a.cache + head_at + max(id, 0) * a.page_stride;
        const int off = kb & (a.page - 1);
        const uint8_t *kp = p + off * D;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < kKWords / 4; ++i) *(u4 *)&k[t][4 * i] = *(const u4 *)(kp + at.k + 4 * t * D + 16 * i);
        ks = fabsf(scalar<float>(p + rec.scales() + off / kBlock * 16));
    }
    __device__ void load_v(const AttendParams &a, const Record8 &rec, const Offsets &at, int64_t head_at, int kb, int id) {
        const uint8_t *p = a.cache + head_at + max(id, 0) * a.page_stride;
        const int off = kb & (a.page - 1);
        const uint8_t *vp = p + off * D;
#pragma unroll
        for (int i = 0; i < kVWords / 4; ++i) *(u4 *)&v[4 * i] = *(const u4 *)(vp + at.v + 16 * i);
        vs = scalar<float>(p + rec.scales() + off / kBlock * 16 + 4);
    }
    // where the pair of channels 2 Pair, 2 Pair + 1 of key j lies: 16 bits of a word
    static constexpr int v_word(int pair, int j) { return (pair / (D / 64) * (D / 4) + j * (D / 32) + pair % (D / 64) * 2) / 4; }
    static constexpr int v_half(int pair, int j) { return (j * (D / 32) + pair % (D / 64) * 2) / 2 & 1; }

    // Of keys vk .. vk + 7 of this lane, those outside [lo, hi), which no column sees, count as zeros of V.
    __device__ void drop(int vk, bool fine, int lo, int hi) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool dead = !fine || vk + j >= hi || vk + j < lo;
#pragma unroll
            for (int p = 0; p < D / 32; ++p) {
                const unsigned bits = v_half(p, j) ? 0xFFFF0000u : 0xFFFFu;
                v[v_word(p, j)] = dead ? v[v_word(p, j)] & ~bits : v[v_word(p, j)];
            }
        }
        if (!fine) vs = 0.0f;
    }
    // NaNs of V go from the codes to the channels of the columns that see them; seen: bit j of each tile's, keys vk + j.
    template <int Tiles>
    __device__ void spread(v4f (&acc)[Tiles][D / 16], const unsigned (&seen)[Tiles]) {
        u4 pa[Tiles];
#pragma unroll
        for (int u = 0; u < Tiles; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) pa[u][j] = (seen[u] >> (2 * j) & 1 ? 0x3F80u : 0) | (seen[u] >> (2 * j + 1) & 1 ? 0x3F800000u : 0);
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
            u4 va = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int shift = 16 * v_half(n / 2, j) + 8 * (n & 1);
                unsigned &w = v[v_word(n / 2, j)];
                const bool bad = nan_code(w >> shift);
                va[j >> 1] |= bad ? (j & 1 ? 0x3F800000u : 0x3F80u) : 0u;
                w = bad ? w & ~(255u << shift) : w;
            }
#pragma unroll
            for (int u = 0; u < Tiles; ++u) {
                const v4f count = mfma(va, pa[u], v4f{0, 0, 0, 0});      // how many such keys each column sees, by channel
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[u][n][i] = count[i] > 0 ? __builtin_nanf("") : acc[u][n][i];
            }
        }
    }
};

// Tiles of 16 columns that share each key's operands, their keys dealt to the eight waves 32 at a time; `splits` workgroups
// share a tile's keys.  Each wave keeps its own maximum, sum and O of all columns, in registers, and they meet once at the end.
// Two tiles where a request and kv head have more rows than one holds, as steps with drafted tokens do: unpacking a key's codes costs
// the vector unit more than its products cost the matrix core, and is done once for both.  On inputs that rotate 64 sessions' up to 5
// tokens on up to 4,097 keys, 32 heads on 8 x 128 in bf16, 272 MB, take 72 us (3.8 TB/s, a large copy 5.2), 2 tokens on 200,003 and 100,001
// keys of 2 x 128, 154 MB, 48 us (3.2 TB/s: 336 of 512 resident workgroups have keys).  On one input again and again, which the memory-side
// cache holds in part: 64 and 37; the former 100 with a tile a workgroup.  One token on 733 keys of 8 x 64: 7 us, two splits of at most
// two steps and their join.
constexpr int kLogShift = 14;      // of P in attend8_kernel

template <class T, int D, int Tiles>
__global__ __launch_bounds__(kAttendThreads, D == 256 || Tiles == 2 ? 2 : 4) void attend8_kernel(AttendParams a) {
    constexpr int kChannels = D / 16, kRow = D + 4, kCols = 16 * Tiles;
    using Raw = typename T::Raw;
    __shared__ float s_m[Tiles][kAttendWaves][16], s_l[Tiles][kAttendWaves][16];
    __shared__ float s_o[4][16][kRow];
    __shared__ int s_last;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    int id = blockIdx.x;
    const int hk = id % a.kv_heads;
    id /= a.kv_heads;
    const int turn = id / a.requests, b = (id + turn) % a.requests;       // turned on: see attend_kernel
    const int tile = turn % a.tiles, split = turn / a.tiles;

    const int f0 = a.first ? a.first[b] : b, f1 = a.first ? a.first[b + 1] : b + 1;
    const int q0 = max(f0, 0), q1 = min(f1, a.n_rows), rows = (q1 - q0) * a.group, row0 = tile * kCols;
    if (q1 <= q0 || row0 >= rows) return;
    const int held = max(min(min(a.lens[b], a.max_len), a.width * a.page), 0);
    const int place0 = held - (f1 - q0);                    // of the first token
    auto end_of = [&](int r) { return max(place0 + r / a.group + 1, 0); };
    auto begin_of = [&](int r) { return a.window ? max(place0 + r / a.group + 1 - a.window, 0) : 0; };
    // keys [lo, hi) of this lane's columns; of the whole tile: tokens rise with the column
    const int row_last = min(row0 + kCols, rows) - 1;
    const int hi_min = end_of(row0), hi_max = end_of(row_last), lo_min = begin_of(row0), lo_max = begin_of(row_last), start = lo_min & ~31;
    const int mine = max((hi_max - start + a.chunk - 1) / a.chunk, 1);     // splits with keys in them
    if (split >= mine) return;
    const int k0 = start + split * a.chunk, k1 = min(k0 + a.chunk, hi_max);
    int hi[Tiles], lo[Tiles];
    Queries<D, 1> q[Tiles];
#pragma unroll
    for (int u = 0; u < Tiles; ++u) {
        const int row = min(row0 + 16 * u + c, rows - 1);
        hi[u] = end_of(row), lo[u] = begin_of(row);
        q[u].template load<T>((const Raw *)a.q + (q0 + row / a.group) * a.q_row + (hk * a.group + row % a.group) * a.q_head, a.vec, a.scale < 0);
    }
    // the scale's sign is in the queries; a scale of zero would make 0 * -inf of a key not seen
    const float to_log2 = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);

    const Record8 rec{a.page, D};
    const int64_t head_at = hk * rec.bytes();
    const int *table = a.table + b * a.table_stride;
    const int last_page = max(held - 1, 0) >> a.page_shift;
    auto page_of = [&](int key) {
        const int p = scalar<int>(table + min(key >> a.page_shift, last_page));
        return (unsigned)p < (unsigned)a.n_pages ? p : -1;
    };

    v4f acc[Tiles][kChannels];      // O^T: channel (D/16)(4g + i) + n of column c in acc[.][n][i], in units of 2^(r - kCodeShift)
    float m[Tiles], l[Tiles];       // largest score so far, this lane's share of the sum, times 2^kLogShift
    int r = kNoExponent;
#pragma unroll
    for (int u = 0; u < Tiles; ++u) {
        m[u] = -INFINITY, l[u] = 0;
#pragma unroll
        for (int n = 0; n < kChannels; ++n) acc[u][n] = v4f{0, 0, 0, 0};
    }
    constexpr int kStride = 32 * kAttendWaves;
    int kb = k0 + 32 * wave;
    if (kb < k1) {
        // The next step's K is read into this one's registers as soon as the scores are formed, V after the sums; pages are
        // looked up a step ahead.
        const typename KeyTile8<D>::Offsets at(rec);
        KeyTile8<D> x;
        int id0 = page_of(kb), n0 = page_of(kb + kStride);
        x.load_k(a, rec, at, head_at, kb, id0);
        x.load_v(a, rec, at, head_at, kb, id0);
        for (;;) {
            const int nb = kb + kStride < k1 ? kb + kStride : kb, l0 = nb == kb ? id0 : n0;
            n0 = page_of(nb + kStride);
            v4f s[Tiles][2];
#pragma unroll
            for (int u = 0; u < Tiles; ++u) s[u][0] = s[u][1] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const u4 k8 = codes8<T>(x.k[t][2 * i], x.k[t][2 * i + 1]);
#pragma unroll
                    for (int u = 0; u < Tiles; ++u) s[u][t] = mfma16<T>(k8, q[u].b[0][i], s[u][t]);
                }
            const float ks = x.ks;
            __builtin_amdgcn_sched_barrier(0);
            x.load_k(a, rec, at, head_at, nb, l0);
#pragma unroll
            for (int u = 0; u < Tiles; ++u) s[u][0] *= ks, s[u][1] *= ks;
            if (kb + 32 > hi_min || kb < lo_max || id0 < 0) {
                const int vk = kb + 8 * g;
                unsigned seen[Tiles];
#pragma unroll
                for (int u = 0; u < Tiles; ++u) {
                    const int end = id0 < 0 ? kb : hi[u];
                    seen[u] = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const bool see = (vk + j < end) & (vk + j >= lo[u]);
                        seen[u] |= see ? 1u << j : 0u;
                        s[u][j >> 2][j & 3] = see ? s[u][j >> 2][j & 3] : -INFINITY;
                    }
                }
                x.drop(vk, id0 >= 0, lo_min, hi_max);
                if (x.vs < 0) x.template spread<Tiles>(acc, seen);
            }
            const int e = exponent_of(x.vs);
            if (e > r) {
                const float keep = power_of_two(r - e);
#pragma unroll
                for (int u = 0; u < Tiles; ++u)
#pragma unroll
                    for (int n = 0; n < kChannels; ++n) acc[u][n] *= keep;
                r = e;
            }
            const float scale = code_scale(e, r);
            u4 p[Tiles];
#pragma unroll
            for (int u = 0; u < Tiles; ++u) {
                float top = fmaxf(fmaxf(fmaxf(s[u][0][0], s[u][0][1]), fmaxf(s[u][0][2], s[u][0][3])),
                                  fmaxf(fmaxf(s[u][1][0], s[u][1][1]), fmaxf(s[u][1][2], s[u][1][3])));
                top = column_max(top);
                if (__any(top > m[u])) {
                    const float m2 = fmaxf(m[u], top);
                    const float keep = m[u] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m[u] - m2) * to_log2);
                    m[u] = m2;
                    l[u] *= keep;
#pragma unroll
                    for (int n = 0; n < kChannels; ++n) acc[u][n] *= keep;
                }
                const float shift = m[u] == -INFINITY ? 0.0f : m[u];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // subtracted first: s to_log2 - m to_log2 in one rounding is not 0 at s = m, and large scores overflow by it
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][j >> 1][2 * (j & 1)] - shift, to_log2, (float)kLogShift));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][j >> 1][2 * (j & 1) + 1] - shift, to_log2, (float)kLogShift));
                    p[u][j] = pack_f16(p0, p1);
                    l[u] += p0 + p1;
                }
            }
            unrolled<D / 32>([&](auto pair) {      // two channels at a time
                constexpr int kPair = decltype(pair)::value;
                u4 even, odd;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned au = scaled2(x.v[x.v_word(kPair, 2 * j)], x.v_half(kPair, 2 * j), scale);
                    const unsigned bu = scaled2(x.v[x.v_word(kPair, 2 * j + 1)], x.v_half(kPair, 2 * j + 1), scale);
                    even[j] = __builtin_amdgcn_perm(bu, au, 0x05040100u);
                    odd[j] = __builtin_amdgcn_perm(bu, au, 0x07060302u);
                }
#pragma unroll
                for (int u = 0; u < Tiles; ++u) {
                    acc[u][2 * kPair] = mfma16<F16>(even, p[u], acc[u][2 * kPair]);
                    acc[u][2 * kPair + 1] = mfma16<F16>(odd, p[u], acc[u][2 * kPair + 1]);
                }
            });
            __builtin_amdgcn_sched_barrier(0);
            x.load_v(a, rec, at, head_at, nb, l0);
            if (nb == kb) break;
            kb = nb, id0 = l0;
        }
    }

    // the eight waves' sums into one, tile by tile, each brought to the common maximum and unit first
    const int64_t at = ((int64_t)b * a.kv_heads + hk) * a.tiles + tile;
    float *all = a.part + at * (a.splits + a.groups) * kCols * kRow;      // 32-bit offsets: see attend_shape
    auto finish = [&](int col, int quad, v4f o, float top, float total) {
        const int row = row0 + col, t = row / a.group, h = hk * a.group + row % a.group;
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
    const float unit = power_of_two(r - kCodeShift - kLogShift);
#pragma unroll
    for (int u = 0; u < Tiles; ++u) {
        const float sum = column_sum(l[u]) * power_of_two(-kLogShift);
        if (g == 0) s_m[u][wave][c] = m[u], s_l[u][wave][c] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < Tiles; ++u) {
        const int live = min(rows - row0 - 16 * u, 16);
        float M = s_m[u][0][c];
#pragma unroll
        for (int w = 1; w < kAttendWaves; ++w) M = fmaxf(M, s_m[u][w][c]);
        const float f = (M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m[u] - M) * to_log2)) * unit;
        float *mine_o = &s_o[wave & 3][c][kChannels * 4 * g];
#pragma unroll
        for (int round = 0; round < 2; ++round) {
            if (wave >> 2 == round && c < live)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int n = 0; n < kChannels; n += 4) {
                        v4f y = {acc[u][n][i] * f, acc[u][n + 1][i] * f, acc[u][n + 2][i] * f, acc[u][n + 3][i] * f};
                        v4f *o = (v4f *)(mine_o + kChannels * i + n);
                        if (round) y += *o;
                        *o = y;
                    }
            __syncthreads();
        }
        constexpr int kQuads = D / 4;       // 4 channels a thread from here on
        for (int v = threadIdx.x; v < live * kQuads; v += kAttendThreads) {
            const int col = v / kQuads, quad = v % kQuads;
            v4f o = *(v4f *)&s_o[0][col][4 * quad];
#pragma unroll
            for (int w = 1; w < 4; ++w) o += *(v4f *)&s_o[w][col][4 * quad];
            float top = s_m[u][0][col], total = 0;
#pragma unroll
            for (int w = 1; w < kAttendWaves; ++w) top = fmaxf(top, s_m[u][w][col]);
#pragma unroll
            for (int w = 0; w < kAttendWaves; ++w)      // with no maximum the sums are 0, or NaN
                total += s_l[u][w][col] * (top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((s_m[u][w][col] - top) * to_log2));
            if (mine == 1) {
                finish(16 * u + col, quad, o, top, total);
            } else {
                const unsigned place = (split * kCols + 16 * u + col) * kRow;
                store_shared(all, place + 4 * quad, o);
                if (quad == 0) store_shared(all, place + D, v4f{top, total, 0, 0});
            }
        }
        if (u + 1 < Tiles) __syncthreads();
    }
    if (mine > 1) join<D, kCols>(a, at, split, mine, min(rows - row0, kCols), to_log2, &s_last, finish);
}

// ---- many query rows: prompts ----
//
// A workgroup takes 128 columns, a wave 32 of them, and goes over the keys 64 at a time, K and V as 16-bit values in LDS, two buffers
// deep: see lm_attend.h.  4 prompts of up to 2,047 tokens on up to 4,095 keys, 32 heads on 8 x 128 in bf16, 162 GFLOP: 219 to 234 us a
// call (0.72 PFLOP/s; a large product 1.22); through a window of 1,000, up to 4,001 on 8,191, 16 heads on 4 in f16, 77 GFLOP: 135 to 152.
// Under the profiler, which both take longer with (256 to 274 and 150 to 160): at 64 channels 189 and 117, at 256 657 and 420.
// No unit is full: of 253 us 204 are left without loads and unpacking, 224 with a quarter of the products with V, 215 with
// an eighth of those with K, 239 without exponentials; the matrix cores are busy for a third of the cycles, the vector units for
// 44%.  The rest is waiting: whether one workgroup's products meet the other's exponentials is left to chance.  (Tried: 64 columns a wave, 358, by its registers; 256 columns a workgroup, four waves unpacking K and four V,
// 274 and 204 through the window, whose one workgroup a unit waits as one.)

constexpr float kPromptLogShift = 9.0f;      // of P: maxima lag by up to 2^6

// One thread's share of 64 keys' bytes: of K a quarter of a key's channels, of V half the channels of an entry of 8 keys; the scales
// of both blocks.
template <int D>
struct PromptBytes8 {
    unsigned k[D / 16], v[D / 16];
    float ks[2], vs[2];

    struct Offsets {
        unsigned k, v;
        int block;           // this wave's, of two

        __device__ Offsets(const Record8 &rec) {
            const int t = threadIdx.x, quarter = t & 3, r = (t >> 1) & 15, half = t & 1;
            k = ((t >> 2) & (kBlock - 1)) * D + quarter * (D / 4);
            v = rec.v_codes() + ((t >> 5) & 3) * (8 * D) + r * (D / 2) + half * (D / 4);
            block = __builtin_amdgcn_readfirstlane(t >> 7);
        }
    };
    // What is made of the bytes is made after this point, not before (the compiler would).
    __device__ void pin() {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) asm volatile("" : "+v"(k[i]));
#pragma unroll
        for (int i = 0; i < D / 16; ++i) asm volatile("" : "+v"(v[i]));
    }
    // [lo, hi): what any column sees; the scales of blocks outside it, or without a page, may be anything
    __device__ void load(const AttendParams &a, const Record8 &rec, const Offsets &at, int64_t head_at, int kb, const int (&ids)[2], int lo, int hi) {
        const int own = kb + at.block * kBlock;
        const uint8_t *kp = a.cache + max(at.block ? ids[1] : ids[0], 0) * a.page_stride + head_at + (own & (a.page - 1)) * D;
#pragma unroll
        for (int i = 0; i < D / 64; ++i) *(u4 *)&k[4 * i] = *(const u4 *)(kp + at.k + 16 * i);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) *(u4 *)&v[4 * i] = *(const u4 *)(kp + at.v + 16 * i);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const v2f s = scalar<v2f>(a.cache + max(ids[j], 0) * a.page_stride + head_at + rec.scales() + ((kb + j * kBlock) & (a.page - 1)) / kBlock * 16);
            const bool live = ids[j] >= 0 && kb + j * kBlock < hi && kb + (j + 1) * kBlock > lo;
            ks[j] = live ? fabsf(s[0]) : 1.0f, vs[j] = live ? s[1] : 0.0f;
        }
    }
};

template <class T, int D>
struct alignas(16) PromptTile8 {
    static constexpr int kKRow = D * 2 + 16, kVRow = kPromptKeys * 2 + 16;     // bytes; the pads spread rows over banks
    uint8_t k[kPromptKeys * kKRow], v[D * kVRow];
    uint8_t nan[kPromptKeys / 8][D];        // of a marked tile: 8 keys' NaNs of a row of v

    // the code of this thread's channel i (of D/32) of key j (of 8)
    static constexpr int word_of(int i, int j) { return (j * (D / 32) + i) / 4; }
    static constexpr int shift_of(int i, int j) { return (j * (D / 32) + i) % 4 * 8; }

    // What no column sees becomes zeros.  NaNs of keys that some column sees are taken out of a tile that has them at an edge, where
    // some column does not see some key, and marked; marked becomes kb.
    __device__ void clean(PromptBytes8<D> &x, int block, int kb, bool edge, bool fine, int lo, int hi, int &marked) {
        if (!edge && fine) return;
        const int t = threadIdx.x, a8 = t >> 5, r = (t >> 1) & 15, half = t & 1;
        const bool has = edge && fine && (block ? x.vs[1] : x.vs[0]) < 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int key = kb + 8 * a8 + j;
            const bool dead = !fine || key >= hi || key < lo;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) x.v[word_of(i, j)] = dead ? x.v[word_of(i, j)] & ~(255u << shift_of(i, j)) : x.v[word_of(i, j)];
        }
        // (all marks of a tile that any thread marks are written: a tile has two blocks, one of which may have none)
        if (edge)
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                unsigned bits = 0;
                if (has)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const bool bad = nan_code(x.v[word_of(i, j)] >> shift_of(i, j));
                        bits |= bad ? 1u << j : 0u;
                        x.v[word_of(i, j)] = bad ? x.v[word_of(i, j)] & ~(255u << shift_of(i, j)) : x.v[word_of(i, j)];
                    }
                nan[a8][(half * (D / 32) + i) * 16 + r] = (uint8_t)bits;
                if (bits) marked = kb;
            }
    }
    // V lies transposed, row 16j + r holding channel (D/16) r + j.
    __device__ void stage(const PromptBytes8<D> &x, float scale) {
        const int t = threadIdx.x, key = t >> 2, quarter = t & 3;
        uint8_t *krow = k + key * kKRow + quarter * (D / 2);
#pragma unroll
        for (int w = 0; w < D / 32; ++w) *(u4 *)(krow + 16 * w) = codes8<T>(x.k[2 * w], x.k[2 * w + 1]);
        const int a8 = t >> 5, r = (t >> 1) & 15, half = t & 1;
#pragma unroll
        for (int i = 0; i < D / 32; i += 2) {
            u4 even, odd;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned p = scaled2(x.v[word_of(i, 2 * j)], shift_of(i, 2 * j) != 0, scale);
                const unsigned q = scaled2(x.v[word_of(i, 2 * j + 1)], shift_of(i, 2 * j + 1) != 0, scale);
                even[j] = __builtin_amdgcn_perm(q, p, 0x05040100u);
                odd[j] = __builtin_amdgcn_perm(q, p, 0x07060302u);
            }
            const int n = half * (D / 32) + i;
            *(u4 *)(v + (n * 16 + r) * kVRow + a8 * 16) = even;
            *(u4 *)(v + ((n + 1) * 16 + r) * kVRow + a8 * 16) = odd;
        }
    }
    // Scores of the keys that a column does not see become -inf; what it sees of marked NaNs is put into their channels.  ends: where the
    // column's keys end, of each block.  (Conditions that look at pages key by key are compiled so that scores keep their
    // values where the look alone is false.)
    __device__ void mask(v16f (&s)[2], v16f (&acc)[D / 32], int kb, int h, int lo, const int (&ends)[2], bool marked) const {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int key = kb + 32 * (i >> 4) + 16 * (i >> 3 & 1) + 8 * h + (i & 7);
            s[i >> 4][i & 15] = ((key < ends[i >> 4]) & (key >= lo)) ? s[i >> 4][i & 15] : -INFINITY;
        }
        if (!marked) return;
        unsigned long long seen = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int from = min(max(lo - kb - 32 * j, 0), 32), to = min(max(ends[j] - kb - 32 * j, 0), 32);
            if (from < to) seen |= (unsigned long long)(0xFFFFFFFFu >> (32 - (to - from)) << from) << (32 * j);
        }
#pragma unroll
        for (int n = 0; n < D / 32; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int row = 32 * n + 8 * (i >> 2) + 4 * h + (i & 3);
                unsigned bad = 0;
                for (int g = 0; g < 8; ++g) bad |= nan[g][row] & (unsigned)(seen >> (8 * g)) & 255u;
                acc[n][i] = bad ? __builtin_nanf("") : acc[n][i];
            }
    }
};

template <class T, int D>
__global__ __launch_bounds__(kPromptThreads, D == 256 ? 1 : 2) void attend8_prompt_kernel(AttendParams a) {
    constexpr int kSteps = D / 16, kChannels = D / 32, kCols = kPromptCols;
    using Raw = typename T::Raw;
    using Tile = PromptTile8<T, D>;
    __shared__ Tile s_tile[2];
    __shared__ int s_marked[2];       // the tile of each buffer that has marked NaNs

    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), h = lane >> 5, c = lane & 31;
    // the last tiles of a prompt see the most keys: they go first
    int id = blockIdx.x;
    const int hk = id % a.kv_heads;
    id /= a.kv_heads;
    const int turn = id / a.requests, b = (id + turn) % a.requests;       // turned on: see attend_kernel
    const int tile = a.tiles - 1 - turn;

    const int f0 = a.first ? a.first[b] : b, f1 = a.first ? a.first[b + 1] : b + 1;
    const int q0 = max(f0, 0), q1 = min(f1, a.n_rows), rows = (q1 - q0) * a.group, row0 = tile * kCols;
    if (q1 <= q0 || row0 >= rows) return;
    const int held = max(min(min(a.lens[b], a.max_len), a.width * a.page), 0);
    const int place0 = held - (f1 - q0);
    auto end_of = [&](int r) { return max(place0 + r / a.group + 1, 0); };
    auto begin_of = [&](int r) { return a.window ? max(place0 + r / a.group + 1 - a.window, 0) : 0; };
    const int row_last = min(row0 + kCols, rows) - 1;
    const int hi_min = end_of(row0), hi_max = end_of(row_last), lo_min = begin_of(row0), lo_max = begin_of(row_last);
    const int k0 = lo_min & ~(kPromptKeys - 1), k1 = hi_max;

    // this wave's columns
    const int wrow0 = row0 + wave * 32, wlast = min(wrow0 + 32, rows) - 1, row = min(wrow0 + c, rows - 1);
    const int whi_min = end_of(min(wrow0, rows - 1)), whi_max = end_of(max(wlast, 0)), wlo_min = begin_of(min(wrow0, rows - 1)),
              wlo_max = begin_of(max(wlast, 0));
    const int hi = end_of(row), lo = begin_of(row), tok = row / a.group, head = hk * a.group + row % a.group;
    u4 q[kSteps];
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
            q[ks] = *(u4 *)raw;
        }
    }
    const float to_log2 = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);

    const Record8 rec{a.page, D};
    const int64_t head_at = hk * rec.bytes();
    const int *table = a.table + b * a.table_stride;
    const int last_page = max(held - 1, 0) >> a.page_shift;
    auto page_of = [&](int key) {
        const int p = scalar<int>(table + min(key >> a.page_shift, last_page));
        return (unsigned)p < (unsigned)a.n_pages ? p : -1;
    };
    auto pages_of = [&](int kb, int (&ids)[2]) { ids[0] = page_of(kb), ids[1] = page_of(kb + kBlock); };

    v16f acc[kChannels];
#pragma unroll
    for (int n = 0; n < kChannels; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n][i] = 0;
    float m = -INFINITY, l = 0;
    int r = kNoExponent;      // of the sums; below, r_now and r_next: of what is staged in the two buffers

    auto edge_at = [&](int kb) { return kb + kPromptKeys > hi_min || kb < lo_max; };
    if (k0 < k1) {
        PromptBytes8<D> bytes;
        const typename PromptBytes8<D>::Offsets offsets(rec);
        int ids[2], ids2[2];
        pages_of(k0, ids);
        bytes.load(a, rec, offsets, head_at, k0, ids, lo_min, hi_max);
        if (t < 2) s_marked[t] = -1;
        __syncthreads();
        auto exponent = [&] { return max(exponent_of(bytes.vs[0]), exponent_of(bytes.vs[1])); };
        auto own_scale = [&](int unit) { return code_scale(exponent_of(offsets.block ? bytes.vs[1] : bytes.vs[0]), unit); };
        int r_now = exponent();
        float ks[2] = {bytes.ks[0], bytes.ks[1]};
        bool gone[2] = {ids[0] < 0, ids[1] < 0};
        s_tile[0].clean(bytes, offsets.block, k0, edge_at(k0), !(offsets.block ? gone[1] : gone[0]), lo_min, hi_max, s_marked[0]);
        s_tile[0].stage(bytes, own_scale(r_now));
        pages_of(k0 + kPromptKeys, ids);
        bytes.load(a, rec, offsets, head_at, k0 + kPromptKeys, ids, lo_min, hi_max);
        pages_of(k0 + 2 * kPromptKeys, ids2);
        __syncthreads();
        int buf = 0;
        // While a tile is worked on, the next one is unpacked (between the products of Q and K, which leave the vector
        // unit free) and the one after that is on its way from memory; behind the last one the last page is read again.
        for (int kb = k0; kb < k1; kb += kPromptKeys, buf ^= 1) {
            const int nb = kb + kPromptKeys;
            Tile &next = s_tile[buf ^ 1];
            const Tile &x = s_tile[buf];
            if (D < 256) __builtin_amdgcn_s_setprio(0);
            const bool next_gone[2] = {ids[0] < 0, ids[1] < 0};
            next.clean(bytes, offsets.block, nb, edge_at(nb), !(offsets.block ? next_gone[1] : next_gone[0]), lo_min, hi_max, s_marked[buf ^ 1]);
            int r_next = r_now;
            float next_ks[2];
            const bool active = kb < whi_max && nb > wlo_min;
            v16f s[2];
            {
                // all operands first, so that no product waits for its own; the two halves' products in turn, the next
                // tile's unpacking between them
                const int krow = 16 * (c >> 4) + 8 * ((c >> 2) & 1) + 4 * ((c >> 3) & 1) + (c & 3);
                constexpr int kAhead = kSteps < 8 ? kSteps : 8;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[j][i] = 0;
#pragma unroll
                for (int k8 = 0; k8 < kSteps; k8 += kAhead) {
                    u4 kk[2][kAhead];
#pragma unroll
                    for (int ks8 = 0; ks8 < kAhead; ++ks8)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            kk[j][ks8] = *(const u4 *)(x.k + (32 * j + krow) * Tile::kKRow + 32 * (k8 + ks8) + 16 * h);
                    __builtin_amdgcn_sched_barrier(0);
                    if (k8 + kAhead >= kSteps) bytes.pin();
#pragma unroll
                    for (int ks8 = 0; ks8 < kAhead; ++ks8)
#pragma unroll
                        for (int j = 0; j < 2; ++j) s[j] = mfma32x<T>(kk[j][ks8], q[k8 + ks8], s[j]);
                    if (k8 + kAhead >= kSteps) {
                        r_next = max(r_now, exponent());
                        next_ks[0] = bytes.ks[0], next_ks[1] = bytes.ks[1];
                        next.stage(bytes, own_scale(r_next));
#pragma unroll
                        for (int i = 0; i < 2 * kAhead; ++i) {
                            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(0x202, 4, 0);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            ids[0] = ids2[0], ids[1] = ids2[1];
            bytes.load(a, rec, offsets, head_at, kb + 2 * kPromptKeys, ids, lo_min, hi_max);
            pages_of(kb + 3 * kPromptKeys, ids2);
            if (active) {
                // a tile can be an edge, its NaNs marked, for other waves' columns and whole for this one's
                const bool marked = s_marked[buf] == kb;
                if (kb + kPromptKeys > whi_min || kb < wlo_max || gone[0] || gone[1] || marked) {
                    const int ends[2] = {gone[0] ? kb : hi, gone[1] ? kb : hi};
                    x.mask(s, acc, kb, h, lo, ends, marked);
                }
                if (r_now > r) {
                    const float keep = power_of_two(r - r_now);
#pragma unroll
                    for (int n = 0; n < kChannels; ++n) acc[n] *= keep;
                    r = r_now;
                }
                float top0 = s[0][0], top1 = s[1][0];
#pragma unroll
                for (int i = 1; i < 16; ++i) top0 = fmaxf(top0, s[0][i]), top1 = fmaxf(top1, s[1][i]);
                float top = fmaxf(top0 * ks[0], top1 * ks[1]);
                {
                    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                    top = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
                }
                // sums are brought to a new maximum only where it has outgrown the old one by 2^6
                if (__any((top - m) * to_log2 > 6.0f)) {
                    const float m2 = fmaxf(m, top);
                    const float keep = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - m2) * to_log2);
                    m = m2;
                    l *= keep;
#pragma unroll
                    for (int n = 0; n < kChannels; ++n) acc[n] *= keep;
                }
                const float shift = m == -INFINITY ? 0.0f : m * to_log2;
                if (__any(fabsf(shift) > 0x1p24f)) {
                    // s to_log2 - shift in one rounding is not 0 at s = m: nothing beside what it is beyond such scores
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float y = s[j][i] * ks[j];
                            s[j][i] = (m == -INFINITY ? y : y - m) * to_log2 + kPromptLogShift;
                        }
                } else {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        // a product of zero would make 0 * -inf of a key not seen; scores below 2^102 come to nothing at this one
                        const float by = fmaxf(to_log2 * ks[j], 0x1p-126f);
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[j][i] = __builtin_fmaf(s[j][i], by, kPromptLogShift - shift);
                    }
                }
                // 16 keys at a time: their products with V run beside the next ones' exponentials
                u4 p[4];
                auto exponentials = [&](int g) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float e0 = __builtin_amdgcn_exp2f(s[g >> 1][8 * (g & 1) + 2 * j]);
                        const float e1 = __builtin_amdgcn_exp2f(s[g >> 1][8 * (g & 1) + 2 * j + 1]);
                        l += e0 + e1;
                        p[g][j] = pack_f16(e0, e1);
                    }
                };
                u4 vv[2][kChannels];
                auto operands = [&](int g) {
#pragma unroll
                    for (int n = 0; n < kChannels; ++n) vv[g & 1][n] = *(const u4 *)(x.v + (32 * n + c) * Tile::kVRow + 32 * g + 16 * h);
                };
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
                    for (int n = 0; n < kChannels; ++n) acc[n] = mfma32x<F16>(vv[g & 1][n], p[g], acc[n]);
#pragma unroll
                    for (int i = 0; i < kChannels; ++i) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
                        __builtin_amdgcn_sched_group_barrier(0x400, 8 / kChannels > 0 ? 8 / kChannels : 1, 1);
                        __builtin_amdgcn_sched_group_barrier(0x002, 4, 1);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            r_now = r_next, ks[0] = next_ks[0], ks[1] = next_ks[1], gone[0] = next_gone[0], gone[1] = next_gone[1];
            __syncthreads();
        }
    }
    {
        const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
        l = __uint_as_float(y[0]) + __uint_as_float(y[1]);
    }
    if (wrow0 + c >= rows) return;
    const float unit = power_of_two(r - kCodeShift), inv = l == 0.0f ? 0.0f : 1.0f / l;
    Raw *out = (Raw *)a.out + (int64_t)(q0 + tok) * a.out_row + head * a.out_head;
    // entry e of D/16 channels from acc[n][8 b + ..]: this lane has the entries 4h + i and 8 + 4h + i
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v[D / 16];
#pragma unroll
            for (int n = 0; n < kChannels; ++n) v[2 * n] = acc[n][4 * half + i], v[2 * n + 1] = acc[n][8 + 4 * half + i];
            alignas(8) Raw w[D / 16];
#pragma unroll
            for (int j = 0; j < D / 16; ++j) w[j] = T::put(T::held(v[j] * inv * unit));
            Raw *o = out + (8 * half + 4 * h + i) * (D / 16);
            if (a.vec_out)
#pragma unroll
                for (int j = 0; j < D / 64; ++j) ((u2 *)o)[j] = ((u2 *)w)[j];
            else
#pragma unroll
                for (int j = 0; j < D / 16; ++j) o[j] = w[j];
        }
    if (a.lse && h == 0)
        a.lse[(int64_t)(q0 + tok) * a.heads + head] = l == 0.0f ? -INFINITY : m * to_log2 * kLn2 + (logf(l) - kPromptLogShift * kLn2);
}

}  // namespace pklm
