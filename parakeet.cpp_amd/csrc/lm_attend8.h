// lm_attend8.h -- how attention takes its operands from the 8-bit cache (pk_kv8_attend): codes of 8 bits, a scale for 32 tokens.
//
// A step of 32 keys, and a wave's share of a prompt's 64, lie in one block: on one page, under one scale of K and one
// of V, which is the same in the whole wave.  A code has four significant bits, so that it is exact in bf16 with the scale,
// a power of two, applied in the conversion.
//
// What lies at keys that no column sees may be anything: their V codes become zeros.  A block that holds a NaN has a
// negative scale of V; where some columns see such a key and others do not its NaNs are taken out and put into the
// channels of the columns that see them.
#pragma once

#include "lm_attend.h"
#include "lm_cache8.h"

namespace pklm {

// 4 codes as 4 bf16
__device__ inline u2 unpack4(unsigned w, float scale) {
    return u2{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false)),
              __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))};
}
__device__ inline bool nan_code(unsigned code) { return (code & 0x7Fu) == 0x7Fu; }

template <int D, bool Small>
struct KeyOffsets8 {
    unsigned k, v;

    __device__ KeyOffsets8(const Record8 &rec) {
        const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
        k = (8 * (c >> 2) + (c & 3)) * D + g * (D / 4);
        v = rec.v_codes() + g * (8 * D) + c * (D / 2);
    }
};

// One step's operands of a lane: 32 keys, of K two rows' D/4 channels, of V 8 keys' D/16 channels.
template <int D>
struct KeyTile8 {
    static constexpr int kKWords = D / 16, kVWords = D / 8;
    unsigned k[2][kKWords], v[kVWords];
    float ks, vs;
    using VScales = float;

    __device__ static const uint8_t *record(const AttendParams &a, int64_t head_at, int id) {
        return a.cache + head_at + max(id, 0) * a.page_stride;
    }
    template <bool Small>
    __device__ void load_k(const AttendParams &a, const Record8 &rec, const KeyOffsets8<D, Small> &at, int64_t head_at, int kb, int id, int) {
        const uint8_t *p = record(a, head_at, id);
        const int off = kb & (a.page - 1);
        const uint8_t *kp = p + off * D;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < kKWords / 4; ++i) *(u4 *)&k[t][4 * i] = *(const u4 *)(kp + at.k + 4 * t * D + 16 * i);
        ks = fabsf(*(const float *)(p + rec.scales() + off / kBlock * 16));
    }
    template <bool Small>
    __device__ void load_v(const AttendParams &a, const Record8 &rec, const KeyOffsets8<D, Small> &at, int64_t head_at, int kb, int id, int) {
        const uint8_t *p = record(a, head_at, id);
        const int off = kb & (a.page - 1);
        const uint8_t *vp = p + off * D;
#pragma unroll
        for (int i = 0; i < kVWords / 4; ++i) *(u4 *)&v[4 * i] = *(const u4 *)(vp + at.v + 16 * i);
        vs = *(const float *)(p + rec.scales() + off / kBlock * 16 + 4);
    }
    // channels 8 step .. of key row t as bf16
    __device__ u4 k8(int t, int step) const {
        const u2 lo = unpack4(k[t][2 * step], ks), hi = unpack4(k[t][2 * step + 1], ks);
        return u4{lo[0], lo[1], hi[0], hi[1]};
    }
    __device__ static float v_scale(float vs, int) { return fabsf(vs); }
    // where the pair of channels 2 Pair, 2 Pair + 1 of key j lies: 16 bits of a word
    static constexpr int v_word(int pair, int j) { return (pair / (D / 64) * (D / 4) + j * (D / 32) + pair % (D / 64) * 2) / 4; }
    static constexpr int v_half(int pair, int j) { return (j * (D / 32) + pair % (D / 64) * 2) / 2 & 1; }
    template <int Pair>
    __device__ unsigned v_pair(int j, float scale) const {
        const unsigned w = v[v_word(Pair, j)];
        return v_half(Pair, j) ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))
                               : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
    }

    // Keys vk .. vk + 7 of this lane: [lo, hi) is what its column sees, [lo_all, hi_all) what any column sees.  Scores
    // of keys not seen become -inf.
    template <class Softmax>
    __device__ void mask(Softmax &sm, v4f (&s)[2], float &vs, int vk, bool fine, int lo, int hi, int lo_all, int hi_all) {
        unsigned seen = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int key = vk + j;
            if (fine && key < hi && key >= lo) seen |= 1u << j;
            else s[j >> 2][j & 3] = -INFINITY;
            const bool dead = !fine || key >= hi_all || key < lo_all;
#pragma unroll
            for (int p = 0; p < D / 32; ++p) {
                const unsigned bits = v_half(p, j) ? 0xFFFF0000u : 0xFFFFu;
                v[v_word(p, j)] = dead ? v[v_word(p, j)] & ~bits : v[v_word(p, j)];
            }
        }
        if (!fine) vs = 1.0f;
        if (vs < 0) {
            u4 pa;
#pragma unroll
            for (int j = 0; j < 4; ++j) pa[j] = (seen >> (2 * j) & 1 ? 0x3F80u : 0) | (seen >> (2 * j + 1) & 1 ? 0x3F800000u : 0);
#pragma unroll
            for (int n = 0; n < D / 16; ++n) {
                u4 va = {0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int shift = 16 * v_half(n / 2, j) + 8 * (n & 1);
                    unsigned &w = v[v_word(n / 2, j)];
                    if (nan_code(w >> shift)) {
                        va[j >> 1] |= j & 1 ? 0x3F800000u : 0x3F80u;
                        w &= ~(255u << shift);
                    }
                }
                const v4f count = mfma(va, pa, v4f{0, 0, 0, 0});      // how many such keys each column sees, by channel
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (count[i] > 0) sm.acc[n][i] = __builtin_nanf("");
            }
        }
    }
};

// A wave's keys of 64, of K and of V: one block.
template <int D, bool Small>
struct PromptOffsets8 {
    unsigned k, v;

    __device__ PromptOffsets8(const AttendParams &a, const Record8 &rec) {
        const int t = threadIdx.x, quarter = t & 3, r = (t >> 1) & 15, half = t & 1;
        k = ((t >> 2) & (kBlock - 1)) * D + quarter * (D / 4);
        v = rec.v_codes() + ((t >> 5) & 3) * (8 * D) + r * (D / 2) + half * (D / 4);
    }
    static constexpr bool kTwoPages = false;
    __device__ int k_key() const { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 7) * kBlock; }
    __device__ int v_key() const { return k_key(); }
};

// One thread's share of 64 keys' bytes: of K a quarter of a key's channels, of V half the channels of an entry of 8 keys.
template <int D>
struct PromptBytes8 {
    unsigned k[D / 16], v[D / 16];
    float ks, vs;

    __device__ void pin() {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) asm volatile("" : "+v"(k[i]));
#pragma unroll
        for (int i = 0; i < D / 16; ++i) asm volatile("" : "+v"(v[i]));
    }
    template <bool Small>
    __device__ void load(const AttendParams &a, const PromptOffsets8<D, Small> &at, int64_t head_at, int kb, int id, int) {
        const uint8_t *p = a.cache + max(id, 0) * a.page_stride + head_at;
        const int off = (kb + at.k_key()) & (a.page - 1);
        const uint8_t *kp = p + off * D;
#pragma unroll
        for (int i = 0; i < D / 64; ++i) *(u4 *)&k[4 * i] = *(const u4 *)(kp + at.k + 16 * i);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) *(u4 *)&v[4 * i] = *(const u4 *)(kp + at.v + 16 * i);
        const v2f s = *(const v2f *)(p + Record8{a.page, D}.scales() + off / kBlock * 16);
        ks = fabsf(s[0]), vs = s[1];
    }
};

template <int D>
struct alignas(16) PromptTile8 {
    static constexpr int kKRow = D * 2 + 16, kVRow = kPromptKeys * 2 + 16;     // bytes; the pads spread rows over banks
    uint8_t k[kPromptKeys * kKRow], v[D * kVRow];
    uint8_t nan[kPromptKeys / 8][D];        // of a marked tile: 8 keys' NaNs of a row of v

    // the code of this thread's channel i (of D/32) of key j (of 8)
    static constexpr int word_of(int i, int j) { return (j * (D / 32) + i) / 4; }
    static constexpr int shift_of(int i, int j) { return (j * (D / 32) + i) % 4 * 8; }

    // NaNs of keys that some column sees are taken out of a tile that has them at an edge, where some column does not see some
    // key, and marked; marked becomes kb.
    __device__ void clean(PromptBytes8<D> &x, int kb, bool edge, bool fine, int lo, int hi, int &marked) {
        if (!edge && fine) return;
        const int t = threadIdx.x, a8 = t >> 5, r = (t >> 1) & 15, half = t & 1;
        const bool has = edge && fine && x.vs < 0;
        if (!fine) x.vs = 1.0f;
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
                    for (int j = 0; j < 8; ++j)
                        if (nan_code(x.v[word_of(i, j)] >> shift_of(i, j))) {
                            bits |= 1u << j;
                            x.v[word_of(i, j)] &= ~(255u << shift_of(i, j));
                        }
                nan[a8][(half * (D / 32) + i) * 16 + r] = (uint8_t)bits;
                if (bits) marked = kb;
            }
    }
    __device__ void stage(const PromptBytes8<D> &x) {
        const int t = threadIdx.x, key = t >> 2, quarter = t & 3;
        uint8_t *krow = k + key * kKRow + quarter * (D / 2);
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
            const u2 lo = unpack4(x.k[2 * w], x.ks), hi = unpack4(x.k[2 * w + 1], x.ks);
            *(u4 *)(krow + 16 * w) = u4{lo[0], lo[1], hi[0], hi[1]};
        }
        const int a8 = t >> 5, r = (t >> 1) & 15, half = t & 1;
        const float scale = fabsf(x.vs);
#pragma unroll
        for (int i = 0; i < D / 32; i += 2) {
            u4 even, odd;
            auto pair = [&](int j) {
                const unsigned w = x.v[word_of(i, j)];
                return shift_of(i, j) ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))
                                      : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
            };
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned p = pair(2 * j), q = pair(2 * j + 1);
                even[j] = __builtin_amdgcn_perm(q, p, 0x05040100u);
                odd[j] = __builtin_amdgcn_perm(q, p, 0x07060302u);
            }
            const int n = half * (D / 32) + i;
            *(u4 *)(v + (n * 16 + r) * kVRow + a8 * 16) = even;
            *(u4 *)(v + ((n + 1) * 16 + r) * kVRow + a8 * 16) = odd;
        }
    }
    // Scores of the keys outside [lo, hi) or without a page, which this column does not see, become -inf.  What it sees of marked
    // NaNs is put into their channels.
    template <class Paged>
    __device__ void mask(v16f (&s)[2], v16f (&acc)[D / 32], int kb, int h, int lo, int hi, bool marked, Paged paged) const {
        // A block of keys has a page or has none, so that its keys' bounds say it all.  (A look at the page of each key in the condition
        // is compiled so that scores keep their values where the look alone is false.)
        const int ends[2] = {paged(kb) ? hi : kb, paged(kb + kBlock) ? hi : kb};
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int key = kb + 32 * (i >> 4) + 16 * (i >> 3 & 1) + 8 * h + (i & 7);
            s[i >> 4][i & 15] = ((key < ends[i >> 4]) & (key >= lo)) ? s[i >> 4][i & 15] : -INFINITY;
        }
        if (!marked) return;
        const int from = min(max(lo - kb, 0), 64), to = min(max(hi - kb, 0), 64);
        const unsigned long long seen = from < to ? (~0ull >> (64 - (to - from))) << from : 0;      // keys without a page have no marks
#pragma unroll
        for (int n = 0; n < D / 32; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int row = 32 * n + 8 * (i >> 2) + 4 * h + (i & 3);
                unsigned bad = 0;
                for (int g = 0; g < 8; ++g) bad |= nan[g][row] & (unsigned)(seen >> (8 * g)) & 255u;
                if (bad) acc[n][i] = __builtin_nanf("");
            }
    }
};

struct Kv8 {
    using Rec = Record8;
    // of a vector unit: twice the codes' registers of the 4-bit cache
    template <class T, int D>
    static constexpr int kWaves = D == 256 || __is_same(T, F16) ? 2 : 4;
    template <int D, bool Small>
    using Offsets = KeyOffsets8<D, Small>;
    template <int D>
    using Tile = KeyTile8<D>;
    template <int D, bool Small>
    using PromptOffsets = PromptOffsets8<D, Small>;
    template <int D>
    using PromptBytes = PromptBytes8<D>;
    template <int D>
    using PromptTile = PromptTile8<D>;
};

}  // namespace pklm
