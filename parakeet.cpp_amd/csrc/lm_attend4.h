// lm_attend4.h -- how attention takes its operands from the 4-bit cache (pk_kv4_attend): codes of 4 bits, a scale byte for 32
// channels of a token.
#pragma once

#include "lm_attend.h"

namespace pklm {

// 8 codes as 8 bf16
__device__ inline u4 unpack8(unsigned w, float scale) {
    u4 r;
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
    return r;
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
    using VScales = u2;

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
    // channels 8 ks .. of key row t as bf16
    __device__ u4 k8(int t, int step) const {
        const unsigned sb = D == 256 ? ks[t] >> (8 * (step / 4)) & 255u : ks[t];
        return unpack8(k[t][step], __uint_as_float(sb << 23));
    }
    __device__ static float v_scale(u2 vs, int j) { return __uint_as_float((vs[j >> 2] >> (8 * (j & 3)) & 255u) << 23); }
    // channels 2 Pair and 2 Pair + 1 of key j as bf16
    template <int Pair>
    __device__ unsigned v_pair(int j, float scale) const {
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v_word(j, Pair / 4), scale, Pair % 4));
    }

    // Keys vk .. vk + 7 of this lane: [lo, hi) is what its column sees, [lo_all, hi_all) what any column sees.  Scores
    // of keys not seen become -inf.  What lies at keys that no column sees may be anything: their V scale becomes 1.  A
    // NaN block of V that only some columns see is taken out, and those columns are made NaN.
    template <class Softmax>
    __device__ void mask(Softmax &sm, v4f (&s)[2], u2 &vs, int vk, bool fine, int lo, int hi, int lo_all, int hi_all) const {
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
                    for (int t = 0; t < D / 16; ++t) sm.acc[t][i] = __builtin_nanf("");
        }
    }
};

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

    // which keys of 64 this thread's bytes of K and of V are, where that tells their pages
    static constexpr bool kTwoPages = Small;
    __device__ int k_key() const { return Small ? threadIdx.x >> 2 : 0; }
    __device__ int v_key() const { return (threadIdx.x >> 5) * 8; }
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

    // Scores of the keys outside [lo, hi) or without a page, which this column does not see, become -inf.  What it sees of marked
    // blocks makes their channels NaN.
    template <class Paged>
    __device__ void mask(v16f (&s)[2], v16f (&acc)[D / 32], int kb, int h, int lo, int hi, bool marked, Paged paged) const {
        unsigned bad = 0;             // channel blocks whose NaN this column sees
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int at = 32 * (i >> 4) + 16 * (i >> 3 & 1) + 8 * h + (i & 7), key = kb + at;
            const bool see = key < hi && key >= lo && paged(key);
            if (!see) s[i >> 4][i & 15] = -INFINITY;
            else if (marked)
#pragma unroll
                for (int j = 0; j < D / 32; ++j) bad |= (unsigned)nan[at][j] << j;
        }
        bad |= (unsigned)__shfl_xor((int)bad, 32);
        if (__any(bad != 0))
#pragma unroll
            for (int n = 0; n < D / 32; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = (8 * (i >> 2) + 4 * h + (i & 3)) & 15;
                    if (bad >> (r * (D / 16) / 32) & 1) acc[n][i] = __builtin_nanf("");
                }
    }
};

struct Kv4 {
    using Rec = Record;
    template <class T, int D>
    static constexpr int kWaves = D == 256 ? 2 : 4;      // of a vector unit
    template <int D, bool Small>
    using Offsets = KeyOffsets<D, Small>;
    template <int D>
    using Tile = KeyTile<D>;
    template <int D, bool Small>
    using PromptOffsets = pklm::PromptOffsets<D, Small>;
    template <int D>
    using PromptBytes = pklm::PromptBytes<D>;
    template <int D>
    using PromptTile = pklm::PromptTile<D>;
};

}  // namespace pklm
