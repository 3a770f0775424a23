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

// Where the codes of a lane's 8 channels (of V those from 8c) of the row at offset `off` of its page lie: in K two runs of 4; in V
// the D/32 channels of 256 / D half entries, which are D/4 bytes, 8 tokens, apart.
template <int D, bool V>
struct Codes8 {
    int lo, hi;

    __device__ Codes8(const Record8 &rec, int off, int c, const LaneChannels<D> &ch)
        : lo(V ? rec.v_codes() + (off >> 3) * (8 * D) + c * 64 + (off & 7) * (D / 32) : off * D + ch.lo), hi(V ? lo + D / 4 : off * D + ch.hi) {}
    __device__ void put(uint8_t *rec, u2 code) const {
        if (V && D == 64) {
#pragma unroll
            for (int i = 0; i < 4; ++i) *(uint16_t *)(rec + lo + i * (D / 4)) = (uint16_t)(code[i >> 1] >> 16 * (i & 1));
        } else if (V && D == 256) {
            *(u2 *)(rec + lo) = code;
        } else {
            *(unsigned *)(rec + lo) = code[0], *(unsigned *)(rec + hi) = code[1];
        }
    }
    __device__ u2 get(const uint8_t *rec) const {
        if (V && D == 64) {
            unsigned w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = *(const uint16_t *)(rec + lo + i * (D / 4));
            return u2{w[0] | w[1] << 16, w[2] | w[3] << 16};
        }
        if (V && D == 256) return *(const u2 *)(rec + lo);
        return u2{*(const unsigned *)(rec + lo), *(const unsigned *)(rec + hi)};
    }
};

// The run's rows that a thread has of a unit, a head of K or of V, as they come from memory.
template <class T, int D, bool Halves>
struct UnitRows {
    static constexpr int kLanes = D / 8, kRows = kTurnThreads / kLanes, kPasses = kBlock / kRows;
    Four<typename T::Raw> lo[kPasses], hi[kPasses];
    unsigned before;                          // the block's scale

    // of V eight adjacent threads take 8 rows, so that they write runs of bytes
    template <bool V>
    __device__ static int c() { return V ? (threadIdx.x >> 3) % kLanes : threadIdx.x % kLanes; }
    template <bool V>
    __device__ static int row(int p) { return p * kRows + (V ? (threadIdx.x & 7) + 8 * (threadIdx.x / (8 * kLanes)) : threadIdx.x / kLanes); }

    template <bool V>
    __device__ void load(const pk_kv8_append_desc &a, int h, int64_t row0, int n, int slot0, int page_shift, bool wide) {
        using Raw = typename T::Raw;
        const int o0 = slot0 & (kBlock - 1), page_off = (slot0 & (a.page - 1)) - o0;
        const Record8 rec{a.page, D};
        const uint8_t *at = (const uint8_t *)a.cache + (int64_t)(slot0 >> page_shift) * a.page_stride + h * rec.bytes();
        before = o0 ? *(const unsigned *)(at + rec.scales() + (page_off / kBlock) * 16 + (V ? 4 : 0)) : 0;
        const int64_t x_row = V ? a.v_row : a.k_row;
        const Raw *x = (V ? (const Raw *)a.v + h * a.v_head : (const Raw *)a.k + h * a.k_head) + row0 * x_row;
        const LaneChannels<D> ch(c<V>(), !V && Halves);
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            const int r = row<V>(p) - o0;
            if (r >= 0 && r < n) {
                if (Halves || wide) {
                    lo[p] = *(const Four<Raw> *)(x + r * x_row + ch.lo), hi[p] = *(const Four<Raw> *)(x + r * x_row + ch.hi);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) lo[p].v[i] = x[r * x_row + ch.lo + i], hi[p].v[i] = x[r * x_row + ch.hi + i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) lo[p].v[i] = hi[p].v[i] = 0;
            }
        }
    }
};

// A barrier for values in LDS alone: rows on their way from memory stay so.
__device__ inline void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// One head's K or V rows, a run, into one block from its offset o0 on, on a workgroup: the largest magnitude, the scale, the
// codes.  Rows before o0 are held already: the block keeps the larger of both scales, and where that has grown they are
// rounded again.  (A power of two more drops at most the last bit of subnormal codes, below 2^-9 of the scale.)  s_top: a
// place for each wave, not the one of the call before; next(): what is to be on its way meanwhile.
template <bool V, class T, int D, class Turn, class Next>
__device__ inline void append_rows(const pk_kv8_append_desc &a, const Turn &turn, const TurnTable<D> &table, const UnitRows<T, D, Turn::halves> &rows, int h,
                                   int n, int slot0, int page_shift, unsigned *s_top, Next next) {
    using Rows = UnitRows<T, D, Turn::halves>;
    constexpr int kRows = Rows::kRows, kPasses = Rows::kPasses;
    const int t = threadIdx.x, o0 = slot0 & (kBlock - 1), page_off = (slot0 & (a.page - 1)) - o0;
    const int c = Rows::template c<V>(), first = Rows::template row<V>(0);
    const Record8 rec{a.page, D};
    uint8_t *at = (uint8_t *)a.cache + (int64_t)(slot0 >> page_shift) * a.page_stride + h * rec.bytes();
    unsigned *scale_at = (unsigned *)(at + rec.scales() + (page_off / kBlock) * 16 + (V ? 4 : 0));
    unsigned before = rows.before;
    const LaneChannels<D> ch(c, !V && Turn::halves);
    float x[kPasses][8];
#pragma unroll
    for (int p = 0; p < kPasses; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[p][i] = T::get(rows.lo[p].v[i]), x[p][4 + i] = T::get(rows.hi[p].v[i]);
    next();
    if (!V && (turn.norm || turn.rot)) {
        float w[8];
        load_weights(a.k_weight, ch, w);
#pragma unroll
        for (int p = 0; p < kPasses; ++p)
            if (p * kRows < o0 + n && (p + 1) * kRows > o0) {
                const int r = p * kRows + first - o0;
                norm_and_turn<D>(x[p], c, turn, table, min(max(r, 0), n - 1), w);
                // rows beside the run are zeros, whose norm with an eps of 0 is NaN: they count for nothing
#pragma unroll
                for (int i = 0; i < 8; ++i) x[p][i] = r >= 0 && r < n ? x[p][i] : 0.0f;
            }
    }
    auto largest = [&](unsigned below) {
        unsigned top = 0;
#pragma unroll
        for (int p = 0; p < kPasses; ++p)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned m = __float_as_uint(x[p][i]) & 0x7FFFFFFFu;
                top = max(top, m < below ? m : 0u);
            }
        return wave_scan(top, 0u, [](unsigned u, unsigned v) { return max(u, v); });      // in lane 63
    };
    const unsigned top_any = largest(0xFFFFFFFFu);
    const bool mine_bad = __any(top_any >= 0x7F800000u);
    unsigned top = mine_bad ? largest(0x7F800000u) : top_any;
    if ((t & 63) == 63) s_top[t >> 6] = top | (mine_bad ? 0x80000000u : 0u);
    // every wave has the scale before it lets the others go on, who write the new one
    asm volatile("" : "+v"(before));
    lds_barrier();
    top = s_top[0];
#pragma unroll
    for (int v = 1; v < kTurnWaves; ++v) top = max(top & 0x7FFFFFFFu, s_top[v] & 0x7FFFFFFFu) | ((top | s_top[v]) & 0x80000000u);
    bool bad = top >> 31;
    top &= 0x7FFFFFFFu;
    if (bad)
#pragma unroll
        for (int p = 0; p < kPasses; ++p)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[p][i] = (__float_as_uint(x[p][i]) & 0x7F800000u) == 0x7F800000u ? __builtin_nanf("") : x[p][i];
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
                if (p * kRows + first < o0) {
                    const Codes8<D, V> place(rec, page_off + p * kRows + first, c, ch);
                    float y[8];
                    decode8(place.get(at), from, y);
                    place.put(at, encode8(y, to));
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
        const int r = p * kRows + first;
        if (r >= o0 && r < o0 + n) Codes8<D, V>(rec, page_off + r, c, ch).put(at, encode8(x[p], scale));
    }
    if (t == 0) {
        *scale_at = (unsigned)s << 23 | (bad ? 0x80000000u : 0u);
        if (V) *(u2 *)(scale_at + 1) = u2{0, 0};
    }
}

// A workgroup has `rows` rows of the call (at most kTurnRows) and takes the runs that begin in them: rows one after the other
// whose slots are one after the other in one block, 32 at most, the last of them perhaps behind its own rows.  It goes over
// the run's heads of K and of V, its waves over those of the queries where they are given.  Rows without a slot are runs of one,
// for their query.  26,617 rows of 32 query heads on 8 x 128 in bf16 with norms, 600 MB, take 186 us (3.2 TB/s; a large copy
// 5.2), 421 with a head of K or V a wave, whose registers leave two waves a vector unit, 204 without the next head's rows on their way:
// memory, the wait for each block's largest magnitude, and queries that a workgroup begins behind all its K and V.  In f32, 1.15 GB,
// 298 us; with half of the channels turned, or partners beside each other, 216 in bf16 and 339 in f32.  (f32 spills 2 to 18 registers at 64 and
// 128 channels, the latter forms in 16 bits up to 6 at 128.)  A step of 64 sessions, 215 rows: 10 us, the chain from slots to angles,
// norm, scale and codes.
template <class T, int D, bool Halves>
__global__ __launch_bounds__(kTurnThreads, D == 256 ? 2 : 4) void append_kernel(pk_kv8_append_desc a, int rows, int page_shift, int wide_q, int wide_kv) {
    using Raw = typename T::Raw;
    __shared__ TurnTable<D> s_table;
    __shared__ unsigned s_top[2][kTurnWaves];
    const Turn<Halves> turn{a.inv_freq, a.pos, a.rot_dim, a.norm, a.interleaved, a.eps};
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
    bool first = true;
    int turns = 0;
    while (begins) {
        const int l = __builtin_ctzll(begins);
        begins &= begins - 1;
        const int slot0 = lane_value(slot, l), n = 1 + __builtin_ctzll(~(going >> (l + 1)));
        const int64_t row0 = (int64_t)blockIdx.x * rows - 1 + l;
        // a unit's rows are on their way while the one before is worked on, the first ones' while the angles are
        UnitRows<T, D, Halves> rows;
        const int units = slot0 >= 0 ? 2 * a.kv_heads : 0;
        auto load = [&](int u) {
            if (u >= units) return;
            if (u < a.kv_heads) rows.template load<false>(a, u, row0, n, slot0, page_shift, wide_kv);
            else rows.template load<true>(a, u - a.kv_heads, row0, n, slot0, page_shift, wide_kv);
        };
        load(blockIdx.y);
        if (a.rot_dim) {
            if (!first) lds_barrier();
            s_table.fill(turn, row0, n);
            lds_barrier();
            first = false;
        }
        for (int u = blockIdx.y; u < units; u += gridDim.y, ++turns) {
            auto next = [&] { load(u + gridDim.y); };
            if (u < a.kv_heads) append_rows<false, T, D>(a, turn, s_table, rows, u, n, slot0, page_shift, s_top[turns & 1], next);
            else append_rows<true, T, D>(a, turn, s_table, rows, u - a.kv_heads, n, slot0, page_shift, s_top[turns & 1], next);
        }
        for (int h = blockIdx.y * kTurnWaves + wave; h < a.heads; h += gridDim.y * kTurnWaves)
            turn_rows<T, D, 4>((const Raw *)a.q + h * a.q_head, a.q_row, wide_q & 1, (Raw *)a.q_out + h * a.q_out_head, a.q_out_row, wide_q & 2,
                            a.q_weight, turn, s_table, row0, n, threadIdx.x & 63);
    }
}

// Rows out of the cache: 8 channels a thread, of V eight adjacent threads the same channels of 8 rows, whose entries lie side by side.
// 26,617 rows of 8 x 128, 163 MB read and written: 39 us, 4.2 TB/s, on inputs that rotate or not.
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
    decode8(Codes8<D, V>(rec, off, c, LaneChannels<D>(c, false)).get(at), __uint_as_float(s), x);
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
