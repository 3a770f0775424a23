// lm_rope.h -- norms of queries and keys for each head and the position rotation (pk_qk_rope, and on the way into the
// 8-bit cache pk_kv8_append).
//
// A row of D channels of one head is D/8 lanes' 8 channels, so that a wave holds 512 / D rows and the norm's sum stays within a
// row's lanes.  Where all channels are turned, in halves, a lane has 4 channels of the lower half and their partners in the upper one;
// with partners beside each other, 8 adjacent channels; so no value crosses lanes.  (Partners through shuffles: 16,385 rows of
// 32 + 8 heads x 128 took 88 us.)  Only a part's rotation in halves needs shuffles.  The angles of a token are the same for all its heads: a workgroup works out the sines
// and cosines of its rows once, into LDS, and its waves go over the heads.  An angle is pos * inv_freq in f64, in turns
// less the whole ones: in f32 a position of 200,000 has lost 2^-7 of a radian.
#pragma once

#include "lm_cache.h"
#include "lm_common.h"
#include "parakeet_lm.h"

namespace pklm {

constexpr int kTurnThreads = 256, kTurnWaves = kTurnThreads / 64, kTurnRows = 32;

// Sum over the D/8 lanes of a row.
template <int Lanes>
__device__ inline float row_sum(float v) {
    v += from_lane<0xB1, 0xF>(v, 0.0f);                 // lane ^ 1
    v += from_lane<0x4E, 0xF>(v, 0.0f);                 // lane ^ 2
    v += from_lane<0x141, 0xF>(v, 0.0f);                // the other four of eight
    if (Lanes > 8) v += from_lane<0x140, 0xF>(v, 0.0f); // the other eight of sixteen
    if (Lanes > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

// How rows are normed and turned.  Halves: all channels are, in halves, and rows are aligned to four channels; a lane's 8 are
// 4 of each half.
template <bool Halves>
struct Turn {
    static constexpr bool halves = Halves;
    const float *inv_freq;
    const int *pos;              // nullable where nothing is turned
    int rot, norm, interleaved;
    float eps;

    __device__ bool live(int64_t row) const { return !pos || pos[row] >= 0; }
};

// A lane's 8 channels of a row: 4 from lo, 4 from hi.
template <int D>
struct LaneChannels {
    int lo, hi;
    __device__ LaneChannels(int c, bool halves) : lo(halves ? 4 * c : 8 * c), hi(halves ? D / 2 + 4 * c : 8 * c + 4) {}
};
template <class Raw>
struct alignas(4 * sizeof(Raw)) Four {
    Raw v[4];
};
template <class T, int D>
__device__ inline void load_channels(const typename T::Raw *row, const LaneChannels<D> &at, bool wide, float (&x)[8]) {
    using Raw = typename T::Raw;
    Four<Raw> lo, hi;
    if (wide) {
        lo = *(const Four<Raw> *)(row + at.lo), hi = *(const Four<Raw> *)(row + at.hi);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) lo.v[i] = row[at.lo + i], hi.v[i] = row[at.hi + i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = T::get(lo.v[i]), x[4 + i] = T::get(hi.v[i]);
}
template <class T, int D>
__device__ inline void store_channels(typename T::Raw *row, const LaneChannels<D> &at, bool wide, const float (&x)[8]) {
    using Raw = typename T::Raw;
    Four<Raw> lo, hi;
#pragma unroll
    for (int i = 0; i < 4; ++i) lo.v[i] = T::put(x[i]), hi.v[i] = T::put(x[4 + i]);
    if (wide) {
        *(Four<Raw> *)(row + at.lo) = lo, *(Four<Raw> *)(row + at.hi) = hi;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) row[at.lo + i] = lo.v[i], row[at.hi + i] = hi.v[i];
    }
}

template <int D>
struct TurnTable {
    float c[kTurnRows * D / 2], s[kTurnRows * D / 2];

    // the angles of the n rows from row0; a barrier on either side
    template <class Turn>
    __device__ void fill(const Turn &turn, int64_t row0, int n) {
        const int half = turn.rot / 2;
        for (int i = threadIdx.x; i < n * half; i += kTurnThreads) {
            const int r = i / half, j = i - r * half;
            double t = (double)turn.pos[row0 + r] * (double)turn.inv_freq[j] * 0.15915494309189533577;
            t -= rint(t);
            sincospif(2.0f * (float)t, &s[r * half + j], &c[r * half + j]);
        }
    }
};

// A lane's 8 channels of a row, the lane_c'th of its lanes: normed with the weights w, turned by the angles of the table's row r.
template <int D, class Turn>
__device__ inline void norm_and_turn(float (&x)[8], int lane_c, const Turn &turn, const TurnTable<D> &table, int r, const float (&w)[8]) {
    if (turn.norm) {
        float sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(x[i], x[i], sum);
        const float inv = 1.0f / sqrtf(row_sum<D / 8>(sum) * (1.0f / D) + turn.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= inv * w[i];
    }
    if (!Turn::halves && turn.rot == 0) return;
    const int half = Turn::halves ? D / 2 : turn.rot / 2;
    if (Turn::halves) {
        const v4f c = *(const v4f *)&table.c[r * half + 4 * lane_c], s = *(const v4f *)&table.s[r * half + 4 * lane_c];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = x[i], b = x[4 + i];
            x[i] = a * c[i] - b * s[i], x[4 + i] = a * s[i] + b * c[i];
        }
    } else if (turn.interleaved) {
        if (8 * lane_c < turn.rot) {
            const v4f c = *(const v4f *)&table.c[r * half + 4 * lane_c], s = *(const v4f *)&table.s[r * half + 4 * lane_c];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = x[2 * i], b = x[2 * i + 1];
                x[2 * i] = a * c[i] - b * s[i], x[2 * i + 1] = a * s[i] + b * c[i];
            }
        }
    } else {
        // the other channel of a pair is half channels, whole lanes, away
        const int lanes = half / 8, lane = threadIdx.x & 63;
        const bool low = lane_c < lanes, in = lane_c < 2 * lanes;
        const int from = in ? (low ? lane + lanes : lane - lanes) : lane;
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __shfl(x[i], from);
        if (in) {
            const int at = r * half + 8 * (low ? lane_c : lane_c - lanes);
#pragma unroll
            for (int i4 = 0; i4 < 8; i4 += 4) {
                const v4f c = *(const v4f *)&table.c[at + i4], s = *(const v4f *)&table.s[at + i4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i4 + i] = x[i4 + i] * c[i] + (low ? -y[i4 + i] : y[i4 + i]) * s[i];
            }
        }
    }
}

template <int D>
__device__ inline void load_weights(const float *weight, const LaneChannels<D> &at, float (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = weight ? weight[i < 4 ? at.lo + i : at.hi + i - 4] : 1.0f;
}

// One head's rows row0 .. row0 + n, n <= kTurnRows, from x into y, on one wave: Batch passes' loads together.  (One pass at
// a time leaves too little on its way: 16,385 rows of 32 + 8 heads x 128, 8-byte partners through shuffles, took 104 us, 4 at a time 88.)
template <class T, int D, int Batch, class Turn>
__device__ inline void turn_some(const typename T::Raw *x, int64_t x_row, bool wide, typename T::Raw *y, int64_t y_row, bool y_wide,
                                 const float (&w)[8], const Turn &turn, const TurnTable<D> &table, int64_t row0, int n, int lane) {
    constexpr int kLanes = D / 8, kRows = 64 / kLanes;
    const int c = lane % kLanes;
    const LaneChannels<D> at(c, Turn::halves);
    for (int r0 = 0; r0 < n; r0 += kRows * Batch) {
        float v[Batch][8];
        bool live[Batch];
#pragma unroll
        for (int p = 0; p < Batch; ++p) {
            const int r = r0 + p * kRows + lane / kLanes;
            const int64_t row = row0 + min(r, n - 1);
            load_channels<T, D>(x + row * x_row, at, Turn::halves || wide, v[p]);
            live[p] = r < n && turn.live(row);
        }
#pragma unroll
        for (int p = 0; p < Batch; ++p) {
            const int r = r0 + p * kRows + lane / kLanes;
            if (Batch > 1 && r0 + p * kRows >= n) break;
            norm_and_turn<D>(v[p], c, turn, table, min(r, n - 1), w);
            if (live[p]) store_channels<T, D>(y + (row0 + r) * y_row, at, Turn::halves || y_wide, v[p]);
        }
    }
}
template <class T, int D, int Batch, class Turn>
__device__ inline void turn_rows(const typename T::Raw *x, int64_t x_row, bool wide, typename T::Raw *y, int64_t y_row, bool y_wide,
                                 const float *weight, const Turn &turn, const TurnTable<D> &table, int64_t row0, int n, int lane) {
    float w[8];
    load_weights(weight, LaneChannels<D>(lane % (D / 8), Turn::halves), w);
    if (n <= 512 / D) turn_some<T, D, 1>(x, x_row, wide, y, y_row, y_wide, w, turn, table, row0, n, lane);
    else turn_some<T, D, Batch>(x, x_row, wide, y, y_row, y_wide, w, turn, table, row0, n, lane);
}

// Memory bounds it: 16,385 rows (2,048 of them left out) of 32 + 8 heads x 128 in bf16 with norms, 294 MB, take 74 us on inputs that
// rotate, 4.0 TB/s, where a large copy reaches 5.2; 62 on one input again and again, which the memory-side cache holds in part, as
// in the next figures.  4 passes' loads a wave of 16-bit types (2: 65; at 64 channels, where 4 are all rows, 28.5 and 29.6; f32
// has no registers for them), 8 waves a vector unit.  In f32 134 us (588 MB, 4.4 TB/s).  With half of the channels turned, or partners beside
// each other, 103 in bf16 and 168 in f32: four waves a vector unit.  One row of 16 heads takes 3 us, a launch and the sines.
template <class T, int D, bool Halves>
__global__ __launch_bounds__(kTurnThreads, !Halves || D == 256 ? 4 : 8) void rope_kernel(pk_qk_rope_desc a, int rows, int wide_q, int wide_k) {
    using Raw = typename T::Raw;
    __shared__ TurnTable<D> s_table;
    const Turn<Halves> turn{a.inv_freq, a.pos, a.rot_dim, a.norm, a.interleaved, a.eps};
    const int64_t row0 = (int64_t)blockIdx.x * rows;
    const int n = (int)min((int64_t)rows, a.n_rows - row0), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (a.rot_dim) {
        // a padded call's last workgroups, all of whose rows are left out, read none
        const bool live = turn.live(row0 + min((int)(threadIdx.x & 63), n - 1));
        s_table.fill(turn, row0, n);
        if (!__any(live)) return;
        __syncthreads();
    }
    constexpr int kBatch = sizeof(Raw) == 2 && D > 64 ? 4 : 2;
    for (int u = blockIdx.y * kTurnWaves + wave; u < a.heads + a.kv_heads; u += gridDim.y * kTurnWaves) {
        // what follows from the lane is worked out behind this, not in front of the angles and the loop, over which it would be spilled:
        // with 2 passes 48 registers instead of 62 and 10 spilled, 215 rows 4.2 us, not 5.7
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        if (u < a.heads)
            turn_rows<T, D, kBatch>((const Raw *)a.q + u * a.q_head, a.q_row, wide_q & 1, (Raw *)a.q_out + u * a.q_out_head, a.q_out_row, wide_q & 2,
                            a.q_weight, turn, s_table, row0, n, lane);
        else
            turn_rows<T, D, kBatch>((const Raw *)a.k + (u - a.heads) * a.k_head, a.k_row, wide_k & 1, (Raw *)a.k_out + (u - a.heads) * a.k_out_head,
                            a.k_out_row, wide_k & 2, a.k_weight, turn, s_table, row0, n, lane);
    }
}

}  // namespace pklm
