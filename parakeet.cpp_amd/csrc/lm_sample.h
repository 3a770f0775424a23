// lm_sample.h -- one token per row of logits (pk_sample).
#pragma once

#include "lm_common.h"
#include "parakeet_lm.h"

namespace pklm {

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;

// f32 order as unsigned order; both zeros alike
__device__ inline unsigned order_key(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// floor(total * part / 2^31), part <= 2^31
__device__ inline unsigned long long share(unsigned long long total, unsigned long long part) {
    return (total >> 31) * part + (((total & 0x7FFFFFFFull) * part) >> 31);
}

struct RowFilter {
    float top, inv;      // largest logit, 1 / temperature
    __device__ unsigned weight(float x) const {
        if (x == -INFINITY) return 0;
        const float z = x == top ? 0.0f : (x - top) * inv;
        return (unsigned)rintf(expf(z) * 1073741824.0f);
    }
};

template <class T>
__device__ inline float logit(const typename T::Raw *row, int i) {
    const float x = T::get(row[i]);
    return x != x ? -INFINITY : x;
}

// One workgroup a row.  The kept set is a prefix of the order (falling logit, rising index), so it is one cut: a key and
// how many of that key's tokens.  The cut is found digit by digit from histograms of (count, weight).
template <class T>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(pk_sample_desc a) {
    using Raw = typename T::Raw;
    typedef unsigned long long u64;
    __shared__ u64 s_top, s_mass[256], s_wm[kSampleWaves], s_r[4];
    __shared__ unsigned s_cnt[256], s_wc[kSampleWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.vocab, b = blockIdx.x;
    const Raw *row = (const Raw *)a.logits + (int64_t)b * a.logits_row;

    // the largest logit, lowest index
    u64 best = 0;
    for (int i = tid; i < V; i += kSampleThreads) {
        const u64 k = (u64)order_key(logit<T>(row, i)) << 32 | (0xFFFFFFFFu - (unsigned)i);
        best = best > k ? best : k;
    }
    if (tid == 0) s_top = 0;
    __syncthreads();
    for (int d = 32; d; d >>= 1) {
        const u64 o = __shfl_xor(best, d);
        best = best > o ? best : o;
    }
    if (lane == 0) atomicMax(&s_top, best);
    __syncthreads();
    best = s_top;
    const unsigned top_key = (unsigned)(best >> 32);
    const int top_at = (int)(0xFFFFFFFFu - (unsigned)best);
    const float temperature = a.temperature ? a.temperature[b] : 1.0f;
    const bool none = top_key == order_key(-INFINITY);
    if (none || !(temperature > 0)) {
        if (tid == 0) {
            a.token[b] = none ? -1 : top_at;
            if (a.prob) a.prob[b] = none ? 0.0f : 1.0f;
            if (a.kept) a.kept[b] = none ? 0 : 1;
        }
        return;
    }
    const RowFilter f{logit<T>(row, top_at), fminf(1.0f / temperature, 3e38f)};
    const int top_k = a.top_k ? a.top_k[b] : 0;
    const float top_p = a.top_p ? a.top_p[b] : 1.0f, min_p = a.min_p ? a.min_p[b] : 0.0f;
    const u64 P = (u64)(fminf(fmaxf(top_p, 0.0f), 1.0f) * 2147483648.0f);
    const unsigned least = (unsigned)ceilf(fminf(fmaxf(min_p, 0.0f), 1.0f) * 1073741824.0f);

    // sums over all, then the cut by count, then the cut by weight
    u64 cut_mass = 0;            // weight of the kept prefix so far
    unsigned cut_key = 0, cut_ties = 0xFFFFFFFFu;   // kept: key > cut_key, or the first cut_ties of cut_key
    auto block_sum = [&](u64 m, unsigned n) {
        for (int d = 32; d; d >>= 1) m += __shfl_xor(m, d), n += __shfl_xor(n, d);
        __syncthreads();
        if (lane == 0) s_wm[wave] = m, s_wc[wave] = n;
        __syncthreads();
        if (tid == 0) {
            u64 M = 0;
            unsigned N = 0;
            for (int w = 0; w < kSampleWaves; ++w) M += s_wm[w], N += s_wc[w];
            s_r[0] = M, s_r[1] = N;
        }
        __syncthreads();
    };
    {
        u64 m = 0;
        for (int i = tid; i < V; i += kSampleThreads) m += f.weight(logit<T>(row, i));
        block_sum(m, 0);
        cut_mass = s_r[0];
    }
    // the key in which a running count (by_count) or weight first reaches `want` (>= 1, and reached)
    auto find = [&](bool by_count, u64 want, unsigned &key, unsigned &ties, u64 &before) {
        unsigned prefix = 0;
        u64 above_c = 0, above_m = 0;
        unsigned here = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) s_cnt[tid] = 0, s_mass[tid] = 0;
            __syncthreads();
            for (int i = tid; i < V; i += kSampleThreads) {
                const float x = logit<T>(row, i);
                const unsigned k = order_key(x);
                if (shift == 24 || (k >> (shift + 8)) == prefix) {
                    atomicAdd(&s_cnt[k >> shift & 255u], 1u);
                    atomicAdd(&s_mass[k >> shift & 255u], (u64)f.weight(x));
                }
            }
            __syncthreads();
            if (tid == 0) {
                int d = 255;
                u64 c = above_c, m = above_m;
                for (; d > 0; --d) {
                    if ((by_count ? c + s_cnt[d] : m + s_mass[d]) >= want) break;
                    c += s_cnt[d], m += s_mass[d];
                }
                s_r[0] = (u64)d, s_r[1] = c, s_r[2] = m, s_r[3] = s_cnt[d];
            }
            __syncthreads();
            prefix = prefix << 8 | (unsigned)s_r[0];
            above_c = s_r[1], above_m = s_r[2], here = (unsigned)s_r[3];
        }
        key = prefix, ties = here;
        before = by_count ? above_c : above_m;
        if (by_count) s_wm[0] = above_m;     // read back below, before the next use
    };
    auto weight_of_key = [&](unsigned k) {
        return f.weight(__uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k));
    };
    if (top_k > 0 && top_k < V) {
        u64 before;
        find(true, (u64)top_k, cut_key, cut_ties, before);
        __syncthreads();
        cut_ties = (unsigned)(top_k - before);
        cut_mass = s_wm[0] + (u64)cut_ties * weight_of_key(cut_key);
    }
    const u64 need = share(cut_mass, P);
    if (need == 0) {
        cut_key = top_key, cut_ties = 1;
    } else {
        unsigned key, ties;
        u64 before;
        find(false, need, key, ties, before);
        const u64 w = weight_of_key(key);
        const unsigned t = (unsigned)((need - before + w - 1) / w);
        if (key > cut_key || (key == cut_key && t < cut_ties)) cut_key = key, cut_ties = t;
    }
    // waves own runs of the row: which tie is the last, sums, then the token
    const int seg = (V + kSampleWaves * 64 - 1) / (kSampleWaves * 64) * 64, w0 = min(wave * seg, V), w1 = min(w0 + seg, V);
    unsigned n = 0;
    for (int i = w0 + lane; i < w1; i += 64) n += order_key(logit<T>(row, i)) == cut_key;
    for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
    __syncthreads();
    if (lane == 0) s_wc[wave] = n;
    __syncthreads();
    unsigned ties_before = 0;
    for (int w = 0; w < wave; ++w) ties_before += s_wc[w];
    u64 mass = 0;
    unsigned kept = 0, seen = ties_before;
    auto weigh = [&](int i, unsigned &run) -> unsigned {    // the kept weight of lane's token, ~0u where not kept
        const float x = i < w1 ? logit<T>(row, i) : -INFINITY;
        const unsigned k = i < w1 ? order_key(x) : 0;
        const u64 tie = __ballot(i < w1 && k == cut_key);
        const unsigned rank = run + __popcll(tie & ((1ull << lane) - 1));
        run += __popcll(tie);
        const bool in = i < w1 && (k > cut_key || (k == cut_key && rank < cut_ties));
        const unsigned w = in ? f.weight(x) : 0;
        return in && (w >= least || i == top_at) ? w : ~0u;
    };
    for (int i0 = w0; i0 < w1; i0 += 64) {
        const unsigned w = weigh(i0 + lane, seen);
        if (w != ~0u) mass += w, ++kept;
    }
    for (int d = 32; d; d >>= 1) mass += __shfl_xor(mass, d), kept += __shfl_xor(kept, d);
    __syncthreads();
    if (lane == 0) s_wm[wave] = mass, s_wc[wave] = kept;
    __syncthreads();
    u64 total = 0, lead = 0;
    unsigned all = 0;
    for (int w = 0; w < kSampleWaves; ++w) {
        if (w < wave) lead += s_wm[w];
        total += s_wm[w], all += s_wc[w];
    }
    u64 U = (u64)(fminf(fmaxf(a.u[b], 0.0f), 1.0f) * 2147483648.0f);
    if (U > 0x7FFFFFFFull) U = 0x7FFFFFFFull;
    const u64 t = share(total, U);
    if (lead > t || lead + s_wm[wave] <= t) return;         // another wave's run has the token
    seen = ties_before;
    for (int i0 = w0; i0 < w1; i0 += 64) {
        const unsigned w = weigh(i0 + lane, seen);
        const u64 run = wave_scan((u64)(w == ~0u ? 0 : w));
        const u64 hit = __ballot(lead + run > t);
        if (hit) {
            const int at = __ffsll(hit) - 1;
            if (lane == at) {
                a.token[b] = i0 + lane;
                if (a.prob) a.prob[b] = (float)w / (float)total;
                if (a.kept) a.kept[b] = (int)all;
            }
            return;
        }
        lead += __shfl(run, 63);
    }
}

}  // namespace pklm
