// lm_verify.h -- drafted tokens against the target's probabilities (pk_verify).
//
// Weights are pk_sample's whole numbers, w = round(2^30 exp((x - max) / T)), so that their sums are exact in any order.  What is
// compared and drawn from follows from them in single f64 steps, p = w (1 / sum w): the same wherever it is worked out.  A
// refused draft's successor is drawn from max(p - q, 0) in steps of 2^-52, whole numbers again, whose sum is at most 2^52 and a
// half step for each token.
#pragma once

#include "lm_common.h"
#include "lm_sample.h"
#include "parakeet_lm.h"

namespace pklm {

constexpr int kNever = 0x7FFFFFFF;

// One row's weights: the logits' largest, 1 / T, and where the largest alone counts its place.
struct RowWeights {
    RowRule rule;
    bool greedy;
    int top_at;
    double inv_sum;

    __device__ void settings(const float *temperature, int b) {
        const float t = temperature ? temperature[b] : 1.0f;
        greedy = !(t > 0);
        rule.inv = greedy ? 1.0f : fminf(1.0f / t, 3e38f);
    }
    __device__ unsigned weight(float x, int i) const {
        if (greedy) return i == top_at && x != -INFINITY ? 1u << 30 : 0u;
        return rule.weight(x);
    }
    __device__ void total(u64 sum) { inv_sum = sum ? 1.0 / (double)sum : 0.0; }
    __device__ double share_of(unsigned w) const { return __dmul_rn((double)w, inv_sum); }
};

__device__ inline double uniform(float u) {
    const u64 v = part31(u);
    return (double)(v > 0x7FFFFFFFull ? 0x7FFFFFFFull : v) * 0x1p-31;
}
__device__ inline u64 left_of(double p, double q) { return p > q ? (u64)(__dadd_rn(p, -q) * 0x1p52) : 0; }

// Rows of a request: [begin, begin + n) of the call's.
struct RequestRows {
    int begin, n;
    __device__ RequestRows(const pk_verify_desc &a, int b) {
        const int f0 = max(a.first[b], 0), f1 = min(a.first[b + 1], a.n_rows);
        begin = f0, n = min(max(f1 - f0, 0), a.max_new);
    }
    // the draft of its row j, -1: none
    __device__ int draft(const pk_verify_desc &a, int j) const {
        const int d = j + 1 < n ? a.tokens[begin + j + 1] : -1;
        return d >= 0 && d < a.vocab ? d : -1;
    }
};

__device__ inline void verify_counts(const pk_verify_desc &a, int b, int n, int accepted) {
    a.accepted[b] = accepted;
    if (a.lens_out) a.lens_out[b] = a.lens[b] - max(n - 1 - accepted, 0);
}

// What a row came to: a draft that was accepted, or the token drawn in its place.
struct alignas(16) RowVerdict {
    int ok, token;
    float prob;
    int unused;
};

// A request's rows on a workgroup each, tokens in registers as sample_row_kernel has them.  Every row that refuses its
// draft draws its own token, whether or not an earlier row has refused; the request's last workgroup to arrive has the rows'
// verdicts and writes them up to the first refusal.
template <class T, int BS, int E, bool Draft>
__global__ __launch_bounds__(BS) void verify_row_kernel(pk_verify_desc a, int *arrived, RowVerdict *verdicts) {
    constexpr int kWaves = BS / 64;
    __shared__ float s_max[2][kWaves];
    __shared__ int s_at[2][kWaves];
    __shared__ u64 s_sum[2][kWaves];
    __shared__ RowVerdict s_verdict;
    __shared__ int s_flag;
    using Raw = typename T::Raw;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), V = a.vocab;
    const int b = blockIdx.x / a.max_new, j = blockIdx.x % a.max_new;
    const RequestRows rows(a, b);
    if (rows.n == 0 && j == 0 && tid == 0) verify_counts(a, b, 0, 0);
    if (j >= rows.n) return;
    const int r = rows.begin + j, d = rows.draft(a, j);
    constexpr int kSources = Draft ? 2 : 1;
    const bool drafted = d >= 0;
    const int n = (V + BS - 1) / BS, base = wave * n * 64 + lane, end = min((wave + 1) * n * 64, V);
    const Raw *row[2] = {(const Raw *)a.logits + (int64_t)r * a.logits_row, Draft ? (const Raw *)a.draft + (int64_t)r * a.draft_row : nullptr};
    float x[kSources][E], at_draft[2];
    RowWeights rw[2];
    rw[0].settings(a.temperature, b);
    if (Draft) rw[1].settings(a.draft_temperature, b);
#pragma unroll
    for (int q = 0; q < kSources; ++q) {
        const bool on = q == 0 || drafted;      // without a draft its row is not read
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = base + e * 64;
            x[q][e] = on && i < end ? logit<T>(row[q], i) : -INFINITY;
        }
        at_draft[q] = drafted ? logit<T>(row[q], d) : -INFINITY;
    }
    // the largest, and its first place
#pragma unroll
    for (int q = 0; q < kSources; ++q) {
        float top = x[q][0];
#pragma unroll
        for (int e = 1; e < E; ++e) top = fmaxf(top, x[q][e]);
        top = wave_max(top);
        if (lane == 0) s_max[q][wave] = top;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kSources; ++q) {
        float top = s_max[q][0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, s_max[q][w]);
        rw[q].rule.top = top;
        int at = kNever;
        if (rw[q].greedy)
#pragma unroll
            for (int e = 0; e < E; ++e) at = min(at, x[q][e] == top ? base + e * 64 : kNever);
        at = lane_value(wave_scan(at, kNever, [](int u, int v) { return min(u, v); }), 63);
        if (lane == 0) s_at[q][wave] = at;
    }
    __syncthreads();
    unsigned w[kSources][E];
#pragma unroll
    for (int q = 0; q < kSources; ++q) {
        int at = s_at[q][0];
#pragma unroll
        for (int v = 1; v < kWaves; ++v) at = min(at, s_at[q][v]);
        rw[q].top_at = at;
        u64 sum = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            w[q][e] = rw[q].weight(x[q][e], base + e * 64);
            sum += w[q][e];
        }
        sum = wave_sum(sum);
        if (lane == 0) s_sum[q][wave] = sum;
    }
    __syncthreads();
    u64 total[2] = {0, 0};
#pragma unroll
    for (int q = 0; q < kSources; ++q) {
#pragma unroll
        for (int v = 0; v < kWaves; ++v) total[q] += s_sum[q][v];
        rw[q].total(total[q]);
    }
    const double p_draft = drafted ? rw[0].share_of(rw[0].weight(at_draft[0], d)) : 0.0;
    const double q_draft = Draft ? rw[1].share_of(rw[1].weight(at_draft[1], d)) : 1.0;
    const bool ok = drafted && __dmul_rn(uniform(a.u[r]), q_draft) < p_draft;
    if (ok || total[0] == 0) {
        if (tid == 0) s_verdict = RowVerdict{ok, ok ? d : -1, ok ? (float)p_draft : 0.0f, 0};
    } else {
        // what is left to draw from
        u64 left[E], mass = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            left[e] = w[0][e];
            if (drafted) left[e] = Draft ? left_of(rw[0].share_of(w[0][e]), rw[1].share_of(w[kSources - 1][e])) : base + e * 64 == d ? 0 : left[e];
            mass += left[e];
        }
        mass = wave_sum(mass);
        __syncthreads();                         // s_sum may still be read
        if (lane == 0) s_sum[1][wave] = mass;
        __syncthreads();
        u64 all = 0, lead = 0;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) {
            if (v < wave) lead += s_sum[1][v];
            all += s_sum[1][v];
        }
        if (all == 0) {                          // nothing: from the target itself
#pragma unroll
            for (int e = 0; e < E; ++e) left[e] = w[0][e];
            mass = s_sum[0][wave], all = total[0], lead = 0;
#pragma unroll
            for (int v = 0; v < kWaves; ++v)
                if (v < wave) lead += s_sum[0][v];
        }
        const u64 u = part31(a.u_draw[b]), t = share(all, u > 0x7FFFFFFFull ? 0x7FFFFFFFull : u);
        if (lead <= t && t < lead + mass)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const u64 run = wave_scan(left[e]), sum = lane_value(run, 63);
                if (lead <= t && t < lead + sum) {
                    const u64 hit = __ballot(lead + run > t);
                    if (lane == __ffsll(hit) - 1) s_verdict = RowVerdict{0, base + e * 64, (float)rw[0].share_of(w[0][e]), 0};
                }
                lead += sum;
            }
    }
    __syncthreads();
    RowVerdict *mine = verdicts + (int64_t)b * a.max_new;
    if (tid == 0) store_shared4((unsigned *)(mine + j), 0, __builtin_bit_cast(u4, s_verdict));
    if (!last_to_arrive(&arrived[b], rows.n, &s_flag) || wave != 0) return;
    int stop = kNever;
    for (int j0 = 0; j0 < rows.n; j0 += 64) {
        RowVerdict v{1, 0, 0, 0};
        if (j0 + lane < rows.n) v = __builtin_bit_cast(RowVerdict, load_shared4((const unsigned *)(mine + j0), 4 * lane));
        const u64 refused = __ballot(!v.ok);
        if (stop == kNever && refused) stop = j0 + __ffsll(refused) - 1;
        if (j0 + lane < rows.n) {
            const bool kept = j0 + lane <= stop;
            a.out[rows.begin + j0 + lane] = kept ? v.token : -1;
            if (a.prob) a.prob[rows.begin + j0 + lane] = kept ? v.prob : 0.0f;
        }
    }
    if (lane == 0) verify_counts(a, b, rows.n, stop);
}

// ---- rows too long for one workgroup's registers ----
//
// Three launches over chunks of rows: each chunk's largest logit and its place; its weight; then, of each request's first row
// that refuses its draft alone, what each chunk has left to draw from, of which the request's last chunk to arrive draws.
// A launch's workgroups work out for themselves what follows from the launch before.

struct SplitVerify {
    float *chunk_max;       // [rows][2][chunks], of the target and of the draft
    int *chunk_at;          // likewise
    u64 *chunk_sum;         // likewise
    u64 *left;              // [requests][chunks]
    int *arrived;           // [requests], zero between calls
    int chunks, per, sources;
};

// A workgroup's chunk of a row: (request, row of it, source) and the tokens [i0, i1).
struct VerifyChunk {
    int b, j, q, chunk;
    __device__ VerifyChunk(const pk_verify_desc &a, const SplitVerify &w) {
        int64_t id = blockIdx.x;
        chunk = (int)(id % w.chunks), id /= w.chunks;
        q = (int)(id % w.sources), id /= w.sources;
        j = (int)(id % a.max_new), b = (int)(id / a.max_new);
    }
};

template <class T>
__device__ inline const typename T::Raw *verify_row(const pk_verify_desc &a, int q, int r) {
    using Raw = typename T::Raw;
    return q ? (const Raw *)a.draft + (int64_t)r * a.draft_row : (const Raw *)a.logits + (int64_t)r * a.logits_row;
}

// The weights' rule of a row, from its chunks' maxima.
__device__ inline void row_rule(const pk_verify_desc &a, const SplitVerify &w, int b, int64_t place, int q, RowWeights &rw) {
    rw.settings(q ? a.draft_temperature : a.temperature, b);
    const float *m = w.chunk_max + (place * 2 + q) * w.chunks;
    const int *at = w.chunk_at + (place * 2 + q) * w.chunks;
    float top = m[0];
    int top_at = at[0];
    for (int c = 1; c < w.chunks; ++c)
        if (m[c] > top) top = m[c], top_at = at[c];
    rw.rule.top = top, rw.top_at = top_at;
}

template <class T>
__global__ __launch_bounds__(kSplitThreads) void verify_max_kernel(pk_verify_desc a, SplitVerify w) {
    __shared__ float s_max[kRuns];
    __shared__ int s_at[kRuns];
    const VerifyChunk c(a, w);
    const RequestRows rows(a, c.b);
    if (c.j >= rows.n || (c.q && rows.draft(a, c.j) < 0)) return;
    const auto *row = verify_row<T>(a, c.q, rows.begin + c.j);
    const int tid = threadIdx.x, size = w.per * kSplitThreads, i0 = c.chunk * size, i1 = min(i0 + size, a.vocab);
    float top = -INFINITY;
    int at = kNever;
    for (int i = i0 + tid; i < i1; i += kBatch * kSplitThreads) {
        float x[kBatch];
        load_batch<T>(row, i, kSplitThreads, i1, x);
#pragma unroll
        for (int e = 0; e < kBatch; ++e)
            if (x[e] > top) top = x[e], at = i + e * kSplitThreads;
    }
    const float wave_top = wave_max(top);
    at = lane_value(wave_scan(top == wave_top ? at : kNever, kNever, [](int u, int v) { return min(u, v); }), 63);
    if ((tid & 63) == 0) s_max[tid >> 6] = wave_top, s_at[tid >> 6] = at;
    __syncthreads();
    if (tid == 0) {
        float m = s_max[0];
        int p = s_at[0];
        for (int v = 1; v < kRuns; ++v)
            if (s_max[v] > m || (s_max[v] == m && s_at[v] < p)) m = s_max[v], p = s_at[v];
        const int64_t place = (((int64_t)c.b * a.max_new + c.j) * 2 + c.q) * w.chunks + c.chunk;
        w.chunk_max[place] = m, w.chunk_at[place] = p;
    }
}

template <class T>
__global__ __launch_bounds__(kSplitThreads) void verify_sum_kernel(pk_verify_desc a, SplitVerify w) {
    __shared__ u64 s_sum[kRuns];
    const VerifyChunk c(a, w);
    const RequestRows rows(a, c.b);
    if (c.j >= rows.n || (c.q && rows.draft(a, c.j) < 0)) return;
    const auto *row = verify_row<T>(a, c.q, rows.begin + c.j);
    const int tid = threadIdx.x, size = w.per * kSplitThreads, i0 = c.chunk * size, i1 = min(i0 + size, a.vocab);
    const int64_t place = (int64_t)c.b * a.max_new + c.j;
    float x[kBatch];
    load_batch<T>(row, i0 + tid, kSplitThreads, i1, x);       // on its way while the rule is worked out
    RowWeights rw;
    row_rule(a, w, c.b, place, c.q, rw);
    u64 sum = 0;
    for (int i = i0 + tid;;) {
#pragma unroll
        for (int e = 0; e < kBatch; ++e) sum += rw.weight(x[e], i + e * kSplitThreads);
        i += kBatch * kSplitThreads;
        if (i - tid >= i1) break;
        load_batch<T>(row, i, kSplitThreads, i1, x);
    }
    sum = wave_sum(sum);
    if ((tid & 63) == 0) s_sum[tid >> 6] = sum;
    __syncthreads();
    if (tid < 64) {
        sum = wave_sum(tid < kRuns ? s_sum[tid] : 0);
        if (tid == 0) w.chunk_sum[(place * 2 + c.q) * w.chunks + c.chunk] = sum;
    }
}

template <class T>
__global__ __launch_bounds__(kSplitThreads) void verify_draw_kernel(pk_verify_desc a, SplitVerify w) {
    __shared__ u64 s_sum[kRuns], s_base;
    __shared__ int s_stop, s_flag, s_chunk;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), V = a.vocab;
    const int b = blockIdx.x / w.chunks, chunk = blockIdx.x % w.chunks;
    const RequestRows rows(a, b);
    if (rows.n == 0) {
        if (chunk == 0 && tid == 0) verify_counts(a, b, 0, 0);
        return;
    }
    // a row's rules with their sums; by a whole wave
    auto rules = [&](int j, int d, RowWeights (&rw)[2]) {
        const int64_t place = (int64_t)b * a.max_new + j;
        u64 sum = 0;
        for (int q = 0; q < (d >= 0 ? w.sources : 1); ++q) {
            row_rule(a, w, b, place, q, rw[q]);
            const u64 s = wave_sum(lane < w.chunks ? w.chunk_sum[(place * 2 + q) * w.chunks + lane] : 0);
            rw[q].total(s);
            if (q == 0) sum = s;
        }
        return sum;
    };
    auto draft_share = [&](int j, int d, const RowWeights (&rw)[2], double &q) {
        q = w.sources > 1 ? rw[1].share_of(rw[1].weight(logit<T>(verify_row<T>(a, 1, rows.begin + j), d), d)) : 1.0;
        return rw[0].share_of(rw[0].weight(logit<T>(verify_row<T>(a, 0, rows.begin + j), d), d));
    };
    // the first row that refuses its draft, a row a wave
    if (tid == 0) s_stop = kNever;
    __syncthreads();
    for (int j0 = 0;; j0 += kRuns) {
        const int j = j0 + wave;
        if (j < rows.n) {
            const int d = rows.draft(a, j);
            bool ok = false;
            if (d >= 0) {
                RowWeights rw[2];
                rules(j, d, rw);
                double q;
                const double p = draft_share(j, d, rw, q);
                ok = __dmul_rn(uniform(a.u[rows.begin + j]), q) < p;
            }
            if (!ok && lane == 0) atomicMin(&s_stop, j);
        }
        __syncthreads();
        if (s_stop != kNever) break;             // the last row has no draft
    }
    const int stop = s_stop;
    if (chunk == 0) {
        for (int j = wave; j < rows.n; j += kRuns) {
            if (j == stop) continue;
            int token = -1;
            float prob = 0;
            if (j < stop) {
                token = rows.draft(a, j);
                RowWeights rw[2];
                rules(j, token, rw);
                double q;
                prob = (float)draft_share(j, token, rw, q);
            }
            if (lane == 0) {
                a.out[rows.begin + j] = token;
                if (a.prob) a.prob[rows.begin + j] = prob;
            }
        }
        if (tid == 0) verify_counts(a, b, rows.n, stop);
    }
    const int d = rows.draft(a, stop), r = rows.begin + stop;
    RowWeights rw[2];
    const u64 total = rules(stop, d, rw);
    const bool drafted = d >= 0, two = drafted && w.sources > 1;
    const auto *x_row = verify_row<T>(a, 0, r), *y_row = two ? verify_row<T>(a, 1, r) : x_row;
    auto left = [&](int i, bool any) -> u64 {
        if (i >= V) return 0;
        const unsigned wt = rw[0].weight(logit<T>(x_row, i), i);
        if (any || !drafted) return wt;
        if (!two) return i == d ? 0 : wt;
        return left_of(rw[0].share_of(wt), rw[1].share_of(rw[1].weight(logit<T>(y_row, i), i)));
    };
    // a chunk is kRuns runs of 64 per tokens, a wave each
    auto run_sum = [&](int ch, bool any) {
        u64 mass = 0;
        const int i0 = (ch * kRuns + wave) * 64 * w.per + lane;
#pragma unroll 4
        for (int e = 0; e < w.per; ++e) mass += left(i0 + e * 64, any);
        return wave_sum(mass);
    };
    auto chunk_total = [&]() {
        u64 s = 0;
        for (int v = 0; v < kRuns; ++v) s += s_sum[v];
        return s;
    };
    {
        const u64 mass = run_sum(chunk, false);
        if (lane == 0) s_sum[wave] = mass;
        __syncthreads();
        if (tid == 0) put_shared(&w.left[(int64_t)b * w.chunks + chunk], chunk_total());
    }
    if (!last_to_arrive(&w.arrived[b], w.chunks, &s_flag)) return;
    const u64 of_chunk = lane < w.chunks ? get_shared(&w.left[(int64_t)b * w.chunks + lane]) : 0;
    u64 all = wave_sum(of_chunk), mine = of_chunk;
    const bool any = all == 0;                   // nothing: from the target itself
    if (any) {
        all = total;
        mine = lane < w.chunks ? w.chunk_sum[((int64_t)b * a.max_new + stop) * 2 * w.chunks + lane] : 0;
    }
    if (all == 0) {
        if (tid == 0) {
            a.out[r] = -1;
            if (a.prob) a.prob[r] = 0;
        }
        return;
    }
    const u64 u = part31(a.u_draw[b]), t = share(all, u > 0x7FFFFFFFull ? 0x7FFFFFFFull : u);
    if (wave == 0) {
        const u64 before = wave_scan(mine) - mine;
        if (before <= t && t < before + mine) s_chunk = lane, s_base = before;
    }
    __syncthreads();
    const int ch = s_chunk;
    const u64 mass = run_sum(ch, any);
    if (lane == 0) s_sum[wave] = mass;
    __syncthreads();
    u64 lead = s_base;
    for (int v = 0; v < wave; ++v) lead += s_sum[v];
    if (lead > t || lead + mass <= t) return;
    const int i0 = (ch * kRuns + wave) * 64 * w.per + lane;
    for (int e = 0; e < w.per; ++e) {
        const int i = i0 + e * 64;
        const u64 run = wave_scan(left(i, any)), sum = lane_value(run, 63);
        if (lead <= t && t < lead + sum) {
            const u64 hit = __ballot(lead + run > t);
            if (lane == __ffsll(hit) - 1) {
                a.out[r] = i;
                if (a.prob) a.prob[r] = (float)rw[0].share_of(rw[0].weight(logit<T>(x_row, i), i));
            }
            break;
        }
        lead += sum;
    }
}

}  // namespace pklm
