// lm_verify.h -- drafted tokens against the target's probabilities (pk_verify).
//
// Weights are whole numbers, w = round(2^30 exp((x - max) / T)), as pk_sample's but for the last bits of the exponential, so that
// their sums are exact in any order.  What is compared and drawn from follows from them in single f64 steps, p = w (1 / sum w):
// the same wherever it is worked out.  A refused draft's successor is drawn from max(p - q, 0) in steps of 2^-52, whole
// numbers again, whose sum is at most 2^52 and a half step for each token.
#pragma once

#include <type_traits>

#include "lm_common.h"
#include "lm_sample.h"
#include "parakeet_lm.h"

namespace pklm {

// Single steps: neither is fused with the other, as the compiler would where it may (HIP's __dmul_rn and __dadd_rn are plain
// operators, which it fuses).
__device__ inline double product(double a, double b) {
#pragma clang fp contract(off)
    return a * b;
}
__device__ inline double difference(double a, double b) {
#pragma clang fp contract(off)
    return a - b;
}

constexpr int kNever = 0x7FFFFFFF;
constexpr float kMostLogit = 0x1.fffffep127f;         // +inf counts as this

// One row's weights: the logits' largest, log2(e) / T, and where the largest alone counts its place.
struct RowWeights {
    float top, to_log2;
    bool greedy;
    int top_at;
    double inv_sum;

    __device__ void settings(const float *temperature, int b) {
        const float t = temperature ? temperature[b] : 1.0f;
        greedy = !(t > 0);
        to_log2 = fminf(fmaxf(1.4426950408889634f / (greedy ? 1.0f : t), 1e-38f), 3e38f);
    }
    // a row of -inf has no weight, in one with +inf those are alike
    __device__ void largest(float x) { top = x == -INFINITY ? 0.0f : fminf(x, kMostLogit); }
    // exp2 of one rounded product: off by 2^-23 and 2^-24 of the exponent, 2^-19 of itself where weights end.  (The library's expf takes
    // half as long again: weights are what bounds long rows.)  The median of -200, 0 and the exponent is -200 for -inf and NaN.
    __device__ float weight_f(float x, int i) const {
        if (greedy) return i == top_at ? 1073741824.0f : 0.0f;
        return rintf(__builtin_amdgcn_exp2f(__builtin_amdgcn_fmed3f((x - top) * to_log2, -200.0f, 0.0f)) * 1073741824.0f);
    }
    __device__ unsigned weight(float x, int i) const { return (unsigned)weight_f(x, i); }
    __device__ void total(u64 sum) { inv_sum = sum ? 1.0 / (double)sum : 0.0; }
    __device__ double share_of(unsigned w) const { return product((double)w, inv_sum); }
};

// 8 adjacent logits of a row, from i on, as they come from memory; rows need not be aligned.
template <class T>
struct Tokens8 {
    typename T::Raw raw[8];

    __device__ void load(const typename T::Raw *row, int i, int end) {
        if (i + 8 <= end) {
            __builtin_memcpy(raw, row + i, sizeof(raw));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) raw[e] = i < end ? row[min(i + e, end - 1)] : (typename T::Raw)0;
        }
    }
    // -inf behind the row's end
    __device__ float get(int e, int i, int end) const { return i + e >= end ? -INFINITY : T::get(raw[e]); }
    // f(e, value) of each, of a wave's pass that may reach past the row's end
    template <class F>
    __device__ void each(int i, int end, F f) const {
        if (__all(i + 8 <= end)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f(e, T::get(raw[e]));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f(e, get(e, i, end));
        }
    }
};
__device__ inline int wave_min(int v) { return lane_value(wave_scan(v, kNever, [](int a, int b) { return min(a, b); }), 63); }

__device__ inline double uniform(float u) {
    const u64 v = part31(u);
    return (double)(v > 0x7FFFFFFFull ? 0x7FFFFFFFull : v) * 0x1p-31;
}
// In steps of 2^-52, cut to whole ones: at most 2^52, so that added to 2^52 they are the low bits.
__device__ inline u64 left_of(double p, double q) {
    const double d = difference(p, q);
    return d > 0 ? __double_as_longlong(trunc(d * 0x1p52) + 0x1p52) - __double_as_longlong(0x1p52) : 0;
}

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

// One launch, bound by its latency: 5 rows of 8,193 logits in f32 take 8.0 us a call, 256 requests of up to 6 rows of 1,027 with draft logits
// 9.6.
//
// A request has `each` workgroups, a row on each, or several in turn (Turns, which takes up to a tenth longer by its registers) where there
// may be more rows.  Tokens are in registers: wave w has tokens ((w n + g) 64 + lane) 8 + e of a row, g < n <= G.  Every row that
// refuses its draft draws its own token, whether or not an earlier row has refused; the request's last row to arrive has the rows'
// verdicts and writes them up to the first refusal.
template <class T, int BS, int G, bool Draft, bool Turns>
__global__ __launch_bounds__(BS) void verify_row_kernel(pk_verify_desc a, int each, int *arrived, RowVerdict *verdicts) {
    constexpr int kWaves = BS / 64, E = 8 * G, kSources = Draft ? 2 : 1;
    __shared__ float s_max[2][kWaves];
    __shared__ int s_at[2][kWaves];
    __shared__ u64 s_sum[2][kWaves], s_left[kWaves];
    __shared__ RowVerdict s_verdict;
    __shared__ int s_flag;
    using Raw = typename T::Raw;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Of Turns most may have no row: those go last.  Turned on by a request, so that one's rows are not all on one XCD.
    const int first = Turns ? blockIdx.x / a.requests : blockIdx.x % each;
    const int b = Turns ? (blockIdx.x + first) % a.requests : blockIdx.x / each;
    const RequestRows rows(a, b);
    if (rows.n == 0 && first == 0 && tid == 0) verify_counts(a, b, 0, 0);
#pragma nounroll
    for (int j = first; j < rows.n; j += each) {
        // what follows from these is worked out for each row, not once in front of them all, over which it would be spilled
        int lane = tid & 63, V = a.vocab;
        if (Turns) asm volatile("" : "+v"(lane), "+s"(V));
        const int r = rows.begin + j, d = rows.draft(a, j);
        const bool drafted = d >= 0;
        const int n = (V + 8 * BS - 1) / (8 * BS);
        auto index = [&](int g) { return ((wave * n + g) * 64 + lane) * 8; };
        const Raw *row[2] = {(const Raw *)a.logits + (int64_t)r * a.logits_row, Draft ? (const Raw *)a.draft + (int64_t)r * a.draft_row : nullptr};
        Tokens8<T> raw[kSources][G];
        float at_draft[2];
        RowWeights rw[2];
#pragma unroll
        for (int q = 0; q < kSources; ++q) {
            const int end = q == 0 || drafted ? V : 0;      // without a draft its row is not read
#pragma unroll
            for (int g = 0; g < G; ++g) raw[q][g].load(row[q], g < n ? index(g) : end, end);
            at_draft[q] = drafted ? logit<T>(row[q], d) : -INFINITY;
            rw[q].settings(q ? a.draft_temperature : a.temperature, b);
        }
        float x[kSources][E];
#pragma unroll
        for (int q = 0; q < kSources; ++q) {
            const int end = q == 0 || drafted ? V : 0;
            float top = -INFINITY;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                x[q][e] = raw[q][e / 8].get(e % 8, e / 8 < n ? index(e / 8) : end, end);
                top = fmaxf(top, x[q][e]);
            }
            top = wave_max(top);
            if (lane == 0) s_max[q][wave] = top;
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < kSources; ++q) {
            float top = s_max[q][0];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) top = fmaxf(top, s_max[q][w]);
            rw[q].largest(top), rw[q].top_at = kNever;
        }
        if (rw[0].greedy || (Draft && rw[1].greedy)) {       // the first place of the largest; no NaN is as large as it
#pragma unroll
            for (int q = 0; q < kSources; ++q) {
                int at = kNever;
#pragma unroll
                for (int e = E - 1; e >= 0; --e) at = x[q][e] >= rw[q].top ? index(e / 8) + e % 8 : at;
                at = wave_min(at);
                if (lane == 0) s_at[q][wave] = at;
            }
            __syncthreads();
#pragma unroll
            for (int q = 0; q < kSources; ++q)
#pragma unroll
                for (int v = 0; v < kWaves; ++v) rw[q].top_at = min(rw[q].top_at, s_at[q][v]);
        }
        unsigned w[kSources][E];
#pragma unroll
        for (int q = 0; q < kSources; ++q) {
            u64 sum = 0;
#pragma unroll
            for (int g = 0; g < G; ++g)
                if (g < n)
#pragma unroll
                    for (int e = 8 * g; e < 8 * g + 8; ++e) {
                        w[q][e] = rw[q].weight(x[q][e], index(g) + e % 8);
                        sum += w[q][e];
                    }
                else
#pragma unroll
                    for (int e = 8 * g; e < 8 * g + 8; ++e) w[q][e] = 0;
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
        const bool ok = drafted && product(uniform(a.u[r]), q_draft) < p_draft;
        if (ok || total[0] == 0) {
            if (tid == 0) s_verdict = RowVerdict{ok, ok ? d : -1, ok ? (float)p_draft : 0.0f, 0};
        } else {
            // what is left to draw from
            std::conditional_t<Draft, u64, unsigned> left[E];
            u64 mass = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                left[e] = w[0][e];
                if (drafted && Draft) left[e] = left_of(rw[0].share_of(w[0][e]), rw[1].share_of(w[kSources - 1][e]));
                if (drafted && !Draft) left[e] = index(e / 8) + e % 8 == d ? 0 : left[e];
                mass += left[e];
            }
            mass = wave_sum(mass);
            if (lane == 0) s_left[wave] = mass;
            __syncthreads();
            u64 all = 0, lead = 0;
#pragma unroll
            for (int v = 0; v < kWaves; ++v) {
                if (v < wave) lead += s_left[v];
                all += s_left[v];
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
                for (int g = 0; g < G; ++g) {
                    u64 own = 0;
#pragma unroll
                    for (int e = 0; e < 8; ++e) own += left[8 * g + e];
                    const u64 run = wave_scan(own);
                    u64 at = lead + run - own;
                    if (at <= t && t < at + own)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            if (at <= t && t < at + left[8 * g + e])
                                s_verdict = RowVerdict{0, index(g) + e, (float)rw[0].share_of(w[0][8 * g + e]), 0};
                            at += left[8 * g + e];
                        }
                    lead += lane_value(run, 63);
                }
        }
        __syncthreads();
        auto write = [&](int at, const RowVerdict &v, bool kept) {
            a.out[rows.begin + at] = kept ? v.token : -1;
            if (a.prob) a.prob[rows.begin + at] = kept ? v.prob : 0.0f;
        };
        if (rows.n == 1) {
            if (tid == 0) write(0, s_verdict, true), verify_counts(a, b, 1, 0);
            return;
        }
        RowVerdict *mine = verdicts + rows.begin;
        if (tid == 0) store_shared4((unsigned *)(mine + j), 0, __builtin_bit_cast(u4, s_verdict));
        if (!last_to_arrive(&arrived[b], rows.n, &s_flag)) {
            if (Turns) continue;
            return;
        }
        if (wave != 0) return;
        int stop = kNever;
        for (int j0 = 0; j0 < rows.n; j0 += 64) {
            RowVerdict v{1, 0, 0, 0};
            if (j0 + lane < rows.n) v = __builtin_bit_cast(RowVerdict, load_shared4((const unsigned *)(mine + j0), 4 * lane));
            const u64 refused = __ballot(!v.ok || j0 + lane == rows.n - 1);
            if (stop == kNever && refused) stop = j0 + __ffsll(refused) - 1;
            if (j0 + lane < rows.n) write(j0 + lane, v, j0 + lane <= stop);
        }
        if (lane == 0) verify_counts(a, b, rows.n, stop);
        return;
    }
}

// ---- rows too long for one workgroup's registers ----
//
// Three launches over chunks of rows: each chunk's largest logit and its place; its weight; then, of each request's first row
// that refuses its draft alone, what each chunk has left to draw from, of which the request's last chunk to arrive draws.
// A launch's workgroups work out for themselves what follows from the launch before.  64 requests of up to 5 rows of 128,001 in bf16 with draft
// logits, 57 MB: 18 us (memory; 15 on one input again and again), 17 (the vector unit: 28 million exponentials, the rows again from the
// cache behind the L2) and 31 (the chain to each request's row, its own exponentials and f64 sums, the drawn chunk summed again and
// searched).

// Of the first two launches, and of the draws, whose workgroups each find the row that they draw from: 256 and 512 threads.  (64 requests of up
// to 5 rows of 128,001 in bf16 with draft logits on 256, 512 and 1,024: 24, 28, 35 us the two, 29, 21, 27 the draws.)
constexpr int kVerifyThreads = 256, kVerifyWaves = kVerifyThreads / 64, kVerifyPass = 8 * kVerifyThreads;
constexpr int kDrawThreads = 512, kDrawWaves = kDrawThreads / 64, kDrawPass = 8 * kDrawThreads;

struct SplitVerify {
    float *chunk_max;       // [rows of the call][2][chunks], of the target and of the draft
    int *chunk_at;          // likewise; where the largest alone counts
    u64 *chunk_sum;         // likewise
    u64 *left;              // [requests][chunks]
    int *arrived;           // [requests], zero between calls
    int chunks, passes, sources;        // a chunk is passes * kVerifyPass tokens, a wave's part of it in one run
    int draw_chunks, draw_passes;       // likewise, with kDrawPass, of the one row of a request that is drawn from
};

// The request of the call's row r, the first one that ends behind it: by a whole wave, among 64 runs of requests, then in the run.
static_assert(PK_LM_MAX_REQUESTS <= 64 * 64, "a lane looks at one run, then at one request");
__device__ inline int request_of(const pk_verify_desc &a, int r) {
    const int lane = threadIdx.x & 63, run = (a.requests + 63) / 64;
    auto behind = [&](int request) { return __ballot(a.first[min(request + 1, a.requests)] > r); };
    const u64 runs = behind((lane + 1) * run - 1);
    int b = runs ? __builtin_ctzll(runs) * run : a.requests - 1;
    if (run > 1) {
        const u64 in = behind(b + lane);
        b += in ? __builtin_ctzll(in) : 0;
    }
    return min(b, a.requests - 1);
}

// A workgroup's chunk of a row of the call: its request and place in it, none where j is not below rows.n.
struct VerifyChunk {
    int q, chunk, r, b, j;
    RequestRows rows;
    __device__ VerifyChunk(const pk_verify_desc &a, const SplitVerify &w)
        : q(blockIdx.x / w.chunks % w.sources), chunk(blockIdx.x % w.chunks), r(blockIdx.x / w.chunks / w.sources), b(request_of(a, r)), rows(a, b) {
        j = r >= rows.begin ? r - rows.begin : rows.n;
    }
    __device__ bool none(const pk_verify_desc &a) const { return j >= rows.n || (q && rows.draft(a, j) < 0); }
    __device__ int64_t place(const SplitVerify &w) const { return ((int64_t)r * 2 + q) * w.chunks + chunk; }
};

template <class T>
__device__ inline const typename T::Raw *verify_row(const pk_verify_desc &a, int q, int r) {
    using Raw = typename T::Raw;
    return q ? (const Raw *)a.draft + (int64_t)r * a.draft_row : (const Raw *)a.logits + (int64_t)r * a.logits_row;
}
// The first token of this lane in a pass of a chunk of so many waves.
template <int Waves>
__device__ inline int verify_token(int passes, int chunk, int pass) {
    return ((chunk * Waves + (int)(threadIdx.x >> 6)) * passes + pass) * 512 + (int)(threadIdx.x & 63) * 8;
}

// The rule of row r of the call, from its chunks' maxima, and its weight where the chunks have theirs: by a whole wave.
__device__ inline u64 row_rule(const pk_verify_desc &a, const SplitVerify &w, int b, int r, int q, RowWeights &rw, bool summed) {
    const int lane = threadIdx.x & 63;
    const int64_t at = ((int64_t)r * 2 + q) * w.chunks + lane;
    rw.settings(q ? a.draft_temperature : a.temperature, b);
    const bool in = lane < w.chunks;
    const float m = in ? w.chunk_max[at] : -INFINITY;
    const u64 sum = summed && in ? w.chunk_sum[at] : 0;
    const int p = rw.greedy && in ? w.chunk_at[at] : kNever;
    const float top = wave_max(m);
    rw.largest(top);
    rw.top_at = rw.greedy && top != -INFINITY ? wave_min(m == top ? p : kNever) : kNever;
    const u64 total = summed ? wave_sum(sum) : 0;
    rw.total(total);
    return total;
}

template <class T>
__global__ __launch_bounds__(kVerifyThreads) void verify_max_kernel(pk_verify_desc a, SplitVerify w) {
    __shared__ float s_max[kVerifyWaves];
    __shared__ int s_at[kVerifyWaves];
    const VerifyChunk c(a, w);
    if (c.none(a)) return;
    const auto *row = verify_row<T>(a, c.q, c.r);
    const int tid = threadIdx.x, V = a.vocab;
    RowWeights rw;
    rw.settings(c.q ? a.draft_temperature : a.temperature, c.b);
    float top = -INFINITY;
    int at = kNever;
    for (int p0 = 0; p0 < w.passes; p0 += 2) {
        Tokens8<T> x[2];
        int i[2];
#pragma unroll
        for (int p = 0; p < 2; ++p) i[p] = p0 + p < w.passes ? verify_token<kVerifyWaves>(w.passes, c.chunk, p0 + p) : V, x[p].load(row, i[p], V);
#pragma unroll
        for (int p = 0; p < 2; ++p)
            x[p].each(i[p], V, [&](int e, float v) {
                if (rw.greedy && v > top && top < kMostLogit) at = i[p] + e;
                top = fmaxf(top, v);
            });
    }
    top = fminf(top, kMostLogit);
    const float wave_top = wave_max(top);
    at = rw.greedy ? wave_min(top == wave_top ? at : kNever) : kNever;
    if ((tid & 63) == 0) s_max[tid >> 6] = wave_top, s_at[tid >> 6] = at;
    __syncthreads();
    if (tid == 0) {
        float m = s_max[0];
        int p = s_at[0];
        for (int v = 1; v < kVerifyWaves; ++v)
            if (s_max[v] > m || (s_max[v] == m && s_at[v] < p)) m = s_max[v], p = s_at[v];
        w.chunk_max[c.place(w)] = m, w.chunk_at[c.place(w)] = p;
    }
}

template <class T>
__global__ __launch_bounds__(kVerifyThreads) void verify_sum_kernel(pk_verify_desc a, SplitVerify w) {
    __shared__ u64 s_sum[kVerifyWaves];
    const VerifyChunk c(a, w);
    if (c.none(a)) return;
    const auto *row = verify_row<T>(a, c.q, c.r);
    const int tid = threadIdx.x, V = a.vocab;
    Tokens8<T> x;
    x.load(row, verify_token<kVerifyWaves>(w.passes, c.chunk, 0), V);       // on its way while the rule is worked out
    RowWeights rw;
    row_rule(a, w, c.b, c.r, c.q, rw, false);
    u64 sum = 0;
    for (int p = 0; p < w.passes; ++p) {
        const int i = verify_token<kVerifyWaves>(w.passes, c.chunk, p);
        Tokens8<T> y;
        y.load(row, p + 1 < w.passes ? verify_token<kVerifyWaves>(w.passes, c.chunk, p + 1) : V, V);
        unsigned two = 0;                              // of at most 2^30 each
        x.each(i, V, [&](int e, float v) {
            two += rw.weight(v, i + e);
            if (e & 1) sum += two, two = 0;
        });
        x = y;
    }
    sum = wave_sum(sum);
    if ((tid & 63) == 0) s_sum[tid >> 6] = sum;
    __syncthreads();
    if (tid < 64) {
        sum = wave_sum(tid < kVerifyWaves ? s_sum[tid] : 0);
        if (tid == 0) w.chunk_sum[c.place(w)] = sum;
    }
}

template <class T>
__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(pk_verify_desc a, SplitVerify w) {
    __shared__ u64 s_sum[kDrawWaves], s_base;
    __shared__ int s_stop[2], s_flag, s_chunk;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), V = a.vocab;
    const int b = blockIdx.x / w.draw_chunks, chunk = blockIdx.x % w.draw_chunks;
    const RequestRows rows(a, b);
    if (rows.n == 0) {
        if (chunk == 0 && tid == 0) verify_counts(a, b, 0, 0);
        return;
    }
    const bool two_sources = w.sources > 1;
    RowWeights target, draft;
    // p and q of a row's draft; by a whole wave
    auto shares = [&](int j, int d, double &q) {
        const float x = logit<T>(verify_row<T>(a, 0, rows.begin + j), d), y = two_sources ? logit<T>(verify_row<T>(a, 1, rows.begin + j), d) : 0.0f;
        row_rule(a, w, b, rows.begin + j, 0, target, true);
        q = 1.0;
        if (two_sources) {
            row_rule(a, w, b, rows.begin + j, 1, draft, true);
            q = draft.share_of(draft.weight(y, d));
        }
        return target.share_of(target.weight(x, d));
    };
    // The first row that refuses its draft, a row a wave; those in front of it stay.  Rounds of rows have two places in turn, since a
    // wave may look at a round's after another has begun the next.
    if (tid < 2) s_stop[tid] = kNever;
    __syncthreads();
    int stop = kNever;
    for (int j0 = 0, round = 0; stop == kNever; j0 += kDrawWaves, round ^= 1) {      // ends: the last row has no draft
        const int j = j0 + wave, d = j < rows.n ? rows.draft(a, j) : -1;
        double p = 0, q = 1;
        if (d >= 0) p = shares(j, d, q);
        const bool ok = d >= 0 && product(uniform(a.u[rows.begin + j]), q) < p;
        if (!ok && lane == 0 && j < rows.n) atomicMin(&s_stop[round], j);
        __syncthreads();
        stop = s_stop[round];
        if (chunk == 0 && lane == 0 && j < min(rows.n, stop)) {
            a.out[rows.begin + j] = d;
            if (a.prob) a.prob[rows.begin + j] = (float)p;
        }
    }
    if (chunk == 0) {
        for (int j = stop + 1 + tid; j < rows.n; j += kDrawThreads) {
            a.out[rows.begin + j] = -1;
            if (a.prob) a.prob[rows.begin + j] = 0.0f;
        }
        if (tid == 0) verify_counts(a, b, rows.n, stop);
    }
    const int d = rows.draft(a, stop), r = rows.begin + stop;
    const bool drafted = d >= 0, two = drafted && two_sources;
    const auto *x_row = verify_row<T>(a, 0, r), *y_row = two ? verify_row<T>(a, 1, r) : x_row;
    const u64 total = row_rule(a, w, b, r, 0, target, true);
    if (two) row_rule(a, w, b, r, 1, draft, true);
    // What is left of a lane's 8 tokens of a pass, whole numbers in f64, whose sums are exact: of p - q in steps of 2^-52 at most 2^52
    // and a step a token, of weights at most 2^50.
    const double scale_p = target.inv_sum * 0x1p52, scale_q = two ? draft.inv_sum * 0x1p52 : 0.0;
    struct Pass {
        Tokens8<T> x, y;
    };
    auto load_pass = [&](int ch, int pass, bool any, Pass &of) {
        const int i = pass < w.draw_passes ? verify_token<kDrawWaves>(w.draw_passes, ch, pass) : V;
        of.x.load(x_row, i, V);
        if (two && !any) of.y.load(y_row, i, V);
    };
    auto left_of_pass = [&](int ch, int pass, bool any, const Pass &of, double (&left)[8]) {
        const int i = verify_token<kDrawWaves>(w.draw_passes, ch, pass);
        of.x.each(i, V, [&](int e, float v) { left[e] = (double)target.weight_f(v, i + e); });
        if (any || !drafted) return;
        if (two)
            of.y.each(i, V, [&](int e, float v) {
                left[e] = trunc(fmax(difference(product(left[e], scale_p), product((double)draft.weight_f(v, i + e), scale_q)), 0.0));
            });
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) left[e] = i + e == d ? 0.0 : left[e];
    };
    auto run_sum = [&](int ch, bool any) {
        double mass = 0;
        Pass now, next;
        load_pass(ch, 0, any, now);
        for (int p = 0; p < w.draw_passes; ++p) {
            load_pass(ch, p + 1, any, next);
            double left[8];
            left_of_pass(ch, p, any, now, left);
#pragma unroll
            for (int e = 0; e < 8; ++e) mass += left[e];
            now = next;
        }
        return wave_sum((u64)mass);
    };
    {
        const u64 mass = run_sum(chunk, false);
        if (lane == 0) s_sum[wave] = mass;
        __syncthreads();
        if (tid == 0) {
            u64 s = 0;
            for (int v = 0; v < kDrawWaves; ++v) s += s_sum[v];
            put_shared(&w.left[(int64_t)b * w.draw_chunks + chunk], s);
        }
    }
    if (!last_to_arrive(&w.arrived[b], w.draw_chunks, &s_flag)) return;
    const u64 mine = lane < w.draw_chunks ? get_shared(&w.left[(int64_t)b * w.draw_chunks + lane]) : 0;
    u64 all = wave_sum(mine);
    const bool any = all == 0;                   // nothing: from the target itself
    if (any) all = total;
    if (all == 0) {
        if (tid == 0) {
            a.out[r] = -1;
            if (a.prob) a.prob[r] = 0;
        }
        return;
    }
    const u64 u = part31(a.u_draw[b]), t = share(all, u > 0x7FFFFFFFull ? 0x7FFFFFFFull : u);
    // the chunk in which the drawn weight falls: from the chunks' sums, or (seldom) chunk by chunk
    if (wave == 0 && !any) {
        const u64 before = wave_scan(mine) - mine;
        if (before <= t && t < before + mine) s_chunk = lane, s_base = before;
    }
    __syncthreads();
    int ch = any ? 0 : s_chunk;
    u64 lead = any ? 0 : s_base, mass = 0;
    for (;; ++ch) {                              // ends: t is below the sum over all chunks
        mass = run_sum(ch, any);
        if (lane == 0) s_sum[wave] = mass;
        __syncthreads();
        u64 of_chunk = 0;
        for (int v = 0; v < kDrawWaves; ++v) of_chunk += s_sum[v];
        if (t < lead + of_chunk || ch + 1 >= w.draw_chunks) break;
        lead += of_chunk;
        __syncthreads();
    }
    for (int v = 0; v < wave; ++v) lead += s_sum[v];
    if (lead > t || lead + mass <= t) return;
    for (int p = 0; p < w.draw_passes; ++p) {
        Pass now;
        double left[8];
        u64 own = 0;
        load_pass(ch, p, any, now);
        left_of_pass(ch, p, any, now, left);
#pragma unroll
        for (int e = 0; e < 8; ++e) own += (u64)left[e];
        const u64 run = wave_scan(own), sum = lane_value(run, 63);
        u64 at = lead + run - own;
        if (at <= t && t < at + own) {
            const int i0 = verify_token<kDrawWaves>(w.draw_passes, ch, p);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (at <= t && t < at + (u64)left[e]) {
                    a.out[r] = i0 + e;
                    if (a.prob) a.prob[r] = (float)target.share_of(target.weight(logit<T>(x_row, i0 + e), i0 + e));
                }
                at += (u64)left[e];
            }
        }
        lead += sum;
    }
}

}  // namespace pklm
