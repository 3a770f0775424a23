// lm_sample.h -- one token per row of logits (pk_sample).
//
// Weights are whole numbers, so sums are exact and the same in any order, and atomics may build them.  In the order
// (falling logit, rising index) the kept tokens are a prefix, so the filters come down to one cut: the last kept token.
// Every token has a rank word, its logit's ordered bits (those that its type has) over its inverted index; kept is
// rank >= cut.
//
// To find the cut, tokens are binned by their distance from the largest logit, (max - x) / T in bins of 22/1,024
// (weights round to none at 21.5), and the bins' (count, weight) sums are scanned.  That names the bin in which
// the count reaches top_k or the weight reaches top_p's share, and the tokens of that bin are listed; of a small top_k those
// up to that bin.  A short list is sorted, each word's place the number of larger ones: the cut is a place in it, and of a
// list with all kept tokens the token too.  In a longer one, and where a bin has more tokens than a list holds (many equal
// logits), the cut's rank word is found eight bits at a time.
#pragma once

#include "lm_common.h"
#include "parakeet_lm.h"

namespace pklm {

typedef unsigned long long u64;

constexpr float kReach = 22.0f;            // distance that the bins cover
constexpr float kWeighed = -21.6f;         // a distance beyond this has no weight: exp(-21.6) < 2^-31
constexpr int kCountShift = 46;            // (count, weight) of up to 2^15 tokens in one word: 2^15 2^30 < 2^46
constexpr u64 kMassMask = (1ull << kCountShift) - 1;

// f32 order as unsigned order; both zeros alike
__device__ inline unsigned order_key(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr int kIndexBits = 20;             // PK_LM_MAX_VOCAB
// floor(total * part / 2^31), part <= 2^31
__device__ inline u64 share(u64 total, u64 part) { return (total >> 31) * part + (((total & 0x7FFFFFFFull) * part) >> 31); }
__device__ inline u64 part31(float p) { return (u64)(fminf(fmaxf(p, 0.0f), 1.0f) * 2147483648.0f); }

// One row's settings and what follows from its largest logit.
struct RowRule {
    float top, inv;
    unsigned least;      // min_p's weight
    int k;               // how many at most
    u64 p;               // top_p in 2^-31
    bool k_on, p_on;
    int spare;           // low bits that no logit of this type has in f32

    __device__ u64 rank(float x, int i) const {
        return (u64)(order_key(x) >> spare) << kIndexBits | (unsigned)((1 << kIndexBits) - 1 - i);
    }
    __device__ float logit_of(u64 rank) const {
        const unsigned k = (unsigned)(rank >> kIndexBits) << spare;
        return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~(k | ((1u << spare) - 1)));
    }

    template <class T>
    __device__ void settings(const pk_sample_desc &a, int b) {
        spare = __is_same(T, F32) ? 0 : __is_same(T, F16) ? 13 : 16;
        const float t = a.temperature ? a.temperature[b] : 1.0f;
        const bool greedy = !(t > 0);
        inv = greedy ? 1.0f : fminf(1.0f / t, 3e38f);
        const int top_k = a.top_k ? a.top_k[b] : 0;
        k = greedy ? 1 : top_k;
        k_on = greedy || (top_k > 0 && top_k < a.vocab);
        p = part31(a.top_p ? a.top_p[b] : 1.0f);
        p_on = p < 0x80000000ull;
        least = (unsigned)ceilf(fminf(fmaxf(a.min_p ? a.min_p[b] : 0.0f, 0.0f), 1.0f) * 1073741824.0f);
    }
    __device__ float distance(float x) const { return x == top ? 0.0f : (x - top) * inv; }
    __device__ unsigned weight(float x) const {
        return x == -INFINITY ? 0u : (unsigned)rintf(expf(distance(x)) * 1073741824.0f);
    }
    // the steps from x to the bin are monotone, so bins keep the order; tokens without a weight are in none, or the last
    template <int Bins>
    __device__ int bin(float x) const { return (int)fminf(distance(x) * (-Bins / kReach), (float)(Bins - 1)); }
};

template <class T>
__device__ inline float logit(const typename T::Raw *row, int i) {
    const float x = T::get(row[i]);
    return x != x ? -INFINITY : x;
}

// Where a cut was found: the token's rank word and the weight up to it, itself included.
struct Cut {
    u64 rank, mass;
};

__device__ inline int index_of(u64 rank) { return (1 << kIndexBits) - 1 - (int)(rank & ((1 << kIndexBits) - 1)); }

// What a workgroup of BS threads keeps in LDS to find a cut: List, the most tokens that are listed.
template <int BS, int Bins, int List = BS>
struct CutScratch {
    static constexpr int kThreads = BS, kBins = Bins, kCounted = BS / 4;
    u64 mass[Bins];                  // (count, weight) of a bin in one word; then running weight
    unsigned count[Bins];            // running count of tokens
    u64 list[List], list_mass[BS];   // rank words, falling once sorted; running weight
    unsigned list_w[List];           // weight
    u64 wave_mass[BS / 64];
    unsigned wave_count[BS / 64];
    u64 digit_mass[256];
    unsigned digit_count[256];
    u64 digit_at[4];                 // tokens and weight before the digit reached, its weight, its tokens
    unsigned differ[2];
    int n[2], bin[2], found[2];      // by count, by weight: tokens listed, bin reached, place in the list
    int digit;

    // before the barrier that precedes everything below
    __device__ void clear() {
        for (int i = threadIdx.x; i < Bins; i += BS) mass[i] = 0, count[i] = 0;
        if (threadIdx.x < 2) n[threadIdx.x] = 0, bin[threadIdx.x] = -1;
    }
    __device__ u64 mass_to(int b) const { return b < 0 ? 0 : mass[b]; }
    __device__ unsigned count_to(int b) const { return b < 0 ? 0 : count[b]; }

    // a running sum over the threads: what lies before this one's, from its wave's inclusive sum
    __device__ u64 before(u64 inclusive, u64 own) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 63) wave_mass[wave] = inclusive;
        __syncthreads();
        u64 v = inclusive - own;
#pragma unroll
        for (int w = 0; w < BS / 64; ++w)
            if (w < wave) v += wave_mass[w];
        return v;
    }

    // Running sums of m, c, Bins / BS a thread (bin tid Bins / BS + i), into mass and count.
    __device__ void scan(u64 (&m)[Bins / BS], unsigned (&c)[Bins / BS]) {
        constexpr int kPer = Bins / BS;
        const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
#pragma unroll
        for (int i = 1; i < kPer; ++i) m[i] += m[i - 1], c[i] += c[i - 1];
        const unsigned ic = wave_scan(c[kPer - 1]);
        if (lane == 63) wave_count[wave] = ic;
        const u64 bm = before(wave_scan(m[kPer - 1]), m[kPer - 1]);
        unsigned bc = ic - c[kPer - 1];
#pragma unroll
        for (int w = 0; w < BS / 64; ++w)
            if (w < wave) bc += wave_count[w];
#pragma unroll
        for (int i = 0; i < kPer; ++i) mass[tid * kPer + i] = bm + m[i], count[tid * kPer + i] = bc + c[i];
        __syncthreads();
    }

    // Running sums of count (in place) alone.
    __device__ void scan_counts() {
        constexpr int kPer = Bins / BS;
        const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
        unsigned c[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) c[i] = count[tid * kPer + i] + (i ? c[i - 1] : 0);
        const unsigned ic = wave_scan(c[kPer - 1]);
        if (lane == 63) wave_count[wave] = ic;
        __syncthreads();
        unsigned bc = ic - c[kPer - 1];
#pragma unroll
        for (int w = 0; w < BS / 64; ++w)
            if (w < wave) bc += wave_count[w];
#pragma unroll
        for (int i = 0; i < kPer; ++i) count[tid * kPer + i] = bc + c[i];
        __syncthreads();
    }

    // The bin in which the running count (kind 0) or weight (kind 1) reaches `want`; -1: never.  Once a kind.
    __device__ int reach(int kind, u64 want) {
        for (int i = threadIdx.x; i < Bins; i += BS) {
            const u64 here = kind ? mass[i] : count[i];
            const u64 prior = i == 0 ? 0 : kind ? mass[i - 1] : count[i - 1];
            if (prior < want && want <= here) bin[kind] = i;
        }
        __syncthreads();
        return bin[kind];
    }

    // list[0 .. n), n <= kCounted, into falling order, its weights and running weights: each word's place is the number of
    // larger ones, some lanes a word.
    __device__ void sort(int n_list, const RowRule &rule) {
        constexpr int kLanes = BS / kCounted;
        const int tid = threadIdx.x, j = tid / kLanes;
        const u64 v = j < n_list ? list[j] : 0;
        int larger = 0;
#pragma unroll 4
        for (int i = tid % kLanes; i < n_list; i += kLanes) larger += list[i] > v;
#pragma unroll
        for (int d = kLanes / 2; d; d >>= 1) larger += __shfl_xor(larger, d);
        __syncthreads();
        if (j < n_list && tid % kLanes == 0) list[larger] = v;
        __syncthreads();
        const u64 w = tid < n_list ? rule.weight(rule.logit_of(list[tid])) : 0;
        const u64 run = before(wave_scan(w), w) + w;
        if (tid < n_list) list_mass[tid] = run, list_w[tid] = (unsigned)w;
        __syncthreads();
    }

    // Weights of an unsorted list.
    __device__ void weigh(int n_list, const RowRule &rule) {
        for (int i = threadIdx.x; i < n_list; i += BS) list_w[i] = rule.weight(rule.logit_of(list[i]));
        __syncthreads();
    }

    // The place in the sorted list at which mass0 and its running weight reach `want`.
    __device__ int place(int n_list, u64 mass0, u64 want) {
        const int tid = threadIdx.x;
        if (tid < n_list && mass0 + list_mass[tid] >= want && (tid == 0 || mass0 + list_mass[tid - 1] < want)) found[1] = tid;
        __syncthreads();
        return found[1];
    }
};

// The token at which the count (kind 0) or the weight (kind 1) reaches `want`, among all that `each` gives (each(f) calls
// f(rank, weight) for this thread's ones; some has one of the ranks): eight bits of the rank words at a time, from the
// highest in which any two differ, until one token is left.
// Packed: at most 2^15 tokens, counts and weights in one word.
template <bool Packed = false, class Scratch, class Each>
__device__ inline Cut cut_by_digits(Scratch &s, int kind, u64 want, u64 some, Each each) {
    if (threadIdx.x < 2) s.differ[threadIdx.x] = 0;
    __syncthreads();
    {
        u64 d = 0;
        each([&](u64 r, unsigned) { d |= r ^ some; });
        const unsigned lo = (unsigned)d, hi = (unsigned)(d >> 32);
        if (lo) atomicOr(&s.differ[0], lo);
        if (hi) atomicOr(&s.differ[1], hi);
    }
    __syncthreads();
    const u64 differ = (u64)s.differ[1] << 32 | s.differ[0];
    // not yet known, from the lowest.  (Without a choice on differ == 0: the compiler makes it a scalar select on a condition
    // that it has in a vector compare's result.)
    int bits = 63 - __builtin_clzll(differ << 1 | 1);
    u64 prefix = some >> bits, c0 = 0, m0 = 0;       // rank words have at most 52 bits
    while (bits > 0) {
        const int width = min(bits, 8), shift = bits - width;
        for (int i = threadIdx.x; i < 256; i += Scratch::kThreads) {
            s.digit_mass[i] = 0;
            if (!Packed) s.digit_count[i] = 0;
        }
        __syncthreads();
        each([&](u64 r, unsigned w) {
            if (r >> bits == prefix) {
                const int d = (int)(r >> shift) & ((1 << width) - 1);
                if (!Packed) atomicAdd(&s.digit_count[d], 1u);
                atomicAdd(&s.digit_mass[d], Packed ? (1ull << kCountShift) | w : (u64)w);
            }
        });
        __syncthreads();
        if (threadIdx.x < 64) {
            // four digits a lane, the largest first
            u64 m[4];
            unsigned c[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 255 - (4 * threadIdx.x + i);
                m[i] = s.digit_mass[d] + (i ? m[i - 1] : 0);
                c[i] = Packed ? 0 : s.digit_count[d] + (i ? c[i - 1] : 0);
            }
            u64 bm = wave_scan(m[3]) - m[3], bc = 0;
            if (Packed) {
                bc = bm >> kCountShift, bm &= kMassMask;
#pragma unroll
                for (int i = 0; i < 4; ++i) c[i] = (unsigned)(m[i] >> kCountShift), m[i] &= kMassMask;
            } else {
                bc = wave_scan(c[3]) - c[3];
            }
            bm += m0, bc += c0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u64 pm = bm + (i ? m[i - 1] : 0), pc = bc + (i ? c[i - 1] : 0);
                if (kind ? pm < want && want <= bm + m[i] : pc < want && want <= bc + c[i]) {
                    s.digit = 255 - (4 * (int)threadIdx.x + i);
                    s.digit_at[0] = pc, s.digit_at[1] = pm, s.digit_at[2] = bm + m[i] - pm, s.digit_at[3] = bc + c[i] - pc;
                }
            }
        }
        __syncthreads();
        c0 = s.digit_at[0], m0 = s.digit_at[1], prefix = prefix << width | (unsigned)s.digit, bits = shift;
        if (s.digit_at[3] == 1) break;
        __syncthreads();
    }
    // the one token with this prefix
    each([&](u64 r, unsigned w) {
        if (r >> bits == prefix) s.digit_mass[0] = r, s.digit_mass[1] = w;
    });
    __syncthreads();
    const Cut cut{s.digit_mass[0], m0 + s.digit_mass[1]};
    __syncthreads();
    return cut;
}

// The same of an unsorted list with weights.
template <class Scratch>
__device__ inline Cut cut_in_list(Scratch &s, int n, int kind, u64 want) {
    return cut_by_digits<true>(s, kind, want, s.list[0], [&](auto f) {
        for (int i = threadIdx.x; i < n; i += Scratch::kThreads) f(s.list[i], s.list_w[i]);
    });
}

// The cut of a row whose bins are scanned.  list(kind, bin) lists a bin's tokens; each(f) and some are as above.
template <class Scratch, class List, class Each>
__device__ inline u64 find_cut(Scratch &s, const RowRule &rule, u64 some, List list, Each each) {
    // the token in bin b at which the count or the weight reaches `want`
    auto cut_at = [&](int kind, int b, u64 want) {
        const int n = s.count_to(b) - s.count_to(b - 1);
        if (n > Scratch::kThreads) return cut_by_digits(s, kind, want, some, each);
        list(kind, b);
        s.weigh(n, rule);
        const u64 c0 = s.count_to(b - 1), m0 = s.mass_to(b - 1);
        Cut c = cut_in_list(s, n, kind, want - (kind ? m0 : c0));
        c.mass += m0;
        return c;
    };
    u64 cut = 0, total = s.mass[Scratch::kBins - 1];
    if (rule.k_on) {
        const int b = s.reach(0, (u64)rule.k);
        if (b >= 0) {
            const Cut c = cut_at(0, b, (u64)rule.k);
            cut = c.rank, total = c.mass;
        }
    }
    if (rule.p_on) {
        u64 need = share(total, rule.p);
        need = need ? need : 1;              // the first token is kept whatever the share
        const u64 c = cut_at(1, s.reach(1, need), need).rank;
        cut = cut > c ? cut : c;
    }
    return cut;
}

// Sets a row's results.
__device__ inline void answer(const pk_sample_desc &a, int b, int token, unsigned w, u64 total, unsigned kept) {
    a.token[b] = token;
    if (a.prob) a.prob[b] = total ? (float)w / (float)total : 0.0f;
    if (a.kept) a.kept[b] = (int)kept;
}
__device__ inline u64 drawn(const pk_sample_desc &a, int b, u64 total) {
    const u64 u = part31(a.u[b]);
    return share(total, u > 0x7FFFFFFFull ? 0x7FFFFFFFull : u);
}

// The drawn token of the first `kept` of a sorted list, at most kCounted: each is compared with each.
template <class Scratch>
__device__ inline void answer_from_list(Scratch &s, const pk_sample_desc &a, int b, const RowRule &rule, int kept) {
    const int tid = threadIdx.x;
    const unsigned least = max(rule.least, 1u);
    if (tid < kept && s.list_w[tid] >= least && (tid == kept - 1 || s.list_w[tid + 1] < least)) s.found[0] = tid + 1;
    __syncthreads();
    kept = s.found[0];
    const u64 total = s.list_mass[kept - 1], t = drawn(a, b, total);
    int lanes = 64;
    while (lanes > 1 && kept * lanes > Scratch::kThreads) lanes >>= 1;
    const int j = tid / lanes;
    const int own = j < kept ? index_of(s.list[j]) : 0;
    u64 before = 0;
#pragma unroll 4
    for (int i = tid & (lanes - 1); i < kept; i += lanes) {
        const unsigned w = s.list_w[i];
        before += index_of(s.list[i]) < own ? w : 0;
    }
    for (int d = lanes >> 1; d; d >>= 1) before += __shfl_xor(before, d);
    if (j < kept && (tid & (lanes - 1)) == 0) {
        const unsigned w = s.list_w[j];
        if (before <= t && t < before + w) answer(a, b, index_of(s.list[j]), w, total, kept);
    }
}

// Sorts an unsorted list, n <= BS, whose first rule.k <= kCounted tokens are wanted; of more than kCounted those alone are
// kept.  Returns how many are.
template <class Scratch>
__device__ inline int shorten(Scratch &s, const RowRule &rule, int n) {
    if (n > Scratch::kCounted) {
        const int tid = threadIdx.x;
        s.weigh(n, rule);
        const Cut c = cut_in_list(s, n, 0, (u64)rule.k);
        const u64 v = tid < n ? s.list[tid] : 0;
        if (tid == 0) s.n[1] = 0;
        __syncthreads();
        if (v >= c.rank && tid < n) s.list[atomicAdd(&s.n[1], 1)] = v;
        __syncthreads();
        n = rule.k;
    }
    s.sort(n, rule);
    return n;
}

// A row on one workgroup, its tokens in registers: wave w has tokens (w n + e) 64 + lane, e < n <= E.  The logits are read
// once and the rest is a chain of barriers, so latency bounds it: one row of 8,193 logits with top-k and top-p 8.1 us, 512
// rows of 1,027 with filters of their own 11.5 us.
template <class T, int BS, int E>
__global__ __launch_bounds__(BS) void sample_row_kernel(pk_sample_desc a) {
    constexpr int kWaves = BS / 64, kBins = 1024;
    __shared__ CutScratch<BS, kBins> s;
    __shared__ float s_max[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), V = a.vocab, b = blockIdx.x;
    const auto *row = (const typename T::Raw *)a.logits + (int64_t)b * a.logits_row;
    const int n = (V + BS - 1) / BS, base = wave * n * 64 + lane, end = min((wave + 1) * n * 64, V);
    float x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = base + e * 64;
        x[e] = i < end ? logit<T>(row, i) : -INFINITY;
    }
    RowRule rule;
    rule.settings<T>(a, b);
    float top = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) top = fmaxf(top, x[e]);
    top = wave_max(top);
    if (lane == 0) s_max[wave] = top;
    s.clear();
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, s_max[w]);
    rule.top = top;
    if (top == -INFINITY) {
        if (tid == 0) answer(a, b, -1, 0, 0, 0);
        return;
    }
    // groups of four tokens a thread: the last one's may lie behind the row, as -inf
    auto tokens = [&](auto f) {
#pragma unroll
        for (int g = 0; g < E; g += 4)
            if (g < n)
#pragma unroll
                for (int e = g; e < g + 4; ++e) f(e);
    };
    if (rule.k_on && rule.k <= s.kCounted) {
        // Few by count: the bins only count, and only the listed tokens' weights are worked out.  64 rows of 8,193 logits by
        // a top_k of up to 200: 12.5 us, 14.5 with every token's weight; by top_p too 11.9, and 17.1.
        int bin[E];
        tokens([&](int e) {
            bin[e] = rule.distance(x[e]) > kWeighed ? rule.bin<kBins>(x[e]) : kBins;
            if (bin[e] < kBins) atomicAdd(&s.count[bin[e]], 1u);
        });
        __syncthreads();
        s.scan_counts();
        const int at = s.reach(0, (u64)rule.k), last = at < 0 ? kBins - 1 : at, listed = s.count[last];
        if (listed <= BS) {
            tokens([&](int e) {
                if (bin[e] <= last) s.list[atomicAdd(&s.n[0], 1)] = rule.rank(x[e], base + e * 64);
            });
            __syncthreads();
            const int left0 = shorten(s, rule, listed);
            int left = min(rule.k, left0);
            if (rule.p_on) {
                const u64 need = share(s.list_mass[left - 1], rule.p);
                left = s.place(left, 0, need ? need : 1) + 1;
            }
            answer_from_list(s, a, b, rule, left);
            return;
        }
        __syncthreads();
        s.clear();
        __syncthreads();
    }
    unsigned w[E];
    tokens([&](int e) { w[e] = rule.weight(x[e]); });
    u64 cut = 0;
    if (rule.k_on || rule.p_on) {
        int bin[E];
        tokens([&](int e) {
            bin[e] = w[e] ? rule.bin<kBins>(x[e]) : kBins;
            if (w[e]) atomicAdd(&s.mass[bin[e]], (1ull << kCountShift) | w[e]);
        });
        __syncthreads();
        constexpr int kPer = kBins / BS;
        u64 bm[kPer];
        unsigned bc[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const u64 both = s.mass[tid * kPer + i];
            bm[i] = both & kMassMask, bc[i] = (unsigned)(both >> kCountShift);
        }
        s.scan(bm, bc);
        auto each = [&](auto f) {            // seldom wanted: from memory again
            for (int i = tid; i < V; i += BS) {
                const float y = logit<T>(row, i);
                const unsigned wt = rule.weight(y);
                if (wt) f(rule.rank(y, i), wt);
            }
        };
        auto list = [&](int kind, int at) {
            tokens([&](int e) {
                if (bin[e] == at) s.list[atomicAdd(&s.n[kind], 1)] = rule.rank(x[e], base + e * 64);
            });
            __syncthreads();
        };
        cut = find_cut(s, rule, rule.rank(top, 0), list, each);
    }
    // kept weights; each wave's sum, then the token in the wave that the drawn weight falls to
    const float cut_x = cut ? rule.logit_of(cut) : -INFINITY;
    const int cut_i = cut ? index_of(cut) : 0;
    u64 mass = 0;
    unsigned kept = 0;
    tokens([&](int e) {
        const bool in = w[e] && w[e] >= rule.least && (x[e] > cut_x || (x[e] == cut_x && base + e * 64 <= cut_i));
        w[e] = in ? w[e] : 0;
        mass += w[e], kept += in;
    });
    mass = wave_sum(mass), kept = wave_sum(kept);
    __syncthreads();                         // wave_mass may still be read
    if (lane == 0) s.wave_mass[wave] = mass, s.wave_count[wave] = kept;
    __syncthreads();
    u64 total = 0, lead = 0;
    unsigned all = 0;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
        if (v < wave) lead += s.wave_mass[v];
        total += s.wave_mass[v], all += s.wave_count[v];
    }
    const u64 t = drawn(a, b, total);
    if (lead > t || lead + mass <= t) return;
    u64 sum[E];
    tokens([&](int e) { sum[e] = wave_sum((u64)w[e]); });
    tokens([&](int e) {
        if (lead <= t && t < lead + sum[e]) {
            const u64 hit = __ballot(lead + wave_scan((u64)w[e]) > t);
            if (lane == __ffsll(hit) - 1) answer(a, b, base + e * 64, w[e], total, all);
        }
        lead += sum[e];
    });
}

// ---- rows too long for one workgroup's registers ----
//
// Three launches over chunks of rows: the largest logit of each chunk; the bins' sums of each chunk, which the row's last
// chunk to arrive adds up and names the bins to list from; the kept weight of each chunk's 16 runs with the listed
// tokens beside, from which the row's last chunk finds the cut, the run and the token.  A row is read three times (64 rows
// of 128,001 in bf16 past the L2 each time: 16 MB a launch).  One such row by top_p: 4.6 + 9.9 + 17.0 us under a profiler, 27 us
// one call after another; 64 rows each with its own filters 5.2 + 15.4 + 27.2 and 46 us.  The chain at a row's end bounds
// it: bins and lists that meet in memory, scans and digits, a barrier after each.  Two workgroups a unit (64 registers): 256
// rows 116 us, one with 128 registers 157; 64 rows 46.6 and 45.2.  A list of 4,096: at 1,024, 64 rows of 262,144 often had
// more than that in the bin of the cut and took 772 us, not 70.

constexpr int kSplitThreads = 1024, kSplitBins = 1024, kSplitCap = 4096, kRuns = kSplitThreads / 64, kMaxChunks = 32;

// What is listed of a row: the tokens of the bins first .. last, and of bin_k.
struct RowPick {
    int first, last, bin_k, n;
    u64 total, mass_first, mass_k;  // weight of the row; before first; before bin_k less what first .. last hold
    unsigned count_k, unused;       // tokens before bin_k, likewise
};

// Whether a row is cut by a count so small that its bins only count: weights are worked out for the listed tokens alone.
// (64 rows of 128,001 by top-k and top-p 54.9 us, 57.2 without; of 262,144 64.9 and 71.3.)
__device__ inline bool few_by_count(const RowRule &rule) { return rule.k_on && rule.k <= kSplitThreads / 4; }

struct SplitRows {
    float *chunk_max;               // [rows][chunks]
    u64 *hist;                      // [rows][chunks][kSplitBins] (count, weight)
    RowPick *pick;                  // [rows]
    u64 *run_mass;                  // [rows][chunks * kRuns]
    u64 *list_rank;                 // [rows][kSplitCap]
    unsigned *run_kept;
    int *arrived_hist, *arrived_pick, *listed;       // [rows], zero between calls
    int row0, chunks, per;          // first row of this launch; tokens of a run: 64 per
};

template <class V>
__device__ inline void put_shared(V *p, V v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <class V>
__device__ inline V get_shared(const V *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Whether this workgroup is the last of `of` to get here; what each had put_shared before is then seen by it.
__device__ inline bool last_to_arrive(int *counter, int of, int *s_flag) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
        *s_flag = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == of - 1;
        if (*s_flag) put_shared(counter, 0);
    }
    __syncthreads();
    return *s_flag;
}

// kBatch logits, step apart, from memory together: -inf at and behind `end`.
constexpr int kBatch = 8;
template <class T>
__device__ inline void load_batch(const typename T::Raw *row, int i, int step, int end, float (&x)[kBatch]) {
    typename T::Raw raw[kBatch];
#pragma unroll
    for (int e = 0; e < kBatch; ++e) raw[e] = row[min(i + e * step, end - 1)];
#pragma unroll
    for (int e = 0; e < kBatch; ++e) {
        x[e] = T::get(raw[e]);
        if (x[e] != x[e] || i + e * step >= end) x[e] = -INFINITY;
    }
}

template <class T>
__global__ __launch_bounds__(kSplitThreads) void sample_max_kernel(pk_sample_desc a, SplitRows w) {
    __shared__ float s_max[kRuns];
    const int tid = threadIdx.x, chunk = blockIdx.x % w.chunks, r = blockIdx.x / w.chunks;
    const auto *row = (const typename T::Raw *)a.logits + (int64_t)(w.row0 + r) * a.logits_row;
    const int size = w.per * kSplitThreads, i0 = chunk * size, i1 = min(i0 + size, a.vocab);
    float top = -INFINITY;
    for (int i = i0 + tid; i < i1; i += kBatch * kSplitThreads) {
        float x[kBatch];
        load_batch<T>(row, i, kSplitThreads, i1, x);
#pragma unroll
        for (int e = 0; e < kBatch; ++e) top = fmaxf(top, x[e]);
    }
    top = wave_max(top);
    if ((tid & 63) == 0) s_max[tid >> 6] = top;
    __syncthreads();
    if (tid < 64) {
        top = wave_max(s_max[tid % kRuns]);
        if (tid == 0) w.chunk_max[r * w.chunks + chunk] = top;
    }
}

__device__ inline float row_max(const SplitRows &w, int r) {
    float top = w.chunk_max[r * w.chunks];
    for (int c = 1; c < w.chunks; ++c) top = fmaxf(top, w.chunk_max[r * w.chunks + c]);
    return top;
}

template <class T>
__global__ __launch_bounds__(kSplitThreads, 8) void sample_hist_kernel(pk_sample_desc a, SplitRows w) {
    static_assert(kSplitBins == kSplitThreads, "a bin a thread");
    __shared__ CutScratch<kSplitThreads, kSplitBins> s;
    __shared__ int s_flag;
    const int tid = threadIdx.x, chunk = blockIdx.x % w.chunks, r = blockIdx.x / w.chunks;
    const auto *row = (const typename T::Raw *)a.logits + (int64_t)(w.row0 + r) * a.logits_row;
    const int size = w.per * kSplitThreads, i0 = chunk * size, i1 = min(i0 + size, a.vocab);
    float x[kBatch];
    load_batch<T>(row, i0 + tid, kSplitThreads, i1, x);       // on its way while the settings are read
    RowRule rule;
    rule.settings<T>(a, w.row0 + r);
    rule.top = row_max(w, r);
    s.clear();
    if ((!rule.k_on && !rule.p_on) || rule.top == -INFINITY) return;
    __syncthreads();
    const bool few = few_by_count(rule);
    for (int i = i0 + tid;;) {
        if (few) {
#pragma unroll
            for (int e = 0; e < kBatch; ++e)
                if (rule.distance(x[e]) > kWeighed) atomicAdd(&s.mass[rule.bin<kSplitBins>(x[e])], 1ull << kCountShift);
        } else {
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                const unsigned wt = rule.weight(x[e]);
                if (wt) atomicAdd(&s.mass[rule.bin<kSplitBins>(x[e])], (1ull << kCountShift) | wt);
            }
        }
        i += kBatch * kSplitThreads;
        if (i - tid >= i1) break;
        load_batch<T>(row, i, kSplitThreads, i1, x);
    }
    __syncthreads();
    u64 *hist = w.hist + (int64_t)r * w.chunks * kSplitBins;
    put_shared(&hist[(int64_t)chunk * kSplitBins + tid], s.mass[tid]);
    if (!last_to_arrive(&w.arrived_hist[r], w.chunks, &s_flag)) return;

    // two bins of every other chunk a thread, so that all loads are on their way together
    const int pair = tid & 511, half = tid >> 9;
    u64 m2[2] = {0, 0};
    unsigned c2[2] = {0, 0};
#pragma unroll 8
    for (int c = half; c < w.chunks; c += 2) {
        const u4 v = load_shared4((const unsigned *)hist, 2 * (c * kSplitBins + 2 * pair));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const u64 both = (u64)v[2 * i + 1] << 32 | v[2 * i];
            m2[i] += both & kMassMask, c2[i] += (unsigned)(both >> kCountShift);
        }
    }
    __syncthreads();
    if (half)
        for (int i = 0; i < 2; ++i) s.mass[2 * pair + i] = m2[i], s.count[2 * pair + i] = c2[i];
    __syncthreads();
    if (!half)
        for (int i = 0; i < 2; ++i) s.mass[2 * pair + i] += m2[i], s.count[2 * pair + i] += c2[i];
    __syncthreads();
    u64 mass[1] = {s.mass[tid]};
    unsigned count[1] = {s.count[tid]};
    s.scan(mass, count);
    auto mass_to = [&](int bin) { return s.mass_to(bin); };
    auto count_to = [&](int bin) { return s.count_to(bin); };
    RowPick p{kSplitBins, kSplitBins - 1, -1, 0, 0, 0, 0, 0, 0};
    if (few) {
        p.bin_k = s.reach(0, (u64)rule.k);
        p.first = 0, p.last = p.bin_k < 0 ? kSplitBins - 1 : p.bin_k;
        p.n = (int)count_to(p.last);
        if (tid == 0) w.pick[r] = p;
        return;
    }
    u64 low = s.mass[kSplitBins - 1], high = low;          // between which the kept total after top_k lies
    if (rule.k_on) {
        p.bin_k = s.reach(0, (u64)rule.k);
        if (p.bin_k >= 0) p.first = p.last = p.bin_k, low = mass_to(p.bin_k - 1), high = mass_to(p.bin_k);
    }
    if (rule.p_on) {
        const u64 need_low = share(low, rule.p), need_high = share(high, rule.p);
        const int b0 = s.reach(1, need_low ? need_low : 1);
        __syncthreads();                                    // b0 is read by all before it is written again
        const int b1 = s.reach(1, need_high ? need_high : 1);
        p.first = p.bin_k >= 0 ? min(b0, p.bin_k) : b0, p.last = p.bin_k >= 0 ? min(b1, p.bin_k) : b1;
    }
    if (tid == 0) {
        const unsigned ranged = count_to(p.last) - count_to(p.first - 1);
        const bool apart = p.bin_k > p.last;
        p.total = s.mass[kSplitBins - 1], p.mass_first = mass_to(p.first - 1);
        if (p.bin_k >= 0) {
            p.mass_k = mass_to(p.bin_k - 1) - (apart ? mass_to(p.last) - p.mass_first : 0);
            p.count_k = count_to(p.bin_k - 1) - (apart ? ranged : 0);
            if (!apart) p.mass_k = p.mass_first, p.count_k = count_to(p.first - 1);
        }
        p.n = (int)(ranged + (apart ? count_to(p.bin_k) - count_to(p.bin_k - 1) : 0));
        w.pick[r] = p;
    }
}

template <class T>
__global__ __launch_bounds__(kSplitThreads, 8) void sample_pick_kernel(pk_sample_desc a, SplitRows w) {
    __shared__ CutScratch<kSplitThreads, kSplitBins, kSplitCap> s;
    __shared__ u64 s_run[kMaxChunks * kRuns], s_row[kMaxChunks];
    __shared__ int s_flag, s_at;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int chunk = blockIdx.x % w.chunks, r = blockIdx.x / w.chunks, b = w.row0 + r, V = a.vocab, runs = w.chunks * kRuns;
    const auto *row = (const typename T::Raw *)a.logits + (int64_t)b * a.logits_row;
    const int run = chunk * kRuns + wave, run_size = 64 * w.per;
    const int from = run * run_size + lane, end = min((run + 1) * run_size, V);
    float x[kBatch];
    if (from - lane < end) load_batch<T>(row, from, 64, end, x);      // on its way while the settings are read
    RowPick p = w.pick[r];
    RowRule rule;
    rule.settings<T>(a, b);
    rule.top = row_max(w, r);
    if (rule.top == -INFINITY) {
        if (chunk == 0 && tid == 0) answer(a, b, -1, 0, 0, 0);
        return;
    }
    if (!rule.k_on && !rule.p_on) p = RowPick{kSplitBins, kSplitBins - 1, -1, 0, 0, 0, 0, 0, 0};
    const bool few = few_by_count(rule), crowded = p.n > (few ? kSplitThreads : kSplitCap);
    if (!crowded) {
        if (tid == 0) s.n[0] = 0;
        __syncthreads();
        // this wave's run: what lies in the bins before the listed ones is kept whatever the cut
        u64 mass = 0;
        unsigned kept = 0;
        for (int i0 = from; i0 - lane < end; i0 += 64 * kBatch) {
            if (i0 != from) load_batch<T>(row, i0, 64, end, x);
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                const int bin = rule.bin<kSplitBins>(x[e]);
                if (bin > p.last && bin != p.bin_k) continue;      // most tokens: no weight is worked out
                const unsigned wt = few ? rule.distance(x[e]) > kWeighed : rule.weight(x[e]);
                if (wt && bin < p.first) {
                    if (wt >= rule.least) mass += wt, ++kept;
                } else if (wt) {
                    const int at = atomicAdd(&s.n[0], 1);
                    if (at < kSplitCap) s.list[at] = rule.rank(x[e], i0 + e * 64);
                }
            }
        }
        mass = wave_sum(mass), kept = wave_sum(kept);
        if (lane == 0) put_shared(&w.run_mass[(int64_t)r * runs + run], mass), put_shared(&w.run_kept[(int64_t)r * runs + run], kept);
        // the chunk's listed tokens, behind those of the chunks that came before it
        __syncthreads();
        const int n = min(s.n[0], kSplitCap);
        if (tid == 0 && n) s_at = __hip_atomic_fetch_add(&w.listed[r], n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        for (int j = tid; j < n; j += kSplitThreads) {
            const int at = s_at + j;
            if (at < kSplitCap) put_shared(&w.list_rank[(int64_t)r * kSplitCap + at], s.list[j]);
        }
    }
    if (!last_to_arrive(&w.arrived_pick[r], w.chunks, &s_flag)) return;

    u64 cut = 0;
    unsigned kept = 0;
    if (!crowded) {
        const int n = p.n;
        for (int i = tid; i < n; i += kSplitThreads) s.list[i] = get_shared(&w.list_rank[(int64_t)r * kSplitCap + i]);
        if (tid < runs) {
            s_run[tid] = get_shared(&w.run_mass[(int64_t)r * runs + tid]);
            kept = get_shared(&w.run_kept[(int64_t)r * runs + tid]);
        }
        if (tid == 0) put_shared(&w.listed[r], 0);
        __syncthreads();
        if (n) {
            if (few || n <= s.kCounted) {
                const int sorted = few ? shorten(s, rule, n) : n;
                if (!few) s.sort(n, rule);
                u64 total = p.total;
                int left = sorted;                   // of the list
                if (p.bin_k >= 0) left = rule.k - (int)p.count_k;
                if (p.bin_k >= 0 || few) total = p.mass_k + s.list_mass[left - 1];
                if (rule.p_on) {
                    const u64 need = share(total, rule.p);
                    left = min(left, s.place(left, p.mass_first, need ? need : 1) + 1);
                }
                if (p.first == 0) {
                    answer_from_list(s, a, b, rule, left);
                    return;
                }
                cut = s.list[left - 1];
            } else {
                s.weigh(n, rule);
                u64 total = p.total;
                if (p.bin_k >= 0) {
                    const Cut c = cut_in_list(s, n, 0, (u64)rule.k - p.count_k);
                    cut = c.rank, total = p.mass_k + c.mass;
                }
                if (rule.p_on) {
                    const u64 need = share(total, rule.p);
                    const Cut c = cut_in_list(s, n, 1, (need ? need : 1) - p.mass_first);
                    cut = cut > c.rank ? cut : c.rank;
                }
            }
            for (int i = tid; i < n; i += kSplitThreads)
                if (s.list[i] >= cut && s.list_w[i] >= rule.least) {
                    atomicAdd(&s_run[index_of(s.list[i]) / run_size], (u64)s.list_w[i]);
                    ++kept;
                }
        }
    } else {
        // more tokens at the cut than the list holds: this workgroup goes over the row by itself, over the tokens that the
        // bins counted (a count by logits alone has some whose weight is none, so that it may reach k where weights do not)
        auto each = [&](auto f) {
            for (int i = tid; i < V; i += kSplitThreads) {
                const float x = logit<T>(row, i);
                const unsigned wt = rule.weight(x);
                if (few ? rule.distance(x) > kWeighed : wt != 0) f(rule.rank(x, i), wt);
            }
        };
        u64 total = p.total;
        if (p.bin_k >= 0) {
            const Cut c = cut_by_digits(s, 0, (u64)rule.k, rule.rank(rule.top, 0), each);
            cut = c.rank, total = c.mass;
        }
        if (rule.p_on) {
            const u64 need = share(total, rule.p);
            const Cut c = cut_by_digits(s, 1, need ? need : 1, rule.rank(rule.top, 0), each);
            cut = cut > c.rank ? cut : c.rank;
        }
        for (int q = wave; q < runs; q += kRuns) {
            u64 mass = 0;
            for (int e = 0; e < w.per; ++e) {
                const int i = q * run_size + e * 64 + lane;
                if (i >= V) break;
                const float x = logit<T>(row, i);
                const unsigned wt = rule.weight(x);
                if (wt && wt >= rule.least && rule.rank(x, i) >= cut) mass += wt, ++kept;
            }
            mass = wave_sum(mass);
            if (lane == 0) s_run[q] = mass;
        }
    }
    kept = wave_sum(kept);
    if (lane == 0) s.wave_count[wave] = kept;
    __syncthreads();
    // running sums over the runs (at most 512: the first waves), then the one in which the drawn weight falls
    {
        u64 m = tid < runs ? s_run[tid] : 0;
        const u64 im = wave_scan(m);
        if (lane == 63) s.wave_mass[wave] = im;
        __syncthreads();
        u64 before = im - m, total = 0;
        for (int v = 0; v < kRuns; ++v) {
            if (v < wave) before += s.wave_mass[v];
            total += s.wave_mass[v];
        }
        const u64 t = drawn(a, b, total);
        if (tid < runs && before <= t && t < before + m) s.bin[0] = tid, s.digit_at[0] = before;
        __syncthreads();
        const int q = s.bin[0];
        const u64 lead = s.digit_at[0];
        unsigned all = 0;
        for (int v = 0; v < kRuns; ++v) all += s.wave_count[v];
        // its rows of 64 tokens, two a wave at most
        unsigned wt[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int e = wave + h * kRuns, i = q * run_size + e * 64 + lane;
            wt[h] = 0;
            if (e < w.per && i < V) {
                const float x = logit<T>(row, i);
                const unsigned v = rule.weight(x);
                if (v && v >= rule.least && rule.rank(x, i) >= cut) wt[h] = v;
            }
            const u64 sum = wave_sum((u64)wt[h]);
            if (lane == 0 && e < w.per) s_row[e] = sum;
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int e = wave + h * kRuns;
            if (e >= w.per) break;
            u64 at = lead;
            for (int v = 0; v < e; ++v) at += s_row[v];
            if (at > t || at + s_row[e] <= t) continue;
            const u64 hit = __ballot(at + wave_scan((u64)wt[h]) > t);
            if (lane == __ffsll(hit) - 1) answer(a, b, q * run_size + e * 64 + lane, wt[h], total, all);
        }
    }
}

}  // namespace pklm
