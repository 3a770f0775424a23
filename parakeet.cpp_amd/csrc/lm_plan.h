// lm_plan.h -- page tables and slot maps from request lengths (pk_kv_plan).
#pragma once

#include "lm_common.h"
#include "parakeet_lm.h"

namespace pklm {

constexpr int kPlanThreads = 256;
constexpr int kPlanTokens = 4;   // consecutive tokens of one thread: one 16-byte store for each map

// Three running sums over the requests: new tokens (where a token's request is found), pages lacked (where its page
// is in the ring), pages given up (where they go behind the ring's end).  Every workgroup makes all three in its LDS
// from the two length arrays, at most 32 KB of reads, so that nothing is exchanged between workgroups and one launch
// does it all; each then takes its share of the tokens and of the pages given up.  Latency alone counts: lengths are read
// once, and a thread's four tokens, mostly of one request, take their pages in two loads together.  One request with one new
// token: 3.0 us, which is a launch and four loads that wait for each other.  512 requests of up to 8,191 tokens, 254,000
// slots and positions (2.2 MB): 7.8 us, most of it the three sums.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(pk_kv_plan_desc a, int shift, int wide) {
    __shared__ int s_first[PK_LM_MAX_REQUESTS + 1], s_lack[PK_LM_MAX_REQUESTS + 1], s_free[PK_LM_MAX_REQUESTS + 1];
    __shared__ int s_old[PK_LM_MAX_REQUESTS], s_new[PK_LM_MAX_REQUESTS];
    __shared__ int s_wave[3][kPlanThreads / 64], s_used;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int B = a.requests, page = 1 << shift, most = a.width << shift;
    auto pages = [&](int n) { return (n + page - 1) >> shift; };
    for (int b = tid; b < B; b += kPlanThreads) s_old[b] = a.old_len[b], s_new[b] = a.new_len[b];
    const int count = min(max(a.state[1], 0), a.n_pages);
    int head = a.state[0] % a.n_pages;
    if (head < 0) head += a.n_pages;
    if (tid == 0) s_used = 0;
    if (tid == 0 && B == 0) s_first[0] = s_free[0] = 0;   // no thread below has a last request
    __syncthreads();

    // this thread's run of requests, their sums, and what lies before them
    const int per = (B + kPlanThreads - 1) / kPlanThreads, b0 = min(tid * per, B), b1 = min(b0 + per, B);
    int tokens = 0, lack = 0;
    for (int b = b0; b < b1; ++b) {
        const int o = s_old[b], n = s_new[b];
        if (o < 0 || n < 0 || o > most || n > most) continue;
        tokens += max(n - o, 0);
        lack += max(pages(n) - pages(o), 0);
    }
    const int st = wave_scan(tokens), sl = wave_scan(lack);
    if (lane == 63) s_wave[0][wave] = st, s_wave[1][wave] = sl;
    __syncthreads();
    int at = st - tokens, al = sl - lack, freed = 0, used = 0;
    for (int w = 0; w < wave; ++w) at += s_wave[0][w], al += s_wave[1][w];
    for (int b = b0; b < b1; ++b) {
        const int o = s_old[b], n = s_new[b];
        const bool ranged = !(o < 0 || n < 0 || o > most || n > most);
        const int had = ranged ? pages(o) : 0, want = ranged ? pages(n) : 0;
        const int need = max(want - had, 0);
        const bool ok = ranged && (need == 0 || al + need <= count);
        s_first[b] = at;
        s_lack[b] = ok ? al : -1;                       // -1: not served
        if (ranged) at += max(n - o, 0);
        al += need;
        if (ok && need) used = al;
        s_free[b] = ok ? max(had - want, 0) : 0;
        freed += s_free[b];
        if (blockIdx.x == 0) {
            a.ok[b] = ok;
            a.lens[b] = ok ? n : o;
            a.first[b] = s_first[b];
        }
    }
    const int sf = wave_scan(freed);
    if (lane == 63) s_wave[2][wave] = sf;
    if (used) atomicMax(&s_used, used);
    if (b0 < b1 && b1 == B) s_first[B] = at;
    __syncthreads();
    int af = sf - freed;
    for (int w = 0; w < wave; ++w) af += s_wave[2][w];
    for (int b = b0; b < b1; ++b) {
        const int f = s_free[b];
        s_free[b] = af;
        af += f;
    }
    if (b0 < b1 && b1 == B) s_free[B] = af;
    __syncthreads();
    const int total = s_first[B], gone = s_free[B];
    if (blockIdx.x == 0 && tid == 0) {
        a.first[B] = total;
        a.state_out[0] = (head + s_used) % a.n_pages;
        a.state_out[1] = min(count - s_used + gone, a.n_pages);
    }

    // A slot, -1 where the id is no page: negative, or so large that its slots are past 32 bits and would wrap to others.
    auto slot_at = [&](int id, int q) {
        return (unsigned)id <= (unsigned)INT32_MAX >> shift ? (id << shift) + (q & (page - 1)) : -1;
    };
    // page j of request b, which holds `had` pages and takes new ones from place `al` of the ring on
    auto page_at = [&](int b, int j, int had, int al_b) {
        const int64_t place = (int64_t)head + al_b + (j - had);
        const int *p = j < had ? a.table + b * a.table_stride + j : a.ring + (place >= a.n_pages ? place - a.n_pages : place);
        return *p;
    };
    const int64_t stride = (int64_t)gridDim.x * kPlanThreads, me = (int64_t)blockIdx.x * kPlanThreads + tid;
    for (int64_t t0 = me * kPlanTokens; t0 < max(total, a.n_tokens); t0 += stride * kPlanTokens) {
        v4i slot = {-1, -1, -1, -1}, pos = {-1, -1, -1, -1};
        if (t0 < total) {
            int b = 0, hi = B;                          // the last request that begins at or before t0
            while (hi - b > 1) {
                const int mid = (b + hi) >> 1;
                if (s_first[mid] <= t0) b = mid; else hi = mid;
            }
            if (t0 + kPlanTokens <= s_first[b + 1]) {
                const int al_b = s_lack[b];
                if (al_b >= 0) {
                    const int o = s_old[b], p = o + (int)(t0 - s_first[b]), had = pages(o);
                    const int j0 = p >> shift, j1 = (p + kPlanTokens - 1) >> shift;
                    const int id0 = page_at(b, j0, had, al_b), id1 = page_at(b, j1, had, al_b);
#pragma unroll
                    for (int i = 0; i < kPlanTokens; ++i) {
                        const int q = p + i, id = q >> shift == j0 ? id0 : id1;
                        slot[i] = slot_at(id, q);
                        pos[i] = q;
                        // a new page's first token is new: it enters the page into the table
                        if ((q & (page - 1)) == 0) a.table[b * a.table_stride + (q >> shift)] = id;
                    }
                }
            } else {
                for (int i = 0; i < kPlanTokens; ++i) {
                    const int64_t t = t0 + i;
                    if (t >= total) break;
                    while (t >= s_first[b + 1]) ++b;
                    const int al_b = s_lack[b];
                    if (al_b < 0) continue;
                    const int o = s_old[b], q = o + (int)(t - s_first[b]);
                    const int id = page_at(b, q >> shift, pages(o), al_b);
                    slot[i] = slot_at(id, q);
                    pos[i] = q;
                    if ((q & (page - 1)) == 0) a.table[b * a.table_stride + (q >> shift)] = id;
                }
            }
        }
        if (t0 + kPlanTokens <= a.n_tokens && wide) {
            *(v4i *)(a.slots + t0) = slot;
            if (a.pos) *(v4i *)(a.pos + t0) = pos;
        } else {
#pragma unroll
            for (int i = 0; i < kPlanTokens; ++i)
                if (t0 + i < a.n_tokens) {
                    a.slots[t0 + i] = slot[i];
                    if (a.pos) a.pos[t0 + i] = pos[i];
                }
        }
    }
    for (int64_t f = me; f < gone; f += stride) {       // pages given up, in the order of the requests
        int b = 0, hi = B;
        while (hi - b > 1) {
            const int mid = (b + hi) >> 1;
            if (s_free[mid] <= f) b = mid; else hi = mid;
        }
        if (count + f >= a.n_pages) continue;           // a ring that says it holds more than there are
        const int r = (int)(((int64_t)head + count + f) % a.n_pages);
        a.ring[r] = a.table[b * a.table_stride + pages(s_new[b]) + (f - s_free[b])];
    }
}

}  // namespace pklm
