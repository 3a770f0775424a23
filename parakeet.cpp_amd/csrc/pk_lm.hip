// pk_lm.hip -- language-model serving operators: host side + C ABI of parakeet_lm.h.
//
// Each entry point checks its descriptor, chooses a launch and enqueues it on the caller's stream.  The kernels are in
// lm_plan.h, lm_cache.h, lm_attend.h and lm_sample.h.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>

#include "last_error.h"
#include "lm_attend.h"
#include "lm_attend_host.h"
#include "lm_cache.h"
#include "lm_host.h"
#include "lm_plan.h"
#include "lm_sample.h"
#include "parakeet_lm.h"

namespace {

using namespace pklm;

bool page_ok(int page) { return page == 16 || page == 32 || page == 64 || page == 128 || page == 256; }

// What pk_kv4_store, _load and _attend ask of the cache; 0 = fine.
int check_cache(const char *what, const void *cache, int64_t page_stride, int page, int n_pages, int heads, int dim) {
    if (!page_ok(page)) return pk_fail(PK_ERR_UNSUPPORTED, "%s: pages of %d tokens (16, 32, 64, 128 or 256)", what, page);
    if (dim != 64 && dim != 128 && dim != 256)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128 or 256)", what, dim);
    if (heads <= 0 || n_pages <= 0) return pk_fail(PK_ERR_ARG, "%s: %d heads, %d pages", what, heads, n_pages);
    if ((int64_t)n_pages * page > INT32_MAX)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d pages of %d tokens: slots are 32 bits", what, n_pages, page);
    if (!cache || !aligned(cache, 16)) return pk_fail(PK_ERR_ARG, "%s: the cache is NULL or not aligned to 16 bytes", what);
    const Record rec{page, dim};
    if (page_stride % 16 || page_stride < heads * rec.bytes())
        return pk_fail(PK_ERR_ARG, "%s: page_stride %lld bytes (a multiple of 16, at least %lld)", what, (long long)page_stride,
                       (long long)(heads * rec.bytes()));
    return PK_OK;
}

// Several passes a thread where there are values for it: 24,577 rows of 8 heads x 128 in bf16 take 53.4 us, 54.8 in single
// passes, 40,000 rows 93.3 and 98.0; 8,192 rows 19.7 and 18.3, 24,577 of 2 heads x 64 in f32 15.9 and 14.5.
bool many_rows(const pk_kv4_rows_desc &d) { return (int64_t)d.n_rows * d.heads * d.head_dim >= 1 << 24; }
int64_t row_groups(const pk_kv4_rows_desc &d) {
    const int each = kRowThreads * 8 / d.head_dim * (many_rows(d) ? kRowPasses : 1);
    return ((int64_t)d.n_rows + each - 1) / each;
}

template <class T, int D, bool Store>
void launch_rows(const pk_kv4_rows_desc &d, int wide, hipStream_t s) {
    const bool many = many_rows(d);
    const dim3 grid((unsigned)row_groups(d), 2 * d.heads);
    if (many) rows_kernel<T, D, Store, kRowPasses><<<grid, kRowThreads, 0, s>>>(d, log2i(d.page), wide);
    else rows_kernel<T, D, Store, 1><<<grid, kRowThreads, 0, s>>>(d, log2i(d.page), wide);
}

template <class T, bool Store>
void launch_rows(const pk_kv4_rows_desc &d, int wide, hipStream_t s) {
    if (d.head_dim == 64) launch_rows<T, 64, Store>(d, wide, s);
    else if (d.head_dim == 128) launch_rows<T, 128, Store>(d, wide, s);
    else launch_rows<T, 256, Store>(d, wide, s);
}

template <bool Store>
int rows_call(const char *what, const pk_kv4_rows_desc *d, void *stream) {
    pk_fail_clear();
    if (!d) return pk_fail(PK_ERR_ARG, "%s: no descriptor", what);
    if (int rc = check_cache(what, d->cache, d->page_stride, d->page, d->n_pages, d->heads, d->head_dim)) return rc;
    if (d->n_rows < 0) return pk_fail(PK_ERR_ARG, "%s: %d rows", what, d->n_rows);
    if (d->n_rows == 0) return PK_OK;
    const int size = d->dtype == PK_DTYPE_F32 ? 4 : 2;
    if (d->dtype != PK_DTYPE_F32 && d->dtype != PK_DTYPE_F16 && d->dtype != PK_DTYPE_BF16)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: dtype %d", what, d->dtype);
    if (!d->k || !d->v || !d->slots) return pk_fail(PK_ERR_ARG, "%s: NULL rows or slots", what);
    if (!aligned(d->k, size) || !aligned(d->v, size) || !aligned(d->slots, 4))
        return pk_fail(PK_ERR_ARG, "%s: rows or slots not aligned to their type", what);
    if (d->heads > 32767) return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d heads (at most 32767)", what, d->heads);
    if (row_groups(*d) > most_groups(kRowThreads))
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d rows of %d channels in one call", what, d->n_rows, d->head_dim);
    const int per = 16 / size;
    const int wide = aligned(d->k, 16) && aligned(d->v, 16) && d->k_row % per == 0 && d->k_head % per == 0 &&
                     d->v_row % per == 0 && d->v_head % per == 0;
    const hipStream_t s = (hipStream_t)stream;
    if (d->dtype == PK_DTYPE_F32) launch_rows<F32, Store>(*d, wide, s);
    else if (d->dtype == PK_DTYPE_F16) launch_rows<F16, Store>(*d, wide, s);
    else launch_rows<BF16, Store>(*d, wide, s);
    return launched(what);
}

// Sampling.  A row of up to kRowVocab logits is one workgroup's, its tokens in registers, 16 a thread; longer rows are cut in
// chunks, in three launches.  Rows of 16,384 in f32 with filters, microseconds on one workgroup and in chunks: 1 row 9.8 and
// 18.4, 64 rows 21.6 and 23.8, 512 rows 48 and 96.
constexpr int kRowVocab = 16384, kSplitRowsMost = 512, kSplitGroups = 2048;

struct SampleShape {
    int per, chunks, rows;       // tokens a thread takes of a chunk, chunks of a row, rows of a launch
    // counters first, the same place for every shape: they are zero between calls
    static constexpr int64_t kCounterBytes = 3 * kSplitRowsMost * 4;
    int64_t max_at, hist_at, pick_at, run_mass_at, list_rank_at, run_kept_at, bytes;
};

SampleShape sample_shape(int rows, int vocab) {
    SampleShape s{};
    if (vocab <= kRowVocab) return s;
    // As many chunks a row as give each of the card's 256 units one, 2 to 16: more are slow to add up.  128,001 logits in
    // bf16, microseconds at 4, 8, 16 and 32 chunks: one row by top-p 43.8, 33.5, 28.3, 29.6; 8 rows 43.8, 33.4, 30.0,
    // 34.5; 64 rows each with its own filters 45.7, 46.3, 60.9, 95.8; 256 rows 115, 144, 206 at 4, 8 and 16.  256 rows of
    // 32,000 at 2 and 4: 43.1, 58.5.
    const int aim = std::min(std::max(256 / std::max(rows, 1), 2), 16);
    s.per = std::min(std::max((vocab + aim * kSplitThreads - 1) / (aim * kSplitThreads), 4), kMaxChunks);
    s.chunks = (vocab + s.per * kSplitThreads - 1) / (s.per * kSplitThreads);
    s.rows = std::min({rows, kSplitRowsMost, std::max(kSplitGroups / s.chunks, 1)});
    int64_t at = SampleShape::kCounterBytes;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const int64_t n = s.rows, runs = (int64_t)s.chunks * kRuns;
    s.max_at = take(n * s.chunks * 4);
    s.hist_at = take(n * s.chunks * kSplitBins * 8);
    s.pick_at = take(n * sizeof(RowPick));
    s.run_mass_at = take(n * runs * 8);
    s.list_rank_at = take(n * kSplitCap * 8);
    s.run_kept_at = take(n * runs * 4);
    s.bytes = at;
    return s;
}

// A workgroup of 256 or of 1,024 threads a row: the larger is quicker by itself, of the smaller four fit in its place.  Rows of
// 2,000 logits, microseconds: 256 rows 12.2 and 10.2, 384 rows 12.4 and 16.1; of 1,000: 64 rows 9.5 and 9.8, 512 rows
// 10.8 and 17.3; of 4,000: 64 rows 14.7 and 10.8, 512 rows 19.1 and 20.7 (without filters 12.2 and 10.9).
int row_threads(const pk_sample_desc &d) { return d.vocab <= 1024 || (d.vocab <= 2048 && d.rows > 256) ? 256 : 1024; }

template <class T>
void launch_sample(const pk_sample_desc &d, const SampleShape &sh, hipStream_t s) {
    const unsigned rows = (unsigned)d.rows;
    if (d.vocab <= 1024) sample_row_kernel<T, 256, 4><<<rows, 256, 0, s>>>(d);
    else if (row_threads(d) == 256) sample_row_kernel<T, 256, 8><<<rows, 256, 0, s>>>(d);
    else if (d.vocab <= 4096) sample_row_kernel<T, 1024, 4><<<rows, 1024, 0, s>>>(d);
    else if (d.vocab <= kRowVocab) sample_row_kernel<T, 1024, 16><<<rows, 1024, 0, s>>>(d);
    else {
        char *w = (char *)d.workspace;
        SplitRows p;
        p.arrived_hist = (int *)w, p.arrived_pick = p.arrived_hist + kSplitRowsMost, p.listed = p.arrived_pick + kSplitRowsMost;
        p.chunk_max = (float *)(w + sh.max_at), p.hist = (u64 *)(w + sh.hist_at), p.pick = (RowPick *)(w + sh.pick_at);
        p.run_mass = (u64 *)(w + sh.run_mass_at), p.list_rank = (u64 *)(w + sh.list_rank_at);
        p.run_kept = (unsigned *)(w + sh.run_kept_at);
        p.chunks = sh.chunks, p.per = sh.per;
        for (p.row0 = 0; p.row0 < d.rows; p.row0 += sh.rows) {
            const unsigned grid = (unsigned)(std::min(sh.rows, d.rows - p.row0) * sh.chunks);
            sample_max_kernel<T><<<grid, kSplitThreads, 0, s>>>(d, p);
            if (d.temperature || d.top_k || d.top_p) sample_hist_kernel<T><<<grid, kSplitThreads, 0, s>>>(d, p);
            sample_pick_kernel<T><<<grid, kSplitThreads, 0, s>>>(d, p);
        }
    }
}

// attend_prompt_kernel takes calls of more than kPromptRows query rows to a request and kv head that give it kPromptGroups
// workgroups or more, which the card holds at a time; attend_kernel splits long axes and takes the others.  The host has
// bounds alone: where requests stay below them, workgroups stay empty and the others' keys make a tail.  32 heads on 8 of 128
// channels in bf16, requests x new tokens on up to 8,191 keys, microseconds of the prompt kernel and of the other:
//   workgroups             256                           512                                      1,024
//   requests all alike     2 x 512: 226, 231             4 x 512: 278, 462; 16 x 128: 307, 512
//   lengths spread evenly  4 x 256: 225, 132             4 x 512: 244, 224; 16 x 128: 233, 186    4 x 1,024: 314, 400
//   one request            1 x 1,024: 224, 223           1 x 2,048: 269, 412                      1 x 4,096: 435, 709
//   without keys held      4 x 256: 18, 21               4 x 512: 25, 42; 16 x 128: 17, 31
// f16 at 512, 16 x 128: alike 486, 660; spread, on 6,000 keys 264, 175.  bf16 rows of 256 channels at 512, 4 x 512: alike 803,
// 952; spread, on 6,000 keys 399, 365.  So 512 costs up to half where lengths are spread on long axes, and a higher
// bound would cost as much or more where they are not.  64 requests of spread lengths on up to 2,047 keys: 64 rows each 69
// and 43, 96 rows 69 and 55, 128 rows 70 and 70.  Not f16 rows of 256, which its registers do not hold: two requests of up
// to 1,024 new tokens, 24 heads on 8 (384), 314 and 240 on up to 2,047 keys, 1,067 and 602 on 6,000.
constexpr int kPromptRows = 128, kPromptGroups = 512;

struct HostKv4 {
    static int check(const char *what, const void *cache, int64_t page_stride, int page, int n_pages, int heads, int dim) {
        return check_cache(what, cache, page_stride, page, n_pages, heads, dim);
    }
    static bool prompt(const pk_kv4_attend_desc &d, int64_t rows, int64_t groups) {
        return rows > kPromptRows && groups >= kPromptGroups && !(d.dtype == PK_DTYPE_F16 && d.head_dim == 256);
    }
    static int tile_cols(int64_t, int) { return 16; }
};

template <class T, int D>
void launch_attend(const AttendParams &p, bool prompt, unsigned grid, hipStream_t s) {
    // pages of whole key tiles: addresses are worked out a wave at a time.  A prompt of 512 tokens x 4 on up to 8,191 keys
    // takes 431 us with f16 rows of 128 then, 443 otherwise; of D = 256, whose registers are full, 664 and 526.
    if constexpr (D == 256 && __is_same(T, BF16)) {
        if (prompt) return attend_prompt_kernel<T, D, true><<<grid, kPromptThreads, 0, s>>>(p);
    } else if constexpr (D < 256) {
        if (prompt && p.page < kPromptKeys) return attend_prompt_kernel<T, D, true><<<grid, kPromptThreads, 0, s>>>(p);
        if (prompt) return attend_prompt_kernel<T, D, false><<<grid, kPromptThreads, 0, s>>>(p);
    }
    if (p.page < 32) attend_kernel<T, D, true><<<grid, kAttendThreads, 0, s>>>(p);
    else attend_kernel<T, D, false><<<grid, kAttendThreads, 0, s>>>(p);
}

template <class T>
void launch_attend(const AttendParams &p, bool prompt, int dim, unsigned grid, hipStream_t s) {
    if (dim == 64) launch_attend<T, 64>(p, prompt, grid, s);
    else if (dim == 128) launch_attend<T, 128>(p, prompt, grid, s);
    else launch_attend<T, 256>(p, prompt, grid, s);
}

}  // namespace

extern "C" {

PK_API int pk_kv_plan(const pk_kv_plan_desc *d, void *stream) {
    pk_fail_clear();
    const char *what = "pk_kv_plan";
    if (!d) return pk_fail(PK_ERR_ARG, "%s: no descriptor", what);
    if (d->requests < 0 || d->requests > PK_LM_MAX_REQUESTS)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d requests (at most %d)", what, d->requests, PK_LM_MAX_REQUESTS);
    if (!page_ok(d->page)) return pk_fail(PK_ERR_UNSUPPORTED, "%s: pages of %d tokens (16, 32, 64, 128 or 256)", what, d->page);
    if (d->width <= 0 || d->n_pages <= 0 || d->n_tokens < 0)
        return pk_fail(PK_ERR_ARG, "%s: table width %d, %d pages, %d tokens", what, d->width, d->n_pages, d->n_tokens);
    if ((int64_t)d->n_pages * d->page > INT32_MAX || (int64_t)std::max(d->requests, 1) * d->width * d->page > INT32_MAX)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d requests x %d pages, %d pages of %d tokens: positions and slots are 32 bits", what, d->requests,
                       d->width, d->n_pages, d->page);
    if (!d->ring || !d->state || !d->state_out || !d->first || (d->n_tokens && !d->slots) ||
        (d->requests && (!d->old_len || !d->new_len || !d->table || !d->lens || !d->ok)))
        return pk_fail(PK_ERR_ARG, "%s: NULL array", what);
    if (d->requests > 1 && d->table_stride < d->width)
        return pk_fail(PK_ERR_ARG, "%s: table rows %lld apart, %d wide", what, (long long)d->table_stride, d->width);
    if (d->state == d->state_out || d->lens == d->old_len || d->lens == d->new_len)
        return pk_fail(PK_ERR_ARG, "%s: state_out and lens are written while state and the lengths are read", what);
    const int wide = aligned(d->slots, 16) && aligned(d->pos, 16);
    const int64_t per = kPlanThreads * kPlanTokens;
    const unsigned grid = (unsigned)std::min<int64_t>(std::max<int64_t>((d->n_tokens + per - 1) / per, 1), 512);
    plan_kernel<<<grid, kPlanThreads, 0, (hipStream_t)stream>>>(*d, log2i(d->page), wide);
    return launched(what);
}

PK_API int pk_kv4_store(const pk_kv4_rows_desc *d, void *stream) { return rows_call<true>("pk_kv4_store", d, stream); }
PK_API int pk_kv4_load(const pk_kv4_rows_desc *d, void *stream) { return rows_call<false>("pk_kv4_load", d, stream); }

PK_API int pk_kv4_attend_workspace(const pk_kv4_attend_desc *d, int64_t *bytes) {
    return attend_workspace<HostKv4>("pk_kv4_attend", d, bytes);
}

PK_API int pk_kv4_attend(const pk_kv4_attend_desc *d, void *stream) {
    return attend_call<HostKv4>("pk_kv4_attend", d, [&](const AttendParams &p, const AttendShape &s, unsigned grid) {
        if (d->dtype == PK_DTYPE_F16) launch_attend<F16>(p, s.prompt, d->head_dim, grid, (hipStream_t)stream);
        else launch_attend<BF16>(p, s.prompt, d->head_dim, grid, (hipStream_t)stream);
    });
}

static int sample_check(const char *what, const pk_sample_desc *d) {
    if (!d) return pk_fail(PK_ERR_ARG, "%s: no descriptor", what);
    if (d->rows < 0 || d->vocab <= 0 || d->vocab > PK_LM_MAX_VOCAB)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d rows of %d logits (1 .. %d)", what, d->rows, d->vocab, PK_LM_MAX_VOCAB);
    return PK_OK;
}

PK_API int pk_sample_workspace(const pk_sample_desc *d, int64_t *bytes) {
    pk_fail_clear();
    if (int rc = sample_check("pk_sample_workspace", d)) return rc;
    if (!bytes) return pk_fail(PK_ERR_ARG, "pk_sample_workspace: NULL result");
    *bytes = sample_shape(d->rows, d->vocab).bytes;
    return PK_OK;
}

PK_API int pk_sample(const pk_sample_desc *d, void *stream) {
    pk_fail_clear();
    const char *what = "pk_sample";
    if (int rc = sample_check(what, d)) return rc;
    if (d->rows == 0) return PK_OK;
    if (!d->logits || !d->u || !d->token) return pk_fail(PK_ERR_ARG, "%s: NULL array", what);
    if (d->dtype != PK_DTYPE_F32 && d->dtype != PK_DTYPE_F16 && d->dtype != PK_DTYPE_BF16)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: dtype %d", what, d->dtype);
    if (!aligned(d->logits, d->dtype == PK_DTYPE_F32 ? 4 : 2)) return pk_fail(PK_ERR_ARG, "%s: logits not aligned to their type", what);
    if (d->vocab <= kRowVocab && d->rows > most_groups(row_threads(*d)))
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d rows of %d logits in one call", what, d->rows, d->vocab);
    const SampleShape sh = sample_shape(d->rows, d->vocab);
    if (sh.bytes > 0 && (!d->workspace || !aligned(d->workspace, 16) || d->workspace_bytes < sh.bytes))
        return pk_fail(PK_ERR_ARG, "%s: a workspace of %lld bytes is wanted, aligned to 16 (%lld given)", what, (long long)sh.bytes,
                       (long long)(d->workspace ? d->workspace_bytes : 0));
    const hipStream_t s = (hipStream_t)stream;
    if (d->dtype == PK_DTYPE_F32) launch_sample<F32>(*d, sh, s);
    else if (d->dtype == PK_DTYPE_F16) launch_sample<F16>(*d, sh, s);
    else launch_sample<BF16>(*d, sh, s);
    return launched(what);
}

}  // extern "C"
