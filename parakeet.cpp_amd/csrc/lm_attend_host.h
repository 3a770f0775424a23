// lm_attend_host.h -- host side of attention over a paged cache (pk_kv4_attend, pk_kv8_attend): checks, the choice of kernel and
// how a call's work is dealt out.  C is the cache's kind, as in lm_attend.h, with what the host asks of it:
//   check(...)            of a call's cache
//   prompt(call, rows, groups)   whether its kernel for prompts takes a call of `rows` to a request and kv head, in so many workgroups
//   tile_cols(rows, D)    query rows of the other kernel's workgroup, of `rows` of a request and kv head
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "lm_attend.h"
#include "lm_host.h"

namespace pklm {

// Arrival counters of the tiles whose keys are split, at the workspace's beginning whatever the call's shape, so that
// no call's partial sums lie where another's counters are.  A split call has at most kSplitWork tiles times splits, and
// a tile 1 + (splits + 15) / 16 counters.
constexpr int kSplitWork = 512, kCounters = 4 * kSplitWork;
// How a call's work is dealt out, from its host-known sizes alone.
struct AttendShape {
    bool prompt;             // the kernel for prompts; else the one that splits a long axis
    int cols;                // query rows a workgroup
    int tiles, chunk, splits, groups;
    int64_t part_bytes;
    int64_t bytes() const { return splits > 1 ? kCounters * 4 + part_bytes : 0; }
};

template <class C>
int attend_shape(const char *what, const pk_kv4_attend_desc &d, AttendShape &s) {
    const int64_t rows = (int64_t)d.max_new * (d.heads / d.kv_heads), pairs = (int64_t)d.requests * d.kv_heads;
    const int64_t prompt_tiles = (rows + kPromptCols - 1) / kPromptCols;
    auto too_many = [&] {
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: %lld requests x kv heads of %lld query rows in one call", what, (long long)pairs,
                       (long long)rows);
    };
    if (pairs > most_groups(kPromptThreads)) return too_many();
    s.prompt = C::prompt(d, rows, pairs * prompt_tiles);
    s.cols = s.prompt ? kPromptCols : C::tile_cols(rows, d.head_dim);
    const int64_t tiles = (rows + s.cols - 1) / s.cols, step = 32 * kAttendWaves;
    // keys of one tile: its rows span at most as many tokens
    const int64_t keys = d.window ? std::min<int64_t>(d.max_len, (int64_t)d.window + s.cols + 64) : d.max_len;
    // Split where the tiles leave the card short of work (512 workgroups are resident), into no less than 512 keys.
    // 200,003 and 100,001 keys on 2 kv heads, 64 sessions of up to 4,097 keys on 8, 8 of up to 32,000: 29.5, 35.8 and 40.6
    // us; for twice as many splits 34.3, 37.2 and 43.3, for half as many 29.3, 36.1 and 46.0.
    const int64_t want = kSplitWork, least = 512, each = std::max<int64_t>(pairs * tiles, 1);
    int64_t splits = s.prompt ? 1 : std::max<int64_t>(std::min<int64_t>(want / each, (keys + least - 1) / least), 1);
    const int64_t chunk = std::max<int64_t>(((keys + splits - 1) / splits + step - 1) / step * step, step);
    splits = std::max<int64_t>((keys + chunk - 1) / chunk, 1);
    if (pairs * tiles * splits > most_groups(s.prompt ? kPromptThreads : kAttendThreads)) return too_many();
    // a tile's partial sums are reached by 32-bit byte offsets
    static_assert((kSplitWork + (kSplitWork + kJoin - 1) / kJoin) * 32 * (256 + 4) * 4ll < 1ll << 31, "at most kSplitWork splits");
    s.tiles = (int)tiles, s.chunk = (int)chunk, s.splits = (int)splits;
    s.groups = (int)((splits + kJoin - 1) / kJoin);
    s.part_bytes = pairs * tiles * (splits + s.groups) * s.cols * (d.head_dim + 4) * 4;
    return PK_OK;
}

inline int attend_check(const char *what, const pk_kv4_attend_desc *d) {
    if (!d) return pk_fail(PK_ERR_ARG, "%s: no descriptor", what);
    if (d->dtype != PK_DTYPE_F16 && d->dtype != PK_DTYPE_BF16) return pk_fail(PK_ERR_UNSUPPORTED, "%s: dtype %d (f16 or bf16)", what, d->dtype);
    if (d->heads <= 0 || d->kv_heads <= 0 || d->heads % d->kv_heads)
        return pk_fail(PK_ERR_ARG, "%s: %d query heads on %d kv heads", what, d->heads, d->kv_heads);
    if (d->requests < 0 || d->n_rows < 0 || d->max_new < 0 || d->max_len < 0 || d->window < 0 || d->width <= 0)
        return pk_fail(PK_ERR_ARG, "%s: %d requests, %d rows, max_new %d, max_len %d, window %d, table width %d", what, d->requests, d->n_rows,
                       d->max_new, d->max_len, d->window, d->width);
    if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128 or 256)", what, d->head_dim);
    if (!std::isfinite(d->scale)) return pk_fail(PK_ERR_ARG, "%s: a scale of %g", what, d->scale);
    if ((int64_t)std::max(d->n_rows, d->max_new) * (d->heads / d->kv_heads) > INT32_MAX - 4096)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d rows, max_new %d, %d query heads a kv head: row numbers are 32 bits", what, d->n_rows, d->max_new,
                       d->heads / d->kv_heads);
    // positions are 32 bits, some steps past the last key included
    if ((int64_t)d->width * d->page > INT32_MAX - 4096 || d->max_len > INT32_MAX - 4096)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: a table of %d pages of %d tokens, max_len %d: positions are 32 bits", what, d->width, d->page,
                       d->max_len);
    return PK_OK;
}

template <class C>
int attend_workspace(const char *what, const pk_kv4_attend_desc *d, int64_t *bytes) {
    pk_fail_clear();
    if (int rc = attend_check(what, d)) return rc;
    if (!bytes) return pk_fail(PK_ERR_ARG, "%s_workspace: NULL result", what);
    AttendShape s;
    if (int rc = attend_shape<C>(what, *d, s)) return rc;
    *bytes = s.bytes();
    return PK_OK;
}

template <class C, class Launch>
int attend_call(const char *what, const pk_kv4_attend_desc *d, Launch launch) {
    pk_fail_clear();
    if (int rc = attend_check(what, d)) return rc;
    if (int rc = C::check(what, d->cache, d->page_stride, d->page, d->n_pages, d->kv_heads, d->head_dim)) return rc;
    if (d->n_rows == 0 || d->requests == 0 || d->max_new == 0) return PK_OK;
    if (!d->q || !d->out || !d->table || !d->lens) return pk_fail(PK_ERR_ARG, "%s: NULL array", what);
    if (!aligned(d->q, 2) || !aligned(d->out, 2) || !aligned(d->lse, 4))
        return pk_fail(PK_ERR_ARG, "%s: q, out or lse not aligned to its type", what);
    if (!d->first && (d->n_rows != d->requests || d->max_new != 1))
        return pk_fail(PK_ERR_ARG, "%s: without first, one query per request: %d rows, %d requests, max_new %d", what, d->n_rows, d->requests, d->max_new);
    if (d->requests > 1 && d->table_stride < d->width)
        return pk_fail(PK_ERR_ARG, "%s: table rows %lld apart, %d wide", what, (long long)d->table_stride, d->width);
    AttendShape sh;
    if (int rc = attend_shape<C>(what, *d, sh)) return rc;
    if (sh.bytes() > 0 && (!d->workspace || !aligned(d->workspace, 16) || d->workspace_bytes < sh.bytes()))
        return pk_fail(PK_ERR_ARG, "%s: a workspace of %lld bytes is wanted, aligned to 16 (%lld given)", what, (long long)sh.bytes(),
                       (long long)(d->workspace ? d->workspace_bytes : 0));
    AttendParams p;
    p.q = d->q, p.out = d->out, p.lse = d->lse, p.cache = (const uint8_t *)d->cache;
    p.table = d->table, p.lens = d->lens, p.first = d->first;
    p.arrived = (int *)d->workspace;
    p.part = (float *)((char *)d->workspace + kCounters * 4);
    p.q_row = d->q_row, p.q_head = d->q_head, p.out_row = d->out_row, p.out_head = d->out_head;
    p.page_stride = d->page_stride, p.table_stride = d->table_stride;
    p.n_rows = d->n_rows, p.requests = d->requests, p.heads = d->heads, p.kv_heads = d->kv_heads;
    p.page = d->page, p.page_shift = log2i(d->page), p.n_pages = d->n_pages, p.width = d->width;
    p.max_len = d->max_len, p.window = d->window, p.group = d->heads / d->kv_heads;
    p.tiles = sh.tiles, p.splits = sh.splits, p.groups = sh.groups, p.chunk = sh.chunk, p.scale = d->scale;
    p.vec = aligned(d->q, 16) && d->q_row % 8 == 0 && d->q_head % 8 == 0;
    p.vec_out = aligned(d->out, 8) && d->out_row % 4 == 0 && d->out_head % 4 == 0;
    const unsigned grid = (unsigned)((int64_t)d->requests * d->kv_heads * sh.tiles * sh.splits);
    launch(p, sh, grid);
    return launched(what);
}

}  // namespace pklm
