// pk_lm_step.hip -- host side + C ABI of parakeet_lm.h's operators of a step with drafted tokens: norms and rotation, the
// 8-bit cache, attention over it, verification.  The kernels are in lm_rope.h, lm_cache8.h, lm_attend8.h and lm_verify.h.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "lm_attend8.h"
#include "lm_attend_host.h"
#include "lm_cache8.h"
#include "lm_host.h"
#include "lm_rope.h"
#include "lm_verify.h"
#include "parakeet_lm.h"

namespace {

using namespace pklm;

// What pk_kv8_append, _load and _attend ask of the cache; 0 = fine.
int check_cache8(const char *what, const void *cache, int64_t page_stride, int page, int n_pages, int heads, int dim) {
    if (page != 32 && page != 64 && page != 128 && page != 256)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: pages of %d tokens (32, 64, 128 or 256)", what, page);
    if (dim != 64 && dim != 128 && dim != 256) return pk_fail(PK_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128 or 256)", what, dim);
    if (heads <= 0 || n_pages <= 0) return pk_fail(PK_ERR_ARG, "%s: %d heads, %d pages", what, heads, n_pages);
    if ((int64_t)n_pages * page > INT32_MAX)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d pages of %d tokens: slots are 32 bits", what, n_pages, page);
    if (!cache || !aligned(cache, 16)) return pk_fail(PK_ERR_ARG, "%s: the cache is NULL or not aligned to 16 bytes", what);
    const Record8 rec{page, dim};
    if (page_stride % 16 || page_stride < heads * rec.bytes())
        return pk_fail(PK_ERR_ARG, "%s: page_stride %lld bytes (a multiple of 16, at least %lld)", what, (long long)page_stride,
                       (long long)(heads * rec.bytes()));
    return PK_OK;
}

// What pk_qk_rope and pk_kv8_append ask of the norm and the rotation.
int check_turn(const char *what, int dim, int rot, const float *inv_freq, const int32_t *pos, int norm, float eps, const float *qw, const float *kw) {
    if (rot < 0 || rot > dim || rot % 16) return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d of %d channels turned (a multiple of 16)", what, rot, dim);
    if (rot && (!inv_freq || !pos)) return pk_fail(PK_ERR_ARG, "%s: NULL positions or inv_freq", what);
    if (norm && !(eps >= 0 && std::isfinite(eps))) return pk_fail(PK_ERR_ARG, "%s: an eps of %g", what, eps);
    if (!aligned(inv_freq, 4) || !aligned(pos, 4) || !aligned(qw, 4) || !aligned(kw, 4))
        return pk_fail(PK_ERR_ARG, "%s: positions, inv_freq or weights not aligned to their type", what);
    return PK_OK;
}

// Whether `each` channels of any row are aligned to their bytes.
bool wide_rows(const void *p, int64_t row, int64_t head, int size, int each = 4) {
    return aligned(p, each * size) && row % each == 0 && head % each == 0;
}

// Rows of a workgroup, workgroups beside it on the same rows.
struct TurnGrid {
    int rows, parts;
    int64_t groups;
};
// As many rows as leave 128 groups of them, whole blocks where that is more than half a block; beside each, as many parts of the heads as
// make 2,048 workgroups.  32 heads on 8 x 128 in bf16, one input again and again, microseconds where 1,024, 128 and 32 groups are left: 1,000 rows normed
// and turned 9.4, 8.6, 10.6; up to 4 x 200 appended 22, 15, 12, 4 x 1,000 56, 24, 24; a token of 64 sessions 7.5, 7.6, 11.1.  With parts
// up to 1,024, 2,048 and 4,096 workgroups: 16,385 rows 79, 61, 67, up to 4 x 200 appended 17.5, 14.8, 14.1.
TurnGrid turn_grid(int n_rows, int parts, int least) {
    TurnGrid g;
    g.rows = (int)std::min<int64_t>(std::max<int64_t>(n_rows / 128, least), kTurnRows);
    if (g.rows > kTurnRows / 2) g.rows = kTurnRows;
    g.groups = ((int64_t)n_rows + g.rows - 1) / g.rows;
    g.parts = (int)std::min<int64_t>(std::max<int64_t>((2048 + g.groups - 1) / g.groups, 1), std::max(parts, 1));
    return g;
}

template <class F>
void by_type(int dtype, F f) {
    if (dtype == PK_DTYPE_F32) f(F32{});
    else if (dtype == PK_DTYPE_F16) f(F16{});
    else f(BF16{});
}
template <class F>
void by_dim(int dim, F f) {
    if (dim == 64) f(std::integral_constant<int, 64>{});
    else if (dim == 128) f(std::integral_constant<int, 128>{});
    else f(std::integral_constant<int, 256>{});
}

struct HostKv8 {
    static int check(const char *what, const void *cache, int64_t page_stride, int page, int n_pages, int heads, int dim) {
        return check_cache8(what, cache, page_stride, page, n_pages, heads, dim);
    }
    // The prompt kernel does not split keys: it takes calls that fill the card with workgroups, or half of it where no request has many
    // more keys than new tokens; rows of 256 channels, which the other kernel takes 16 columns at a time, from a quarter on.  32 heads
    // on 8 in bf16, new tokens and keys up to the numbers given, spread evenly over the requests, microseconds of the other kernel and of it:
    //   workgroups         128 channels                            64 channels                           256 channels
    //   128                512 on 8,191: 123, 199; on 512: 21, 20                                        512 on 8,191: 482, 391
    //   256                4 x 256 on 8,191: 149, 207;             94, 157;                              514, 394
    //                      on 2,047: 58, 56; on 512: 31, 20        37, 44; 18, 16
    //   512                4 x 512 on 8,191: 258, 259;             159, 199;                             970, 567
    //                      64 x 24 on 2,047: 75, 72                42, 56                                232, 214
    //   1,024              4 x 1,024 on 8,191: 471, 336            275, 258                              1,832, 894
    // 64 x 16 on 2,047, half a tile's rows, at 128 channels: 61, 73.
    static bool prompt(const pk_kv4_attend_desc &d, int64_t rows, int64_t groups) {
        const int64_t keys = d.window ? std::min<int64_t>(d.max_len, (int64_t)d.window + d.max_new) : d.max_len;
        if (rows < 96) return false;
        if (d.head_dim == 256) return groups >= 128;
        return groups >= (d.head_dim == 64 ? 1024 : 512) || (groups >= 256 && keys <= (d.head_dim == 64 ? 2 : 8) * (int64_t)d.max_new);
    }
    // Two tiles that share each key's operands, where registers hold them.  32 heads on 8 x 128 in bf16, in one tile and in two: 64
    // sessions' up to 5 tokens (20 rows) on up to 4,097 keys 94 and 65 us, 4 x 20 tokens on 8,191 keys 39 and 24, 64 x 20 on 1,000 keys 47
    // and 47; but one session's 6 tokens on 8,191 keys, whose splits do not fill the card, 13 and 17, which this rule does not see.
    static int tile_cols(int64_t rows, int dim) { return rows <= 16 || dim == 256 ? 16 : 32; }
};

template <class T>
void launch_attend8(const AttendParams &p, const AttendShape &sh, int dim, unsigned grid, hipStream_t s) {
    by_dim(dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (sh.prompt) attend8_prompt_kernel<T, D><<<grid, kPromptThreads, 0, s>>>(p);
        else if (sh.cols == 16) attend8_kernel<T, D, 1><<<grid, kAttendThreads, 0, s>>>(p);
        else if constexpr (D < 256) attend8_kernel<T, D, 2><<<grid, kAttendThreads, 0, s>>>(p);
    });
}

// Verification.  Rows of up to kVerifyVocab logits are a workgroup's each, in one launch, 16 tokens a lane at most; longer ones, which
// no workgroup's registers hold, are cut in chunks.  Up to 5 f32 rows of 16,384 logits with draft logits, of 1 request and of 256, take 11 and 34
// us in one launch, 23 and 44 in three.  Fewer threads make room for more rows: 256 requests' rows of 4,001 take 12 us on 512 threads each,
// 26 on 1,024, of 8,001 19 and 28; one's of 4,001 7.4 and 9.1.
//
// In one launch a request has as many workgroups as it may bring rows.  Where that bound says nothing (it is all rows of the call) or
// is far, it has twice the mean's, or what makes kVerifyGroups in all, and they take its rows in turn: with the bound and without,
// 256 requests' 5 rows of 1,027 with draft logits take 10.4 and 10.5 us, 64 requests' 5 of 4,001 7.5 and 9.0, one request's 300 rows of
// 1,027 among 63 of one row 11.2 and 17.5.  Half of kVerifyGroups: 10.5, 7.7 and 25.9.  Several launches have workgroups for the call's
// rows alone.
constexpr int kVerifyVocab = 16384, kVerifyGroups = 8192, kVerifyMost = 1 << 17;

struct VerifyShape {
    bool turns;          // see verify_row_kernel
    int each;
    int64_t groups;      // workgroups of it, or of the first launch of several
    int passes, chunks, draw_passes, draw_chunks;        // see SplitVerify
    // counters first, the same place for every shape: they are zero between calls
    static constexpr int64_t kCounterBytes = PK_LM_MAX_REQUESTS * 4;
    int64_t max_at, at_at, sum_at, left_at, bytes;
};

VerifyShape verify_shape(const pk_verify_desc &d) {
    VerifyShape s{};
    const int64_t requests = std::max(d.requests, 1), most = std::max(std::min(d.max_new, d.n_rows), 1);
    const int64_t mean = (d.n_rows + requests - 1) / requests;
    if (d.vocab <= kVerifyVocab) {
        const bool known = (d.max_new < d.n_rows || requests == 1) && requests * most <= kVerifyMost;
        s.each = (int)(known ? most : std::min(most, std::max(2 * mean, kVerifyGroups / requests)));
        s.turns = s.each < most, s.groups = requests * s.each;
        s.bytes = VerifyShape::kCounterBytes + d.n_rows * (int64_t)sizeof(RowVerdict);
        return s;
    }
    // As many chunks as make `want` workgroups, 64 of a row at most (a lane has one each), of two passes at least.  Requests of up to 5 rows
    // of 128,001 in bf16 with draft logits: the first two launches in 2,048, 4,096, 8,192 and 16,384 take 31, 23, 25, 27 us for 64, 12.3, 13.5,
    // 11.3, 11.5 for 16; the draws of 64, of which two fit a unit, in 256, 512 and 1,024 28, 21, 27.
    auto cut = [&](int64_t each, int &chunks, int &passes, int64_t want, int pass) {
        const int64_t aim = std::min<int64_t>(std::max<int64_t>(want / std::max<int64_t>(each, 1), 1), 64);
        passes = (int)std::max<int64_t>(2, (d.vocab + aim * pass - 1) / (aim * pass));
        chunks = (d.vocab + passes * pass - 1) / (passes * pass);
    };
    const int64_t rows = d.n_rows, sources = d.draft ? 2 : 1;
    cut(std::min(requests * most, 2 * rows) * sources, s.chunks, s.passes, 8192, kVerifyPass);
    cut(d.requests, s.draw_chunks, s.draw_passes, 512, kDrawPass);
    s.groups = rows * sources * s.chunks;
    int64_t at = VerifyShape::kCounterBytes;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    s.max_at = take(rows * 2 * s.chunks * 4), s.at_at = take(rows * 2 * s.chunks * 4), s.sum_at = take(rows * 2 * s.chunks * 8);
    s.left_at = take((int64_t)d.requests * s.draw_chunks * 8);
    s.bytes = at;
    return s;
}

int verify_check(const char *what, const pk_verify_desc *d) {
    if (!d) return pk_fail(PK_ERR_ARG, "%s: no descriptor", what);
    if (d->requests < 0 || d->requests > PK_LM_MAX_REQUESTS)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d requests (at most %d)", what, d->requests, PK_LM_MAX_REQUESTS);
    if (d->n_rows < 0 || d->max_new < 0 || d->vocab <= 0 || d->vocab > PK_LM_MAX_VOCAB)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d rows, max_new %d, %d logits (1 .. %d)", what, d->n_rows, d->max_new, d->vocab, PK_LM_MAX_VOCAB);
    if ((int64_t)d->requests * d->max_new > INT32_MAX || verify_shape(*d).groups > most_groups(1024))       // threads of the largest workgroup
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d requests of up to %d rows, %d in all, in one call", what, d->requests, d->max_new, d->n_rows);
    return PK_OK;
}

// Whether two arrays of n whole numbers have a place in common.
bool overlap(const int32_t *a, const int32_t *b, int64_t n) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return (x < y ? y - x : x - y) < (uintptr_t)n * sizeof(int32_t);
}

template <class T, int BS, int G>
void launch_verify_rows(const pk_verify_desc &d, const VerifyShape &sh, hipStream_t s) {
    int *arrived = (int *)d.workspace;
    auto *verdicts = (RowVerdict *)((char *)d.workspace + VerifyShape::kCounterBytes);
    auto launch = [&](auto draft, auto turns) {
        verify_row_kernel<T, BS, G, draft.value, turns.value><<<(unsigned)sh.groups, BS, 0, s>>>(d, sh.each, arrived, verdicts);
    };
    if (sh.turns) d.draft ? launch(std::true_type{}, std::true_type{}) : launch(std::false_type{}, std::true_type{});
    else d.draft ? launch(std::true_type{}, std::false_type{}) : launch(std::false_type{}, std::false_type{});
}

template <class T>
void launch_verify(const pk_verify_desc &d, const VerifyShape &sh, hipStream_t s) {
    if (d.vocab <= 2048) return launch_verify_rows<T, 256, 1>(d, sh, s);
    if (d.vocab <= 4096) return launch_verify_rows<T, 512, 1>(d, sh, s);
    if (d.vocab <= 8192) return launch_verify_rows<T, 512, 2>(d, sh, s);
    if (d.vocab <= kVerifyVocab) return launch_verify_rows<T, 1024, 2>(d, sh, s);
    char *w = (char *)d.workspace;
    SplitVerify p;
    p.arrived = (int *)w, p.chunk_max = (float *)(w + sh.max_at), p.chunk_at = (int *)(w + sh.at_at), p.chunk_sum = (u64 *)(w + sh.sum_at);
    p.left = (u64 *)(w + sh.left_at);
    p.chunks = sh.chunks, p.passes = sh.passes, p.sources = d.draft ? 2 : 1;
    p.draw_chunks = sh.draw_chunks, p.draw_passes = sh.draw_passes;
    if (sh.groups) verify_max_kernel<T><<<(unsigned)sh.groups, kVerifyThreads, 0, s>>>(d, p);
    if (sh.groups) verify_sum_kernel<T><<<(unsigned)sh.groups, kVerifyThreads, 0, s>>>(d, p);
    verify_draw_kernel<T><<<(unsigned)(d.requests * p.draw_chunks), kDrawThreads, 0, s>>>(d, p);
}

}  // namespace

extern "C" {

PK_API int pk_qk_rope(const pk_qk_rope_desc *d, void *stream) {
    pk_fail_clear();
    const char *what = "pk_qk_rope";
    if (!d) return pk_fail(PK_ERR_ARG, "%s: no descriptor", what);
    if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128 or 256)", what, d->head_dim);
    if (!float_type(d->dtype)) return pk_fail(PK_ERR_UNSUPPORTED, "%s: dtype %d", what, d->dtype);
    if (d->n_rows < 0 || d->heads < 0 || d->kv_heads < 0 || d->heads + (int64_t)d->kv_heads > 65535)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d rows of %d and %d heads (at most 65535)", what, d->n_rows, d->heads, d->kv_heads);
    if (int rc = check_turn(what, d->head_dim, d->rot_dim, d->inv_freq, d->pos, d->norm, d->eps, d->q_weight, d->k_weight)) return rc;
    if (d->n_rows == 0 || d->heads + d->kv_heads == 0) return PK_OK;
    const int size = type_size(d->dtype);
    if ((d->heads && (!d->q || !d->q_out)) || (d->kv_heads && (!d->k || !d->k_out))) return pk_fail(PK_ERR_ARG, "%s: NULL rows", what);
    if (!aligned(d->q, size) || !aligned(d->k, size) || !aligned(d->q_out, size) || !aligned(d->k_out, size))
        return pk_fail(PK_ERR_ARG, "%s: rows not aligned to their type", what);
    const TurnGrid g = turn_grid(d->n_rows, (d->heads + d->kv_heads + kTurnWaves - 1) / kTurnWaves, 512 / d->head_dim);
    if (g.groups * g.parts > most_groups(kTurnThreads)) return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d rows in one call", what, d->n_rows);
    const int wide_q = wide_rows(d->q, d->q_row, d->q_head, size) | wide_rows(d->q_out, d->q_out_row, d->q_out_head, size) << 1;
    const int wide_k = wide_rows(d->k, d->k_row, d->k_head, size) | wide_rows(d->k_out, d->k_out_row, d->k_out_head, size) << 1;
    const bool halves = d->rot_dim == d->head_dim && !d->interleaved && (wide_q == 3 || !d->heads) && (wide_k == 3 || !d->kv_heads);
    by_type(d->dtype, [&](auto t) {
        by_dim(d->head_dim, [&](auto dim) {
            const dim3 grid((unsigned)g.groups, g.parts);
            if (halves) rope_kernel<decltype(t), dim.value, true><<<grid, kTurnThreads, 0, (hipStream_t)stream>>>(*d, g.rows, wide_q, wide_k);
            else rope_kernel<decltype(t), dim.value, false><<<grid, kTurnThreads, 0, (hipStream_t)stream>>>(*d, g.rows, wide_q, wide_k);
        });
    });
    return launched(what);
}

PK_API int pk_kv8_append(const pk_kv8_append_desc *d, void *stream) {
    pk_fail_clear();
    const char *what = "pk_kv8_append";
    if (!d) return pk_fail(PK_ERR_ARG, "%s: no descriptor", what);
    if (int rc = check_cache8(what, d->cache, d->page_stride, d->page, d->n_pages, d->kv_heads, d->head_dim)) return rc;
    if (!float_type(d->dtype)) return pk_fail(PK_ERR_UNSUPPORTED, "%s: dtype %d", what, d->dtype);
    if (d->n_rows < 0 || d->heads < 0 || d->heads + 2 * (int64_t)d->kv_heads > 65535)
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d rows of %d and 2 x %d heads (at most 65535)", what, d->n_rows, d->heads, d->kv_heads);
    if (int rc = check_turn(what, d->head_dim, d->rot_dim, d->inv_freq, d->pos, d->norm, d->eps, d->q_weight, d->k_weight)) return rc;
    if (d->n_rows == 0) return PK_OK;
    const int size = type_size(d->dtype);
    if (!d->k || !d->v || !d->slots || (d->heads && (!d->q || !d->q_out))) return pk_fail(PK_ERR_ARG, "%s: NULL rows or slots", what);
    if (!aligned(d->k, size) || !aligned(d->v, size) || !aligned(d->q, size) || !aligned(d->q_out, size) || !aligned(d->slots, 4))
        return pk_fail(PK_ERR_ARG, "%s: rows or slots not aligned to their type", what);
    const TurnGrid g = turn_grid(d->n_rows, std::max(2 * d->kv_heads, (d->heads + kTurnWaves - 1) / kTurnWaves), 1);
    if (g.groups * g.parts > most_groups(kTurnThreads)) return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d rows in one call", what, d->n_rows);
    const int wide_q = wide_rows(d->q, d->q_row, d->q_head, size) | wide_rows(d->q_out, d->q_out_row, d->q_out_head, size) << 1;
    const int wide_kv = wide_rows(d->k, d->k_row, d->k_head, size) && wide_rows(d->v, d->v_row, d->v_head, size);
    const bool halves = d->rot_dim == d->head_dim && !d->interleaved && (wide_q == 3 || !d->heads) && wide_kv;
    by_type(d->dtype, [&](auto t) {
        by_dim(d->head_dim, [&](auto dim) {
            const dim3 grid((unsigned)g.groups, g.parts);
            const int shift = log2i(d->page);
            if (halves) append_kernel<decltype(t), dim.value, true><<<grid, kTurnThreads, 0, (hipStream_t)stream>>>(*d, g.rows, shift, wide_q, wide_kv);
            else append_kernel<decltype(t), dim.value, false><<<grid, kTurnThreads, 0, (hipStream_t)stream>>>(*d, g.rows, shift, wide_q, wide_kv);
        });
    });
    return launched(what);
}

PK_API int pk_kv8_load(const pk_kv4_rows_desc *d, void *stream) {
    pk_fail_clear();
    const char *what = "pk_kv8_load";
    if (!d) return pk_fail(PK_ERR_ARG, "%s: no descriptor", what);
    if (int rc = check_cache8(what, d->cache, d->page_stride, d->page, d->n_pages, d->heads, d->head_dim)) return rc;
    if (d->n_rows < 0) return pk_fail(PK_ERR_ARG, "%s: %d rows", what, d->n_rows);
    if (d->n_rows == 0) return PK_OK;
    if (!float_type(d->dtype)) return pk_fail(PK_ERR_UNSUPPORTED, "%s: dtype %d", what, d->dtype);
    const int size = type_size(d->dtype);
    if (!d->k || !d->v || !d->slots) return pk_fail(PK_ERR_ARG, "%s: NULL rows or slots", what);
    if (!aligned(d->k, size) || !aligned(d->v, size) || !aligned(d->slots, 4))
        return pk_fail(PK_ERR_ARG, "%s: rows or slots not aligned to their type", what);
    if (d->heads > 32767) return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d heads (at most 32767)", what, d->heads);
    const int each = kRowThreads * 8 / d->head_dim;
    const int64_t groups = ((int64_t)d->n_rows + each - 1) / each;
    if (groups * 2 * d->heads > most_groups(kRowThreads))
        return pk_fail(PK_ERR_UNSUPPORTED, "%s: %d rows of %d channels in one call", what, d->n_rows, d->head_dim);
    const int wide = wide_rows(d->k, d->k_row, d->k_head, size, 16 / size) && wide_rows(d->v, d->v_row, d->v_head, size, 16 / size);
    by_type(d->dtype, [&](auto t) {
        by_dim(d->head_dim, [&](auto dim) {
            load8_kernel<decltype(t), dim.value><<<dim3((unsigned)groups, 2 * d->heads), kRowThreads, 0, (hipStream_t)stream>>>(*d, log2i(d->page), wide);
        });
    });
    return launched(what);
}

PK_API int pk_kv8_attend_workspace(const pk_kv4_attend_desc *d, int64_t *bytes) {
    return attend_workspace<HostKv8>("pk_kv8_attend", d, bytes);
}

PK_API int pk_kv8_attend(const pk_kv4_attend_desc *d, void *stream) {
    return attend_call<HostKv8>("pk_kv8_attend", d, [&](const AttendParams &p, const AttendShape &s, unsigned grid) {
        if (d->dtype == PK_DTYPE_F16) launch_attend8<F16>(p, s, d->head_dim, grid, (hipStream_t)stream);
        else launch_attend8<BF16>(p, s, d->head_dim, grid, (hipStream_t)stream);
    });
}

PK_API int pk_verify_workspace(const pk_verify_desc *d, int64_t *bytes) {
    pk_fail_clear();
    if (int rc = verify_check("pk_verify_workspace", d)) return rc;
    if (!bytes) return pk_fail(PK_ERR_ARG, "pk_verify_workspace: NULL result");
    *bytes = verify_shape(*d).bytes;
    return PK_OK;
}

PK_API int pk_verify(const pk_verify_desc *d, void *stream) {
    pk_fail_clear();
    const char *what = "pk_verify";
    if (int rc = verify_check(what, d)) return rc;
    if (!float_type(d->dtype)) return pk_fail(PK_ERR_UNSUPPORTED, "%s: dtype %d", what, d->dtype);
    if (d->requests == 0) return PK_OK;
    // without rows the requests' counts are written all the same
    if (d->n_rows > 0 && d->max_new == 0) return pk_fail(PK_ERR_ARG, "%s: max_new 0", what);
    if (!d->first || !d->u_draw || !d->accepted || (d->n_rows > 0 && (!d->logits || !d->tokens || !d->u || !d->out)))
        return pk_fail(PK_ERR_ARG, "%s: NULL array", what);
    if (d->lens_out && (!d->lens || overlap(d->lens_out, d->lens, d->requests)))
        return pk_fail(PK_ERR_ARG, "%s: lens_out without lens, or over lens", what);
    if (overlap(d->out, d->tokens, d->n_rows)) return pk_fail(PK_ERR_ARG, "%s: out is written while tokens are read", what);
    const int size = type_size(d->dtype);
    if (!aligned(d->logits, size) || !aligned(d->draft, size)) return pk_fail(PK_ERR_ARG, "%s: logits not aligned to their type", what);
    const VerifyShape sh = verify_shape(*d);
    if (!d->workspace || !aligned(d->workspace, 16) || d->workspace_bytes < sh.bytes)
        return pk_fail(PK_ERR_ARG, "%s: a workspace of %lld bytes is wanted, aligned to 16 (%lld given)", what, (long long)sh.bytes,
                       (long long)(d->workspace ? d->workspace_bytes : 0));
    by_type(d->dtype, [&](auto t) { launch_verify<decltype(t)>(*d, sh, (hipStream_t)stream); });
    return launched(what);
}

}  // extern "C"
