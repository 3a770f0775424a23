/*
 * parakeet_lm.h -- C ABI of the language-model serving operators
 * (libparakeet_hip.so, the library of parakeet_hip.h).
 *
 * A voice pipeline that decodes speech with this library and answers with a
 * decoder-only model needs, beside that model's matrix products:
 *
 *   pk_kv_plan      which pages of the cache each session's tokens go to
 *   pk_kv4_store    key and value rows into a paged cache held in 4 bits
 *   pk_kv4_load     rows back out of it
 *   pk_kv4_attend   attention over that cache: single tokens and whole prompts
 *   pk_sample       the next token from logits and given uniform numbers
 *
 * Conventions.  Every call checks its descriptor on the host, enqueues its
 * kernels on the caller's stream (a hipStream_t, NULL = the default stream)
 * and returns; it allocates nothing, waits for nothing and may be captured
 * into a graph.  All pointers are device pointers of the current device, int32
 * unless said otherwise; strides are in elements.  Returns a PK_* status of
 * parakeet_hip.h; pk_last_error() has the message.  What only the device can
 * see (lengths, page ids, slots) is bounds-checked there: entries out of range
 * are skipped, never dereferenced.
 *
 * The cache.  A token's row of one head, D channels, is held in blocks of 32:
 * 4-bit floating point codes (sign, values 0 .5 1 1.5 2 3 4 6) and one scale
 * byte s that stands for 2^(s - 127); s = 255 marks a block that held a NaN or
 * an infinity and stands for NaNs.  17 bytes per 32 values.  A page holds
 * `page` tokens (16, 32, 64, 128 or 256).  The record of one (page, kv head) is
 *
 *   K codes [page][D/2] | V codes [page/8][16][8][D/32] | K scales [page][D/32] | V scales [D/32][page]
 *
 * page * (D + D/16) bytes; low nibbles hold the even channels.  V entry [a][r][i]
 * holds channels r*D/16 .. (r+1)*D/16 of token 8a + i: the order in which the
 * matrix instructions take 8 tokens' values.  A record lies at
 *   cache + id * page_stride + head * page * (D + D/16).
 * A slot is a token's place: page id * page + offset.
 */
#ifndef PARAKEET_LM_H
#define PARAKEET_LM_H

#include "parakeet_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { PK_DTYPE_F32 = 0, PK_DTYPE_F16 = 1, PK_DTYPE_BF16 = 2 };

#define PK_LM_MAX_REQUESTS 4096   /* requests per pk_kv_plan call */
#define PK_LM_MAX_VOCAB 1048576   /* logits per pk_sample row */

/* Page tables and slot maps.  Request b holds old_len[b] tokens and is to hold
 * new_len[b].  Pages it lacks are taken from the front of a ring of free page
 * ids, in the order of the requests, as long as the running sum of the pages
 * lacked is within the ring's count; a request that needs none is always
 * served, one that is not served keeps its length.  Pages given up are appended
 * behind the ring's end (for the next call).  Lengths below 0 or above
 * width * page make a request not served. */
typedef struct pk_kv_plan_desc {
    const int32_t *old_len, *new_len;   /* [requests] */
    int32_t *table;                     /* [requests][width], rows table_stride apart: page ids; entries of new pages
                                           are written, entries past a request's length are never read */
    int32_t *ring;                      /* [n_pages] free page ids, a ring */
    const int32_t *state;               /* {head, count} of the ring */
    int32_t *state_out;                 /* {head, count} after the call; not state itself */
    int32_t *lens;                      /* out [requests] lengths after the call; neither old_len nor new_len */
    int32_t *ok;                        /* out [requests] 1 = served */
    int32_t *first;                     /* out [requests + 1]: new tokens before request b (served or not) */
    int32_t *slots;                     /* out [n_tokens]: slot of each new token, -1 for tokens of requests not served,
                                           behind the last token, and on page ids that are negative or have no 32-bit slots */
    int32_t *pos;                       /* out [n_tokens]: its position in its request, -1 for tokens of requests not served
                                           and behind the last token; nullable */
    int64_t table_stride;
    int32_t requests, width, n_pages, page, n_tokens;
} pk_kv_plan_desc;
PK_API int pk_kv_plan(const pk_kv_plan_desc *desc, void *stream);

/* Rows k, v [n_rows][heads][head_dim] (strides per row and per head, channels
 * adjacent) into the cache at slots[n_rows], or from there.  Rows whose slot is
 * outside the cache are skipped; of rows stored to one slot in one call any mix
 * may be left there.  Blocks are rounded to the nearest code, ties
 * to the even code, under the power of two that puts the largest of the 32
 * values between 3.5 and 7 (kept to 2^-120 .. 2^125, so that smaller blocks
 * vanish and the largest stay finite; f16 rows over 57,344 are held as 65,536,
 * which f16 results, of pk_kv4_attend too, give as 65,504). */
typedef struct pk_kv4_rows_desc {
    void *k, *v;                        /* read by pk_kv4_store, written by pk_kv4_load */
    const int32_t *slots;
    void *cache;
    int64_t k_row, k_head, v_row, v_head;   /* strides */
    int64_t page_stride;                /* bytes between pages */
    int32_t n_rows, heads, head_dim, dtype, page, n_pages;
} pk_kv4_rows_desc;
PK_API int pk_kv4_store(const pk_kv4_rows_desc *desc, void *stream);
PK_API int pk_kv4_load(const pk_kv4_rows_desc *desc, void *stream);

/* Attention: out = softmax(scale * q . K^T) V for every query head.  Request b
 * brings queries first[b] .. first[b + 1] of q, its last tokens: query i stands
 * at position p = lens[b] - (first[b + 1] - first[b]) + i and sees the keys at
 * positions 0 .. p, with a window the last `window` of them (its own included).
 * A query that sees no key gives zeros and an lse of -inf, as does one whose
 * scores overflow to -inf all.  Query head h reads kv head
 * h / (heads / kv_heads).  Scores, sums and O are f32; probabilities are rounded
 * before the product with V, for bf16 results to bf16, which adds to the error
 * of a result's own rounding (0.0022 of the results' norm instead of 0.0016 over
 * prompts of 2,047), for f16 results to two bf16, 16 bits, which does not. */
typedef struct pk_kv4_attend_desc {
    const void *q;                      /* f16 or bf16 [n_rows][heads][head_dim] */
    void *out;                          /* as q */
    float *lse;                         /* out [n_rows][heads], natural logarithm of the softmax sum; nullable */
    const void *cache;
    const int32_t *table;               /* [requests][width], rows table_stride apart */
    const int32_t *lens;                /* [requests] tokens held, those of q included */
    const int32_t *first;               /* [requests + 1]; NULL: one query per request */
    void *workspace;                    /* pk_kv4_attend_workspace() bytes, zeroed once before its first use; nullable where
                                           that is 0.  One call at a time may use it. */
    int64_t workspace_bytes;
    int64_t q_row, q_head, out_row, out_head;   /* strides */
    int64_t page_stride, table_stride;
    int32_t n_rows, requests, heads, kv_heads, head_dim, dtype, page, n_pages, width;
    int32_t max_new;                    /* no request brings more queries */
    int32_t max_len;                    /* no request holds more tokens (longer ones are cut there) */
    int32_t window;                     /* 0 = none */
    float scale;                        /* finite */
} pk_kv4_attend_desc;
PK_API int pk_kv4_attend(const pk_kv4_attend_desc *desc, void *stream);
/* Bytes of workspace that the call wants (host arithmetic; pointers are not looked at). */
PK_API int pk_kv4_attend_workspace(const pk_kv4_attend_desc *desc, int64_t *bytes);

/* One token per row.  Weights are whole numbers, w = round(2^30 exp((x - max) /
 * temperature)) in f32 steps, so that no result depends on the order of a sum.
 * By falling logit (equal ones: rising index) the first top_k tokens are kept;
 * of these the ones with less than top_p of their weight before them; of these
 * the ones with at least min_p of the largest weight; the first always.  The
 * token is the first, by rising index, whose running kept weight exceeds u
 * times the kept total.  temperature <= 0 (or NaN): the largest logit, lowest
 * index, alone.  NaN logits count as -inf; a row of -inf gives token -1. */
typedef struct pk_sample_desc {
    const void *logits;                 /* [rows][vocab], rows logits_row apart */
    const float *u;                     /* [rows] uniform in [0, 1) */
    const float *temperature;           /* [rows], NULL = 1 */
    const int32_t *top_k;               /* [rows], NULL or an entry <= 0 = off */
    const float *top_p;                 /* [rows], NULL or an entry >= 1 = off */
    const float *min_p;                 /* [rows], NULL or an entry <= 0 = off */
    int32_t *token;                     /* out [rows] */
    float *prob;                        /* out [rows]: its share of the kept weight; nullable */
    int32_t *kept;                      /* out [rows]: how many tokens were kept; nullable */
    void *workspace;                    /* pk_sample_workspace() bytes, zeroed once before its first use; nullable where
                                           that is 0.  One call at a time may use it. */
    int64_t workspace_bytes;
    int64_t logits_row;
    int32_t rows, vocab, dtype, reserved;
} pk_sample_desc;
PK_API int pk_sample(const pk_sample_desc *desc, void *stream);
PK_API int pk_sample_workspace(const pk_sample_desc *desc, int64_t *bytes);

#ifdef __cplusplus
}
#endif
#endif
