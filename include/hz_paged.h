/*
 * hz_paged.h — C ABI of the paged operators on MI355X (gfx950): rows of tokens whose keys and values lie in a
 * pool of pages, for walkers or requests of very different lengths, and rotations by positions of
 * several axes. They stand next to the token operators (hz_token.h), whose conventions hold here. The
 * reference has no counterpart.
 *
 *   hz_qk_rotary_fwd / _bwd   rotation of queries and keys by positions of several axes (row and column of a
 *                             lattice site, layer, time), with or without the norms of hz_qk_norm_rotary
 *   hz_paged_append           new tokens' keys and values into their slots
 *   hz_paged_attention        attention of new tokens over the slots of their rows; the weights that
 *                             each slot has had are added up on request
 *   hz_paged_evict            the slots of the least such weight given up, the cache closed over them in place
 *
 * A cache is k and v [pages, page_size, Hk, D]: strides in elements of the page, slot and head axes (the
 * fields batch, token and head; multiples of 8, a head's D elements are contiguous). Row b has the slots
 * 0 .. n_b - 1 with n_b = lengths[b], clamped to [0, table_width page_size]; slot j lies in page
 * page_table[b, j / page_size] at j % page_size. Rows may share pages that no call writes. A number outside
 * [0, pages) is no page: its slots are not seen by the attention, not written by the append and not moved by the
 * eviction (whose results count them as slots like others, by their scores). Slots from n_b on are neither read nor written; those below must hold finite values.
 */
#ifndef HZ_PAGED_H
#define HZ_PAGED_H

#include "hz_token.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HZ_ROTARY_MAX_AXES 16 /* most axes of a position */

/*
 * The rotation of hz_qk_norm_rotary with the angle t = positions[b, n, axes[p]] * freqs[p] of pair p: positions
 * [B, N, n_axes] int32 (NULL: n, one axis), axes [n_freqs] int32 (NULL: 0; a number outside [0, n_axes)
 * leaves its pair as it is). norm 1: behind the norms, as there. norm 0: the rotation alone; w_q, w_k and
 * eps are not used. The other fields and their limits as there.
 */
typedef struct {
  hz_qk_norm_rotary rotary;
  const int32_t* axes;
  int64_t n_axes;
  int32_t norm;
} hz_qk_rotary;

int hz_qk_rotary_fwd(hipStream_t stream, const hz_qk_rotary* p);

/*
 * Its reverse mode, as hz_qk_norm_rotary_bwd's. norm 0: the cotangents turned back by -t; q and k are not read (data
 * may be NULL), dw_q and dw_k must be NULL, and no workspace is needed.
 */
int64_t hz_qk_rotary_workspace(int64_t B, int64_t N, int64_t D, int32_t norm);
int hz_qk_rotary_bwd(hipStream_t stream, const hz_qk_rotary* p, void* dq, void* dk, float* dw_q, float* dw_k,
                     void* workspace, int64_t workspace_bytes);

/* page_table [B, table_width] and lengths [B] int32; D a multiple of 8 up to HZ_TOKEN_MAX_HEAD;
 * table_width * page_size below 2^30. */
typedef struct {
  hz_token_tensor k, v;
  const int32_t *page_table, *lengths;
  int64_t B, pages, page_size, table_width, Hk, D;
  int32_t dtype;
} hz_paged_cache;

/*
 * Token i of the N new ones of row b (k, v [B, N, Hk, D], strided) goes into slot lengths[b] - N + i: lengths count
 * the new tokens already. Tokens of negative slots (the front of a row shorter than N) are left out. (lengths[b] clamped as
 * everywhere: beyond the table's slots, the row's last ones take the new tokens.) B N Hk heads, in pieces of 16 bytes, are at most 2^32 - 256.
 */
int hz_paged_append(hipStream_t stream, const hz_paged_cache* cache, const hz_token_tensor* k, const hz_token_tensor* v,
                    int64_t N);

/*
 * Attention of the last Nq tokens of each row: query i stands at p_i = n_b - Nq + i and sees the slots
 * j <= p_i. Scores, caps, slopes and shared key heads as hz_token_attention's with `causal` and kv_len = lengths;
 * q [B, Nq, H, D] strided, out [B, Nq, H, D]. A query that sees no slot gets zeros.
 * scores_out [B, Hk, table_width * page_size] float32 or NULL: with P the softmax,
 *     scores_out[b, g, j] = decay scores[b, g, j] + sum over i and the query heads h of key head g of P_hij
 * for j < n_b, and 0 from n_b on. scores (NULL: zeros) may be scores_out itself; 16-byte aligned both. scores_out may not
 * overlap anything else that is read. With scores_out the workspace holds B Nq H table_width page_size floats and more, whatever the lengths.
 * The slots are read once for up to 32 of the Nq H / Hk queries and heads of a key head (float32 with D above 64: 16), and again for every 32 more.
 */
typedef struct {
  hz_paged_cache cache;
  hz_token_tensor q;
  void* out;
  const float *slopes, *scores;
  float* scores_out;
  int64_t Nq, H;
  float scale, softcap, decay;
} hz_paged_attention_args;

int64_t hz_paged_attention_workspace(const hz_paged_attention_args* p);
int hz_paged_attention(hipStream_t stream, const hz_paged_attention_args* p, void* workspace, int64_t workspace_bytes);

/*
 * Rows longer than `budget` keep that many slots of each key head: the first `sinks`, the last `recent`, and of the others
 * those of the largest scores [B, Hk, table_width * page_size] float32 (equal ones: the lowest slot first; a NaN
 * is less than any number). The k-th kept slot at or behind the budget, in ascending order, then moves to the k-th slot
 * below it that was given up; the others stay where they are. Other rows stay as they are.
 *   lengths_out [B]                min(n_b, budget)
 *   sources [B, Hk, m] with m = min(budget, table_width * page_size): the slot whose token lies at s now; -1 from
 *                                  lengths_out[b] on
 *   scores_out (as scores; may not overlap it): the kept ones at their new slots, 0 from lengths_out[b] on
 * scores may not lie in the caches. The outputs may not be lengths or page_table. budget >= 1, sinks + recent <= budget. Rows that are cut
 * must not share pages with other rows, and no row may have a page twice.
 */
typedef struct {
  hz_paged_cache cache;
  const float* scores;
  float* scores_out;
  int32_t *sources, *lengths_out;
  int64_t budget, sinks, recent;
} hz_paged_evict_args;

int64_t hz_paged_evict_workspace(const hz_paged_evict_args* p);
int hz_paged_evict(hipStream_t stream, const hz_paged_evict_args* p, void* workspace, int64_t workspace_bytes);

#ifdef __cplusplus
}
#endif

#endif /* HZ_PAGED_H */
