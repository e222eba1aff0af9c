/*
 * hz_token.h — C ABI of the token operators on MI355X (gfx950): what an autoregressive wavefunction
 * over the same sites needs next to the MHSEA kernels (hz_mhsea.h). The reference has no counterpart.
 *
 *   hz_qk_norm_rotary_fwd / _bwd   RMS norms of queries and keys for each head, with the position
 *                                  rotation in the same pass
 *   hz_token_attention_fwd / _bwd  attention with shared key heads, capped scores, a distance bias and
 *                                  causal, prefix, document and length masks; single tokens over a cache
 *   hz_bucket_bias_fwd / _bwd      a learned relative position bias by buckets, in the bias layouts of
 *                                  hz_mhsea.h, and its table's gradient
 *
 * Conventions as hz_mhsea.h: device pointers, 16-byte aligned (integer arrays, slopes and weights: as
 * their elements), enqueue-only on `stream`, nothing allocated (scratch memory is the caller's
 * `workspace`, whose size in bytes a *_workspace call gives; calls that may overlap need one each),
 * outputs fully overwritten, deterministic (no atomics on global memory), 0 or an HZ_E* status with
 * hz_last_error(). Every axis is at least 1 long. Tensors with strides are given by their strides in elements of the batch, token and
 * head axes (multiples of 8; a head's D elements are contiguous; 0 is a broadcast axis); the others
 * are C-contiguous. dtype: HZ_DTYPE_F32 or HZ_DTYPE_BF16.
 */
#ifndef HZ_TOKEN_H
#define HZ_TOKEN_H

#include <stdint.h>
#include <hip/hip_runtime_api.h>

#include "hz_mhsea.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HZ_TOKEN_MAX_HEAD 128     /* largest head dimension of the attention */
#define HZ_ROTARY_MAX_HEAD 256    /* largest head dimension of the norms */
#define HZ_BUCKET_MAX 512         /* most buckets of a relative position bias */
#define HZ_BUCKET_MAX_RANGE 4096  /* largest R: buckets holds the distances -R .. R */
#define HZ_BUCKET_MAX_TABLE 32832 /* most entries of (n_buckets + 1) rows of H, rounded up to 64 */

/* A strided [B, N, heads, D] tensor: strides in elements. */
typedef struct {
  void* data;
  int64_t batch, token, head;
} hz_token_tensor;

/*
 * Norms of queries and keys for each head, then the rotation by position:
 *     r   = 1 / sqrt(mean_d x_d^2 + eps),   y = x r w                        (w NULL: ones)
 *     pair p of the first 2 n_freqs elements: angle t = positions[b, n] * freqs[p] (in float64)
 *         (y_a, y_b) -> (y_a cos t - y_b sin t, y_b cos t + y_a sin t)
 *         a = p, b = p + n_freqs; or, interleaved, a = 2 p, b = 2 p + 1
 * q [B, N, H, D], k [B, N, Hk, D] (strided) -> q_out, k_out (strided: k_out may lie in a cache); the
 * outputs may not overlap the inputs. w_q, w_k [D] float32; freqs [n_freqs] float64, in radians a
 * position; positions [B, N] int32 (NULL: n). D a multiple of 8 up to HZ_ROTARY_MAX_HEAD; n_freqs
 * a multiple of 4, 2 n_freqs <= D, 0: no rotation.
 */
typedef struct {
  hz_token_tensor q, k, q_out, k_out;
  const float *w_q, *w_k;
  const double* freqs;
  const int32_t* positions;
  int64_t B, N, H, Hk, D, n_freqs;
  float eps;
  int32_t interleaved, dtype;
} hz_qk_norm_rotary;

int hz_qk_norm_rotary_fwd(hipStream_t stream, const hz_qk_norm_rotary* p);

/*
 * Its reverse mode. q, k and the options as in the forward; q_out and k_out are the cotangents of
 * its outputs. With g the cotangent turned back by -t:
 *     dw_d = sum over rows of g_d x_d r,   dx = r (g w - x r mean_d(g w x r))
 * dq [B, N, H, D], dk [B, N, Hk, D]; dw_q, dw_k [D] float32 (NULL: not wanted).
 */
int64_t hz_qk_norm_rotary_workspace(int64_t B, int64_t N, int64_t D);
int hz_qk_norm_rotary_bwd(hipStream_t stream, const hz_qk_norm_rotary* p, void* dq, void* dk, float* dw_q,
                          float* dw_k, void* workspace, int64_t workspace_bytes);

/*
 * Attention of Nq query tokens over Nk key tokens. Head h of the queries uses key head h / (H / Hk).
 * Row b holds n_b = kv_len[b] keys (NULL: Nk; other values are clamped to [0, Nk]) and its queries are
 * the tokens at positions p_i = n_b - Nq + i:
 *     x_ij = scale q_i . k_j
 *     s_ij = softcap tanh(x_ij / softcap)   (softcap 0: x_ij)   - slopes[h] |p_i - j|   (slopes NULL: 0)
 *     visible(i, j):  j < n_b
 *                     and (not causal, or j <= p_i, or j < prefix[b])                  (prefix NULL: 0)
 *                     and (documents NULL, or p_i >= 0 and documents[b, p_i] = documents[b, j] >= 0)
 *     out_i = sum_j softmax over the visible j of s_ij, times v_j;   lse_i = log sum_j exp s_ij
 * A query that sees no key gets zeros and lse = -inf. Keys from n_b on and tokens of a negative document
 * (padding) are never used, whatever they hold; the other tokens' values must be finite.
 * q [B, Nq, H, D], k, v [B, Nk, Hk, D] strided; out [B, Nq, H, D]; lse [B, Nq, H] float32 or NULL (a
 * forward without a reverse pass). slopes [H] float32, prefix [B], documents [B, Nk] and kv_len [B]
 * int32. D a multiple of 8 up to HZ_TOKEN_MAX_HEAD, H a multiple of Hk, Nq, Nk < 2^30, B H ceil(Nq / 128) and, with
 * lse, B Hk ceil(Nk / 128) at most 2^20, B Nk at most 2^31 with documents; prefix only with causal.
 * out_low [B, Nq, H, D] or NULL, for bfloat16: what out's rounding left out, rounded to bfloat16. The
 * reverse pass takes rowsum(dout out) from both where it is given: from out alone the row sum's error is as large
 * as that of all other roundings of dq and dk together.
 * The weights of the products with v and the score gradients are rounded to bfloat16 for bfloat16
 * tensors (and the rounded weights are summed); for float32 ones every product keeps float32's precision (three bfloat16 parts an operand,
 * split_f32.h, whose remarks on values that are not finite or above 3.39e38 hold).
 */
typedef struct {
  hz_token_tensor q, k, v;
  void *out, *out_low;
  float* lse;
  const float* slopes;
  const int32_t *prefix, *documents, *kv_len;
  int64_t B, Nq, Nk, H, Hk, D;
  float scale, softcap;
  int32_t causal, dtype;
} hz_token_attention;

int64_t hz_token_attention_fwd_workspace(const hz_token_attention* p);
int hz_token_attention_fwd(hipStream_t stream, const hz_token_attention* p, void* workspace, int64_t workspace_bytes);

/*
 * Its reverse mode for the cotangent dout (strided) of out; out and lse are the forward's:
 *     P = exp(s - lse),  dP = dout v^T,  dS = P (dP - rowsum(dout out)) (1 - tanh^2(x / softcap))
 *     dq = scale dS k,  dk = scale sum over the key head's query heads of dS^T q,  dv = the same of P^T dout
 * P is at most 1. Rows whose lse is above 32 in size (256 for bfloat16) have their largest score and sum formed again, so that
 * their weights keep their precision at any size of the scores.
 * dq [B, Nq, H, D], dk, dv [B, Nk, Hk, D]; what no visible pair reaches is zero.
 */
int64_t hz_token_attention_bwd_workspace(const hz_token_attention* p);
int hz_token_attention_bwd(hipStream_t stream, const hz_token_attention* p, const hz_token_tensor* dout, void* dq,
                           void* dk, void* dv, void* workspace, int64_t workspace_bytes);

/*
 * Learned relative position bias: with d = clamp(k_positions[b, j] - q_positions[b, i], -R, R),
 *     e[b, i, j, h] = table[buckets[R + d], h]
 * table [n_buckets, H] float32; buckets [2 R + 1] int32 (a number outside [0, n_buckets) gives a zero
 * bias and no gradient); q_positions [B, Nq], k_positions [B, Nk] int32; e [B, Nq, H, Nk], or
 * [B, Nq, Nk, H] with HZ_FLAG_E_QKH. n_buckets <= HZ_BUCKET_MAX, R <= HZ_BUCKET_MAX_RANGE, H <= 256,
 * (n_buckets + 1) ceil64(H) <= HZ_BUCKET_MAX_TABLE (the table lies in LDS).
 */
int hz_bucket_bias_fwd(hipStream_t stream, const float* table, const int32_t* buckets, const int32_t* q_positions,
                       const int32_t* k_positions, void* e, int64_t B, int64_t Nq, int64_t Nk, int64_t H,
                       int64_t n_buckets, int64_t R, int dtype, int flags);

/* dtable[m, h] = sum of de[b, i, j, h] over the (b, i, j) of bucket m; float32 sums. de must be finite (with
 * HZ_FLAG_E_QKH a value that is not makes every bucket of its head NaN). */
int64_t hz_bucket_bias_workspace(int64_t B, int64_t Nq, int64_t Nk, int64_t H, int64_t n_buckets, int dtype, int flags);
int hz_bucket_bias_bwd(hipStream_t stream, const void* de, const int32_t* buckets, const int32_t* q_positions,
                       const int32_t* k_positions, float* dtable, void* workspace, int64_t workspace_bytes, int64_t B,
                       int64_t Nq, int64_t Nk, int64_t H, int64_t n_buckets, int64_t R, int dtype, int flags);

#ifdef __cplusplus
}
#endif

#endif /* HZ_TOKEN_H */
