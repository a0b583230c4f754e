/*
 * primitiv_b200 -- C ABI of the operators of an attention layer: rotary positions, norms of queries
 * and keys with the rotation in the same pass, and attention over packed sequences, each with its
 * backward pass.
 *
 * The reference has none of these; what stands between them (the products of queries, keys and
 * values, the output product) is b200_matmul_*.  Same conventions as primitiv_b200_ops.h: device
 * pointers, return codes, `mode` selects the storage type (float for the fp32 modes, IEEE half for
 * B200_MODE_FP16), launches go to `stream`, backward passes add into a gradient with `accumulate`
 * = 1 and overwrite it with 0.  Nothing here allocates device memory, uses atomics or waits for
 * the GPU, so every call can be captured into a graph, and the same call gives the same bits.
 *
 * They write arrays that products read next: a program that keeps operand planes
 * (b200_operand_cache_enable) invalidates y, gx, gq, gk, gv and the gains' gradients after each call, as
 * after any write of its own (b200_operand_cache_invalidate).
 *
 * A tensor of heads is Shape({head, heads, tokens}): element (d, h, t) lies at
 *     d + head * h + ld * t,        ld >= head * heads, in elements.
 * `ld` (0 = dense) lets an operator work in the output of one product that holds queries, keys and
 * values of a token side by side, Shape({head * (heads_q + 2 heads_k), tokens}).  A minibatch of
 * Shape({head, heads, T}, batch) is the same as batch * T tokens.
 */
#ifndef PRIMITIV_B200_ATTENTION_H_
#define PRIMITIV_B200_ATTENTION_H_

#include "primitiv_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- rotary positions -----------------------------------------------------------------------
 *
 * The first `rot` elements of each head are turned in pairs, the others are copied:
 *     (a, b) -> amplitude * (a cos t - b sin t, b cos t + a sin t),   t = position * freqs[pair].
 * PAIRS: pair p is elements (2p, 2p + 1).  HALVES: elements (p, p + rot/2). */
enum { B200_ROTARY_PAIRS = 0, B200_ROTARY_HALVES = 1 };

/* Frequencies for rot/2 pairs, in radians per position (a pure host function):
 *     PLAIN     base^(-2p/rot)
 *     LINEAR    divided by `factor`: positions interpolated
 *     BASE      PLAIN with base * factor^(rot/(rot - 2)): the slowest pair is interpolated by
 *               `factor`, the fastest not at all
 *     BY_PARTS  pairs that turn less than once in `original` positions as LINEAR, more than 32
 *               times as PLAIN, between the two a blend that is linear in p: the share of LINEAR is
 *               (p - first) / (last - first) between 0 and 1, first = floor(pair(32)), last = ceil(pair(1)),
 *               pair(n) = rot ln(original / (2 pi n)) / (2 ln base), whether or not there are such pairs;
 *               amplitude 1 + 0.1 ln(factor), 1 in the other forms
 * `amplitude_host` may be NULL. */
enum { B200_ROTARY_PLAIN = 0, B200_ROTARY_LINEAR, B200_ROTARY_BASE, B200_ROTARY_BY_PARTS };
B200_API int b200_rotary_frequencies(uint32_t rot, double base, int scaling, double factor, double original,
                                     double *freqs_host, double *amplitude_host);

/* y = turned x; gx (+)= gy turned back, the transposed map.  head <= 256, rot even and <= head.
 * `freqs`: rot/2 doubles on the device.  `positions`: one per token, or NULL for 0, 1, 2, ...  Angles
 * position * freqs[pair] are formed and reduced in 64 bits, far positions with what the products round off, and
 * rounded to 32 bits then: at any position they are right to 2^-26 of a turn.
 * y may be x, and gx may be gy, with the same ld and without accumulate. */
B200_API int b200_rotary_fw(b200_ctx *ctx, int mode, const void *x, void *y, uint32_t head, uint32_t heads,
                            uint32_t tokens, uint64_t x_ld, uint64_t y_ld, uint32_t rot, int layout,
                            const double *freqs, float amplitude, const uint32_t *positions, void *stream);
B200_API int b200_rotary_bw(b200_ctx *ctx, int mode, const void *gy, void *gx, uint32_t head, uint32_t heads,
                            uint32_t tokens, uint64_t gy_ld, uint64_t gx_ld, uint32_t rot, int layout,
                            const double *freqs, float amplitude, const uint32_t *positions, int accumulate,
                            void *stream);

/* The same behind a norm of each head:  n = x / sqrt(mean(x^2) + eps), y = turned (n * gain).
 * The first heads_q heads of a token take gain_q, the next heads_k take gain_k (`head` elements each;
 * either count may be 0, then its gain may be NULL).  rot = 0 norms without turning.
 *     g = gy turned back;  ggain (+)= sum over tokens and heads of g n;
 *     gx (+)= (g gain - n mean(g gain n)) / sqrt(mean(x^2) + eps)
 * ggain_q / ggain_k may be NULL to skip both sums.  `scratch`: B200_NORM_ROTARY_SCRATCH floats of the
 * caller's, whose contents do not matter before or after; not needed (NULL) without the sums.
 * y may be x; gx may be gy without accumulate, and must not be x. */
#define B200_NORM_ROTARY_SCRATCH (512u * 512u)
B200_API int b200_norm_rotary_fw(b200_ctx *ctx, int mode, const void *x, const void *gain_q, const void *gain_k,
                                 void *y, uint32_t head, uint32_t heads_q, uint32_t heads_k, uint32_t tokens,
                                 uint64_t x_ld, uint64_t y_ld, uint32_t rot, int layout, const double *freqs,
                                 float amplitude, const uint32_t *positions, float eps, void *stream);
B200_API int b200_norm_rotary_bw(b200_ctx *ctx, int mode, const void *x, const void *gain_q, const void *gain_k,
                                 const void *gy, void *gx, void *ggain_q, void *ggain_k, float *scratch,
                                 uint32_t head, uint32_t heads_q, uint32_t heads_k, uint32_t tokens,
                                 uint64_t x_ld, uint64_t gy_ld, uint64_t gx_ld, uint32_t rot, int layout,
                                 const double *freqs, float amplitude, const uint32_t *positions, float eps,
                                 int accumulate_x, int accumulate_gain, void *stream);

/* ---- attention ---------------------------------------------------------------------------------
 *
 * For each sequence and each head h of q, with h' = h / (heads_q / heads_k) its head of k and v:
 *     s[i][j] = scale * sum_d q[i][d] k[j][d]         p = softmax over the j that i sees
 *     y[i][d] = sum_j p[i][j] v[j][d]                 lse[h][i] = log(sum_j exp(s[i][j]))
 * causal: query i of lq sees key j of lk when j <= i + lk - lq (the last query sees every key);
 * otherwise every query sees every key of its sequence.  A query that sees no key has y = 0,
 * lse = -infinity and no part in any gradient.  Keys, values and queries outside a sequence are never
 * used, whatever they hold.  Within a sequence a NaN or an infinity is not lost: it reaches every result
 * that depends on it, as a NaN or as what the formula makes of it: a query whose scores are all -infinity
 * has lse = -infinity too, but NaNs in y.  (Where a product gives such a value the weight zero, behind the diagonal of a causal
 * sequence, it may reach further, as a NaN: one of v or gy, and in the gradients one of any input.)
 *
 * Sequence i has its queries in rows q_starts[i], q_starts[i] + 1, ... of q, y (and their
 * gradients), its keys in rows k_starts[i], ... of k and v.  There are
 *     q_starts[i + 1] - q_starts[i] of them, or q_lens[i] if that is fewer (q_lens may be NULL);
 * starts must not decrease; what passes rows_q / rows_k is cut off.  Without q_starts (NULL),
 * sequence i has the rows from i * (rows_q / seqs) up to the next one's; the same for the keys.
 * So packed sequences, a padded minibatch, and a cache with room for more keys than it holds are all
 * the same call.  The arrays are on the DEVICE and are read by the kernels: a captured graph follows
 * them.  max_q / max_k say how long a sequence can be (0: not known); longer ones are cut.  They
 * choose the kernel: max_q = 1 is a step of generation.
 * Rows times heads, on either side, may be 2^31 - 2^16 at most, and heads_q * head less than 2^31
 * (B200_ERR_TOO_LARGE); offsets in elements may pass 32 bits.
 *
 * Arithmetic.  Scores, softmax statistics and all sums are in 32 bits.  B200_MODE_FP16: the weights p and, in
 * the gradients, ds (scaled by a power of two) are rounded to half as operands of their products, which
 * the tensor cores' rate asks for; delta = sum gy y is formed from y as it was stored.  So the error, by 2-norms,
 * is 2.6e-4 of y, 2.9e-4 of gv and 3.1e-4 of gq and gk (up to 3.7e-4 where causal sequences are shorter than
 * about 100) where rounding the results alone makes 2.1e-4; keys share one scale of ds with all queries that see them.
 * B200_MODE_FP32_3XTF32: three TF32 passes over operands split in two, which lose at most 2^-21 of an
 * operand.  B200_MODE_FP32_3XFP16 is the same here: its planes of halves are for products that find their operands
 * in memory.  B200_MODE_TF32: one pass, operands of 11 bits.  An infinity becomes a NaN where it is split.
 *
 * Rows of y and lse that belong to no sequence are left as they were.  Gradients of such rows are zero:
 * stored with accumulate = 0, left alone with 1. */
typedef struct b200_attention {
  uint32_t head, heads_q, heads_k;    /* head <= 256; heads_q a multiple of heads_k */
  uint32_t rows_q, rows_k;            /* tokens of q and y; of k and v */
  uint32_t seqs, max_q, max_k;
  uint64_t q_ld, k_ld, v_ld, y_ld;    /* 0 = dense; a gradient lies as what it is the gradient of */
  const uint32_t *q_starts, *q_lens;  /* seqs + 1 and seqs numbers on the device, or NULL */
  const uint32_t *k_starts, *k_lens;
  int32_t causal;
  float scale;
} b200_attention;

/* lse: Shape({rows_q, heads_q}) of float, or NULL where no backward pass follows.  y may not overlap q, k or v. */
B200_API int b200_attention_fw(b200_ctx *ctx, int mode, const b200_attention *plan_host, const void *q, const void *k,
                               const void *v, void *y, float *lse, void *stream);
/* gq, gk and gv from gy and from what the forward pass read and wrote.  No two of the arrays may
 * overlap, except that gq, gk and gv may lie side by side as q, k and v may.  `scratch`: floats of the caller's,
 * as many as b200_attention_bw_scratch says, whose contents do not matter before or after. */
B200_API int b200_attention_bw(b200_ctx *ctx, int mode, const b200_attention *plan_host, const void *q, const void *k,
                               const void *v, const void *y, const float *lse, const void *gy, void *gq, void *gk,
                               void *gv, float *scratch, int accumulate, void *stream);
B200_API int b200_attention_bw_scratch(const b200_attention *plan_host, uint64_t *floats_host);

#ifdef __cplusplus
}
#endif

#endif  /* PRIMITIV_B200_ATTENTION_H_ */
