/* libosmos MI355X - the rows between a decoder block's products: the root-mean-square norm with the residual's addition,
   in the forms that the products read; rotary positions, on packed rows or on their way into the paged cache
   (osmos_attn.h); and the choice of the next token from a row of logits. no counterpart in the reference's kernel ABI.

   types are osmos_attn.h's (OSMOS_F32, _F16, _BF16). every call is queued on `stream` (a hipStream_t) and never waited
   for, allocates nothing and may be captured into a graph; false = refused, nothing queued (among what is: more rows than a
   launch of fewer than 2^32 threads holds, at 64 a row or more, 1024 for osmos_sample). */
#ifndef OSMOS_ROWS_H
#define OSMOS_ROWS_H

#include <stdbool.h>
#include <stdint.h>

#include "osmos_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define OSMOS_NORM_MAX_DIM 65536u

/* s = x + add (float, rounded once); y = (s r) (weight + offset), each product rounded, with r = 1 / sqrt(mean of s^2 + eps)
   rounded once from float64 (the squares are exact and summed in float64, in an order that type and dim alone fix: a row's bits
   do not depend on the other rows, on their number or on what else is written). n rows of dim values, row t at x + t x_stride
   (values). outputs, any of them:
     sum      s, rounded once to `type`; may be x or add (in place)
     out      y, rounded once to out_type
     x16      y as mm_x16's tiles (include/osmos/gpu/mm.h), the bytes that mm_x16 makes of float rows y, the rows past n up to a
              whole tile zero; *overflow (wanted with it) set to 1 for a value past F16's range, left as it is otherwise
     codes    y as q8_round's codes and scales (include/osmos/gpu/q8.h), the bytes that q8_round makes of float rows y
   weight: dim values of weight_type, NULL for ones. refused: no rows or output, dim over OSMOS_NORM_MAX_DIM, or not whole
   16s (x16) or 32s (codes), eps under 0, more than one row at a stride under dim; x16 and codes are 16-byte aligned. the
   other pointers are aligned to their values. out, x16, codes and scales overlap no input */
typedef struct OsmosNorm
{
  const void *x, *add;  /* of `type`; add NULL: none */
  void *sum;
  const void *weight;
  void *out, *x16;
  int32_t *overflow;
  int8_t *codes;
  float *scales;        /* n x dim / 32 */
  uint64_t x_stride, add_stride, sum_stride, out_stride;
  uint32_t type, weight_type, out_type;
  uint32_t n, dim;
  float eps, offset;
} OsmosNorm;

bool osmos_norm(const OsmosNorm *a, void *stream);

/* rotary positions: a head's pair i < rot / 2 turned by position x turns[i] whole turns, (a, b) -> (a c - b s, b c + a s) with
   c and s the angle's cosine and sine times `scale`; the values from rot on stay. the product is formed exactly and its
   fraction of a turn in float64, so that far positions turn by turns[i] as exactly as near ones, up to 2^53 turns (a table's
   own rounding to float64 grows with the position: osmos_rope_turns' first pair, unscaled, is 2^-25 of a turn off at 2^31). */
#define OSMOS_ROPE_HALVES 0u /* pair i: values i and i + rot / 2 */
#define OSMOS_ROPE_PAIRS 1u  /* pair i: values 2 i and 2 i + 1 */

/* what the turns of a longer context are made from: base^(-2 i / rot) radians a token, then
     LINEAR   all divided by factor
     NTK      base times factor^(rot / (rot - 2)) instead
     YARN     pairs that make `slow` turns or less in `context` tokens divided by factor, those of `fast` or more as they are, a
              ramp over the pairs' numbers between; the cosines and sines times 0.1 ln(factor) + 1
     BANDS    the same with `low` and `high` turns and a ramp over the turns */
#define OSMOS_ROPE_PLAIN 0u
#define OSMOS_ROPE_LINEAR 1u
#define OSMOS_ROPE_NTK 2u
#define OSMOS_ROPE_YARN 3u
#define OSMOS_ROPE_BANDS 4u
typedef struct OsmosRopeScaling
{
  uint32_t kind;
  double base, factor, context;
  double low, high;  /* turns: BANDS' low and high, YARN's slow and fast */
} OsmosRopeScaling;
/* host code: turns[0 .. rot / 2), whole turns a token (to be copied to the device), and *scale. false: a number out of range */
bool osmos_rope_turns(const OsmosRopeScaling *s, uint32_t rot, double *turns, float *scale);

typedef struct OsmosRope
{
  const double *turns;  /* rot / 2, on the device */
  const float *q_weight, *k_weight; /* NULL, or dim values: each head of q (of k) is first normed, y = x / sqrt(mean of x^2 +
                           eps) (weight + offset), in float */
  const void *q, *k;    /* rows of `type`, row t's head h at q + t q_stride + h q_head (values); 16-byte aligned rows and heads */
  void *q_out, *k_out;  /* of out_type; may be q and k themselves with the same strides and type */
  uint64_t q_stride, q_head, k_stride, k_head, q_out_stride, q_out_head, k_out_stride, k_out_head;
  uint32_t type, out_type;
  uint32_t heads, kv_heads; /* kv_heads 0: no k */
  uint32_t n, dim;      /* dim a multiple of 8 up to OSMOS_ATTN_MAX_DIM */
  uint32_t rot;         /* even, up to dim */
  uint32_t layout;
  float scale, eps, offset;
} OsmosRope;

/* row t at position pos[t] (device memory; may be negative) */
bool osmos_rope(const OsmosRope *a, const int32_t *pos, void *stream);
/* the step's rows at their tokens' places, q into q_out, k turned and v as it is into the layer's pages as osmos_kv_append
   writes them (k_out and its strides unused; a->dim and kv_heads are the cache's): v's rows of `type` as k's. what
   osmos_kv_append leaves out is left out; the q rows of no token (behind the last sequence, of one that takes no part, past
   max_len) are left as they are */
bool osmos_rope_append(const OsmosRope *a, const OsmosKv *kv, uint32_t layer, const OsmosKvStep *step, const void *v,
                       uint64_t v_stride, uint64_t v_head, void *stream);

/* one token for each row of logits. token i of a row has the weight exp(logit / temperature) (in float64 arithmetic); the
   tokens stand in the order of their logits, the greatest first, the lower index first among equals; of these are kept
     the first top_k (0 or less: all),
     of those the first whose weights sum up to top_p of theirs (1 or more: all; at least one token), and
     those of at least min_p times the greatest weight (0 or less: all; over 1: as 1);
   drawn is the first kept token whose running sum of weights passes u (0 <= u < 1) times the kept ones' sum. temperature 0,
   less or NaN: the first token. a logit of -infinity or NaN is never chosen nor kept, +infinity counts as its type's
   greatest value; a row of nothing else gives token -1, prob 0, kept 0. the sums are whole numbers of 2^-42 of the greatest weight: a
   weight under 2^-44.5 of it counts as zero, and the tokens of each 23rd of an octave are summed and then rounded to such a unit, so
   that one of under 2^-43 by itself adds nothing. NaN in top_p or min_p: that limit does not hold; u is clamped into its range, NaN
   counts as 0. outputs overlap neither inputs nor one another.
   the same call gives the same answer, and a row's answer does not depend on the other rows. */
#define OSMOS_SAMPLE_MAX_VOCAB (1u << 20)
typedef struct OsmosSample
{
  const void *logits;   /* n rows of `vocab` values of `type`, row t at logits + t stride; aligned to their values */
  const float *u;       /* n */
  const float *temperature, *top_p, *min_p; /* n each, or NULL: 1, 1, 0 */
  const int32_t *top_k; /* n, or NULL: 0 */
  int32_t *token;       /* n */
  float *prob;          /* n, or NULL: the drawn token's part of the kept weights */
  int32_t *kept;        /* n, or NULL: how many tokens were kept */
  float *probs;         /* n x vocab, or NULL: every token's part of the kept weights, 0 for those not kept */
  uint64_t stride;
  uint32_t type, n, vocab;
} OsmosSample;

/* the device memory (256-byte aligned) that the call needs as its workspace, 0 for none; what a workspace holds before a call
   does not matter, and calls that share one are ordered on one stream */
uint64_t osmos_sample_workspace(const OsmosSample *a);
bool osmos_sample(const OsmosSample *a, void *workspace, uint64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif
