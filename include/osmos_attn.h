/* libosmos MI355X - a paged cache of keys and values on the device, and the attention that reads it: the rows that stand
   between a decoder layer's dense products (mm.h, mv.h) and its experts. no counterpart in the reference's kernel ABI.

   a cache is one piece of device memory, [layer][keys, values][page][head][slot][dim]: page p holds `page` tokens in
   each of 2 `layers` planes. a sequence's token t lies in slot t % page of page table[t / page]. values are F16, BF16 or
   F8 (OCP e4m3; a stored value stands for itself times scale[layer][keys, values][head]).

   a step is the rows that a call brings: sequence s the rows start[s] .. start[s + 1] - 1, its last tokens of len[s]
   (len counts them already), so that row t is token len[s] - (start[s + 1] - t). every call takes the step's numbers
   from device memory and clamps what it reads there: a row or a page id out of range is left out (its keys count as
   masked, its values are not written), never followed.

   every call is queued on `stream` (a hipStream_t) and never waited for, allocates nothing and may be captured into a
   graph; false = refused, nothing queued. */
#ifndef OSMOS_ATTN_H
#define OSMOS_ATTN_H

#include <stdbool.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define OSMOS_F32 0u     /* (the GGUF ids) */
#define OSMOS_F16 1u
#define OSMOS_BF16 30u
#define OSMOS_F8 0x200u  /* e4m3, saturating at 448; no GGUF id */
#define OSMOS_ATTN_MAX_DIM 256u
#define OSMOS_ATTN_MAX_STRIDE (1u << 24) /* values between two packed rows of keys or values */
#define OSMOS_KV_MAX_PAGE 4096u
#define OSMOS_KV_MAX_PAGE_VALUES (1u << 28) /* heads x page x dim */
#define OSMOS_KV_MAX_REQUESTS 1024u

typedef struct OsmosKv
{
  void *data;           /* osmos_kv_bytes bytes, 16-byte aligned */
  const float *scale;   /* F8: 2 layers x heads floats on the device, or NULL for ones; other types: NULL */
  uint32_t type;        /* OSMOS_F16, OSMOS_BF16 or OSMOS_F8 */
  uint32_t layers, pages;
  uint32_t page;        /* tokens a page: a power of two up to OSMOS_KV_MAX_PAGE */
  uint32_t heads, dim;  /* dim: a multiple of 16 up to OSMOS_ATTN_MAX_DIM; heads x page x dim up to
                           OSMOS_KV_MAX_PAGE_VALUES */
} OsmosKv;

typedef struct OsmosKvStep
{
  const int32_t *start; /* n_seq + 1 row numbers, ascending, the last at most n_tok */
  const int32_t *len;   /* seqs: the tokens of each sequence, the step's among them */
  const int32_t *table; /* seqs rows of table_stride page ids; ids past a sequence's pages are not read */
  const int32_t *seq;   /* n_seq: the step's sequences' rows in len and table; NULL: 0 .. n_seq - 1 */
  uint32_t n_seq, n_tok;
  uint32_t max_tok;     /* no sequence brings more rows */
  uint32_t max_len;     /* no sequence has more tokens: later keys are left out */
  uint32_t seqs, table_stride;
  const int32_t *live;  /* n_seq, or NULL: 0 for a sequence that takes no part in this step (osmos_kv_grow's `done`, as its
                           tokens are not in len): its rows are not written, and see no key */
} OsmosKvStep;

/* the bytes of a cache's data; 0 for a shape or type out of range */
uint64_t osmos_kv_bytes(const OsmosKv *kv);

/* the step's rows into the pages: k and v n_tok rows of heads x dim values of `type` (F32, F16 or BF16; row t at
   k + t k_stride values, 16-byte aligned rows), each value rounded once to the cache's type (nearest, ties to even;
   F8: the float quotient value / scale, saturating; NaN stays NaN). */
bool osmos_kv_append(const OsmosKv *kv, uint32_t layer, const OsmosKvStep *step, uint32_t type, const void *k,
                     uint64_t k_stride, const void *v, uint64_t v_stride, void *stream);

/* softmax(scale q k^T) v for the step's rows: row t's head h at q + t q_stride + h q_head (values; likewise out), over
   its kv head h / (heads / kv heads). a row sees the tokens of its sequence up to its own, with `window` (0: all) the
   last `window` of them. a row that sees none gets zeros. lse (may be NULL): n_tok x heads, the logarithm of the
   row's sum of exp(scale q k), -infinity for a row that sees none. what is masked has no influence, infinities and NaN
   among it. q and out F32, F16 or BF16. products on the matrix units in the keys' type (F8: q's, F16 for F32), sums
   and softmax in F32: an F32 q and the probabilities (times a power of two in F16) are rounded to that type first, a q past
   F16's range to an infinity. */
typedef struct OsmosAttn
{
  const void *q;
  void *out;
  float *lse;
  uint64_t q_stride, q_head, out_stride, out_head;
  uint32_t q_type, out_type;
  uint32_t heads;       /* a multiple of the kv heads */
  uint32_t window;
  float scale;
} OsmosAttn;

/* keys and values as packed rows, laid out as q is (for prompts that need no cache): F16 or BF16 */
typedef struct OsmosKvRows
{
  const void *k, *v;
  uint64_t k_stride, k_head, v_stride, v_head;
  uint32_t type, heads, dim;
} OsmosKvRows;

/* the most device memory (256-byte aligned) that an attention call over the step needs as its workspace, 0 for none; a
   workspace is written before it is read, and calls that share one are ordered on one stream */
uint64_t osmos_attn_workspace(const OsmosAttn *a, uint32_t kv_heads, uint32_t dim, const OsmosKvStep *step);
/* whole prompts: row t's keys are its sequence's rows up to t (step->len, table, seq, live unused: NULL) */
bool osmos_attn_prompt(const OsmosAttn *a, const OsmosKvRows *kv, const OsmosKvStep *step, void *workspace,
                       uint64_t workspace_bytes, void *stream);
/* rows over the cache (the step's own among its tokens: osmos_kv_append goes first) */
bool osmos_attn_chunk(const OsmosAttn *a, const OsmosKv *kv, uint32_t layer, const OsmosKvStep *step, void *workspace,
                      uint64_t workspace_bytes, void *stream);
/* osmos_attn_chunk where every sequence brings one row or none (max_tok 1): the cache read once for each 16 query heads of a kv
   head, split over its length.
   refused: n_seq sequences of max_len tokens, or of what a table row holds, past 2^32 tiles of 32 tokens */
bool osmos_attn_token(const OsmosAttn *a, const OsmosKv *kv, uint32_t layer, const OsmosKvStep *step, void *workspace,
                      uint64_t workspace_bytes, void *stream);

/* which pages are whose, on the device: ref[p] how many sequences hold page p (0: free), len and table as in
   OsmosKvStep, a table row's ids past its pages -1. the operations take request lists of up to
   OSMOS_KV_MAX_REQUESTS sequences in device memory and act in stream order with no host round trip; their outcome is
   fixed by the lists' order. `done` (n, may be NULL): 1 for a request carried out, 0 for a refused one, which changes
   nothing. a step queued behind osmos_kv_grow takes its `done` as OsmosKvStep's live: without it a refused sequence's
   rows would be written over the last tokens it has, in pages that others may hold too. */
typedef struct OsmosKvPool
{
  int32_t *ref;         /* pages, 16-byte aligned */
  int32_t *len;         /* seqs */
  int32_t *table;       /* seqs x table_stride */
  void *scratch;        /* osmos_kv_scratch bytes, 16-byte aligned: written before it is read */
  uint32_t seqs, table_stride;
} OsmosKvPool;

uint64_t osmos_kv_scratch(const OsmosKv *kv);
/* sequence seq[i] gets add[i] (at least 0) more tokens: pages for them from the lowest free ids, in the requests' order.
   a last, partly filled page that others hold too is first copied to one of its own; the last of its holders keeps it.
   refused: a sequence out of range or earlier in the list, more tokens than its table row holds, and, from the first
   request on that the free pages do not cover, all */
bool osmos_kv_grow(const OsmosKv *kv, const OsmosKvPool *pool, const int32_t *seq, const int32_t *add, uint32_t n,
                   int32_t *done, void *stream);
/* the empty sequence to[i] gets all tokens of from[i], holding the same pages. refused: a sequence out of range, a `to`
   that has tokens or is earlier in the list, a `from` that is a `to` of the list */
bool osmos_kv_fork(const OsmosKv *kv, const OsmosKvPool *pool, const int32_t *from, const int32_t *to, uint32_t n,
                   int32_t *done, void *stream);
/* sequences emptied, their pages let go (a sequence listed twice or out of range: nothing more) */
bool osmos_kv_free(const OsmosKv *kv, const OsmosKvPool *pool, const int32_t *seq, uint32_t n, void *stream);
/* the pages in use moved to ids 0 .. live - 1: the j-th of those past them to the j-th free id below, the tables
   following; live (may be NULL): how many there are */
bool osmos_kv_compact(const OsmosKv *kv, const OsmosKvPool *pool, int32_t *live, void *stream);
/* page from[i] of every plane to page to[i] (an id out of range: that pair left out); no `to` twice or among `from` */
bool osmos_kv_copy(const OsmosKv *kv, const int32_t *from, const int32_t *to, uint32_t n, void *stream);

#ifdef __cplusplus
}
#endif

#endif
