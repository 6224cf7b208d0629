/* More than one continuation of a sequence over a paged cache, on gfx950: drafted tokens that
 * form a tree, beams, and the pages and states that both share, move and free.
 *
 * Conventions as in tf_decode.h: device pointers, work enqueued on `stream`, nothing
 * allocated, nothing synchronised, 0 or an error code with tfd_last_error()'s text.  A page
 * holds 16 positions; position p of a row lies in page page_table[p / 16], row p % 16.  Values
 * that memory is indexed with are checked on the device: a bad one raises a bit in `err` (NULL:
 * nothing) and its access is left out.  The reference decodes one continuation a sequence
 * (fast/engine.py:239-271); the formulas here are this library's definition. */
#ifndef TF_SEARCH_H
#define TF_SEARCH_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* device error bits besides tf_decode.h's */
#define TFD_ERR_ROW_RANGE 64  /* a parent, path or count outside its range */
#define TFD_ERR_NO_PAGES 128  /* more pages wanted than are free */

/* ---- drafted trees ------------------------------------------------------------------ */
#define TFD_TREE_MAX_NODES 256
/* Masks and depths of each row's tree: node t's parent is parents[t] < t, -1 a root.  Bit n
 * of masks[row][t] (words = ceil(nodes / 64) 64-bit words) is set where n is t or one of its
 * ancestors; depths[row][t] counts them, less one.  Nodes from counts[row] on (counts NULL:
 * none) get empty masks and depth 0.  parents [rows][nodes], nodes <= 256.  A parent outside
 * its range raises TFD_ERR_ROW_RANGE and counts as -1. */
int tfd_tree_masks(const int32_t* parents, const int32_t* counts, int rows, int nodes,
                   uint64_t* masks, int32_t* depths, int32_t* err, void* stream);
/* The path that the picks follow: from node 0, the lowest child whose token is its parent's
 * pick, and so on.  path [rows][nodes]: the nodes in order, -1 behind them; accepted[row]: how
 * many (0 for a row of no nodes); next[row]: the last one's pick (-1). */
int tfd_tree_accept(const int32_t* tokens, const int32_t* parents, const int32_t* picks,
                    const int32_t* counts, int rows, int nodes, int32_t* path,
                    int32_t* accepted, int32_t* next, void* stream);

/* tf_decode.h's tfd_panel_qkv_append for drafted nodes: row m is rotated to position pos[m] (that
 * of its depth), and its key and value go to position slot[m] of sequence seq[m]'s pages; a
 * row with slot[m] < 0 is not there. */
int tfd_tree_qkv_append(const float* part, int slices, int M, int heads, int kv_heads,
                        int head_dim, const void* gamma_q, const void* gamma_k,
                        const void* cos_table, const void* sin_table, int rope_rows,
                        const int32_t* pos, const int32_t* slot, const int32_t* seq,
                        const int32_t* page_table, int max_pages, void* k_pool, void* v_pool,
                        int num_pages, float scale, float eps, void* q_out, int32_t* err,
                        void* stream);
/* Attention of drafted nodes.  Row b's nodes have their keys and values at positions
 * lengths[b] + t of its pages.  Node t attends to every position below lengths[b] and to node n
 * where bit n of masks[b][t] is set and n < counts[b]:
 *   out = sum_j softmax_j(scale q . k_j) v_j,
 * scores and sums in f32, one rounding of the output; the probabilities, a product's operands,
 * are sums of two bf16 (2^-16 of each).  With `rounded` they may be one bf16 (2^-8), for speed,
 * where tfd_tree_attn_form says many.  A node that sees nothing gets zeros.  What a node does not
 * see takes no part, values that are not finite included, nor do positions of a page that is none
 * of the pool's (TFD_ERR_PAGE_RANGE).  q bf16, rows / nodes / heads q_row / q_node / q_head
 * elements apart (multiples of 8; q, the pools and out 16-byte aligned).  out:
 * [rows][nodes][heads][head_dim], or
 * with out_panel the rows x nodes rows of tf_decode.h's panel order.  Nodes from counts[b] on
 * are not written.  head_dim 64, 128 or 256; heads a multiple of kv_heads; nodes <= 256; up to
 * 2^26 positions a row.  work: tfd_tree_attn_work_bytes, 16-byte aligned, contents free, one
 * call's at a time. */
typedef struct {
  const void* q;
  int64_t q_row, q_node, q_head;
  const void* k_pool;
  const void* v_pool;
  const int32_t* page_table; /* [rows][max_pages] */
  const int32_t* lengths;    /* [rows] */
  const int32_t* counts;     /* [rows] or NULL */
  const uint64_t* masks;     /* [rows][nodes][ceil(nodes / 64)] */
  int rows, nodes, heads, kv_heads, head_dim, max_pages, num_pages;
  float scale;
  void* out;
  int out_panel;
  void* work;
  int64_t work_bytes;
  int32_t* err;
  int rounded;
} TfdTreeAttnArgs;
int64_t tfd_tree_attn_work_bytes(int rows, int nodes, int heads, int kv_heads, int head_dim,
                                 int max_pages);
/* How a call of these sizes runs on the current device, for tests and measurements: form = 16s of
 * columns that a wave with its own positions takes (0: waves share positions and each takes
 * other columns), waves of a block, blocks for a row's columns, splits of its positions. */
int tfd_tree_attn_form(int rows, int nodes, int heads, int kv_heads, int head_dim, int max_pages,
                       int32_t form[4]);
int tfd_tree_attn(const TfdTreeAttnArgs* args, void* stream);

/* ---- beams -------------------------------------------------------------------------- */
#define TFD_BEAM_MAX 64
#define TFD_BEAM_MAX_VOCAB 1048576
/* The next beams of `groups` sequences of `beams` each.  Row r = group * beams + beam:
 *   candidate  token t of row r: score[r] + x_t - log(sum_u exp(x_u)); a finished row (done)
 *              offers itself alone, its score as it is and the token eos.  A logit that is NaN
 *              or -inf is no candidate and not in the sum, +inf counts as the largest f32; a
 *              row whose score is NaN or infinite offers nothing;
 *   rank       the candidate's score / max(length, 1) ^ penalty, length = lengths[r] + 1 (a
 *              finished row: lengths[r]), in 64 bits.  The sum in a score's logarithm is one of
 *              f32 exponentials, up to 2^-22 of it off: two rows' candidates that lie closer
 *              than that may come in either order, a row's own and equal rows' never;
 *   beams      the best of a group's candidates, in falling rank; equal ones by the lower row,
 *              in a row by the larger logit, then the lower token.
 * Out, per place: parents (row numbers), tokens, scores (f32), lengths and done (a parent's, or
 * eos was taken).  Places for which no candidate is left hold their own row as parent, token
 * -1, score -inf, and that row's length and done.  eos -1: no token finishes.
 * logits f32, bf16 or f16 [rows][ldl]; lengths NULL: zeros, done NULL: none (uint8).
 * vocab <= 2^20, groups <= 65535, beams <= 64, rows x vocab / 1024 below 2^23.  work:
 * tfd_beam_work_bytes, 16-byte aligned, contents free, one call's at a time.  The outputs must
 * not be the inputs. */
typedef struct {
  const void* logits;
  int64_t ldl;
  int type;
  const float* scores;
  const int32_t* lengths;
  const uint8_t* done;
  int groups, beams, vocab, eos;
  double penalty;
  int32_t* parents;
  int32_t* tokens;
  float* scores_out;
  int32_t* lengths_out;
  uint8_t* done_out;
  void* work;
  int64_t work_bytes;
} TfdBeamArgs;
int64_t tfd_beam_work_bytes(int groups, int beams, int vocab);
int tfd_beam_select(const TfdBeamArgs* args, void* stream);

/* Rows of `n` tensors moved to the rows that continue them, in place: row r becomes what row
 * parents[r] was.  Groups of `beams` rows (<= 64); a parent lies in its row's group (another one
 * raises TFD_ERR_ROW_RANGE and leaves the row as it is).  `states`: a device array; first_block
 * = the running sum of tfd_state_blocks of the tensors before, `blocks` the sum of all (below
 * 2^24; a block takes 4 KiB of a row, fewer of tensors whose rows are no multiples of 16 bytes). */
typedef struct {
  void* base;         /* [rows][row_bytes] */
  int64_t row_bytes;
  int64_t first_block;
} TfdState;
int64_t tfd_state_blocks(const void* base, int64_t row_bytes);
int tfd_reorder_states(const TfdState* states, int n, int64_t blocks, const int32_t* parents,
                       int groups, int beams, int32_t* err, void* stream);

/* ---- pages -------------------------------------------------------------------------- */
#define TFD_PAGES_MAX_ROWS 1024
/* One tensor of pages: [num_pages][heads][16][row_bytes], 16-byte aligned, row_bytes a multiple
 * of 16. */
typedef struct {
  void* base;
  int64_t page_bytes; /* heads * 16 * row_bytes */
  int32_t heads, row_bytes;
} TfdPool;
/* A cache's pages: table int32 [rows][max_pages], -1 for no page, and refs int32 [num_pages],
 * the table entries that name a page (0: free).  scratch: int32 [TFD_PAGES_SCRATCH], zero before
 * the first call and left ready by each.  Calls on one cache are stream-ordered. */
#define TFD_PAGES_SCRATCH(rows, max_pages, num_pages) \
  (3 * (int64_t)(num_pages) + (int64_t)(rows) * (max_pages) + 2 * (int64_t)(rows) + 16)
typedef struct {
  const TfdPool* pools;   /* device array */
  int n_pools;
  int64_t max_page_bytes; /* the largest of theirs */
  int32_t* table;
  int32_t* refs;
  int rows, max_pages, num_pages;
  int32_t* scratch;
  int32_t* err;
} TfdPages;
/* Row r becomes what row parents[r] was: its pages up to lengths[parents[r]] are shared and
 * lengths_out[r] is that length.  parents[r] = -1 empties the row (length 0); = r leaves its
 * entries as they are.  Without parents, the rows with which[r] != 0 are emptied and lengths and
 * lengths_out are not used.  A page that no entry names any more is free. */
int tfd_pages_fork(const TfdPages* pages, const int32_t* parents, const uint8_t* which,
                   const int32_t* lengths, int32_t* lengths_out, void* stream);
/* Pages for positions lengths[r] .. lengths[r] + n - 1 of every row (n: counts[r], or n_all with
 * counts NULL), each the row's own: where there is none, or where others share it, the row
 * gets a free page, and what a shared page holds below lengths[r] is copied (all pools).  If all
 * that share a page want it, the first of them keeps it.  New pages are the free ones of lowest
 * number, in the order of rows and positions.  With none left the entry becomes -1 and
 * TFD_ERR_NO_PAGES is raised; positions past max_pages raise TFD_ERR_POS_RANGE. */
int tfd_pages_take(const TfdPages* pages, const int32_t* lengths, const int32_t* counts,
                   int n_all, void* stream);
/* Page dst[i] of every pool becomes page src[i]; no page is in both lists or twice in dst.  A pair
 * with a number outside the pools raises TFD_ERR_PAGE_RANGE and is left out. */
int tfd_pages_copy(const TfdPages* pages, const int32_t* src, const int32_t* dst, int n,
                   void* stream);
/* Positions lengths[r] + path[r][i] move to lengths[r] + i, i < counts[r], in every pool, and
 * lengths_out[r] = lengths[r] + counts[r].  path [rows][nodes] rises strictly from 0 on along a
 * row (else TFD_ERR_ROW_RANGE, the row stays and keeps its length). */
int tfd_pages_keep(const TfdPages* pages, const int32_t* lengths, const int32_t* path,
                   const int32_t* counts, int nodes, int32_t* lengths_out, void* stream);
/* The pages in use move to the numbers 0 .. live - 1: those from `live` on, in rising order, to
 * the free ones below it, in rising order.  live: one int32. */
int tfd_pages_compact(const TfdPages* pages, int32_t* live, void* stream);

#ifdef __cplusplus
}
#endif

#endif
