/* hk -- a paged KV cache: append, attention, fork and compaction, exported by
 * libhk.so next to hk.h.
 *
 * Where hk_attention_decode reads the contiguous cache of one sequence, these
 * calls serve many sequences from one pool of pages, which sequences may share
 * (a common prompt, several answers to it).  No counterpart in the reference:
 * its engine keeps one cache [kv head][slot][64] on the host
 * (npu_llm/runtime/qwen_engine.py:52-63).
 *
 * Token j of sequence s is in slot j % page_size of page
 * table[s][j / page_size].  The pool of a layer is
 * [page][kv head][page_size][head_dim], keys and values apart.  All state is
 * the caller's device memory; the calls are asynchronous on `stream` (a
 * hipStream_t, NULL = the default stream), read their sizes from the device
 * and allocate nothing, so a captured call serves every later length.
 * hk_init comes first; the memory is of the device that is current at the
 * call.
 *
 * A generation step is one hk_paged_fork that makes room for the new tokens
 * (child = parent, keep = length), then per layer hk_paged_append and
 * hk_paged_attention.  The new tokens are the last ones of `length`.  A fork
 * that was refused leaves the lengths as they were, and an append after it
 * would store over the last tokens of the history, in pages that other
 * sequences may share.  So a caller who enqueues the step without a look at
 * the fork's status words in between (or captures it) names them in
 * cache->status: hk_paged_append then does nothing while the first of them is
 * not HK_PAGED_DONE.  (hk_paged_attention changes no cache; after a refused
 * fork its rows are those of the older tokens and say nothing.)
 *
 * Device contents are not seen by the host, so they are not refused but have
 * a meaning, and no memory outside the described one is touched whatever they
 * hold: a table entry outside [0, pages) has no page (its slots are never
 * seen, and what would be stored there is dropped), a length counts as one in
 * [0, table_width * page_size], a sequence outside [0, seqs) as one of length
 * 0, and `first` as values in [0, tokens].  Calls that write the same memory
 * must be ordered by the caller, as with any kernel.
 *
 * Arrays of int32 and float32 are aligned to 4 bytes, others as said below.
 *
 * A call that returns HK_ERR_HIP could not make one of its launches (an error
 * that an earlier HIP call has left is not taken for that).  After a fork, or a
 * compaction in place, that returns it the cache is not to be used further:
 * its tables may name pages that nobody has filled.
 */
#ifndef HK_PAGED_H
#define HK_PAGED_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HK_PAGED_BF16 0 /* dtype: bf16 bits */
#define HK_PAGED_E4M3 1 /* dtype: OCP e4m3 times a float32 scale per layer and kv head */

/* Bytes of device memory that hk_paged_attention, hk_paged_fork and
 * hk_paged_compact use while they run, 256-byte aligned and set to zero once
 * before its first use (the calls leave it fit for the next).  Calls that may
 * overlap in time each need their own. */
#define HK_PAGED_WORKSPACE 100663296

#define HK_PAGED_MAX_BATCH 4096 /* sequences in one call */

typedef struct hk_paged_cache {
  void* k;              /* pools: layer l, page p at (l * layer_stride + p * page_stride) elements */
  void* v;
  const float* k_scale; /* [layers, kv_heads], finite and positive (HK_PAGED_E4M3), else NULL */
  const float* v_scale;
  int32_t* table;       /* [seqs, table_width] pages; -1 from the sequence's last page on */
  int32_t* length;      /* [seqs] tokens, the new ones of this step included */
  int32_t* refs;        /* [pages] table entries that name the page; 0: free */
  int64_t layer_stride; /* elements, at least kv_heads * page_size * head_dim, multiples of 16 bytes */
  int64_t page_stride;
  int32_t layers;
  int32_t kv_heads;
  int32_t head_dim;     /* 64 or 128 */
  int32_t page_size;    /* 16, 32, 64, 128 or 256 slots */
  int32_t pages;
  int32_t seqs;
  int32_t table_width;  /* pages of a sequence at most */
  int32_t dtype;        /* HK_PAGED_BF16 or HK_PAGED_E4M3 */
  const int32_t* status; /* optional: the status words of the step's hk_paged_fork, for hk_paged_append */
} hk_paged_cache;

/* The batch of an append or an attention: entry b is sequence seqs[b] (seqs
 * NULL: sequence b), and its new tokens are rows first[b] .. first[b + 1] - 1
 * of the `tokens` rows, the last first[b + 1] - first[b] tokens of its length.
 * `first` has n + 1 values that do not decrease; an entry may have no rows.
 * Rows of no entry are left as they were. */

/* RoPE and KV append for one layer: of each row (q heads, k heads, v heads,
 * bf16, rows `qkv_stride` elements apart) the queries go to q_out (bf16, rows
 * q_out_stride apart; the rows of qkv themselves if q_out == qkv and the
 * strides are equal; NULL: no queries), the keys and values into their pages.
 * x1 cos - x2 sin, x2 cos + x1 sin over the two halves of a head, one rounding
 * to bf16 (the numbers hk_attention_decode appends); HK_PAGED_E4M3: rounded
 * from x / scale instead, saturated at +-448.  cos and sin: [positions,
 * head_dim / 2] float32 with positions >= table_width * page_size, or both
 * NULL for no rotation.  Tokens at negative positions (more rows than length)
 * are dropped, and their queries left as they were.  A sequence is listed
 * once.  Fewer than 2^24 tokens.  Pointers and strides are multiples of 16
 * bytes.  With cache->status, neither pages nor q_out are written unless its
 * first word is HK_PAGED_DONE. */
int hk_paged_append(const hk_paged_cache* cache, int32_t layer, const uint16_t* qkv, int64_t qkv_stride,
                    const float* rope_cos, const float* rope_sin, int32_t positions, const int32_t* seqs,
                    const int32_t* first, int32_t n, int32_t tokens, int32_t q_heads, uint16_t* q_out,
                    int64_t q_out_stride, void* stream);

/* Causal grouped-query attention of the batch's new tokens over their cached
 * slots, the new ones included: the row at position p of head h sees the slots
 * j <= p, with `window` > 0 only those with j > p - window, of kv head
 * h / (q_heads / kv_heads).  out = sum_j softmax_j(scale q . k_j) v_j (bf16,
 * rows out_stride elements apart); lse (optional, float32 [tokens, q_heads]) =
 * ln sum_j exp(scale q . k_j), by which results over parts of a context are
 * joined.  A row that sees nothing gets zeros and -inf.  Slots that a row does
 * not see have no influence on it, whatever they hold.  scale is finite and
 * positive; a score above float32's range makes its row NaN.
 * out may be q itself, if the strides are equal.  max_new: the largest count
 * of rows of one entry, as far as the caller knows it; it chooses between
 * forms of the kernel and every value gives the same result, up to float32
 * summation order.  At most 2^30 rows
 * (tokens x q_heads).  Pointers and strides are multiples of 16 bytes. */
int hk_paged_attention(const hk_paged_cache* cache, int32_t layer, const uint16_t* q, int64_t q_stride,
                       const int32_t* seqs, const int32_t* first, int32_t n, int32_t tokens, int32_t max_new,
                       int32_t q_heads, float scale, int32_t window, uint16_t* out, int64_t out_stride, float* lse,
                       void* workspace, void* stream);

/* Status words of hk_paged_fork. */
#define HK_PAGED_DONE 0
#define HK_PAGED_BAD_ENTRY 1 /* status[1]: the first entry that is not valid */
#define HK_PAGED_FULL 2      /* status[1]: pages that are missing */

/* All n entries at once: sequence child[i] becomes the first keep[i] tokens of
 * sequence parent[i] as they were before the call, with pages for grow[i]
 * tokens more; its length becomes keep[i] + grow[i].  Pages that keep fills are
 * shared; of a partly filled last page the child gets its own copy (its first
 * keep % page_size slots, every layer), or the page itself if nobody else
 * keeps it.  What the children held before is released first, and new pages
 * are the free ones of lowest number, in order of entries.  So
 *   next tokens     child = parent, keep = length, grow = their count
 *   a second answer child another sequence, keep = length (or less: a prefix)
 *   taking back     child = parent, keep < length
 *   freeing         keep = grow = 0
 * and beams are reordered in one call.  Device arrays: child NULL: i; parent
 * NULL: child[i]; keep NULL: length[parent[i]]; grow NULL: 0; they may be the
 * cache's own `length`.  An entry is valid if child is in [0, seqs) and no
 * earlier entry's, 0 <= keep <= length[parent] (parent in [0, seqs), or any
 * value where keep is 0), grow >= 0, keep + grow fits the table, and the partly
 * filled page is there.  status (device, 2 words): HK_PAGED_DONE, or why
 * nothing at all was changed.  refs has to be what the tables say.  One
 * sequence may be the parent of several entries.  n <= seqs. */
int hk_paged_fork(const hk_paged_cache* cache, const int32_t* child, const int32_t* parent, const int32_t* keep,
                  const int32_t* grow, int32_t n, int32_t* status, void* workspace, void* stream);

/* Moves the live pages (refs > 0) into the first pages of the pool: with L of
 * them, the i-th live page from L on goes to the i-th free page below L, in
 * every layer.  table_out [seqs, table_width] and refs_out [pages] receive the
 * tables and counts (cache->table and cache->refs themselves: in place; else
 * those stay as they were, and the moved pages are still at their old place
 * too), live_out (device) L.  Pages from L on are free afterwards. */
int hk_paged_compact(const hk_paged_cache* cache, int32_t* table_out, int32_t* refs_out, int32_t* live_out,
                     void* workspace, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HK_PAGED_H */
