/* C-ABI of the attention side of a decoder layer: a paged key-value cache, the store of new tokens into it (norms of
 * queries and keys per head, position rotation), attention of new tokens over it, and its page bookkeeping.  Exported
 * by the same library as xcb_moe.h, with the same rules: plain device pointers and sizes, an explicit cudaStream_t,
 * no allocation, no host synchronisation (read_status excepted), XCB_OK or an XCB_ERR_* code, argument errors found
 * on the host before any launch, what only the device can see reported as bits of a status word.
 *
 * The reference has no attention operator; these entry points have no counterpart there. */
#ifndef XCB_ATTN_H_
#define XCB_ATTN_H_

#include "xcb_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- element types ---- */
#define XCB_DTYPE_BF16 0
#define XCB_DTYPE_F16 1
#define XCB_DTYPE_E4M3 2            /* cache only: value = code * scale of the kv head                     */
#define XCB_DTYPE_F32 3             /* norm weights only                                                   */

/* ---- device status bits, beside those of xcb_moe.h ---- */
#define XCB_STATUS_BAD_PAGE 16      /* a page id outside [0, num_pages), or a token without a page: not stored, not
                                       attended                                                             */
#define XCB_STATUS_BAD_SEQ 32       /* a sequence id or length that a call cannot take: that entry was left out */
#define XCB_STATUS_NO_PAGES 64      /* xcb_kv_extend found too few free pages: no sequence grew            */

/* A paged cache: kv [layers][2][num_pages][kv_heads][page_size][head_dim], keys at [..][0], values at [..][1].
 * Token j of sequence s lies in page page_table[s * max_pages + j / page_size], at j % page_size.  A sequence's
 * entries past its last page are -1.  A page may belong to several sequences; refcounts[p] says to how many. */
typedef struct XcbKvCache {
  int32_t layers, num_pages, kv_heads, page_size, head_dim;  /* head_dim * element bytes % 16 == 0, head_dim <= 256 */
  int32_t dtype;                    /* XCB_DTYPE_BF16, _F16 or _E4M3                                       */
  int32_t max_seqs, max_pages;      /* rows and columns of page_table                                      */
  void* kv;                         /* 16-byte aligned                                                     */
  int32_t* page_table;
  int32_t* seq_lens;                /* [max_seqs] tokens in each sequence                                  */
  int32_t* refcounts;               /* [num_pages], 0 = free; NULL where no page operation is called       */
  const float* k_scale;             /* [kv_heads] or NULL (1.0); used with XCB_DTYPE_E4M3 alone            */
  const float* v_scale;
  int32_t* status;                  /* one word, zeroed by the owner at set-up                             */
} XcbKvCache;

/* ---- norms, rotation and store of new tokens ----
 * For each token t and head: y = x * rsqrt(mean(x^2) + eps) * (w + weight_offset) (left out where w is NULL), then
 * the first rotary_dim values turn by positions[t] * f_i in pairs (i, i + rotary_dim / 2), or (2i, 2i + 1) with
 * interleaved; cos and sin are multiplied by mscale.  All in 32 bits, rounded once.  turns[i] = f_i / (2 pi) as a
 * fraction of 2^64: angles are exact modulo a full turn at any position.
 * With a cache, turned keys and the values go to slot positions[t] of sequence seqs[t] (seqs[t] < 0: padding, not
 * stored); e4m3 stores saturate at +-448 times the scale.  Two tokens of a call may not share a slot, and the
 * page must not be shared with another sequence (xcb_kv_extend sees to that).  q_out may be q, k_out may be k.
 * At most 2^30 tokens a call. */
typedef struct XcbRopeArgs {
  int32_t tokens, q_heads, kv_heads, head_dim;
  int32_t rotary_dim;               /* even, 0 <= rotary_dim <= head_dim                                   */
  int32_t interleaved;
  int32_t dtype;                    /* of q, k, v and the outputs: XCB_DTYPE_BF16 or _F16                  */
  int32_t weight_dtype;             /* of the norm weights: dtype or XCB_DTYPE_F32                         */
  float eps, weight_offset, mscale;
  int32_t layer;                    /* of the cache                                                        */
  const void* q;                    /* [tokens, q_heads, head_dim], rows contiguous, 16-byte aligned       */
  const void* k;                    /* [tokens, kv_heads, head_dim], or NULL with kv_heads = 0             */
  const void* v;                    /* with a cache only                                                   */
  int64_t q_stride[2], k_stride[2], v_stride[2], q_out_stride[2], k_out_stride[2];  /* elements: token, head */
  void* q_out;                      /* or NULL                                                             */
  void* k_out;                      /* or NULL                                                             */
  const void* q_weight;             /* [head_dim] or NULL                                                  */
  const void* k_weight;
  const int32_t* positions;         /* [tokens]                                                            */
  const int32_t* seqs;              /* [tokens], with a cache                                              */
  const uint64_t* turns;            /* [rotary_dim / 2]                                                    */
} XcbRopeArgs;
int xcb_qk_norm_rope(const XcbKvCache* cache, const XcbRopeArgs* args, cudaStream_t stream);

/* ---- attention of new tokens over the cache ----
 * q [batch, new_tokens, q_heads, head_dim]: the last new_tokens tokens of sequence seqs[b] (or b where seqs is NULL),
 * already stored.  Token i stands at p = seq_lens - new_tokens + i and sees the positions j <= p, with a window only
 * p - window < j.  out = softmax(scale * q k^T) v per head; q head h reads kv head h / (q_heads / kv_heads).  A token
 * that sees nothing (an empty sequence, p < 0, no page) gets zeros and lse = -inf.  What is not seen is not read
 * into the result, whatever it holds; infinite values that are seen make their dimension infinite (NaN where both signs
 * or a NaN are seen).  lse (natural logarithm of the sum of exponentials) is optional.  At most 65536 new tokens, 65536
 * query heads, 2^20 sequences, and 2^20 rows (new_tokens * q_heads / kv_heads) a call. */
typedef struct XcbAttnArgs {
  int32_t batch, new_tokens, q_heads, dtype, layer, window;  /* window 0: all                              */
  float scale;
  const void* q;
  int64_t q_stride[3];              /* elements: batch, token, head; multiples of 8, head_dim contiguous   */
  void* out;                        /* [batch, new_tokens, q_heads, head_dim] contiguous, dtype            */
  float* lse;                       /* fp32 [batch, new_tokens, q_heads] or NULL                           */
  const int32_t* seqs;              /* [batch] or NULL                                                     */
} XcbAttnArgs;
/* Workspace of any call of this cache shape, group (q_heads / kv_heads) and new_tokens on the current device (parts of
 * sequences that several blocks share).  It needs no set-up (xcb_attn_workspace_init does nothing but refuse NULL), and
 * one that is larger than asked for serves as well; calls that share one must be ordered.  XCB_ERR_UNSUPPORTED: 2^32 or
 * more rows in one layer's keys (num_pages * kv_heads * page_size), or 2^31 or more chunks of 64 positions over all
 * sequences, kv heads and row tiles. */
size_t xcb_attn_workspace_bytes(const XcbKvCache* cache, int32_t q_heads, int32_t new_tokens);
int xcb_attn_workspace_init(void* workspace, size_t bytes, cudaStream_t stream);
int xcb_paged_attention(const XcbKvCache* cache, const XcbAttnArgs* args, void* workspace, size_t workspace_bytes,
                        cudaStream_t stream);

/* ---- page bookkeeping ----
 * All counts and ids are read and written on the device; calls on one cache must be ordered.  The workspace is
 * zeroed once with xcb_kv_workspace_init. */
size_t xcb_kv_workspace_bytes(const XcbKvCache* cache);
int xcb_kv_workspace_init(const XcbKvCache* cache, void* workspace, size_t bytes, cudaStream_t stream);
/* Room for new_tokens[i] more tokens in sequence seqs[i]: the lowest free pages go to the sequences in list order, and
 * seq_lens grows.  A last page that is part full and shared is replaced by a copy first (in list order before the
 * sequence's other new pages); where all its holders grow in this call, the first in the list keeps it.  Too few free
 * pages: nothing changes, XCB_STATUS_NO_PAGES.  A sequence id out of range or listed before, a negative growth, or
 * one past max_pages is left out, XCB_STATUS_BAD_SEQ. */
int xcb_kv_extend(const XcbKvCache* cache, const int32_t* seqs, const int32_t* new_tokens, int32_t n, void* workspace,
                  size_t workspace_bytes, cudaStream_t stream);
/* Sequence dst[i], which must be empty, becomes a copy of src[i] that shares its pages.  An entry whose dst is not
 * empty, was listed before, or is a src of this call is left out, XCB_STATUS_BAD_SEQ. */
int xcb_kv_fork(const XcbKvCache* cache, const int32_t* src, const int32_t* dst, int32_t n, cudaStream_t stream);
/* Sequence seqs[i] keeps its first lens[i] tokens (lens NULL: none); pages that no sequence holds any more are free.
 * An id out of range or listed before, or a length outside [0, seq_lens], is left out, XCB_STATUS_BAD_SEQ. */
int xcb_kv_truncate(const XcbKvCache* cache, const int32_t* seqs, const int32_t* lens, int32_t n, cudaStream_t stream);
/* Live pages move down: with L pages live, those at ids >= L fill the free ids below L, both in ascending order, and
 * the tables follow.  Afterwards the pages [L, num_pages) are free. */
int xcb_kv_compact(const XcbKvCache* cache, void* workspace, size_t workspace_bytes, cudaStream_t stream);
/* Contents of page src[i] to page dst[i], in all layers.  A dst may appear once and may not be a src.  A pair with an
 * id out of range is left out, XCB_STATUS_BAD_PAGE. */
int xcb_kv_copy_pages(const XcbKvCache* cache, const int32_t* src, const int32_t* dst, int32_t n, cudaStream_t stream);
/* Synchronise, read the status bits, clear them: XCB_OK if none were set, else XCB_ERR_DEVICE. */
int xcb_kv_read_status(const XcbKvCache* cache, int32_t* device_status, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* XCB_ATTN_H_ */
