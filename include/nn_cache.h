/* nn_cache.h -- a paged cache of keys and values: the append of new tokens, attention
 * that reads it, and the way back out.
 *
 * A serving program calls them in this order for every layer: one projection makes
 * queries, keys and values of the new tokens; launch_cache_append normalises and rotates
 * queries and keys and writes keys and values to the pages of their requests;
 * launch_cache_attention_forward reads the pages.  They have no counterpart in the
 * reference and follow the conventions of nn_attention.h: device pointers, the stream
 * last, asynchronous, no state between calls, nothing allocated, every call fit for
 * capture, descriptions read during the call only, refusals recorded for
 * nnhip_get_last_error().
 */
#ifndef NN_CACHE_H
#define NN_CACHE_H

#include "nn_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------
 * The cache
 * ------------------------------------------------------------------------
 * Two pools, of keys and of values, of `pages` pages each.  Token p of request r lies in
 * page table[r, p / page_tokens] of both, in slot p % page_tokens.  A page is
 * [kv_heads] of blocks, and a block is, with d = head_dim:
 *   NN_CACHE_PLAIN: page_tokens rows of d values of the call's dtype, each row padded
 *     with zeros to a multiple of 16 bytes;
 *   NN_CACHE_MXFP4: page_tokens rows of 16 G bytes, then page_tokens rows of G scales
 *     (a byte each), G = d / 32 rounded up.  Feature i of a row is the 4 bits i of it,
 *     the low half of a byte first: 3 bits that stand for 0, 0.5, 1, 1.5, 2, 3, 4, 6
 *     and a sign, times 2^(scale - 127) with the scale of its 32 features.  A scale of
 *     255 makes them NaN.
 * An entry of the table that is no page (below 0, or `pages` or more) holds no tokens:
 * what is appended to it is dropped, attention does not see it and reads of it give
 * zeros.  Entries past a request's last token are not used and may hold anything.
 * Requests may share pages that no call writes. */
typedef enum { NN_CACHE_PLAIN = 0, NN_CACHE_MXFP4 } NnCacheKind;

typedef struct {
    int kind;        /* NnCacheKind */
    int page_tokens; /* a power of two, 16 .. 4096 */
    int pages;       /* of each pool */
    int requests;    /* rows of the table */
    int table_pages; /* entries of a row; table_pages * page_tokens up to 2^30 - 4096 */
    const int* table;
    void *k, *v;     /* the pools, pages * nnhip_cache_page_bytes() each, 16-byte aligned */
} NnCache;

/* Bytes of a page of one pool (0 after a refusal); `dtype` as in the calls. */
size_t nnhip_cache_page_bytes(const NnCache* c, int dtype, int kv_heads, int head_dim);

/* ------------------------------------------------------------------------
 * Append
 * ------------------------------------------------------------------------
 * Row t of q, k and v belongs to token place[t] of request request[t] (NULL: t).
 * q_out and the cached key are the rows turned by `rope`, as launch_qk_norm_rope_forward
 * has it (q_weight and k_weight with the norm only); without `norm` they are turned but
 * not normalised.  Values are stored as they are.
 *
 * To 4 bits: of 32 features x (keys: in 64 bits throughout, so that a code does not
 * depend on the order of a sum), the exponent is the least e of -120 .. 125 with
 * max|x| <= 7 * 2^e, and each |x| 2^-e is rounded to the nearest of the 8 sizes, half
 * way to the even code: off by half a step at most, as 7 still rounds to 6.  (From
 * 7 * 2^125 on, sizes end at 6 * 2^125.)  If any of the 32 is infinite or NaN all are NaN.
 *
 * place[t] < 0: row t is no token (a padded batch): what it holds has no effect, and nothing is
 * written for it.  A
 * request that is none, or a place past the table, is an entry that is no page: q_out is
 * written, key and value are dropped.  No two rows of a call may have the same slot;
 * which of them it then holds, and whether whole, is not defined. */
typedef struct {
    NnQkNormRope rope;      /* head_dim up to 128, kv_heads from 1; k_out_stride is not used */
    int norm;
    long long v_stride[2];  /* of (token, head) */
    const int* request;     /* [tokens], or NULL */
    const int* place;       /* [tokens] */
} NnCacheAppend;

/* q_out at q_out_stride; it may be q itself if the strides are equal.  With heads = 0 q
   and q_out are ignored. */
void launch_cache_append(void* q_out, const void* q, const void* k, const void* v,
    const NnCacheAppend* a, const NnCache* c, hipStream_t s);

/* ------------------------------------------------------------------------
 * Read
 * ------------------------------------------------------------------------
 * k[t], v[t] = the key and value of token place[t] of request request[t] (NULL: t), as
 * the values that they stand for: exact in both types, and infinite from 2^128 on (scales
 * of 253 and 254, which no append writes).  Rows with place[t] < 0 are left as they are. */
typedef struct {
    int dtype;              /* NnDtype of k and v, and of plain pages */
    int tokens;
    int kv_heads, head_dim;
    long long k_stride[2], v_stride[2]; /* of (token, head) */
    const int* request;     /* [tokens], or NULL */
    const int* place;       /* [tokens] */
} NnCacheRead;

void launch_cache_read(void* k, void* v, const NnCacheRead* a, const NnCache* c, hipStream_t s);

/* ------------------------------------------------------------------------
 * Attention
 * ------------------------------------------------------------------------
 * launch_attention_forward with keys and values from the cache: request b of the batch
 * is row b of the table, key j its token j.  All of NnAttention's terms and masks but
 * documents (a request is one), with these differences: k_stride and v_stride are not
 * used; len_k, which has to fit in the table, bounds k_len; keys of entries that are no
 * page are not seen.  What seen pages hold up to k_len should be finite (and values below
 * 2^119 / len_k in size: fp32 sums have shares of up to 2^8); slots behind k_len may hold
 * anything.
 *
 * With bf16 tensors queries, probabilities and plain pages are bf16 and 4-bit values,
 * which bf16 holds exactly, meet them there; with fp32 tensors all products are of fp32
 * values.
 *
 * `workspace`: nnhip_cache_attention_workspace floats (NULL if that is 0), zero-filled
 * before its first use; every launch leaves it fit for the next, also of another shape
 * that it is large enough for, and its size serves every call of a smaller batch or of
 * fewer queries or keys too.  launch_attention_forward leaves a workspace as fit, and
 * takes one that this call has left, so one of the larger size serves both; what
 * anything else has written to is to be filled with zeros again.  Launches that may run
 * concurrently need separate workspaces. */
size_t nnhip_cache_attention_workspace(const NnAttention* a, const NnCache* c);
void launch_cache_attention_forward(void* out, float* lse, const void* q,
    const NnAttention* a, const NnCache* c, float* workspace, hipStream_t s);

#ifdef __cplusplus
}
#endif

#endif /* NN_CACHE_H */
