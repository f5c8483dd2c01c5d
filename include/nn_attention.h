/* nn_attention.h -- launch layer of the attention operators.
 *
 * A transformer block calls them in this order: one projection makes queries,
 * keys and values; launch_qk_norm_rope_* normalises each head's query and key
 * and rotates it by its position; launch_attention_* mixes the values.  They
 * have no counterpart in the reference and follow the conventions of nn_hip.h:
 * device pointers unless stated otherwise, the stream last, asynchronous, no
 * state between calls, workspaces lent by the caller, refusals recorded for
 * nnhip_get_last_error().  The descriptions (NnQkNormRope, NnAttention) are
 * host memory and read during the call only.
 *
 * Tensors hold fp32 or bf16 values; sums, softmax statistics, norms and the
 * gradients of weights and biases are fp32 (or wider) for both.  With bf16
 * tensors two things are rounded to bf16 before a sum: the probabilities and score
 * gradients that are multiplied with values, queries, keys and dout (each by up to
 * 2^-8 of itself, which about adds the result's own rounding once more), and the
 * output from which dq takes its row sum <dout, out> (dk, dv and dbias take an fp32
 * one).
 *
 * The last dimension of every tensor is contiguous; the other strides are the
 * caller's, counted in elements, so that the parts of one projection's rows, and
 * caches with a head's tokens together, are read where they lie.  Pointers and
 * strides that are multiples of 16 bytes (with head_dim * size too) get 16-byte
 * accesses; any others are taken element by element, slower.
 *
 * What a call reads may repeat rows (strides of 0); what it writes, outputs and
 * gradients at the strides of their inputs, may not, and is refused.  Gradients of
 * inputs that repeat rows are for the caller to form from those of their copies.
 *
 * Nothing allocates, issues a memset or synchronises: every call can be
 * captured into a graph.  Results do not depend on the order in which
 * workgroups run.
 */
#ifndef NN_ATTENTION_H
#define NN_ATTENTION_H

#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum { NN_F32 = 0, NN_BF16 } NnDtype;

/* Which keys a query sees: all, those up to its own position, or those up to its
   own position and the first `prefix` ones. */
typedef enum { NN_MASK_NONE = 0, NN_MASK_CAUSAL, NN_MASK_PREFIX } NnMask;

/* ------------------------------------------------------------------------
 * Norm of each head's query and key with the position rotation
 * ------------------------------------------------------------------------
 * For each token t and head: y = x * rsqrt(mean(x^2) + eps) * weight over the
 * head_dim features; then each pair p < rot_dim / 2 of (y_a, y_b) turns by the
 * angle pos[t, axis(p)] * freq[p]:
 *     out_a = y_a cos - y_b sin,  out_b = y_a sin + y_b cos
 * with (a, b) = (p, p + rot_dim / 2), or (2p, 2p + 1) if interleaved, and
 * axis(p) = p / (rot_dim / 2 / axes).  Features from rot_dim on are not turned.
 * Angles are formed and reduced in 64 bits, so far positions keep their sine. */
typedef struct {
    int dtype;               /* NnDtype of q, k, their outputs and gradients */
    int tokens;              /* tokens * (heads + kv_heads) below 2^31, 2^30 at most for the gradients */
    int heads, kv_heads;     /* either may be 0: its pointers are then ignored */
    int head_dim;            /* 1 .. 256 */
    int rot_dim;             /* even, 0 .. head_dim */
    int axes;                /* >= 1, a divisor of rot_dim / 2 */
    int interleaved;
    float eps;
    long long q_stride[2], k_stride[2];         /* of (token, head): inputs and their gradients */
    long long q_out_stride[2], k_out_stride[2]; /* outputs and their gradients */
    const float* q_weight;   /* [head_dim], or NULL for 1 */
    const float* k_weight;
    const int* pos;          /* [tokens, axes] */
    const double* freq;      /* [rot_dim / 2], radians a position */
} NnQkNormRope;

/* q_out, k_out: written at q_out_stride, k_out_stride; they may be q and k
   themselves if the strides are equal. */
void launch_qk_norm_rope_forward(void* q_out, void* k_out, const void* q, const void* k,
    const NnQkNormRope* a, hipStream_t s);

/* dq, dk (layout of q, k) from dq_out, dk_out (layout of the outputs) and the
   forward pass's inputs; dq_weight, dk_weight [head_dim] are overwritten, and may be
   NULL where they are not wanted.  `workspace`: nnhip_qk_norm_rope_workspace
   floats, needed if either weight gradient is. */
size_t nnhip_qk_norm_rope_workspace(const NnQkNormRope* a);
void launch_qk_norm_rope_backward(void* dq, void* dk, float* dq_weight, float* dk_weight,
    const void* dq_out, const void* dk_out, const void* q, const void* k,
    const NnQkNormRope* a, float* workspace, hipStream_t s);

/* ------------------------------------------------------------------------
 * Attention
 * ------------------------------------------------------------------------
 * Query i of request b stands at position P = q_start[b] + i; key j at j.  Head h
 * reads key head h / (heads / kv_heads).
 *     x_ij = scale * <q_i, k_j>
 *     x_ij = softcap * tanh(x_ij / softcap)                  if softcap > 0
 *     x_ij += bias[bucket[clamp(j - P, -m, m) + m], h]       if buckets > 0, m = max_distance
 *     p_ij = exp(x_ij) / sum_j exp(x_ij) over the keys that i sees
 *     out_i = sum_j p_ij v_j,  lse_i = log sum_j exp(x_ij)
 * Query i sees key j if j < k_len[b]; and, by `mask`, j <= P or (prefix only)
 * j < prefix[b]; and, with documents, doc_q[b, i] == doc_k[b, j] >= 0.  A query
 * that sees nothing gets out = 0, lse = -inf and zero gradients.  Keys past k_len
 * or of a negative document, and queries that see nothing, may hold anything, NaN
 * among it; what other keys and values hold should be finite, as masked entries
 * of a tile are multiplied by zero. */
typedef struct {
    int dtype;              /* NnDtype of q, k, v, out and their gradients */
    int batch, len_q, len_k; /* lengths up to 2^30 - 4096 */
    int heads, kv_heads;    /* heads a multiple of kv_heads */
    int head_dim;           /* 1 .. 128 */
    float scale;            /* > 0 */
    float softcap;          /* 0: none; scale / softcap and 1.45 softcap are normal fp32 values */
    int mask;               /* NnMask */
    int buckets;            /* 0: no bias */
    int max_distance;       /* 0 .. 1023 */
    long long q_stride[3], k_stride[3], v_stride[3]; /* of (batch, token, head): tensors and their gradients */
    long long out_stride[3];                         /* out and its gradient */
    const int* q_start;     /* [batch], any value, or NULL for len_k - len_q */
    const int* k_len;       /* [batch], or NULL for len_k */
    const int* prefix;      /* [batch], for NN_MASK_PREFIX */
    const int* doc_q;       /* [batch, len_q], or NULL (both or neither) */
    const int* doc_k;       /* [batch, len_k] */
    const int* bucket;      /* [2 max_distance + 1], values in 0 .. buckets - 1 */
    const float* bias;      /* [buckets, heads] */
} NnAttention;

/* out, lse [batch, heads, len_q].  `workspace`: nnhip_attention_forward_workspace
   floats (NULL if that is 0), zero-filled before its first use; every launch leaves
   it fit for the next, also of another shape that it is large enough for.  Its size
   serves every call of a smaller batch or of fewer queries or keys too, so that of a
   program's largest call serves all of them.  Launches that may run concurrently need
   separate workspaces. */
size_t nnhip_attention_forward_workspace(const NnAttention* a);
void launch_attention_forward(void* out, float* lse, const void* q, const void* k, const void* v,
    const NnAttention* a, float* workspace, hipStream_t s);

/* dq, dk, dv (layouts of q, k, v) and dbias [buckets, heads] (NULL if not wanted)
   from dout, the forward pass's inputs and its out and lse.  All are overwritten.
   `workspace`: nnhip_attention_backward_workspace floats (they serve every smaller
   batch and shorter lengths), nothing to be filled. */
size_t nnhip_attention_backward_workspace(const NnAttention* a);
void launch_attention_backward(void* dq, void* dk, void* dv, float* dbias, const void* dout,
    const void* q, const void* k, const void* v, const void* out, const float* lse,
    const NnAttention* a, float* workspace, hipStream_t s);

#ifdef __cplusplus
}
#endif

#endif /* NN_ATTENTION_H */
