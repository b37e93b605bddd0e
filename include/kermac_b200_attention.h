/*
 * kermac_b200 C-ABI, attention: the part of libkermac_b200.so that kermac_b200.h does not declare.  Same conventions: plain
 * pointers, sizes and element strides; device pointers of the current device; asynchronous on `stream`; 0, a KM_ERR_* or a
 * cudaError_t is returned and kermac_b200_last_error() has the message.  No call allocates, and none keeps anything from one
 * call to the next.  The reference has no such operator; kernel_matvec with normalised weights.
 */
#ifndef KERMAC_B200_ATTENTION_H
#define KERMAC_B200_ATTENTION_H

#include "kermac_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Attention: out[l, n, h] = sum_m softmax_m(scale * <q[l, n, h], k[l, m, hk]>) * v[l, m, hk], hk = h / (heads / key_heads),
 * over the keys that the query sees: the normalised form of kernel_matvec, whose weights never reach memory either.
 * A query that sees no key gets zeros and lse = -inf.
 *
 * A KmHeads is a tensor [l][row][head][channel] with contiguous channels; strides are in elements, and stride_l = 0
 * broadcasts it over the batch.  Scores, softmax statistics and sums are 32-bit whatever `type`; with 16-bit types the
 * weights are rounded to that type for the product with v (and, in the gradient, their gradients for theirs).
 */
#define KM_TYPE_FLOAT32  0
#define KM_TYPE_BFLOAT16 1
#define KM_TYPE_FLOAT16  2
typedef struct KmHeads {
    void*   ptr;
    int64_t stride_l, stride_row, stride_head;
} KmHeads;

typedef struct KmAttentionArgs {
    int32_t l, n, m;              /* batch entries, queries, (own) keys */
    int32_t heads, key_heads, d;  /* heads is a multiple of key_heads; 1 <= d <= 256 channels */
    int32_t type;                 /* KM_TYPE_* of every KmHeads */
    int32_t prefix;               /* kermac_b200_prefix_attention: keys of the prefix that the batch shares, else 0 */
    KmHeads q, k, v, out;         /* k and v have the same batch: both stride_l = 0, or both not */
    KmHeads k_prefix, v_prefix;   /* stride_l is not used */
    const int32_t* lengths; int64_t lengths_stride;      /* keys of each batch entry, NULL: m; values outside [0, m] are
                                                            taken as the nearest of the two.  Later rows of k and v are not read into any result. */
    float*  lse; int64_t lse_stride_l, lse_stride_head;  /* [l][head][n]: natural logarithm of the sum of the exponentials.
                                                            Output (may be NULL) of the forward pass, input of the gradient */
    float   scale;                /* finite, not negative */
    int32_t kv_batch;             /* gradient: batch entries of grad_k and grad_v, l or 1 (k and v broadcast: the sum over l) */
    int32_t q_batch;              /* gradient: batch entries of grad_q, l or 1 */
    KmHeads grad_out, grad_q, grad_k, grad_v;            /* gradient only; `out` is then an input */
    void*   scratch; int64_t scratch_bytes;              /* see the _scratch_bytes functions; 16-byte aligned */
} KmAttentionArgs;

/* Every query sees the lengths[l] keys of its batch entry. */
int kermac_b200_cross_attention(const KmAttentionArgs* args, void* stream);
/* Every query sees the `prefix` keys that the batch shares, which are read once for all, and those of its own entry's keys that
 * are not behind it: the n queries are the entry's newest tokens, so query i sees own key j when j <= lengths[l] - n + i. */
int kermac_b200_prefix_attention(const KmAttentionArgs* args, void* stream);
/* grad_q, grad_k and grad_v from grad_out and the forward pass's out and lse.  Every row is written, those of keys behind
 * lengths[l] with zeros.  The sums have a fixed order: equal calls give equal bits. */
int kermac_b200_cross_attention_grad(const KmAttentionArgs* args, void* stream);
/* Bytes of scratch that the three calls use (0: none), with MB = 2^20 bytes.
 * Forward: partial sums where keys are divided, 512 MB at most, and copies of float32 inputs of up to 64 channels, 384 bytes a row of a
 * head of each of them (whatever d is), 1024 MB at most.  These two calls take less or none, and are slower then.  But where there are both
 * a prefix and own keys a row has a part for each: 8 * l * n * heads * (d + 2) bytes at least, however much that is, and without it the
 * call is refused.
 * Gradient: 4 * l * n * heads bytes, with float16 a 64th of that and 4 bytes for 64 keys of a head besides; 4 * l * n * heads * d for the sum
 * over the batch where q_batch is 1 and l is not; where sums are divided 256 MB at most for each of the three gradients.  It needs all of it. */
int64_t kermac_b200_cross_attention_scratch_bytes(const KmAttentionArgs* args);
int64_t kermac_b200_prefix_attention_scratch_bytes(const KmAttentionArgs* args);
int64_t kermac_b200_cross_attention_grad_scratch_bytes(const KmAttentionArgs* args);
/* Writes which kernels a call of `kind` (0 cross, 1 prefix, 2 gradient) launches into buf (NUL terminated, truncated). */
int kermac_b200_describe_attention(const KmAttentionArgs* args, int32_t kind, char* buf, int32_t buf_len);

#ifdef __cplusplus
}
#endif
#endif /* KERMAC_B200_ATTENTION_H */
