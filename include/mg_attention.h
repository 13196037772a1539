/*
 * mg_attention.h -- C ABI of the attention operators of the B200 (sm_100a)
 * library: attention over whole rows with its gradients, rotary positions, and
 * attention of one new token over a paged key-value cache.
 *
 * They stand beside mg_matmul_softmax (mg_gemm.h), which writes the scores of
 * rows of at most 256 keys: here no score reaches memory, rows have any length
 * and the scores may be capped, biased by distance and masked by documents or a
 * prefix. The same rules hold: plain C, status codes (mg_last_error() has the
 * message), work enqueued on the caller's stream on the current device, scratch
 * from mg_set_allocator's allocator or the library's own stream-ordered pool.
 * The library's first call on a device (of any function) sets the device up and
 * cannot be captured into a graph; every later one can.
 */
#ifndef MG_ATTENTION_H
#define MG_ATTENTION_H

#include "mg_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum mg_dtype { MG_F32 = 0, MG_BF16 = 1 } mg_dtype;

#define MG_MAX_HEAD_DIM 128

/* Attention of q [batch, heads, q_len, head_dim] over k, v [batch, kv_heads,
 * k_len, head_dim]; heads is a multiple of kv_heads, and query head h reads
 * key-value head h / (heads / kv_heads). Query i stands at position
 * i + k_len - q_len, key j at position j.
 *   t[i][j] = scale * q[i] . k[j];  s = cap > 0 ? cap * tanh(t / cap) : t
 *   s -= slopes[h] * |position(i) - j|                  (slopes not NULL)
 * Key j is seen by query i if
 *   (causal == 0 or j <= position(i) or j < prefix[b])  (prefix NULL: 0) and
 *   (documents NULL or documents[b][j] == documents[b][position(i)] >= 0);
 * a query at a negative position has no document and sees no key where
 * documents are given.
 *   lse[i] = log sum exp(s[i][j]), out[i] = sum exp(s[i][j] - lse[i]) v[j]
 * over the seen keys; a query that sees none gets out = 0, lse = -inf.
 * Keys of a negative document are padding: what k and v hold there is never
 * used, nor is q or dout of a query of a negative document. Elsewhere v (and in the
 * backward pass k, q, dout) has to be finite also where a mask hides it from
 * some queries.
 * The backward pass takes each weight from the forward's lse of the same call, exp(s - lse).
 * fp32 tensors, and those that run on the CUDA cores, have a row's weights divided by their
 * sum; 16-bit ones on the tensor cores keep lse's rounding, a relative 2^-24 * |lse|. In 16-bit
 * calls the weights, and dS, are rounded to 16 bits for their products; sums, softmax
 * statistics and delta are kept in 32.
 * Scores and biases are resolved up to 2^28 in size; a row with larger ones may
 * come out as NaN.
 * scale lies within +-1e30, cap is 0 or within 1e-30..1e30. Strides are in
 * elements, for {batch, head, row}; head_dim is contiguous. Outputs must not
 * share memory with an input or with each other (MG_ERR_INVALID; views of one buffer
 * that lie between one another are fine), but `out` may be q itself, with the same
 * strides. Tensors whose rows start on 16-byte boundaries and hold a
 * multiple of 8 elements run on the tensor cores, others on the CUDA cores. */
typedef struct mg_attention_desc {
    int32_t dtype;                       /* mg_dtype of q, k, v, out and the gradients */
    int32_t batch, heads, kv_heads, q_len, k_len, head_dim;
    int32_t causal;
    float scale, cap;
    int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];
    int64_t dout_stride[3], dq_stride[3], dk_stride[3], dv_stride[3];  /* backward only */
    const float* slopes;                 /* [heads] or NULL */
    const int32_t* documents;            /* [batch][k_len] or NULL */
    const int32_t* prefix;               /* [batch] or NULL; needs causal */
} mg_attention_desc;

/* out and lse ([batch][heads][q_len] fp32, contiguous). */
mg_status mg_attention(const mg_attention_desc* d, void* out, float* lse, const void* q, const void* k,
                       const void* v, void* stream);

/* Gradients of sum(dout * out) with respect to q, k and v, from the forward's
 * out and lse:
 *   P = exp(s - lse), its rows summing to one, dV = P^T dout, delta = rowsum(dout * out),
 *   dS = P * (dout V^T - delta) * scale * (1 - tanh^2), dQ = dS K, dK = dS^T Q,
 * dK and dV summed over the query heads that share a key-value head.
 * Deterministic: no atomics. The slopes are constants. */
mg_status mg_attention_backward(const mg_attention_desc* d, void* dq, void* dk, void* dv, const void* dout,
                                const void* q, const void* k, const void* v, const void* out,
                                const float* lse, void* stream);

/* Rotary positions on q [batch, heads, len, head_dim] and k [batch, kv_heads,
 * len, head_dim] (k may be NULL) in one launch. Of each head the first
 * 2 * pairs elements turn, pair p by the angle positions[b][l] *
 * frequencies[p]: (a, b) -> magnitude * (a cos - b sin, a sin + b cos), with
 * inverse != 0 by the opposite angle (the gradient of the forward call). Pair p
 * is (2p, 2p + 1) if interleaved, else (p, p + pairs). The rest is copied.
 * The angle is reduced in 64-bit fixed point: exact for any int32 position.
 * Outputs may be the inputs themselves (same strides) but not share memory with
 * them, the other input or each other otherwise (MG_ERR_INVALID). */
typedef struct mg_rotary_desc {
    int32_t dtype;
    int32_t batch, heads, kv_heads, len, head_dim, pairs;
    int32_t interleaved, inverse;
    float magnitude;
    int64_t q_stride[3], k_stride[3], out_q_stride[3], out_k_stride[3];
    int64_t position_stride;             /* between batches; 0: all share one row */
    const int32_t* positions;            /* [batch][len] */
    const double* frequencies;           /* [pairs], radians a position */
} mg_rotary_desc;

mg_status mg_rotary(const mg_rotary_desc* d, void* out_q, void* out_k, const void* q, const void* k,
                    void* stream);

/* Attention of one new token per request over a paged key-value cache:
 * q, out [batch, heads, head_dim], lse [batch][heads]. Key j of request b is
 * row j % page_size of page block_table[b][j / page_size], for j <
 * lengths[b]; the query stands at position lengths[b] - 1. cap and slopes as
 * in mg_attention. With k_new and v_new ([batch, kv_heads, head_dim]) the
 * token's own key and value are taken from there and written to the cache at
 * position lengths[b] - 1. A length of 0 gives out = 0, lse = -inf and writes
 * nothing. A length beyond the table is cut off there: the call attends to the
 * keys that the table holds, from the last one's position, and the request
 * appends nothing. A page outside the pool is skipped (never read or written).
 * Both set MG_ERR_INVALID in mg_device_status(). Requests must not share the
 * page that they append to, nor keys and values theirs; k_new and v_new may lie in
 * the cache, but not where the call appends. Outputs must not share memory with an
 * input or with each other, but `out` may be q itself, with the same strides. */
typedef struct mg_paged_desc {
    int32_t dtype;
    int32_t batch, heads, kv_heads, head_dim, page_size, pages, table_width;
    float scale, cap;
    int64_t q_stride[2], out_stride[2];          /* {batch, head} */
    int64_t k_stride[3], v_stride[3];            /* {page, row of the page, head} */
    int64_t k_new_stride[2], v_new_stride[2];    /* {batch, head} */
    int64_t table_stride;                        /* between requests */
    const float* slopes;                         /* [heads] or NULL */
    const int32_t* block_table;
    const int32_t* lengths;                      /* [batch] */
} mg_paged_desc;

mg_status mg_paged_attention(const mg_paged_desc* d, void* out, float* lse, const void* q, void* k_pages,
                             void* v_pages, const void* k_new, const void* v_new, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MG_ATTENTION_H */
