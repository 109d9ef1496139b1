/* rlipv2_attention.h -- C ABI of cross attention to states of another length (gfx950).
 *
 *   S = scale q k^T,  P = softmax over the keys that count,  out = (P * keep * keep_scale) v
 *
 *   query [B, Lq, heads, D], key / value [B, Lk, kv_heads, D]: bf16 or float32, element strides (batch, token, head), elements
 *       of a head contiguous, every row 16-byte aligned, token strides not negative and below 64 MB.  Query head h reads key head h / (heads / kv_heads).
 *   padding  [B, Lk] bytes, nonzero = the key does not count (row stride padding_stride; NULL: all count)
 *   lengths  [B] int32: keys [0, lengths[b]) count (clamped to 0 .. Lk; NULL: all)
 *   keep     [B, heads, Lq, Lk] bytes, contiguous: dropout keep mask of the probabilities (NULL: none); kept ones are multiplied
 *            by keep_scale
 *   out, grad_query [B, Lq, heads, D], grad_key, grad_value [B, Lk, kv_heads, D]: contiguous, the operands' type
 *   out_low  as out, bf16 only, may be NULL: what rounding took from out.  The backward call's delta = rowsum(grad_out out) is taken
 *            from out + out_low; without it the gradients of query and key carry out's rounding as well.  Not used where
 *            cross_attention_short_keys(args) holds (delta is computed from the probabilities).
 *   stats    [B, heads, Lq] float32: log2 of the row's sum of exp(S), +infinity for a row without keys (written by the forward
 *            call, read by the backward call; may be NULL in a forward call)
 *   delta    [B, heads, Lq] float32: scratch of the backward call
 *
 * A row without a key that counts gives zeros, and no gradient.  Where lengths or Lk leave one key, the gradients of query and key are
 * exactly zero.  Keys and values that do not count are never multiplied with:
 * their NaNs and infinities stay where they are, their gradients are zero.  scale >= 1e-30 and finite.
 * Supported: D a multiple of 8 up to 256, heads a multiple of kv_heads, dtype MSDA_BF16 or MSDA_F32.  Results do not depend on
 * anything but the operands (no atomics: repeated calls give the same bits).  Nothing allocates or synchronises; work is enqueued
 * on `stream`.  Return value: 0 or an msda_status code (rlipv2_msda.h). */
#ifndef RLIPV2_ATTENTION_H
#define RLIPV2_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct cross_attention_args {
    int32_t dtype, B, heads, kv_heads, Lq, Lk, D;
    float scale;
    float keep_scale;
    int32_t reserved;
    const void *query, *key, *value;
    int64_t query_stride[3], key_stride[3], value_stride[3];
    const void *padding;
    int64_t padding_stride;
    const void *lengths;
    const void *keep;
    void *out;
    void *out_low;
    void *stats;
    /* backward call only; grad_key and grad_value may both be NULL (states that are not trained) */
    const void *grad_out;
    int64_t grad_out_stride[3];
    void *grad_query, *grad_key, *grad_value;
    void *delta;
    /* cross_attention_workspace_bytes(args, backward) bytes of device memory, 16-byte aligned (may be NULL if that is 0): partial results
     * of as many workgroups as fit on the card, and for long float32 forward calls 8 bytes a query row */
    void *workspace;
    size_t workspace_bytes;
} cross_attention_args;

/* sizeof(cross_attention_args), for bindings that lay the struct out themselves */
size_t cross_attention_args_bytes(void);
/* whether sizes and type are supported (pointers and strides are not looked at) */
int cross_attention_supported(const cross_attention_args *args);
/* whether the backward call reads no out_low */
int cross_attention_short_keys(const cross_attention_args *args);
size_t cross_attention_workspace_bytes(const cross_attention_args *args, int backward);
int cross_attention_forward(const cross_attention_args *args, void *stream);
int cross_attention_backward(const cross_attention_args *args, void *stream);

#ifdef __cplusplus
}
#endif
#endif
