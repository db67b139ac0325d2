/* SPDX-License-Identifier: MIT
 *
 * Log-probabilities of given tokens under rows of logits, on the GPU: what a
 * teacher-forced pass over a search's sequences needs, with the entropy of each
 * row and its most likely tokens, and the logits' gradient. Additions of
 * libdbs_hip.so beside the search itself (dbs_cuda.h, dbs_hip.h); the reference
 * has no counterpart.
 *
 * Every pointer is device memory, every call is asynchronous on `stream` (a
 * hipStream_t, NULL = the default stream) and returns a dbs_cuda status:
 * DBS_CUDA_STATUS_INVALID_ARGUMENT where sizes, strides or pointers are refused,
 * before anything is launched. Nothing is allocated, read back or waited for, so
 * a call can be captured into a graph.
 */
#pragma once

#include "dbs_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rows of `vocab` logits x, [outer, inner, vocab] with the strides of the first
 * two in elements (a row is contiguous), and a token t for each, tokens [outer *
 * inner] (int32, or int64 with tokens_i64). With p = softmax(x):
 *   logprobs      [rows]       log p_t
 *   entropy       [rows]       -sum_v p_v log p_v            (or NULL)
 *   top_logprobs  [rows, top]  the `top` largest log p_v, largest first, of equal
 *   top_tokens    [rows, top]  ones the lowest v first       (both NULL: top = 0)
 *   stats         [rows, 4]    what the gradient needs of the row (or NULL)
 * A row whose token lies outside [0, vocab) is not read: logprobs 0, entropy 0,
 * top_logprobs -inf, top_tokens -1. A row of -inf alone (nothing is possible):
 * logprobs -inf, entropy 0, top_logprobs -inf. A row that holds NaN or +inf: NaN,
 * top_tokens -1. Sums are held in 32 bits. vocab is at most 2^30, top at most 64 and
 * at most vocab, rows fewer than 2^24. What is written shares no memory with what is
 * read. */
typedef struct BeamgradTokenLogprobs {
    const void* logits;
    int32_t data_type; /* DBS_CUDA_DTYPE_F32, _F16 or _BF16 */
    int32_t outer;
    int32_t inner;
    int32_t vocab;
    int64_t strides[2];
    const void* tokens;
    int32_t tokens_i64;
    int32_t top;
    float* logprobs;
    float* entropy;
    float* top_logprobs;
    int64_t* top_tokens;
    float* stats;
} BeamgradTokenLogprobs;

/* Workspace bytes of the call (0: it needs none), or -1 where its sizes are refused. */
DBS_CUDA_EXPORT int64_t beamgrad_token_logprobs_workspace_size(const BeamgradTokenLogprobs* args);

/* `workspace`: 16-byte aligned, of at least the size above. */
DBS_CUDA_EXPORT int beamgrad_token_logprobs(const BeamgradTokenLogprobs* args, void* workspace, int64_t workspace_bytes,
                                            void* stream);

/* The logits' gradient, [outer, inner, vocab] contiguous in their type, from the
 * gradients of the outputs (float32, contiguous; NULL: zeros). args as in the
 * call, whose stats and top_tokens are read; its other outputs are not. With
 * A = g + sum_j g_j over the row's alternatives j and H its entropy,
 *   grad_v = -p_v (A + g_H (log p_v + H)) + [v = t] g + sum_j [v = top_j] g_j,
 * computed in 32 bits and rounded once; zeros where the row was not read or nothing
 * in it is possible, NaN where it holds NaN or +inf. In the logits' own place it is
 * refused. */
DBS_CUDA_EXPORT int beamgrad_token_logprobs_backward(const BeamgradTokenLogprobs* args, const float* grad_logprobs,
                                                     const float* grad_entropy, const float* grad_top, void* grad_logits,
                                                     void* stream);

#ifdef __cplusplus
}
#endif
