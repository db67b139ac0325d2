/* SPDX-License-Identifier: MIT
 *
 * The state of a model in a beam search, on the GPU: attention over a paged
 * cache of keys and values, the pages of that cache, the eviction of tokens by the
 * attention that they get, rotary positions, and the reordering of dense states. Additions of libdbs_hip.so beside the search itself
 * (dbs_cuda.h, dbs_hip.h); the reference has no counterpart.
 *
 * Every pointer is device memory unless said otherwise, every call is
 * asynchronous on `stream` (a hipStream_t, NULL = the default stream) and
 * returns a dbs_cuda status: DBS_CUDA_STATUS_INVALID_ARGUMENT where sizes,
 * strides or pointers are refused, before anything is launched. Nothing is
 * allocated, read back or waited for, so a call can be captured into a graph.
 *
 * Data types are DBS_CUDA_DTYPE_F32, _F16 and _BF16.
 *
 * A page table holds S sequences: pages [S, P] (the pages of each sequence in
 * order, -1 past its last), lengths [S] (tokens held) and refs [n_pages] (how
 * many sequences hold each page; 0: it is free); S * P is at most 2^30. Values
 * read from device memory are checked where they are used: an entry that is no
 * page of the pool counts as -1, a length is cut to [0, P * page_tokens], a token
 * without a page is seen by no query and written nowhere.
 */
#pragma once

#include "dbs_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Attention of the last tokens of S sequences over their cached keys and
 * values. q [S, N, H, D]; the pools k and v [n_pages, page_tokens, Hkv, D];
 * head h reads the cache's head h / (H / Hkv). Of sequence s the last
 * counts[s] tokens of its lengths[s] ask (all N where counts is NULL; at most
 * N and lengths[s]); the tokens ahead of them are its prefix, which every
 * asking token sees. Of the asking tokens, token i sees itself and
 *   - without parents: the asking tokens before it,
 *   - with parents [S, N]: its parent, the parent's parent, and so on, up to a
 *     parent that is not an earlier asking token (-1).
 * out[s, i, h] = sum_j p_j v_j, p = softmax over the seen j of scale * q . k_j;
 * lse[s, i, h] = log of the sum of exp(scale * q . k_j). Rows i >= counts[s]:
 * out 0, lse -inf.
 *
 * beams > 1: sequences come in groups of `beams`, S a multiple of it, and the
 * live ones of group b (counts > 0) hold the same pages for the whole pages
 * within their first shared[b] tokens (an int32 [S / beams] array; NULL: none).
 * Those pages are read once for the group.
 *
 * D is a multiple of 8 up to 256, H a multiple of Hkv, N <= 512 with parents.
 * Rows are contiguous in D; the other strides (in elements) and the base
 * pointers are multiples of 16 bytes. out and lse are contiguous. */
typedef struct BeamgradAttention {
    const void* q;
    const void* k;
    const void* v;
    int32_t data_type;
    int32_t sequences; /* S */
    int32_t tokens;    /* N */
    int32_t heads;     /* H */
    int32_t kv_heads;  /* Hkv */
    int32_t head_dim;  /* D */
    int32_t beams;
    int32_t page_tokens;
    int32_t n_pages;
    int32_t table_pages; /* P */
    int64_t q_strides[3]; /* sequence, token, head */
    int64_t k_strides[3]; /* page, token, head */
    int64_t v_strides[3];
    const int32_t* pages; /* [S, P], contiguous */
    const int32_t* lengths;
    const int32_t* counts;  /* or NULL */
    const int32_t* parents; /* or NULL */
    const int32_t* shared;  /* or NULL */
    float scale;            /* positive, finite times log2(e) */
    int32_t reserved;       /* 0 */
    void* out;
    float* lse; /* or NULL */
} BeamgradAttention;

/* Workspace bytes of the call, or -1 where its sizes are refused: partial results
 * in float32, two tiles of up to 128 rows for each of the card's workgroups (up to two
 * a CU); with `shared` also one for each tile of a launch, which takes as many groups as
 * 256 MB of them allow, and one at least. */
DBS_CUDA_EXPORT int64_t beamgrad_tree_attention_workspace_size(const BeamgradAttention* args);

/* `workspace`: 16-byte aligned, of at least the size above. */
DBS_CUDA_EXPORT int beamgrad_tree_attention(const BeamgradAttention* args, void* workspace, int64_t workspace_bytes,
                                            void* stream);

/* Pools of a cache: n pools of n_pages pages of page_tokens tokens each, a
 * token's row of row_bytes[i] contiguous bytes in pool i at base[i] + page *
 * page_stride[i] + token * token_stride[i] (bytes). The arrays are host
 * memory, read before the call returns. All pools are paged by one table. They
 * may lie in one buffer, in turns too, but no byte may be two pools' or two tokens':
 * the calls write them in many places at once, and refuse pools that meet. */
typedef struct BeamgradPools {
    void* const* base;
    const int64_t* row_bytes;
    const int64_t* page_stride;
    const int64_t* token_stride;
    int32_t n;
    int32_t n_pages;
    int32_t page_tokens;
    int32_t reserved; /* 0 */
} BeamgradPools;

/* A call reads one table and writes another, no part of which may lie in the first
 * or in another part (refused). */
typedef struct BeamgradTable {
    int32_t* pages; /* [sequences, table_pages], contiguous */
    int32_t* lengths;
    int32_t* refs; /* [n_pages] */
} BeamgradTable;

/* The table after a step of a beam search: sequence s continues sequence
 * parents[s] of `from` (int32, or int64 with parents_i64; outside [0, S): it
 * holds nothing). Whole pages are shared. A last page that is not full goes to
 * the first sequence that continues its holder; every other one gets a free page
 * and a copy of its tokens, in every pool. Free pages are taken in order of
 * their number, for the sequences in order; a sequence that finds none holds
 * nothing. */
DBS_CUDA_EXPORT int64_t beamgrad_fork_pages_workspace_size(int sequences);
DBS_CUDA_EXPORT int beamgrad_fork_pages(const BeamgradPools* pools, const BeamgradTable* from, const void* parents,
                                        int parents_i64, int sequences, int table_pages, const BeamgradTable* to,
                                        void* workspace, int64_t workspace_bytes, void* stream);

/* Room for counts[s] >= 0 more tokens: pages are taken from the free ones in
 * order of their number, for the sequences in order. A sequence for which the
 * pool or the table has too few keeps its pages and its length; after one for which
 * the pool has, every later one that needs a page does too. Takes some us, and 0.9
 * for every 1000 pages of the pool. */
DBS_CUDA_EXPORT int64_t beamgrad_extend_pages_workspace_size(int n_pages);
DBS_CUDA_EXPORT int beamgrad_extend_pages(const BeamgradTable* from, const int32_t* counts, int sequences,
                                          int table_pages, int n_pages, int page_tokens, const BeamgradTable* to,
                                          void* workspace, int64_t workspace_bytes, void* stream);

/* news[i] (pool i's rows, at news[i] + s * news_strides[2 i] + j *
 * news_strides[2 i + 1] bytes) for the last counts[s] tokens of each sequence (all
 * `tokens` where counts is NULL; at most `tokens` and lengths[s]): row j to the
 * j-th of them. news that lie in a pool are refused. Where sequences hold one page
 * together (refs > 1), none may write to it: extend_pages after fork_pages leaves every
 * sequence its new tokens' pages to itself. */
DBS_CUDA_EXPORT int beamgrad_write_tokens(const BeamgradPools* pools, const void* const* news,
                                          const int64_t* news_strides, const int32_t* pages, const int32_t* lengths,
                                          const int32_t* counts, int sequences, int table_pages, int tokens,
                                          void* stream);

/* Of the last drafted[s] tokens, keep[s, 0 .. kept[s]) stay (numbers among the
 * drafted ones, ascending; the first that is not ends the list), moved
 * together in every pool; the others' pages are given back. The drafted tokens
 * lie in pages of their sequence alone, as extend_pages after fork_pages leaves
 * them. keep is [sequences, width]. */
DBS_CUDA_EXPORT int beamgrad_keep_tokens(const BeamgradPools* pools, const BeamgradTable* from, const int32_t* drafted,
                                         const int32_t* keep, const int32_t* kept, int sequences, int table_pages,
                                         int width, const BeamgradTable* to, void* stream);

/* to[i][b, k] = from[i][b, parents[b, k]], zeros where parents is outside
 * [0, beams): n dense states [examples, beams, row_bytes[i]]; from[i] == to[i]
 * for every i moves the rows in place. Otherwise no state that is written may meet
 * one that is read; two that are written never may. At most 4096 beams. */
DBS_CUDA_EXPORT int beamgrad_reorder_states(const void* const* from, void* const* to, const int64_t* row_bytes, int n,
                                            const void* parents, int parents_i64, int examples, int beams,
                                            void* stream);

/* Its gradient: to[i][b, p] = the sum over the k with parents[b, k] == p of
 * from[i][b, k], in order of k in 32 bits, rounded once. Rows of `elements[i]`
 * values of data_type. */
DBS_CUDA_EXPORT int beamgrad_reorder_states_backward(const void* const* from, void* const* to, const int64_t* elements,
                                                     int n, int data_type, const void* parents, int parents_i64,
                                                     int examples, int beams, void* stream);

/* Rotary positions: of every head of n tensors [sequences, tokens, heads[i],
 * head_dim[i]] the first 2 * pairs values turn in pairs, by the angles position *
 * frequency[f] of pair f,
 *   (a, b) -> scale * (a cos - b sin, a sin + b cos),
 * values 2 f and 2 f + 1 with `interleaved`, f and pairs + f without; with `inverse`
 * by the angles' negatives, which is the gradient. The rest of a head is copied. Tokens
 * n >= counts[s] (counts may be NULL) become zeros, or stay as they are in place. Angles
 * are computed in 64 bits: their sines and cosines are good to 32 up to 2^50, of either sign.
 *
 * from, to, heads, head_dim and the strides are host arrays, read before the call
 * returns; strides are of sequences, tokens and heads (three for each tensor), in
 * elements, and a head is contiguous. from[i] == to[i] for every i (with equal strides)
 * turns in place; otherwise no memory that is written may meet what is read. No two rows
 * that are written may meet; where sequences, tokens and heads lie in three steps of which
 * none continues another, what lies between the rows of the smallest counts as written too. head_dim is at most 1024, sequences * tokens fewer than 2^26, strides at
 * most 2^40. */
typedef struct BeamgradRotary {
    const void* const* from;
    void* const* to;
    const int32_t* heads;
    const int32_t* head_dim;
    const int64_t* from_strides;
    const int64_t* to_strides;
    int32_t n;
    int32_t data_type;
    int32_t sequences;
    int32_t tokens;
    int32_t pairs;
    int32_t interleaved;
    int32_t inverse;
    float scale;
    const void* positions; /* int32, or int64 with positions_i64 */
    int64_t position_strides[2]; /* sequence, token, in elements */
    int32_t positions_i64;
    int32_t reserved; /* 0 */
    const double* frequencies; /* [pairs] */
    const int32_t* counts;
} BeamgradRotary;

DBS_CUDA_EXPORT int beamgrad_rotary(const BeamgradRotary* args, void* stream);

/* The attention that cached tokens get, of the last tokens of S sequences as
 * beamgrad_tree_attention has them (the fields alike): with p_ihj the weight that
 * asking token i gives token j in head h, exp(scale * q . k_j - lse[s, i, h]) where it
 * sees it, and the heads h of the cache's head g,
 *   weights[s, g, j] += sum_i sum_h p_ihj   for the tokens ahead of the asking ones,
 *   weights[s, g, j]  = sum_i sum_h p_ihj   for the asking ones,
 * summed in 32 bits and in an order that does not change from run to run. Tokens
 * without a page, and places past a sequence's length, keep what they have. A row whose
 * lse is -inf gives nothing. lse [S, N, H] is what beamgrad_tree_attention leaves,
 * contiguous; weights [S, Hkv, ...] has weight_strides (elements) and room for
 * table_pages * page_tokens places, contiguous, and shares no memory with q, k or lse. */
typedef struct BeamgradWeights {
    const void* q;
    const void* k;
    int32_t data_type;
    int32_t sequences; /* S */
    int32_t tokens;    /* N */
    int32_t heads;     /* H */
    int32_t kv_heads;  /* Hkv */
    int32_t head_dim;  /* D */
    int32_t page_tokens;
    int32_t n_pages;
    int32_t table_pages; /* P */
    float scale;         /* positive, finite times log2(e) */
    int64_t q_strides[3]; /* sequence, token, head */
    int64_t k_strides[3]; /* page, token, head */
    int64_t weight_strides[2]; /* sequence, head */
    const int32_t* pages; /* [S, P], contiguous */
    const int32_t* lengths;
    const int32_t* counts;  /* or NULL */
    const int32_t* parents; /* or NULL */
    const float* lse;
    float* weights;
} BeamgradWeights;

DBS_CUDA_EXPORT int64_t beamgrad_accumulate_weights_workspace_size(const BeamgradWeights* args);
DBS_CUDA_EXPORT int beamgrad_accumulate_weights(const BeamgradWeights* args, void* workspace, int64_t workspace_bytes,
                                                void* stream);

/* A cache cut to its heaviest tokens. Of a sequence of more than b tokens (b =
 * budgets[s], or `budget` where that is NULL) the last r = min(recent, b) stay, the
 * first f = min(first, b - r), and of those between the b - r - f with the largest
 * weights, of equal ones the earlier; NaN counts as less than every number. They move
 * together in their order, in place in every pool, and the pages that hold no token
 * any more are given back. n_weights sets of weights, one for each pools.n / n_weights
 * pools in turn: weights[i] [sequences, heads, table_pages * page_tokens] float32 with
 * weight_strides[2 i], [2 i + 1] (elements, host arrays) chooses for every head by itself,
 * a pool's row being `heads` parts of equal length. to_weights[i], contiguous, gets the
 * weights of the tokens that stay, zeros behind them.
 *
 * A sequence of at most b tokens stays as it is, as does one that has no page for one of
 * its tokens, or that would write to a page that others hold too (refs != 1): its
 * places are copied, weights too. b < 0 counts as 0. At most 65535 sequences, 1024 heads,
 * rows of 2 MB. */
typedef struct BeamgradEviction {
    const float* const* weights;
    const int64_t* weight_strides;
    float* const* to_weights;
    int32_t n_weights;
    int32_t heads;
    const int32_t* budgets; /* device, [sequences], or NULL */
    int32_t budget;
    int32_t recent;
    int32_t first;
    int32_t reserved; /* 0 */
} BeamgradEviction;

DBS_CUDA_EXPORT int64_t beamgrad_evict_tokens_workspace_size(const BeamgradPools* pools, const BeamgradEviction* args,
                                                             int sequences, int table_pages);
DBS_CUDA_EXPORT int beamgrad_evict_tokens(const BeamgradPools* pools, const BeamgradEviction* args,
                                          const BeamgradTable* from, int sequences, int table_pages,
                                          const BeamgradTable* to, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
