/* SPDX-License-Identifier: MIT
 *
 * The state of a model in a beam search, on the GPU: attention over a paged
 * cache of keys and values, the pages of that cache, and the reordering of
 * dense states. Additions of libdbs_hip.so beside the search itself
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

#ifdef __cplusplus
}
#endif
