/*
 * Attention over a paged cache of keys and values, next to the search over its keys: a decoder's step appends its tokens' rows,
 * attends to the recent ones in full and to those of the far ones that a search named, and joins the two parts.
 * No counterpart in the reference.
 *
 * The cache is two device tensors [n_pages, page_size, n_heads, dim], keys and values, f16, bf16 or f32, of any strides that put
 * every row of `dim` elements on a 16-byte boundary (the row itself is contiguous); dim is at most 256 and a row a multiple of 16
 * bytes long.  A token's slot is page * page_size + its place in the page: the id under which the token's key goes into an index,
 * so that the ids that a search returns are slots.  `pages` (i32 [n_sequences, width]) names the pages of each sequence in the order
 * of its positions: position i is in pages[sequence, i / page_size] at place i % page_size; an entry that is no page of the cache
 * (-1, say) holds no tokens.
 *
 * All tensors are on the device of the handle.  Queries and outputs have the cache's element type; query head i reads the rows of
 * head i / (n_query_heads / n_heads).  Scores, softmax and sums are held in 32 bits; outputs are rounded once.  Where nothing may be
 * attended to, the output row is 0 and its lse -inf.  Weights below 2^-100 of the largest may count as 0, in attention over f16 those
 * below 2^-38 (times an infinite value that is no number).  The calls only enqueue work on the handle's stream and can be captured.
 * Results do not depend on anything but the arguments, the GPU's number of SMs and the clusters of thread blocks that it holds at once.
 */
#ifndef CUVS_B200_KV_CACHE_H_
#define CUVS_B200_KV_CACHE_H_

#include "cuvs_core_c_api.h"
#include "cuvs_ivf_pq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Writes the rows of new tokens to their places and, with frequencies, turns keys and queries by their positions on the way.
 * new_keys, new_values: [n_tokens, n_heads, dim]; pages: i32 [n_sequences, width]; positions: i32 [n_tokens]; sequences: i32
 * [n_tokens], the sequence of each token, or NULL: token i is one of sequence i; queries, rotated: [n_tokens, n_query_heads, dim], or
 * both NULL (`rotated` may be `queries`); frequencies: f64 or f32 [n_pairs], n_pairs <= dim / 2, or NULL: nothing is turned; pair i
 * of a row is its columns (i, i + n_pairs), interleaved: (2i, 2i + 1), turned by position * frequencies[i] radians; further columns
 * stay.  slots: i64 [n_tokens], receives the tokens' slots.
 * A token whose position is negative, whose sequence does not exist or whose page is not in the cache gets slot -1 and is not
 * written; the query row of a token with a negative position is copied as it is.  Two tokens of a call must not have the same slot. */
CUVS_EXPORT cuvsError_t cuvsKvCacheAppend(cuvsResources_t res, DLManagedTensor* keys, DLManagedTensor* values,
                                          DLManagedTensor* new_keys, DLManagedTensor* new_values, DLManagedTensor* pages,
                                          DLManagedTensor* positions, DLManagedTensor* sequences, DLManagedTensor* queries,
                                          DLManagedTensor* frequencies, bool interleaved, DLManagedTensor* slots,
                                          DLManagedTensor* rotated);

/* Attention of one token per sequence to the sequence's positions 0 .. lengths[i] - 1, or the last `window` of them (window > 0; 0:
 * all).  queries, out: [n_sequences, n_query_heads, dim]; lengths: i32 [n_sequences] (what exceeds the table's width is not there;
 * a negative length is 0); scores are scale * q.k; filter: NO_FILTER or BITSET over slots; lse: f32 [n_sequences, n_query_heads],
 * the natural logarithm of the softmax's denominator.  workspace: u8 [cuvsKvCacheAttentionWorkspace bytes] that no other call uses
 * until this one's work is done, or NULL: the handle's own for this stream (refused while the stream is being captured: what is replayed
 * needs one to itself). */
CUVS_EXPORT cuvsError_t cuvsKvCacheAttention(cuvsResources_t res, DLManagedTensor* keys, DLManagedTensor* values,
                                             DLManagedTensor* queries, DLManagedTensor* pages, DLManagedTensor* lengths, float scale,
                                             int64_t window, cuvsFilter filter, DLManagedTensor* out, DLManagedTensor* lse,
                                             DLManagedTensor* workspace);
/* Bytes that cuvsKvCacheAttention needs for tensors of these shapes; it depends on shapes, window and element type alone. */
CUVS_EXPORT cuvsError_t cuvsKvCacheAttentionWorkspace(cuvsResources_t res, DLManagedTensor* keys, DLManagedTensor* queries,
                                                      DLManagedTensor* pages, int64_t window, size_t* bytes);

/* Attention of every query head of a token to the slots that its list names: candidates i64 [n_tokens, n_query_heads,
 * n_candidates], as a search over the keys returns them.  Ids that are no slots (the search's "no such neighbour", -1) and slots
 * whose bit of the filter is 0 are skipped; a slot that is named twice counts twice.  queries, out: [n_tokens, n_query_heads, dim];
 * lse: f32 [n_tokens, n_query_heads]. */
CUVS_EXPORT cuvsError_t cuvsKvCacheAttendCandidates(cuvsResources_t res, DLManagedTensor* keys, DLManagedTensor* values,
                                                    DLManagedTensor* queries, DLManagedTensor* candidates, float scale,
                                                    cuvsFilter filter, DLManagedTensor* out, DLManagedTensor* lse);

/* Joins parts of one softmax over disjoint sets of rows: parts [n_parts, n_tokens, n_heads, dim] (any 16-byte strides) and their
 * lse, f32 [n_parts, n_tokens, n_heads] (any strides), give out [n_tokens, n_heads, dim] and lse f32 [n_tokens, n_heads].  What the
 * row of a part holds whose lse is -inf does not count. */
CUVS_EXPORT cuvsError_t cuvsKvCacheMergeParts(cuvsResources_t res, DLManagedTensor* parts, DLManagedTensor* parts_lse,
                                              DLManagedTensor* out, DLManagedTensor* lse);

/* The calls above on arrays that are described by words: op 0 append, 1 attention, 2 attend candidates, 3 merge parts.  The
 * tensors come in the order of the calls, each as ndim | type code << 32 | bits << 40 | lanes << 48; address; device type | device
 * id << 32; the shape; the strides in elements -- or as one word 0 where there is none -- with a filter as a u32 tensor in the place
 * of its argument; behind them the scalars: {interleaved}, {window, bits of the f32 scale}, {bits of the scale}, {}.  The
 * work goes to `stream`, whatever the handle's own is, and is waited for if `sync`.  Returns a cuvsError_t, or 2 where the call needs a
 * workspace to itself (attention that is captured): nothing was done then. */
CUVS_EXPORT int cuvsB200KvCacheArrays(cuvsResources_t res, cudaStream_t stream, int op, const int64_t* words, int64_t n_words, bool sync);
/* The same for a caller in Python: tensors as Python objects (of the type that the table of DLPack exchange functions is from, or none),
 * read in place; the caller holds the interpreter's lock.  `integer`: interleaved, or the window.  Does not wait: cuvsB200KvCacheWait
 * does, without the lock. */
CUVS_EXPORT cuvsError_t cuvsB200SetTensorExchange(const void* table, const void* none);
CUVS_EXPORT int cuvsB200KvCacheTensors(cuvsResources_t res, cudaStream_t stream, int op, void* t0, void* t1, void* t2, void* t3, void* t4,
                                       void* t5, void* t6, void* t7, void* t8, void* t9, void* t10, int64_t integer, float scale, bool sync);
CUVS_EXPORT cuvsError_t cuvsB200KvCacheWait(cuvsResources_t res, cudaStream_t stream);
/* cuvsKvCacheAttentionWorkspace on the words of keys, queries, pages and {window}. */
CUVS_EXPORT cuvsError_t cuvsB200KvCacheWorkspaceArrays(cuvsResources_t res, const int64_t* words, int64_t n_words, size_t* bytes);
/* The checks of such a call alone, for a handle of `device`: touches no GPU and reads no tensor. */
CUVS_EXPORT cuvsError_t cuvsB200KvCacheCheck(int device, int op, const int64_t* words, int64_t n_words);

#ifdef __cplusplus
}
#endif
#endif
