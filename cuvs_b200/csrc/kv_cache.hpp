// Attention over a paged cache of keys and values: what the entry points check and hand to the kernels.
#pragma once

#include "common.hpp"
#include "kv_place.hpp"

#include <cstdint>

// These calls go by the stream that they are given and touch nothing of the handle but its count of launches and, under a lock, its workspaces
// of streams: several threads may make them through one handle, and one more may search through it meanwhile.
namespace cuvs_b200::kv {

inline void count_launches(resources& res, uint64_t n) { res.launches += n; }

enum class elem { f16, bf16, f32 };

// An array as its caller describes it (strides in elements); no data and ndim = 0: not given.
struct tensor {
  char* data       = nullptr;
  int code         = 0;
  int bits         = 0;
  int ndim         = 0;
  int device_type  = 0;
  int device_id    = 0;
  int64_t shape[4]  = {0, 0, 0, 0};
  int64_t stride[4] = {0, 0, 0, 0};
  bool given() const { return ndim != 0; }
};

// Rows of one head: keys and values [n_pages, page_size, n_heads, dim] at any strides (in elements) that leave every row on a
// 16-byte boundary.  A slot is page * page_size + place in the page.
struct cache_view {
  const char* keys;
  const char* values;
  int64_t k_page, k_token, k_head;
  int64_t v_page, v_token, v_head;
  // For reading: the same strides of pages and tokens in units of 1 << unit_shift bytes, small enough that a row's place fits 32 bits.
  uint32_t k_page_units, k_token_units, v_page_units, v_token_units, unit_shift;
  int64_t n_slots;
  int32_t n_pages;
  page_divisor page;
  uint32_t n_heads;
  uint32_t dim;
  const uint32_t* filter;  // bit i: slot i may be attended; nullptr: all
};

// [n, n_heads, dim] rows at any 16-byte strides
struct rows_view {
  char* data;
  int64_t row, head;
};

struct append_args {
  cache_view cache;
  elem type;
  uint32_t n_tokens, n_sequences, table_width;
  int64_t table_stride;  // from one sequence's row of `pages` to the next
  const char* keys;  // new rows [n_tokens, n_heads, dim]
  const char* values;
  int64_t k_row, k_head, v_row, v_head;
  uint32_t n_query_heads;  // 0: no queries
  rows_view queries, rotated;
  const int32_t* pages;      // [n_sequences, table_width]
  const int32_t* positions;  // [n_tokens]
  const int32_t* sequences;  // [n_tokens], nullptr: token i is one of sequence i
  const void* frequencies;   // [n_pairs] f64, or f32
  bool frequencies_f32;
  uint32_t n_pairs;
  bool interleaved;
  int64_t* slots;  // [n_tokens]
};
void append(resources& res, cudaStream_t stream, const append_args& a);

struct attention_args {
  cache_view cache;
  elem type;
  uint32_t n_sequences, n_query_heads, table_width;
  int64_t table_stride;
  rows_view queries, out;
  const int32_t* pages;    // [n_sequences, table_width]
  const int32_t* lengths;  // [n_sequences]
  float scale;
  int64_t window;  // 0: none
  float* lse;      // [n_sequences, n_query_heads]
  char* workspace;
  size_t workspace_bytes;
};
// How many bytes of workspace attention() wants, by sizes alone.
size_t attention_workspace(const resources& res, elem type, uint32_t n_sequences, uint32_t n_query_heads, uint32_t n_heads, uint32_t dim,
                           uint64_t capacity, int64_t window);
void attention(resources& res, cudaStream_t stream, const attention_args& a);

struct candidates_args {
  cache_view cache;
  elem type;
  uint32_t n_tokens, n_query_heads, n_candidates;
  rows_view queries, out;
  const int64_t* candidates;  // [n_tokens, n_query_heads, n_candidates]
  float scale;
  float* lse;  // [n_tokens, n_query_heads]
};
void attend_candidates(resources& res, cudaStream_t stream, const candidates_args& a);

struct merge_args {
  elem type;
  uint32_t n_parts, n_tokens, n_heads, dim;
  const char* parts;  // [n_parts, n_tokens, n_heads, dim]
  int64_t p_part, p_row, p_head;
  const float* parts_lse;  // [n_parts, n_tokens, n_heads]
  int64_t l_part, l_row, l_head;
  rows_view out;
  float* lse;  // [n_tokens, n_heads]
};
void merge_parts(resources& res, cudaStream_t stream, const merge_args& a);

}  // namespace cuvs_b200::kv
