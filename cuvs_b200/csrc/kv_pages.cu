// Trees of drafted tokens, and what is left of them: ancestors and positions from parents, the rows of the path that was kept, copies of pages.
#include "kv_rows.cuh"

#include <algorithm>

namespace cuvs_b200::kv {

namespace {

// ---- draft_tree ---------------------------------------------------------------------------------------------------------------
//
// A token reaches itself and what its parent reaches.  Every token looks 1, 2, 4, .. steps up: after k rounds `up` is the ancestor 2^k steps up
// (or how the way ends) and the token's bits are those of the 2^k - 1 nearest ancestors and its own; a round adds the bits of `up` and takes
// its `up`.  ceil(log2 n) rounds see a whole tree in whatever order its tokens stand, and a way that has not ended by then goes in a circle.
//
// What bounds it: the latency of a launch and of the rounds, which one block makes per sequence in shared memory, a thread per token with the token's
// words in registers.  (A thread per word, with their divisions: 64 trees of 255 tokens 10.7 us.)
constexpr int32_t kNoToken = -2, kFollows = -1;

__global__ void __launch_bounds__(1024) draft_tree_kernel(draft_tree_args a)
{
  chain_begin();
  constexpr uint32_t kMost = 32;  // words of 1,024 tokens
  extern __shared__ uint32_t s_words[];
  const uint32_t n = a.n_drafted, words = (n + 31) / 32, pitch = words | 1u, sequence = blockIdx.x, token = threadIdx.x;
  int32_t* s_up        = reinterpret_cast<int32_t*>(s_words + n * pitch);
  const bool exists    = token < n;
  const int64_t length = max(a.lengths[sequence], 0);
  const int32_t parent = exists ? a.parents[int64_t(sequence) * a.parents_stride + token] : kNoToken;
  int32_t up           = parent >= kFollows && parent < int32_t(n) ? parent : kNoToken;
  uint32_t bits[kMost];
#pragma unroll
  for (uint32_t word = 0; word < kMost; word++) {
    if (word >= words) { break; }
    bits[word] = word == token / 32 ? 1u << (token & 31u) : 0u;
    if (exists) { s_words[token * pitch + word] = bits[word]; }
  }
  if (exists) { s_up[token] = up; }
  __syncthreads();
  for (uint32_t reach = 1; reach < n; reach *= 2) {  // the way of a chain of n tokens ends n steps up
    int32_t next = up;
    if (up >= 0) {
#pragma unroll
      for (uint32_t word = 0; word < kMost; word++) {
        if (word >= words) { break; }
        bits[word] |= s_words[up * pitch + word];
      }
      next = s_up[up];
    }
    if (__syncthreads_or(up >= 0) == 0) { break; }  // all have read; all ways have ended
    if (up >= 0) {
#pragma unroll
      for (uint32_t word = 0; word < kMost; word++) {
        if (word >= words) { break; }
        s_words[token * pitch + word] = bits[word];
      }
      up          = next;
      s_up[token] = up;
    }
    __syncthreads();
  }
  int64_t position = length - 1;
#pragma unroll
  for (uint32_t word = 0; word < kMost; word++) {
    if (word >= words) { break; }
    position += __popc(bits[word]);
  }
  const bool there = up == kFollows && position <= 0x7FFFFFFF;
  if (exists) {
    s_up[token] = there;
    a.positions[size_t(sequence) * n + token] = there ? int32_t(position) : -1;
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < n * words; i += blockDim.x) {
    const uint32_t of = i / words;
    a.mask[size_t(sequence) * n * words + i] = s_up[of] != 0 ? s_words[of * pitch + (i - of * words)] : 0u;
  }
}

// ---- keep_path ----------------------------------------------------------------------------------------------------------------
//
// Row length + path[i] of a sequence moves to length + i.  Entries ascend, so path[i] >= i: a row's new place is never one that a later entry
// still has to be read from, only its own or one that was read before.  A warp has some 16-byte columns of a sequence's rows, and each of its lanes
// moves its column entry by entry, a few at a time (all of them read before one is written).
//
// What bounds it: latency, for rows are few: the launch, the path, the table, the rows.
constexpr int kKeepWarps = 4;

__global__ void __launch_bounds__(kKeepWarps * 32) keep_path_kernel(keep_path_args a, uint32_t slices)
{
  chain_begin();
  constexpr int AHEAD     = 8;
  const uint32_t lane     = threadIdx.x & 31u;
  const uint32_t sequence = blockIdx.x / slices, slice = blockIdx.x - sequence * slices;
  const int32_t* path     = a.paths + int64_t(sequence) * a.paths_stride;
  const int32_t* table    = a.pages + int64_t(sequence) * a.table_stride;
  const int32_t length    = max(a.lengths[sequence], 0);
  // how far the path goes: every entry is greater than the one before it, and the new length is a number of 32 bits
  uint32_t n = 0;
  for (uint32_t i0 = 0; i0 < a.n_entries; i0 += 32) {
    const uint32_t i     = i0 + lane;
    const int32_t entry  = i < a.n_entries ? path[i] : -1;
    const int32_t before = i > 0 && i < a.n_entries ? path[i - 1] : -1;
    const unsigned bad   = __ballot_sync(kAllLanes, !(entry > before && int64_t(length) + entry < 0x7FFFFFFF));
    n                    = bad != 0u ? i0 + __ffs(int(bad)) - 1 : i0 + 32;
    if (bad != 0u) { break; }
  }
  const uint32_t pieces = a.row_bytes / 16, columns = 2 * a.cache.n_heads * pieces;  // keys, then values
  const uint32_t column = (slice * kKeepWarps + (threadIdx.x >> 5)) * 32 + lane;
  const bool has        = column < columns;
  const bool of_values  = column >= columns / 2;
  const uint32_t at     = of_values ? column - columns / 2 : column;
  const uint32_t head   = at / pieces, piece = at - head * pieces;
  const int64_t size    = a.row_bytes / a.cache.dim;
  char* rows            = const_cast<char*>(of_values ? a.cache.values + int64_t(head) * a.cache.v_head * size
                                                      : a.cache.keys + int64_t(head) * a.cache.k_head * size) + piece * 16;
  const int64_t page_on = (of_values ? a.cache.v_page : a.cache.k_page) * size, token_on = (of_values ? a.cache.v_token : a.cache.k_token) * size;
  for (uint32_t i0 = 0; i0 < n; i0 += 32) {
    // lane i looks up the places of entry i0 + i
    const uint32_t i = i0 + lane;
    int64_t from = -1, to = -1;
    if (i < n && path[i] != int32_t(i)) {
      from = slot_of(table, a.table_width, length + path[i], a.cache.page, a.cache.n_pages);
      to   = slot_of(table, a.table_width, length + int32_t(i), a.cache.page, a.cache.n_pages);
    }
    const bool moves = from >= 0 && to >= 0;
    uint32_t from_page, from_place, to_page, to_place;
    split_slot(a.cache, moves ? from : 0, from_page, from_place);
    split_slot(a.cache, moves ? to : 0, to_page, to_place);
    unsigned left = __ballot_sync(kAllLanes, moves);
    while (left != 0u) {
      uint4 x[AHEAD];
      char* target[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; u++) {
        const bool some     = left != 0u;
        const int of        = some ? __ffs(int(left)) - 1 : 0;
        const char* source  = rows + __shfl_sync(kAllLanes, from_page, of) * page_on + __shfl_sync(kAllLanes, from_place, of) * token_on;
        char* const place   = rows + __shfl_sync(kAllLanes, to_page, of) * page_on + __shfl_sync(kAllLanes, to_place, of) * token_on;
        target[u]           = some && has ? place : nullptr;
        x[u]                = load_piece(source, some && has);
        left &= left - 1u;
      }
#pragma unroll
      for (int u = 0; u < AHEAD; u++) {
        if (target[u] != nullptr) { *reinterpret_cast<uint4*>(target[u]) = x[u]; }
      }
    }
  }
  if (slice == 0 && threadIdx.x == 0) { a.kept[sequence] = length + int32_t(n); }
}

// ---- copy_pages ---------------------------------------------------------------------------------------------------------------
//
// What bounds it: HBM, every row read and written once.  A page is a grid of rows of 16-byte pieces, keys and values; a thread has every so many-th
// piece of a pair's two pages and eight of them in flight.
constexpr int kCopyThreads = 256;

__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(copy_pages_args a, uint32_t slices, page_divisor pieces, page_divisor inner,
                                                                  bool heads_inside)
{
  chain_begin();
  constexpr int AHEAD  = 8;
  const uint32_t pair  = blockIdx.x / slices, slice = blockIdx.x - pair * slices;
  const int32_t source = a.sources[pair], target = a.targets[pair];
  if (source < 0 || source >= a.cache.n_pages || target < 0 || target >= a.cache.n_pages) { return; }
  const int64_t size   = a.row_bytes / a.cache.dim;
  const uint32_t half  = a.cache.n_heads * a.cache.page.size * pieces.size, all = 2 * half;  // below 2^31
  const char* k_from   = a.cache.keys + source * (a.cache.k_page * size);
  const char* v_from   = a.cache.values + source * (a.cache.v_page * size);
  char* k_to           = const_cast<char*>(a.cache.keys) + target * (a.cache.k_page * size);
  char* v_to           = const_cast<char*>(a.cache.values) + target * (a.cache.v_page * size);
  // strides from one row to the next in the order in which they lie
  const int64_t k_in = (heads_inside ? a.cache.k_head : a.cache.k_token) * size, k_out = (heads_inside ? a.cache.k_token : a.cache.k_head) * size;
  const int64_t v_in = (heads_inside ? a.cache.v_head : a.cache.v_token) * size, v_out = (heads_inside ? a.cache.v_token : a.cache.v_head) * size;
  for (uint32_t i0 = slice * kCopyThreads * AHEAD + threadIdx.x; i0 < all; i0 += slices * kCopyThreads * AHEAD) {
    uint4 x[AHEAD];
    char* to[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; u++) {
      const uint32_t i     = i0 + u * kCopyThreads;
      const bool of_values = i >= half;
      uint32_t row, piece, out, in;
      split_place(min(of_values ? i - half : i, half - 1), pieces, row, piece);
      split_place(row, inner, out, in);
      const int64_t at = (of_values ? out * v_out + in * v_in : out * k_out + in * k_in) + piece * 16;
      x[u]  = load_piece((of_values ? v_from : k_from) + at, i < all);
      to[u] = (of_values ? v_to : k_to) + at;
    }
#pragma unroll
    for (int u = 0; u < AHEAD; u++) {
      if (i0 + u * kCopyThreads < all) { *reinterpret_cast<uint4*>(to[u]) = x[u]; }
    }
  }
}

}  // namespace

void draft_tree(resources& res, cudaStream_t stream, const draft_tree_args& a)
{
  if (a.n_sequences == 0 || a.n_drafted == 0) { return; }
  const uint32_t words = ceildiv(a.n_drafted, 32u);
  const size_t smem    = size_t(a.n_drafted) * ((words | 1u) + 1) * sizeof(uint32_t);
  if (smem > 48 * 1024) { ensure_dynamic_smem(reinterpret_cast<const void*>(draft_tree_kernel), smem); }
  const uint32_t threads = round_up(a.n_drafted, 32u);
  launch_chained(draft_tree_kernel, dim3(a.n_sequences), threads, smem, stream, a);
  count_launches(res, 1);
}

void keep_path(resources& res, cudaStream_t stream, const keep_path_args& a)
{
  if (a.n_sequences == 0) { return; }
  const uint32_t columns = 2 * a.cache.n_heads * (a.row_bytes / 16);
  const uint32_t slices  = ceildiv(columns, uint32_t(kKeepWarps * 32));
  launch_chained(keep_path_kernel, dim3(a.n_sequences * slices), kKeepWarps * 32, 0, stream, a, slices);
  count_launches(res, 1);
}

void copy_pages(resources& res, cudaStream_t stream, const copy_pages_args& a)
{
  if (a.n_pairs == 0) { return; }
  // until there are 16 blocks of an SM, or a thread has its eight pieces
  const uint32_t pieces = a.row_bytes / 16, all = 2 * a.cache.n_heads * a.cache.page.size * pieces;
  const uint32_t slices = std::max(1u, std::min(ceildiv(all, uint32_t(kCopyThreads * 8)), ceildiv(uint32_t(res.sm_count) * 16, a.n_pairs)));
  const bool heads_inside = a.cache.k_head < a.cache.k_token;
  launch_chained(copy_pages_kernel, dim3(a.n_pairs * slices), kCopyThreads, 0, stream, a, slices, divisor_of(pieces),
                 divisor_of(heads_inside ? a.cache.n_heads : a.cache.page.size), heads_inside);
  count_launches(res, 1);
}

}  // namespace cuvs_b200::kv
