// Who does what when query heads attend to lists of rows: units, tiles, shares, clusters, and the joining of what several blocks have of
// a unit.
//
// A unit is a (sequence, key head, block of query heads) with its list of rows, cut into tiles.  Two ways to deal the tiles out:
//
// Shares.  All units' tiles stand in one row, and each of a fixed number of resident blocks takes an equal, contiguous share of it,
// whatever the lengths are (they are known on the device alone: every warp finds its block's share from them itself).  A unit that lies in
// one share is finished there; of a unit that several share, each block leaves a part (top, sum and weighted sum in 32 bits), and a second
// kernel joins the parts in the order of the blocks.
//
// Clusters.  One cluster of blocks per unit, whose blocks take equal runs of its tiles and join their parts through each other's shared
// memory: one launch and no workspace, but no balance between units.
//
// Nothing depends on the order in which blocks run.
#pragma once

#include "kv_rows.cuh"

#include <cooperative_groups.h>

namespace cuvs_b200::kv {

// Warps of a block: small blocks, several to an SM, balance best; where units are fewer than SMs, one large block has an SM's warps for one
// unit.
constexpr int kSmall = 4, kLarge = 12;

struct work_view {
  uint32_t n_sequences;
  uint32_t n_units;      // per sequence: key heads x blocks of query heads
  uint32_t n_blocks_of;  // blocks of query heads of one key head
  uint32_t group;        // query heads of one key head
  uint32_t cluster;      // blocks of a unit's cluster; 0: shares
};

// ---- lists --------------------------------------------------------------------------------------------------------------------

// All positions of a sequence, or its last ones.  A tile begins at a multiple of 16 positions, so that 16 rows lie in one page where pages
// are multiples of 16.
struct positions {
  const int32_t* pages;
  const int32_t* lengths;
  int64_t table_stride;
  int64_t window;
  uint32_t width;

  struct list {
    const int32_t* table;
    uint32_t first, end, base;
  };
  __device__ __forceinline__ uint32_t open(const cache_view& c, uint32_t sequence, uint32_t tile, list& l) const
  {
    attended(lengths[sequence], window, width, c.page_size, l.first, l.end);
    l.table = pages + int64_t(sequence) * table_stride;
    l.base  = l.first & ~15u;
    return l.end > l.first ? (l.end - l.base + tile - 1) / tile : 0u;
  }
  __device__ __forceinline__ void select(const cache_view&, const work_view&, uint32_t, uint32_t, list&) const {}
  // What memory says about row i of the list (-1: it is none); to be looked at later, when it has arrived.
  __device__ __forceinline__ int64_t name(const cache_view& c, const list& l, uint32_t i) const
  {
    const uint32_t at = l.base + i;
    if (at < l.first || at >= l.end) { return -1; }
    uint32_t column, place;
    split_place(at, c.page_size, c.page_shift, column, place);
    return int64_t(l.table[column]);  // at < end: the column is inside the table
  }
  // Its page and place in it; false: it has none.
  __device__ __forceinline__ bool place(const cache_view& c, const list& l, uint32_t i, int64_t name, int64_t& page, uint32_t& place) const
  {
    uint32_t column;
    split_place(l.base + i, c.page_size, c.page_shift, column, place);
    page = name;
    return name >= 0 && name < c.n_pages;
  }
};

// Slots that are named one by one, n for each query head of a token.
struct named_slots {
  const int64_t* ids;
  uint32_t n;

  struct list {
    const int64_t* ids;
  };
  __device__ __forceinline__ uint32_t open(const cache_view&, uint32_t, uint32_t tile, list&) const { return (n + tile - 1) / tile; }
  __device__ __forceinline__ void select(const cache_view&, const work_view& w, uint32_t token, uint32_t unit, list& l) const
  {
    l.ids = ids + (int64_t(token) * w.n_units + unit) * n;
  }
  __device__ __forceinline__ int64_t name(const cache_view&, const list& l, uint32_t i) const { return i < n ? l.ids[i] : -1; }
  __device__ __forceinline__ bool place(const cache_view& c, const list&, uint32_t, int64_t name, int64_t& page, uint32_t& place) const
  {
    const bool there = name >= 0 && name < c.n_slots;
    split_slot(c, there ? name : 0, page, place);
    return there;
  }
};

// ---- shares -------------------------------------------------------------------------------------------------------------------

struct share {
  uint64_t total;   // tiles of all units
  uint32_t blocks;  // that have a share
  __device__ uint64_t start(uint32_t block) const { return block * total / blocks; }
};

// The number of all tiles; every warp sums it up for itself.
template <int TILE, class Lists>
__device__ __forceinline__ uint64_t all_tiles(const cache_view& c, const work_view& w, const Lists& lists)
{
  uint64_t sum = 0;
  typename Lists::list l;
#pragma unroll 4
  for (uint32_t b = threadIdx.x & 31u; b < w.n_sequences; b += 32) { sum += lists.open(c, b, TILE, l); }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { sum += __shfl_xor_sync(kAllLanes, sum, o); }
  return sum * w.n_units;
}
template <int TILE>
__device__ __forceinline__ uint64_t all_tiles(const cache_view& c, const work_view& w, const named_slots& lists)
{
  named_slots::list l;
  return uint64_t(lists.open(c, 0, TILE, l)) * w.n_sequences * w.n_units;
}

// The sequence that tile `at` of all belongs to, and the number of tiles before that sequence.
template <int TILE, class Lists>
__device__ __forceinline__ uint32_t sequence_of(const cache_view& c, const work_view& w, const Lists& lists, uint64_t at, uint64_t& before)
{
  const uint32_t lane = threadIdx.x & 31u;
  before              = 0;
  for (uint32_t b0 = 0; b0 < w.n_sequences; b0 += 32) {  // comes to an end inside: `at` is less than the number of all tiles
    typename Lists::list l;
    const uint64_t mine = b0 + lane < w.n_sequences ? uint64_t(lists.open(c, b0 + lane, TILE, l)) * w.n_units : 0u;
    uint64_t up         = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t t = __shfl_up_sync(kAllLanes, up, o);
      if (lane >= uint32_t(o)) { up += t; }
    }
    const unsigned past = __ballot_sync(kAllLanes, before + up > at);
    if (past != 0u) {
      const int found = __ffs(int(past)) - 1;
      before += __shfl_sync(kAllLanes, up - mine, found);
      return b0 + found;
    }
    before += __shfl_sync(kAllLanes, up, 31);
  }
  return w.n_sequences;
}
template <int TILE>
__device__ __forceinline__ uint32_t sequence_of(const cache_view& c, const work_view& w, const named_slots& lists, uint64_t at, uint64_t& before)
{
  named_slots::list l;
  const uint64_t each     = uint64_t(lists.open(c, 0, TILE, l)) * w.n_units;
  const uint32_t sequence = uint32_t(at / each);
  before                  = sequence * each;
  return sequence;
}

// ---- parts --------------------------------------------------------------------------------------------------------------------

// Two parts per block: 0 of a unit that a block before began, 1 of a unit that this block begins and a later one goes on with.
struct parts_view {
  float* acc;     // [2 blocks][rows][dim]
  float2* stats;  // [2 blocks][rows] top (of scores in powers of two), sum
  // about the unit that block i - 1 begins and block i goes on with: the tile behind its end (0: there is none), sequence | unit << 32
  uint64_t* unit;  // [blocks + 1][2]
  uint32_t rows;   // query heads of a unit, at most
};

inline size_t part_bytes(uint32_t blocks, uint32_t rows, uint32_t dim)
{
  return round_up<size_t>(size_t(2) * blocks * rows * (dim * sizeof(float) + sizeof(float2)), 16) + size_t(blocks + 1) * 16;
}
inline parts_view parts_at(char* workspace, uint32_t blocks, uint32_t rows, uint32_t dim)
{
  parts_view p;
  p.acc   = reinterpret_cast<float*>(workspace);
  p.stats = reinterpret_cast<float2*>(p.acc + size_t(2) * blocks * rows * dim);
  p.unit  = reinterpret_cast<uint64_t*>(workspace + part_bytes(blocks, rows, dim) - size_t(blocks + 1) * 16);
  p.rows  = rows;
  return p;
}

struct result_view {
  rows_view out;
  float* lse;  // [n_sequences, query heads]
};

template <typename T>
__device__ __forceinline__ void store_piece(const rows_view& out, uint32_t sequence, uint32_t head, uint32_t piece, const float* x)
{
  reinterpret_cast<uint4*>(out.data + (int64_t(sequence) * out.row + int64_t(head) * out.head) * int64_t(sizeof(T)))[piece] = floats_to_piece<T>(x);
}

// What a block's warps have of a unit, in shared memory: weighted sums [warps][rows][acc_row], top and sum [warps][rows]; `joined` [rows] is
// for the block's own.
struct block_state {
  float* acc;
  float2* stats;
  float2* joined;
  uint32_t acc_row;
};

// Joins the warps: the block's sums become output rows (whole), a part in the workspace, or warp 0's sums (for the cluster).
enum { TO_OUTPUT, TO_PART, TO_CLUSTER };
template <typename T, int WARPS>
__device__ __forceinline__ void join_warps(const cache_view& c, const work_view& w, const block_state& s, uint32_t rows, uint32_t sequence,
                                           uint32_t head0, const result_view& result, int to, const parts_view& parts, uint32_t part)
{
  constexpr uint32_t E  = kPerPiece<T>;
  const uint32_t pieces = c.dim / E;
  for (uint32_t i = threadIdx.x; i < rows * pieces; i += WARPS * 32) {
    const uint32_t r = i / pieces, piece = i - r * pieces;
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < WARPS; v++) { top = fmaxf(top, s.stats[v * parts.rows + r].x); }
    const float safe = finite_top(top);
    float sum        = 0.0f;
    float x[E]       = {};
#pragma unroll
    for (int v = 0; v < WARPS; v++) {
      const float2 st = s.stats[v * parts.rows + r];
      const float f   = exp2f(st.x - safe);
      sum             = fmaf(st.y, f, sum);
      const float4* a = reinterpret_cast<const float4*>(s.acc + (size_t(v) * parts.rows + r) * s.acc_row + piece * E);
#pragma unroll
      for (uint32_t e = 0; e < E; e += 4) {
        const float4 y = a[e / 4];
        x[e]           = fmaf(y.x, f, x[e]);
        x[e + 1]       = fmaf(y.y, f, x[e + 1]);
        x[e + 2]       = fmaf(y.z, f, x[e + 2]);
        x[e + 3]       = fmaf(y.w, f, x[e + 3]);
      }
    }
    if (to == TO_OUTPUT) {
      const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
      for (uint32_t e = 0; e < E; e++) { x[e] *= scale; }
      store_piece<T>(result.out, sequence, head0 + r, piece, x);
      if (piece == 0) { result.lse[size_t(sequence) * (w.group * c.n_heads) + head0 + r] = (safe + log2f(sum)) * kLn2; }
    } else {
      float* base = to == TO_PART ? parts.acc + (size_t(part) * parts.rows + r) * c.dim : s.acc + size_t(r) * s.acc_row;
      float4* a   = reinterpret_cast<float4*>(base + piece * E);
#pragma unroll
      for (uint32_t e = 0; e < E; e += 4) { a[e / 4] = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]); }
      if (piece == 0) { (to == TO_PART ? parts.stats + size_t(part) * parts.rows : s.joined)[r] = make_float2(top, sum); }
    }
  }
}

// Joins the blocks of a cluster, whose sums lie in warp 0's place of each: every block writes a share of the output.
template <typename T, int WARPS>
__device__ __forceinline__ void join_cluster(const cache_view& c, const work_view& w, const block_state& s, uint32_t rows, uint32_t sequence,
                                             uint32_t head0, const result_view& result)
{
  constexpr uint32_t E  = kPerPiece<T>;
  const uint32_t pieces = c.dim / E;
  auto cluster          = cooperative_groups::this_cluster();
  cluster.sync();
  for (uint32_t i = cluster.block_rank() * (WARPS * 32) + threadIdx.x; i < rows * pieces; i += w.cluster * (WARPS * 32)) {
    const uint32_t r = i / pieces, piece = i - r * pieces;
    float top = -INFINITY;
    for (uint32_t v = 0; v < w.cluster; v++) { top = fmaxf(top, cluster.map_shared_rank(s.joined, v)[r].x); }
    const float safe = finite_top(top);
    float sum        = 0.0f;
    float x[E]       = {};
#pragma unroll 4
    for (uint32_t v = 0; v < w.cluster; v++) {
      const float2 st = cluster.map_shared_rank(s.joined, v)[r];
      const float f   = exp2f(st.x - safe);
      sum             = fmaf(st.y, f, sum);
      const float4* a = reinterpret_cast<const float4*>(cluster.map_shared_rank(s.acc, v) + size_t(r) * s.acc_row + piece * E);
#pragma unroll
      for (uint32_t e = 0; e < E; e += 4) {
        const float4 y = a[e / 4];
        x[e]           = fmaf(y.x, f, x[e]);
        x[e + 1]       = fmaf(y.y, f, x[e + 1]);
        x[e + 2]       = fmaf(y.z, f, x[e + 2]);
        x[e + 3]       = fmaf(y.w, f, x[e + 3]);
      }
    }
    const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (uint32_t e = 0; e < E; e++) { x[e] *= scale; }
    store_piece<T>(result.out, sequence, head0 + r, piece, x);
    if (piece == 0) { result.lse[size_t(sequence) * (w.group * c.n_heads) + head0 + r] = (safe + log2f(sum)) * kLn2; }
  }
  cluster.sync();  // no block leaves while others read its shared memory
}

// Rows of sequences that attend to nothing: they have no tiles in any share.
template <typename T, int WARPS, int TILE, class Lists>
__device__ __forceinline__ void empty_rows(const cache_view& c, const work_view& w, const Lists& lists, const result_view& result)
{
  constexpr uint32_t E   = kPerPiece<T>;
  const uint32_t heads   = w.group * c.n_heads;
  const float nothing[8] = {};
  for (uint32_t b = blockIdx.x; b < w.n_sequences; b += gridDim.x) {
    typename Lists::list l;
    if (lists.open(c, b, TILE, l) != 0u) { continue; }
    for (uint32_t i = threadIdx.x; i < heads * (c.dim / E); i += WARPS * 32) {
      store_piece<T>(result.out, b, i / (c.dim / E), i % (c.dim / E), nothing);
    }
    for (uint32_t i = threadIdx.x; i < heads; i += WARPS * 32) { result.lse[size_t(b) * heads + i] = -INFINITY; }
  }
}

// Goes through what the block has to do, unit by unit: body(sequence, unit, list, tile0, tile1) leaves its warps' state in shared memory.
template <typename T, int WARPS, int TILE, class Lists, class Body>
__device__ __forceinline__ void each_unit(const cache_view& c, const work_view& w, const Lists& lists, const result_view& result,
                                          const parts_view& parts, const block_state& s, Body&& body)
{
  typename Lists::list l;
  uint64_t unfinished = 0, where = 0;
  share all{};
  uint32_t sequence = 0, unit = 0, n = 0;     // n: tiles of a unit
  uint64_t at = 0, stop = 0, before = 0;      // tiles: the next one, the share's end, those before the sequence
  if (w.cluster != 0u) {
    const uint32_t which = blockIdx.x / w.cluster, rank = blockIdx.x - which * w.cluster;
    sequence = which / w.n_units;
    unit     = which - sequence * w.n_units;
    n        = lists.open(c, sequence, TILE, l);
    at       = uint64_t(rank) * n / w.cluster;
    stop     = uint64_t(rank + 1) * n / w.cluster;
  } else {
    all.total  = all_tiles<TILE>(c, w, lists);
    all.blocks = uint32_t(min(uint64_t(gridDim.x), all.total));
    if (blockIdx.x < all.blocks) {
      at       = all.start(blockIdx.x);
      stop     = all.start(blockIdx.x + 1);
      sequence = sequence_of<TILE>(c, w, lists, at, before);
      if (sequence < w.n_sequences) { n = lists.open(c, sequence, TILE, l); }
    }
  }
  bool more = w.cluster != 0u || at < stop;
  while (more) {
    uint64_t begin = 0, last = stop;
    if (w.cluster == 0u) {
      while (at >= before + uint64_t(n) * w.n_units) {  // on to the next sequence that has tiles
        before += uint64_t(n) * w.n_units;
        if (++sequence >= w.n_sequences) { break; }
        n = lists.open(c, sequence, TILE, l);
      }
      if (sequence >= w.n_sequences) { break; }  // lengths that changed meanwhile
      unit  = uint32_t((at - before) / n);
      begin = before + uint64_t(unit) * n;
      last  = min(stop, begin + n);
    }
    lists.select(c, w, sequence, unit, l);
    body(sequence, unit, l, uint32_t(at - begin), uint32_t(last - begin));
    const uint32_t head = unit / w.n_blocks_of, of = unit - head * w.n_blocks_of;
    const uint32_t rows = min(parts.rows, w.group - of * parts.rows), head0 = head * w.group + of * parts.rows;
    __syncthreads();
    if (w.cluster > 1u) {
      join_warps<T, WARPS>(c, w, s, rows, sequence, head0, result, TO_CLUSTER, parts, 0);
      join_cluster<T, WARPS>(c, w, s, rows, sequence, head0, result);
      return;
    }
    const bool whole = w.cluster == 1u || (at == begin && last == begin + n);
    join_warps<T, WARPS>(c, w, s, rows, sequence, head0, result, whole ? TO_OUTPUT : TO_PART, parts, 2 * blockIdx.x + (at == begin ? 1u : 0u));
    __syncthreads();
    if (at == begin && !whole) {
      unfinished = begin + n;
      where      = uint64_t(sequence) | uint64_t(unit) << 32;
    }
    at   = last;
    more = w.cluster == 0u && at < stop;
  }
  if (w.cluster != 0u) { return; }
  if (parts.unit != nullptr && threadIdx.x == 0) {
    parts.unit[2 * (blockIdx.x + 1)]     = unfinished;
    parts.unit[2 * (blockIdx.x + 1) + 1] = where;
    if (blockIdx.x == 0) {
      parts.unit[0] = all.total;
      parts.unit[1] = all.blocks;
    }
  }
  empty_rows<T, WARPS, TILE>(c, w, lists, result);
}

// ---- joining parts ------------------------------------------------------------------------------------------------------------

constexpr int kJoinWarps = 8;

// One block per share that begins inside a unit begun by the block before.  SPLIT warps take turns at the parts of a row.
template <typename T, int SPLIT>
__global__ void __launch_bounds__(kJoinWarps * 32)
join_kernel(work_view w, parts_view parts, uint32_t dim, uint32_t n_heads, result_view result)
{
  chain_begin();
  constexpr int E      = 4;
  const uint32_t i     = blockIdx.x + 1;
  const uint64_t stop  = parts.unit[2 * i];
  if (stop == 0u) { return; }
  const uint64_t where = parts.unit[2 * i + 1];
  const share s{parts.unit[0], uint32_t(parts.unit[1])};
  const uint32_t sequence = uint32_t(where), unit = uint32_t(where >> 32);
  const uint32_t head = unit / w.n_blocks_of, of = unit - head * w.n_blocks_of;
  const uint32_t rows = min(parts.rows, w.group - of * parts.rows);
  const uint32_t head0 = head * w.group + of * parts.rows;
  // the part that begins the unit, then the first parts of all blocks whose share begins before the unit's end
  // (block j's share begins at j * total / blocks, rounded down: before `stop` as long as j * total < stop * blocks)
  const uint32_t behind = uint32_t(min((stop * s.blocks + s.total - 1) / s.total, uint64_t(s.blocks)));
  const uint32_t n    = 1 + behind - i;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  auto part_at = [&](uint32_t p) { return p == 0 ? 2 * (i - 1) + 1 : 2 * (i + p - 1); };
  __shared__ float s_acc[SPLIT > 1 ? kJoinWarps : 1][256];
  for (uint32_t r = blockIdx.y * (kJoinWarps / SPLIT) + warp / SPLIT; r < rows; r += gridDim.y * (kJoinWarps / SPLIT)) {
    float top = -INFINITY;
    for (uint32_t p = lane; p < n; p += 32) { top = fmaxf(top, parts.stats[size_t(part_at(p)) * parts.rows + r].x); }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { top = fmaxf(top, __shfl_xor_sync(kAllLanes, top, o)); }
    const float safe = finite_top(top);
    float sum        = 0.0f;
    for (uint32_t p = lane; p < n; p += 32) {
      const float2 st = parts.stats[size_t(part_at(p)) * parts.rows + r];
      sum             = fmaf(st.y, exp2f(st.x - safe), sum);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { sum += __shfl_xor_sync(kAllLanes, sum, o); }
    const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
    float x[2][E]     = {};
#pragma unroll 8
    for (uint32_t p = warp % SPLIT; p < n; p += SPLIT) {
      const uint32_t part = part_at(p);
      const float weight  = exp2f(parts.stats[size_t(part) * parts.rows + r].x - safe);
      const float4* a     = reinterpret_cast<const float4*>(parts.acc + (size_t(part) * parts.rows + r) * dim);
#pragma unroll
      for (int v = 0; v < 2; v++) {
        if ((lane + 32u * v) * E < dim) {
          const float4 y = a[lane + 32 * v];
          x[v][0]        = fmaf(weight, y.x, x[v][0]);
          x[v][1]        = fmaf(weight, y.y, x[v][1]);
          x[v][2]        = fmaf(weight, y.z, x[v][2]);
          x[v][3]        = fmaf(weight, y.w, x[v][3]);
        }
      }
    }
    if constexpr (SPLIT > 1) {
#pragma unroll
      for (int v = 0; v < 2; v++) {
#pragma unroll
        for (int e = 0; e < E; e++) { s_acc[warp][(lane + 32 * v) * E + e] = x[v][e]; }
      }
      __syncthreads();  // SPLIT is all of the block's warps: they take the same turns
      T* o = reinterpret_cast<T*>(result.out.data) + int64_t(sequence) * result.out.row + int64_t(head0 + r) * result.out.head;
      for (uint32_t d = threadIdx.x; d < dim; d += kJoinWarps * 32) {
        float y = 0.0f;
#pragma unroll
        for (int v = 0; v < kJoinWarps; v++) { y += s_acc[v][d]; }
        o[d] = from_float<T>(y * scale);
      }
      __syncthreads();
    } else {
      T* o = reinterpret_cast<T*>(result.out.data) + int64_t(sequence) * result.out.row + int64_t(head0 + r) * result.out.head;
#pragma unroll
      for (int v = 0; v < 2; v++) {
        const uint32_t d = (lane + 32u * v) * E;
        if (d < dim) {
          alignas(16) T y[E];
#pragma unroll
          for (int e = 0; e < E; e++) { y[e] = from_float<T>(x[v][e] * scale); }
          if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<uint2*>(o + d) = *reinterpret_cast<const uint2*>(y);
          } else {
            *reinterpret_cast<uint4*>(o + d) = *reinterpret_cast<const uint4*>(y);
          }
        }
      }
    }
    if (warp % SPLIT == 0 && lane == 0) { result.lse[size_t(sequence) * (w.group * n_heads) + head0 + r] = (safe + log2f(sum)) * kLn2; }
  }
}

// ---- copies into shared memory ------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t shared_address(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void copy_piece(uint32_t to, const void* from, bool there)
{
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait()
{
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A warp's way through its rows of a unit, ahead of the copies: what memory says about a row two tiles ahead, the word of the filter one tile
// ahead.  Lane i (modulo CHUNK) looks after row i of the warp's CHUNK rows of a tile.
template <int WARPS, int CHUNK, class Lists>
struct row_stream {
  const cache_view& c;
  const Lists& lists;
  const typename Lists::list& l;
  uint32_t base, tile_rows, tile1;
  int64_t name_0, name_1;
  uint32_t word_0;

  __device__ __forceinline__ row_stream(const cache_view& c_, const Lists& lists_, const typename Lists::list& l_, uint32_t warp, uint32_t tile0,
                                        uint32_t tile1_)
    : c(c_), lists(lists_), l(l_), base(warp * CHUNK + (threadIdx.x & 31u) % CHUNK), tile_rows(WARPS * CHUNK), tile1(tile1_)
  {
    name_0 = name(tile0);
    name_1 = name(tile0 + 1);
    word_0 = word(tile0, name_0);
  }
  __device__ __forceinline__ int64_t name(uint32_t tile) const { return tile < tile1 ? lists.name(c, l, base + tile * tile_rows) : -1; }
  __device__ __forceinline__ uint32_t word(uint32_t tile, int64_t name) const
  {
    if (c.filter == nullptr) { return 0u; }
    int64_t page;
    uint32_t place;
    return lists.place(c, l, base + tile * tile_rows, name, page, place) ? c.filter[(page * int64_t(c.page_size) + place) >> 5] : 0u;
  }
  // The place of this lane's row of `tile` (false: it is not to be read), and on to the next.
  __device__ __forceinline__ bool next(uint32_t tile, int64_t& page, uint32_t& place)
  {
    const int64_t name_2  = name(tile + 2);
    const uint32_t word_1 = word(tile + 1, name_1);
    bool there            = lists.place(c, l, base + tile * tile_rows, name_0, page, place);
    if (there && c.filter != nullptr) { there = ((word_0 >> (uint32_t(page * int64_t(c.page_size) + place) & 31u)) & 1u) != 0u; }
    name_0 = name_1;
    name_1 = name_2;
    word_0 = word_1;
    return there;
  }
};

// ---- host ---------------------------------------------------------------------------------------------------------------------

template <typename... Params, typename... Args>
void launch_units(resources& res, void (*kernel)(Params...), uint32_t blocks, uint32_t threads, uint32_t cluster, size_t smem,
                  Args&&... args)
{
  if (smem > 48 * 1024) { ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem); }
  cudaLaunchAttribute attrs[2]{};
  attrs[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id                                         = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x                           = std::max(cluster, 1u);
  attrs[1].val.clusterDim.y                           = 1;
  attrs[1].val.clusterDim.z                           = 1;
  cudaLaunchConfig_t config{};
  config.gridDim          = blocks;
  config.blockDim         = threads;
  config.dynamicSmemBytes = smem;
  config.stream           = res.stream;
  config.attrs            = attrs;
  config.numAttrs         = cluster > 1 ? 2 : 1;
  CUDA_TRY(cudaLaunchKernelEx(&config, kernel, std::forward<Args>(args)...));
  res.launches++;
}

// What a call launches, by type and sizes alone.
struct plan {
  uint32_t rows;      // query heads of a unit
  uint32_t chunk;     // rows of the cache that a warp takes of a tile
  uint32_t resident;  // small blocks of an SM
  uint32_t warps;     // of a block
  uint32_t blocks;
  uint32_t cluster;   // 0: shares
  bool join;          // a unit may lie in several shares
};

// `most`: rows of a unit, at most; `large`: whether there are large blocks; `shares`: whether there may be shares.
inline void deal_out(const resources& res, plan& p, uint64_t units, uint64_t most, bool large, bool shares)
{
  const uint64_t sms = uint64_t(res.sm_count), resident = sms * p.resident;
  p.join = false;
  if (units <= sms) {
    p.warps              = large ? kLarge : kSmall;
    const uint64_t tiles = ceildiv<uint64_t>(most, p.warps * p.chunk);
    uint32_t cluster     = 1;
    while (cluster < 8 && 2 * cluster * units <= sms && cluster < tiles) { cluster *= 2; }
    if (!shares || ceildiv<uint64_t>(tiles, cluster) <= 4) {
      p.blocks  = uint32_t(units * cluster);
      p.cluster = cluster;
      return;
    }
  }
  const uint64_t tiles = std::max<uint64_t>(1, ceildiv<uint64_t>(most, kSmall * p.chunk));
  p.warps              = kSmall;
  if (!shares) {
    p.blocks  = uint32_t(units);
    p.cluster = 1;
  } else {
    p.blocks  = uint32_t(std::min(resident, units * tiles));
    p.cluster = 0;
    p.join    = tiles > 1 && p.blocks > 1;
  }
}

template <typename T>
void launch_join(resources& res, const plan& p, const work_view& w, const parts_view& parts, uint32_t dim, uint32_t n_heads,
                 const result_view& result)
{
  // Few units have many parts each: a block per row and all of its warps on the row's parts; else a warp per row.
  const uint64_t units = uint64_t(w.n_units) * w.n_sequences;
  if (p.blocks / units >= 16) {
    launch_chained(join_kernel<T, kJoinWarps>, dim3(p.blocks - 1, std::min(p.rows, w.group)), kJoinWarps * 32, 0, res.stream, w, parts, dim,
                   n_heads, result);
  } else {
    launch_chained(join_kernel<T, 1>, dim3(p.blocks - 1, 1), kJoinWarps * 32, 0, res.stream, w, parts, dim, n_heads, result);
  }
  res.launches++;
}

}  // namespace cuvs_b200::kv
