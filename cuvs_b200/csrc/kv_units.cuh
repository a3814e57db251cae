// Who does what when query heads attend to lists of rows: units, chunks, shares, clusters, and the joining of what several have of a unit.
//
// A unit is a (sequence, key head, block of query heads) with its list of rows, cut into chunks of as many rows as a warp takes at a time.
// Two ways to deal the chunks out:
//
// Shares.  All units' chunks stand in one row, and each of the resident blocks takes an equal, contiguous share of it, whatever the lengths
// are (they are known on the device alone: every warp finds its block's share from them itself).  What a unit costs beside its rows counts too.
// A block's warps take a unit's chunks in turn, copy the first rows of the next unit while they finish this one, and join through shared
// memory at its end.  A unit that lies in one share is finished there; of a unit that several share, each block leaves a part (top, sum and
// weighted sum in 32 bits), and a second kernel joins the parts in the order of the shares.
//   What else was tried: warps with shares of their own, which need no barrier but leave four times the parts (32 requests of up to 16,384 tokens
// 170 us against 148, 256 of up to 1,024 87 against 80); parts joined in a tree by whichever block came last, without the second kernel (12 us at
// the end of one long list); shares that get smaller in rounds, taken by whoever is done (four ends of pieces instead of one: 118 us
// against 94 on one list of 250,000); shares of equal chunks whatever the units cost (16 requests of up to 2,000 tokens 32 us, 16 now).
//
// Clusters.  One cluster of blocks per unit, whose warps take its chunks in turn and join their parts through shared memory, their own and
// each other's: no workspace, one launch and the shortest way to the end, but no balance between units: for few units with few rows.
//
// Nothing depends on the order in which blocks run.
#pragma once

#include "kv_plan.hpp"
#include "kv_rows.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

namespace cuvs_b200::kv {

struct work_view {
  uint32_t n_sequences;
  uint32_t n_units;      // per sequence: key heads x blocks of query heads
  uint32_t n_blocks_of;  // blocks of query heads of one key head
  uint32_t group;        // query heads of one key head
  uint32_t cluster;      // blocks of a unit's cluster; 0: shares
  uint32_t cost;         // of a unit beside its rows (queries, joining, writing), in chunks: what it counts for where shares are dealt out
  // Weights are held times `room`, a power of two that keeps the sum of a whole list below 1: weighted sums, which are divided by it at their end,
  // stay below the largest value then, and finite where the answer is (times 1, 1,500 rows of 3e38 gave infinity).  What that costs is at the
  // other end of the range: values below 1e-25 in lists of 2^17 rows lose digits.  `back` = 1 / room.
  float room, back;
};

// For lists of `rows` at most.
inline void make_room(work_view& w, uint64_t rows)
{
  int bits = 1;
  while (bits < 32 && (uint64_t(1) << (bits - 1)) < rows) { bits++; }
  w.room = std::ldexp(1.0f, -bits);
  w.back = std::ldexp(1.0f, bits);
}

// ---- lists --------------------------------------------------------------------------------------------------------------------

// All positions of a sequence, or its last ones.  A list begins at a multiple of 16 positions, so that 16 rows lie in one page where pages
// are multiples of 16.
struct positions {
  static constexpr bool kShares    = true;
  static constexpr uint32_t kLeast = kLeastShare;  // chunks of a share, at least: one for each warp of a block
  using name_type               = int32_t;
  const int32_t* pages;
  const int32_t* lengths;
  int64_t table_stride;
  int64_t window;
  uint32_t width;

  struct list {
    const int32_t* table;
    uint32_t first, end, base;
  };
  __device__ __forceinline__ uint32_t open(const cache_view& c, uint32_t sequence, uint32_t chunk, list& l) const
  {
    attended(lengths[sequence], window, width, c.page.size, l.first, l.end);
    l.table = pages + int64_t(sequence) * table_stride;
    l.base  = l.first & ~15u;
    return l.end > l.first ? (l.end - l.base + chunk - 1) / chunk : 0u;
  }
  __device__ __forceinline__ void select(const cache_view&, const work_view&, uint32_t, uint32_t, list&) const {}
  // What memory says about row i of the list (-1: it is none); to be looked at later, when it has arrived.
  __device__ __forceinline__ int32_t name(const cache_view& c, const list& l, uint32_t i) const
  {
    const uint32_t at = l.base + i;
    if (at < l.first || at >= l.end) { return -1; }
    uint32_t column, place;
    split_place(at, c.page, column, place);
    return l.table[column];  // at < end: the column is inside the table
  }
  // Its page and place in it; false: it has none.
  __device__ __forceinline__ bool place(const cache_view& c, const list& l, uint32_t i, int32_t name, uint32_t& page, uint32_t& place) const
  {
    uint32_t column;
    split_place(l.base + i, c.page, column, place);
    page = uint32_t(name);
    return name >= 0 && name < c.n_pages;
  }
};

// Slots that are named one by one, n for each query head of a token.
struct named_slots {
  static constexpr bool kShares = false;  // lists are equally long
  using name_type               = int64_t;
  const int64_t* ids;
  uint32_t n;

  struct list {
    const int64_t* ids;
  };
  __device__ __forceinline__ uint32_t open(const cache_view&, uint32_t, uint32_t chunk, list&) const { return (n + chunk - 1) / chunk; }
  __device__ __forceinline__ void select(const cache_view&, const work_view& w, uint32_t token, uint32_t unit, list& l) const
  {
    l.ids = ids + (int64_t(token) * w.n_units + unit) * n;
  }
  __device__ __forceinline__ int64_t name(const cache_view&, const list& l, uint32_t i) const { return i < n ? l.ids[i] : -1; }
  __device__ __forceinline__ bool place(const cache_view& c, const list&, uint32_t, int64_t name, uint32_t& page, uint32_t& place) const
  {
    const bool there = name >= 0 && name < c.n_slots;
    split_slot(c, there ? name : 0, page, place);
    return there;
  }
};

// ---- shares -------------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint64_t quotient(uint64_t a, uint32_t b)
{
  return a >> 32 == 0 ? uint64_t(uint32_t(a) / b) : a / b;  // the short division where it is enough
}

// `total` chunks of all units dealt out in `count` equal shares: one for every block, or fewer of `least` chunks each.
struct share {
  uint64_t total, each;
  uint32_t count, longer;  // the first `longer` get `each` + 1, the others `each`
  __device__ __forceinline__ share(uint64_t total_, uint32_t most, uint32_t least)
    : total(total_), each(0), count(uint32_t(min(uint64_t(most), ceildiv<uint64_t>(total_, least)))), longer(0)
  {
    if (count != 0u) {
      each   = quotient(total, count);
      longer = uint32_t(total - each * count);
    }
  }
  __device__ __forceinline__ uint64_t start(uint32_t i) const { return i * each + min(i, longer); }
  __device__ __forceinline__ uint32_t of(uint64_t chunk) const  // the share that has it
  {
    const uint64_t middle = longer * (each + 1);
    return chunk < middle ? uint32_t(quotient(chunk, uint32_t(each + 1))) : longer + uint32_t(quotient(chunk - middle, uint32_t(each)));
  }
};

// The sequences that a lane looks at: kAtOnce neighbours of every 32 * kAtOnce, their lengths asked for together.
constexpr uint32_t kAtOnce = 4;
template <int CHUNK, class Lists>
__device__ __forceinline__ uint64_t chunks_at(const cache_view& c, const work_view& w, const Lists& lists, uint32_t first, uint32_t (&n)[kAtOnce])
{
  uint64_t sum = 0;
#pragma unroll
  for (uint32_t i = 0; i < kAtOnce; i++) {
    typename Lists::list l;
    n[i] = first + i < w.n_sequences ? lists.open(c, first + i, CHUNK, l) : 0u;
    if (n[i] != 0u) { n[i] += w.cost; }
    sum += n[i];
  }
  return sum;
}

// The number of all chunks, with the units' costs, which come before their chunks; every warp sums it up for itself.
template <int CHUNK, class Lists>
__device__ __forceinline__ uint64_t all_chunks(const cache_view& c, const work_view& w, const Lists& lists)
{
  uint64_t sum = 0;
  uint32_t n[kAtOnce];
  for (uint32_t b = (threadIdx.x & 31u) * kAtOnce; b < w.n_sequences; b += 32 * kAtOnce) { sum += chunks_at<CHUNK>(c, w, lists, b, n); }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { sum += __shfl_xor_sync(kAllLanes, sum, o); }
  return sum * w.n_units;
}

// The sequence that chunk `at` of all belongs to, and the number of chunks before that sequence.
template <int CHUNK, class Lists>
__device__ __forceinline__ uint32_t sequence_of(const cache_view& c, const work_view& w, const Lists& lists, uint64_t at, uint64_t& before)
{
  const uint32_t lane = threadIdx.x & 31u;
  before              = 0;
  for (uint32_t b0 = 0; b0 < w.n_sequences; b0 += 32 * kAtOnce) {  // comes to an end inside: `at` is less than the number of all chunks
    uint32_t n[kAtOnce];
    const uint64_t mine = chunks_at<CHUNK>(c, w, lists, b0 + lane * kAtOnce, n) * w.n_units;
    uint64_t up         = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t t = __shfl_up_sync(kAllLanes, up, o);
      if (lane >= uint32_t(o)) { up += t; }
    }
    const unsigned past = __ballot_sync(kAllLanes, before + up > at);
    if (past != 0u) {
      const int found   = __ffs(int(past)) - 1;
      uint32_t sequence = b0 + found * kAtOnce;
      before += __shfl_sync(kAllLanes, up - mine, found);
#pragma unroll
      for (uint32_t i = 0; i + 1 < kAtOnce; i++) {
        const uint64_t here = uint64_t(__shfl_sync(kAllLanes, n[i], found)) * w.n_units;
        if (sequence == b0 + found * kAtOnce + i && before + here <= at) {
          before += here;
          sequence++;
        }
      }
      return sequence;
    }
    before += __shfl_sync(kAllLanes, up, 31);
  }
  return w.n_sequences;
}

// ---- parts --------------------------------------------------------------------------------------------------------------------

// Two parts per share: 0 of a unit that a share before began, 1 of a unit that this share begins and a later one goes on with.
struct parts_view {
  float* acc;     // [2 shares][rows][dim]
  float2* stats;  // [2 shares][rows] top (of scores in powers of two), sum
  uint4* begun;   // [shares] the unit that share i begins and does not end: sequence, unit, how many parts it has (0: there is none)
  uint32_t shares;
  uint32_t rows;  // query heads of a unit, at most
};

inline size_t part_bytes(uint32_t shares, uint32_t rows, uint32_t dim)
{
  return size_t(shares) * (sizeof(uint4) + 2 * rows * (dim * sizeof(float) + sizeof(float2)));
}
inline parts_view parts_at(char* workspace, uint32_t shares, uint32_t rows, uint32_t dim)
{
  parts_view p;
  p.begun  = reinterpret_cast<uint4*>(workspace);
  p.acc    = reinterpret_cast<float*>(p.begun + shares);
  p.stats  = reinterpret_cast<float2*>(p.acc + size_t(2) * shares * rows * dim);
  p.shares = shares;
  p.rows   = rows;
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

// Joins the warps: the block's sums become output rows, or warp 0's sums (for the cluster).
template <typename T, int WARPS>
__device__ __forceinline__ void join_warps(const cache_view& c, const work_view& w, const block_state& s, uint32_t rows, uint32_t sequence,
                                           uint32_t head0, const result_view& result, bool clustered, const parts_view& parts)
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
      const float f   = power_of_2(st.x - safe);
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
    if (!clustered) {
      const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
      for (uint32_t e = 0; e < E; e++) { x[e] *= scale; }
      store_piece<T>(result.out, sequence, head0 + r, piece, x);
      if (piece == 0) { result.lse[size_t(sequence) * (w.group * c.n_heads) + head0 + r] = (safe + log2f(sum * w.back)) * kLn2; }
    } else {
      float4* a = reinterpret_cast<float4*>(s.acc + size_t(r) * s.acc_row + piece * E);
#pragma unroll
      for (uint32_t e = 0; e < E; e += 4) { a[e / 4] = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]); }
      if (piece == 0) { s.joined[r] = make_float2(top, sum); }
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
      const float f   = power_of_2(st.x - safe);
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
    if (piece == 0) { result.lse[size_t(sequence) * (w.group * c.n_heads) + head0 + r] = (safe + log2f(sum * w.back)) * kLn2; }
  }
  cluster.sync();  // no block leaves while others read its shared memory
}

// Rows of sequences that attend to nothing: they have no chunks in any share.
template <typename T, int WARPS, int CHUNK, class Lists>
__device__ __forceinline__ void empty_rows(const cache_view& c, const work_view& w, const Lists& lists, const result_view& result)
{
  constexpr uint32_t E   = kPerPiece<T>;
  const uint32_t heads   = w.group * c.n_heads;
  const float nothing[8] = {};
  for (uint32_t b = blockIdx.x; b < w.n_sequences; b += gridDim.x) {
    typename Lists::list l;
    if (lists.open(c, b, CHUNK, l) != 0u) { continue; }
    for (uint32_t i = threadIdx.x; i < heads * (c.dim / E); i += WARPS * 32) {
      store_piece<T>(result.out, b, i / (c.dim / E), i % (c.dim / E), nothing);
    }
    for (uint32_t i = threadIdx.x; i < heads; i += WARPS * 32) { result.lse[size_t(b) * heads + i] = -INFINITY; }
  }
}

// ---- joining parts ------------------------------------------------------------------------------------------------------------

constexpr int kJoinWarps = 16, kJoinAlone = 16;

// A row of a unit with n parts, of which this warp takes every `step`-th from `from` on: their top and sum, and the weighted sum in columns
// 4 * lane and 128 + 4 * lane on.
__device__ __forceinline__ void join_some(const parts_view& parts, uint32_t share, uint32_t n, uint32_t r, uint32_t dim, uint32_t from, uint32_t step,
                                          float& top, float& sum, float (&x)[2][4])
{
  const uint32_t lane = threadIdx.x & 31u;
  auto place          = [&](uint32_t p) { return size_t(p == 0 ? 2 * share + 1 : 2 * (share + p)) * parts.rows + r; };
  top                 = -INFINITY;
  sum                 = 0.0f;
#pragma unroll
  for (int v = 0; v < 2; v++) { x[v][0] = x[v][1] = x[v][2] = x[v][3] = 0.0f; }
  for (uint32_t p0 = from; p0 < n; p0 += 8 * step) {
    float2 st[8];
    uint4 y[2][8];
#pragma unroll
    for (uint32_t i = 0; i < 8; i++) {
      const uint32_t p = p0 + i * step;
      const bool there = p < n;
      const size_t at  = place(there ? p : 0u);
      st[i]            = there ? parts.stats[at] : make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int v = 0; v < 2; v++) {
        const uint32_t column = 4 * lane + 128u * v;
        y[v][i]               = load_piece(parts.acc + at * dim + column, there && column < dim);
      }
    }
    float next = top;
#pragma unroll
    for (uint32_t i = 0; i < 8; i++) { next = fmaxf(next, st[i].x); }
    const float safe = finite_top(next), keep = power_of_2(top - safe);
    top = next;
    sum *= keep;
#pragma unroll
    for (int v = 0; v < 2; v++) {
#pragma unroll
      for (int e = 0; e < 4; e++) { x[v][e] *= keep; }
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; i++) {
      const float f = power_of_2(st[i].x - safe);
      sum           = fmaf(st[i].y, f, sum);
#pragma unroll
      for (int v = 0; v < 2; v++) {
        x[v][0] = fmaf(__uint_as_float(y[v][i].x), f, x[v][0]);
        x[v][1] = fmaf(__uint_as_float(y[v][i].y), f, x[v][1]);
        x[v][2] = fmaf(__uint_as_float(y[v][i].z), f, x[v][2]);
        x[v][3] = fmaf(__uint_as_float(y[v][i].w), f, x[v][3]);
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ void write_joined(const work_view& w, const result_view& result, uint32_t sequence, uint32_t head, uint32_t heads,
                                             uint32_t dim, float top, float sum, const float (&x)[2][4])
{
  const uint32_t lane = threadIdx.x & 31u;
  const float scale   = sum == 0.0f ? 0.0f : 1.0f / sum;
  T* o                = reinterpret_cast<T*>(result.out.data) + int64_t(sequence) * result.out.row + int64_t(head) * result.out.head;
#pragma unroll
  for (int v = 0; v < 2; v++) {
    const uint32_t column = 4 * lane + 128u * v;
    if (column >= dim) { continue; }
    alignas(16) T z[4];
#pragma unroll
    for (int e = 0; e < 4; e++) { z[e] = from_float<T>(x[v][e] * scale); }
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint2*>(o + column) = *reinterpret_cast<const uint2*>(z);
    } else {
      *reinterpret_cast<uint4*>(o + column) = *reinterpret_cast<const uint4*>(z);
    }
  }
  if (lane == 0) { result.lse[size_t(sequence) * heads + head] = (finite_top(top) + log2f(sum * w.back)) * kLn2; }
}

// Every warp looks at its (share, row) pairs: rows of a few parts are joined by the warp alone, those of many by the block's warps together.
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32)
join_kernel(work_view w, parts_view parts, uint32_t dim, uint32_t n_heads, result_view result)
{
  chain_begin();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, heads = w.group * n_heads;
  __shared__ uint32_t s_many[kJoinWarps], s_n;
  __shared__ float4 s_x[kJoinWarps][64];
  __shared__ float2 s_stats[kJoinWarps];
  // neighbouring warps have different shares: the rows of a unit with many parts are those of different blocks
  const uint32_t pairs = parts.shares * parts.rows, stride = gridDim.x * kJoinWarps;
  auto row_of = [&](uint32_t pair, uint32_t& share, uint32_t& r, uint4& unit, uint32_t& head) -> bool {
    r                = pair / parts.shares;
    share            = pair - r * parts.shares;
    unit             = parts.begun[share];
    const uint32_t h = unit.y / w.n_blocks_of, of = unit.y - h * w.n_blocks_of;
    head             = h * w.group + of * parts.rows + r;
    return unit.z != 0u && of * parts.rows + r < w.group;
  };
  float top, sum, x[2][4];
  for (uint32_t base = blockIdx.x * kJoinWarps; base < pairs; base += stride) {
    if (threadIdx.x == 0) { s_n = 0u; }
    __syncthreads();
    uint32_t share, r, head;
    uint4 unit;
    if (base + warp < pairs && row_of(base + warp, share, r, unit, head)) {
      if (unit.z <= uint32_t(kJoinAlone)) {
        join_some(parts, share, unit.z, r, dim, 0u, 1u, top, sum, x);
        write_joined<T>(w, result, unit.x, head, heads, dim, top, sum, x);
      } else if (lane == 0) {
        s_many[atomicAdd(&s_n, 1u)] = base + warp;
      }
    }
    __syncthreads();
    const uint32_t many = s_n;
    for (uint32_t i = 0; i < many; i++) {
      row_of(s_many[i], share, r, unit, head);
      join_some(parts, share, unit.z, r, dim, warp, kJoinWarps, top, sum, x);
      s_x[warp][lane]      = make_float4(x[0][0], x[0][1], x[0][2], x[0][3]);
      s_x[warp][lane + 32] = make_float4(x[1][0], x[1][1], x[1][2], x[1][3]);
      if (lane == 0) { s_stats[warp] = make_float2(top, sum); }
      __syncthreads();
      if (warp == 0) {
        top = -INFINITY;
#pragma unroll
        for (int v = 0; v < kJoinWarps; v++) { top = fmaxf(top, s_stats[v].x); }
        const float safe = finite_top(top);
        sum              = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++) { x[0][e] = x[1][e] = 0.0f; }
#pragma unroll
        for (int v = 0; v < kJoinWarps; v++) {
          const float f = power_of_2(s_stats[v].x - safe);
          sum           = fmaf(s_stats[v].y, f, sum);
#pragma unroll
          for (int u = 0; u < 2; u++) {
            const float4 y = s_x[v][lane + 32 * u];
            x[u][0]        = fmaf(y.x, f, x[u][0]);
            x[u][1]        = fmaf(y.y, f, x[u][1]);
            x[u][2]        = fmaf(y.z, f, x[u][2]);
            x[u][3]        = fmaf(y.w, f, x[u][3]);
          }
        }
        write_joined<T>(w, result, unit.x, head, heads, dim, top, sum, x);
      }
      __syncthreads();
    }
  }
}

// ---- pieces -------------------------------------------------------------------------------------------------------------------

// What a share has of one unit: its chunks [chunk, end), which may be all of it.
struct piece {
  uint32_t sequence, unit, chunk, end;
  uint32_t n_parts;  // of a unit that the piece begins and does not end
  bool begins, whole;
};

// A block's way through its share, piece by piece; all its warps go it.
template <int CHUNK, class Lists>
struct walk {
  const cache_view& c;
  const work_view& w;
  const Lists& lists;
  typename Lists::list l;  // of the sequence that the walk is at
  share all;
  uint64_t at, stop, before;
  uint32_t sequence, n, which;  // `which`: the share

  __device__ __forceinline__ walk(const cache_view& c_, const work_view& w_, const Lists& lists_, uint32_t most, uint32_t which_)
    : c(c_), w(w_), lists(lists_), all(all_chunks<CHUNK>(c_, w_, lists_), most, Lists::kLeast), at(0), stop(0), before(0), sequence(0), n(0), which(which_)
  {
    if (which >= all.count) { return; }
    at       = all.start(which);
    stop     = all.start(which + 1);
    sequence = sequence_of<CHUNK>(c, w, lists, at, before);
    if (sequence < w.n_sequences) {
      open();
    } else {  // lengths that changed meanwhile
      at = stop;
    }
  }
  __device__ __forceinline__ void open()
  {
    n = lists.open(c, sequence, CHUNK, l);
    if (n != 0u) { n += w.cost; }
  }
  __device__ __forceinline__ bool next(piece& p)
  {
    while (at < stop) {
      while (at >= before + uint64_t(n) * w.n_units) {  // on to the next sequence that has chunks
        before += uint64_t(n) * w.n_units;
        if (++sequence >= w.n_sequences) {
          at = stop;
          return false;
        }
        open();
      }
      p.unit              = uint32_t(quotient(at - before, n));
      const uint64_t unit = before + uint64_t(p.unit) * n, begin = unit + w.cost, end = unit + n, from = max(at, begin), to = min(stop, end);
      at                  = to;
      if (from >= to) { continue; }  // of the unit's cost alone
      p.sequence = sequence;
      p.chunk    = uint32_t(from - begin);
      p.end      = uint32_t(to - begin);
      p.begins   = from == begin;
      p.whole    = p.begins && to == end;
      if (p.begins && !p.whole) { p.n_parts = min(all.of(end - 1), all.count - 1u) - which + 1u; }
      return true;
    }
    return false;
  }
};

// ---- copies into shared memory ------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t shared_address(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

// `bytes`: 16, or 0: then nothing is read, and zeros are written.
__device__ __forceinline__ void copy_piece(uint32_t to, const void* from, uint32_t bytes)
{
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait()
{
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A warp's way through its chunks of a piece, ahead of the copies: what memory says about a row two chunks ahead, the word of the filter one
// chunk ahead.  Lane i (modulo CHUNK) looks after row i of a chunk.
template <int CHUNK, class Lists>
struct row_stream {
  using name_type = typename Lists::name_type;
  const cache_view& c;
  const Lists& lists;
  typename Lists::list l;
  uint32_t chunk, end, step;  // the next chunk to copy, the piece's end
  name_type name_0, name_1;
  uint32_t word_0;

  __device__ __forceinline__ row_stream(const cache_view& c_, const Lists& lists_) : c(c_), lists(lists_), chunk(0), end(0), step(1) {}
  __device__ __forceinline__ void attach(const typename Lists::list& l_, uint32_t chunk_, uint32_t end_, uint32_t step_)
  {
    l      = l_;
    chunk  = chunk_;
    end    = end_;
    step   = step_;
    name_0 = name(chunk);
    name_1 = name(chunk + step);
    word_0 = word(chunk, name_0);
  }
  __device__ __forceinline__ bool done() const { return chunk >= end; }
  __device__ __forceinline__ uint32_t row(uint32_t at) const { return at * CHUNK + (threadIdx.x & 31u) % CHUNK; }
  __device__ __forceinline__ name_type name(uint32_t at) const { return at < end ? lists.name(c, l, row(at)) : name_type(-1); }
  __device__ __forceinline__ uint32_t word(uint32_t at, name_type name) const
  {
    if (c.filter == nullptr) { return 0u; }
    uint32_t page, place;
    return lists.place(c, l, row(at), name, page, place) ? c.filter[(uint64_t(page) * c.page.size + place) >> 5] : 0u;
  }
  // The place of this lane's row of the next chunk (false: it is not to be read), and on to the one after.
  __device__ __forceinline__ bool next(uint32_t& page, uint32_t& place)
  {
    const name_type name_2 = name(chunk + 2 * step);
    const uint32_t word_1  = word(chunk + step, name_1);
    bool there             = lists.place(c, l, row(chunk), name_0, page, place);
    if (c.filter != nullptr) { there = there && ((word_0 >> ((page * c.page.size + place) & 31u)) & 1u) != 0u; }
    name_0 = name_1;
    name_1 = name_2;
    word_0 = word_1;
    chunk += step;
    return there;
  }
};

// ---- the way of a block -------------------------------------------------------------------------------------------------------

constexpr uint32_t kEmpty = 0xFFFFFFFFu;  // in the place of a stage's mask: no chunk of any piece is there

// Goes through everything the block has to do.  A warp's stages are filled a few chunks ahead, over the ends of pieces: the first chunks of the
// next one come while the last ones of this are worked on and its sums are written.  `hooks`:
//   attach(unit)                       where the rows to be copied next lie
//   copy(stage, page, place, there)    copies of a chunk's rows; returns which of them are read
//   start(sequence, unit)              queries; sums to zero
//   consume(stage, mask)               the rows of a stage
//   close()                            a warp's lanes have the warp's sums
//   send(i, to), receive(i, from)      a warp's sums to another, the i-th of kPortions portions of kPortion floats
//   to_rows(...)                       the warp's sums become output rows, or a part
//   to_shared()                        the warp's sums into the block's state
// `s_mask`: the warp's [STAGES]; `exchange`: room for half the warps' portions; the block's state may lie where the stages are.
template <typename T, int WARPS, int CHUNK, int STAGES, class Lists, class Hooks>
__device__ __forceinline__ void run_units(const cache_view& c, const work_view& w, const Lists& lists, const result_view& result,
                                          const parts_view& parts, const block_state& state, float* exchange, uint32_t* s_mask, Hooks& hooks)
{
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  uint32_t filling = 0, emptying = 0;  // stages
  row_stream<CHUNK, Lists> stream(c, lists);
  auto fill = [&] {  // the next stage, with a chunk if the stream has one
    uint32_t mask = kEmpty;
    if (!stream.done()) {
      uint32_t page, place;
      const bool there = stream.next(page, place);
      mask             = hooks.copy(filling, page, place, there);
    }
    if (lane == 0) { s_mask[filling] = mask; }
    copies_end_group();
    filling = filling + 1 == STAGES ? 0 : filling + 1;
  };
  auto heads_of = [&](uint32_t unit, uint32_t& rows, uint32_t& head0) {
    const uint32_t head = unit / w.n_blocks_of, of = unit - head * w.n_blocks_of;
    rows  = min(parts.rows, w.group - of * parts.rows);
    head0 = head * w.group + of * parts.rows;
  };
  uint32_t rows, head0;

  if (!Lists::kShares || w.cluster != 0u) {
    typename Lists::list l;
    const uint32_t which = blockIdx.x / w.cluster, rank = blockIdx.x - which * w.cluster;
    const uint32_t sequence = which / w.n_units, unit = which - sequence * w.n_units;
    const uint32_t n = lists.open(c, sequence, CHUNK, l);
    lists.select(c, w, sequence, unit, l);
    hooks.attach(unit);
    stream.attach(l, uint32_t(uint64_t(rank) * n / w.cluster) + warp, uint32_t(uint64_t(rank + 1) * n / w.cluster), WARPS);
    hooks.start(sequence, unit);
#pragma unroll 1
    for (int i = 0; i < STAGES; i++) { fill(); }
    while (true) {
      copies_wait<STAGES - 1>();
      __syncwarp();
      const uint32_t mask = s_mask[emptying];
      if (mask == kEmpty) { break; }
      if (mask != 0u) { hooks.consume(emptying, mask); }
      __syncwarp();
      emptying = emptying + 1 == STAGES ? 0 : emptying + 1;
      fill();
    }
    copies_wait<0>();
    hooks.close();
    heads_of(unit, rows, head0);
    __syncthreads();  // shared memory changes hands: from rows to sums
    hooks.to_shared();
    __syncthreads();
    join_warps<T, WARPS>(c, w, state, rows, sequence, head0, result, w.cluster > 1u, parts);
    if (w.cluster > 1u) { join_cluster<T, WARPS>(c, w, state, rows, sequence, head0, result); }
    return;
  }

  if constexpr (Lists::kShares) {
    walk<CHUNK, Lists> path(c, w, lists, parts.shares, blockIdx.x);
    piece now, then;
    auto turn_to = [&](const piece& p) {
      hooks.attach(p.unit);
      stream.attach(path.l, p.chunk + warp, p.end, WARPS);
    };
    bool found = __syncthreads_and(path.next(now)) != 0, more = false;
    uint4 begun = make_uint4(0, 0, 0, 0);
    if (found) { turn_to(now); }
    // `more`: the piece behind this one, once the stream has come to it
    bool looked  = false;
    auto fill_on = [&] {
      if (stream.done() && !looked) {
        looked = true;
        more   = path.next(then);
        if (more) { turn_to(then); }
      }
      fill();
    };
    if (found) {
#pragma unroll 1
      for (int i = 0; i < STAGES; i++) { fill_on(); }
    }
    while (found) {
      hooks.start(now.sequence, now.unit);
      uint32_t left = now.end > now.chunk + warp ? ceildiv<uint32_t>(now.end - now.chunk - warp, WARPS) : 0u;
      while (left != 0u) {
        copies_wait<STAGES - 1>();
        __syncwarp();
        const uint32_t mask = s_mask[emptying];
        if (mask != kEmpty) {  // (a stage may be empty where a piece was shorter than the stages are many)
          left--;
          if (mask != 0u) { hooks.consume(emptying, mask); }
        }
        __syncwarp();
        emptying = emptying + 1 == STAGES ? 0 : emptying + 1;
        fill_on();
      }
      hooks.close();
      heads_of(now.unit, rows, head0);
      if (!looked) {
        more = path.next(then);
        if (more) { turn_to(then); }
      }
      // the upper half of the warps to the lower, until the first has all
#pragma unroll
      for (int half = WARPS / 2; half > 0; half /= 2) {
#pragma unroll
        for (int i = 0; i < Hooks::kPortions; i++) {
          if (int(warp) >= half && int(warp) < 2 * half) { hooks.send(i, exchange + (warp - half) * Hooks::kPortion); }
          __syncthreads();
          if (int(warp) < half) { hooks.receive(i, exchange + warp * Hooks::kPortion); }
          if (half > 1 || i + 1 < Hooks::kPortions) { __syncthreads(); }
        }
      }
      // The warps found this out each for itself.  They go on together, or none does: lengths that somebody changes while the kernel runs must not
      // leave one of them waiting for the others.
      found = __syncthreads_and(more) != 0;
      if (warp == 0) { hooks.to_rows(rows, now.sequence, head0, now.whole, 2 * blockIdx.x + (now.begins ? 1u : 0u)); }
      if (now.begins && !now.whole) { begun = make_uint4(now.sequence, now.unit, now.n_parts, 0); }
      now    = then;
      looked = false;
      more   = false;
    }
    copies_wait<0>();
    if (parts.begun != nullptr && threadIdx.x == 0) { parts.begun[blockIdx.x] = begun; }
    empty_rows<T, WARPS, CHUNK>(c, w, lists, result);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

template <typename... Params, typename... Args>
void launch_units(cudaStream_t stream, void (*kernel)(Params...), uint32_t blocks, uint32_t threads, uint32_t cluster, size_t smem, Args&&... args)
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
  config.stream           = stream;
  config.attrs            = attrs;
  config.numAttrs         = cluster > 1 ? 2 : 1;
  CUDA_TRY(cudaLaunchKernelEx(&config, kernel, std::forward<Args>(args)...));
}

template <typename T>
void launch_join(const resources& res, cudaStream_t stream, const plan& p, const work_view& w, const parts_view& parts, uint32_t dim,
                 uint32_t n_heads, const result_view& result)
{
  const uint32_t blocks = std::min<uint32_t>(ceildiv<uint32_t>(parts.shares * parts.rows, kJoinWarps), uint32_t(res.sm_count) * 4);
  launch_chained(join_kernel<T>, dim3(blocks), kJoinWarps * 32, 0, stream, w, parts, dim, n_heads, result);
}

}  // namespace cuvs_b200::kv
