// Who does what when query heads attend to lists of rows: units, chunks, shares, clusters, and the joining of what several have of a unit.
//
// A unit is a (sequence, key head, block of query heads) with its list of rows, cut into chunks of as many rows as a warp takes at a time.
// Two ways to deal the chunks out:
//
// Shares.  All units' chunks stand in one row, and each of a fixed number of teams -- the resident blocks, or their warps -- takes an equal,
// contiguous share of it, whatever the lengths are (they are known on the device alone: every warp finds its share from them itself).  A
// unit that lies in one share is finished there; of a unit that several share, each team leaves a part (top, sum and weighted sum in 32
// bits).  Parts are joined in a tree, eight neighbours at a time, by whichever of the eight comes last; the order of the sums does not
// depend on who that is.  Warps as teams need no barrier and never wait for one another between units: for many units.  Blocks as teams
// leave a quarter of the parts: for few and long ones.
//
// Clusters.  One cluster of blocks per unit, whose blocks take equal runs of its chunks and join their parts through each other's shared
// memory: no workspace and the shortest way to the end, but no balance between units: for few units with few rows.
#pragma once

#include "kv_rows.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace cuvs_b200::kv {

// Warps of a block: small blocks, several to an SM, balance best; where units are fewer than SMs, one large block has an SM's warps for one
// unit.
constexpr int kSmall     = 4;
constexpr int kMostTeams = 24;  // warps of an SM, at most, where they are teams

struct work_view {
  uint32_t n_sequences;
  uint32_t n_units;      // per sequence: key heads x blocks of query heads
  uint32_t n_blocks_of;  // blocks of query heads of one key head
  uint32_t group;        // query heads of one key head
  uint32_t cluster;      // blocks of a unit's cluster; 0: shares
  bool warp_teams;       // of shares: warps, else blocks
};

// ---- lists --------------------------------------------------------------------------------------------------------------------

// All positions of a sequence, or its last ones.  A list begins at a multiple of 16 positions, so that 16 rows lie in one page where pages
// are multiples of 16.
struct positions {
  static constexpr bool kShares = true;
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
    attended(lengths[sequence], window, width, c.page_size, l.first, l.end);
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
    split_place(at, c.page_size, c.page_shift, column, place);
    return l.table[column];  // at < end: the column is inside the table
  }
  // Its page and place in it; false: it has none.
  __device__ __forceinline__ bool place(const cache_view& c, const list& l, uint32_t i, int32_t name, uint32_t& page, uint32_t& place) const
  {
    uint32_t column;
    split_place(l.base + i, c.page_size, c.page_shift, column, place);
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
    int64_t p;
    split_slot(c, there ? name : 0, p, place);
    page = uint32_t(p);
    return there;
  }
};

// ---- shares -------------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint64_t quotient(uint64_t a, uint32_t b)
{
  return a >> 32 == 0 ? uint64_t(uint32_t(a) / b) : a / b;  // the short division where it is enough
}

// `total` chunks of all units dealt out to `teams` (at most one per chunk): the first `longer` get `each` + 1, the others `each`.
struct share {
  uint64_t total, each;
  uint32_t teams, longer;
  __device__ __forceinline__ share(uint64_t total_, uint32_t most)
    : total(total_), each(0), teams(uint32_t(min(uint64_t(most), total_))), longer(0)
  {
    if (teams != 0u) {
      each   = quotient(total, teams);
      longer = uint32_t(total - each * teams);
    }
  }
  __device__ __forceinline__ uint64_t start(uint32_t team) const { return team * each + min(team, longer); }
  __device__ __forceinline__ uint32_t team_of(uint64_t chunk) const
  {
    const uint64_t edge = longer * (each + 1);  // `each` is below 2^32 as long as there are fewer than 2^32 chunks per team
    return chunk < edge ? uint32_t(quotient(chunk, uint32_t(each + 1))) : longer + uint32_t(quotient(chunk - edge, uint32_t(each)));
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
    sum += n[i];
  }
  return sum;
}

// The number of all chunks; every warp sums it up for itself.
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

constexpr uint32_t kFan    = 8;  // parts that are joined at a time
constexpr uint32_t kLevels = 4;  // of the tree, at most: fewer than 4,096 teams

// Two parts per team: 0 of a unit that a team before began, 1 of a unit that this team begins and a later one goes on with.
struct parts_view {
  uint32_t* arrived;  // [levels][2 teams] how many of a node's parts are there; 0 between calls
  float* acc;         // [2 teams][rows][dim]
  float2* stats;      // [2 teams][rows] top (of scores in powers of two), sum
  uint32_t teams;
  uint32_t rows;  // query heads of a unit, at most
};

// A workspace begins with `arrived`, as large as any call's, so that calls of different sizes can follow one another in it.
inline size_t arrived_bytes(uint32_t teams) { return size_t(kLevels) * 2 * teams * sizeof(uint32_t); }
inline size_t arrived_bytes(const resources& res) { return round_up<size_t>(arrived_bytes(uint32_t(res.sm_count) * kMostTeams), 256); }
inline size_t part_bytes(uint32_t teams, uint32_t rows, uint32_t dim)
{
  return size_t(2) * teams * rows * (dim * sizeof(float) + sizeof(float2));
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
    if (piece == 0) { result.lse[size_t(sequence) * (w.group * c.n_heads) + head0 + r] = (safe + log2f(sum)) * kLn2; }
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

// Joins a unit's n parts, of which this team has just written number k: up the tree as long as the team is the last of its node to come.
// Part 0 is the second of team `first`, part i the first of team first + i.  A node's joined part takes the place of its first one.
template <typename T, int THREADS, uint32_t B>
__device__ __forceinline__ void join_tree(const cache_view& c, const work_view& w, const parts_view& parts, uint32_t first, uint32_t n, uint32_t k,
                                          uint32_t rows, uint32_t sequence, uint32_t head0, const result_view& result)
{
  constexpr int E = 4;
  const uint32_t thread = THREADS == 32 ? threadIdx.x & 31u : threadIdx.x;
  auto place  = [&](uint32_t p) { return p == 0 ? 2 * first + 1 : 2 * (first + p); };
  auto team_sync = [] {
    if constexpr (THREADS == 32) {
      __syncwarp();
    } else {
      __syncthreads();
    }
  };
  __shared__ uint32_t s_last;  // of block teams
  uint32_t step = 1;           // parts of a node's child
  for (uint32_t level = 0; level < kLevels; level++, step *= kFan) {
    const uint32_t node    = k / (step * kFan) * (step * kFan);  // its first part
    const uint32_t members = min(kFan, (n - node + step - 1) / step);
    const bool root        = node == 0 && n <= step * kFan;
    if (members > 1) {
      __threadfence();
      team_sync();
      uint32_t last = 0;
      if (thread == 0) { last = atomicInc(parts.arrived + size_t(level) * 2 * parts.teams + place(node), members - 1) == members - 1; }
      if constexpr (THREADS == 32) {
        last = __shfl_sync(kAllLanes, last, 0);
      } else {
        if (thread == 0) { s_last = last; }
        __syncthreads();
        last = s_last;
      }
      if (last == 0u) { return; }
      __threadfence();
      // a row's pieces of four columns lie side by side in the team's threads; B for a thread at a time
      const uint32_t pieces = c.dim / E, items = rows * pieces;
      for (uint32_t i0 = thread; i0 < items; i0 += B * THREADS) {
        float2 st[B][kFan];
        float4 y[B][kFan];
#pragma unroll
        for (uint32_t u = 0; u < B; u++) {
          const uint32_t i = min(i0 + u * THREADS, items - 1), r = i / pieces, piece = i - r * pieces;
#pragma unroll
          for (uint32_t m = 0; m < kFan; m++) {
            const size_t at = size_t(place(node + min(m, members - 1) * step)) * parts.rows + r;
            st[u][m]        = __ldcg(parts.stats + at);
            y[u][m]         = __ldcg(reinterpret_cast<const float4*>(parts.acc + at * c.dim) + piece);
          }
        }
#pragma unroll
        for (uint32_t u = 0; u < B; u++) {
          const uint32_t i = i0 + u * THREADS, r = i / pieces, piece = i - r * pieces;
          if (i >= items) { continue; }
          float top = -INFINITY, sum = 0.0f;
#pragma unroll
          for (uint32_t m = 0; m < kFan; m++) { top = fmaxf(top, st[u][m].x); }  // (the last member again and again does no harm here)
          const float safe = finite_top(top);
          float x[E]       = {};
#pragma unroll
          for (uint32_t m = 0; m < kFan; m++) {
            if (m < members) {
              const float f = power_of_2(st[u][m].x - safe);
              sum           = fmaf(st[u][m].y, f, sum);
              x[0]          = fmaf(y[u][m].x, f, x[0]);
              x[1]          = fmaf(y[u][m].y, f, x[1]);
              x[2]          = fmaf(y[u][m].z, f, x[2]);
              x[3]          = fmaf(y[u][m].w, f, x[3]);
            }
          }
          if (root) {
            const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
            T* o = reinterpret_cast<T*>(result.out.data) + int64_t(sequence) * result.out.row + int64_t(head0 + r) * result.out.head + piece * E;
            alignas(16) T z[E];
#pragma unroll
            for (int e = 0; e < E; e++) { z[e] = from_float<T>(x[e] * scale); }
            if constexpr (sizeof(T) == 2) {
              *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(z);
            } else {
              *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(z);
            }
            if (piece == 0) { result.lse[size_t(sequence) * (w.group * c.n_heads) + head0 + r] = (safe + log2f(sum)) * kLn2; }
          } else {
            // other threads of the team still read this row's old top and sum: both are written when all have read
            const size_t at = size_t(place(node)) * parts.rows + r;
            reinterpret_cast<float4*>(parts.acc + at * c.dim)[piece] = make_float4(x[0], x[1], x[2], x[3]);
          }
        }
      }
      if (!root) {
        team_sync();
        for (uint32_t r = thread; r < rows; r += THREADS) {
          float top = -INFINITY, sum = 0.0f;
          for (uint32_t m = 0; m < members; m++) { top = fmaxf(top, __ldcg(parts.stats + size_t(place(node + m * step)) * parts.rows + r).x); }
          const float safe = finite_top(top);
          for (uint32_t m = 0; m < members; m++) {
            const float2 s = __ldcg(parts.stats + size_t(place(node + m * step)) * parts.rows + r);
            sum            = fmaf(s.y, power_of_2(s.x - safe), sum);
          }
          parts.stats[size_t(place(node)) * parts.rows + r] = make_float2(top, sum);
        }
      }
    }
    if (root) { return; }
  }
}

// Goes through what the team has to do, unit by unit.  body(sequence, unit, list, chunk, end, step): the warp's chunks of a unit, into its
// registers; to_shared(): from there into the block's shared memory; to_rows(...): from there to output rows, or a part.
template <typename T, int WARPS, int CHUNK, uint32_t B, class Lists, class Body, class ToShared, class ToRows>
__device__ __forceinline__ void each_unit(const cache_view& c, const work_view& w, const Lists& lists, const result_view& result,
                                          const parts_view& parts, const block_state& s, Body&& body, ToShared&& to_shared, ToRows&& to_rows)
{
  const uint32_t warp = threadIdx.x >> 5;
  typename Lists::list l;
  auto heads_of = [&](uint32_t unit, uint32_t& rows, uint32_t& head0) {
    const uint32_t head = unit / w.n_blocks_of, of = unit - head * w.n_blocks_of;
    rows  = min(parts.rows, w.group - of * parts.rows);
    head0 = head * w.group + of * parts.rows;
  };
  uint32_t rows, head0;
  if (w.cluster != 0u) {
    const uint32_t which = blockIdx.x / w.cluster, rank = blockIdx.x - which * w.cluster;
    const uint32_t sequence = which / w.n_units, unit = which - sequence * w.n_units;
    const uint32_t n = lists.open(c, sequence, CHUNK, l);
    lists.select(c, w, sequence, unit, l);
    body(sequence, unit, l, uint32_t(uint64_t(rank) * n / w.cluster) + warp, uint32_t(uint64_t(rank + 1) * n / w.cluster), WARPS);
    heads_of(unit, rows, head0);
    __syncthreads();  // shared memory changes hands: from rows to sums
    to_shared();
    __syncthreads();
    join_warps<T, WARPS>(c, w, s, rows, sequence, head0, result, w.cluster > 1u ? TO_CLUSTER : TO_OUTPUT, parts, 0);
    if (w.cluster > 1u) { join_cluster<T, WARPS>(c, w, s, rows, sequence, head0, result); }
    return;
  }
  if constexpr (Lists::kShares) {
    const share all(all_chunks<CHUNK>(c, w, lists), parts.teams);
    const uint32_t team = w.warp_teams ? blockIdx.x * WARPS + warp : blockIdx.x;
    if (team < all.teams) {
      uint64_t at = all.start(team), before;  // chunks: the next one, those before the sequence
      const uint64_t stop = all.start(team + 1);
      uint32_t sequence   = sequence_of<CHUNK>(c, w, lists, at, before);
      uint32_t n          = sequence < w.n_sequences ? lists.open(c, sequence, CHUNK, l) : 0u;
      while (at < stop) {
        while (at >= before + uint64_t(n) * w.n_units) {  // on to the next sequence that has chunks
          before += uint64_t(n) * w.n_units;
          if (++sequence >= w.n_sequences) { break; }
          n = lists.open(c, sequence, CHUNK, l);
        }
        if (sequence >= w.n_sequences) { break; }  // lengths that changed meanwhile
        const uint32_t unit  = uint32_t(quotient(at - before, n));
        const uint64_t begin = before + uint64_t(unit) * n, end = begin + n, last = min(stop, end);
        lists.select(c, w, sequence, unit, l);
        body(sequence, unit, l, uint32_t(at - begin) + (w.warp_teams ? 0u : warp), uint32_t(last - begin), w.warp_teams ? 1u : uint32_t(WARPS));
        heads_of(unit, rows, head0);
        const bool whole    = at == begin && last == end;
        const uint32_t part = uint32_t(2 * team + (at == begin ? 1 : 0));
        if (w.warp_teams) {
          to_rows(rows, sequence, head0, whole, part);
        } else {
          __syncthreads();  // shared memory changes hands: from rows to sums
          to_shared();
          __syncthreads();
          join_warps<T, WARPS>(c, w, s, rows, sequence, head0, result, whole ? TO_OUTPUT : TO_PART, parts, part);
        }
        if (!whole) {
          const uint32_t first = all.team_of(begin), n_parts = all.team_of(end - 1) - first + 1u;
          if (w.warp_teams) {
            join_tree<T, 32, B>(c, w, parts, first, n_parts, team - first, rows, sequence, head0, result);
          } else {
            join_tree<T, WARPS * 32, B>(c, w, parts, first, n_parts, team - first, rows, sequence, head0, result);
          }
        }
        if (!w.warp_teams) { __syncthreads(); }
        at = last;
      }
    }
    empty_rows<T, WARPS, CHUNK>(c, w, lists, result);
  }
}

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

// A warp's way through its chunks of a unit, ahead of the copies: what memory says about a row two chunks ahead, the word of the filter one
// chunk ahead.  Lane i (modulo CHUNK) looks after row i of a chunk.
template <int CHUNK, class Lists>
struct row_stream {
  using name_type = typename Lists::name_type;
  const cache_view& c;
  const Lists& lists;
  const typename Lists::list& l;
  uint32_t end, step;  // chunks
  name_type name_0, name_1;
  uint32_t word_0;

  __device__ __forceinline__ row_stream(const cache_view& c_, const Lists& lists_, const typename Lists::list& l_, uint32_t chunk, uint32_t end_,
                                        uint32_t step_)
    : c(c_), lists(lists_), l(l_), end(end_), step(step_)
  {
    name_0 = name(chunk);
    name_1 = name(chunk + step);
    word_0 = word(chunk, name_0);
  }
  __device__ __forceinline__ uint32_t row(uint32_t chunk) const { return chunk * CHUNK + (threadIdx.x & 31u) % CHUNK; }
  __device__ __forceinline__ name_type name(uint32_t chunk) const { return chunk < end ? lists.name(c, l, row(chunk)) : name_type(-1); }
  __device__ __forceinline__ uint32_t word(uint32_t chunk, name_type name) const
  {
    if (c.filter == nullptr) { return 0u; }
    uint32_t page, place;
    return lists.place(c, l, row(chunk), name, page, place) ? c.filter[(uint64_t(page) * c.page_size + place) >> 5] : 0u;
  }
  // The place of this lane's row of `chunk` (false: it is not to be read), and on to the next.
  __device__ __forceinline__ bool next(uint32_t chunk, uint32_t& page, uint32_t& place)
  {
    const name_type name_2 = name(chunk + 2 * step);
    const uint32_t word_1  = word(chunk + step, name_1);
    bool there             = lists.place(c, l, row(chunk), name_0, page, place);
    if (c.filter != nullptr) { there = there && ((word_0 >> ((page * c.page_size + place) & 31u)) & 1u) != 0u; }
    name_0 = name_1;
    name_1 = name_2;
    word_0 = word_1;
    return there;
  }
};

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

// What a call launches, by type and sizes alone.
struct plan {
  uint32_t rows;      // query heads of a unit
  uint32_t chunk;     // rows of the cache that a warp takes at a time
  uint32_t resident;  // small blocks of an SM
  uint32_t large;     // warps of a large block; 0: there is none
  uint32_t warps;     // of a block
  uint32_t blocks;
  uint32_t cluster;   // 0: shares
  bool warp_teams;
  bool parts;         // a unit may lie in several shares
  uint32_t teams() const { return warp_teams ? blocks * warps : blocks; }
};

// `most`: rows of a unit, at most; `shares`: whether there may be any.
inline void deal_out(const resources& res, plan& p, uint64_t units, uint64_t most, bool shares)
{
  const uint64_t sms = uint64_t(res.sm_count), resident = std::min<uint64_t>(sms * p.resident, 4095 / kSmall);  // a tree holds 4,095 parts
  p.parts = p.warp_teams = false;
  if (units <= sms) {
    p.warps               = p.large ? p.large : kSmall;
    const uint64_t chunks = ceildiv<uint64_t>(most, p.warps * p.chunk);
    uint32_t cluster      = 1;
    while (cluster < 8 && 2 * cluster * units <= sms && cluster < chunks) { cluster *= 2; }
    if (!shares || ceildiv<uint64_t>(chunks, cluster) <= 4) {
      p.blocks  = uint32_t(units * cluster);
      p.cluster = cluster;
      return;
    }
  }
  p.warps = kSmall;
  if (!shares) {
    p.blocks  = uint32_t(units);
    p.cluster = 1;
  } else {
    const uint64_t chunks = std::max<uint64_t>(1, ceildiv<uint64_t>(most, p.chunk));
    p.warp_teams          = units >= 2 * resident;
    p.blocks              = uint32_t(std::min(resident, ceildiv<uint64_t>(units * chunks, kSmall)));
    p.cluster             = 0;
    p.parts               = chunks > 1 && p.teams() > 1;
  }
}

}  // namespace cuvs_b200::kv
