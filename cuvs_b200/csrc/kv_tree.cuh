// What the two kinds of attention of drafted tokens share: whose keys a token sees, how the work is dealt out, and the joining of parts.
//
//   S_k = scale q.k,  then cap tanh(S_k / cap),  then S_k - slope (position of q - position of k),  lse = log sum exp S_k,  o = sum exp(S_k - lse) v_k
//
// A unit is a (sequence, key head); its rows are the drafted tokens' query heads of that key head, row = token * group + head, in blocks of rows.  Its
// keys, the sequence's tokens and the drafted ones behind them, are cut into tiles.  All units' tiles stand in one row, of which every share takes an equal,
// contiguous part (kv_units.cuh); the row blocks of a unit are different thread blocks of the same share, which go through the same tiles
// at the same time, so that the second one finds them in L2.  A unit that lies in one share is finished there; of one that several shares
// have, each leaves a part (top, sum, weighted sum in 32 bits), and a second kernel joins the parts in the order of the shares.
//
// Most tiles are seen whole by all rows.  The others -- with drafted keys, at the edge of a window, with slots that are not there -- get a word of 32 bits
// for each row and 32 keys.
#pragma once

#include "kv_units.cuh"

namespace cuvs_b200::kv {

// Two 32-bit numbers in one operation.
struct two {
  uint64_t v;
  __device__ __forceinline__ two() {}
  __device__ __forceinline__ two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ two fma2(two a, two b, two c)
{
  two d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}
__device__ __forceinline__ two mul2(two a, two b)
{
  two d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ two add2(two a, two b)
{
  two d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}

struct tree_view {
  uint32_t n_drafted, group, n_rows;  // n_rows = n_drafted * group, of a unit
  uint32_t n_blocks_of;               // row blocks of a unit
  const int32_t* lengths;
  const int32_t* positions;
  int64_t positions_stride;
  const uint32_t* mask;
  int64_t mask_sequence, mask_token;
  const float* slopes;
  int64_t window;
  drafted_rows_view queries, out;
  float* lse;
  float scale_log2;  // scores in powers of two: scale * log2(e)
  float scale_cap, cap_log2;  // scale / cap, cap * log2(e); cap_log2 = 0: no cap
  float cap_near[5];          // cap_log2 tanh(y) = y (cap_near[0] + cap_near[1] y^2 + ..) for |y| below kTanhNear
};
// tanh(y) / y by least squares at Chebyshev's points of y^2: to 2^-27.
constexpr float kTanhNear = 0.4f;
constexpr float kTanh[5]  = {1.0f, -0.333333283662796f, 0.13332538306713104f, -0.0537162646651268f, 0.019272800534963608f};

// The keys of a sequence and its drafted tokens, as far as any of them may be seen.  What is in the list of positions of one token is in this one: the
// window is that of a token at position `length`, and those after it see no key before its first.
struct drafted_lists {
  static constexpr bool kShares    = true;
  static constexpr uint32_t kLeast = 2;
  const int32_t* lengths;
  int64_t window;
  uint32_t width, n_drafted;

  struct list {
    uint32_t length, first, end, base;  // keys [first, end); tiles begin at `base`
  };
  __device__ __forceinline__ uint32_t open(const cache_view& c, uint32_t sequence, uint32_t tile, list& l) const
  {
    const int64_t n = max(lengths[sequence], 0), capacity = min(int64_t(width) * c.page.size, int64_t(1) << 31);
    l.length = uint32_t(n);
    l.end    = uint32_t(min(n + n_drafted, capacity));
    l.first  = window > 0 && n + 1 > window ? uint32_t(n + 1 - window) : 0u;
    if (l.first > l.end) { l.first = l.end; }
    l.base = l.first & ~15u;
    return l.end > l.first ? (l.end - l.base + tile - 1) / tile : 0u;
  }
};

// Which of the 32 keys from `at` on a drafted token sees, as far as that does not depend on the cache.  `own`: its position, `row`: its row of the mask.
__device__ __forceinline__ uint32_t seen_keys(const tree_view& t, const drafted_lists::list& l, const int32_t* positions, int32_t own,
                                              const uint32_t* row, uint32_t at)
{
  if (own < 0 || uint32_t(own) < l.length) { return 0u; }
  uint32_t seen = 0;
  const int64_t before = int64_t(l.length) - at;  // keys of the sequence itself
  if (before > 0) { seen = before >= 32 ? 0xFFFFFFFFu : (1u << before) - 1u; }
  if (t.window > 0) {
    const int64_t gone = int64_t(own) - t.window + 1 - at;  // keys that are too far away
    if (gone > 0) { seen = gone >= 32 ? 0u : seen & ~((1u << gone) - 1u); }
  }
  if (before < 32) {
    // drafted token k is bit k - first of the word
    const int64_t first   = -before;
    const uint32_t words  = (t.n_drafted + 31) / 32;
    uint32_t drafted      = 0;
    if (first < 0) {
      drafted = row[0] << uint32_t(before);
    } else if (first < int64_t(t.n_drafted)) {
      const uint32_t word = uint32_t(first) / 32, by = uint32_t(first) & 31u;
      drafted             = row[word] >> by;
      if (by != 0u && word + 1 < words) { drafted |= row[word + 1] << (32u - by); }
    }
    const int64_t there = int64_t(t.n_drafted) - first;  // (bits behind the last token do not count)
    if (there < 32) { drafted &= there <= 0 ? 0u : (1u << there) - 1u; }
    for (uint32_t left = drafted; left != 0u; left &= left - 1u) {
      const uint32_t bit = __ffs(int(left)) - 1;
      const int32_t of   = positions[first + bit];
      const bool far     = t.window > 0 && int64_t(own) - of >= t.window;
      if (of < 0 || uint32_t(of) < l.length || far) { drafted &= ~(1u << bit); }
    }
    seen |= drafted;
  }
  return seen;
}

// ---- parts --------------------------------------------------------------------------------------------------------------------

// Two parts of every thread block, as in parts_view (`begun` is that of shares), each of `rows` rows: weighted sums as [columns / 4][rows] float4, so
// that threads of neighbouring rows write what lies together.
struct tree_parts {
  float4* acc;
  float2* stats;  // [parts][rows] top (of scores in powers of two), sum
  uint4* begun;   // [entries] sequence, key head, how many parts (0: there is none), the share that has the first
  uint32_t entries;  // one for each unit, or, where these are more than the shares, for the one unit that a share begins and does not end
  uint32_t shares, blocks_of, rows, quads;
  bool by_unit;
  __device__ __forceinline__ size_t part(uint32_t share, uint32_t block, uint32_t slot) const
  {
    return (size_t(share) * blocks_of + block) * 2 + slot;
  }
};
inline size_t tree_part_bytes(uint32_t shares, uint32_t blocks_of, uint32_t rows, uint32_t dim)
{
  return size_t(shares) * (sizeof(uint4) + size_t(blocks_of) * 2 * rows * (ceildiv(dim, 4u) * sizeof(float4) + sizeof(float2)));
}
inline tree_parts tree_parts_at(char* workspace, uint32_t shares, uint32_t blocks_of, uint32_t rows, uint32_t dim, uint64_t units)
{
  tree_parts p;
  p.by_unit   = units <= shares;
  p.entries   = p.by_unit ? uint32_t(units) : shares;
  p.shares    = shares;
  p.blocks_of = blocks_of;
  p.rows      = rows;
  p.quads     = ceildiv(dim, 4u);
  p.begun     = reinterpret_cast<uint4*>(workspace);
  p.acc       = reinterpret_cast<float4*>(p.begun + shares);
  p.stats     = reinterpret_cast<float2*>(p.acc + size_t(shares) * blocks_of * 2 * rows * p.quads);
  return p;
}

// Where row `r` of a unit goes.
template <typename T>
__device__ __forceinline__ T* out_row(const tree_view& t, uint32_t sequence, uint32_t head, uint32_t r)
{
  const uint32_t token = r / t.group, g = r - token * t.group;
  return reinterpret_cast<T*>(t.out.data) + int64_t(sequence) * t.out.sequence + int64_t(token) * t.out.token +
         int64_t(head * t.group + g) * t.out.head;
}
__device__ __forceinline__ float* lse_at(const tree_view& t, uint32_t sequence, uint32_t head, uint32_t n_heads, uint32_t r)
{
  const uint32_t token = r / t.group, g = r - token * t.group;
  return t.lse + (size_t(sequence) * t.n_drafted + token) * (t.group * n_heads) + head * t.group + g;
}

template <typename T>
__device__ __forceinline__ void store_quad(T* to, float4 x)
{
  alignas(16) T z[4] = {from_float<T>(x.x), from_float<T>(x.y), from_float<T>(x.z), from_float<T>(x.w)};
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(z);
  } else {
    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(z);
  }
}

// What sequences have no keys at all: they are in no share.  By `threads` threads of each block.
template <typename T>
__device__ __forceinline__ void empty_tree_rows(const cache_view& c, uint32_t n_sequences, const drafted_lists& lists, const tree_view& t,
                                                const tree_parts& parts, uint32_t thread, uint32_t threads)
{
  for (uint32_t b = blockIdx.x; b < n_sequences; b += gridDim.x) {
    drafted_lists::list l;
    if (lists.open(c, b, 16, l) != 0u) { continue; }
    const uint32_t quads = c.dim / 4;
    for (uint32_t h = 0; h < c.n_heads; h++) {
      if (parts.begun != nullptr && parts.by_unit && thread == 0) { parts.begun[b * c.n_heads + h] = make_uint4(0, 0, 0, 0); }
      for (uint32_t i = thread; i < t.n_rows * quads; i += threads) {
        const uint32_t r = i / quads;
        store_quad<T>(out_row<T>(t, b, h, r) + (i - r * quads) * 4, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
      }
      for (uint32_t r = thread; r < t.n_rows; r += threads) { *lse_at(t, b, h, c.n_heads, r) = -INFINITY; }
    }
  }
}

// What the join finds of a piece that begins its unit; `last`: of the share's last such unit, if entries are those of shares.
__device__ __forceinline__ void note_begun(const tree_parts& parts, const piece& p, uint32_t n_heads, uint32_t which, uint4& last)
{
  const uint4 entry = make_uint4(p.sequence, p.unit, p.whole ? 0u : p.n_parts, which);
  if (parts.begun != nullptr && parts.by_unit) {
    parts.begun[p.sequence * n_heads + p.unit] = entry;
  } else {
    last = entry;
  }
}

// ---- joining parts ------------------------------------------------------------------------------------------------------------

constexpr int kTreeJoinWarps = 8;

// A block has 32 rows (a lane each) of a unit and 8 column quads.  Of few parts a warp takes its quad of all of them; of many, warps share
// the parts of one quad after the other.
template <typename T, bool MANY>
__global__ void __launch_bounds__(kTreeJoinWarps * 32)
tree_join_kernel(tree_view t, tree_parts parts, uint32_t dim, uint32_t n_heads, float shift)
{
  chain_begin();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t groups = ceildiv(min(parts.rows, t.n_rows), 32u);
  const uint32_t entry = blockIdx.x / (groups * parts.blocks_of), rest = blockIdx.x - entry * (groups * parts.blocks_of);
  const uint32_t block = rest / groups, r = (rest - block * groups) * 32 + lane;
  uint4 unit = parts.begun[entry];
  // (an entry that nothing has written, where lengths changed meanwhile or a block gave up, leads nowhere else; those of shares are always written)
  if (parts.by_unit) { unit.x = entry / n_heads, unit.y = entry - unit.x * n_heads; }
  const uint32_t share = unit.w, n = share < parts.shares ? min(unit.z, parts.shares - share) : 0u, row = block * parts.rows + r;
  if (n == 0u || block * parts.rows + (r - lane) >= t.n_rows) { return; }
  const bool there = r < parts.rows && row < t.n_rows;
  const uint32_t rr = min(r, parts.rows - 1u);
  auto part = [&](uint32_t p) { return p == 0 ? parts.part(share, block, 1) : parts.part(share + p, block, 0); };
  constexpr int AHEAD = 4;
  __shared__ float4 s_x[MANY ? kTreeJoinWarps : 1][32];
  __shared__ float2 s_stats[MANY ? kTreeJoinWarps : 1][32];

  auto add = [&](uint32_t quad, uint32_t first, uint32_t step, float& top, float& sum, float4& x) {
    top = -INFINITY;
    sum = 0.0f;
    x   = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t p0 = first; p0 < n; p0 += step * AHEAD) {
      float2 st[AHEAD];
      float4 y[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; i++) {
        const uint32_t p = p0 + i * step;
        const size_t at  = part(min(p, n - 1u));
        st[i]            = p < n ? parts.stats[at * parts.rows + rr] : make_float2(-INFINITY, 0.0f);
        y[i]             = p < n && quad < parts.quads ? parts.acc[(at * parts.quads + quad) * parts.rows + rr] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
      float next = top;
#pragma unroll
      for (int i = 0; i < AHEAD; i++) { next = fmaxf(next, st[i].x); }
      const float safe = finite_top(next), keep = power_of_2(top - safe);
      top = next;
      sum *= keep;
      x.x *= keep, x.y *= keep, x.z *= keep, x.w *= keep;
#pragma unroll
      for (int i = 0; i < AHEAD; i++) {
        // (a part that saw nothing has a sum of 0, one whose scores are all no numbers has one that is none either)
        const float f = power_of_2(st[i].x - safe);
        sum           = fmaf(st[i].y, f, sum);
        if (st[i].x == -INFINITY) { continue; }
        x.x           = fmaf(y[i].x, f, x.x);
        x.y           = fmaf(y[i].y, f, x.y);
        x.z           = fmaf(y[i].z, f, x.z);
        x.w           = fmaf(y[i].w, f, x.w);
      }
    }
  };
  auto write = [&](uint32_t quad, float top, float sum, float4 x) {
    const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (there && quad < parts.quads) {
      store_quad<T>(out_row<T>(t, unit.x, unit.y, row) + quad * 4, make_float4(x.x * scale, x.y * scale, x.z * scale, x.w * scale));
    }
    if (there && quad == 0) { *lse_at(t, unit.x, unit.y, n_heads, row) = (finite_top(top) + log2f(sum) - shift) * kLn2; }
  };
  float top, sum;
  float4 x;
  if constexpr (!MANY) {
    const uint32_t quad = blockIdx.y * kTreeJoinWarps + warp;
    if (quad >= parts.quads) { return; }
    add(quad, 0u, 1u, top, sum, x);
    write(quad, top, sum, x);
  } else {
    const uint32_t quad = blockIdx.y;
    add(quad, warp, kTreeJoinWarps, top, sum, x);
    s_x[warp][lane]     = x;
    s_stats[warp][lane] = make_float2(top, sum);
    __syncthreads();
    if (warp != 0u) { return; }
    top = -INFINITY;
#pragma unroll
    for (int v = 0; v < kTreeJoinWarps; v++) { top = fmaxf(top, s_stats[v][lane].x); }
    const float safe = finite_top(top);
    sum              = 0.0f;
    x                = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int v = 0; v < kTreeJoinWarps; v++) {
      const float2 st = s_stats[v][lane];
      const float f = power_of_2(st.x - safe);
      sum           = fmaf(st.y, f, sum);
      if (st.x == -INFINITY) { continue; }
      const float4 y = s_x[v][lane];
      x.x            = fmaf(y.x, f, x.x);
      x.y            = fmaf(y.y, f, x.y);
      x.z            = fmaf(y.z, f, x.z);
      x.w            = fmaf(y.w, f, x.w);
    }
    write(quad, top, sum, x);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

// How a call's work is dealt out.
struct tree_plan {
  uint32_t rows;       // of a row block
  uint32_t blocks_of;  // row blocks of a unit
  uint32_t shares;
  uint32_t tile;       // keys
  uint32_t cost;       // of a unit beside its tiles, in tiles
  bool parts;          // a unit may lie in several shares
  bool sets_aside;     // sums in tensor memory may be longer than kChain tiles
};
// Tiles that a sum in tensor memory is carried over.  The tensor core cuts off what it adds to a sum, always towards 0: some 7e-7 of the sum for a tile
// of 64 keys, so that fp16 outputs of 200,000 keys in one share were 1.6e-3 too small (half a step of theirs is 4.9e-4).  After so many tiles a
// sum is set aside -- in the workspace, added in 32 bits, rounded, to those before it -- and begun anew.  With 32 tiles 2.3e-5 is lost, with 64 5.0e-5; one
// request of 250,001 + 64 tokens takes 356 us with either, 340 without.
constexpr uint32_t kChain = 32;
// `units` of `most` keys each, at most; `blocks`: thread blocks that the GPU holds at once; `least`: tiles of a share.
inline tree_plan deal_out_tree(uint32_t blocks, uint32_t rows, uint32_t tile, uint32_t cost, uint32_t least, uint64_t units, uint32_t n_rows, uint64_t most)
{
  tree_plan p;
  p.rows      = rows;
  p.tile      = tile;
  p.cost      = cost;
  p.blocks_of = ceildiv(n_rows, rows);
  const uint64_t tiles = std::max<uint64_t>(1, ceildiv<uint64_t>(most, tile));
  p.shares = uint32_t(std::max<uint64_t>(1, std::min<uint64_t>(blocks / p.blocks_of, ceildiv<uint64_t>(units * (tiles + cost), least))));
  p.parts  = p.shares > 1 && tiles > 1;
  p.sets_aside = false;
  return p;
}

constexpr uint32_t tree_columns(uint32_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Everything that a kernel for rows of one type is called with.
struct tree_call {
  cache_view c;
  work_view w;
  drafted_lists lists;
  tree_view t;
  tree_parts parts;
  tree_plan plan;
  const int32_t* pages;
  int64_t table_stride;
  float4* aside;       // of every thread block: sums that were set aside, [columns / 4][rows]
  float shift;         // weights are held times 2^shift
  uint32_t* report;    // host word that is set where a wait runs out
  uint32_t limit, skip_tile;  // of waits; for tests of them
};
template <typename T>
void attend_tree16(cudaStream_t stream, const tree_call& call);
template <>
void attend_tree16<__half>(cudaStream_t stream, const tree_call& call);
template <>
void attend_tree16<__nv_bfloat16>(cudaStream_t stream, const tree_call& call);

template <typename T>
void launch_tree_join(cudaStream_t stream, const tree_plan& p, uint64_t units, const tree_view& t, const tree_parts& parts, uint32_t dim,
                      uint32_t n_heads, float shift)
{
  const uint32_t items = parts.entries * p.blocks_of * ceildiv(std::min(p.rows, t.n_rows), 32u), quads = ceildiv(dim, 4u);
  // Many parts of few units: warps share them.
  if (uint64_t(p.shares) > 8 * units) {
    launch_chained(tree_join_kernel<T, true>, dim3(items, quads), kTreeJoinWarps * 32, 0, stream, t, parts, dim, n_heads, shift);
  } else {
    launch_chained(tree_join_kernel<T, false>, dim3(items, ceildiv(quads, uint32_t(kTreeJoinWarps))), kTreeJoinWarps * 32, 0, stream, t, parts, dim,
                   n_heads, shift);
  }
}

}  // namespace cuvs_b200::kv
