// Attention of query heads to rows of a paged cache with 32-bit products: to a sequence's 32-bit rows (`attention`), and to the rows of any
// type that a search named for each head (`attend_candidates`).
//
// What bounds it: HBM, through the bytes in flight: rows of a few hundred bytes that lie anywhere.  Every warp copies its rows into its own
// part of shared memory a stage ahead; a group of lanes -- as many as a row has 16-byte pieces -- then reads them as registers and carries a
// softmax of its own (running top, sum of weights, weighted sum of values), joined at the end.  64 tokens x 32 heads x 1,000 candidates of 128
// bf16: 163-166 us for the 0.99 GB that random rows bring from DRAM (6.0 TB/s; loaded into registers four rows at a time: 187); 32-bit rows of
// one head, 64 columns, with a window and a filter: 26 us with the join for 116 MB, bound by instructions (loaded into registers: 45).
#include "kv_attention.hpp"

#include <algorithm>
#include <type_traits>

namespace cuvs_b200::kv {

namespace {

// Rows of a chunk, by the 16-byte pieces that a row has room for in shared memory: 4 KB of keys for several query heads, 2 KB for one, which
// leaves room for more warps; 16 at most (a chunk's mask has 16 bits).
constexpr uint32_t chunk_of(uint32_t pieces, uint32_t heads)
{
  const uint32_t rows = (heads == 1 ? 128 : 256) / pieces;
  return rows < 16 ? rows : 16;
}
// Small blocks of an SM and warps of a large block: what registers leave room for (the way through shares takes some).
constexpr uint32_t resident_of(uint32_t heads, bool shares) { return heads > 1 ? 3 : shares ? 4 : 6; }
constexpr int large_of(uint32_t heads, bool shares) { return heads > 1 ? 12 : shares ? 16 : 24; }

// LANES lanes have a row, PIECES 16-byte pieces each; R query heads share its reading.
template <typename T, int LANES, int PIECES, int R, int WARPS, bool SHARES>
struct rows_shape {
  static constexpr int kPitch    = LANES * PIECES * 16;                    // bytes of a row in shared memory
  static constexpr int kChunk    = chunk_of(LANES * PIECES, R);            // rows of a warp's stage
  static constexpr int kStages   = kPitch < 128 ? 4 : R == 1 && SHARES ? 3 : 2;
  static constexpr int kGroups   = 32 / LANES;
  static constexpr int kTurns    = kChunk / kGroups;                       // rows of a lane group in a stage
  static constexpr int kColumns  = LANES * PIECES * kPerPiece<T>;
  static constexpr int kStage    = 2 * kChunk * kPitch;
  static constexpr int kStatsAt  = WARPS * kStages * kStage;
  static constexpr int kJoinedAt = kStatsAt + WARPS * R * 8;
  static constexpr int kMaskAt   = kJoinedAt + R * 8;
  static constexpr int kPortion  = (2 + PIECES * kPerPiece<T>) * 32;         // floats that a warp sends another: the sums of a query head
  static constexpr int kExchangeAt = kMaskAt + WARPS * 16;
  static constexpr int kShared   = kExchangeAt + (WARPS == kSmall && SHARES ? WARPS / 2 * kPortion * 4 : 0);
  static_assert(kChunk <= 16, "masks of 16 bits");
  static_assert(WARPS * R * kColumns * 4 <= kStatsAt, "the warps' sums take the stages' place");
};

template <typename T, int LANES, int PIECES, int R, int WARPS, bool SHARES>
struct rows_hooks {
  using shape                    = rows_shape<T, LANES, PIECES, R, WARPS, SHARES>;
  static constexpr int E         = kPerPiece<T>;
  static constexpr int CHUNK     = shape::kChunk;
  static constexpr int U         = shape::kTurns < 4 ? shape::kTurns : 4;  // rows that a lane group takes at a time
  static constexpr int ROWS      = LANES == 32 ? 1 : 32 / LANES;           // a copy of a warp: one piece of every lane (of 64: two), so many rows

  static constexpr int kPortion  = shape::kPortion;
  static constexpr int kPortions = R;

  const cache_view& c;
  const work_view& w;
  const rows_view& queries;
  const result_view& result;
  const parts_view& parts;
  const block_state& state;
  float scale_log2;
  uint32_t warp, lane, group, gl;
  const char* stages;
  uint32_t buffers, copy_row, copy_piece_of;
  const char *keys, *values;
  float q[R][PIECES][E], acc[R][PIECES][E], top[R], sum[R];

  __device__ __forceinline__ rows_hooks(const cache_view& c_, const work_view& w_, const rows_view& queries_, const result_view& result_,
                                        const parts_view& parts_, const block_state& state_, const char* smem, float scale_log2_)
    : c(c_), w(w_), queries(queries_), result(result_), parts(parts_), state(state_), scale_log2(scale_log2_), warp(threadIdx.x >> 5),
      lane(threadIdx.x & 31u), group((threadIdx.x & 31u) / LANES), gl((threadIdx.x & 31u) % LANES)
  {
    stages        = smem + warp * (shape::kStages * shape::kStage);
    buffers       = shared_address(stages);
    copy_row      = LANES == 32 ? 0u : lane / LANES;
    copy_piece_of = LANES == 32 ? lane : lane % LANES;
  }
  __device__ __forceinline__ uint32_t pieces() const { return c.dim / E; }

  __device__ __forceinline__ void attach(uint32_t unit)
  {
    const uint32_t head = unit / w.n_blocks_of;
    keys                = c.keys + int64_t(head) * c.k_head * int64_t(sizeof(T));
    values              = c.values + int64_t(head) * c.v_head * int64_t(sizeof(T));
  }

  __device__ __forceinline__ uint32_t copy(uint32_t stage, uint32_t page, uint32_t place, bool there)
  {
    const uint32_t mask = __ballot_sync(kAllLanes, there) & ((1u << CHUNK) - 1u);
    if (mask == 0u) { return 0u; }
    const uint32_t to   = buffers + stage * shape::kStage + copy_row * shape::kPitch + copy_piece_of * 16;
    const uint32_t k_at = there ? page * c.k_page_units + place * c.k_token_units : 0u;
    const uint32_t v_at = there ? page * c.v_page_units + place * c.v_token_units : 0u;
#pragma unroll
    for (int i = 0; i < CHUNK / ROWS; i++) {
      const char* k_from = keys + (uint64_t(__shfl_sync(kAllLanes, k_at, copy_row + i * ROWS)) << c.unit_shift);
      const char* v_from = values + (uint64_t(__shfl_sync(kAllLanes, v_at, copy_row + i * ROWS)) << c.unit_shift);
      const bool read    = ((mask >> (copy_row + i * ROWS)) & 1u) != 0u;
#pragma unroll
      for (int p = 0; p < PIECES; p++) {
        const uint32_t piece = copy_piece_of + p * 32, bytes = read && piece < pieces() ? 16u : 0u;
        const uint32_t at    = to + i * (ROWS * shape::kPitch) + p * 512;
        copy_piece(at, k_from + (piece < pieces() ? piece * 16 : 0), bytes);
        copy_piece(at + CHUNK * shape::kPitch, v_from + (piece < pieces() ? piece * 16 : 0), bytes);
      }
    }
    return mask;
  }

  __device__ __forceinline__ void start(uint32_t sequence, uint32_t unit)
  {
    const uint32_t head = unit / w.n_blocks_of, of = unit - head * w.n_blocks_of;
    const uint32_t rows = min(uint32_t(R), w.group - of * R), head0 = head * w.group + of * R;
    const char* first   = queries.data + (int64_t(sequence) * queries.row + int64_t(head0) * queries.head) * int64_t(sizeof(T));
#pragma unroll
    for (int r = 0; r < R; r++) {
      top[r] = -INFINITY;
      sum[r] = 0.0f;
#pragma unroll
      for (int p = 0; p < PIECES; p++) {
        const uint32_t j = gl + p * LANES;
        uint4 x          = make_uint4(0, 0, 0, 0);
        if (uint32_t(r) < rows && j < pieces()) { x = reinterpret_cast<const uint4*>(first + int64_t(r) * queries.head * int64_t(sizeof(T)))[j]; }
        piece_to_floats<T>(x, q[r][p]);
#pragma unroll
        for (int e = 0; e < E; e++) { acc[r][p][e] = 0.0f; }
      }
    }
  }

  // A lane group's sums of U values over its lanes: halves of the lanes take halves of the values, so that lane gl ends with the sum of value
  // own(gl) alone: 5 exchanges of four values over 16 lanes instead of 16.
  __device__ __forceinline__ uint32_t own() const { return gl / (LANES / U); }
  __device__ __forceinline__ float own_sum(float (&v)[U]) const
  {
#pragma unroll
    for (int n = U, o = LANES / 2; n > 1; n /= 2, o /= 2) {
      const bool upper = (gl & uint32_t(o)) != 0u;
#pragma unroll
      for (int i = 0; i < n / 2; i++) {
        const float give = upper ? v[i] : v[i + n / 2];
        v[i]             = (upper ? v[i + n / 2] : v[i]) + __shfl_xor_sync(kAllLanes, give, o);
      }
    }
#pragma unroll
    for (int o = LANES / U / 2; o > 0; o /= 2) { v[0] += __shfl_xor_sync(kAllLanes, v[0], o); }
    return v[0];
  }

  __device__ __forceinline__ void consume(uint32_t stage, uint32_t mask)
  {
    const char* k_rows = stages + stage * shape::kStage;
    const char* v_rows = k_rows + CHUNK * shape::kPitch;
#pragma unroll 1
    for (int u0 = 0; u0 < shape::kTurns; u0 += U) {
      float part[R][U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t row = uint32_t(u0 + u) * shape::kGroups + group;
        float x[PIECES][E];
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
          piece_to_floats<T>(*reinterpret_cast<const uint4*>(k_rows + row * shape::kPitch + (gl + p * LANES) * 16), x[p]);
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
          float s = 0.0f;
#pragma unroll
          for (int p = 0; p < PIECES; p++) {
#pragma unroll
            for (int e = 0; e < E; e++) { s = fmaf(q[r][p][e], x[p][e], s); }
          }
          part[r][u] = s;
        }
      }
      const bool ok = ((mask >> (uint32_t(u0 + own()) * shape::kGroups + group)) & 1u) != 0u;
#pragma unroll
      for (int r = 0; r < R; r++) {
        const float s     = own_sum(part[r]);
        const float score = ok ? s * scale_log2 : -INFINITY;
        float next        = fmaxf(top[r], score);
#pragma unroll
        for (int o = LANES / 2; o >= LANES / U; o /= 2) { next = fmaxf(next, __shfl_xor_sync(kAllLanes, next, o)); }
        const float safe = finite_top(next);
        const float keep = power_of_2(top[r] - safe);
        top[r]           = next;
        const float weight = power_of_2(score - safe) * w.room;
        sum[r]             = sum[r] * keep + weight;  // of the lane's own rows, until close()
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
#pragma unroll
          for (int e = 0; e < E; e++) { acc[r][p][e] *= keep; }
        }
#pragma unroll
        for (int u = 0; u < U; u++) { part[r][u] = __shfl_sync(kAllLanes, weight, u * (LANES / U), LANES); }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t row = uint32_t(u0 + u) * shape::kGroups + group;
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
          float x[E];
          piece_to_floats<T>(*reinterpret_cast<const uint4*>(v_rows + row * shape::kPitch + (gl + p * LANES) * 16), x);
#pragma unroll
          for (int r = 0; r < R; r++) {
#pragma unroll
            for (int e = 0; e < E; e++) { acc[r][p][e] = fmaf(part[r][u], x[e], acc[r][p][e]); }
          }
        }
      }
    }
  }

  // the lanes of a group, then the warp's lane groups
  __device__ __forceinline__ void close()
  {
#pragma unroll
    for (int r = 0; r < R; r++) {
#pragma unroll
      for (int o = LANES / 2; o >= LANES / U; o /= 2) { sum[r] += __shfl_xor_sync(kAllLanes, sum[r], o); }
#pragma unroll
      for (int o = LANES; o < 32; o <<= 1) {
        const float other = __shfl_xor_sync(kAllLanes, top[r], o);
        const float next  = fmaxf(top[r], other);
        const float safe  = finite_top(next);
        const float own = power_of_2(top[r] - safe), theirs = power_of_2(other - safe);
        sum[r] = sum[r] * own + __shfl_xor_sync(kAllLanes, sum[r], o) * theirs;
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
#pragma unroll
          for (int e = 0; e < E; e++) { acc[r][p][e] = acc[r][p][e] * own + __shfl_xor_sync(kAllLanes, acc[r][p][e], o) * theirs; }
        }
        top[r] = next;
      }
    }
  }

  // a lane's own values to the same lane of another warp
  __device__ __forceinline__ void send(int r, float* to) const
  {
    to[lane]      = top[r];
    to[lane + 32] = sum[r];
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
#pragma unroll
      for (int e = 0; e < E; e++) { to[lane + 32 * (2 + p * E + e)] = acc[r][p][e]; }
    }
  }
  __device__ __forceinline__ void receive(int r, const float* from)
  {
    const float other = from[lane], next = fmaxf(top[r], other), safe = finite_top(next);
    const float own = power_of_2(top[r] - safe), theirs = power_of_2(other - safe);
    sum[r] = sum[r] * own + from[lane + 32] * theirs;
    top[r] = next;
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
#pragma unroll
      for (int e = 0; e < E; e++) { acc[r][p][e] = acc[r][p][e] * own + from[lane + 32 * (2 + p * E + e)] * theirs; }
    }
  }

  __device__ __forceinline__ void to_floats(float* row, int r) const
  {
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        if (gl + p * LANES < pieces()) {
          *reinterpret_cast<float4*>(row + (gl + p * LANES) * E + e) = make_float4(acc[r][p][e], acc[r][p][e + 1], acc[r][p][e + 2], acc[r][p][e + 3]);
        }
      }
    }
  }
  __device__ __forceinline__ void to_shared() const
  {
#pragma unroll
    for (int r = 0; r < R; r++) {
      if (group == 0) { to_floats(state.acc + (warp * R + r) * shape::kColumns, r); }
      if (lane == 0) { state.stats[warp * R + r] = make_float2(top[r], sum[r]); }
    }
  }
  __device__ __forceinline__ void to_rows(uint32_t rows, uint32_t sequence, uint32_t head0, bool whole, uint32_t part) const
  {
    if (group != 0) { return; }
#pragma unroll
    for (int r = 0; r < R; r++) {
      if (uint32_t(r) >= rows) { continue; }
      if (whole) {
        const float scale = sum[r] == 0.0f ? 0.0f : 1.0f / sum[r];
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
          if (gl + p * LANES < pieces()) {
            float x[E];
#pragma unroll
            for (int e = 0; e < E; e++) { x[e] = acc[r][p][e] * scale; }
            store_piece<T>(result.out, sequence, head0 + r, gl + p * LANES, x);
          }
        }
        if (gl == 0) { result.lse[size_t(sequence) * (w.group * c.n_heads) + head0 + r] = (finite_top(top[r]) + log2f(sum[r] * w.back)) * kLn2; }
      } else {
        to_floats(parts.acc + (size_t(part) * parts.rows + r) * c.dim, r);
        if (gl == 0) { parts.stats[size_t(part) * parts.rows + r] = make_float2(top[r], sum[r]); }
      }
    }
  }
};

template <typename T, int LANES, int PIECES, int R, int WARPS, class Lists>
__global__ void __launch_bounds__(WARPS * 32, WARPS == kSmall ? resident_of(R, Lists::kShares) : 1)
rows_kernel(cache_view c, work_view w, Lists lists, rows_view queries, result_view result, float scale_log2, parts_view parts)
{
  using shape = rows_shape<T, LANES, PIECES, R, WARPS, Lists::kShares>;
  extern __shared__ __align__(128) char smem[];
  const block_state state{reinterpret_cast<float*>(smem), reinterpret_cast<float2*>(smem + shape::kStatsAt),
                          reinterpret_cast<float2*>(smem + shape::kJoinedAt), shape::kColumns};
  uint32_t* s_mask = reinterpret_cast<uint32_t*>(smem + shape::kMaskAt) + (threadIdx.x >> 5) * shape::kStages;
  chain_begin();
  rows_hooks<T, LANES, PIECES, R, WARPS, Lists::kShares> hooks(c, w, queries, result, parts, state, smem, scale_log2);
  run_units<T, WARPS, shape::kChunk, shape::kStages>(c, w, lists, result, parts, state, reinterpret_cast<float*>(smem + shape::kExchangeAt), s_mask,
                                                     hooks);
}

// How rows of so many 16-byte pieces are read.
template <class Fn>
void by_pieces(uint32_t pieces, Fn&& fn)
{
  using std::integral_constant;
  if (pieces <= 4) {
    fn(integral_constant<int, 4>{}, integral_constant<int, 1>{});
  } else if (pieces <= 8) {
    fn(integral_constant<int, 8>{}, integral_constant<int, 1>{});
  } else if (pieces <= 16) {
    fn(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  } else if (pieces <= 32) {
    fn(integral_constant<int, 32>{}, integral_constant<int, 1>{});
  } else {
    fn(integral_constant<int, 32>{}, integral_constant<int, 2>{});
  }
}

uint32_t room_of(uint32_t pieces)
{
  uint32_t room = 0;
  by_pieces(pieces, [&](auto lanes, auto n) { room = decltype(lanes)::value * decltype(n)::value; });
  return room;
}

plan attention_plan(const resources& res, elem type, uint64_t sequences, uint32_t n_heads, uint32_t group, uint32_t dim, uint64_t capacity,
                    int64_t window)
{
  // The cost of a unit is what the end of one piece and the start of the next take a block: 2.5 us for eight heads of 16 bits, against the 0.35 us of
  // a chunk.  With shares of equal chunks those with many short units were done last (16 requests of up to 2,000 tokens, 128 units: 32 us, 16
  // with it).  32-bit rows of one to eight heads: 0, 4, 8, 16 chunks are 55, 44, 42, 42 us for one head (64 requests of up to 1,000 tokens, 8 key
  // heads), 79, 55, 46, 48 for four, 47, 35, 30, 30 for eight (2 key heads).
  // A window may begin anywhere in 16 positions.
  const uint64_t most = window > 0 && uint64_t(window) < capacity ? std::min(capacity, uint64_t(window) + 15) : capacity;
  plan p{};
  if (type == elem::f32) {
    p.rows     = dim > 128 ? std::min(group, 4u) : group > 4 ? 8 : group;
    p.rows     = p.rows == 3 ? 4 : p.rows;
    p.chunk    = chunk_of(room_of(dim / 4), p.rows);
    p.resident = resident_of(p.rows, true);
    p.large    = large_of(p.rows, true);
    p.cost     = 8;
  } else {
    const uint32_t d = padded(dim), eights = group <= 8 ? 1 : group <= 16 || d == 256 ? 2 : 4;
    p.rows     = 8 * eights;
    p.chunk    = 16;
    p.resident = d == 256 ? 1 : eights == 4 ? 2 : 3;
    p.large    = mma_large_of(d, eights);
    p.cost     = 8 * eights * (d == 256 ? 2 : 1);
  }
  deal_out(uint32_t(res.sm_count), res.clusters_at_once, p, sequences * n_heads * ceildiv(group, p.rows), most, true);
  return p;
}

template <typename T, int LANES, int PIECES, int R, class Lists, typename... Args>
void launch_rows(cudaStream_t stream, const plan& p, Args&&... args)
{
  constexpr int LARGE = large_of(R, Lists::kShares);
  if (p.warps == uint32_t(LARGE)) {
    launch_units(stream, rows_kernel<T, LANES, PIECES, R, LARGE, Lists>, p.blocks, LARGE * 32, p.cluster,
                 rows_shape<T, LANES, PIECES, R, LARGE, Lists::kShares>::kShared, args...);
  } else {
    launch_units(stream, rows_kernel<T, LANES, PIECES, R, kSmall, Lists>, p.blocks, kSmall * 32, p.cluster,
                 rows_shape<T, LANES, PIECES, R, kSmall, Lists::kShares>::kShared, args...);
  }
}

template <typename T>
void launch_candidates(resources& res, cudaStream_t stream, const candidates_args& a)
{
  const uint32_t group = a.n_query_heads / a.cache.n_heads, pieces = a.cache.dim / kPerPiece<T>;
  const named_slots lists{a.candidates, a.n_candidates};
  parts_view parts{};
  plan p{};
  p.rows = parts.rows = 1;
  p.chunk             = chunk_of(room_of(pieces), 1);
  p.resident          = resident_of(1, false);
  p.large             = large_of(1, false);
  deal_out(uint32_t(res.sm_count), res.clusters_at_once, p, uint64_t(a.n_tokens) * a.n_query_heads, a.n_candidates, false);
  work_view w{a.n_tokens, a.n_query_heads, group, group, p.cluster, 0};
  make_room(w, a.n_candidates);
  by_pieces(pieces, [&](auto lanes, auto n) {
    constexpr int LANES = decltype(lanes)::value, PIECES = decltype(n)::value;
    if constexpr (sizeof(T) == 4 || PIECES == 1) {
      launch_rows<T, LANES, PIECES, 1, named_slots>(stream, p, a.cache, w, lists, a.queries, result_view{a.out, a.lse}, a.scale * kLog2E, parts);
    }
  });
}

}  // namespace

size_t attention_workspace(const resources& res, elem type, uint32_t n_sequences, uint32_t n_query_heads, uint32_t n_heads, uint32_t dim,
                           uint64_t capacity, int64_t window)
{
  const plan p = attention_plan(res, type, n_sequences, n_heads, n_query_heads / n_heads, dim, capacity, window);
  return p.parts ? part_bytes(p.blocks, p.rows, dim) : 0;
}

void attention(resources& res, cudaStream_t stream, const attention_args& a)
{
  if (a.n_sequences == 0) { return; }
  const cache_view& c  = a.cache;
  const uint32_t group = a.n_query_heads / c.n_heads;
  const plan p         = attention_plan(res, a.type, a.n_sequences, c.n_heads, group, c.dim, uint64_t(a.table_width) * c.page.size, a.window);
  const uint32_t of    = ceildiv(group, p.rows);
  const uint64_t longest = uint64_t(a.table_width) * c.page.size;
  work_view w{a.n_sequences, c.n_heads * of, of, group, p.cluster, p.cost};
  make_room(w, a.window > 0 ? std::min(longest, uint64_t(a.window)) : longest);
  const positions lists{a.pages, a.lengths, a.table_stride, a.window, a.table_width};
  const result_view result{a.out, a.lse};
  parts_view parts{};
  if (p.parts) { parts = parts_at(a.workspace, p.blocks, p.rows, c.dim); }
  parts.shares = p.blocks;
  parts.rows   = p.rows;
  count_launches(res, p.parts ? 2 : 1);
  auto join = [&](auto type) {
    if (p.parts) { launch_join<decltype(type)>(res, stream, p, w, parts, c.dim, c.n_heads, result); }
  };
  if (a.type == elem::f16) {
    attention16<__half>(stream, a, p, w, lists, result, parts);
    return join(__half{});
  }
  if (a.type == elem::bf16) {
    attention16<__nv_bfloat16>(stream, a, p, w, lists, result, parts);
    return join(__nv_bfloat16{});
  }
  by_pieces(c.dim / 4, [&](auto lanes, auto n) {
    constexpr int LANES = decltype(lanes)::value, PIECES = decltype(n)::value;
    auto go = [&](auto r) {
      launch_rows<float, LANES, PIECES, decltype(r)::value, positions>(stream, p, c, w, lists, a.queries, result, a.scale * kLog2E, parts);
    };
    using std::integral_constant;
    if (p.rows == 1) {
      go(integral_constant<int, 1>{});
    } else if (p.rows == 2) {
      go(integral_constant<int, 2>{});
    } else if (p.rows == 4) {
      go(integral_constant<int, 4>{});
    } else if constexpr (PIECES == 1) {
      go(integral_constant<int, 8>{});
    }
  });
  join(float{});
}

void attend_candidates(resources& res, cudaStream_t stream, const candidates_args& a)
{
  if (a.n_tokens == 0) { return; }
  count_launches(res, 1);
  switch (a.type) {
    case elem::f16: return launch_candidates<__half>(res, stream, a);
    case elem::bf16: return launch_candidates<__nv_bfloat16>(res, stream, a);
    default: return launch_candidates<float>(res, stream, a);
  }
}

}  // namespace cuvs_b200::kv
