// Attention of query heads to rows of a paged cache with 32-bit products: to a sequence's 32-bit rows (`attention`), and to the rows of any
// type that a search named for each head (`attend_candidates`).
//
// What bounds it: HBM, through the bytes in flight: rows of a few hundred bytes that lie anywhere.  Every warp copies its rows into its own
// part of shared memory a stage ahead; a group of lanes -- as many as a row has 16-byte pieces -- then reads them as registers and carries a
// softmax of its own (running top, sum of weights, weighted sum of values), joined at the end.
#include "kv_attention.hpp"

#include <algorithm>
#include <type_traits>

namespace cuvs_b200::kv {

namespace {

// LANES lanes have a row, PIECES 16-byte pieces each; R query heads share its reading.
template <typename T, int LANES, int PIECES, int R, int WARPS>
struct rows_shape {
  static constexpr int kPitch    = LANES * PIECES * 16;                    // bytes of a row in shared memory
  static constexpr int kChunk    = kPitch <= 128 ? 32 : 4096 / kPitch;     // rows of a warp's stage
  static constexpr int kStages   = kPitch < 128 ? 4 : 2;
  static constexpr int kTile     = WARPS * kChunk;
  static constexpr int kGroups   = 32 / LANES;
  static constexpr int kTurns    = kChunk / kGroups;                       // rows of a lane group in a stage
  static constexpr int kColumns  = LANES * PIECES * kPerPiece<T>;
  static constexpr int kStage    = 2 * kChunk * kPitch;
  static constexpr int kStatsAt  = WARPS * kStages * kStage;
  static constexpr int kJoinedAt = kStatsAt + WARPS * R * 8;
  static constexpr int kMaskAt   = kJoinedAt + R * 8;
  static constexpr int kShared   = kMaskAt + WARPS * kStages * 4;
  static_assert(WARPS * R * kColumns * 4 <= kStatsAt, "the warps' sums take the stages' place");
};

template <typename T, int LANES, int PIECES, int R, int WARPS, class Lists>
__global__ void __launch_bounds__(WARPS * 32, WARPS == kSmall ? 3 : 1)
rows_kernel(cache_view c, work_view w, Lists lists, rows_view queries, result_view result, float scale_log2, parts_view parts)
{
  using shape          = rows_shape<T, LANES, PIECES, R, WARPS>;
  constexpr int E      = kPerPiece<T>;
  constexpr int S      = shape::kStages;
  constexpr int CHUNK  = shape::kChunk;
  constexpr int PR     = LANES * PIECES;
  constexpr int U      = 4;  // rows that a lane group takes at a time
  extern __shared__ __align__(128) char smem[];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t group = lane / LANES, gl = lane % LANES;
  const block_state state{reinterpret_cast<float*>(smem), reinterpret_cast<float2*>(smem + shape::kStatsAt),
                          reinterpret_cast<float2*>(smem + shape::kJoinedAt), shape::kColumns};
  uint32_t* s_mask       = reinterpret_cast<uint32_t*>(smem + shape::kMaskAt) + warp * S;
  const char* stages     = smem + warp * (S * shape::kStage);
  const uint32_t buffers = shared_address(stages);
  const uint32_t pieces  = c.dim / E;
  chain_begin();

  each_unit<T, WARPS, shape::kTile>(
    c, w, lists, result, parts, state,
    [&](uint32_t sequence, uint32_t unit, const typename Lists::list& l, uint32_t tile0, uint32_t tile1) {
      const uint32_t head = unit / w.n_blocks_of, of = unit - head * w.n_blocks_of;
      const uint32_t rows  = min(uint32_t(R), w.group - of * R);
      const uint32_t head0 = head * w.group + of * R;
      const char* keys     = c.keys + int64_t(head) * c.k_head * int64_t(sizeof(T));
      const char* values   = c.values + int64_t(head) * c.v_head * int64_t(sizeof(T));
      row_stream<WARPS, CHUNK, Lists> stream(c, lists, l, warp, tile0, tile1);
      auto advance = [&](uint32_t tile) {
        if (tile < tile1) {
          const uint32_t stage = (tile - tile0) % S;
          int64_t page;
          uint32_t place;
          const bool there    = stream.next(tile, page, place);
          const uint32_t mask = __ballot_sync(kAllLanes, there) & uint32_t((uint64_t(1) << CHUNK) - 1u);
          if (lane == 0) { s_mask[stage] = mask; }
          if (mask != 0u) {
            const uint32_t to  = buffers + stage * shape::kStage;
            const int64_t k_at = page * c.k_page + int64_t(place) * c.k_token;
            const int64_t v_at = page * c.v_page + int64_t(place) * c.v_token;
#pragma unroll
            for (int i = 0; i < CHUNK * PR / 32; i++) {
              const uint32_t piece = (lane + 32u * i) % PR, row = (lane + 32u * i) / PR;
              const int64_t k   = __shfl_sync(kAllLanes, k_at, row);
              const int64_t v   = __shfl_sync(kAllLanes, v_at, row);
              const bool read   = ((mask >> row) & 1u) != 0u && piece < pieces;
              const uint32_t at = to + row * shape::kPitch + piece * 16u;
              copy_piece(at, read ? keys + k * int64_t(sizeof(T)) + piece * 16 : c.keys, read);
              copy_piece(at + CHUNK * shape::kPitch, read ? values + v * int64_t(sizeof(T)) + piece * 16 : c.values, read);
            }
          }
        }
        copies_end_group();  // past the unit's end an empty one
      };

      float q[R][PIECES][E], acc[R][PIECES][E] = {}, top[R], sum[R];
#pragma unroll
      for (int r = 0; r < R; r++) {
        top[r] = -INFINITY;
        sum[r] = 0.0f;
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
          const uint32_t j = gl + p * LANES;
          uint4 x          = make_uint4(0, 0, 0, 0);
          if (uint32_t(r) < rows && j < pieces) {
            x = reinterpret_cast<const uint4*>(queries.data + (int64_t(sequence) * queries.row + int64_t(head0 + r) * queries.head) *
                                                                int64_t(sizeof(T)))[j];
          }
          piece_to_floats<T>(x, q[r][p]);
        }
      }
#pragma unroll
      for (int i = 0; i < S; i++) { advance(tile0 + i); }

      for (uint32_t tile = tile0; tile < tile1; tile++) {
        copies_wait<S - 1>();
        __syncwarp();
        const uint32_t stage = (tile - tile0) % S;
        const uint32_t mask  = s_mask[stage];
        if (mask != 0u) {
          const char* k_rows = stages + stage * shape::kStage;
          const char* v_rows = k_rows + CHUNK * shape::kPitch;
#pragma unroll 1
          for (int u0 = 0; u0 < shape::kTurns; u0 += U) {
            float score[R][U];
#pragma unroll
            for (int u = 0; u < U; u++) {
              const uint32_t row = uint32_t(u0 + u) * shape::kGroups + group;
              float x[PIECES][E];
#pragma unroll
              for (int p = 0; p < PIECES; p++) {
                piece_to_floats<T>(*reinterpret_cast<const uint4*>(k_rows + row * shape::kPitch + (gl + p * LANES) * 16), x[p]);
              }
              const bool ok = ((mask >> row) & 1u) != 0u;
#pragma unroll
              for (int r = 0; r < R; r++) {
                float s = 0.0f;
#pragma unroll
                for (int p = 0; p < PIECES; p++) {
#pragma unroll
                  for (int e = 0; e < E; e++) { s = fmaf(q[r][p][e], x[p][e], s); }
                }
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) { s += __shfl_xor_sync(kAllLanes, s, o); }
                score[r][u] = ok ? s * scale_log2 : -INFINITY;
              }
            }
#pragma unroll
            for (int r = 0; r < R; r++) {
              float next = top[r];
#pragma unroll
              for (int u = 0; u < U; u++) { next = fmaxf(next, score[r][u]); }
              const float safe = finite_top(next);
              const float keep = exp2f(top[r] - safe);
              top[r]           = next;
              sum[r] *= keep;
#pragma unroll
              for (int p = 0; p < PIECES; p++) {
#pragma unroll
                for (int e = 0; e < E; e++) { acc[r][p][e] *= keep; }
              }
#pragma unroll
              for (int u = 0; u < U; u++) {
                score[r][u] = exp2f(score[r][u] - safe);
                sum[r] += score[r][u];
              }
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
                  for (int e = 0; e < E; e++) { acc[r][p][e] = fmaf(score[r][u], x[e], acc[r][p][e]); }
                }
              }
            }
          }
        }
        __syncwarp();
        advance(tile + S);
      }
      copies_wait<0>();
      __syncthreads();  // shared memory changes hands: from rows to sums
#pragma unroll
      for (int r = 0; r < R; r++) {
#pragma unroll
        for (int o = LANES; o < 32; o <<= 1) {
          const float other = __shfl_xor_sync(kAllLanes, top[r], o);
          const float next  = fmaxf(top[r], other);
          const float safe  = finite_top(next);
          const float own = exp2f(top[r] - safe), theirs = exp2f(other - safe);
          sum[r] = sum[r] * own + __shfl_xor_sync(kAllLanes, sum[r], o) * theirs;
#pragma unroll
          for (int p = 0; p < PIECES; p++) {
#pragma unroll
            for (int e = 0; e < E; e++) { acc[r][p][e] = acc[r][p][e] * own + __shfl_xor_sync(kAllLanes, acc[r][p][e], o) * theirs; }
          }
          top[r] = next;
        }
        if (group == 0) {
#pragma unroll
          for (int p = 0; p < PIECES; p++) {
#pragma unroll
            for (int e = 0; e < E; e += 4) {
              *reinterpret_cast<float4*>(state.acc + (warp * R + r) * shape::kColumns + (gl + p * LANES) * E + e) =
                make_float4(acc[r][p][e], acc[r][p][e + 1], acc[r][p][e + 2], acc[r][p][e + 3]);
            }
          }
        }
        if (lane == 0) { state.stats[warp * R + r] = make_float2(top[r], sum[r]); }
      }
    });
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

uint32_t chunk_of(uint32_t pieces)
{
  uint32_t chunk = 0;
  by_pieces(pieces, [&](auto lanes, auto n) { chunk = rows_shape<float, decltype(lanes)::value, decltype(n)::value, 1, kSmall>::kChunk; });
  return chunk;
}

plan attention_plan(const resources& res, elem type, uint64_t sequences, uint32_t n_heads, uint32_t group, uint32_t dim, uint64_t capacity,
                    int64_t window)
{
  // a window may begin anywhere in 16 positions
  const uint64_t most = window > 0 && uint64_t(window) < capacity ? std::min(capacity, uint64_t(window) + 15) : capacity;
  plan p{};
  bool large = true;
  if (type == elem::f32) {
    p.rows     = dim > 128 ? std::min(group, 4u) : group > 4 ? 8 : group;
    p.rows     = p.rows == 3 ? 4 : p.rows;
    p.chunk    = chunk_of(dim / 4);
    p.resident = 3;
  } else {
    const uint32_t d = padded(dim), eights = group <= 8 ? 1 : group <= 16 || d == 256 ? 2 : 4;
    p.rows     = 8 * eights;
    p.chunk    = 16;
    p.resident = d == 256 ? 1 : eights == 4 ? 2 : 3;
    large      = has_large(d, eights);
  }
  deal_out(res, p, sequences * n_heads * ceildiv(group, p.rows), most, large, true);
  return p;
}

template <typename T, int LANES, int PIECES, int R, class Lists, typename... Args>
void launch_rows(resources& res, const plan& p, Args&&... args)
{
  if (p.warps == uint32_t(kLarge)) {
    launch_units(res, rows_kernel<T, LANES, PIECES, R, kLarge, Lists>, p.blocks, kLarge * 32, p.cluster,
                 rows_shape<T, LANES, PIECES, R, kLarge>::kShared, args...);
  } else {
    launch_units(res, rows_kernel<T, LANES, PIECES, R, kSmall, Lists>, p.blocks, kSmall * 32, p.cluster,
                 rows_shape<T, LANES, PIECES, R, kSmall>::kShared, args...);
  }
}

template <typename T>
void launch_candidates(resources& res, const candidates_args& a)
{
  const uint32_t group = a.n_query_heads / a.cache.n_heads, pieces = a.cache.dim / kPerPiece<T>;
  const named_slots lists{a.candidates, a.n_candidates};
  parts_view parts{};
  plan p{};
  p.rows = parts.rows = 1;
  p.chunk             = chunk_of(pieces);
  p.resident          = 3;
  deal_out(res, p, uint64_t(a.n_tokens) * a.n_query_heads, a.n_candidates, true, false);
  const work_view w{a.n_tokens, a.n_query_heads, group, group, p.cluster};
  by_pieces(pieces, [&](auto lanes, auto n) {
    constexpr int LANES = decltype(lanes)::value, PIECES = decltype(n)::value;
    if constexpr (sizeof(T) == 4 || PIECES == 1) {
      launch_rows<T, LANES, PIECES, 1, named_slots>(res, p, a.cache, w, lists, a.queries, result_view{a.out, a.lse}, a.scale * kLog2E, parts);
    }
  });
}

}  // namespace

size_t attention_workspace(const resources& res, elem type, uint32_t n_sequences, uint32_t n_query_heads, uint32_t n_heads, uint32_t dim,
                           uint64_t capacity, int64_t window)
{
  const plan p = attention_plan(res, type, n_sequences, n_heads, n_query_heads / n_heads, dim, capacity, window);
  return p.join ? part_bytes(p.blocks, p.rows, dim) : 0;
}

void attention(resources& res, const attention_args& a)
{
  if (a.n_sequences == 0) { return; }
  const cache_view& c  = a.cache;
  const uint32_t group = a.n_query_heads / c.n_heads;
  const plan p         = attention_plan(res, a.type, a.n_sequences, c.n_heads, group, c.dim, uint64_t(a.table_width) * c.page_size, a.window);
  const uint32_t of    = ceildiv(group, p.rows);
  const work_view w{a.n_sequences, c.n_heads * of, of, group, p.cluster};
  const positions lists{a.pages, a.lengths, a.table_stride, a.window, a.table_width};
  const result_view result{a.out, a.lse};
  parts_view parts{};
  if (p.join) { parts = parts_at(a.workspace, p.blocks, p.rows, c.dim); }
  parts.rows = p.rows;
  auto join  = [&](auto type) {
    if (p.join) { launch_join<decltype(type)>(res, p, w, parts, c.dim, c.n_heads, result); }
  };
  if (a.type == elem::f16) {
    attention16<__half>(res, a, p, w, lists, result, parts);
    return join(__half{});
  }
  if (a.type == elem::bf16) {
    attention16<__nv_bfloat16>(res, a, p, w, lists, result, parts);
    return join(__nv_bfloat16{});
  }
  by_pieces(c.dim / 4, [&](auto lanes, auto n) {
    constexpr int LANES = decltype(lanes)::value, PIECES = decltype(n)::value;
    auto go = [&](auto r) {
      constexpr int R = decltype(r)::value;
      launch_rows<float, LANES, PIECES, R, positions>(res, p, c, w, lists, a.queries, result, a.scale * kLog2E, parts);
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

void attend_candidates(resources& res, const candidates_args& a)
{
  if (a.n_tokens == 0) { return; }
  switch (a.type) {
    case elem::f16: return launch_candidates<__half>(res, a);
    case elem::bf16: return launch_candidates<__nv_bfloat16>(res, a);
    default: return launch_candidates<float>(res, a);
  }
}

}  // namespace cuvs_b200::kv
