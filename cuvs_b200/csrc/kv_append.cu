// Appending rows to a paged cache: keys and values of new tokens go to the places that the table of pages gives their positions, keys
// (and the queries that come with them) turned by their positions on the way.
//
// Pairs of columns (x1, x2) become (x1 cos a - x2 sin a, x2 cos a + x1 sin a), a = position * frequency.  The angle is formed and reduced
// to half a turn in 64 bits -- a position of a million times a frequency of one leaves 32 bits no digits for the sine.  Sine and cosine are
// taken of its first 32 bits and turned by the rest (to first order: it is below 2^-25), so that they are as exact as the functions are, once
// per token and pair for all of its heads.
#include "kv_rows.cuh"

#include <algorithm>

namespace cuvs_b200::kv {

namespace {

constexpr int kWarps = 8;

// A row is cut into 16-byte pieces.  Where the halves that pair up start on piece boundaries (PAIRED), a step is two pieces, j and
// j + half; else it is one piece, whose pairs lie inside it (ADJACENT) or anywhere in the row (ANYWHERE: then one lane's store must not
// be another's load, and a warp reads all of a row's elements before it writes any).  That last way is the plain one: a row of a lane group in
// flight, partners read one by one: 20,000 tokens of 32 + 2 x 8 heads of 128 f16 269 us with 50 pairs, 107 with 48.
enum { ADJACENT = 0, PAIRED = 1, ANYWHERE = 2 };

// A warp has a token, or some of its rows: its lanes take the token's angles, then go through the rows, each lane at the same pieces of every
// row, so that it holds their sines and cosines in registers; four rows of a lane are in flight at a time.
//
// What bounds it: HBM.  Blocks that went through the rows of eight tokens with the angles in shared memory waited for those (four lanes on
// one bank): 20,000 tokens of 32 + 2 x 8 heads of 128 f16 92 us, now 85 (5.8 TB/s).
template <typename T, int MODE>
__global__ void __launch_bounds__(kWarps * 32)
append_kernel(append_args a, uint32_t log_lanes, uint32_t steps, uint32_t slices, uint32_t rows_of_slice)
{
  chain_begin();
  constexpr int E     = kPerPiece<T>;
  constexpr int AHEAD = 4;
  extern __shared__ __align__(16) float2 s_turn[];
  const uint32_t lane  = threadIdx.x & 31u;
  float2* turn         = s_turn + (threadIdx.x >> 5) * a.n_pairs;  // cos, sin
  const uint64_t task  = uint64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const uint32_t token = uint32_t(task / slices), slice = uint32_t(task - uint64_t(token) * slices);
  if (token >= a.n_tokens) { return; }

  const int32_t pos = a.positions[token];
  const int64_t seq = a.sequences ? int64_t(a.sequences[token]) : int64_t(token);
  int64_t slot      = -1;
  if (seq >= 0 && seq < int64_t(a.n_sequences)) {
    slot = slot_of(a.pages + seq * a.table_stride, a.table_width, pos, a.cache.page, a.cache.n_pages);
  }
  if (slice == 0 && lane == 0) { a.slots[token] = slot; }
  uint32_t page, place;
  split_slot(a.cache, max(slot, int64_t(0)), page, place);
  for (uint32_t pair = lane; pair < a.n_pairs; pair += 32) {
    const double f = a.frequencies_f32 ? double(static_cast<const float*>(a.frequencies)[pair]) : static_cast<const double*>(a.frequencies)[pair];
    const double half_turns = double(max(pos, 0)) * f * 0.31830988618379067154;  // 1 / pi
    const double angle = half_turns - 2.0 * rint(0.5 * half_turns);
    const float near   = float(angle), rest = float(angle - double(near)) * 3.14159265f;
    float s, c;
    sincospif(near, &s, &c);
    turn[pair] = make_float2(fmaf(-s, rest, c), fmaf(c, rest, s));
  }
  __syncwarp();

  const uint32_t heads  = a.cache.n_heads;
  const uint32_t begin  = slice * rows_of_slice;
  const uint32_t end    = min(begin + rows_of_slice, a.n_query_heads + 2 * heads);
  const uint32_t gl     = lane & ((1u << log_lanes) - 1u);
  const uint32_t stride = 32u >> log_lanes;
  // where a row comes from and goes to; whether it is turned (values are not, nor is what has no position)
  auto row_at = [&](uint32_t r, const char*& from, char*& to) -> bool {
    from = nullptr;
    if (r >= end) { return false; }
    if (r < a.n_query_heads) {
      from = a.queries.data + (int64_t(token) * a.queries.row + int64_t(r) * a.queries.head) * int64_t(sizeof(T));
      to   = a.rotated.data + (int64_t(token) * a.rotated.row + int64_t(r) * a.rotated.head) * int64_t(sizeof(T));
      return pos >= 0;
    }
    if (slot < 0) { return false; }
    const uint32_t h = r - a.n_query_heads;
    if (h < heads) {
      from = a.keys + (int64_t(token) * a.k_row + int64_t(h) * a.k_head) * int64_t(sizeof(T));
      to   = const_cast<char*>(a.cache.keys) +
           (int64_t(page) * a.cache.k_page + int64_t(place) * a.cache.k_token + int64_t(h) * a.cache.k_head) * int64_t(sizeof(T));
      return true;
    }
    from = a.values + (int64_t(token) * a.v_row + int64_t(h - heads) * a.v_head) * int64_t(sizeof(T));
    to   = const_cast<char*>(a.cache.values) +
         (int64_t(page) * a.cache.v_page + int64_t(place) * a.cache.v_token + int64_t(h - heads) * a.cache.v_head) * int64_t(sizeof(T));
    return false;
  };

  if constexpr (MODE == ANYWHERE) {
    for (uint32_t r0 = begin; r0 < end; r0 += stride) {
      const char* from;
      char* to;
      const bool turned = row_at(r0 + (lane >> log_lanes), from, to);
      // at most two pieces per lane (log_lanes is 5 for rows of more than 16 pieces); kept until the whole warp has read
      uint4 kept[2];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const uint32_t j = gl + (uint32_t(u) << log_lanes);
        if (from == nullptr || j >= steps) { continue; }
        kept[u] = reinterpret_cast<const uint4*>(from)[j];
        if (turned && j * E < 2 * a.n_pairs) {
          float x[E];
          piece_to_floats<T>(kept[u], x);
#pragma unroll
          for (int e = 0; e < E; e++) {
            const uint32_t column = j * E + e;
            if (column < a.n_pairs) {
              const float2 cs = turn[column];
              x[e]            = x[e] * cs.x - to_float(reinterpret_cast<const T*>(from)[column + a.n_pairs]) * cs.y;
            } else if (column < 2 * a.n_pairs) {
              const float2 cs = turn[column - a.n_pairs];
              x[e]            = x[e] * cs.x + to_float(reinterpret_cast<const T*>(from)[column - a.n_pairs]) * cs.y;
            }
          }
          kept[u] = floats_to_piece<T>(x);
        }
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const uint32_t j = gl + (uint32_t(u) << log_lanes);
        if (from != nullptr && j < steps) { reinterpret_cast<uint4*>(to)[j] = kept[u]; }
      }
    }
  } else {
    const uint32_t half = a.n_pairs / E;  // PAIRED: in pieces
    for (uint32_t j = gl; j < steps; j += 1u << log_lanes) {
      constexpr int PAIRS = MODE == PAIRED ? E : E / 2;  // of a step
      const uint32_t pair = j * PAIRS;
      const bool two      = MODE == PAIRED && j < half;
      const uint32_t at   = MODE == PAIRED && !two ? j + half : j;
      float2 cs[PAIRS];
#pragma unroll
      for (int e = 0; e < PAIRS; e++) { cs[e] = pair + e < a.n_pairs ? turn[pair + e] : make_float2(1.0f, 0.0f); }
      for (uint32_t r0 = begin + (lane >> log_lanes); r0 < end; r0 += AHEAD * stride) {
        uint4 lo[AHEAD], hi[MODE == PAIRED ? AHEAD : 1];
        char* to[AHEAD];
        bool there[AHEAD], turned[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
          const char* from;
          turned[u] = row_at(r0 + u * stride, from, to[u]);
          there[u]  = from != nullptr;
          lo[u]     = load_piece(from + at * 16, there[u]);
          if constexpr (MODE == PAIRED) { hi[u] = load_piece(from + (j + half) * 16, there[u] && two); }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
          if (turned[u] && pair < a.n_pairs) {
            float x[E];
            piece_to_floats<T>(lo[u], x);
            if constexpr (MODE == PAIRED) {
              float y[E];
              piece_to_floats<T>(hi[u], y);
#pragma unroll
              for (int e = 0; e < E; e++) {
                const float v = x[e] * cs[e].x - y[e] * cs[e].y;
                y[e]          = y[e] * cs[e].x + x[e] * cs[e].y;
                x[e]          = v;
              }
              hi[u] = floats_to_piece<T>(y);
            } else {
#pragma unroll
              for (int e = 0; e < E; e += 2) {
                if (pair + e / 2 < a.n_pairs) {
                  const float v = x[e] * cs[e / 2].x - x[e + 1] * cs[e / 2].y;
                  x[e + 1]      = x[e + 1] * cs[e / 2].x + x[e] * cs[e / 2].y;
                  x[e]          = v;
                }
              }
            }
            lo[u] = floats_to_piece<T>(x);
          }
          if (there[u]) {
            reinterpret_cast<uint4*>(to[u])[at] = lo[u];
            if constexpr (MODE == PAIRED) {
              if (two) { reinterpret_cast<uint4*>(to[u])[j + half] = hi[u]; }
            }
          }
        }
      }
    }
  }
}

template <typename T>
void launch(resources& res, cudaStream_t stream, const append_args& a)
{
  constexpr uint32_t E  = kPerPiece<T>;
  const uint32_t pieces = a.cache.dim / E;
  const int mode        = a.interleaved || a.n_pairs == 0 ? ADJACENT : a.n_pairs % E == 0 ? PAIRED : ANYWHERE;
  const uint32_t steps  = mode == PAIRED ? pieces - a.n_pairs / E : pieces;
  uint32_t log_lanes    = 0;
  while (log_lanes < 5 && (1u << log_lanes) < steps) { log_lanes++; }
  // Fewer lanes to a row where more of their turns are full: 40 steps are 5 turns of 8 lanes, or 2 of 32 that are 62% full (14,701 tokens of
  // 9 + 2 x 3 rows of 160 f32, 16 columns turned: 59 us against 70).
  if (mode != ANYWHERE) {
    auto turns = [&](uint32_t log) { return ceildiv(steps, 1u << log) << log; };
    uint32_t best = log_lanes;
    for (uint32_t log = log_lanes; log >= 2; log--) {
      if (turns(log) < turns(best)) { best = log; }
    }
    log_lanes = best;
  }
  // A token's rows go to several warps where tokens are few: until there are 16 warps per SM, or a warp has one turn of rows.
  const uint32_t rows = a.n_query_heads + 2 * a.cache.n_heads, turn = 32u >> log_lanes;
  uint32_t slices     = 1;
  while (uint64_t(a.n_tokens) * slices * 2 <= uint64_t(res.sm_count) * 16 && rows > turn * slices) { slices *= 2; }
  const uint32_t rows_of_slice = round_up(ceildiv(rows, slices), turn);
  const size_t smem            = size_t(kWarps) * a.n_pairs * sizeof(float2);
  auto go                      = [&](auto kernel) {
    launch_chained(kernel, dim3(uint32_t(ceildiv<uint64_t>(uint64_t(a.n_tokens) * slices, kWarps))), kWarps * 32, smem, stream, a, log_lanes,
                   steps, slices, rows_of_slice);
  };
  if (mode == PAIRED) {
    go(append_kernel<T, PAIRED>);
  } else if (mode == ADJACENT) {
    go(append_kernel<T, ADJACENT>);
  } else {
    go(append_kernel<T, ANYWHERE>);
  }
  count_launches(res, 1);
}

}  // namespace

void append(resources& res, cudaStream_t stream, const append_args& a)
{
  if (a.n_tokens == 0) { return; }
  switch (a.type) {
    case elem::f16: return launch<__half>(res, stream, a);
    case elem::bf16: return launch<__nv_bfloat16>(res, stream, a);
    default: return launch<float>(res, stream, a);
  }
}

}  // namespace cuvs_b200::kv
