// Appending rows to a paged cache: keys and values of new tokens go to the places that the table of pages gives their positions, keys
// (and the queries that come with them) turned by their positions on the way.
//
// Pairs of columns (x1, x2) become (x1 cos a - x2 sin a, x2 cos a + x1 sin a), a = position * frequency.  The angle is formed and reduced
// to half a turn in 64 bits -- a position of a million times a frequency of one leaves 32 bits no digits for the sine -- and sine and cosine
// are taken in 32 bits of the rest, once per token and pair for all of its heads.
#include "kv_rows.cuh"

#include <algorithm>

namespace cuvs_b200::kv {

namespace {

constexpr int kThreads = 256;

// A row is cut into 16-byte pieces.  Where the halves that pair up start on piece boundaries (PAIRED), a step is two pieces, j and
// j + half; else it is one piece, whose pairs lie inside it (adjacent pairs) or anywhere in the row (then one thread's store must not
// be another's load: ANYWHERE reads all of a row's elements in a warp before it writes any).
enum { ADJACENT = 0, PAIRED = 1, ANYWHERE = 2 };

template <typename T, int MODE>
__global__ void __launch_bounds__(kThreads)
append_kernel(append_args a, uint32_t tokens_per_block, uint32_t log_lanes, uint32_t steps)
{
  chain_begin();
  constexpr int E = kPerPiece<T>;
  extern __shared__ __align__(16) char smem[];
  float2* turn     = reinterpret_cast<float2*>(smem);                                                    // [tokens][pairs] cos, sin
  int64_t* s_slot  = reinterpret_cast<int64_t*>(smem + size_t(tokens_per_block) * a.n_pairs * sizeof(float2));
  int32_t* s_pos   = reinterpret_cast<int32_t*>(s_slot + tokens_per_block);
  const uint32_t t0 = blockIdx.x * tokens_per_block;
  const uint32_t n  = min(tokens_per_block, a.n_tokens - t0);
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const int32_t pos  = a.positions[t0 + i];
    const int64_t seq  = a.sequences ? int64_t(a.sequences[t0 + i]) : int64_t(t0 + i);
    int64_t slot       = -1;
    if (seq >= 0 && seq < int64_t(a.n_sequences)) {
      slot = slot_of(a.pages + seq * a.table_stride, a.table_width, pos, a.cache.page_size, a.cache.page_shift, a.cache.n_pages);
    }
    s_slot[i] = slot;
    s_pos[i]  = pos;
    if (blockIdx.y == 0) { a.slots[t0 + i] = slot; }
  }
  for (uint32_t i = threadIdx.x; i < n * a.n_pairs; i += kThreads) {
    const uint32_t token = i / a.n_pairs, pair = i - token * a.n_pairs;
    const int32_t pos    = a.positions[t0 + token];
    const double f       = a.frequencies_f32 ? double(static_cast<const float*>(a.frequencies)[pair])
                                             : static_cast<const double*>(a.frequencies)[pair];
    const double half_turns = double(max(pos, 0)) * f * 0.31830988618379067154;  // 1 / pi
    const double whole      = 2.0 * rint(0.5 * half_turns);
    float s, c;
    sincospif(float(half_turns - whole), &s, &c);
    turn[i] = make_float2(c, s);
  }
  __syncthreads();

  const uint32_t heads  = a.cache.n_heads;
  const uint32_t rows   = a.n_query_heads + 2 * heads;
  const uint32_t lane   = threadIdx.x & ((1u << log_lanes) - 1u);
  const uint32_t stride = uint32_t(kThreads) >> log_lanes;
  const uint32_t end    = n * rows;
  for (uint32_t r0 = blockIdx.y * stride; r0 < end; r0 += gridDim.y * stride) {
    const uint32_t r = r0 + (threadIdx.x >> log_lanes);
    const bool here  = r < end;
    const uint32_t i = here ? r / rows : 0u;
    uint32_t head    = here ? r - i * rows : 0u;
    const char* from = nullptr;
    char* to         = nullptr;
    bool turned      = s_pos[i] >= 0;
    const size_t t   = t0 + i;
    if (here) {
      const int64_t slot = s_slot[i];
      if (head < a.n_query_heads) {
        from = a.queries.data + (int64_t(t) * a.queries.row + head * a.queries.head) * sizeof(T);
        to   = a.rotated.data + (int64_t(t) * a.rotated.row + head * a.rotated.head) * sizeof(T);
      } else {
        head -= a.n_query_heads;
        const bool value = head >= heads;
        if (value) { head -= heads; }
        if (slot >= 0) {
          int64_t page;
          uint32_t place;
          split_slot(a.cache, slot, page, place);
          if (value) {
            turned = false;
            from   = a.values + (int64_t(t) * a.v_row + head * a.v_head) * sizeof(T);
            to     = const_cast<char*>(a.cache.values) +
                 (page * a.cache.v_page + place * a.cache.v_token + head * a.cache.v_head) * sizeof(T);
          } else {
            from = a.keys + (int64_t(t) * a.k_row + head * a.k_head) * sizeof(T);
            to   = const_cast<char*>(a.cache.keys) +
                 (page * a.cache.k_page + place * a.cache.k_token + head * a.cache.k_head) * sizeof(T);
          }
        }
      }
    }
    const float2* angles = turn + i * a.n_pairs;
    if constexpr (MODE == PAIRED) {
      const uint32_t half = a.n_pairs / E;
      for (uint32_t j = lane; j < steps; j += 1u << log_lanes) {
        if (from == nullptr) { continue; }
        if (j < half) {
          uint4 lo = reinterpret_cast<const uint4*>(from)[j], hi = reinterpret_cast<const uint4*>(from)[j + half];
          if (turned) {
            float x[E], y[E];
            piece_to_floats<T>(lo, x);
            piece_to_floats<T>(hi, y);
#pragma unroll
            for (int e = 0; e < E; e++) {
              const float2 cs = angles[j * E + e];
              const float u   = x[e] * cs.x - y[e] * cs.y;
              y[e]            = y[e] * cs.x + x[e] * cs.y;
              x[e]            = u;
            }
            lo = floats_to_piece<T>(x);
            hi = floats_to_piece<T>(y);
          }
          reinterpret_cast<uint4*>(to)[j]        = lo;
          reinterpret_cast<uint4*>(to)[j + half] = hi;
        } else {
          reinterpret_cast<uint4*>(to)[j + half] = reinterpret_cast<const uint4*>(from)[j + half];
        }
      }
    } else if constexpr (MODE == ADJACENT) {
      for (uint32_t j = lane; j < steps; j += 1u << log_lanes) {
        if (from == nullptr) { continue; }
        uint4 w = reinterpret_cast<const uint4*>(from)[j];
        if (turned && j * E < 2 * a.n_pairs) {
          float x[E];
          piece_to_floats<T>(w, x);
#pragma unroll
          for (int e = 0; e < E; e += 2) {
            const uint32_t pair = (j * E + e) / 2;
            if (pair < a.n_pairs) {
              const float2 cs = angles[pair];
              const float u   = x[e] * cs.x - x[e + 1] * cs.y;
              x[e + 1]        = x[e + 1] * cs.x + x[e] * cs.y;
              x[e]            = u;
            }
          }
          w = floats_to_piece<T>(x);
        }
        reinterpret_cast<uint4*>(to)[j] = w;
      }
    } else {
      // at most two pieces per lane (log_lanes is 5 for rows of more than 16 pieces); kept until the whole warp has read
      uint4 kept[2];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const uint32_t j = lane + (uint32_t(u) << log_lanes);
        if (from == nullptr || j >= steps) { continue; }
        kept[u] = reinterpret_cast<const uint4*>(from)[j];
        if (turned && j * E < 2 * a.n_pairs) {
          float x[E];
          piece_to_floats<T>(kept[u], x);
#pragma unroll
          for (int e = 0; e < E; e++) {
            const uint32_t column = j * E + e;
            if (column < a.n_pairs) {
              const float2 cs = angles[column];
              x[e] = x[e] * cs.x - to_float(reinterpret_cast<const T*>(from)[column + a.n_pairs]) * cs.y;
            } else if (column < 2 * a.n_pairs) {
              const float2 cs = angles[column - a.n_pairs];
              x[e] = x[e] * cs.x + to_float(reinterpret_cast<const T*>(from)[column - a.n_pairs]) * cs.y;
            }
          }
          kept[u] = floats_to_piece<T>(x);
        }
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const uint32_t j = lane + (uint32_t(u) << log_lanes);
        if (from != nullptr && j < steps) { reinterpret_cast<uint4*>(to)[j] = kept[u]; }
      }
    }
  }
}

template <typename T>
void launch(resources& res, const append_args& a)
{
  constexpr uint32_t E  = kPerPiece<T>;
  const uint32_t pieces = a.cache.dim / E;
  const int mode        = a.interleaved || a.n_pairs == 0 ? ADJACENT : a.n_pairs % E == 0 ? PAIRED : ANYWHERE;
  const uint32_t steps  = mode == PAIRED ? pieces - a.n_pairs / E : pieces;
  uint32_t log_lanes    = 0;
  while (log_lanes < 5 && (1u << log_lanes) < steps) { log_lanes++; }
  // Tokens per block: as many as leave every SM several blocks, eight at most.
  uint32_t per_block = 1;
  while (per_block < 8 && a.n_tokens / (2 * per_block) >= uint32_t(res.sm_count) * 8) { per_block *= 2; }
  const size_t smem = size_t(per_block) * (a.n_pairs * sizeof(float2) + sizeof(int64_t) + sizeof(int32_t));
  const dim3 grid(ceildiv(a.n_tokens, per_block), 1);
  auto go = [&](auto kernel) {
    launch_chained(kernel, grid, kThreads, smem, res.stream, a, per_block, log_lanes, steps);
    CUDA_TRY(cudaGetLastError());
  };
  if (mode == PAIRED) {
    go(append_kernel<T, PAIRED>);
  } else if (mode == ADJACENT) {
    go(append_kernel<T, ADJACENT>);
  } else {
    go(append_kernel<T, ANYWHERE>);
  }
  res.launches++;
}

}  // namespace

void append(resources& res, const append_args& a)
{
  if (a.n_tokens == 0) { return; }
  switch (a.type) {
    case elem::f16: return launch<__half>(res, a);
    case elem::bf16: return launch<__nv_bfloat16>(res, a);
    default: return launch<float>(res, a);
  }
}

}  // namespace cuvs_b200::kv
