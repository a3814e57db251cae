// Attention of drafted tokens to the rows of their sequences in a paged cache, with 32-bit products (the mathematics: kv_tree.cuh).
#include "kv_tree.cuh"
#include "tc_ptx.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace cuvs_b200::kv {

namespace {

constexpr int kThreads = 256;

// What a block's first warp finds of its share, for all of them: lengths that somebody changes meanwhile must not lead them apart.
struct found_piece {
  piece now;
  drafted_lists::list l;
  uint32_t more;
};
template <class Walk>
__device__ __forceinline__ bool next_piece(Walk& path, found_piece& found, piece& now, drafted_lists::list& l)
{
  __syncthreads();
  if (threadIdx.x < 32) {
    const bool more = path.next(now);
    if (threadIdx.x == 0) {
      found.more = more;
      found.now  = now;
      found.l    = path.l;
    }
  }
  __syncthreads();
  now = found.now;
  l   = found.l;
  return found.more != 0u;
}

// Blocks of an SM: what shared memory leaves room for.
constexpr int tree_resident(int columns) { return columns == 64 ? 2 : 1; }

// D: columns of a row in shared memory; BM: rows of a block.  Threads stand in 16 x 16: thread (y, x) has BM / 16 rows, their scores with every 16th key
// and their weighted sums in every 16th four columns.
//
// What bounds it: 32-bit multiply-adds, and the barriers between a tile's steps with few blocks of an SM.  One sequence of 20,000 + 64 tokens, 2 key heads of 4,
// 128 columns: 188 us, 28 TFLOP/s (264 where a tile was loaded between barriers).
template <int D>
struct tree_shape {
  static constexpr int BM     = 64;
  static constexpr int kTile  = D <= 128 ? 64 : 32;
  static constexpr int kRows  = BM / 16;    // of a thread
  static constexpr int kKeys  = kTile / 16;
  static constexpr int kQuads = D / 64;
  static constexpr int kPitch = D + 4;      // floats: 16 lanes' quads of different rows on different banks
  static constexpr int kKAt   = BM * kPitch;
  static constexpr int kStage = 2 * kTile * kPitch;  // keys, values; two of them: a tile is copied while the one before it is worked on
  static constexpr int kPAt   = kKAt + 2 * kStage;
  static constexpr int kSeenAt = kPAt + BM * (kTile + 4);
  static constexpr int kValidAt = kSeenAt + BM * (kTile / 32);
  static constexpr int kPlaceAt = kValidAt + 4;
  static constexpr int kShared = (kPlaceAt + 2 * 3 * kTile) * 4;
  static constexpr int kResident = tree_resident(D);
  static_assert(kResident * (kShared + 1024) <= 233472, "");
};

template <int D>
__global__ void __launch_bounds__(kThreads, tree_shape<D>::kResident)
tree_rows_kernel(cache_view c, work_view w, drafted_lists lists, tree_view t, tree_parts parts, const int32_t* pages, int64_t table_stride, float shift)
{
  using T     = float;
  using shape = tree_shape<D>;
  constexpr int BM = shape::BM;
  constexpr int TILE = shape::kTile, ROWS = shape::kRows, KEYS = shape::kKeys, QUADS = shape::kQuads, PITCH = shape::kPitch, E = kPerPiece<T>;
  chain_begin();
  extern __shared__ __align__(16) float s_mem[];
  float* s_q        = s_mem;
  float* s_p        = s_mem + shape::kPAt;
  uint32_t* s_seen  = reinterpret_cast<uint32_t*>(s_mem + shape::kSeenAt);
  uint32_t* s_valid_of[2] = {reinterpret_cast<uint32_t*>(s_mem + shape::kValidAt), reinterpret_cast<uint32_t*>(s_mem + shape::kValidAt) + 2};
  // of each stage: places of keys, of values, the keys' positions
  auto places = [&](uint32_t stage) { return reinterpret_cast<uint32_t*>(s_mem + shape::kPlaceAt) + stage * (3 * TILE); };
  const uint32_t y = threadIdx.x / 16, x = threadIdx.x % 16;
  const uint32_t which = blockIdx.x / t.n_blocks_of, block = blockIdx.x - which * t.n_blocks_of;
  const uint32_t row0 = block * BM, rows = min(uint32_t(BM), t.n_rows - row0);
  const uint32_t pieces = c.dim / E;

  walk<TILE, drafted_lists> path(c, w, lists, parts.shares, which);
  piece now;
  uint4 begun = make_uint4(0, 0, 0, 0);
  __shared__ found_piece s_found;
  drafted_lists::list l;
  while (next_piece(path, s_found, now, l)) {
    const uint32_t head         = now.unit;
    const int32_t* table        = pages + int64_t(now.sequence) * table_stride;
    const int32_t* positions    = t.positions + int64_t(now.sequence) * t.positions_stride;
    // queries; columns and rows that are none: 0
    for (uint32_t i = threadIdx.x; i < uint32_t(BM * (D / E)); i += kThreads) {
      const uint32_t r = i / (D / E), p = i - r * (D / E);
      float f[E] = {};
      if (r < rows && p < pieces) {
        const uint32_t token = (row0 + r) / t.group, g = row0 + r - token * t.group;
        piece_to_floats<T>(reinterpret_cast<const uint4*>(t.queries.data + (int64_t(now.sequence) * t.queries.sequence + int64_t(token) * t.queries.token +
                                                                            int64_t(head * t.group + g) * t.queries.head) * int64_t(sizeof(T)))[p], f);
      }
#pragma unroll
      for (int e = 0; e < E; e++) { s_q[r * PITCH + p * E + e] = f[e]; }
    }
    int32_t own[ROWS];
    float slope[ROWS], top[ROWS], sum[ROWS], acc[ROWS][QUADS][4];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const uint32_t r = row0 + min(y * ROWS + i, rows - 1u), token = r / t.group;
      own[i]   = positions[token];
      slope[i] = t.slopes != nullptr ? t.slopes[head * t.group + (r - token * t.group)] * kLog2E : 0.0f;
      top[i]   = -INFINITY;
      sum[i]   = 0.0f;
#pragma unroll
      for (int q = 0; q < QUADS; q++) { acc[i][q][0] = acc[i][q][1] = acc[i][q][2] = acc[i][q][3] = 0.0f; }
    }
    int32_t latest = 0;
    if (t.window > 0) {
      for (uint32_t i = 0; i < t.n_drafted; i++) { latest = max(latest, positions[i]); }
    }

    auto look = [&](uint32_t tile, uint32_t stage) {
      if (threadIdx.x >= TILE) { return; }
      const uint32_t at = l.base + tile * TILE + threadIdx.x;
      bool there        = at >= l.first && at < l.end;
      uint32_t column, place;
      split_place(min(at, 0x7FFFFFFFu), c.page, column, place);
      const int32_t page = there ? table[column] : -1;  // at < end: the column is inside the table
      there              = there && page >= 0 && page < c.n_pages;
      if (there && c.filter != nullptr) {
        const uint64_t slot = uint64_t(page) * c.page.size + place;
        there               = (c.filter[slot >> 5] >> (slot & 31u)) & 1u;
      }
      int32_t of = int32_t(at);
      if (there && at >= l.length) {
        of    = positions[at - l.length];
        there = of >= 0 && uint32_t(of) >= l.length;
      }
      uint32_t* at_stage               = places(stage) + threadIdx.x;
      at_stage[0]                      = there ? uint32_t(page) * c.k_page_units + place * c.k_token_units : 0u;
      at_stage[TILE]                   = there ? uint32_t(page) * c.v_page_units + place * c.v_token_units : 0u;
      at_stage[2 * TILE]               = uint32_t(of);
      const uint32_t word = __ballot_sync(kAllLanes, there);
      if ((threadIdx.x & 31u) == 0) { s_valid_of[stage][threadIdx.x / 32] = word; }
    };
    // rows that are not there, and columns behind a row's end: 0
    auto load = [&](uint32_t stage) {
      const uint32_t to = shared_address(s_mem + shape::kKAt + stage * shape::kStage);
      const char *keys = c.keys + int64_t(head) * c.k_head * 4, *values = c.values + int64_t(head) * c.v_head * 4;
#pragma unroll 4
      for (uint32_t i = threadIdx.x; i < uint32_t(TILE * (D / E)); i += kThreads) {
        const uint32_t k = i / (D / E), p = i - k * (D / E);
        const bool there = p < pieces && ((s_valid_of[stage][k / 32] >> (k & 31u)) & 1u) != 0u;
        const uint32_t from = there ? p * 16 : 0u, bytes = there ? 16u : 0u;
        copy_piece(to + (k * PITCH + p * E) * 4, keys + (uint64_t(places(stage)[k]) << c.unit_shift) + from, bytes);
        copy_piece(to + ((TILE + k) * PITCH + p * E) * 4, values + (uint64_t(places(stage)[TILE + k]) << c.unit_shift) + from, bytes);
      }
    };
    look(now.chunk, 0);
    __syncthreads();
    load(0);
    copies_end_group();
    for (uint32_t tile = now.chunk; tile < now.end; tile++) {
      const uint32_t stage = (tile - now.chunk) & 1u, base = l.base + tile * TILE;
      const bool mixed     = int64_t(base) + TILE > int64_t(l.length) || (t.window > 0 && int64_t(base) <= int64_t(latest) - t.window);
      if (tile + 1 < now.end) { look(tile + 1, stage ^ 1u); }
      __syncthreads();
      if (tile + 1 < now.end) { load(stage ^ 1u); }
      copies_end_group();
      const float* s_k        = s_mem + shape::kKAt + stage * shape::kStage;
      const float* s_v        = s_k + TILE * PITCH;
      const uint32_t* s_valid = s_valid_of[stage];
      const int32_t* s_of     = reinterpret_cast<const int32_t*>(places(stage)) + 2 * TILE;
      for (uint32_t i = threadIdx.x; i < uint32_t(BM * (TILE / 32)); i += kThreads) {
        const uint32_t r = i / (TILE / 32), word = i - r * (TILE / 32);
        uint32_t seen = s_valid[word];
        if (r >= rows) {
          seen = 0;
        } else {
          const uint32_t token = (row0 + r) / t.group;
          const int32_t at     = positions[token];
          if (mixed) {
            seen &= seen_keys(t, l, positions, at, t.mask + int64_t(now.sequence) * t.mask_sequence + int64_t(token) * t.mask_token, base + word * 32);
          } else if (at < 0 || uint32_t(at) < l.length) {
            seen = 0;
          }
        }
        s_seen[i] = seen;
      }
      copies_wait<1>();
      __syncthreads();

      float s[ROWS][KEYS] = {};
#pragma unroll 4
      for (int d = 0; d < D; d += 4) {
        float4 q[ROWS], k[KEYS];
#pragma unroll
        for (int i = 0; i < ROWS; i++) { q[i] = *reinterpret_cast<const float4*>(s_q + (y * ROWS + i) * PITCH + d); }
#pragma unroll
        for (int j = 0; j < KEYS; j++) { k[j] = *reinterpret_cast<const float4*>(s_k + (x + 16 * j) * PITCH + d); }
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
#pragma unroll
          for (int j = 0; j < KEYS; j++) {
            s[i][j] = fmaf(q[i].x, k[j].x, s[i][j]);
            s[i][j] = fmaf(q[i].y, k[j].y, s[i][j]);
            s[i][j] = fmaf(q[i].z, k[j].z, s[i][j]);
            s[i][j] = fmaf(q[i].w, k[j].w, s[i][j]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < ROWS; i++) {
        const uint32_t r = y * ROWS + i;
        float next       = top[i];
#pragma unroll
        for (int j = 0; j < KEYS; j++) {
          const uint32_t k = x + 16 * j;
          float score      = t.cap_log2 != 0.0f ? tanhf(s[i][j] * t.scale_cap) * t.cap_log2 : s[i][j] * t.scale_log2;
          if (t.slopes != nullptr) { score = fmaf(slope[i], float(int64_t(s_of[k]) - own[i]), score); }
          s[i][j] = ((s_seen[r * (TILE / 32) + k / 32] >> (k & 31u)) & 1u) != 0u ? score : -INFINITY;
          next             = fmaxf(next, s[i][j]);
        }
#pragma unroll
        for (int o = 8; o > 0; o /= 2) { next = fmaxf(next, __shfl_xor_sync(kAllLanes, next, o)); }
        const float safe = finite_top(next), keep = power_of_2(top[i] - safe);
        top[i] = next;
        sum[i] *= keep;
#pragma unroll
        for (int q = 0; q < QUADS; q++) {
#pragma unroll
          for (int e = 0; e < 4; e++) { acc[i][q][e] *= keep; }
        }
#pragma unroll
        for (int j = 0; j < KEYS; j++) {
          const float p = power_of_2(s[i][j] - safe + shift);
          sum[i] += p;  // of the thread's own keys, until the end
          s_p[r * (TILE + 4) + x + 16 * j] = p;
        }
      }
      __syncthreads();
#pragma unroll 4
      for (int k = 0; k < TILE; k++) {
        float4 v[QUADS];
#pragma unroll
        for (int q = 0; q < QUADS; q++) { v[q] = *reinterpret_cast<const float4*>(s_v + k * PITCH + (x + 16 * q) * 4); }
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
          const float p = s_p[(y * ROWS + i) * (TILE + 4) + k];
          if (mixed && p == 0.0f) { continue; }  // what the row does not see may be infinite, or no number
#pragma unroll
          for (int q = 0; q < QUADS; q++) {
            acc[i][q][0] = fmaf(p, v[q].x, acc[i][q][0]);
            acc[i][q][1] = fmaf(p, v[q].y, acc[i][q][1]);
            acc[i][q][2] = fmaf(p, v[q].z, acc[i][q][2]);
            acc[i][q][3] = fmaf(p, v[q].w, acc[i][q][3]);
          }
        }
      }
      __syncthreads();
    }
    const uint32_t part = uint32_t(parts.part(which, block, now.begins ? 1u : 0u));
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
#pragma unroll
      for (int o = 8; o > 0; o /= 2) { sum[i] += __shfl_xor_sync(kAllLanes, sum[i], o); }
      const uint32_t r = y * ROWS + i;
      if (r >= rows) { continue; }
      const float scale = sum[i] == 0.0f ? 0.0f : 1.0f / sum[i];
#pragma unroll
      for (int q = 0; q < QUADS; q++) {
        const uint32_t quad = x + 16 * q;
        if (quad * 4 >= c.dim) { continue; }
        if (top[i] == -INFINITY) { acc[i][q][0] = acc[i][q][1] = acc[i][q][2] = acc[i][q][3] = 0.0f; }  // 0 times what is no number, of a row that saw nothing
        if (now.whole) {
          store_quad<T>(out_row<T>(t, now.sequence, head, row0 + r) + quad * 4,
                        make_float4(acc[i][q][0] * scale, acc[i][q][1] * scale, acc[i][q][2] * scale, acc[i][q][3] * scale));
        } else {
          parts.acc[(size_t(part) * parts.quads + quad) * BM + r] = make_float4(acc[i][q][0], acc[i][q][1], acc[i][q][2], acc[i][q][3]);
        }
      }
      if (x == 0) {
        if (now.whole) {
          *lse_at(t, now.sequence, head, c.n_heads, row0 + r) = (finite_top(top[i]) + log2f(sum[i]) - shift) * kLn2;
        } else {
          parts.stats[size_t(part) * BM + r] = make_float2(top[i], sum[i]);
        }
      }
    }
    if (now.begins && threadIdx.x == 0) { note_begun(parts, now, c.n_heads, which, begun); }
  }
  if (parts.begun != nullptr && !parts.by_unit && block == 0 && threadIdx.x == 0) { parts.begun[which] = begun; }
  empty_tree_rows<T>(c, w.n_sequences, lists, t, parts, threadIdx.x, kThreads);
}

// ---- few rows -----------------------------------------------------------------------------------------------------------------
//
// Where a unit has few rows the keys' and values' way through shared memory is what counts.  Warps work alone, each on chunks of 4 KB of keys and as
// much of values that it copies a stage ahead.  Scores: some lanes share a key, and each of its pieces is read once for all rows, whose queries are
// broadcast.  Sums: a lane has columns, and reads each value once for all rows, whose weights are broadcast.
//
// What bounds it: the instructions' latency, with twelve warps of an SM (six, whose chunks were twice as large: 92 us for 9 sequences of
// up to 9,000 + 5 tokens, 12 key heads of 64 columns, with a window, slopes and a filter; twelve 80, and 64 to 67 with the rows side by side; HBM asks for 18).

constexpr int kFewMost = 12;  // warps of a block, at most
struct few_lists : drafted_lists {
  static constexpr uint32_t kLeast = kFewMost;  // a chunk for each warp
};

template <int D, int R>
struct few_shape {
  static constexpr int kKeys   = 1024 / D;   // of a chunk
  static constexpr int kParts  = 32 / kKeys; // lanes of a key
  static constexpr int kPitch  = D + 4 * kParts;  // floats: eight lanes' pieces on different banks
  static constexpr int kStage  = 2 * kKeys * kPitch;
  static constexpr int kOwn    = 2 * kStage + R * kKeys * 2;  // of a warp: two stages, weights (each twice)
  static constexpr int kFit    = (232448 / 4 - 64 - R * D) / kOwn;  // (64: what found_piece takes)
  static constexpr int kWarps  = kFit < kFewMost ? kFit : kFewMost;
  static constexpr int kQAt    = kWarps * kOwn;
  static constexpr int kShared = (kQAt + R * D) * 4;
  static constexpr int kColumns = D / 32;    // of a lane
  static_assert(kShared + int(sizeof(found_piece)) <= 232448 && sizeof(found_piece) <= 256 && R * (D + 2) <= kOwn, "");
};

template <int D, int R>
__global__ void __launch_bounds__(few_shape<D, R>::kWarps * 32, 1)
tree_few_kernel(cache_view c, work_view w, few_lists lists, tree_view t, tree_parts parts, const int32_t* pages, int64_t table_stride, float shift)
{
  using shape = few_shape<D, R>;
  constexpr int KEYS = shape::kKeys, PARTS = shape::kParts, PITCH = shape::kPitch, COLUMNS = shape::kColumns, PIECES = D / 4, WARPS = shape::kWarps;
  chain_begin();
  extern __shared__ __align__(16) float s_mem[];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  float* s_own = s_mem + warp * shape::kOwn;
  float* s_p   = s_own + 2 * shape::kStage;
  float* s_q   = s_mem + shape::kQAt;
  const uint32_t which = blockIdx.x / t.n_blocks_of, block = blockIdx.x - which * t.n_blocks_of;
  const uint32_t row0 = block * R, rows = min(uint32_t(R), t.n_rows - row0);
  const uint32_t pieces = c.dim / 4, key_of = lane / PARTS, part_of = lane % PARTS;

  walk<KEYS, few_lists> path(c, w, lists, parts.shares, which);
  piece now;
  uint4 begun = make_uint4(0, 0, 0, 0);
  __shared__ found_piece s_found;
  drafted_lists::list l;
  while (next_piece(path, s_found, now, l)) {
    const uint32_t head         = now.unit;
    const int32_t* table        = pages + int64_t(now.sequence) * table_stride;
    const int32_t* positions    = t.positions + int64_t(now.sequence) * t.positions_stride;
    const char* keys            = c.keys + int64_t(head) * c.k_head * 4;
    const char* values          = c.values + int64_t(head) * c.v_head * 4;
    for (uint32_t i = threadIdx.x; i < uint32_t(R * PIECES); i += WARPS * 32) {
      const uint32_t r = i / PIECES, p = i - r * PIECES;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (r < rows && p < pieces) {
        const uint32_t token = (row0 + r) / t.group, g = row0 + r - token * t.group;
        x = reinterpret_cast<const uint4*>(t.queries.data + (int64_t(now.sequence) * t.queries.sequence + int64_t(token) * t.queries.token +
                                                             int64_t(head * t.group + g) * t.queries.head) * 4)[p];
      }
      reinterpret_cast<uint4*>(s_q)[i] = x;
    }
    // lane r looks after row r: its position, its slope, its row of the mask
    const uint32_t my_row = row0 + min(lane, rows - 1u), my_token = my_row / t.group;
    const int32_t my_at   = positions[my_token];
    const bool my_is      = lane < rows && my_at >= 0 && uint32_t(my_at) >= l.length;
    const float my_slope  = t.slopes != nullptr ? t.slopes[head * t.group + (my_row - my_token * t.group)] * kLog2E : 0.0f;
    const uint32_t* my_mask = t.mask + int64_t(now.sequence) * t.mask_sequence + int64_t(my_token) * t.mask_token;
    int32_t latest = 0;
    if (t.window > 0) {
      for (uint32_t i = lane; i < t.n_drafted; i += 32) { latest = max(latest, positions[i]); }
      latest = __reduce_max_sync(kAllLanes, latest);
    }
    float top[R], sum[R];
    two acc[R][COLUMNS / 2];
#pragma unroll
    for (int r = 0; r < R; r++) {
      top[r] = -INFINITY;
      sum[r] = 0.0f;
#pragma unroll
      for (int e = 0; e < COLUMNS / 2; e++) { acc[r][e] = two(0.0f, 0.0f); }
    }
    __syncthreads();

    // what memory says about this lane's key of a chunk
    auto look = [&](uint32_t chunk, uint32_t& k_at, uint32_t& v_at) -> bool {
      const uint32_t at = l.base + chunk * KEYS + lane;
      if (lane >= uint32_t(KEYS) || chunk >= now.end || at < l.first || at >= l.end) { return false; }
      uint32_t column, place;
      split_place(at, c.page, column, place);
      const int32_t page = table[column];  // at < end: the column is inside the table
      if (page < 0 || page >= c.n_pages) { return false; }
      k_at = uint32_t(page) * c.k_page_units + place * c.k_token_units;
      v_at = uint32_t(page) * c.v_page_units + place * c.v_token_units;
      if (c.filter != nullptr) {
        const uint64_t slot = uint64_t(page) * c.page.size + place;
        if (((c.filter[slot >> 5] >> (slot & 31u)) & 1u) == 0u) { return false; }
      }
      if (at >= l.length) {
        const int32_t of = positions[at - l.length];
        return of >= 0 && uint32_t(of) >= l.length;
      }
      return true;
    };
    // copies of the rows that are there; the others are 0
    auto copy = [&](uint32_t stage, bool there, uint32_t k_at, uint32_t v_at) -> uint32_t {
      const uint32_t valid = __ballot_sync(kAllLanes, there);
      const uint32_t to    = shared_address(s_own + stage * shape::kStage);
#pragma unroll 4
      for (uint32_t i = 0; i < uint32_t(KEYS * PIECES / 32); i++) {
        const uint32_t index = i * 32 + lane, row = index / PIECES, p = index % PIECES;
        const uint32_t bytes = p < pieces && ((valid >> row) & 1u) != 0u ? 16u : 0u, from = p < pieces ? p * 16 : 0u;
        const uint32_t k = __shfl_sync(kAllLanes, k_at, row), v = __shfl_sync(kAllLanes, v_at, row);
        copy_piece(to + (row * PITCH + p * 4) * 4, keys + (uint64_t(k) << c.unit_shift) + from, bytes);
        copy_piece(to + ((KEYS + row) * PITCH + p * 4) * 4, values + (uint64_t(v) << c.unit_shift) + from, bytes);
      }
      copies_end_group();
      return valid;
    };
    uint32_t k_at = 0, v_at = 0, chunk = now.chunk + warp;
    bool there      = look(chunk, k_at, v_at);
    uint32_t valid  = chunk < now.end ? copy(0, there, k_at, v_at) : 0u;
    k_at = v_at     = 0;
    there           = look(chunk + WARPS, k_at, v_at);
    for (uint32_t stage = 0; chunk < now.end; chunk += WARPS, stage ^= 1u) {
      const uint32_t next_valid = copy(stage ^ 1u, there, k_at, v_at);
      k_at = v_at = 0;
      there       = look(chunk + 2 * WARPS, k_at, v_at);
      copies_wait<1>();
      __syncwarp();
      const float* s_k     = s_own + stage * shape::kStage;
      const float* s_v     = s_k + KEYS * PITCH;
      const uint32_t base  = l.base + chunk * KEYS;
      const bool mixed     = int64_t(base) + KEYS > int64_t(l.length) || (t.window > 0 && int64_t(base) <= int64_t(latest) - t.window);
      uint32_t seen        = my_is ? valid : 0u;
      if (mixed && my_is) { seen &= seen_keys(t, l, positions, my_at, my_mask, base); }
      float s[R];
      two s2[R];
#pragma unroll
      for (int r = 0; r < R; r++) { s2[r] = two(0.0f, 0.0f); }
#pragma unroll 4
      for (int d = 0; d < D; d += 4 * PARTS) {
        const float4 k = *reinterpret_cast<const float4*>(s_k + key_of * PITCH + d + part_of * 4);
#pragma unroll
        for (int r = 0; r < R; r++) {
          const float4 q = *reinterpret_cast<const float4*>(s_q + r * D + d + part_of * 4);
          s2[r]          = fma2(two(q.x, q.y), two(k.x, k.y), s2[r]);
          s2[r]          = fma2(two(q.z, q.w), two(k.z, k.w), s2[r]);
        }
      }
#pragma unroll
      for (int r = 0; r < R; r++) {
        float u, v;
        s2[r].get(u, v);
        s[r] = u + v;
#pragma unroll
        for (int o = 1; o < PARTS; o *= 2) { s[r] += __shfl_xor_sync(kAllLanes, s[r], o); }
      }
      // (all rows side by side: those that are none see nothing)
#pragma unroll
      for (int r = 0; r < R; r++) { s[r] = t.cap_log2 != 0.0f ? tanhf(s[r] * t.scale_cap) * t.cap_log2 : s[r] * t.scale_log2; }
      if (t.slopes != nullptr) {
        int32_t of = int32_t(base + key_of);  // the key's position
        if (mixed && base + key_of >= l.length && base + key_of - l.length < t.n_drafted) { of = positions[base + key_of - l.length]; }
#pragma unroll
        for (int r = 0; r < R; r++) {
          s[r] = fmaf(__shfl_sync(kAllLanes, my_slope, r), float(int64_t(of) - __shfl_sync(kAllLanes, my_at, r)), s[r]);
        }
      }
      float next[R];
#pragma unroll
      for (int r = 0; r < R; r++) {
        const uint32_t sees = __shfl_sync(kAllLanes, seen, r);
        s[r]                = ((sees >> key_of) & 1u) != 0u ? s[r] : -INFINITY;
        next[r]             = fmaxf(s[r], top[r]);
      }
#pragma unroll
      for (int o = PARTS; o < 32; o *= 2) {
#pragma unroll
        for (int r = 0; r < R; r++) { next[r] = fmaxf(next[r], __shfl_xor_sync(kAllLanes, next[r], o)); }
      }
      bool higher = false;
#pragma unroll
      for (int r = 0; r < R; r++) { higher = higher || next[r] != top[r]; }
      if (higher) {  // of the whole warp
#pragma unroll
        for (int r = 0; r < R; r++) {
          const float keep = power_of_2(top[r] - finite_top(next[r]));
          top[r]           = next[r];
          sum[r] *= keep;
#pragma unroll
          for (int e = 0; e < COLUMNS / 2; e++) { acc[r][e] = mul2(acc[r][e], two(keep, keep)); }
        }
      }
#pragma unroll
      for (int r = 0; r < R; r++) {
        const float p = power_of_2(s[r] - finite_top(top[r]) + shift);
        if (part_of == 0) {
          sum[r] += p;  // of the lane's own keys, until the end
          reinterpret_cast<float2*>(s_p)[r * KEYS + key_of] = make_float2(p, p);
        }
      }
      __syncwarp();
#pragma unroll 2
      for (int k = 0; k < KEYS; k += 4) {
        two v[4][COLUMNS / 2];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float* row = s_v + (k + i) * PITCH;
          if constexpr (COLUMNS == 2) {
            const float2 x = *reinterpret_cast<const float2*>(row + lane * 2);
            v[i][0]        = two(x.x, x.y);
          } else {
#pragma unroll
            for (int e = 0; e < COLUMNS; e += 4) {
              const float4 x  = *reinterpret_cast<const float4*>(row + e * 32 + lane * 4);
              v[i][e / 2]     = two(x.x, x.y);
              v[i][e / 2 + 1] = two(x.z, x.w);
            }
          }
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
          const float4* p4 = reinterpret_cast<const float4*>(s_p + (r * KEYS + k) * 2);
          const float4 a = p4[0], b = p4[1];
          const two p[4] = {two(a.x, a.y), two(a.z, a.w), two(b.x, b.y), two(b.z, b.w)};
          if (!mixed) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
              for (int e = 0; e < COLUMNS / 2; e++) { acc[r][e] = fma2(p[i], v[i][e], acc[r][e]); }
            }
          } else {  // what a row does not see may be infinite, or no number
            const float weight[4] = {a.x, a.z, b.x, b.z};
#pragma unroll
            for (int i = 0; i < 4; i++) {
              if (weight[i] == 0.0f) { continue; }
#pragma unroll
              for (int e = 0; e < COLUMNS / 2; e++) { acc[r][e] = fma2(p[i], v[i][e], acc[r][e]); }
            }
          }
        }
      }
      __syncwarp();
      valid = next_valid;
    }
    copies_wait<0>();
    __syncwarp();
    // the warps' sums, in the place of their stages: top, sum, columns
#pragma unroll
    for (int r = 0; r < R; r++) {
#pragma unroll
      for (int o = 16; o > 0; o /= 2) { sum[r] += __shfl_xor_sync(kAllLanes, sum[r], o); }
      float* mine = s_own + r * (D + 2);
      if (lane == 0) {
        mine[0] = top[r];
        mine[1] = sum[r];
      }
#pragma unroll
      for (int e = 0; e < COLUMNS; e += 2) {
        float u, v;
        acc[r][e / 2].get(u, v);
        float* at = mine + 2 + (COLUMNS == 2 ? lane * 2 : (e / 4) * 128 + lane * 4 + e % 4);
        at[0]     = u;
        at[1]     = v;
      }
    }
    __syncthreads();
    const size_t part = parts.part(which, block, now.begins ? 1u : 0u);
    for (uint32_t i = threadIdx.x; i < rows * pieces; i += WARPS * 32) {
      const uint32_t r = i / pieces, quad = i - r * pieces;
      float most = -INFINITY;
#pragma unroll
      for (int v = 0; v < WARPS; v++) { most = fmaxf(most, s_mem[v * shape::kOwn + r * (D + 2)]); }
      const float safe = finite_top(most);
      float total = 0.0f, x[4] = {};
#pragma unroll
      for (int v = 0; v < WARPS; v++) {
        const float* of = s_mem + v * shape::kOwn + r * (D + 2);
        const float f   = power_of_2(of[0] - safe);
        total           = fmaf(of[1], f, total);
        if (of[0] == -INFINITY) { continue; }
#pragma unroll
        for (int e = 0; e < 4; e++) { x[e] = fmaf(of[2 + quad * 4 + e], f, x[e]); }
      }
      if (now.whole) {
        const float scale = total == 0.0f ? 0.0f : 1.0f / total;
        store_quad<float>(out_row<float>(t, now.sequence, head, row0 + r) + quad * 4, make_float4(x[0] * scale, x[1] * scale, x[2] * scale, x[3] * scale));
        if (quad == 0) { *lse_at(t, now.sequence, head, c.n_heads, row0 + r) = (safe + log2f(total) - shift) * kLn2; }
      } else {
        parts.acc[(part * parts.quads + quad) * parts.rows + r] = make_float4(x[0], x[1], x[2], x[3]);
        if (quad == 0) { parts.stats[part * parts.rows + r] = make_float2(most, total); }
      }
    }
    if (now.begins && threadIdx.x == 0) { note_begun(parts, now, c.n_heads, which, begun); }
  }
  if (parts.begun != nullptr && !parts.by_unit && block == 0 && threadIdx.x == 0) { parts.begun[which] = begun; }
  empty_tree_rows<float>(c, w.n_sequences, lists, t, parts, threadIdx.x, WARPS * 32);
}

// Rows of a block of the kernel for few, by how many a unit has.
constexpr uint32_t few_rows_of(uint32_t n_rows, uint32_t dim) { return n_rows <= 4 ? 4 : n_rows <= 8 || dim > 128 ? 8 : 16; }
// Which kernel: 4 sequences of 20,000 tokens, 2 key heads, us by warps alone and in tiles of 64 rows: 64 columns 16 rows 46 and 67, 32 rows 68 and 68;
// 128 columns 16 rows 83 and 117, 32 rows 145 and 117; 256 columns 32 rows 222 and 260, 40 rows 273 and 260.  With a window of 4,000 (9 of 9,000, 12 heads)
// 16 rows 155 and 251, 334 and 484, 256 columns 32 rows 1,014 and 1,096.  Of many short units (40 of 306 tokens, 8 heads) 16 rows 66 and 75, 119 and 138, 256
// columns 24 rows 259 and 287 but 32 rows 338 and 291; 300 of 100 tokens 16 rows 120 and 113, 224 and 216, 256 columns 32 rows 603 and 470.
constexpr bool is_few(uint32_t n_rows, uint32_t dim) { return n_rows <= (dim <= 128 ? 16u : 32u); }

tree_plan plan_of(const resources& res, elem type, uint64_t sequences, uint32_t n_drafted, uint32_t n_heads, uint32_t group, uint32_t dim,
                  uint64_t capacity, int64_t window)
{
  const uint32_t n_rows = n_drafted * group, sms = uint32_t(res.sm_count);
  // the keys of the longest list: a window may begin anywhere in 16 positions
  const uint64_t most = window > 0 && uint64_t(window) < capacity ? std::min(capacity, uint64_t(window) + n_drafted + 15) : capacity;
  if (type == elem::f32) {
    const uint32_t columns = tree_columns(dim);
    if (is_few(n_rows, dim)) { return deal_out_tree(sms, few_rows_of(n_rows, dim), 1024 / columns, 24, few_lists::kLeast, sequences * n_heads, n_rows, most); }
    return deal_out_tree(sms * tree_resident(int(columns)), 64, columns <= 128 ? 64 : 32, 2, drafted_lists::kLeast, sequences * n_heads, n_rows, most);
  }
  tree_plan p  = deal_out_tree(sms, dim <= 128 && n_rows > 128 ? 256 : 128, 64, 2, drafted_lists::kLeast, sequences * n_heads, n_rows, most);
  p.sets_aside = most > kChain / 2 * p.tile;  // (the second stream's first turn comes half way)
  return p;
}
// Of a plan's parts, and of what its blocks set aside: rows of two streams of 128, one of more than 128 columns.
size_t part_bytes_of(const tree_plan& p, uint32_t dim) { return p.parts ? tree_part_bytes(p.shares, p.blocks_of, p.rows, dim) : 0; }
size_t aside_bytes_of(const tree_plan& p, uint32_t dim)
{
  return p.sets_aside ? size_t(p.shares) * p.blocks_of * (dim <= 128 ? 256 : 128) * dim * sizeof(float) : 0;
}

// Waits of the kernel on tensor cores (tests make one run out).
std::atomic<uint32_t> g_wait_limit{kSpinLimit}, g_skip_tile{0};

}  // namespace

void set_tree_wait_test(uint32_t limit, uint32_t skip_tile)
{
  g_wait_limit = limit != 0u ? limit : kSpinLimit;
  g_skip_tile  = skip_tile;
}

size_t attend_tree_workspace(const resources& res, elem type, uint32_t n_sequences, uint32_t n_drafted, uint32_t n_query_heads, uint32_t n_heads,
                             uint32_t dim, uint64_t capacity, int64_t window)
{
  if (n_sequences == 0) { return 0; }
  const tree_plan p = plan_of(res, type, n_sequences, n_drafted, n_heads, n_query_heads / n_heads, dim, capacity, window);
  return part_bytes_of(p, dim) + aside_bytes_of(p, dim);
}

void attend_tree(resources& res, cudaStream_t stream, const attend_tree_args& a)
{
  if (a.n_sequences == 0) { return; }
  const cache_view& c     = a.cache;
  const uint32_t group    = a.n_query_heads / c.n_heads;
  const uint64_t capacity = uint64_t(a.table_width) * c.page.size, units = uint64_t(a.n_sequences) * c.n_heads;
  const tree_plan p       = plan_of(res, a.type, a.n_sequences, a.n_drafted, c.n_heads, group, c.dim, capacity, a.window);
  tree_call call{};
  call.c             = c;
  call.plan          = p;
  call.pages         = a.pages;
  call.table_stride  = a.table_stride;
  call.report        = a.report;
  call.limit         = g_wait_limit;
  call.skip_tile     = g_skip_tile;
  tree_view& t       = call.t;
  t.n_drafted        = a.n_drafted;
  t.group            = group;
  t.n_rows           = a.n_drafted * group;
  t.n_blocks_of      = p.blocks_of;
  t.lengths          = a.lengths;
  t.positions        = a.positions;
  t.positions_stride = a.positions_stride;
  t.mask             = a.mask;
  t.mask_sequence    = a.mask_sequence;
  t.mask_token       = a.mask_token;
  t.slopes           = a.slopes;
  t.window           = a.window;
  t.queries          = a.queries;
  t.out              = a.out;
  t.lse              = a.lse;
  t.scale_log2       = a.scale * kLog2E;
  t.scale_cap        = a.cap != 0.0f ? a.scale / a.cap : 0.0f;
  t.cap_log2         = a.cap * kLog2E;
  for (int i = 0; i < 5; i++) { t.cap_near[i] = t.cap_log2 * kTanh[i]; }
  call.lists         = {a.lengths, a.window, a.table_width, a.n_drafted};
  call.w             = {a.n_sequences, c.n_heads, 1, group, 0, p.cost};
  make_room(call.w, capacity);
  // room for the sum of a whole list, and for weights above 1 where a top may be behind; the weights of 16-bit floats have their own (kv_tree_tc.cuh)
  call.shift = a.type == elem::f32 ? std::log2(call.w.room) : a.type == elem::bf16 ? std::log2(call.w.room) - 4.0f : 11.0f;
  if (p.parts) { call.parts = tree_parts_at(a.workspace, p.shares, p.blocks_of, p.rows, c.dim, units); }
  call.parts.shares    = p.shares;
  call.parts.blocks_of = p.blocks_of;
  call.parts.rows      = p.rows;
  if (p.sets_aside) { call.aside = reinterpret_cast<float4*>(a.workspace + part_bytes_of(p, c.dim)); }
  count_launches(res, p.parts ? 2 : 1);

  auto join = [&](auto type) {
    if (p.parts) { launch_tree_join<decltype(type)>(stream, p, units, t, call.parts, c.dim, c.n_heads, call.shift); }
  };
  if (a.type == elem::f16) {
    attend_tree16<__half>(stream, call);
    return join(__half{});
  }
  if (a.type == elem::bf16) {
    attend_tree16<__nv_bfloat16>(stream, call);
    return join(__nv_bfloat16{});
  }
  auto go = [&](auto kernel, const auto& lists, int threads, size_t smem) {
    ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
    launch_chained(kernel, dim3(p.shares * p.blocks_of), threads, smem, stream, c, call.w, lists, t, call.parts, a.pages, a.table_stride, call.shift);
  };
  auto by_columns = [&](auto columns) {
    constexpr int D = decltype(columns)::value;
    if (!is_few(t.n_rows, c.dim)) { return go(tree_rows_kernel<D>, call.lists, kThreads, tree_shape<D>::kShared); }
    if (p.rows == 4) { return go(tree_few_kernel<D, 4>, few_lists{call.lists}, few_shape<D, 4>::kWarps * 32, few_shape<D, 4>::kShared); }
    if (p.rows == 8) { return go(tree_few_kernel<D, 8>, few_lists{call.lists}, few_shape<D, 8>::kWarps * 32, few_shape<D, 8>::kShared); }
    if constexpr (D <= 128) { go(tree_few_kernel<D, 16>, few_lists{call.lists}, few_shape<D, 16>::kWarps * 32, few_shape<D, 16>::kShared); }
  };
  using std::integral_constant;
  switch (tree_columns(c.dim)) {
    case 64: by_columns(integral_constant<int, 64>{}); break;
    case 128: by_columns(integral_constant<int, 128>{}); break;
    default: by_columns(integral_constant<int, 256>{});
  }
  join(float{});
}

}  // namespace cuvs_b200::kv
