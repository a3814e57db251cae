// Attention of drafted tokens to the rows of their sequences in a paged cache, with 32-bit products (the mathematics: kv_tree.cuh).
#include "kv_tree.cuh"

#include <algorithm>
#include <type_traits>

namespace cuvs_b200::kv {

namespace {

constexpr int kThreads = 256;

// Blocks of an SM: what shared memory and registers leave room for.  They hide each other's loads.
constexpr int tree_resident(int columns, int rows) { return columns == 64 ? (rows == 16 ? 4 : 3) : columns == 128 ? (rows == 16 ? 2 : 1) : rows == 16 ? 2 : 1; }

// D: columns of a row in shared memory; BM: rows of a block.  Threads stand in 16 x 16: thread (y, x) has BM / 16 rows, their scores with every 16th key
// and their weighted sums in every 16th four columns.
template <int D, int BM>
struct tree_shape {
  static constexpr int kTile  = D <= 128 ? 64 : 32;
  static constexpr int kRows  = BM / 16;    // of a thread
  static constexpr int kKeys  = kTile / 16;
  static constexpr int kQuads = D / 64;
  static constexpr int kPitch = D + 4;      // floats: 16 lanes' quads of different rows on different banks
  static constexpr int kKAt   = BM * kPitch;
  static constexpr int kVAt   = kKAt + kTile * kPitch;
  static constexpr int kPAt   = kVAt + kTile * kPitch;
  static constexpr int kSeenAt = kPAt + BM * (kTile + 4);
  static constexpr int kValidAt = kSeenAt + BM * (kTile / 32);
  static constexpr int kPlaceAt = kValidAt + 4;
  static constexpr int kShared = (kPlaceAt + 3 * kTile) * 4;
  static constexpr int kResident = tree_resident(D, BM);
  static_assert(kResident * (kShared + 1024) <= 233472, "");
};

template <typename T, int D, int BM>
__global__ void __launch_bounds__(kThreads, tree_shape<D, BM>::kResident)
tree_rows_kernel(cache_view c, work_view w, drafted_lists lists, tree_view t, tree_parts parts, const int32_t* pages, int64_t table_stride, float shift)
{
  using shape = tree_shape<D, BM>;
  constexpr int TILE = shape::kTile, ROWS = shape::kRows, KEYS = shape::kKeys, QUADS = shape::kQuads, PITCH = shape::kPitch, E = kPerPiece<T>;
  chain_begin();
  extern __shared__ __align__(16) float s_mem[];
  float* s_q        = s_mem;
  float* s_k        = s_mem + shape::kKAt;
  float* s_v        = s_mem + shape::kVAt;
  float* s_p        = s_mem + shape::kPAt;
  uint32_t* s_seen  = reinterpret_cast<uint32_t*>(s_mem + shape::kSeenAt);
  uint32_t* s_valid = reinterpret_cast<uint32_t*>(s_mem + shape::kValidAt);
  uint32_t* s_k_at  = reinterpret_cast<uint32_t*>(s_mem + shape::kPlaceAt);
  uint32_t* s_v_at  = s_k_at + TILE;
  int32_t* s_of     = reinterpret_cast<int32_t*>(s_v_at + TILE);  // the keys' positions
  const uint32_t y = threadIdx.x / 16, x = threadIdx.x % 16;
  const uint32_t which = blockIdx.x / t.n_blocks_of, block = blockIdx.x - which * t.n_blocks_of;
  const uint32_t row0 = block * BM, rows = min(uint32_t(BM), t.n_rows - row0);
  const uint32_t pieces = c.dim / E;

  walk<TILE, drafted_lists> path(c, w, lists, parts.shares, which);
  piece now;
  uint4 begun = make_uint4(0, 0, 0, 0);
  while (__syncthreads_and(path.next(now)) != 0) {
    const drafted_lists::list l = path.l;
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

    for (uint32_t tile = now.chunk; tile < now.end; tile++) {
      const uint32_t base = l.base + tile * TILE;
      const bool mixed    = int64_t(base) + TILE > int64_t(l.length) || (t.window > 0 && int64_t(base) <= int64_t(latest) - t.window);
      if (threadIdx.x < TILE) {
        const uint32_t at = base + threadIdx.x;
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
        s_k_at[threadIdx.x] = there ? uint32_t(page) * c.k_page_units + place * c.k_token_units : 0u;
        s_v_at[threadIdx.x] = there ? uint32_t(page) * c.v_page_units + place * c.v_token_units : 0u;
        s_of[threadIdx.x]   = of;
        const uint32_t word = __ballot_sync(kAllLanes, there);
        if ((threadIdx.x & 31u) == 0) { s_valid[threadIdx.x / 32] = word; }
      }
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < uint32_t(TILE * (D / E)); i += kThreads) {
        const uint32_t k = i / (D / E), p = i - k * (D / E);
        const bool there = p < pieces && ((s_valid[k / 32] >> (k & 31u)) & 1u) != 0u;
        const char* from = c.keys + int64_t(head) * c.k_head * int64_t(sizeof(T)) + (uint64_t(s_k_at[k]) << c.unit_shift) + (there ? p * 16 : 0);
        float f[E];
        piece_to_floats<T>(load_piece(from, there), f);
#pragma unroll
        for (int e = 0; e < E; e++) { s_k[k * PITCH + p * E + e] = f[e]; }
        from = c.values + int64_t(head) * c.v_head * int64_t(sizeof(T)) + (uint64_t(s_v_at[k]) << c.unit_shift) + (there ? p * 16 : 0);
        piece_to_floats<T>(load_piece(from, there), f);
#pragma unroll
        for (int e = 0; e < E; e++) { s_v[k * PITCH + p * E + e] = f[e]; }
      }
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
          score            = fmaf(slope[i], float(int64_t(s_of[k]) - own[i]), score);
          s[i][j]          = ((s_seen[r * (TILE / 32) + k / 32] >> (k & 31u)) & 1u) != 0u ? score : -INFINITY;
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

tree_plan plan_of(const resources& res, elem type, uint64_t sequences, uint32_t n_drafted, uint32_t n_heads, uint32_t group, uint32_t dim,
                  uint64_t capacity, int64_t window)
{
  const uint32_t n_rows = n_drafted * group, sms = uint32_t(res.sm_count);
  // the keys of the longest list: a window may begin anywhere in 16 positions
  const uint64_t most = window > 0 && uint64_t(window) < capacity ? std::min(capacity, uint64_t(window) + n_drafted + 15) : capacity;
  if (type == elem::f32) {
    const int rows = n_rows <= 16 ? 16 : 64;
    return deal_out_tree(sms * tree_resident(int(tree_columns(dim)), rows), n_rows <= 16 ? 16 : 64, dim <= 128 ? 64 : 32, 2, sequences * n_heads, n_rows, most);
  }
  return deal_out_tree(sms, dim <= 128 && n_rows > 128 ? 256 : 128, 64, 2, sequences * n_heads, n_rows, most);
}

}  // namespace

size_t attend_tree_workspace(const resources& res, elem type, uint32_t n_sequences, uint32_t n_drafted, uint32_t n_query_heads, uint32_t n_heads,
                             uint32_t dim, uint64_t capacity, int64_t window)
{
  if (n_sequences == 0) { return 0; }
  const tree_plan p = plan_of(res, type, n_sequences, n_drafted, n_heads, n_query_heads / n_heads, dim, capacity, window);
  return p.parts ? tree_part_bytes(p.shares, p.blocks_of, p.rows, dim) : 0;
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
  call.timeouts      = res.pinned + 14;
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
  auto go = [&](auto columns, auto bm) {
    constexpr int D = decltype(columns)::value, BM = decltype(bm)::value;
    auto kernel = tree_rows_kernel<float, D, BM>;
    constexpr size_t smem = tree_shape<D, BM>::kShared;
    ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
    launch_chained(kernel, dim3(p.shares * p.blocks_of), kThreads, smem, stream, c, call.w, call.lists, t, call.parts, a.pages, a.table_stride,
                   call.shift);
  };
  using std::integral_constant;
  auto by_rows = [&](auto columns) {
    if (p.rows == 16) {
      go(columns, integral_constant<int, 16>{});
    } else {
      go(columns, integral_constant<int, 64>{});
    }
  };
  switch (tree_columns(c.dim)) {
    case 64: by_rows(integral_constant<int, 64>{}); break;
    case 128: by_rows(integral_constant<int, 128>{}); break;
    default: by_rows(integral_constant<int, 256>{});
  }
  join(float{});
}

}  // namespace cuvs_b200::kv
