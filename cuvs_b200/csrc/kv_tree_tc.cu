// Attention of drafted tokens to the 16-bit rows of their sequences in a paged cache, on tensor cores (the mathematics: kv_tree.cuh).
//
// A block has 128 query rows, or twice 128, and goes through its share's tiles of 128 keys (64 where rows have more than 128 columns).  One warp issues
// tcgen05.mma: scores S = Q K^T into tensor memory; four warps of 32 rows each, a thread a row, read them, carry the softmax (top and sum in 32
// bits) and write the weights back over them as two 16-bit numbers; the same warp issues O += P V with P from tensor memory.  Four more
// warps copy rows of keys and values, 16 bytes at a time, into a ring of tiles, in the order in which they are wanted, and one finds the way through the
// share.  Two streams of tiles keep the tensor core busy while one of them is at its softmax: the two halves of 256 rows on the same tiles, or even
// and odd tiles of the same 128 rows, whose sums are joined at a unit's end.  Rows of more than 128 columns leave tensor memory room for one
// sum only: there the scores of two tiles take turns.
//
// Sums are brought to a new top only where it is 2^4 above the old one: a turn through tensor memory that few tiles need.
#include "kv_tree_tc.cuh"

#include <algorithm>
#include <type_traits>

namespace cuvs_b200::kv {

namespace {

constexpr int kThreads    = 512;  // two softmax groups, four warps that copy, one that multiplies, one that finds the way
constexpr int kInfos      = 8;    // tiles whose descriptions are kept
constexpr int kPieces     = 2;
constexpr int kReaders    = 13;   // warps that read a piece's description
constexpr uint32_t kLimit = kSpinLimit;

template <int D>
struct tc_shape {
  static constexpr bool kTwo      = D <= 128;
  static constexpr int kTile      = kTwo ? 128 : 64;
  static constexpr int kRows      = kTwo ? 256 : 128;  // of a block, at most
  static constexpr int kPanel     = kTile * 128;       // bytes of 64 columns of a tile
  static constexpr int kTileBytes = kPanel * (D / 64);
  static constexpr int kQPanel    = 128 * 128;
  static constexpr int kQBytes    = kQPanel * (D / 64);
  static constexpr int kExchange  = kQBytes;  // where two groups exchange sums: behind the first 128 rows
  static constexpr int kQRegion   = !kTwo ? kQBytes : 2 * kQBytes > kQBytes + 32768 ? 2 * kQBytes : kQBytes + 32768;
  static constexpr int kMisc      = 3072;
  static constexpr int kStages    = (232448 - kQRegion - kMisc) / kTileBytes < 10 ? (232448 - kQRegion - kMisc) / kTileBytes : 10;
  static constexpr int kBehind    = kStages - 2;  // tiles in flight: one more would wait for what waits for it
  static constexpr int kRingAt    = kQRegion;
  static constexpr int kMiscAt    = kRingAt + kStages * kTileBytes;
  static constexpr int kShared    = kMiscAt + kMisc;
  static constexpr int kSumsAt    = 256;               // first column of the sums in tensor memory
  static_assert(kStages >= 4 && kShared <= 232448, "");
};

// A piece of a unit as the way through the share found it.
struct tree_piece {
  uint32_t sequence, head, chunk, end;
  uint32_t length, first, last, base;
  int32_t latest;
  uint32_t begins, whole;
};

struct tc_shared {
  uint64_t full[10], empty[10];
  uint64_t q_full, q_empty, s_full[2], p_full[2], o_full[2], pv_done, exchanged, drained;
  uint64_t piece_full[kPieces], piece_empty[kPieces];
  tree_piece pieces[kPieces];
  uint32_t valid[kInfos][4], bad[kInfos][4];
  float2 stats[2][128];
  uint32_t tmem, failed;
};
static_assert(sizeof(tc_shared) <= 3072, "");

struct tc_args {
  cache_view c;
  work_view w;
  drafted_lists lists;
  tree_view t;
  tree_parts parts;
  const int32_t* pages;
  int64_t table_stride;
  float shift;
  uint32_t* timeouts;
};

constexpr uint32_t kNoMore = 0xFFFFFFFFu;

// Waits with a limit, after which the block gives up; a whole warp at a time.
struct waiter {
  tc_shared& sh;
  __device__ __forceinline__ bool operator()(const uint64_t& bar, uint32_t parity) const
  {
    if (mbar_wait_warp(smem_u32(&bar), parity & 1u, kLimit)) { return true; }
    *const_cast<volatile uint32_t*>(&sh.failed) = 1u;
    return false;
  }
};

__device__ __forceinline__ void arrive_warp(uint64_t& bar)
{
  __syncwarp();
  if ((threadIdx.x & 31u) == 0u) { mbar_arrive(smem_u32(&bar)); }
}

struct piece_reader {
  uint32_t i = 0;
  __device__ __forceinline__ bool next(tc_shared& sh, const waiter& wait, tree_piece& p)
  {
    if (!wait(sh.piece_full[i % kPieces], i / kPieces)) { return false; }
    p = sh.pieces[i % kPieces];
    arrive_warp(sh.piece_empty[i % kPieces]);
    i++;
    return p.sequence != kNoMore;
  }
};

// Of a piece's 2 n tiles in the order in which they are copied and wanted -- K0 K1 V0 K2 V1 .. -- the place of tile j's values.
__device__ __forceinline__ uint32_t values_at(uint32_t j, uint32_t n) { return j + 1 < n ? 2 * j + 2 : 2 * n - 1; }

// Whether all rows that are there see all keys of the tile that are there.
template <int TILE>
__device__ __forceinline__ bool is_mixed(const tree_view& t, const tree_piece& p, uint32_t base)
{
  return int64_t(base) + TILE > int64_t(p.length) || (t.window > 0 && int64_t(base) <= int64_t(p.latest) - t.window);
}

// ---- copying ------------------------------------------------------------------------------------------------------------------

template <typename T, int D>
__device__ __forceinline__ void copy_role(const tc_args& a, tc_shared& sh, char* smem, const waiter& wait, uint32_t which, uint32_t block)
{
  using shape                = tc_shape<D>;
  constexpr uint32_t TILE    = shape::kTile, ROWS = TILE / 4, PR = D / 8, AT_ONCE = 32 / PR > 0 ? 32 / PR : 1, NB = shape::kStages, BEHIND = shape::kBehind;
  const cache_view& c        = a.c;
  const tree_view& t         = a.t;
  const uint32_t warp        = (threadIdx.x >> 5) & 3u, lane = threadIdx.x & 31u;
  const uint32_t piece       = lane % PR, sub = lane / PR;
  const uint32_t pieces      = c.dim / 8, wide = (pieces + 1) & ~1u;  // products take 16 columns at a time: those behind the row's end are 0
  const uint32_t ring        = smem_u32(smem + shape::kRingAt), q_at = smem_u32(smem);
  const uint32_t row0        = block * shape::kRows, rows = min(uint32_t(shape::kRows), t.n_rows - row0);
  const uint32_t column_from = piece < pieces ? piece * 16 : 0u;
  const uint32_t column_to   = (piece >> 3) * shape::kPanel;
  uint32_t it = 0, sent = 0, tiles = 0, q_turn = 0;
  uint64_t scan = 0;  // 4 bits for each place of the ring: 1 + which info, if the values there have to be looked at
  auto send = [&](uint32_t i) {
    const uint32_t slot = i % NB, info = uint32_t(scan >> (4 * slot)) & 15u;
    if (info != 0u) {
      bool bad = false;
      for (uint32_t r = sub; r < ROWS; r += AT_ONCE) {
        if (piece >= wide || sub >= AT_ONCE) { break; }
        const uint32_t row = warp * ROWS + r;
        const uint4 x = *reinterpret_cast<const uint4*>(smem + shape::kRingAt + slot * shape::kTileBytes + column_to + row * 128 +
                                                        (((piece & 7u) ^ (row & 7u)) << 4));
        constexpr uint32_t kAll = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
        const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          bad = bad || (words[e] & kAll) == kAll || ((words[e] >> 16) & kAll) == kAll;
        }
      }
      if (__any_sync(kAllLanes, bad) && lane == 0) { sh.bad[info - 1][warp] = 1u; }
      scan &= ~(uint64_t(15) << (4 * slot));
    }
    fence_async_smem();
    arrive_warp(sh.full[slot]);
  };
  auto flush = [&] {
    copies_wait<0>();
    for (; sent < it; sent++) { send(sent); }
  };
  // The rows of one tile, of which this lane knows the place of one.
  auto copy = [&](const char* from, uint32_t at, uint32_t there) -> bool {
    if (it >= NB && !wait(sh.empty[it % NB], it / NB - 1)) { return false; }
    const uint32_t to = ring + (it % NB) * shape::kTileBytes + column_to;
#pragma unroll
    for (uint32_t i = 0; i < ROWS / AT_ONCE; i++) {
      const uint32_t r = i * AT_ONCE + sub, row = warp * ROWS + r;
      const uint32_t place = __shfl_sync(kAllLanes, at, r);
      const uint32_t bytes = piece < pieces && ((there >> r) & 1u) != 0u ? 16u : 0u;
      if (piece < wide) { copy_piece(to + row * 128 + (((piece & 7u) ^ (row & 7u)) << 4), from + (uint64_t(place) << c.unit_shift), bytes); }
    }
    copies_end_group();
    it++;
    copies_wait<BEHIND>();
    if (it > BEHIND && sent < it - BEHIND) { send(sent++); }
    return true;
  };

  piece_reader reader;
  tree_piece p;
  while (reader.next(sh, wait, p)) {
    const uint32_t n        = p.end - p.chunk;
    const int32_t* table    = a.pages + int64_t(p.sequence) * a.table_stride;
    const int32_t* positions = t.positions + int64_t(p.sequence) * t.positions_stride;
    const char* keys        = c.keys + int64_t(p.head) * c.k_head * 2 + column_from;
    const char* values      = c.values + int64_t(p.head) * c.v_head * 2 + column_from;
    // queries: they may be replaced once the last scores of the piece before are there
    if (q_turn > 0) {
      flush();
      if (!wait(sh.q_empty, q_turn - 1)) { break; }
    }
    const uint32_t q_rows = rows <= 128 ? 128 : 256;
    for (uint32_t r0 = warp * 32; r0 < q_rows; r0 += 128) {
      const uint32_t mine = r0 + lane, r = row0 + min(mine, rows - 1u), token = r / t.group, g = r - token * t.group;
      const char* from = t.queries.data + (int64_t(p.sequence) * t.queries.sequence + int64_t(token) * t.queries.token +
                                           int64_t(p.head * t.group + g) * t.queries.head) * 2;
      for (uint32_t i = 0; i < 32; i += AT_ONCE) {
        const uint32_t row  = r0 + i + sub;
        const uint64_t at   = __shfl_sync(kAllLanes, reinterpret_cast<uint64_t>(from), (i + sub) & 31u);
        const uint32_t to   = q_at + (row >> 7) * shape::kQBytes + (piece >> 3) * shape::kQPanel + (row & 127u) * 128 + (((piece & 7u) ^ (row & 7u)) << 4);
        if (piece < wide) { copy_piece(to, reinterpret_cast<const char*>(at) + column_from, piece < pieces && row < rows ? 16u : 0u); }
      }
    }
    copies_end_group();
    copies_wait<0>();
    fence_async_smem();
    arrive_warp(sh.q_full);
    q_turn++;

    // what the table says about this lane's key of a tile, asked for a tile ahead
    const uint32_t own_row = warp * ROWS + lane % ROWS;
    auto name = [&](uint32_t tile) -> int32_t {
      const uint32_t at = p.base + tile * TILE + own_row;
      if (tile >= p.end || at < p.first || at >= p.last) { return -1; }
      uint32_t column, place;
      split_place(at, c.page, column, place);
      return table[column];  // at < last: the column is inside the table
    };
    int32_t next = name(p.chunk);
    uint32_t v_at = 0, v_there = 0;  // of the tile before
    bool ok = true;
    for (uint32_t j = 0; j <= n && ok; j++) {
      uint32_t k_at = 0, this_v_at = 0, this_there = 0;
      if (j < n) {
        const uint32_t base = p.base + (p.chunk + j) * TILE, at = base + own_row;
        const int32_t page  = next;
        next                = name(p.chunk + j + 1);
        uint32_t column, place;
        split_place(min(at, 0x7FFFFFFFu), c.page, column, place);
        bool there = page >= 0 && page < c.n_pages;
        if (there && c.filter != nullptr) {
          const uint64_t slot = uint64_t(page) * c.page.size + place;
          there               = ((c.filter[slot >> 5] >> (slot & 31u)) & 1u) != 0u;
        }
        if (there && at >= p.length) {
          const int32_t of = positions[at - p.length];
          there            = of >= 0 && uint32_t(of) >= p.length;
        }
        k_at       = there ? uint32_t(page) * c.k_page_units + place * c.k_token_units : 0u;
        this_v_at  = there ? uint32_t(page) * c.v_page_units + place * c.v_token_units : 0u;
        this_there = __ballot_sync(kAllLanes, there);
        const uint32_t info = tiles % kInfos;
        if (lane == 0) {
          sh.valid[info][warp] = ROWS == 32 ? this_there : this_there & 0xFFFFu;
          sh.bad[info][warp]   = 0u;
        }
        tiles++;
        ok = copy(keys, k_at, this_there);
      }
      // tile j's keys come before tile j - 1's values, which have been named together
      if (j > 0 && ok) {
        const uint32_t base = p.base + (p.chunk + j - 1) * TILE;
        if (is_mixed<TILE>(t, p, base)) {
          const uint32_t info = (tiles - (j < n ? 2 : 1)) % kInfos;
          scan |= uint64_t(info + 1) << (4 * (it % NB));
        }
        ok = copy(values, v_at, v_there);
      }
      v_at    = this_v_at;
      v_there = this_there;
    }
    if (!ok) { break; }
  }
  flush();
}

// ---- multiplying --------------------------------------------------------------------------------------------------------------

template <typename T, int D>
__device__ __forceinline__ void multiply_role(const tc_args& a, tc_shared& sh, char* smem, const waiter& wait, uint32_t block)
{
  using shape              = tc_shape<D>;
  constexpr uint32_t TILE  = shape::kTile, NB = shape::kStages;
  constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : 1u;
  const uint32_t tmem      = sh.tmem;
  const uint32_t rows      = min(uint32_t(shape::kRows), a.t.n_rows - block * shape::kRows);
  const bool both          = shape::kTwo && rows > 128;  // two blocks of rows on the same tiles
  const uint32_t steps     = (a.c.dim + 15) / 16;
  const uint32_t qk        = (1u << 4) | (kType << 7) | (kType << 10) | ((TILE >> 3) << 17) | ((128u >> 4) << 24);
  const uint32_t pv        = (1u << 4) | (kType << 7) | (kType << 10) | (1u << 16) | (((steps * 16) >> 3) << 17) | ((128u >> 4) << 24);
  const uint32_t q_at = smem_u32(smem), ring = smem_u32(smem + shape::kRingAt);
  auto scores_at = [&](uint32_t s) { return tmem + s * TILE; };
  auto sums_at   = [&](uint32_t s) { return tmem + shape::kSumsAt + (shape::kTwo ? s * 128 : 0); };
  auto scores = [&](uint32_t slot, uint32_t s) {
    const uint32_t from = ring + slot * shape::kTileBytes, q = q_at + (both ? s * shape::kQBytes : 0u);
    if (elect_one()) {
      for (uint32_t k = 0; k < steps; k++) {
        const uint32_t panel = k >> 2, in = (k & 3u) * 32;
        tc_mma_f16(scores_at(s), make_desc_sw128(q + panel * shape::kQPanel + in), make_desc_sw128(from + panel * shape::kPanel + in), qk, k != 0u);
      }
      tc_commit(smem_u32(&sh.s_full[s]));
    }
    __syncwarp();
  };
  auto sums = [&](uint32_t slot, uint32_t s, bool add) {
    const uint32_t from = ring + slot * shape::kTileBytes;
    if (elect_one()) {
#pragma unroll 1
      for (uint32_t part = 0; part < 2; part++) {
        for (uint32_t k = 0; k < TILE / 16; k++) {
          tc_mma_f16_ts(sums_at(s), scores_at(s) + part * (TILE / 2) + k * 8, make_desc_sw128_rows(from + k * 2048, shape::kPanel), pv,
                        add || (part | k) != 0u);
        }
      }
    }
    __syncwarp();
  };
  auto commit = [&](uint64_t& bar) {
    if (elect_one()) { tc_commit(smem_u32(&bar)); }
    __syncwarp();
  };

  piece_reader reader;
  tree_piece p;
  uint32_t it = 0, tiles = 0, q_turn = 0, p_turn[2] = {0, 0};
  auto next_full = [&](uint32_t& slot) {
    slot          = it % NB;
    const bool ok = wait(sh.full[slot], it / NB);
    it++;
    return ok;
  };
  while (reader.next(sh, wait, p)) {
    const uint32_t n = p.end - p.chunk;
    uint32_t slot;
    if (!wait(sh.q_full, q_turn++)) { break; }
    tc_fence_after();
    bool ok = true;
    // the first scores
    for (uint32_t s = 0; s < (both || n < 2 ? 1u : 2u) && ok; s++) {
      ok = next_full(slot);
      if (!ok) { break; }
      scores(slot, s);
      if (both) { scores(slot, 1); }
      commit(sh.empty[slot]);
    }
    if (n == 1 || (n == 2 && !both)) { commit(sh.q_empty); }
    for (uint32_t j = 0; j < n && ok; j++) {
      uint32_t k_slot = 0, v_slot = 0;
      const bool more = j + (both ? 1 : 2) < n;
      if (both) {
        // the next tile's keys stand before this one's values in the ring
        if (more && !next_full(k_slot)) { ok = false; break; }
        if (!next_full(v_slot)) { ok = false; break; }
      } else if (!next_full(v_slot)) {
        ok = false;
        break;
      }
      const uint32_t info = (tiles + j) % kInfos;
      for (uint32_t s = both ? 0u : (j & 1u); s < (both ? 2u : (j & 1u) + 1u); s++) {
        if (!wait(sh.p_full[s], p_turn[s]++)) { ok = false; break; }
        tc_fence_after();
        // where values are no numbers the threads of the rows have added them up themselves
        const volatile uint32_t* b = sh.bad[info];
        if ((b[0] | b[1] | b[2] | b[3]) == 0u) { sums(v_slot, s, shape::kTwo && !both ? j > 1 : j > 0); }
        if constexpr (!shape::kTwo) { commit(sh.pv_done); }
        if (both) {
          if (more) { scores(k_slot, s); }
          if (j + 1 == n) { commit(sh.o_full[s]); }
        } else if constexpr (shape::kTwo) {
          if (!more) { commit(sh.o_full[s]); }
        } else {
          if (j + 1 == n) { commit(sh.o_full[0]); }
        }
      }
      if (!ok) { break; }
      commit(sh.empty[v_slot]);
      if (more) {
        if (!both) {
          if (!next_full(k_slot)) { ok = false; break; }
          scores(k_slot, j & 1u);
        }
        commit(sh.empty[k_slot]);
        if (j + (both ? 2 : 3) == n) { commit(sh.q_empty); }
      }
    }
    if (!ok) { break; }
    tiles += n;
  }
  commit(sh.drained);
  wait(sh.drained, 0);
}

// ---- softmax ------------------------------------------------------------------------------------------------------------------

template <typename T, int D, bool SHAPED>
__device__ __forceinline__ void softmax_role(const tc_args& a, tc_shared& sh, char* smem, const waiter& wait, uint32_t which, uint32_t block)
{
  using shape             = tc_shape<D>;
  constexpr uint32_t TILE = shape::kTile, NB = shape::kStages, GROUPS = TILE / 32;
  const tree_view& t      = a.t;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, stream = warp >> 2, quarter = warp & 3u;
  const uint32_t row0 = block * shape::kRows, rows = min(uint32_t(shape::kRows), t.n_rows - row0);
  const bool both      = shape::kTwo && rows > 128;
  const bool alternate = shape::kTwo && !both;
  const uint32_t in    = quarter * 32 + lane, r = both ? stream * 128 + in : in;
  const bool exists    = r < rows;
  const uint32_t row   = row0 + min(r, rows - 1u), token = row / t.group, g = row - token * t.group;
  const bool alive     = __any_sync(kAllLanes, exists);
  const uint32_t lanes = quarter << 21;  // this warp's lanes of tensor memory
  const uint32_t sums  = sh.tmem + lanes + shape::kSumsAt + (shape::kTwo ? stream * 128 : 0);
  const uint32_t width = (a.c.dim + 31) / 32;  // columns of the sums, in 32
  piece_reader reader;
  tree_piece p;
  uint32_t s_turn[2] = {0, 0}, o_turn = 0, x_turn = 0, tiles = 0, items = 0, pv_turn = 0;

  while (reader.next(sh, wait, p)) {
    const uint32_t n = p.end - p.chunk;
    if (!shape::kTwo && stream == 1) { continue; }
    const int32_t* positions = t.positions + int64_t(p.sequence) * t.positions_stride;
    const uint32_t* mask     = t.mask + int64_t(p.sequence) * t.mask_sequence + int64_t(token) * t.mask_token;
    const int32_t own        = positions[token];
    const bool is_token      = exists && own >= 0 && uint32_t(own) >= p.length;
    float slope              = 0.0f;
    if (SHAPED && t.slopes != nullptr) { slope = t.slopes[p.head * t.group + g] * kLog2E; }
    float top = -INFINITY, sum = 0.0f;
    drafted_lists::list l{p.length, p.first, p.last, p.base};
    uint32_t done = 0;  // tiles of this stream
    bool ok = true;
    for (uint32_t j = alternate ? stream : 0u; j < n; j += alternate ? 2u : 1u, done++) {
      const uint32_t buffer = shape::kTwo ? stream : (j & 1u);
      const uint32_t scores = sh.tmem + lanes + buffer * TILE;
      if (!wait(sh.s_full[buffer], s_turn[buffer]++)) { ok = false; break; }
      tc_fence_after();
      if (!alive) {
        arrive_warp(sh.p_full[buffer]);
        continue;
      }
      uint32_t raw[GROUPS][32];
#pragma unroll
      for (uint32_t i = 0; i < GROUPS; i++) { tmem_ld32_async(scores + i * 32, raw[i]); }
      const uint32_t base = p.base + (p.chunk + j) * TILE, info = (tiles + j) % kInfos;
      const bool mixed    = is_mixed<int(TILE)>(t, p, base);
      uint32_t seen[GROUPS];
#pragma unroll
      for (uint32_t i = 0; i < GROUPS; i++) {
        if constexpr (TILE == 128) {
          seen[i] = sh.valid[info][i];
        } else {
          seen[i] = sh.valid[info][2 * i] | (sh.valid[info][2 * i + 1] << 16);
        }
        if (!is_token) { seen[i] = 0u; }
        if (mixed && is_token) { seen[i] &= seen_keys(t, l, positions, own, mask, base + i * 32); }
      }
      float s[GROUPS][32];
#pragma unroll
      for (uint32_t i = 0; i < GROUPS; i++) {
        tmem_ld_wait(raw[i]);
#pragma unroll
        for (int k = 0; k < 32; k++) { s[i][k] = __uint_as_float(raw[i][k]); }
      }
      if constexpr (SHAPED) {
        if (t.cap_log2 != 0.0f) {
#pragma unroll
          for (uint32_t i = 0; i < GROUPS; i++) {
            float most = 0.0f;
#pragma unroll
            for (int k = 0; k < 32; k++) {
              s[i][k] *= t.scale_cap;
              most = fmaxf(most, fabsf(s[i][k]));
            }
            if (__any_sync(kAllLanes, !(most < 0.6f))) {
#pragma unroll
              for (int k = 0; k < 32; k++) { s[i][k] = tanh_any(s[i][k]) * t.cap_log2; }
            } else {
#pragma unroll
              for (int k = 0; k < 32; k++) { s[i][k] = tanh_near(s[i][k]) * t.cap_log2; }
            }
          }
        } else {
#pragma unroll
          for (uint32_t i = 0; i < GROUPS; i++) {
#pragma unroll
            for (int k = 0; k < 32; k++) { s[i][k] *= t.scale_log2; }
          }
        }
        if (t.slopes != nullptr) {
          const float from = float(int64_t(base) - own);
#pragma unroll
          for (uint32_t i = 0; i < GROUPS; i++) {
#pragma unroll
            for (int k = 0; k < 32; k++) {
              float distance = from + float(int(i) * 32 + k);
              if (mixed) {
                const int64_t drafted = int64_t(base) + int(i * 32 + k) - int64_t(p.length);
                if (drafted >= 0 && drafted < int64_t(t.n_drafted)) { distance = float(int64_t(positions[drafted]) - own); }
              }
              s[i][k] = fmaf(slope, distance, s[i][k]);
            }
          }
        }
      }
      bool whole = true;
#pragma unroll
      for (uint32_t i = 0; i < GROUPS; i++) { whole = whole && seen[i] == 0xFFFFFFFFu; }
      if (!__all_sync(kAllLanes, whole)) {
#pragma unroll
        for (uint32_t i = 0; i < GROUPS; i++) {
#pragma unroll
          for (int k = 0; k < 32; k++) { s[i][k] = ((seen[i] >> k) & 1u) != 0u ? s[i][k] : -INFINITY; }
        }
      }
      float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (uint32_t i = 0; i < GROUPS; i++) {
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
#pragma unroll
          for (int e = 0; e < 4; e++) { most[e] = fmaxf(most[e], s[i][k + e]); }
        }
      }
      float highest = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
      if constexpr (!SHAPED) { highest *= t.scale_log2; }  // (a scale above 0)
      // (a top of -inf: nothing was seen, and the sums are 0)
      if (__any_sync(kAllLanes, highest > top + kAhead)) {
        const float next = highest > top + kAhead ? highest : top;
        const float keep = top == -INFINITY ? 1.0f : power_of_2(top - next);
        if (done > 0 && __any_sync(kAllLanes, keep != 1.0f)) {
          if constexpr (!shape::kTwo) {  // the tile before may still be added up
            if (!wait(sh.pv_done, pv_turn + j - 1)) { ok = false; break; }
            tc_fence_after();
          }
          for (uint32_t i = 0; i < width; i++) {
            uint32_t o[32];
            tmem_ld32(sums + i * 32, o);
            uint32_t x[2][16];
#pragma unroll
            for (int k = 0; k < 32; k++) { x[k / 16][k % 16] = __float_as_uint(__uint_as_float(o[k]) * keep); }
            tmem_st16(sums + i * 32, x[0]);
            tmem_st16(sums + i * 32 + 16, x[1]);
          }
          tmem_st_wait();
        }
        sum *= keep;
        top = next;
      }
      const float from = a.shift - finite_top(top);
      float part[4]    = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (uint32_t i = 0; i < GROUPS; i++) {
        uint32_t high[16], low[16];
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const float x = power_of_2(SHAPED ? s[i][k] + from : fmaf(s[i][k], t.scale_log2, from));
          const float y = power_of_2(SHAPED ? s[i][k + 1] + from : fmaf(s[i][k + 1], t.scale_log2, from));
          part[k & 2] += x;
          part[(k & 2) + 1] += y;
          weight_pair<T>::split(x, y, high[k / 2], low[k / 2]);
        }
        tmem_st16(scores + i * 16, high);
        tmem_st16(scores + TILE / 2 + i * 16, low);
      }
      sum += (part[0] + part[1]) + (part[2] + part[3]);
      tmem_st_wait();
      if (mixed) {
        // Values that are no numbers must not reach rows that do not see them, as 0 times them would: each row adds up what it sees.
        const uint32_t at = items + values_at(j, n), slot = at % NB;
        if (!wait(sh.full[slot], at / NB)) { ok = false; break; }
        const volatile uint32_t* b = sh.bad[info];
        if ((b[0] | b[1] | b[2] | b[3]) != 0u) {
          if constexpr (!shape::kTwo) {
            if (j > 0 && !wait(sh.pv_done, pv_turn + j - 1)) { ok = false; break; }
            tc_fence_after();
          }
          const char* v = smem + shape::kRingAt + slot * shape::kTileBytes;
#pragma unroll 1
          for (uint32_t i = 0; i < width; i++) {
            uint32_t o[32];
            if (done > 0) {
              tmem_ld32(sums + i * 32, o);
            } else {
#pragma unroll
              for (int k = 0; k < 32; k++) { o[k] = 0u; }
            }
#pragma unroll 1
            for (uint32_t k0 = 0; k0 < TILE; k0 += 32) {
              uint32_t high[16], low[16];
              tmem_ld16(scores + k0 / 2, high);
              tmem_ld16(scores + TILE / 2 + k0 / 2, low);
#pragma unroll
              for (uint32_t k = 0; k < 32; k++) {
                const float2 pair = weight_pair<T>::join(high[k / 2], low[k / 2]);
                const float x     = (k & 1u) != 0u ? pair.y : pair.x;
                if (x == 0.0f) { continue; }
                const uint32_t key = k0 + k;
#pragma unroll
                for (uint32_t q = 0; q < 4; q++) {
                  const uint32_t column = i * 4 + q;  // in pieces
                  if (column * 8 >= a.c.dim) { break; }
                  float f[8];
                  piece_to_floats<T>(*reinterpret_cast<const uint4*>(v + (column >> 3) * shape::kPanel + key * 128 + (((column & 7u) ^ (key & 7u)) << 4)), f);
#pragma unroll
                  for (int e = 0; e < 8; e++) { o[q * 8 + e] = __float_as_uint(fmaf(x, f[e], __uint_as_float(o[q * 8 + e]))); }
                }
              }
              __syncwarp();
            }
            uint32_t x[2][16];
#pragma unroll
            for (int k = 0; k < 32; k++) { x[k / 16][k % 16] = o[k]; }
            tmem_st16(sums + i * 32, x[0]);
            tmem_st16(sums + i * 32 + 16, x[1]);
          }
          tmem_st_wait();
        }
      }
      tc_fence_before();
      arrive_warp(sh.p_full[buffer]);
    }
    if (!ok) { return; }
    tiles += n;
    items += 2 * n;
    pv_turn += n;
    if (done > 0 || (!alternate && n > 0)) {
      if (!wait(sh.o_full[shape::kTwo ? stream : 0], o_turn++)) { return; }
      tc_fence_after();
    }

    const size_t part_of = a.parts.part(which, block, p.begins ? 1u : 0u);
    auto write = [&](uint32_t quad, const float4& x, float scale) {  // four columns of this row
      if (!exists || quad * 4 >= a.c.dim) { return; }
      if (p.whole) {
        store_quad<T>(out_row<T>(t, p.sequence, p.head, row) + quad * 4, make_float4(x.x * scale, x.y * scale, x.z * scale, x.w * scale));
      } else {
        a.parts.acc[(part_of * a.parts.quads + quad) * a.parts.rows + r] = x;
      }
    };
    auto finish = [&](float top_, float sum_) {
      if (!exists) { return; }
      if (p.whole) {
        *lse_at(t, p.sequence, p.head, a.c.n_heads, row) = (finite_top(top_) + log2f(sum_) - a.shift) * kLn2;
      } else {
        a.parts.stats[part_of * a.parts.rows + r] = make_float2(top_, sum_);
      }
    };
    if (!alternate) {
      if (alive) {
        const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
        for (uint32_t i = 0; i < width; i++) {
          uint32_t o[32];
          tmem_ld32(sums + i * 32, o);
#pragma unroll
          for (uint32_t q = 0; q < 8; q++) {
            float4 x = make_float4(__uint_as_float(o[4 * q]), __uint_as_float(o[4 * q + 1]), __uint_as_float(o[4 * q + 2]), __uint_as_float(o[4 * q + 3]));
            if (top == -INFINITY) { x = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
            write(i * 8 + q, x, scale);
          }
        }
        finish(top, sum);
      }
    } else {
      // Each of the two groups has the sums of every other tile; one finishes the first half of the columns, the other one the second.
      float4* room = reinterpret_cast<float4*>(smem + shape::kExchange);
      constexpr uint32_t HALF = D / 64;  // 32 columns at a time
      sh.stats[stream][in] = make_float2(top, sum);
      float2 other;
      float own_keep = 0.0f, other_keep = 0.0f, joined_top = 0.0f, joined_sum = 0.0f, scale = 0.0f;
#pragma unroll 1
      for (uint32_t i = 0; i < HALF; i++) {
        const uint32_t theirs = (1u - stream) * HALF + i, ours = stream * HALF + i;
        uint32_t o[32];
        if (alive) {
          if (theirs < width) {
            if (done > 0) {
              tmem_ld32(sums + theirs * 32, o);
            } else {
#pragma unroll
              for (int k = 0; k < 32; k++) { o[k] = 0u; }
            }
#pragma unroll
            for (uint32_t q = 0; q < 8; q++) {
              room[(stream * 8 + q) * 128 + in] =
                make_float4(__uint_as_float(o[4 * q]), __uint_as_float(o[4 * q + 1]), __uint_as_float(o[4 * q + 2]), __uint_as_float(o[4 * q + 3]));
            }
          }
        }
        arrive_warp(sh.exchanged);
        if (!wait(sh.exchanged, x_turn++)) { return; }
        if (alive) {
          if (i == 0) {
            other            = sh.stats[1 - stream][in];
            joined_top       = fmaxf(top, other.x);
            const float safe = finite_top(joined_top);
            own_keep         = power_of_2(top - safe);
            other_keep       = power_of_2(other.x - safe);
            joined_sum       = sum * own_keep + other.y * other_keep;
            scale            = joined_sum == 0.0f ? 0.0f : 1.0f / joined_sum;
          }
          if (ours < width) {
            if (done > 0) {
              tmem_ld32(sums + ours * 32, o);
            } else {
#pragma unroll
              for (int k = 0; k < 32; k++) { o[k] = 0u; }
            }
#pragma unroll
            for (uint32_t q = 0; q < 8; q++) {
              const float4 y = room[((1u - stream) * 8 + q) * 128 + in];
              float4 x       = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              if (top != -INFINITY) {
                x = make_float4(__uint_as_float(o[4 * q]) * own_keep, __uint_as_float(o[4 * q + 1]) * own_keep, __uint_as_float(o[4 * q + 2]) * own_keep,
                                __uint_as_float(o[4 * q + 3]) * own_keep);
              }
              if (other.x != -INFINITY) {
                x = make_float4(fmaf(y.x, other_keep, x.x), fmaf(y.y, other_keep, x.y), fmaf(y.z, other_keep, x.z), fmaf(y.w, other_keep, x.w));
              }
              write(ours * 8 + q, x, scale);
            }
          }
        }
        arrive_warp(sh.exchanged);
        if (!wait(sh.exchanged, x_turn++)) { return; }
      }
      if (alive && stream == 0) { finish(joined_top, joined_sum); }
    }
    tc_fence_before();
  }
}

// ---- the way ------------------------------------------------------------------------------------------------------------------

template <int D>
__device__ __forceinline__ void way_role(const tc_args& a, tc_shared& sh, const waiter& wait, uint32_t which, uint32_t block)
{
  constexpr int TILE  = tc_shape<D>::kTile;
  const uint32_t lane = threadIdx.x & 31u;
  walk<TILE, drafted_lists> path(a.c, a.w, a.lists, a.parts.shares, which);
  piece now;
  uint4 begun = make_uint4(0, 0, 0, 0);
  uint32_t i  = 0;
  bool more   = true;
  while (more) {
    more = __all_sync(kAllLanes, path.next(now)) != 0;
    int32_t latest = 0;
    if (more && a.t.window > 0) {
      const int32_t* positions = a.t.positions + int64_t(now.sequence) * a.t.positions_stride;
      for (uint32_t k = lane; k < a.t.n_drafted; k += 32) { latest = max(latest, positions[k]); }
      latest = __reduce_max_sync(kAllLanes, latest);
    }
    if (i >= kPieces && !wait(sh.piece_empty[i % kPieces], i / kPieces - 1)) { return; }
    if (lane == 0) {
      tree_piece p{};
      p.sequence = kNoMore;
      if (more) {
        p = {now.sequence, now.unit, now.chunk, now.end, path.l.length, path.l.first, path.l.end, path.l.base, latest, now.begins, now.whole};
        if (now.begins && !now.whole) { begun = make_uint4(now.sequence, now.unit, now.n_parts, 0); }
      }
      sh.pieces[i % kPieces] = p;
    }
    arrive_warp(sh.piece_full[i % kPieces]);
    i++;
  }
  if (a.parts.begun != nullptr && block == 0 && lane == 0) { a.parts.begun[which] = begun; }
}

template <typename T, int D, bool SHAPED>
__global__ void __launch_bounds__(kThreads, 1) tree_tc_kernel(const __grid_constant__ tc_args a)
{
  using shape = tc_shape<D>;
  extern __shared__ __align__(1024) char smem[];
  tc_shared& sh       = *reinterpret_cast<tc_shared*>(smem + shape::kMiscAt);
  const uint32_t warp = threadIdx.x >> 5;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 32) {
    for (int i = 0; i < shape::kStages; i++) {
      mbar_init(smem_u32(&sh.full[i]), 4);
      mbar_init(smem_u32(&sh.empty[i]), 1);
    }
    mbar_init(smem_u32(&sh.q_full), 4);
    mbar_init(smem_u32(&sh.q_empty), 1);
    for (int i = 0; i < 2; i++) {
      mbar_init(smem_u32(&sh.s_full[i]), 1);
      mbar_init(smem_u32(&sh.p_full[i]), 4);
      mbar_init(smem_u32(&sh.o_full[i]), 1);
    }
    mbar_init(smem_u32(&sh.pv_done), 1);
    mbar_init(smem_u32(&sh.exchanged), 8);
    mbar_init(smem_u32(&sh.drained), 1);
    for (int i = 0; i < kPieces; i++) {
      mbar_init(smem_u32(&sh.piece_full[i]), 1);
      mbar_init(smem_u32(&sh.piece_empty[i]), kReaders);
    }
    sh.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  chain_begin();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t which = blockIdx.x / a.t.n_blocks_of, block = blockIdx.x - which * a.t.n_blocks_of;
  const waiter wait{sh};
  if (warp < 8) {
    registers_up<184>();
    softmax_role<T, D, SHAPED>(a, sh, smem, wait, which, block);
  } else {
    registers_down<72>();
    if (warp < 12) {
      copy_role<T, D>(a, sh, smem, wait, which, block);
    } else if (warp == 12) {
      multiply_role<T, D>(a, sh, smem, wait, block);
    } else if (warp == 13) {
      way_role<D>(a, sh, wait, which, block);
    } else {
      empty_tree_rows<T>(a.c, a.w.n_sequences, a.lists, a.t, threadIdx.x - 14 * 32, 64);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) { asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(sh.tmem) : "memory"); }
  if (threadIdx.x == 0 && sh.failed != 0u) { count_timeout(a.timeouts); }
}

}  // namespace

// One object per type: KV_TYPE is __half or __nv_bfloat16.
template <>
void attend_tree16<KV_TYPE>(cudaStream_t stream, const tree_call& call)
{
  using T = KV_TYPE;
  tc_args a{call.c, call.w, call.lists, call.t, call.parts, call.pages, call.table_stride, call.shift, call.timeouts};
  // a scale above 0 keeps the order of scores: they need not be touched before their largest is known
  const bool shaped = call.t.cap_log2 != 0.0f || call.t.slopes != nullptr || !(call.t.scale_log2 > 0.0f);
  auto go = [&](auto columns) {
    constexpr int D = decltype(columns)::value;
    auto launch     = [&](auto kernel) {
      ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), tc_shape<D>::kShared);
      launch_chained(kernel, dim3(call.plan.shares * call.plan.blocks_of), kThreads, tc_shape<D>::kShared, stream, a);
    };
    if (shaped) {
      launch(tree_tc_kernel<T, D, true>);
    } else {
      launch(tree_tc_kernel<T, D, false>);
    }
  };
  switch (tree_columns(call.c.dim)) {
    case 64: go(std::integral_constant<int, 64>{}); break;
    case 128: go(std::integral_constant<int, 128>{}); break;
    default: go(std::integral_constant<int, 256>{});
  }
}

}  // namespace cuvs_b200::kv
