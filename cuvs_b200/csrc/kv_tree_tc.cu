// Attention of drafted tokens to the 16-bit rows of their sequences in a paged cache, on tensor cores (the mathematics: kv_tree.cuh).
//
// A block has 128 query rows, or twice 128, and goes through its share's tiles of 64 keys.  A warp for each of two streams issues
// tcgen05.mma: scores S = Q K^T into tensor memory; four warps of 32 rows each, a thread a row, read them, carry the softmax (top and sum in 32
// bits) and write the weights back over them as two 16-bit numbers; the stream's warp issues O += P V with P from tensor memory.  Four more
// warps copy rows of keys and values, 16 bytes at a time, into a ring of tiles for each, and one finds the way through the share.  The streams are the two
// halves of 256 rows on the same tiles, or even and odd tiles of the same 128 rows, whose sums are joined at a unit's end.  Each has two tiles of scores,
// so that the next ones are formed while the softmax is at the last.  Rows of more than 128 columns leave tensor memory room for one stream.
//
// Sums are brought to a new top only where it is 2^4 above the old one: a turn through tensor memory that few tiles need.  Every 32 tiles of a stream
// they are set aside, for the tensor core cuts off what it adds (kChain in kv_tree.cuh).
//
// What bounds it: of 256 rows the softmax, 2,300 clocks of 64 keys where the products are 1,800 (with pairs of weights half again those of one
// number).  From replayed graphs with pauses between, and from calls back to back for seconds, for which the power limit leaves lower clocks: one request
// of 250,001 + 64 tokens, 4 key heads of 7, fp16, 354 and 418 us (648 and 549 TFLOP/s of what is asked for); 16 requests of up to 16,384 + 32
// tokens, 8 key heads of 8, bf16, with a cap 264 and 287 us, without 209 and 238.  Of 16 rows HBM and the blocks' starts: the same with 4 tokens of 4 heads each
// 121 us (3.8 TB/s).  Of more than 128 columns one stream, whose scores and weights nothing covers: 32 requests of up to 8,192 + 8 tokens, 2 key heads of
// 8, bf16, 66 us with 192 columns, 74 with 256 (bytes alone: 26, 35).
#include "kv_tree_tc.cuh"

#include <algorithm>
#include <type_traits>

namespace cuvs_b200::kv {

namespace {

constexpr int kThreads    = 512;  // two softmax groups, four warps that copy, one that multiplies, one that finds the way
constexpr int kInfos      = 16;   // tiles whose descriptions are kept: more than can be between copying keys and the softmax
constexpr int kPieces     = 2;
constexpr int kReaders    = 14;   // warps that read a piece's description
constexpr uint32_t kTile  = 64;   // keys
constexpr int kMostStages = 8;    // of keys, and of values
constexpr uint32_t kPatience = 32;  // times the limit: for a piece, which may be all of a sequence

template <int D>
struct tc_shape {
  static constexpr bool kTwo      = D <= 128;          // two streams with sums of their own
  static constexpr int kRows      = kTwo ? 256 : 128;  // of a block, at most
  static constexpr int kPanel     = int(kTile) * 128;  // bytes of 64 columns of a tile
  static constexpr int kTileBytes = kPanel * (D / 64);
  static constexpr int kQPanel    = 128 * 128;
  static constexpr int kQBytes    = kQPanel * (D / 64);
  static constexpr int kExchange  = kQBytes;  // where two groups exchange sums: behind the first 128 rows
  static constexpr int kQRegion   = !kTwo ? kQBytes : 2 * kQBytes > kQBytes + 32768 ? 2 * kQBytes : kQBytes + 32768;
  static constexpr int kMisc      = 3200;  // tc_shared
  static constexpr int kFit       = (232448 - kQRegion - kMisc) / kTileBytes;
  static constexpr int kKeys      = kFit / 2 < kMostStages ? kFit / 2 : kMostStages;  // tiles of keys in flight, and of values
  static constexpr int kValues    = kFit - kKeys < kMostStages ? kFit - kKeys : kMostStages;
  static constexpr int kKeysAt    = kQRegion;
  static constexpr int kValuesAt  = kKeysAt + kKeys * kTileBytes;
  static constexpr int kMiscAt    = kValuesAt + kValues * kTileBytes;
  static constexpr int kShared    = kMiscAt + kMisc;
  static constexpr int kSumsAt    = 256;               // first column of the sums in tensor memory, behind two tiles of scores of each stream
  static_assert(kKeys >= 2 && kValues >= 2 && kShared <= 232448, "");
};

// A piece of a unit as the way through the share found it.
struct tree_piece {
  uint32_t sequence, head, chunk, end;
  uint32_t length, first, last, base;
  int32_t latest;
  uint32_t begins, whole;
};

struct tc_shared {
  uint64_t k_full[kMostStages], k_empty[kMostStages], v_full[kMostStages], v_empty[kMostStages];
  uint64_t q_full, q_empty, s_full[4], p_full[4], pv_done[2], o_full[2], exchanged, drained[2];
  uint64_t piece_full[kPieces], piece_empty[kPieces];
  tree_piece pieces[kPieces];
  uint2 valid[kInfos];  // of the two warps that copy keys: which are there
  uint2 bad[kInfos];    // of the two that copy values: whether any is no number
  float2 stats[2][128];
  uint32_t tmem, failed;
};
static_assert(sizeof(tc_shared) <= 3200, "");

struct tc_args {
  cache_view c;
  work_view w;
  drafted_lists lists;
  tree_view t;
  tree_parts parts;
  const int32_t* pages;
  int64_t table_stride;
  float4* aside;
  float shift;
  uint32_t* report;
  uint32_t limit, skip_tile;  // of waits; for tests: 1 + the tile of each block whose keys nobody is told of (0: none)
};

constexpr uint32_t kNoMore = 0xFFFFFFFFu;

// Waits with a limit, after which the block gives up; a whole warp at a time.
struct waiter {
  tc_shared& sh;
  uint32_t limit;
  __device__ __forceinline__ bool give_up() const
  {
    *const_cast<volatile uint32_t*>(&sh.failed) = 1u;
    return false;
  }
  __device__ __forceinline__ bool operator()(const uint64_t& bar, uint32_t parity) const
  {
    return mbar_wait_warp(smem_u32(&bar), parity & 1u, limit) || give_up();
  }
  // for a piece, or until another warp has given up
  __device__ __forceinline__ bool patiently(const uint64_t& bar, uint32_t parity) const
  {
    for (uint32_t i = 0; i < kPatience; i++) {
      if (mbar_wait_warp(smem_u32(&bar), parity & 1u, limit)) { return true; }
      if (__any_sync(kAllLanes, *const_cast<volatile uint32_t*>(&sh.failed) != 0u)) { break; }
    }
    return give_up();
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
    if (!wait.patiently(sh.piece_full[i % kPieces], i / kPieces)) { return false; }
    p = sh.pieces[i % kPieces];
    arrive_warp(sh.piece_empty[i % kPieces]);
    i++;
    return p.sequence != kNoMore;
  }
};

// The tile of a stream's piece before which sums that have tile `i` are set aside; the two streams' turns do not come at the same time.
__device__ __forceinline__ uint32_t sums_end(uint32_t i, uint32_t stream)
{
  return ((i + stream * (kChain / 2)) / kChain + 1) * kChain - stream * (kChain / 2);
}

// Whether a tile has keys that not all rows see.
__device__ __forceinline__ bool is_mixed(const tree_view& t, const tree_piece& p, uint32_t base)
{
  return int64_t(base) + kTile > int64_t(p.length) || (t.window > 0 && int64_t(base) <= int64_t(p.latest) - t.window);
}

// ---- copying ------------------------------------------------------------------------------------------------------------------

// This thread's arrival, once its copies so far are there.
__device__ __forceinline__ void arrive_behind_copies(uint64_t& bar)
{
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&bar)) : "memory");
}

// Two warps copy keys, two values, half of a tile's rows each.  They never wait for their own copies: a tile's barrier counts them as they arrive, and the
// warp that multiplies orders them before what the tensor core reads.  (A proxy fence by the warps that copy waited for all of their copies in
// flight: 2.5 us a tile.)
template <typename T, int D>
__device__ __forceinline__ void copy_role(const tc_args& a, tc_shared& sh, char* smem, const waiter& wait, uint32_t block)
{
  using shape                = tc_shape<D>;
  constexpr uint32_t PR = D / 8, AT_ONCE = 32 / PR;  // pieces of a row, rows of a copy
  const cache_view& c        = a.c;
  const tree_view& t         = a.t;
  const uint32_t warp        = (threadIdx.x >> 5) & 3u, lane = threadIdx.x & 31u, half = warp & 1u;
  const bool of_values       = warp >= 2;
  const uint32_t piece       = lane % PR, sub = lane / PR;
  const uint32_t pieces      = c.dim / 8, wide = (pieces + 1) & ~1u;  // products take 16 columns at a time: those behind the row's end are 0
  const uint32_t row0        = block * shape::kRows, rows = min(uint32_t(shape::kRows), t.n_rows - row0);
  const uint32_t column_from = piece < pieces ? piece * 16 : 0u;
  const uint32_t stages      = of_values ? shape::kValues : shape::kKeys;
  const uint32_t ring_at     = (of_values ? shape::kValuesAt : shape::kKeysAt) + (piece >> 3) * shape::kPanel + half * (32 * 128);
  const uint32_t ring = smem_u32(smem) + ring_at, q_at = smem_u32(smem);
  uint64_t *full = of_values ? sh.v_full : sh.k_full, *empty = of_values ? sh.v_empty : sh.k_empty;
  const uint32_t page_units = of_values ? c.v_page_units : c.k_page_units, token_units = of_values ? c.v_token_units : c.k_token_units;
  const bool together = c.page.size % 16 == 0;  // (tiles begin at multiples of 16 positions)
  const uint64_t on   = uint64_t(token_units * AT_ONCE) << c.unit_shift;
  uint32_t tiles = 0, q_turn = 0, slot = 0, round = 0;

  piece_reader reader;
  tree_piece p;
  while (reader.next(sh, wait, p)) {
    const uint32_t n         = p.end - p.chunk;
    const int32_t* table     = a.pages + int64_t(p.sequence) * a.table_stride;
    const int32_t* positions = t.positions + int64_t(p.sequence) * t.positions_stride;
    const char* from         = (of_values ? c.values + int64_t(p.head) * c.v_head * 2 : c.keys + int64_t(p.head) * c.k_head * 2) + column_from;
    // what the table says about this lane's key of a tile, asked for a tile ahead
    const uint32_t own_row = half * 32 + lane;
    auto name = [&](uint32_t tile) -> int32_t {
      const uint32_t at = p.base + tile * kTile + own_row;
      if (tile >= p.end || at < p.first || at >= p.last) { return -1; }
      uint32_t column, place;
      split_place(at, c.page, column, place);
      return table[column];  // at < last: the column is inside the table
    };
    int32_t next = name(p.chunk);
    // queries: they may be replaced once the last scores of the piece before are there
    if (q_turn > 0 && !wait(sh.q_empty, q_turn - 1)) { break; }
    const uint32_t q_rows = rows <= 128 ? 128 : 256;
    for (uint32_t r0 = warp * 32; r0 < q_rows; r0 += 128) {
      const uint32_t mine = r0 + lane, r = row0 + min(mine, rows - 1u), token = r / t.group, g = r - token * t.group;
      const char* q = t.queries.data + (int64_t(p.sequence) * t.queries.sequence + int64_t(token) * t.queries.token +
                                        int64_t(p.head * t.group + g) * t.queries.head) * 2;
#pragma unroll 4
      for (uint32_t i = 0; i < 32; i += AT_ONCE) {
        const uint32_t row  = r0 + i + sub;
        const uint64_t at   = __shfl_sync(kAllLanes, reinterpret_cast<uint64_t>(q), i + sub);
        const uint32_t to   = q_at + (row >> 7) * shape::kQBytes + (piece >> 3) * shape::kQPanel + (row & 127u) * 128 + (((piece & 7u) ^ (row & 7u)) << 4);
        if (piece < wide) { copy_piece(to, reinterpret_cast<const char*>(at) + column_from, piece < pieces && row < rows ? 16u : 0u); }
      }
    }
    arrive_behind_copies(sh.q_full);
    q_turn++;

    bool ok = true;
    for (uint32_t j = 0; j < n; j++, tiles++) {
      const uint32_t base = p.base + (p.chunk + j) * kTile, at = base + own_row;
      const int32_t page  = next;
      next                = name(p.chunk + j + 1);
      uint32_t column, place;
      split_place(min(at, 0x7FFFFFFFu), c.page, column, place);
      bool there = page >= 0 && page < c.n_pages;
      if (there && c.filter != nullptr) {
        const uint64_t number = uint64_t(page) * c.page.size + place;
        there                 = ((c.filter[number >> 5] >> (number & 31u)) & 1u) != 0u;
      }
      if (there && at >= p.length) {
        const int32_t of = positions[at - p.length];
        there            = of >= 0 && uint32_t(of) >= p.length;
      }
      const uint32_t units = there ? uint32_t(page) * page_units + place * token_units : 0u;
      const uint32_t rows_there = __ballot_sync(kAllLanes, there);
      if (round > 0 && !wait(empty[slot], round - 1)) { ok = false; break; }
      const uint32_t to = ring + slot * shape::kTileBytes;
      if (together && rows_there == 0xFFFFFFFFu) {
        // all of the warp's rows are there, 16 of them in a page one behind the other
        const uint32_t bytes = piece < pieces ? 16u : 0u, to_piece = to + sub * 128;
#pragma unroll
        for (uint32_t g = 0; g < 2; g++) {
          const char* row = from + (uint64_t(__shfl_sync(kAllLanes, units, g * 16 + sub)) << c.unit_shift);
#pragma unroll
          for (uint32_t i = 0; i < 16; i += AT_ONCE) {
            if (piece < wide) { copy_piece(to_piece + (g * 16 + i) * 128 + (((piece ^ sub ^ i) & 7u) << 4), row, bytes); }
            row += on;
          }
        }
      } else {
#pragma unroll 4
        for (uint32_t i = 0; i < 32; i += AT_ONCE) {
          const uint32_t r     = i + sub;
          const uint32_t where = __shfl_sync(kAllLanes, units, r);
          const uint32_t bytes = piece < pieces && ((rows_there >> r) & 1u) != 0u ? 16u : 0u;
          if (piece < wide) { copy_piece(to + r * 128 + (((piece ^ r) & 7u) << 4), from + (uint64_t(where) << c.unit_shift), bytes); }
        }
      }
      const uint32_t info = tiles % kInfos;
      if (of_values) {
        bool bad = false;
        if (is_mixed(t, p, base)) {  // values that some rows do not see
          copies_end_group();
          copies_wait<0>();
          for (uint32_t r = sub; r < 32 && piece < wide; r += AT_ONCE) {
            const uint4 x = *reinterpret_cast<const uint4*>(smem + ring_at + slot * shape::kTileBytes + r * 128 + (((piece ^ r) & 7u) << 4));
            constexpr uint32_t kAll = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
            const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; e++) { bad = bad || (words[e] & kAll) == kAll || ((words[e] >> 16) & kAll) == kAll; }
          }
        }
        const bool any = __any_sync(kAllLanes, bad);
        if (lane == 0) { (half == 0 ? sh.bad[info].x : sh.bad[info].y) = any; }
      } else if (lane == 0) {
        (half == 0 ? sh.valid[info].x : sh.valid[info].y) = rows_there;
      }
      if (of_values || tiles + 1 != a.skip_tile) {
        arrive_behind_copies(full[slot]);
        arrive_warp(full[slot]);  // what the warp wrote itself
      }
      if (++slot == stages) {
        slot = 0;
        round++;
      }
    }
    if (!ok) { break; }
  }
  copies_end_group();
  copies_wait<0>();
}

// ---- multiplying --------------------------------------------------------------------------------------------------------------

// One warp for each stream: what a warp has to wait for and to look up between its products would leave the tensor core idle (with one warp for
// both streams 3,000 clocks for 64 keys of 2 x 128 rows, of which the products are 1,800).
template <typename T, int D>
__device__ __forceinline__ void multiply_role(const tc_args& a, tc_shared& sh, char* smem, const waiter& wait, uint32_t block, uint32_t stream)
{
  using shape              = tc_shape<D>;
  constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : 1u;
  const uint32_t rows      = min(uint32_t(shape::kRows), a.t.n_rows - block * shape::kRows);
  const bool both          = shape::kTwo && rows > 128;  // two blocks of rows on the same tiles
  const bool alternate     = shape::kTwo && !both;
  const uint32_t steps     = (a.c.dim + 15) / 16;
  const uint32_t qk        = (1u << 4) | (kType << 7) | (kType << 10) | ((kTile >> 3) << 17) | ((128u >> 4) << 24);
  const uint32_t pv        = (1u << 4) | (kType << 7) | (kType << 10) | (1u << 16) | (((steps * 16) >> 3) << 17) | ((128u >> 4) << 24);
  const uint32_t tmem      = __shfl_sync(kAllLanes, sh.tmem, 0);
  const uint32_t scores_at = tmem + stream * (2 * kTile), sums_at = tmem + shape::kSumsAt + stream * 128;
  const uint32_t q_lo      = desc_sw128_lo(smem_u32(smem)) + (both ? stream * (shape::kQBytes >> 4) : 0u);
  const uint32_t k_lo      = desc_sw128_lo(smem_u32(smem + shape::kKeysAt));
  const uint32_t v_lo      = (smem_u32(smem + shape::kValuesAt) >> 4) | (uint32_t(shape::kPanel >> 4) << 16);

  piece_reader reader;
  tree_piece p;
  uint32_t tiles = 0, q_turn = 0, p_turn = 0;  // p_turn: a bit for each buffer
  while (reader.next(sh, wait, p)) {
    const uint32_t n   = p.end - p.chunk;
    const uint32_t own = alternate ? (n + 1 - stream) / 2 : n;  // tiles of this stream
    if (!wait(sh.q_full, q_turn++)) { break; }
    // (A stream passes over the other's tiles.  Copies arrive in their order, so the barrier of a tile is at most one phase behind where the one before
    // it has been seen.)
    auto arrived = [&](const uint64_t& full, uint32_t round) {
      const bool ok = wait(full, round);
      fence_async_smem();  // what was copied, before what the tensor core reads
      return ok;
    };
    auto scores = [&](uint32_t i) {
      const uint32_t j = alternate ? 2 * i + stream : i;
      const uint32_t slot = (tiles + j) % shape::kKeys;
      if (!arrived(sh.k_full[slot], (tiles + j) / shape::kKeys)) { return false; }
      const uint32_t from = k_lo + slot * (shape::kTileBytes >> 4), to = scores_at + (i & 1u) * kTile;
      if (elect_one()) {
        tc_mma_f16_lo<false>(to, q_lo, from, qk);
#pragma unroll
        for (uint32_t k = 1; k < D / 16; k++) {
          if (k < steps) {
            tc_mma_f16_lo<true>(to, q_lo + ((k >> 2) * shape::kQPanel + (k & 3u) * 32) / 16, from + ((k >> 2) * shape::kPanel + (k & 3u) * 32) / 16, qk);
          }
        }
        tc_commit(smem_u32(&sh.s_full[stream * 2 + (i & 1u)]));
        tc_commit(smem_u32(&sh.k_empty[slot]));
        if (i + 1 == own) { tc_commit(smem_u32(&sh.q_empty)); }
      }
      __syncwarp();
      return true;
    };
    if (own == 0) {  // nothing for this stream, but the queries may be replaced
      if (elect_one()) { tc_commit(smem_u32(&sh.q_empty)); }
      __syncwarp();
    }
    bool ok = own < 1 || scores(0);
    ok      = ok && (own < 2 || scores(1));
    for (uint32_t i = 0; i < own && ok; i++) {
      const uint32_t j = alternate ? 2 * i + stream : i, buffer = i & 1u;
      const uint32_t slot = (tiles + j) % shape::kValues;
      if (!arrived(sh.v_full[slot], (tiles + j) / shape::kValues)) { ok = false; break; }
      // where values are no numbers the threads of the rows add them up themselves
      const uint2 bad = sh.bad[(tiles + j) % kInfos];
      const bool good = (bad.x | bad.y) == 0u;
      if (!wait(sh.p_full[stream * 2 + buffer], p_turn >> buffer)) { ok = false; break; }
      p_turn ^= 1u << buffer;
      tc_fence_after();
      const bool anew = i == 0u || sums_end(i - 1, stream) == i;
      if (elect_one()) {
        if (good) {
          // 32 keys of weights stand where their scores stood: 16 columns of the first numbers, 16 of the second
          const uint32_t from = v_lo + slot * (shape::kTileBytes >> 4), w = scores_at + buffer * kTile;
#pragma unroll
          for (uint32_t k = 0; k < kTile / 16; k++) {
            const uint32_t at = w + (k >> 1) * 32 + (k & 1u) * 8;
            tc_mma_f16_ts(sums_at, at, from + k * (2048 >> 4), pv, k != 0u || !anew);
            tc_mma_f16_ts(sums_at, at + 16, from + k * (2048 >> 4), pv, true);
          }
        }
        tc_commit(smem_u32(&sh.pv_done[stream]));
        tc_commit(smem_u32(&sh.v_empty[slot]));
        if (i + 1 == own) { tc_commit(smem_u32(&sh.o_full[stream])); }
      }
      __syncwarp();
      if (i + 2 < own) { ok = scores(i + 2); }
    }
    if (!ok) { break; }
    tiles += n;
  }
  if (elect_one()) { tc_commit(smem_u32(&sh.drained[stream])); }
  __syncwarp();
  // (whatever the limit: nothing may be on its way into tensor memory that is given back)
  if (!mbar_wait_warp(smem_u32(&sh.drained[stream]), 0u, kSpinLimit)) { wait.give_up(); }
}

// ---- softmax ------------------------------------------------------------------------------------------------------------------

// 32 scores from key `at` on, in powers of two: scaled, capped, less what their distance costs.  They stand at `scores` in tensor memory.
__device__ __forceinline__ void shape_scores(const tree_view& t, const tree_piece& p, const int32_t* positions, int32_t own, float slope, uint32_t at,
                                             bool mixed, uint32_t scores, uint32_t (&x)[32])
{
  if (t.cap_log2 != 0.0f) {
    const two by(t.scale_cap, t.scale_cap);
    float most = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; k += 2) {
      const two y = mul2(two(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), by);
      float u, v;
      y.get(u, v);
      most = fmaxf(most, fmaxf(fabsf(u), fabsf(v)));
      tanh_near(y, t.cap_near).get(u, v);
      x[k]     = __float_as_uint(u);
      x[k + 1] = __float_as_uint(v);
    }
    if (__any_sync(kAllLanes, !(most < kTanhNear))) {  // seldom: once more, the long way
      uint32_t y[32];
      tmem_ld32(scores, y);
#pragma unroll
      for (int k = 0; k < 32; k++) {
        const float z = __uint_as_float(y[k]) * t.scale_cap;
        x[k]          = fabsf(z) < kTanhNear ? x[k] : __float_as_uint(tanh_far(z) * t.cap_log2);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 32; k++) { x[k] = __float_as_uint(__uint_as_float(x[k]) * t.scale_log2); }
  }
  if (t.slopes != nullptr) {
    const float from = float(int64_t(at) - own);
    if (!mixed) {
#pragma unroll
      for (int k = 0; k < 32; k++) { x[k] = __float_as_uint(fmaf(slope, from + float(k), __uint_as_float(x[k]))); }
    } else {
#pragma unroll
      for (int k = 0; k < 32; k++) {
        const int64_t drafted = int64_t(at) + k - int64_t(p.length);
        const float distance  = drafted >= 0 && drafted < int64_t(t.n_drafted) ? float(int64_t(positions[drafted]) - own) : from + float(k);
        x[k]                  = __float_as_uint(fmaf(slope, distance, __uint_as_float(x[k])));
      }
    }
  }
}

// Adds the sums of this thread's row and stream that were set aside (`some`: there are) to those in tensor memory, which are set aside in their turn, or
// put back at the piece's end.
template <uint32_t kRows>
__device__ __forceinline__ void add_sums_aside(float4* aside, uint32_t sums, uint32_t dim, bool exists, bool some, float top, float& aside_top, bool back)
{
  const uint32_t width = (dim + 31) / 32;
  const float keep     = some ? power_of_2(aside_top - finite_top(top)) : 0.0f;
#pragma unroll 1
  for (uint32_t i = 0; i < width; i++) {
    float4 y[8];
#pragma unroll
    for (uint32_t q = 0; q < 8; q++) {
      y[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (some && (i * 8 + q) * 4 < dim) { y[q] = aside[(i * 8 + q) * kRows]; }
    }
    __syncwarp();  // (rows that are none ask for nothing; a load from tensor memory is of the whole warp)
    uint32_t o[32];
    tmem_ld32(sums + i * 32, o);
#pragma unroll
    for (uint32_t q = 0; q < 8; q++) {
      y[q] = make_float4(fmaf(y[q].x, keep, __uint_as_float(o[4 * q])), fmaf(y[q].y, keep, __uint_as_float(o[4 * q + 1])),
                         fmaf(y[q].z, keep, __uint_as_float(o[4 * q + 2])), fmaf(y[q].w, keep, __uint_as_float(o[4 * q + 3])));
      if (!back && exists && (i * 8 + q) * 4 < dim) { aside[(i * 8 + q) * kRows] = y[q]; }
      o[4 * q]     = __float_as_uint(y[q].x);
      o[4 * q + 1] = __float_as_uint(y[q].y);
      o[4 * q + 2] = __float_as_uint(y[q].z);
      o[4 * q + 3] = __float_as_uint(y[q].w);
    }
    __syncwarp();
    if (back) { tmem_st32(sums + i * 32, o); }
  }
  if (back) { tmem_st_wait(); }
  aside_top = top;
}
// Out of the way of the loop over tiles, where that is short: 4 requests of 60,000 + 64 tokens, 4 key heads of 8, 64 columns fp16, 166 us, 172 to 190 beside it;
// where scores are capped (16 requests, 128 columns) 293 us, 268 beside it.
template <uint32_t kRows>
__device__ __noinline__ void add_sums_aside_apart(float4* aside, uint32_t sums, uint32_t dim, bool exists, bool some, float top, float& aside_top, bool back)
{
  add_sums_aside<kRows>(aside, sums, dim, exists, some, top, aside_top, back);
}

template <typename T, int D, bool SHAPED>
__device__ __forceinline__ void softmax_role(const tc_args& a, tc_shared& sh, char* smem, const waiter& wait, uint32_t which, uint32_t block)
{
  using shape             = tc_shape<D>;
  const tree_view& t      = a.t;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, stream = warp >> 2, quarter = warp & 3u;
  const uint32_t row0 = block * shape::kRows, rows = min(uint32_t(shape::kRows), t.n_rows - row0);
  const bool both      = shape::kTwo && rows > 128;
  const bool alternate = shape::kTwo && !both;
  const uint32_t in    = quarter * 32 + lane, r = both ? stream * 128 + in : in;
  const bool exists    = r < rows;
  const uint32_t row   = row0 + min(r, rows - 1u), token = row / t.group, g = row - token * t.group;
  const int64_t out_at = int64_t(token) * t.out.token + int64_t(g) * t.out.head;  // of this row, in its sequence and key head
  const bool alive     = __any_sync(kAllLanes, exists);
  const uint32_t lanes = quarter << 21;  // this warp's lanes of tensor memory
  const uint32_t sh_tmem = sh.tmem;
  const uint32_t sums  = sh_tmem + lanes + shape::kSumsAt + (shape::kTwo ? stream * 128 : 0);
  const uint32_t width = (a.c.dim + 31) / 32;  // columns of the sums, in 32
  // (their top stands where the piece's will)
  auto add_aside = [&](float top, uint32_t done, bool back) {
    constexpr uint32_t kRows = shape::kTwo ? 256 : 128;
    float4* const aside      = a.aside + size_t(blockIdx.x) * (a.c.dim / 4) * kRows + stream * 128 + in;
    const bool some          = exists && done > kChain - stream * (kChain / 2);
    if constexpr (SHAPED) {
      add_sums_aside<kRows>(aside, sums, a.c.dim, exists, some, top, sh.stats[stream][in].x, back);
    } else {
      add_sums_aside_apart<kRows>(aside, sums, a.c.dim, exists, some, top, sh.stats[stream][in].x, back);
    }
  };
  piece_reader reader;
  tree_piece p;
  uint32_t s_turn = 0, o_turn = 0, x_turn = 0, tiles = 0, pv_turn = 0;  // s_turn: a bit for each buffer

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
    // tiles that not all rows see whole: from `tail_from` on, and up to `edge_to`
    const int32_t tail_from = int32_t((int64_t(p.length) - int64_t(p.base)) >> 6);
    const int32_t edge_to   = t.window > 0 ? int32_t((int64_t(p.latest) - t.window - int64_t(p.base)) >> 6) : -1;
    uint32_t done = 0;  // tiles of this stream
    bool ok = true;
    // From one turn at setting aside to the next: a test for it inside the loop over tiles cost capped scores 7%.
    const uint32_t step = alternate ? 2u : 1u;
    uint32_t j          = alternate ? stream : 0u;
    while (true) {
      const uint32_t begun = done, full = sums_end(done, stream);
      for (; j < n && done < full; j += step, done++) {
        const uint32_t buffer = stream * 2 + (done & 1u);
        const uint32_t scores = sh_tmem + lanes + buffer * kTile;
        if (!wait(sh.s_full[buffer], s_turn >> (done & 1u))) { ok = false; break; }
        s_turn ^= 1u << (done & 1u);
        tc_fence_after();
        if (!alive) {
          arrive_warp(sh.p_full[buffer]);
          continue;
        }
        uint32_t x[2][32];
        tmem_ld32_async(scores, x[0]);
        tmem_ld32_async(scores + 32, x[1]);
        const uint32_t info = (tiles + j) % kInfos, base = p.base + (p.chunk + j) * kTile;
        const bool mixed    = int32_t(p.chunk + j) >= tail_from || int32_t(p.chunk + j) <= edge_to;
        const uint2 valid   = sh.valid[info];
        const bool whole    = (valid.x & valid.y) == 0xFFFFFFFFu && !mixed;
        tmem_ld_wait(x[0]);
        tmem_ld_wait(x[1]);
        if constexpr (SHAPED) {
#pragma unroll
          for (uint32_t i = 0; i < 2; i++) { shape_scores(t, p, positions, own, slope, base + i * 32, mixed, scores + i * 32, x[i]); }
        }
        if (!whole) {
#pragma unroll
          for (uint32_t i = 0; i < 2; i++) {
            uint32_t seen = i == 0 ? valid.x : valid.y;
            if (mixed) { seen &= seen_keys(t, l, positions, own, mask, base + i * 32); }
#pragma unroll
            for (int k = 0; k < 32; k++) { x[i][k] = ((seen >> k) & 1u) != 0u ? x[i][k] : 0xFF800000u; }
          }
          __syncwarp();
        }
        float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (uint32_t i = 0; i < 2; i++) {
#pragma unroll
          for (int k = 0; k < 32; k += 4) {
#pragma unroll
            for (int e = 0; e < 4; e++) { most[e] = fmaxf(most[e], __uint_as_float(x[i][k + e])); }
          }
        }
        float highest = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
        if constexpr (!SHAPED) { highest *= t.scale_log2; }  // (a scale above 0)
        // (a top of -inf: nothing was seen, and the sums are 0)
        if (__any_sync(kAllLanes, highest > top + kAhead)) {
          const float next = highest > top + kAhead ? highest : top;
          const float keep = top == -INFINITY ? 1.0f : power_of_2(top - next);
          if (done != begun && __any_sync(kAllLanes, keep != 1.0f)) {
            // the tile before may still be added up
            if (!wait(sh.pv_done[stream], pv_turn + done - 1)) { ok = false; break; }
            tc_fence_after();
#pragma unroll 1
            for (uint32_t i = 0; i < width; i++) {
              uint32_t o[32];
              tmem_ld32(sums + i * 32, o);
#pragma unroll
              for (int k = 0; k < 32; k++) { o[k] = __float_as_uint(__uint_as_float(o[k]) * keep); }
              tmem_st32(sums + i * 32, o);
            }
            tmem_st_wait();
          }
          sum *= keep;
          top = next;
        }
        const float from = a.shift - finite_top(top), by = SHAPED ? 1.0f : t.scale_log2;
        const two from2(from, from), by2(by, by);
        two part[2] = {two(0.0f, 0.0f), two(0.0f, 0.0f)};
#pragma unroll
        for (uint32_t i = 0; i < 2; i++) {
          uint32_t pairs[32];
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float u, v;
            fma2(two(__uint_as_float(x[i][k]), __uint_as_float(x[i][k + 1])), by2, from2).get(u, v);
            u = power_of_2(u);
            v = power_of_2(v);
            part[(k / 2) % 2] = add2(part[(k / 2) % 2], two(u, v));
            weight_pair<T>::split(u, v, pairs[k / 2], pairs[16 + k / 2]);
          }
          tmem_st32(scores + i * 32, pairs);
        }
        tmem_st_wait();
        {
          float u, v;
          add2(part[0], part[1]).get(u, v);
          sum += u + v;
        }
        if (mixed) {
          // Values that are no numbers must not reach rows that do not see them, as 0 times them would: each row adds up what it sees.
          const uint32_t slot = (tiles + j) % shape::kValues;
          if (!wait(sh.v_full[slot], (tiles + j) / shape::kValues)) { ok = false; break; }
          const uint2 bad = sh.bad[info];
          if ((bad.x | bad.y) != 0u) {
            if (done > 0 && !wait(sh.pv_done[stream], pv_turn + done - 1)) { ok = false; break; }
            tc_fence_after();
            const char* v = smem + shape::kValuesAt + slot * shape::kTileBytes;
#pragma unroll 1
            for (uint32_t i = 0; i < width; i++) {
              uint32_t o[32];
              if (done != begun) {
                tmem_ld32(sums + i * 32, o);
              } else {
#pragma unroll
                for (int k = 0; k < 32; k++) { o[k] = 0u; }
              }
#pragma unroll 1
              for (uint32_t k0 = 0; k0 < kTile; k0 += 32) {
                uint32_t pairs[32];
                tmem_ld32(scores + k0, pairs);
#pragma unroll
                for (uint32_t k = 0; k < 32; k++) {
                  const float2 pair = weight_pair<T>::join(pairs[k / 2], pairs[16 + k / 2]);
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
              tmem_st32(sums + i * 32, o);
            }
            tmem_st_wait();
          }
        }
        tc_fence_before();
        arrive_warp(sh.p_full[buffer]);
      }
      if (!ok || j >= n) { break; }
      if (alive) {
        // (The scores of the next tile took the place of the weights of the last tile but one, which has been added up then: the barrier is at most one
        // phase behind, and no further one ends before this warp has written its next weights.)
        if (!wait(sh.s_full[stream * 2 + (done & 1u)], s_turn >> (done & 1u)) || !wait(sh.pv_done[stream], pv_turn + done - 1)) { ok = false; break; }
        tc_fence_after();
        add_aside(top, done, false);
        tc_fence_before();
      }
    }
    if (!ok) { return; }
    if (!is_token) {  // whatever stands in the sums of a row that is none
      top = -INFINITY;
      sum = 0.0f;
    }
    tiles += n;
    pv_turn += done;
    if (done > 0) {
      if (!wait(sh.o_full[stream], o_turn++)) { return; }
      tc_fence_after();
      if (done > kChain - stream * (kChain / 2) && alive) { add_aside(top, done, true); }
    }

    const size_t part_of = a.parts.part(which, block, p.begins ? 1u : 0u);
    T* const out         = reinterpret_cast<T*>(t.out.data) + int64_t(p.sequence) * t.out.sequence + out_at + int64_t(p.head * t.group) * t.out.head;
    float4* const part   = a.parts.acc + part_of * a.parts.quads * a.parts.rows + r;
    auto write = [&](uint32_t quad, const float4& x, float scale) {  // four columns of this row
      if (!exists || quad * 4 >= a.c.dim) { return; }
      if (p.whole) {
        store_quad<T>(out + quad * 4, make_float4(x.x * scale, x.y * scale, x.z * scale, x.w * scale));
      } else {
        part[quad * a.parts.rows] = x;
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
          __syncwarp();
        }
        finish(top, sum);
      }
    } else {
      // Each of the two groups has the sums of every other tile; one finishes the first half of the columns, the other one the second.
      float4* room = reinterpret_cast<float4*>(smem + shape::kExchange);
      constexpr uint32_t SIDE = D / 64;  // 32 columns at a time
      sh.stats[stream][in] = make_float2(top, sum);
      float2 other;
      float own_keep = 0.0f, other_keep = 0.0f, joined_top = 0.0f, joined_sum = 0.0f, scale = 0.0f;
#pragma unroll 1
      for (uint32_t i = 0; i < SIDE; i++) {
        const uint32_t theirs = (1u - stream) * SIDE + i, ours = stream * SIDE + i;
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

__device__ __forceinline__ void way_role(const tc_args& a, tc_shared& sh, const waiter& wait, uint32_t which, uint32_t block)
{
  const uint32_t lane = threadIdx.x & 31u;
  walk<int(kTile), drafted_lists> path(a.c, a.w, a.lists, a.parts.shares, which);
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
    if (i >= kPieces && !wait.patiently(sh.piece_empty[i % kPieces], i / kPieces - 1)) {
      begun = make_uint4(0, 0, 0, 0);  // the join must find no entry that an earlier call has left
      break;
    }
    if (lane == 0) {
      tree_piece p{};
      p.sequence = kNoMore;
      if (more) {
        p = {now.sequence, now.unit, now.chunk, now.end, path.l.length, path.l.first, path.l.end, path.l.base, latest, now.begins, now.whole};
        if (now.begins) { note_begun(a.parts, now, a.c.n_heads, which, begun); }
      }
      sh.pieces[i % kPieces] = p;
    }
    arrive_warp(sh.piece_full[i % kPieces]);
    i++;
  }
  if (a.parts.begun != nullptr && !a.parts.by_unit && block == 0 && lane == 0) { a.parts.begun[which] = begun; }
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
  const uint32_t which = blockIdx.x / a.t.n_blocks_of, block = blockIdx.x - which * a.t.n_blocks_of;
  if (threadIdx.x == 32) {
    const bool both = shape::kTwo && a.t.n_rows - block * shape::kRows > 128;
    for (int i = 0; i < kMostStages; i++) {
      mbar_init(smem_u32(&sh.k_full[i]), 64 + 2);
      mbar_init(smem_u32(&sh.v_full[i]), 64 + 2);
      mbar_init(smem_u32(&sh.k_empty[i]), both ? 2 : 1);
      mbar_init(smem_u32(&sh.v_empty[i]), both ? 2 : 1);
    }
    mbar_init(smem_u32(&sh.q_full), 128);
    mbar_init(smem_u32(&sh.q_empty), shape::kTwo ? 2 : 1);
    for (int i = 0; i < 4; i++) {
      mbar_init(smem_u32(&sh.s_full[i]), 1);
      mbar_init(smem_u32(&sh.p_full[i]), 4);
    }
    mbar_init(smem_u32(&sh.pv_done[0]), 1);
    mbar_init(smem_u32(&sh.pv_done[1]), 1);
    mbar_init(smem_u32(&sh.o_full[0]), 1);
    mbar_init(smem_u32(&sh.o_full[1]), 1);
    mbar_init(smem_u32(&sh.exchanged), 8);
    mbar_init(smem_u32(&sh.drained[0]), 1);
    mbar_init(smem_u32(&sh.drained[1]), 1);
    for (int i = 0; i < kPieces; i++) {
      mbar_init(smem_u32(&sh.piece_full[i]), 1);
      mbar_init(smem_u32(&sh.piece_empty[i]), shape::kTwo ? kReaders : kReaders - 1);
    }
    sh.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  chain_begin();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const waiter wait{sh, a.limit};
  if (warp < 8) {
    registers_up<168>();
    softmax_role<T, D, SHAPED>(a, sh, smem, wait, which, block);
  } else {
    registers_down<88>();  // 256 threads of 168 and 256 of 88: what the block was launched with
    if (warp < 12) {
      copy_role<T, D>(a, sh, smem, wait, block);
    } else if (warp == 12) {
      multiply_role<T, D>(a, sh, smem, wait, block, 0);
    } else if (warp == 13) {
      way_role(a, sh, wait, which, block);
    } else if (warp == 14) {
      if constexpr (shape::kTwo) { multiply_role<T, D>(a, sh, smem, wait, block, 1); }
    } else {
      empty_tree_rows<T>(a.c, a.w.n_sequences, a.lists, a.t, a.parts, threadIdx.x - 15 * 32, 32);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) { asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(sh.tmem) : "memory"); }
  if (threadIdx.x == 0 && sh.failed != 0u) {
    *const_cast<volatile uint32_t*>(a.report) = 1u;
    __threadfence_system();
  }
}

}  // namespace

// One object per type: KV_TYPE is __half or __nv_bfloat16.
template <>
void attend_tree16<KV_TYPE>(cudaStream_t stream, const tree_call& call)
{
  using T = KV_TYPE;
  tc_args a{call.c, call.w, call.lists, call.t, call.parts, call.pages, call.table_stride, call.aside, call.shift, call.report, call.limit, call.skip_tile};
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
