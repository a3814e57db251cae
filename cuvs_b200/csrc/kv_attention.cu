// Attention of one token per sequence to the rows of its sequence in a paged cache.
//
//   S_j = scale q.k_j over the positions j that may be attended,  lse = log sum exp S_j,  o = sum exp(S_j - lse) v_j
//
// What bounds it: the rows are read once, 4 bytes of products for each byte of a 16-bit key or value and query head, so with 8 query
// heads to a key head HBM at 6.5 TB/s asks for 52 TFLOP/s: more than the FP32 pipes have left beside the conversions, a fraction of what
// mma.sync has.  Everything here serves keeping loads in flight.
//
// Work.  The positions of every (sequence, key head, block of query heads) -- a unit -- are cut into tiles; all units' tiles stand in one
// row, and each of a fixed number of resident blocks takes an equal, contiguous share of it, whatever the lengths are.  Lengths are known
// on the device alone, so every warp finds its block's share from them itself.  A unit that lies in one block's share is finished there;
// of a unit that several share, each leaves a part (top, sum and weighted sum in 32 bits), and a second kernel joins the parts in the
// order of the blocks.  Nothing depends on the order in which blocks run.
#include "kv_rows.cuh"

#include <algorithm>
#include <type_traits>

namespace cuvs_b200::kv {

namespace {

constexpr int kWarps   = 4;
constexpr int kThreads = kWarps * 32;

// ---- shares -------------------------------------------------------------------------------------------------------------------

struct work_view {
  const int32_t* pages;
  const int32_t* lengths;
  int64_t table_stride;
  int64_t window;
  uint32_t n_sequences, width;
  uint32_t n_units;        // per sequence: key heads x blocks of query heads
  uint32_t n_blocks_of;    // blocks of query heads of one key head
  uint32_t group;          // query heads of one key head
};

// A tile begins at a multiple of 16 positions, so that 16 rows lie in one page where pages are multiples of 16.
template <int TILE>
__device__ __forceinline__ uint32_t tiles_of(const cache_view& c, const work_view& w, uint32_t sequence, uint32_t& first, uint32_t& end)
{
  attended(w.lengths[sequence], w.window, w.width, c.page_size, first, end);
  return end > first ? (end - (first & ~15u) + TILE - 1) / TILE : 0u;
}

struct share {
  uint64_t total;       // tiles of all units
  uint32_t blocks;      // that have a share
  __device__ uint64_t start(uint32_t block) const { return block * total / blocks; }
};

// The number of all tiles; every warp sums it up for itself.
template <int TILE>
__device__ __forceinline__ uint64_t all_tiles(const cache_view& c, const work_view& w)
{
  uint64_t sum = 0;
  uint32_t first, end;
#pragma unroll 4
  for (uint32_t b = threadIdx.x & 31u; b < w.n_sequences; b += 32) { sum += tiles_of<TILE>(c, w, b, first, end); }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { sum += __shfl_xor_sync(kAllLanes, sum, o); }
  return sum * w.n_units;
}

// The sequence that tile `at` of all belongs to, and the number of tiles before that sequence.
template <int TILE>
__device__ __forceinline__ uint32_t sequence_of(const cache_view& c, const work_view& w, uint64_t at, uint64_t& before)
{
  const uint32_t lane = threadIdx.x & 31u;
  before              = 0;
  for (uint32_t b0 = 0; b0 < w.n_sequences; b0 += 32) {  // comes to an end inside: `at` is less than the number of all tiles
    uint32_t first, end;
    const uint64_t mine = b0 + lane < w.n_sequences ? uint64_t(tiles_of<TILE>(c, w, b0 + lane, first, end)) * w.n_units : 0u;
    uint64_t up         = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t t = __shfl_up_sync(kAllLanes, up, o);
      if (lane >= uint32_t(o)) { up += t; }
    }
    const unsigned past = __ballot_sync(kAllLanes, before + up > at);
    if (past != 0u) {
      const int l = __ffs(int(past)) - 1;
      before += __shfl_sync(kAllLanes, up - mine, l);
      return b0 + l;
    }
    before += __shfl_sync(kAllLanes, up, 31);
  }
  return w.n_sequences;
}

// ---- parts --------------------------------------------------------------------------------------------------------------------

// Two parts per block: 0 of a unit that a block before began, 1 of a unit that this block begins and a later one goes on with.
struct parts_view {
  float* acc;     // [2 blocks][rows][dim]
  float2* stats;  // [2 blocks][rows] top (of scores in powers of two), sum
  // about the unit that block i - 1 begins and block i goes on with: the tile behind its end (0: there is none), sequence | unit << 32
  uint64_t* unit;  // [blocks + 1][2]
  uint32_t rows;   // query heads of a unit, at most
};

__host__ __device__ inline size_t part_bytes(uint32_t blocks, uint32_t rows, uint32_t dim)
{
  return round_up<size_t>(size_t(2) * blocks * rows * (dim * sizeof(float) + sizeof(float2)), 16) + size_t(blocks + 1) * 16;
}
inline parts_view parts_at(char* workspace, uint32_t blocks, uint32_t rows, uint32_t dim)
{
  parts_view p;
  p.acc   = reinterpret_cast<float*>(workspace);
  p.stats = reinterpret_cast<float2*>(p.acc + size_t(2) * blocks * rows * dim);
  p.unit  = reinterpret_cast<uint64_t*>(workspace + part_bytes(blocks, rows, dim) - size_t(blocks + 1) * 16);
  p.rows  = rows;
  return p;
}

template <typename T>
__device__ __forceinline__ void store_piece(const rows_view& out, uint32_t sequence, uint32_t head, uint32_t piece, const float* x)
{
  reinterpret_cast<uint4*>(out.data + (int64_t(sequence) * out.row + int64_t(head) * out.head) * int64_t(sizeof(T)))[piece] = floats_to_piece<T>(x);
}

// Rows of sequences that attend to nothing: they have no tiles.
template <typename T, int TILE>
__device__ __forceinline__ void empty_rows(const cache_view& c, const work_view& w, const rows_view& out, float* lse)
{
  constexpr uint32_t E   = kPerPiece<T>;
  const uint32_t heads   = w.group * c.n_heads;
  const float nothing[8] = {};
  for (uint32_t b = blockIdx.x; b < w.n_sequences; b += gridDim.x) {
    uint32_t first, end;
    if (tiles_of<TILE>(c, w, b, first, end) != 0u) { continue; }
    for (uint32_t i = threadIdx.x; i < heads * (c.dim / E); i += kThreads) { store_piece<T>(out, b, i / (c.dim / E), i % (c.dim / E), nothing); }
    for (uint32_t i = threadIdx.x; i < heads; i += kThreads) { lse[size_t(b) * heads + i] = -INFINITY; }
  }
}

// What the block's warps have of a unit (top, sum and weighted sum of every row in shared memory) becomes output rows, or a part.
template <typename T>
__device__ __forceinline__ void finish_unit(const cache_view& c, const work_view& w, const float* s_acc, uint32_t acc_row, const float2* s_stats,
                                            uint32_t rows, uint32_t sequence, uint32_t head0, const rows_view& out, float* lse, bool whole,
                                            const parts_view& parts, uint32_t part)
{
  constexpr uint32_t E  = kPerPiece<T>;
  const uint32_t pieces = c.dim / E;
  for (uint32_t i = threadIdx.x; i < rows * pieces; i += kThreads) {
    const uint32_t r = i / pieces, piece = i - r * pieces;
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < kWarps; v++) { top = fmaxf(top, s_stats[v * parts.rows + r].x); }
    const float safe = finite_top(top);
    float sum        = 0.0f;
    float x[E]       = {};
#pragma unroll
    for (int v = 0; v < kWarps; v++) {
      const float2 st = s_stats[v * parts.rows + r];
      const float s   = exp2f(st.x - safe);
      sum             = fmaf(st.y, s, sum);
      const float* a  = s_acc + (size_t(v) * parts.rows + r) * acc_row + piece * E;
#pragma unroll
      for (uint32_t e = 0; e < E; e++) { x[e] = fmaf(a[e], s, x[e]); }
    }
    if (whole) {
      const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
      for (uint32_t e = 0; e < E; e++) { x[e] *= scale; }
      store_piece<T>(out, sequence, head0 + r, piece, x);
      if (piece == 0) { lse[size_t(sequence) * (w.group * c.n_heads) + head0 + r] = (safe + log2f(sum)) * kLn2; }
    } else {
      float4* a = reinterpret_cast<float4*>(parts.acc + (size_t(part) * parts.rows + r) * c.dim + piece * E);
#pragma unroll
      for (uint32_t e = 0; e < E; e += 4) { a[e / 4] = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]); }
      if (piece == 0) { parts.stats[size_t(part) * parts.rows + r] = make_float2(top, sum); }
    }
  }
}

// Goes through the block's share unit by unit: body(sequence, unit, first, end, tile0, tile1) leaves its rows' state in shared memory.
template <typename T, int TILE, class Body>
__device__ __forceinline__ void each_unit(const cache_view& c, const work_view& w, const rows_view& out, float* lse, const parts_view& parts,
                                          const float* s_acc, uint32_t acc_row, const float2* s_stats, Body&& body)
{
  share s;
  s.total  = all_tiles<TILE>(c, w);
  s.blocks = uint32_t(min(uint64_t(gridDim.x), s.total));
  uint64_t unfinished = 0, where = 0;
  if (blockIdx.x < s.blocks) {
    uint64_t at             = s.start(blockIdx.x);
    const uint64_t stop     = s.start(blockIdx.x + 1);
    uint64_t before;
    uint32_t b = sequence_of<TILE>(c, w, at, before);
    while (at < stop && b < w.n_sequences) {
      uint32_t first, end;
      const uint32_t n = tiles_of<TILE>(c, w, b, first, end);
      while (at < stop && at < before + uint64_t(n) * w.n_units) {
        const uint32_t unit  = uint32_t((at - before) / n);
        const uint64_t begin = before + uint64_t(unit) * n;
        const uint64_t last  = min(stop, begin + n);
        body(b, unit, first, end, uint32_t(at - begin), uint32_t(last - begin));
        const uint32_t head = unit / w.n_blocks_of, of = unit - head * w.n_blocks_of;
        const uint32_t rows = min(parts.rows, w.group - of * parts.rows);
        const bool whole    = at == begin && last == begin + n;
        __syncthreads();
        finish_unit<T>(c, w, s_acc, acc_row, s_stats, rows, b, head * w.group + of * parts.rows, out, lse, whole, parts,
                       2 * blockIdx.x + (at == begin ? 1u : 0u));
        __syncthreads();
        if (at == begin && !whole) {
          unfinished = begin + n;
          where      = uint64_t(b) | uint64_t(unit) << 32;
        }
        at = last;
      }
      before += uint64_t(n) * w.n_units;
      b++;
    }
  }
  if (parts.unit != nullptr && threadIdx.x == 0) {
    parts.unit[2 * (blockIdx.x + 1)]     = unfinished;
    parts.unit[2 * (blockIdx.x + 1) + 1] = where;
    if (blockIdx.x == 0) {
      parts.unit[0] = s.total;
      parts.unit[1] = s.blocks;
    }
  }
}

// ---- joining parts ------------------------------------------------------------------------------------------------------------

constexpr int kJoinWarps = 8;

// One block per share that begins inside a unit begun by the block before.  SPLIT warps take turns at the parts of a row.
template <typename T, int SPLIT>
__global__ void __launch_bounds__(kJoinWarps * 32)
join_kernel(work_view w, parts_view parts, uint32_t dim, uint32_t n_heads, rows_view out, float* lse)
{
  chain_begin();
  constexpr int E      = 4;
  const uint32_t i     = blockIdx.x + 1;
  const uint64_t stop  = parts.unit[2 * i];
  if (stop == 0u) { return; }
  const uint64_t where = parts.unit[2 * i + 1];
  const share s{parts.unit[0], uint32_t(parts.unit[1])};
  const uint32_t sequence = uint32_t(where), unit = uint32_t(where >> 32);
  const uint32_t head = unit / w.n_blocks_of, of = unit - head * w.n_blocks_of;
  const uint32_t rows = min(parts.rows, w.group - of * parts.rows);
  const uint32_t head0 = head * w.group + of * parts.rows;
  // the part that begins the unit, then the first parts of all blocks whose share begins before the unit's end
  // (block j's share begins at j * total / blocks, rounded down: before `stop` as long as j * total < stop * blocks)
  const uint32_t behind = uint32_t(min((stop * s.blocks + s.total - 1) / s.total, uint64_t(s.blocks)));
  const uint32_t n    = 1 + behind - i;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  auto part_at = [&](uint32_t p) { return p == 0 ? 2 * (i - 1) + 1 : 2 * (i + p - 1); };
  __shared__ float s_acc[SPLIT > 1 ? kJoinWarps : 1][256];
  for (uint32_t r = blockIdx.y * (kJoinWarps / SPLIT) + warp / SPLIT; r < rows; r += gridDim.y * (kJoinWarps / SPLIT)) {
    float top = -INFINITY;
    for (uint32_t p = lane; p < n; p += 32) { top = fmaxf(top, parts.stats[size_t(part_at(p)) * parts.rows + r].x); }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { top = fmaxf(top, __shfl_xor_sync(kAllLanes, top, o)); }
    const float safe = finite_top(top);
    float sum        = 0.0f;
    for (uint32_t p = lane; p < n; p += 32) {
      const float2 st = parts.stats[size_t(part_at(p)) * parts.rows + r];
      sum             = fmaf(st.y, exp2f(st.x - safe), sum);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { sum += __shfl_xor_sync(kAllLanes, sum, o); }
    const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
    float x[2][E]     = {};
#pragma unroll 8
    for (uint32_t p = warp % SPLIT; p < n; p += SPLIT) {
      const uint32_t part = part_at(p);
      const float weight  = exp2f(parts.stats[size_t(part) * parts.rows + r].x - safe);
      const float4* a     = reinterpret_cast<const float4*>(parts.acc + (size_t(part) * parts.rows + r) * dim);
#pragma unroll
      for (int v = 0; v < 2; v++) {
        if ((lane + 32u * v) * E < dim) {
          const float4 y = a[lane + 32 * v];
          x[v][0]        = fmaf(weight, y.x, x[v][0]);
          x[v][1]        = fmaf(weight, y.y, x[v][1]);
          x[v][2]        = fmaf(weight, y.z, x[v][2]);
          x[v][3]        = fmaf(weight, y.w, x[v][3]);
        }
      }
    }
    if constexpr (SPLIT > 1) {
#pragma unroll
      for (int v = 0; v < 2; v++) {
#pragma unroll
        for (int e = 0; e < E; e++) { s_acc[warp][(lane + 32 * v) * E + e] = x[v][e]; }
      }
      __syncthreads();  // SPLIT is all of the block's warps: they take the same turns
      T* o = reinterpret_cast<T*>(out.data) + int64_t(sequence) * out.row + int64_t(head0 + r) * out.head;
      for (uint32_t d = threadIdx.x; d < dim; d += kJoinWarps * 32) {
        float y = 0.0f;
#pragma unroll
        for (int v = 0; v < kJoinWarps; v++) { y += s_acc[v][d]; }
        o[d] = from_float<T>(y * scale);
      }
      __syncthreads();
    } else {
      T* o = reinterpret_cast<T*>(out.data) + int64_t(sequence) * out.row + int64_t(head0 + r) * out.head;
#pragma unroll
      for (int v = 0; v < 2; v++) {
        const uint32_t d = (lane + 32u * v) * E;
        if (d < dim) {
          alignas(16) T y[E];
#pragma unroll
          for (int e = 0; e < E; e++) { y[e] = from_float<T>(x[v][e] * scale); }
          if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<uint2*>(o + d) = *reinterpret_cast<const uint2*>(y);
          } else {
            *reinterpret_cast<uint4*>(o + d) = *reinterpret_cast<const uint4*>(y);
          }
        }
      }
    }
    if (warp % SPLIT == 0 && lane == 0) { lse[size_t(sequence) * (w.group * n_heads) + head0 + r] = (safe + log2f(sum)) * kLn2; }
  }
}

// ---- 16-bit rows: tensor cores ------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t shared_address(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void copy_piece(uint32_t to, const void* from, bool there)
{
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait()
{
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at)
{
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_matrices_turned(uint32_t (&r)[4], uint32_t at)
{
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ uint32_t turn_matrix(uint32_t a)
{
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
template <typename T>
__device__ __forceinline__ void multiply_add(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void multiply_add<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void multiply_add<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A weight goes into the product with the values as the sum of two 16-bit numbers, so that its rounding (2^-9 of bf16) is not added to
// that of the output: twice the mma.sync of that product, which has them to spare.  The first is taken a little too small, so that the
// second is never 0 where the weight is not: 0 times an infinite value would be no number.
template <typename T>
struct halves;
template <>
struct halves<__half> {
  static constexpr float kBelow = 0.999f;
  static constexpr float kShift = 14.0f;  // weights are held times 2^14: small ones keep their digits above fp16's smallest numbers
  static __device__ __forceinline__ uint32_t pack(float a, float b)
  {
    const __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
};
template <>
struct halves<__nv_bfloat16> {
  static constexpr float kBelow = 0.99f;
  static constexpr float kShift = 0.0f;
  static __device__ __forceinline__ uint32_t pack(float a, float b)
  {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)); }
};

// D: columns of a row in shared memory (64, 128, 256; what is behind the row's end is 0).  NT: query heads of a unit, in eights.
template <int D, int NT>
struct mma_shape {
  static constexpr int kRows     = 8 * NT;
  static constexpr int kTile     = kWarps * 16;
  static constexpr int kStages   = D == 64 ? 4 : D == 128 ? 2 : 3;
  static constexpr bool kQInRegs = D * NT <= 256;
  static constexpr int kResident = D == 256 ? 1 : NT == 4 ? 2 : 3;  // blocks of an SM
  static constexpr int kRowBytes = D * 2;
  static constexpr int kStage    = 2 * 16 * kRowBytes;                       // 16 keys, 16 values
  static constexpr int kAccRow   = D + 4;                                    // floats: lanes of a store on different banks
  static constexpr int kBuffers  = kWarps * kStages * kStage;
  static constexpr int kAcc      = kWarps * kRows * kAccRow * 4;
  static constexpr int kQBytes   = kQInRegs ? 0 : kRows * kRowBytes;
  static constexpr int kStatsAt  = kBuffers > kAcc ? kBuffers : kAcc;
  static constexpr int kQAt      = kStatsAt + kWarps * kRows * 8;
  static constexpr int kMaskAt   = kQAt + kQBytes;
  static constexpr int kShared   = kMaskAt + kWarps * kStages * 4;
};

// Warps work alone: each has every fourth 16 positions of a unit, copies their rows ahead into its own part of shared memory, and keeps
// its own top, sum and weighted sum.  Scores are formed as keys x queries (S^T: 16 keys by 8 query heads) and outputs as values x weights
// (O^T: 16 columns by 8 heads), so that 8 query heads fill a product.  A thread of quad g, place t has keys g and g + 8 of heads 2t and
// 2t + 1; turning its weights as a matrix makes them the second operand of the second product.
template <typename T, int D, int NT, bool WHOLE_PAGES>
__global__ void __launch_bounds__(kThreads, mma_shape<D, NT>::kResident)
mma_kernel(cache_view c, work_view w, rows_view queries, rows_view out, float* lse, float scale_log2, parts_view parts)
{
  using shape       = mma_shape<D, NT>;
  constexpr int S   = shape::kStages;
  constexpr int PR  = D / 8;  // pieces of a row in shared memory
  extern __shared__ __align__(128) char smem[];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t g = lane >> 2, t = lane & 3u;
  float* s_acc      = reinterpret_cast<float*>(smem);
  float2* s_stats   = reinterpret_cast<float2*>(smem + shape::kStatsAt);
  uint32_t* s_mask  = reinterpret_cast<uint32_t*>(smem + shape::kMaskAt) + warp * S;
  const uint32_t buffers = shared_address(smem) + warp * (S * shape::kStage);
  const uint32_t s_q     = shared_address(smem + shape::kQAt);
  const uint32_t pieces  = c.dim / 8;
  chain_begin();

  each_unit<T, shape::kTile>(
    c, w, out, lse, parts, s_acc, shape::kAccRow, s_stats,
    [&](uint32_t sequence, uint32_t unit, uint32_t first, uint32_t end, uint32_t tile0, uint32_t tile1) {
      const uint32_t head = unit / w.n_blocks_of, of = unit - head * w.n_blocks_of;
      const uint32_t rows  = min(uint32_t(shape::kRows), w.group - of * shape::kRows);
      const uint32_t head0 = head * w.group + of * shape::kRows;
      const int32_t* table = w.pages + int64_t(sequence) * w.table_stride;
      const char* keys     = c.keys + int64_t(head) * c.k_head * 2;
      const char* values   = c.values + int64_t(head) * c.v_head * 2;
      const uint32_t base  = (first & ~15u) + warp * 16u;
      const uint32_t mine  = lane & 15u;  // the row whose place this lane finds

      // ahead of the copies: pages, then words of the filter
      auto page_at = [&](uint32_t tile) -> int32_t {
        const uint32_t at = base + tile * shape::kTile + mine;
        if (tile >= tile1 || at < first || at >= end) { return -1; }
        uint32_t column, place;
        split_place(at, c.page_size, c.page_shift, column, place);
        return page_of(table, w.width, column, c.n_pages);
      };
      auto word_at = [&](uint32_t tile, int32_t page) -> uint32_t {
        if (c.filter == nullptr || page < 0) { return 0u; }
        uint32_t column, place;
        split_place(base + tile * shape::kTile + mine, c.page_size, c.page_shift, column, place);
        return c.filter[(int64_t(page) * c.page_size + place) >> 5];
      };
      auto copy_rows = [&](uint32_t tile, int32_t page, uint32_t word) {
        const uint32_t stage = (tile - tile0) % S;
        if (tile < tile1) {
          uint32_t column, place;
          split_place(base + tile * shape::kTile + mine, c.page_size, c.page_shift, column, place);
          bool there = page >= 0;
          if (there && c.filter != nullptr) { there = (word >> (uint32_t(int64_t(page) * c.page_size + place) & 31u)) & 1u; }
          const uint32_t mask = __ballot_sync(kAllLanes, there) & 0xFFFFu;
          if (lane == 0) { s_mask[stage] = mask; }
          if (mask != 0u) {
            const uint32_t to = buffers + stage * shape::kStage;
            int64_t k_at, v_at;
            if constexpr (WHOLE_PAGES) {
              // all 16 rows are in the page of any of them
              const int l        = __ffs(int(mask)) - 1;
              const int64_t p    = __shfl_sync(kAllLanes, page, l);
              const int64_t from = int64_t(place) - mine;  // of row 0, whichever lane asks
              k_at               = p * c.k_page + from * c.k_token;
              v_at               = p * c.v_page + from * c.v_token;
            } else {
              k_at = int64_t(page) * c.k_page + int64_t(place) * c.k_token;
              v_at = int64_t(page) * c.v_page + int64_t(place) * c.v_token;
            }
#pragma unroll
            for (int i = 0; i < 16 * PR / 32; i++) {
              const uint32_t piece = lane % PR, row = (lane + 32u * i) / PR;
              int64_t k = k_at, v = v_at;
              if constexpr (WHOLE_PAGES) {
                k += row * c.k_token;
                v += row * c.v_token;
              } else {
                k = __shfl_sync(kAllLanes, k_at, row);
                v = __shfl_sync(kAllLanes, v_at, row);
              }
              const bool read   = ((mask >> row) & 1u) != 0u && piece < pieces;
              const uint32_t at = to + row * shape::kRowBytes + ((piece ^ (row & 7u)) << 4);
              copy_piece(at, read ? keys + k * 2 + piece * 16 : c.keys, read);
              copy_piece(at + 16 * shape::kRowBytes, read ? values + v * 2 + piece * 16 : c.values, read);
            }
          }
        }
        copies_end_group();
      };

      // queries: the second operand of the first product
      uint32_t q[shape::kQInRegs ? NT : 1][shape::kQInRegs ? D / 16 : 1][2];
      if constexpr (shape::kQInRegs) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const uint32_t r    = n * 8 + g;
          const char* row     = queries.data + (int64_t(sequence) * queries.row + int64_t(head0 + r) * queries.head) * 2;
#pragma unroll
          for (int k = 0; k < D / 16; k++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const uint32_t column = k * 16 + h * 8 + 2 * t;
              q[n][k][h]            = r < rows && column < c.dim ? *reinterpret_cast<const uint32_t*>(row + column * 2) : 0u;
            }
          }
        }
      } else {
        for (uint32_t i = threadIdx.x; i < uint32_t(shape::kRows * PR); i += kThreads) {
          const uint32_t r = i / PR, piece = i % PR;
          uint4 x          = make_uint4(0, 0, 0, 0);
          if (r < rows && piece < pieces) {
            x = reinterpret_cast<const uint4*>(queries.data + (int64_t(sequence) * queries.row + int64_t(head0 + r) * queries.head) * 2)[piece];
          }
          *reinterpret_cast<uint4*>(smem + shape::kQAt + r * shape::kRowBytes + ((piece ^ (r & 7u)) << 4)) = x;
        }
        __syncthreads();
      }

      float acc[NT][D / 16][4] = {};
      float top[NT][2], sum[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        top[n][0] = top[n][1] = -INFINITY;
        sum[n][0] = sum[n][1] = 0.0f;
      }

      int32_t page_0 = page_at(tile0), page_1 = page_at(tile0 + 1);
      uint32_t word_0 = word_at(tile0, page_0);
      auto advance    = [&](uint32_t tile) {  // copies of `tile`, the word of the next, the page of the one after
        const int32_t page_2  = page_at(tile + 2);
        const uint32_t word_1 = word_at(tile + 1, page_1);
        copy_rows(tile, page_0, word_0);
        page_0 = page_1;
        page_1 = page_2;
        word_0 = word_1;
      };
#pragma unroll
      for (int i = 0; i < S; i++) { advance(tile0 + i); }

      for (uint32_t tile = tile0; tile < tile1; tile++) {
        copies_wait<S - 1>();
        __syncwarp();
        const uint32_t stage = (tile - tile0) % S;
        const uint32_t mask  = s_mask[stage];
        if (mask != 0u) {
          const uint32_t k_rows = buffers + stage * shape::kStage, v_rows = k_rows + 16 * shape::kRowBytes;
          float s[NT][4] = {};
#pragma unroll
          for (int k = 0; k < D / 16; k++) {
            uint32_t a[4];
            const uint32_t row = (lane & 7u) + (lane & 8u), piece = k * 2 + (lane >> 4);
            load_matrices(a, k_rows + row * shape::kRowBytes + ((piece ^ (row & 7u)) << 4));
            if constexpr (shape::kQInRegs) {
#pragma unroll
              for (int n = 0; n < NT; n++) { multiply_add<T>(s[n], a, q[n][k][0], q[n][k][1]); }
            } else {
              // two eights of heads at a time: matrices (heads 0-7, columns 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15)
#pragma unroll
              for (int n = 0; n < NT; n += 2) {
                uint32_t b[4];
                const uint32_t r = n * 8 + (lane & 7u) + ((lane >> 4) << 3), p = k * 2 + ((lane >> 3) & 1u);
                load_matrices(b, s_q + r * shape::kRowBytes + ((p ^ (r & 7u)) << 4));
                multiply_add<T>(s[n], a, b[0], b[1]);
                multiply_add<T>(s[n + 1], a, b[2], b[3]);
              }
            }
          }
          const bool k0 = ((mask >> g) & 1u) != 0u, k1 = ((mask >> (g + 8)) & 1u) != 0u;
          float next[NT][2];
          bool higher = false;
#pragma unroll
          for (int n = 0; n < NT; n++) {
            s[n][0] = k0 ? s[n][0] * scale_log2 : -INFINITY;
            s[n][1] = k0 ? s[n][1] * scale_log2 : -INFINITY;
            s[n][2] = k1 ? s[n][2] * scale_log2 : -INFINITY;
            s[n][3] = k1 ? s[n][3] * scale_log2 : -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; h++) {
              float m = fmaxf(s[n][h], s[n][h + 2]);
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) { m = fmaxf(m, __shfl_xor_sync(kAllLanes, m, o)); }
              next[n][h] = fmaxf(top[n][h], m);
              higher     = higher || next[n][h] > top[n][h];
            }
          }
          if (__any_sync(kAllLanes, higher)) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
              float keep[2];
#pragma unroll
              for (int h = 0; h < 2; h++) {
                keep[h]   = exp2f(top[n][h] - finite_top(next[n][h]));
                top[n][h] = next[n][h];
                sum[n][h] *= keep[h];
              }
#pragma unroll
              for (int d = 0; d < D / 16; d++) {
                acc[n][d][0] *= keep[0];
                acc[n][d][1] *= keep[1];
                acc[n][d][2] *= keep[0];
                acc[n][d][3] *= keep[1];
              }
            }
          }
          uint32_t high[NT][2], low[NT][2];
#pragma unroll
          for (int n = 0; n < NT; n++) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              p[e] = exp2f(s[n][e] - (finite_top(top[n][e & 1]) - halves<T>::kShift));
              sum[n][e & 1] += p[e];
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
              high[n][h]       = halves<T>::pack(p[2 * h] * halves<T>::kBelow, p[2 * h + 1] * halves<T>::kBelow);
              const float2 was = halves<T>::unpack(high[n][h]);
              low[n][h]        = turn_matrix(halves<T>::pack(p[2 * h] - was.x, p[2 * h + 1] - was.y));
              high[n][h]       = turn_matrix(high[n][h]);
            }
          }
#pragma unroll
          for (int d = 0; d < D / 16; d++) {
            uint32_t a[4];
            const uint32_t row = (lane & 7u) + ((lane >> 4) << 3), piece = d * 2 + ((lane >> 3) & 1u);
            load_matrices_turned(a, v_rows + row * shape::kRowBytes + ((piece ^ (row & 7u)) << 4));
#pragma unroll
            for (int n = 0; n < NT; n++) {
              multiply_add<T>(acc[n][d], a, high[n][0], high[n][1]);
              multiply_add<T>(acc[n][d], a, low[n][0], low[n][1]);
            }
          }
        }
        __syncwarp();
        advance(tile + S);
      }
      copies_wait<0>();
      __syncthreads();  // shared memory changes hands: from rows to sums
      const float unshift = exp2f(-halves<T>::kShift);
#pragma unroll
      for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) { sum[n][h] += __shfl_xor_sync(kAllLanes, sum[n][h], o); }
          const uint32_t r = n * 8 + 2 * t + h;
          if (g == 0) { s_stats[warp * shape::kRows + r] = make_float2(top[n][h], sum[n][h] * unshift); }
          float* a = s_acc + (warp * shape::kRows + r) * shape::kAccRow + g;
#pragma unroll
          for (int d = 0; d < D / 16; d++) {
            a[d * 16]     = acc[n][d][h] * unshift;
            a[d * 16 + 8] = acc[n][d][h + 2] * unshift;
          }
        }
      }
    });
  empty_rows<T, shape::kTile>(c, w, out, lse);
}

// ---- 32-bit rows --------------------------------------------------------------------------------------------------------------

// A lane group of LANES lanes has a row's 16-byte pieces, PIECES of them per lane, and reads four rows at a time, keys and values, for the R
// query heads of a unit; products and sums are in 32 bits.
template <int LANES, int PIECES, int R>
__global__ void __launch_bounds__(kThreads)
rows32_kernel(cache_view c, work_view w, rows_view queries, rows_view out, float* lse, float scale_log2, parts_view parts)
{
  constexpr int E      = 4;
  constexpr int GROUPS = 32 / LANES;
  constexpr int U      = 4;
  constexpr int TILE   = kWarps * 32;
  constexpr int COLS   = LANES * PIECES * E;
  __shared__ __align__(16) float s_acc[kWarps * R * COLS];
  __shared__ float2 s_stats[kWarps * R];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t group = lane / LANES, gl = lane % LANES;
  const uint32_t pieces = c.dim / E;
  chain_begin();

  each_unit<float, TILE>(
    c, w, out, lse, parts, s_acc, COLS, s_stats,
    [&](uint32_t sequence, uint32_t unit, uint32_t first, uint32_t end, uint32_t tile0, uint32_t tile1) {
      const uint32_t head = unit / w.n_blocks_of, of = unit - head * w.n_blocks_of;
      const uint32_t rows  = min(uint32_t(R), w.group - of * R);
      const uint32_t head0 = head * w.group + of * R;
      const int32_t* table = w.pages + int64_t(sequence) * w.table_stride;
      const char* keys     = c.keys + int64_t(head) * c.k_head * 4;
      const char* values   = c.values + int64_t(head) * c.v_head * 4;
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
            x = reinterpret_cast<const uint4*>(queries.data + (int64_t(sequence) * queries.row + int64_t(head0 + r) * queries.head) * 4)[j];
          }
          piece_to_floats<float>(x, q[r][p]);
        }
      }
      const uint32_t base = (first & ~15u) + warp * 32u + lane;
      auto place_of       = [&](uint32_t tile, int64_t& k_at, int64_t& v_at) {
        const uint32_t at = base + tile * TILE;
        k_at              = -1;
        v_at              = 0;
        if (tile >= tile1 || at < first || at >= end) { return; }
        uint32_t column, place;
        split_place(at, c.page_size, c.page_shift, column, place);
        const int32_t page = page_of(table, w.width, column, c.n_pages);
        if (page < 0 || !slot_allowed(c, int64_t(page) * c.page_size + place)) { return; }
        k_at = int64_t(page) * c.k_page + int64_t(place) * c.k_token;
        v_at = int64_t(page) * c.v_page + int64_t(place) * c.v_token;
      };
      for (uint32_t tile = tile0; tile < tile1; tile++) {
        int64_t k_at, v_at;
        place_of(tile, k_at, v_at);
        if (!__any_sync(kAllLanes, k_at >= 0)) { continue; }
#pragma unroll 1
        for (int j0 = 0; j0 < 32; j0 += U * GROUPS) {
          uint4 k[U][PIECES], v[U][PIECES];
          bool ok[U];
#pragma unroll
          for (int u = 0; u < U; u++) {
            const int from   = j0 + u * GROUPS + int(group);
            const int64_t kr = __shfl_sync(kAllLanes, k_at, from);
            const int64_t vr = __shfl_sync(kAllLanes, v_at, from);
            ok[u]            = kr >= 0;
#pragma unroll
            for (int p = 0; p < PIECES; p++) {
              const uint32_t j = gl + p * LANES;
              k[u][p] = v[u][p] = make_uint4(0, 0, 0, 0);
              if (ok[u] && j < pieces) {
                k[u][p] = __ldg(reinterpret_cast<const uint4*>(keys + kr * 4) + j);
                v[u][p] = __ldg(reinterpret_cast<const uint4*>(values + vr * 4) + j);
              }
            }
          }
#pragma unroll
          for (int r = 0; r < R; r++) {
            float score[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
              float s = 0.0f;
#pragma unroll
              for (int p = 0; p < PIECES; p++) {
                float x[E];
                piece_to_floats<float>(k[u][p], x);
#pragma unroll
                for (int e = 0; e < E; e++) { s = fmaf(q[r][p][e], x[e], s); }
              }
#pragma unroll
              for (int o = LANES / 2; o > 0; o >>= 1) { s += __shfl_xor_sync(kAllLanes, s, o); }
              score[u] = ok[u] ? s * scale_log2 : -INFINITY;
            }
            float next = top[r];
#pragma unroll
            for (int u = 0; u < U; u++) { next = fmaxf(next, score[u]); }
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
              const float weight = exp2f(score[u] - safe);
              sum[r] += weight;
#pragma unroll
              for (int p = 0; p < PIECES; p++) {
                float x[E];
                piece_to_floats<float>(v[u][p], x);
#pragma unroll
                for (int e = 0; e < E; e++) { acc[r][p][e] = fmaf(weight, x[e], acc[r][p][e]); }
              }
            }
          }
        }
      }
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
            *reinterpret_cast<float4*>(s_acc + (warp * R + r) * COLS + (gl + p * LANES) * E) =
              make_float4(acc[r][p][0], acc[r][p][1], acc[r][p][2], acc[r][p][3]);
          }
        }
        if (lane == 0) { s_stats[warp * R + r] = make_float2(top[r], sum[r]); }
      }
    });
  empty_rows<float, TILE>(c, w, out, lse);
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

// What a call launches, by type and sizes alone.
struct plan {
  uint32_t rows;      // query heads of a unit
  uint32_t tile;
  uint32_t resident;  // blocks of an SM
};

uint32_t padded(uint32_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

plan plan_of(elem type, uint32_t group, uint32_t dim)
{
  if (type == elem::f32) {
    const uint32_t rows = group > 2 && dim > 128 ? 4 : group > 4 ? 8 : group > 2 ? 4 : group;
    return {rows, kWarps * 32, rows == 1 ? 6u : rows == 2 ? 4u : dim > 128 ? 2u : 3u};  // what their registers leave room for
  }
  const uint32_t d  = padded(dim);
  const uint32_t nt = group <= 8 ? 1 : group <= 16 || d == 256 ? 2 : 4;
  return {8 * nt, kWarps * 16, d == 256 ? 1u : nt == 4 ? 2u : 3u};
}

uint64_t most_tiles(const plan& p, uint64_t capacity, int64_t window)
{
  // a window may begin anywhere in 16 positions
  const uint64_t positions = window > 0 && uint64_t(window) < capacity ? std::min(capacity, uint64_t(window) + 15) : capacity;
  return ceildiv<uint64_t>(positions, p.tile);
}

uint32_t blocks_of(const resources& res, const plan& p, uint64_t units, uint64_t tiles)
{
  return uint32_t(std::max<uint64_t>(1, std::min<uint64_t>(uint64_t(res.sm_count) * p.resident, units * std::max<uint64_t>(tiles, 1))));
}

}  // namespace

size_t attention_workspace(const resources& res, elem type, uint32_t n_sequences, uint32_t n_query_heads, uint32_t n_heads, uint32_t dim,
                           uint64_t capacity, int64_t window)
{
  const plan p          = plan_of(type, n_query_heads / n_heads, dim);
  const uint64_t tiles  = most_tiles(p, capacity, window);
  const uint64_t units  = uint64_t(n_sequences) * n_heads * ceildiv(n_query_heads / n_heads, p.rows);
  return tiles <= 1 ? 0 : part_bytes(blocks_of(res, p, units, tiles), p.rows, dim);
}

void attention(resources& res, const attention_args& a)
{
  if (a.n_sequences == 0) { return; }
  const cache_view& c  = a.cache;
  const uint32_t group = a.n_query_heads / c.n_heads;
  const plan p         = plan_of(a.type, group, c.dim);
  work_view w{};
  w.pages        = a.pages;
  w.lengths      = a.lengths;
  w.table_stride = a.table_stride;
  w.window       = a.window;
  w.n_sequences  = a.n_sequences;
  w.width        = a.table_width;
  w.group        = group;
  w.n_blocks_of  = ceildiv(group, p.rows);
  w.n_units      = c.n_heads * w.n_blocks_of;
  const uint64_t units  = uint64_t(w.n_units) * a.n_sequences;
  const uint64_t tiles  = most_tiles(p, uint64_t(a.table_width) * c.page_size, a.window);
  const uint32_t blocks = blocks_of(res, p, units, tiles);
  parts_view parts{};
  parts.rows = p.rows;
  if (tiles > 1) { parts = parts_at(a.workspace, blocks, p.rows, c.dim); }
  const float scale = a.scale * kLog2E;
  auto go           = [&](auto kernel, size_t smem) {
    if (smem > 48 * 1024) { ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem); }
    launch_chained(kernel, dim3(blocks), kThreads, smem, res.stream, c, w, a.queries, a.out, a.lse, scale, parts);
    CUDA_TRY(cudaGetLastError());
    res.launches++;
  };
  auto mma_pages = [&](auto type, auto d, auto nt) {
    using T          = decltype(type);
    constexpr int D  = decltype(d)::value;
    constexpr int NT = decltype(nt)::value;
    if (c.page_size % 16 == 0) {
      go(mma_kernel<T, D, NT, true>, mma_shape<D, NT>::kShared);
    } else {
      go(mma_kernel<T, D, NT, false>, mma_shape<D, NT>::kShared);
    }
  };
  auto mma = [&](auto type) {
    using std::integral_constant;
    const uint32_t d = padded(c.dim), nt = p.rows / 8;
    auto by_rows = [&](auto cols) {
      if (nt == 1) {
        mma_pages(type, cols, integral_constant<int, 1>{});
      } else if (nt == 2) {
        mma_pages(type, cols, integral_constant<int, 2>{});
      } else if constexpr (decltype(cols)::value <= 128) {
        mma_pages(type, cols, integral_constant<int, 4>{});
      }
    };
    if (d == 64) {
      by_rows(integral_constant<int, 64>{});
    } else if (d == 128) {
      by_rows(integral_constant<int, 128>{});
    } else {
      by_rows(integral_constant<int, 256>{});
    }
  };
  auto rows32 = [&](auto lanes, auto pieces) {
    constexpr int L = decltype(lanes)::value, P = decltype(pieces)::value;
    if (p.rows == 1) {
      go(rows32_kernel<L, P, 1>, 0);
    } else if (p.rows == 2) {
      go(rows32_kernel<L, P, 2>, 0);
    } else if (p.rows == 4) {
      go(rows32_kernel<L, P, 4>, 0);
    } else if constexpr (P == 1) {
      go(rows32_kernel<L, P, 8>, 0);
    }
  };
  if (a.type == elem::f16) {
    mma(__half{});
  } else if (a.type == elem::bf16) {
    mma(__nv_bfloat16{});
  } else {
    using std::integral_constant;
    const uint32_t n = c.dim / 4;
    if (n <= 8) {
      rows32(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    } else if (n <= 16) {
      rows32(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    } else if (n <= 32) {
      rows32(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    } else {
      rows32(integral_constant<int, 32>{}, integral_constant<int, 2>{});
    }
  }
  if (tiles <= 1 || blocks == 1) { return; }
  // Few units have many parts each: a block per row and all of its warps on the row's parts; else a warp per row.
  const bool many = blocks / units >= 16;
  auto join       = [&](auto type) {
    using T = decltype(type);
    if (many) {
      launch_chained(join_kernel<T, kJoinWarps>, dim3(blocks - 1, std::min(p.rows, group)), kJoinWarps * 32, 0, res.stream, w, parts, c.dim, c.n_heads,
                     a.out, a.lse);
    } else {
      launch_chained(join_kernel<T, 1>, dim3(blocks - 1, 1), kJoinWarps * 32, 0, res.stream, w, parts, c.dim, c.n_heads, a.out, a.lse);
    }
    CUDA_TRY(cudaGetLastError());
    res.launches++;
  };
  if (a.type == elem::f16) {
    join(__half{});
  } else if (a.type == elem::bf16) {
    join(__nv_bfloat16{});
  } else {
    join(float{});
  }
}

}  // namespace cuvs_b200::kv
