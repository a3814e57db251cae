// Attention of one token per sequence to the 16-bit rows of its sequence in a paged cache.
//
//   S_j = scale q.k_j over the positions j that may be attended,  lse = log sum exp S_j,  o = sum exp(S_j - lse) v_j
//
// What bounds it: the rows are read once, 4 operations for each 16-bit key and value and query head, so with 8 query heads to a key head HBM
// at 6.5 TB/s asks for 52 TFLOP/s: more than the FP32 pipes have left beside the conversions, a fraction of what mma.sync has, which
// takes its operands from registers without tensor memory's detour.  Everything here serves keeping loads in flight.  32 requests of up to 16,384
// tokens, 8 key heads of 8, 128 columns bf16: 149 us with the join for 894 MB (6.0 TB/s); one of 250,000 tokens, 4 key heads of 7: 89 us for 512 MB.
#include "kv_attention.hpp"

#include <algorithm>
#include <type_traits>

namespace cuvs_b200::kv {

namespace {

// ---- 16-bit rows: tensor cores ------------------------------------------------------------------------------------------------

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

// A weight of 32 bits goes into the product with the values as the sum of 16-bit numbers, so that nothing is lost beside what the exponential
// itself is off by: a row of the output is rounded once, at its end.  The products, twice or three times the mma.sync of one number, are to spare.
// No summand is 0 where the weight is not: 0 times an infinite value would be no number.
// `scale`: what weights are held times, `back` = 1 / scale, `to_room`: from there to what sums are left for others to join with.
template <typename T>
struct summands;
template <>
struct summands<__half> {
  // 11 bits, cut off, and the rest rounded to 11 bits: to 2^-22 of the weight.  Weights are held times 2^14, so that small ones keep their digits
  // above fp16's smallest number: it is 2^-38 of the largest weight, and what is below counts for nothing.
  // (Sums of 2^31 values of 65,504 are far from the ends of 32 bits: no room is made for them.)
  static constexpr int kCount = 2;
  static __device__ __forceinline__ float scale(const work_view&) { return 16384.0f; }
  static __device__ __forceinline__ float back(const work_view&) { return 1.0f / 16384.0f; }
  static __device__ __forceinline__ float to_room(const work_view& w) { return w.room * (1.0f / 16384.0f); }
  static __device__ __forceinline__ void split(float a, float b, uint32_t (&part)[kCount])
  {
    constexpr float kSmallest = 5.9604644775390625e-8f;  // 2^-24
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(part[0]) : "f"(b), "f"(a));
    const float2 high = __half22float2(*reinterpret_cast<const __half2*>(&part[0]));
    const __half2 low = __floats2half2_rn(fmaxf(a - high.x, fminf(a, kSmallest)), fmaxf(b - high.y, fminf(b, kSmallest)));
    part[1]           = *reinterpret_cast<const uint32_t*>(&low);
  }
};
template <>
struct summands<__nv_bfloat16> {
  // Three times 8 bits, cut off: all of the weight.  (Two of them, rounded, left the weights of a batch of 32 requests 1.7e-5 off on average: 2^-16.)
  static constexpr int kCount = 3;
  static __device__ __forceinline__ float scale(const work_view& w) { return w.room; }
  static __device__ __forceinline__ float back(const work_view& w) { return w.back; }
  static __device__ __forceinline__ float to_room(const work_view&) { return 1.0f; }
  static __device__ __forceinline__ uint32_t upper(float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); }
  static __device__ __forceinline__ float cut(float a) { return __uint_as_float(__float_as_uint(a) & 0xFFFF0000u); }
  static __device__ __forceinline__ void split(float a, float b, uint32_t (&part)[kCount])
  {
    constexpr float kNothing = 7.52316384526264e-37f;  // 2^-120
    const float a1 = fmaxf(a - cut(a), kNothing), b1 = fmaxf(b - cut(b), kNothing);
    const float a2 = fmaxf(a1 - cut(a1), kNothing), b2 = fmaxf(b1 - cut(b1), kNothing);
    part[0] = upper(a, b);
    part[1] = upper(a1, b1);
    part[2] = upper(a2, b2);
  }
};

// D: columns of a row in shared memory (64, 128, 256; what is behind the row's end is 0).  NT: query heads of a unit, in eights.
template <int D, int NT, int WARPS>
struct mma_shape {
  static constexpr int kRows     = 8 * NT;
  static constexpr int kChunk    = 16;
  static constexpr int kStages   = D == 64 ? 4 : D == 256 && NT == 1 ? 3 : 2;
  static constexpr bool kQInRegs = D * NT <= 256;
  static constexpr int kResident = WARPS > kSmall || D == 256 ? 1 : NT == 4 ? 2 : 3;  // blocks of an SM
  static constexpr int kRowBytes = D * 2;
  static constexpr int kStage    = 2 * 16 * kRowBytes;                       // 16 keys, 16 values
  static constexpr int kAccRow   = D + 4;                                    // floats: lanes of a store on different banks
  static constexpr int kBuffers  = WARPS * kStages * kStage;
  static constexpr int kAcc      = WARPS * kRows * kAccRow * 4;
  static constexpr int kQBytes   = kQInRegs ? 0 : kRows * kRowBytes;       // of a warp
  static constexpr int kStatsAt  = kBuffers > kAcc ? kBuffers : kAcc;
  static constexpr int kJoinedAt = kStatsAt + WARPS * kRows * 8;
  static constexpr int kQAt      = kJoinedAt + kRows * 8;
  static constexpr int kMaskAt   = kQAt + WARPS * kQBytes;
  static constexpr int kPortion  = (D / 16 * 4 + 4) * 32;                    // floats that a warp sends another: the sums of eight heads
  static constexpr int kExchangeAt = kMaskAt + WARPS * 16;
  static constexpr int kShared   = kExchangeAt + (WARPS == kSmall ? WARPS / 2 * kPortion * 4 : 0);
};

// Warps work alone: each copies its rows ahead into its own part of shared memory, and keeps its own top, sum and weighted sum.  Scores are
// formed as keys x queries (S^T: 16 keys by 8 query heads) and outputs as values x weights (O^T: 16 columns by 8 heads), so that 8 query heads fill
// a product.  A thread of quad g, place t has keys g and g + 8 of heads 2t and 2t + 1; turning its weights as a matrix makes them the second
// operand of the second product.
template <typename T, int D, int NT, int WARPS, bool WHOLE_PAGES>
struct mma_hooks {
  using shape                    = mma_shape<D, NT, WARPS>;
  static constexpr int PR        = D / 8;   // pieces of a row in shared memory
  static constexpr int ROWS      = 32 / PR; // a copy of a warp: one piece of every lane, so many rows
  static constexpr int kPortion  = shape::kPortion;
  static constexpr int kPortions = NT;

  const cache_view& c;
  const work_view& w;
  const rows_view& queries;
  const result_view& result;
  const parts_view& parts;
  const block_state& state;
  char* smem;
  float scale_log2;
  uint32_t warp, lane, g, t;
  uint32_t buffers, s_q;
  // Copies: a lane has one piece of every ROWS-th row.  Pieces stand in a row's place by place ^ (row & 7), so that eight rows' pieces of one
  // column lie on different banks; behind the row's end they are 0.
  uint32_t copy_row, copy_swizzle, copy_bytes, copy_from;
  const char *keys, *values;
  float acc[NT][D / 16][4], top[NT][2], sum[NT][2];
  uint32_t q[shape::kQInRegs ? NT : 1][shape::kQInRegs ? D / 16 : 1][2];  // the second operand of the first product

  __device__ __forceinline__ mma_hooks(const cache_view& c_, const work_view& w_, const rows_view& queries_, const result_view& result_,
                                       const parts_view& parts_, const block_state& state_, char* smem_, float scale_log2_)
    : c(c_), w(w_), queries(queries_), result(result_), parts(parts_), state(state_), smem(smem_), scale_log2(scale_log2_),
      warp(threadIdx.x >> 5), lane(threadIdx.x & 31u), g((threadIdx.x & 31u) >> 2), t(threadIdx.x & 3u)
  {
    buffers      = shared_address(smem) + warp * (shape::kStages * shape::kStage);
    s_q          = shared_address(smem + shape::kQAt);
    copy_row     = lane / PR;
    copy_swizzle = ((lane % PR) ^ copy_row) << 4;
    copy_bytes   = lane % PR < c.dim / 8 ? 16u : 0u;
    copy_from    = lane % PR < c.dim / 8 ? (lane % PR) * 16u : 0u;
  }

  __device__ __forceinline__ void attach(uint32_t unit)
  {
    const uint32_t head = unit / w.n_blocks_of;
    keys                = c.keys + int64_t(head) * c.k_head * 2 + copy_from;
    values              = c.values + int64_t(head) * c.v_head * 2 + copy_from;
  }

  __device__ __forceinline__ uint32_t copy(uint32_t stage, uint32_t page, uint32_t place, bool there)
  {
    const uint32_t mask = __ballot_sync(kAllLanes, there) & 0xFFFFu;
    if (mask == 0u) { return 0u; }
    const uint32_t to = buffers + stage * shape::kStage + copy_row * shape::kRowBytes;
    uint32_t k_at, v_at;
    const char *k_from, *v_from;
    if constexpr (WHOLE_PAGES) {
      // all 16 rows are in the page of any of them, whether they are to be read or not; `place` is that of the lane's own row
      page   = __shfl_sync(kAllLanes, page, __ffs(int(mask)) - 1);
      place  = place - (lane & 15u) + copy_row;
      k_from = keys + (uint64_t(page * c.k_page_units + place * c.k_token_units) << c.unit_shift);
      v_from = values + (uint64_t(page * c.v_page_units + place * c.v_token_units) << c.unit_shift);
    } else {
      k_at = there ? page * c.k_page_units + place * c.k_token_units : 0u;
      v_at = there ? page * c.v_page_units + place * c.v_token_units : 0u;
    }
    const uint64_t k_rows_on = uint64_t(c.k_token_units * ROWS) << c.unit_shift, v_rows_on = uint64_t(c.v_token_units * ROWS) << c.unit_shift;
#pragma unroll
    for (int i = 0; i < 16 / ROWS; i++) {
      const uint32_t at = to + i * (ROWS * shape::kRowBytes) + (copy_swizzle ^ ((i * ROWS & 7) << 4));
      if constexpr (!WHOLE_PAGES) {
        k_from = keys + (uint64_t(__shfl_sync(kAllLanes, k_at, copy_row + i * ROWS)) << c.unit_shift);
        v_from = values + (uint64_t(__shfl_sync(kAllLanes, v_at, copy_row + i * ROWS)) << c.unit_shift);
      }
      const uint32_t bytes = ((mask >> (copy_row + i * ROWS)) & 1u) != 0u ? copy_bytes : 0u;
      copy_piece(at, k_from, bytes);
      copy_piece(at + 16 * shape::kRowBytes, v_from, bytes);
      if constexpr (WHOLE_PAGES) {
        k_from += k_rows_on;
        v_from += v_rows_on;
      }
    }
    return mask;
  }

  __device__ __forceinline__ void start(uint32_t sequence, uint32_t unit)
  {
    const uint32_t head = unit / w.n_blocks_of, of = unit - head * w.n_blocks_of;
    const uint32_t rows = min(uint32_t(shape::kRows), w.group - of * shape::kRows), head0 = head * w.group + of * shape::kRows;
    const char* first   = queries.data + (int64_t(sequence) * queries.row + int64_t(head0) * queries.head) * 2;
    if constexpr (shape::kQInRegs) {
#pragma unroll
      for (int n = 0; n < NT; n++) {
        const uint32_t r = n * 8 + g;
        const char* row  = first + int64_t(r) * queries.head * 2;
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
      // the warp's own copy: warps are not at the same piece at the same time
      __syncwarp();
      for (uint32_t i = lane; i < uint32_t(shape::kRows * PR); i += 32) {
        const uint32_t r = i / PR, piece = i % PR;
        uint4 x          = make_uint4(0, 0, 0, 0);
        if (r < rows && piece < c.dim / 8) { x = reinterpret_cast<const uint4*>(first + int64_t(r) * queries.head * 2)[piece]; }
        *reinterpret_cast<uint4*>(smem + shape::kQAt + warp * shape::kQBytes + r * shape::kRowBytes + ((piece ^ (r & 7u)) << 4)) = x;
      }
      __syncwarp();
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int d = 0; d < D / 16; d++) { acc[n][d][0] = acc[n][d][1] = acc[n][d][2] = acc[n][d][3] = 0.0f; }
      top[n][0] = top[n][1] = -INFINITY;
      sum[n][0] = sum[n][1] = 0.0f;
    }
  }

  __device__ __forceinline__ void consume(uint32_t stage, uint32_t mask)
  {
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
          load_matrices(b, s_q + warp * shape::kQBytes + r * shape::kRowBytes + ((p ^ (r & 7u)) << 4));
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
          keep[h]   = power_of_2(top[n][h] - finite_top(next[n][h]));
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
    constexpr int N = summands<T>::kCount;
    uint32_t part[NT][2][N];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        p[e] = power_of_2(s[n][e] - finite_top(top[n][e & 1])) * summands<T>::scale(w);
        sum[n][e & 1] += p[e];
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        summands<T>::split(p[2 * h], p[2 * h + 1], part[n][h]);
#pragma unroll
        for (int i = 0; i < N; i++) { part[n][h][i] = turn_matrix(part[n][h][i]); }
      }
    }
#pragma unroll
    for (int d = 0; d < D / 16; d++) {
      uint32_t a[4];
      const uint32_t row = (lane & 7u) + ((lane >> 4) << 3), piece = d * 2 + ((lane >> 3) & 1u);
      load_matrices_turned(a, v_rows + row * shape::kRowBytes + ((piece ^ (row & 7u)) << 4));
#pragma unroll
      for (int n = 0; n < NT; n++) {
        // The tensor core cuts off what it adds to a sum, always towards 0: it gets the products of these keys alone, and what they come to is
        // added in 32 bits, rounded.  (With a sum of all keys outputs of 300 sequences of 200,000 tokens were 2.9e-4 too small in fp16, 4.6e-4 in
        // bf16.  It costs 8% where 16 query heads or more go with a key head, 0.5% where HBM is what counts.)
        float t[4] = {};
#pragma unroll
        for (int i = 0; i < N; i++) { multiply_add<T>(t, a, part[n][0][i], part[n][1][i]); }
#pragma unroll
        for (int e = 0; e < 4; e++) { acc[n][d][e] += t[e]; }
      }
    }
  }

  __device__ __forceinline__ void close()
  {
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) { sum[n][h] += __shfl_xor_sync(kAllLanes, sum[n][h], o); }
      }
    }
  }

  // a lane's own values to the same lane of another warp
  __device__ __forceinline__ void send(int n, float* to) const
  {
    float4* at = reinterpret_cast<float4*>(to) + lane;
    at[0]      = make_float4(top[n][0], top[n][1], sum[n][0], sum[n][1]);
#pragma unroll
    for (int d = 0; d < D / 16; d++) { at[32 * (d + 1)] = make_float4(acc[n][d][0], acc[n][d][1], acc[n][d][2], acc[n][d][3]); }
  }
  __device__ __forceinline__ void receive(int n, const float* from)
  {
    const float4* at   = reinterpret_cast<const float4*>(from) + lane;
    const float4 stats = at[0];
    float own[2], theirs[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const float other = h == 0 ? stats.x : stats.y, next = fmaxf(top[n][h], other), safe = finite_top(next);
      own[h]    = power_of_2(top[n][h] - safe);
      theirs[h] = power_of_2(other - safe);
      sum[n][h] = sum[n][h] * own[h] + (h == 0 ? stats.z : stats.w) * theirs[h];
      top[n][h] = next;
    }
#pragma unroll
    for (int d = 0; d < D / 16; d++) {
      const float4 y = at[32 * (d + 1)];
      acc[n][d][0]   = acc[n][d][0] * own[0] + y.x * theirs[0];
      acc[n][d][1]   = acc[n][d][1] * own[1] + y.y * theirs[1];
      acc[n][d][2]   = acc[n][d][2] * own[0] + y.z * theirs[0];
      acc[n][d][3]   = acc[n][d][3] * own[1] + y.w * theirs[1];
    }
  }

  __device__ __forceinline__ void to_shared() const
  {
    const float to_room = summands<T>::to_room(w);
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t r = n * 8 + 2 * t + h;
        if (g == 0) { state.stats[warp * shape::kRows + r] = make_float2(top[n][h], sum[n][h] * to_room); }
        float* a = state.acc + (warp * shape::kRows + r) * shape::kAccRow + g;
#pragma unroll
        for (int d = 0; d < D / 16; d++) {
          a[d * 16]     = acc[n][d][h] * to_room;
          a[d * 16 + 8] = acc[n][d][h + 2] * to_room;
        }
      }
    }
  }

  // A store of a warp is eight neighbouring columns of four rows.
  __device__ __forceinline__ void to_rows(uint32_t rows, uint32_t sequence, uint32_t head0, bool whole, uint32_t part) const
  {
    const float to_room = summands<T>::to_room(w);
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t r = n * 8 + 2 * t + h;
        if (r >= rows) { continue; }
        if (whole) {
          const float scale = sum[n][h] == 0.0f ? 0.0f : 1.0f / sum[n][h];
          T* o = reinterpret_cast<T*>(result.out.data) + int64_t(sequence) * result.out.row + int64_t(head0 + r) * result.out.head + g;
#pragma unroll
          for (int d = 0; d < D / 16; d++) {
            if (d * 16 + g < c.dim) { o[d * 16] = from_float<T>(acc[n][d][h] * scale); }
            if (d * 16 + 8 + g < c.dim) { o[d * 16 + 8] = from_float<T>(acc[n][d][h + 2] * scale); }
          }
          if (g == 0) {
            result.lse[size_t(sequence) * (w.group * c.n_heads) + head0 + r] = (finite_top(top[n][h]) + log2f(sum[n][h] * summands<T>::back(w))) * kLn2;
          }
        } else {
          float* a = parts.acc + (size_t(part) * parts.rows + r) * c.dim + g;
#pragma unroll
          for (int d = 0; d < D / 16; d++) {
            if (d * 16 + g < c.dim) { a[d * 16] = acc[n][d][h] * to_room; }
            if (d * 16 + 8 + g < c.dim) { a[d * 16 + 8] = acc[n][d][h + 2] * to_room; }
          }
          if (g == 0) { parts.stats[size_t(part) * parts.rows + r] = make_float2(top[n][h], sum[n][h] * to_room); }
        }
      }
    }
  }
};

template <typename T, int D, int NT, int WARPS, bool WHOLE_PAGES>
__global__ void __launch_bounds__(WARPS * 32, mma_shape<D, NT, WARPS>::kResident)
mma_kernel(cache_view c, work_view w, positions lists, rows_view queries, result_view result, float scale_log2, parts_view parts)
{
  using shape = mma_shape<D, NT, WARPS>;
  extern __shared__ __align__(128) char smem[];
  const block_state state{reinterpret_cast<float*>(smem), reinterpret_cast<float2*>(smem + shape::kStatsAt),
                          reinterpret_cast<float2*>(smem + shape::kJoinedAt), shape::kAccRow};
  uint32_t* s_mask = reinterpret_cast<uint32_t*>(smem + shape::kMaskAt) + (threadIdx.x >> 5) * shape::kStages;
  chain_begin();
  mma_hooks<T, D, NT, WARPS, WHOLE_PAGES> hooks(c, w, queries, result, parts, state, smem, scale_log2);
  run_units<T, WARPS, shape::kChunk, shape::kStages>(c, w, lists, result, parts, state, reinterpret_cast<float*>(smem + shape::kExchangeAt), s_mask,
                                                     hooks);
}

}  // namespace

// One object per type: KV_TYPE is __half or __nv_bfloat16.
template <>
void attention16<KV_TYPE>(cudaStream_t stream, const attention_args& a, const plan& p, const work_view& w, const positions& lists,
                          const result_view& result, const parts_view& parts)
{
  using T     = KV_TYPE;
  auto launch = [&](auto d, auto nt, auto warps) {
    constexpr int D = decltype(d)::value, NT = decltype(nt)::value, WARPS = decltype(warps)::value;
    auto go = [&](auto kernel) {
      launch_units(stream, kernel, p.blocks, WARPS * 32, p.cluster, mma_shape<D, NT, WARPS>::kShared, a.cache, w, lists, a.queries, result,
                   a.scale * kLog2E, parts);
    };
    if (a.cache.page.size % 16 == 0) {
      go(mma_kernel<T, D, NT, WARPS, true>);
    } else {
      go(mma_kernel<T, D, NT, WARPS, false>);
    }
  };
  using std::integral_constant;
  auto by_rows = [&](auto cols) {
    constexpr int D = decltype(cols)::value;
    auto by_warps   = [&](auto nt) {
      if constexpr (mma_large_of(D, decltype(nt)::value) != 0) {
        if (p.warps != uint32_t(kSmall)) { return launch(cols, nt, integral_constant<int, mma_large_of(D, decltype(nt)::value)>{}); }
      }
      launch(cols, nt, integral_constant<int, kSmall>{});
    };
    if (p.rows == 8) {
      by_warps(integral_constant<int, 1>{});
    } else if (p.rows == 16) {
      by_warps(integral_constant<int, 2>{});
    } else if constexpr (D <= 128) {
      by_warps(integral_constant<int, 4>{});
    }
  };
  const uint32_t d = padded(a.cache.dim);
  if (d == 64) {
    by_rows(integral_constant<int, 64>{});
  } else if (d == 128) {
    by_rows(integral_constant<int, 128>{});
  } else {
    by_rows(integral_constant<int, 256>{});
  }
}

}  // namespace cuvs_b200::kv
