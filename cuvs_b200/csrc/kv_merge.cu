// Joining parts of one softmax: parts o_p of disjoint sets of rows, each with the logarithm lse_p of its denominator, give
//   lse = log sum_p exp(lse_p),   o = sum_p exp(lse_p - lse) o_p.
// A part that attended to nothing (lse_p = -inf) has weight 0, and what its row holds does not count.  Weights are divided by their sum before rows
// are multiplied by them: sums of values next to the largest stay finite.
//
// What bounds it: HBM (every part is read once, the result written once), through the bytes in flight.  A group of lanes has a row.  It
// asks for the first eight parts' pieces at once and, while they come, for the lse; its lanes take the weights of as many parts as there
// are lanes.  Asking for rows only when their weights were known moved 4.1 TB/s (8 parts of 4,096 x 32 rows of 128 bf16: 74 us).
#include "kv_rows.cuh"

namespace cuvs_b200::kv {

namespace {

constexpr int kThreads = 256;

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads, 4) merge_kernel(merge_args a, uint32_t pieces)
{
  chain_begin();
  constexpr int E         = kPerPiece<T>;
  constexpr int AHEAD     = 8;
  const uint32_t lane     = threadIdx.x % LANES;
  const uint64_t asked    = (uint64_t(blockIdx.x) * kThreads + threadIdx.x) / LANES;
  const uint32_t n_rows   = a.n_tokens * a.n_heads;  // below 2^31
  const uint32_t r        = uint32_t(min(asked, uint64_t(n_rows - 1)));  // groups behind the last row take part in the shuffles
  const uint32_t token    = r / a.n_heads, head = r - token * a.n_heads;
  const float* lse        = a.parts_lse + int64_t(token) * a.l_row + int64_t(head) * a.l_head;
  const char* rows        = a.parts + (int64_t(token) * a.p_row + int64_t(head) * a.p_head) * int64_t(sizeof(T));
  const int64_t part_size = a.p_part * int64_t(sizeof(T));

  uint4 v[AHEAD];
  auto ask = [&](uint32_t j, uint32_t p0) {
#pragma unroll
    for (int q = 0; q < AHEAD; q++) {
      const uint32_t p = p0 + q;
      v[q]             = load_piece(rows + int64_t(p) * part_size + j * 16, p < a.n_parts && j < pieces);
    }
  };
  ask(lane, 0);
  float first = -INFINITY;  // of the first LANES parts, kept
  float top   = -INFINITY;
  for (uint32_t p = lane; p < a.n_parts; p += LANES) {
    const float x = lse[int64_t(p) * a.l_part];
    if (p == lane) { first = x; }
    top = fmaxf(top, x);
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) { top = fmaxf(top, __shfl_xor_sync(kAllLanes, top, o)); }
  top         = finite_top(top);
  float total = 0.0f;
  for (uint32_t p = lane; p < a.n_parts; p += LANES) { total += expf((p == lane ? first : lse[int64_t(p) * a.l_part]) - top); }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) { total += __shfl_xor_sync(kAllLanes, total, o); }
  const float scale = total == 0.0f ? 0.0f : 1.0f / total;

  for (uint32_t j0 = 0; j0 < pieces; j0 += LANES) {
    const uint32_t j = j0 + lane;
    float acc[E]     = {};
    float mine       = 0.0f;
    for (uint32_t p0 = 0; p0 < a.n_parts; p0 += AHEAD) {
      if (j0 != 0 || p0 != 0) { ask(j, p0); }
      if (p0 % LANES == 0) { mine = p0 + lane < a.n_parts ? expf((p0 == 0 ? first : lse[int64_t(p0 + lane) * a.l_part]) - top) * scale : 0.0f; }
#pragma unroll
      for (int q = 0; q < AHEAD; q++) {
        const float w = __shfl_sync(kAllLanes, mine, (p0 + q) % LANES, LANES);
        float x[E];
        piece_to_floats<T>(v[q], x);
#pragma unroll
        for (int e = 0; e < E; e++) { acc[e] = w != 0.0f ? fmaf(w, x[e], acc[e]) : acc[e]; }
      }
    }
    if (asked < n_rows && j < pieces) {
      reinterpret_cast<uint4*>(a.out.data + (int64_t(token) * a.out.row + int64_t(head) * a.out.head) * int64_t(sizeof(T)))[j] =
        floats_to_piece<T>(acc);
    }
  }
  if (asked < n_rows && lane == 0) { a.lse[r] = top + logf(total); }
}

template <typename T>
void launch(resources& res, cudaStream_t stream, const merge_args& a)
{
  const uint32_t pieces = a.dim / kPerPiece<T>;
  const uint64_t rows   = uint64_t(a.n_tokens) * a.n_heads;
  auto go               = [&](auto kernel, uint32_t lanes) {
    launch_chained(kernel, dim3(uint32_t(ceildiv<uint64_t>(rows, kThreads / lanes))), kThreads, 0, stream, a, pieces);
      count_launches(res, 1);
  };
  if (pieces <= 8) {
    go(merge_kernel<T, 8>, 8);
  } else if (pieces <= 16) {
    go(merge_kernel<T, 16>, 16);
  } else {
    go(merge_kernel<T, 32>, 32);
  }
}

}  // namespace

void merge_parts(resources& res, cudaStream_t stream, const merge_args& a)
{
  if (a.n_tokens == 0 || a.n_heads == 0) { return; }
  switch (a.type) {
    case elem::f16: return launch<__half>(res, stream, a);
    case elem::bf16: return launch<__nv_bfloat16>(res, stream, a);
    default: return launch<float>(res, stream, a);
  }
}

}  // namespace cuvs_b200::kv
