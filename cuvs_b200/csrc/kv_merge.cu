// Joining parts of one softmax: parts o_p of disjoint sets of rows, each with the logarithm lse_p of its denominator, give
//   lse = log sum_p exp(lse_p),   o = sum_p exp(lse_p - lse) o_p.
// A part that attended to nothing (lse_p = -inf) has weight 0 and is not read.
#include "kv_rows.cuh"

namespace cuvs_b200::kv {

namespace {

constexpr int kThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kThreads) merge_kernel(merge_args a, uint32_t log_lanes, uint32_t pieces)
{
  chain_begin();
  constexpr int E       = kPerPiece<T>;
  const uint32_t lane   = threadIdx.x & ((1u << log_lanes) - 1u);
  const uint64_t r      = (uint64_t(blockIdx.x) * kThreads + threadIdx.x) >> log_lanes;
  if (r >= uint64_t(a.n_tokens) * a.n_heads) { return; }
  const int64_t token = int64_t(r / a.n_heads), head = int64_t(r - uint64_t(token) * a.n_heads);
  const float* lse    = a.parts_lse + token * a.l_row + head * a.l_head;
  float top           = -INFINITY;
  for (uint32_t p = 0; p < a.n_parts; p++) { top = fmaxf(top, lse[p * a.l_part]); }
  top         = finite_top(top);
  float total = 0.0f;
  for (uint32_t p = 0; p < a.n_parts; p++) { total += expf(lse[p * a.l_part] - top); }
  const float scale = total == 0.0f ? 0.0f : 1.0f / total;
  for (uint32_t j = lane; j < pieces; j += 1u << log_lanes) {
    float acc[E] = {};
#pragma unroll 4
    for (uint32_t p = 0; p < a.n_parts; p++) {
      const float w = expf(lse[p * a.l_part] - top);
      if (w == 0.0f) { continue; }
      const uint4 v = reinterpret_cast<const uint4*>(a.parts + (p * a.p_part + token * a.p_row + head * a.p_head) * int64_t(sizeof(T)))[j];
      float x[E];
      piece_to_floats<T>(v, x);
#pragma unroll
      for (int e = 0; e < E; e++) { acc[e] = fmaf(w, x[e], acc[e]); }
    }
#pragma unroll
    for (int e = 0; e < E; e++) { acc[e] *= scale; }
    reinterpret_cast<uint4*>(a.out.data + (token * a.out.row + head * a.out.head) * int64_t(sizeof(T)))[j] = floats_to_piece<T>(acc);
  }
  if (lane == 0) { a.lse[r] = top + logf(total); }
}

template <typename T>
void launch(resources& res, const merge_args& a)
{
  const uint32_t pieces = a.dim / kPerPiece<T>;
  uint32_t log_lanes    = 0;
  while (log_lanes < 5 && (1u << log_lanes) < pieces) { log_lanes++; }
  const uint64_t rows = uint64_t(a.n_tokens) * a.n_heads;
  launch_chained(merge_kernel<T>, dim3(uint32_t(ceildiv<uint64_t>(rows, kThreads >> log_lanes))), kThreads, 0, res.stream, a, log_lanes,
                 pieces);
  CUDA_TRY(cudaGetLastError());
  res.launches++;
}

}  // namespace

void merge_parts(resources& res, const merge_args& a)
{
  if (a.n_tokens == 0 || a.n_heads == 0) { return; }
  switch (a.type) {
    case elem::f16: return launch<__half>(res, a);
    case elem::bf16: return launch<__nv_bfloat16>(res, a);
    default: return launch<float>(res, a);
  }
}

}  // namespace cuvs_b200::kv
