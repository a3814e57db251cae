// Attention of one query head over the rows of the cache that a search named.
//
// One block per (token, query head).  A warp takes 32 rows of the list at a time: every lane finds the place of one of them, then groups
// of lanes -- as many as a row has 16-byte pieces -- read four rows each, keys and values together, and carry a softmax of their own
// (running top, sum of weights, weighted sum of values); the groups, then the warps, are joined at the end.
#include "kv_rows.cuh"

#include <algorithm>

namespace cuvs_b200::kv {

namespace {

constexpr int kWarps = 8;

template <typename T, int LANES, int PIECES>
__global__ void __launch_bounds__(kWarps * 32)
rows_kernel(cache_view c, const int64_t* __restrict__ candidates, uint32_t n_candidates, rows_view queries, rows_view out, float* lse, uint32_t n_query_heads, float scale_log2)
{
  chain_begin();
  constexpr int E      = kPerPiece<T>;
  constexpr int GROUPS = 32 / LANES;
  constexpr int U      = 4;
  __shared__ float s_top[kWarps], s_sum[kWarps];
  __shared__ float s_out[kWarps][LANES * PIECES * E];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t group = lane / LANES, gl = lane % LANES;
  const uint64_t list  = blockIdx.x;
  const uint32_t token = uint32_t(list / n_query_heads), qh = uint32_t(list - uint64_t(token) * n_query_heads);
  const uint32_t head  = qh / (n_query_heads / c.n_heads);
  const uint32_t n_pieces = c.dim / E;
  const char* keys   = c.keys + int64_t(head) * c.k_head * sizeof(T);
  const char* values = c.values + int64_t(head) * c.v_head * sizeof(T);

  float q[PIECES][E];
#pragma unroll
  for (int v = 0; v < PIECES; v++) {
    const uint32_t j = gl + v * LANES;
    const uint4 w    = j < n_pieces ? reinterpret_cast<const uint4*>(queries.data + (int64_t(token) * queries.row + int64_t(qh) * queries.head) *
                                                                                      int64_t(sizeof(T)))[j]
                                    : make_uint4(0, 0, 0, 0);
    piece_to_floats<T>(w, q[v]);
  }
  float top = -INFINITY, sum = 0.0f;
  float acc[PIECES][E] = {};
  for (uint32_t base = warp * 32u; base < n_candidates; base += kWarps * 32u) {
    int64_t k_at = -1, v_at = 0;
    if (base + lane < n_candidates) {
      const int64_t slot = candidates[list * n_candidates + base + lane];
      if (slot >= 0 && slot < c.n_slots && slot_allowed(c, slot)) {
        int64_t page;
        uint32_t place;
        split_slot(c, slot, page, place);
        k_at = page * c.k_page + int64_t(place) * c.k_token;
        v_at = page * c.v_page + int64_t(place) * c.v_token;
      }
    }
#pragma unroll 1
    for (int j0 = 0; j0 < 32; j0 += U * GROUPS) {
      uint4 k[U][PIECES], v[U][PIECES];
      bool ok[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int from      = j0 + u * GROUPS + int(group);
        const int64_t kr    = __shfl_sync(kAllLanes, k_at, from);
        const int64_t vr    = __shfl_sync(kAllLanes, v_at, from);
        ok[u]               = kr >= 0;
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
          const uint32_t j = gl + p * LANES;
          k[u][p] = v[u][p] = make_uint4(0, 0, 0, 0);
          if (ok[u] && j < n_pieces) {
            k[u][p] = __ldg(reinterpret_cast<const uint4*>(keys + kr * int64_t(sizeof(T))) + j);
            v[u][p] = __ldg(reinterpret_cast<const uint4*>(values + vr * int64_t(sizeof(T))) + j);
          }
        }
      }
      float score[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        float s = 0.0f;
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
          float x[E];
          piece_to_floats<T>(k[u][p], x);
#pragma unroll
          for (int e = 0; e < E; e++) { s = fmaf(q[p][e], x[e], s); }
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) { s += __shfl_xor_sync(kAllLanes, s, o); }
        score[u] = ok[u] ? s * scale_log2 : -INFINITY;
      }
      float next = top;
#pragma unroll
      for (int u = 0; u < U; u++) { next = fmaxf(next, score[u]); }
      const float safe = finite_top(next);
      const float keep = exp2f(top - safe);
      top              = next;
      sum *= keep;
#pragma unroll
      for (int p = 0; p < PIECES; p++) {
#pragma unroll
        for (int e = 0; e < E; e++) { acc[p][e] *= keep; }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const float w = exp2f(score[u] - safe);
        sum += w;
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
          float x[E];
          piece_to_floats<T>(v[u][p], x);
#pragma unroll
          for (int e = 0; e < E; e++) { acc[p][e] = fmaf(w, x[e], acc[p][e]); }
        }
      }
    }
  }
  // the warp's groups
#pragma unroll
  for (int o = LANES; o < 32; o <<= 1) {
    const float other = __shfl_xor_sync(kAllLanes, top, o);
    const float next  = fmaxf(top, other);
    const float safe  = finite_top(next);
    const float mine = exp2f(top - safe), theirs = exp2f(other - safe);
    sum = sum * mine + __shfl_xor_sync(kAllLanes, sum, o) * theirs;
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
#pragma unroll
      for (int e = 0; e < E; e++) { acc[p][e] = acc[p][e] * mine + __shfl_xor_sync(kAllLanes, acc[p][e], o) * theirs; }
    }
    top = next;
  }
  if (group == 0) {
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
#pragma unroll
      for (int e = 0; e < E; e++) { s_out[warp][(gl + p * LANES) * E + e] = acc[p][e]; }
    }
  }
  if (lane == 0) {
    s_top[warp] = top;
    s_sum[warp] = sum;
  }
  __syncthreads();
  float all = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWarps; w++) { all = fmaxf(all, s_top[w]); }
  const float safe = finite_top(all);
  float total      = 0.0f;
#pragma unroll
  for (int w = 0; w < kWarps; w++) { total += s_sum[w] * exp2f(s_top[w] - safe); }
  const float scale = total == 0.0f ? 0.0f : 1.0f / total;
  T* o = reinterpret_cast<T*>(out.data) + int64_t(token) * out.row + int64_t(qh) * out.head;
  for (uint32_t d = threadIdx.x; d < c.dim; d += kWarps * 32) {
    float x = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; w++) { x += s_out[w][d] * exp2f(s_top[w] - safe); }
    o[d] = from_float<T>(x * scale);
  }
  if (threadIdx.x == 0) { lse[list] = (safe + log2f(total)) * kLn2; }
}

template <typename T>
void launch(resources& res, const candidates_args& a)
{
  const uint32_t pieces = a.cache.dim / kPerPiece<T>;
  auto go               = [&](auto kernel) {
    launch_chained(kernel, dim3(a.n_tokens * a.n_query_heads), kWarps * 32, 0, res.stream, a.cache, a.candidates, a.n_candidates, a.queries,
                   a.out, a.lse, a.n_query_heads, a.scale * kLog2E);
    CUDA_TRY(cudaGetLastError());
  };
  if (pieces <= 4) {
    go(rows_kernel<T, 4, 1>);
  } else if (pieces <= 8) {
    go(rows_kernel<T, 8, 1>);
  } else if (pieces <= 16) {
    go(rows_kernel<T, 16, 1>);
  } else if (pieces <= 32) {
    go(rows_kernel<T, 32, 1>);
  } else if constexpr (sizeof(T) == 4) {
    go(rows_kernel<T, 32, 2>);
  }
  res.launches++;
}

}  // namespace

void attend_candidates(resources& res, const candidates_args& a)
{
  if (a.n_tokens == 0) { return; }
  switch (a.type) {
    case elem::f16: return launch<__half>(res, a);
    case elem::bf16: return launch<__nv_bfloat16>(res, a);
    default: return launch<float>(res, a);
  }
}

}  // namespace cuvs_b200::kv
