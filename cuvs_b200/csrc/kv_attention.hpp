// What kv_rows.cu, which plans a call, and kv_attention.cu, which has the kernels for 16-bit rows, share.
#pragma once

#include "kv_units.cuh"

namespace cuvs_b200::kv {

// Columns of a row in the kernels' shared memory.
inline uint32_t padded(uint32_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
// Warps of the large block of the kernel for so many columns and eights of query heads; 0: its threads' registers leave no room for one.
constexpr int mma_large_of(uint32_t columns, uint32_t eights) { return columns <= 128 && eights <= 2 ? 12 : 0; }

template <typename T>
void attention16(cudaStream_t stream, const attention_args& a, const plan& p, const work_view& w, const positions& lists, const result_view& result,
                 const parts_view& parts);
template <>
void attention16<__half>(cudaStream_t stream, const attention_args& a, const plan& p, const work_view& w, const positions& lists,
                         const result_view& result, const parts_view& parts);
template <>
void attention16<__nv_bfloat16>(cudaStream_t stream, const attention_args& a, const plan& p, const work_view& w, const positions& lists,
                                const result_view& result, const parts_view& parts);

}  // namespace cuvs_b200::kv
