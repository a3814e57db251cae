// How the work of a call is dealt out, by type and sizes and by what the GPU holds at once.  For a host compiler.
#pragma once

#include <cuvs/core/b200_common.hpp>

#include <algorithm>
#include <cstdint>

namespace cuvs_b200::kv {

// Warps of a block: small blocks, several to an SM, balance best; where units are fewer than SMs, one large block has an SM's warps for one
// unit.
constexpr int kSmall = 4;
// Chunks of a share, at least.
constexpr uint32_t kLeastShare = 4;

struct plan {
  uint32_t rows;      // query heads of a unit
  uint32_t chunk;     // rows of the cache that a warp takes at a time
  uint32_t resident;  // small blocks of an SM
  uint32_t large;     // warps of a large block; 0: there is none
  uint32_t warps;     // of a block
  uint32_t blocks;
  uint32_t cluster;   // 0: shares
  uint32_t cost;      // of a unit beside its rows, in chunks
  bool parts;         // a unit may lie in several shares
};

// `units` with `most` rows each, at most; `shares`: whether there may be any.
//   Clusters are as large as fit on the GPU at once, one block to an SM: 15 of eight blocks and 33 of four on one whose 148 SMs would hold 18 and
// 37.  One more waits for all the others (bf16, sequences of 3,000 tokens: 15 units in clusters of eight 8.5 us, 16 units 15.6, and in clusters of
// four 10.4).
//   They are taken where a warp has four chunks at most: 8 units of 4,096 tokens (3 each) 9.3 us, 12.1 in shares; 6,144 (4) 10.8 and 12.8; 8,192
// (6) 12.8 and 14.0; 2 units of 6,144 (4) 10.7 and 11.5, 8,192 (6) 12.5 and 12.0; 32-bit rows of four heads, 8 units of 3,000 (4) 12.6 and
// 13.6, 4,096 (6) 15.7 and 15.2.
inline void deal_out(uint32_t sm_count, const uint32_t (&clusters_at_once)[4], plan& p, uint64_t units, uint64_t most, bool shares)
{
  const uint64_t sms = sm_count, resident = sms * p.resident;
  p.parts = false;
  if (units <= sms) {
    p.warps               = p.large ? p.large : kSmall;
    const uint64_t chunks = ceildiv<uint64_t>(most, p.warps * p.chunk);
    uint32_t cluster      = 1;
    for (int log = 1; log <= 3 && units <= clusters_at_once[log] && cluster < chunks; log++) { cluster = 1u << log; }
    if (!shares || ceildiv<uint64_t>(chunks, cluster) <= 4) {
      p.blocks  = uint32_t(units * cluster);
      p.cluster = cluster;
      return;
    }
  }
  p.warps = kSmall;
  if (!shares) {
    p.blocks  = uint32_t(units);
    p.cluster = 1;
  } else {
    const uint64_t chunks = std::max<uint64_t>(1, ceildiv<uint64_t>(most, p.chunk));
    p.blocks              = uint32_t(std::min(resident, units * ceildiv<uint64_t>(chunks, kLeastShare)));
    p.cluster             = 0;
    p.parts               = chunks > 1;
  }
}

}  // namespace cuvs_b200::kv
