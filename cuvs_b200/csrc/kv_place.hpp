// Where a sequence's position lies in a paged cache.  For the device, and for a host compiler.
#pragma once

#include <cuvs/core/b200_common.hpp>

#include <cstdint>

namespace cuvs_b200::kv {

// Division of numbers below 2^31 by the page size as one product (Granlund and Montgomery, Division by invariant integers using
// multiplication, 1994): with l = ceil(log2 size) and m = floor(2^(31 + l) / size) + 1, which is below 2^32, n / size = n m >> (31 + l).
struct page_divisor {
  uint32_t size, factor, shift;
};
inline page_divisor divisor_of(uint32_t size)
{
  uint32_t l = 0;
  while ((uint64_t(1) << l) < size) { l++; }
  return {size, uint32_t((uint64_t(1) << (31 + l)) / size + 1), 31 + l};
}

// Page column and place in the page of a position (below 2^31).
CUVS_HD inline void split_place(uint32_t at, const page_divisor& by, uint32_t& page, uint32_t& place)
{
  page  = uint32_t(uint64_t(at) * by.factor >> by.shift);
  place = at - page * by.size;
}

// The page of the cache in column `column` of a sequence's row of the table, -1 where there is none.
CUVS_HD inline int32_t page_of(const int32_t* row, uint32_t width, uint32_t column, int32_t n_pages)
{
  if (column >= width) { return -1; }
  const int32_t page = row[column];
  return page >= 0 && page < n_pages ? page : -1;
}

// The slot of position `at` of a sequence; -1: the position has none.
CUVS_HD inline int64_t slot_of(const int32_t* row, uint32_t width, int32_t at, const page_divisor& by, int32_t n_pages)
{
  if (at < 0) { return -1; }
  uint32_t column, place;
  split_place(uint32_t(at), by, column, place);
  const int32_t page = page_of(row, width, column, n_pages);
  return page < 0 ? -1 : int64_t(page) * by.size + place;
}

// First and one past the last position that a token attends to: the last `window` (0: all) of `length`, as far as the table reaches.
CUVS_HD inline void attended(int32_t length, int64_t window, uint32_t width, uint32_t page_size, uint32_t& first, uint32_t& end)
{
  const int64_t n = length < 0 ? 0 : length, capacity = int64_t(width) * page_size;
  end   = uint32_t(n < capacity ? n : capacity);
  first = window > 0 && n > window ? uint32_t(n - window) : 0u;
  if (first > end) { first = end; }
}

}  // namespace cuvs_b200::kv
