// The part of DLPack 1.x's table of exchange functions that a call needs to read the description of a Python tensor in place (published
// in the DLPack specification: a type's attribute __dlpack_c_exchange_api__ is a capsule named "dlpack_exchange_api" with this table).
#pragma once

#include <dlpack/dlpack.h>

#include <cstdint>

namespace cuvs_b200 {

struct tensor_exchange {
  uint32_t major, minor;
  const void* previous;
  void* allocate;               // not used here
  void* managed_from_python;    // not used here
  void* python_from_managed;    // not used here
  int (*from_python)(void* object, DLTensor* out);  // borrowed: shape and strides are the tensor's; 0, or -1 with a Python error set
  void* current_stream;         // not used here
};

}  // namespace cuvs_b200
