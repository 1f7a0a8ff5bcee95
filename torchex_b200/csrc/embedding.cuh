// What the lookup of table rows and its gradient share.
#pragma once

#include <climits>

#include "vector_io.cuh"

namespace texb {

// Lanes that walk one row of `vectors` accesses: a power of two, at most a warp.
inline int lanes_of(int64_t vectors) {
  int l = 1;
  while (l < 32 && l < vectors) l *= 2;
  return l;
}

// Widest access that the start of every row and the length of a row allow.
inline int access_bytes(int elem, int dim, const void* a, const void* b) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | uintptr_t(int64_t(dim) * elem);
  if (bits % 16 == 0) return 16;
  if (bits % 4 == 0) return 4;
  return elem;
}

inline int check_embedding_sizes(int id_bytes, int64_t n, int dtype, int64_t vocab, int dim) {
  if (id_bytes != 4 && id_bytes != 8)
    return fail(TEXB_ERR_INVALID_ARGUMENT, "id_bytes must be 4 or 8, got %d", id_bytes);
  if (!dtype_known(dtype)) return fail(TEXB_ERR_INVALID_ARGUMENT, "embedding: unknown dtype %d", dtype);
  if (n < 0 || vocab < 0 || dim < 1) return fail(TEXB_ERR_INVALID_ARGUMENT, "embedding: bad sizes");
  if (n > INT_MAX - 65536 || vocab > INT_MAX - 65536)
    return fail(TEXB_ERR_UNSUPPORTED, "embedding: tokens and vocab must be below 2^31 - 65536");
  return TEXB_OK;
}

}  // namespace texb
