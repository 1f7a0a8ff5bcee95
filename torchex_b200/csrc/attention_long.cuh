// What the kernels of the attention within segments for long segments share.
#pragma once

#include "attention.cuh"
#include "tcgen05.cuh"

namespace texb {
namespace attention {

constexpr int kLongTile = 128;
constexpr int kLongRows = 2 * kLongTile;
constexpr int kLongThreads = 512;

// Descriptions of the tensors for the copy engine (columns, heads, rows; boxes of 64 columns of one head), where
// the rows lie in segment order.
struct Maps {
  CUtensorMap q, k, v, g;
  int used;
};

// False where the copy engine cannot describe the tensor (then the rows are copied 16 bytes at a time).
bool make_map(CUtensorMap* map, const Problem& a, const View& x, int heads, int box_rows, int dtype);  // attention.cu

// Copies ROWS rows from position pos0 on (zeros from `end` on) into a tile of blocks of 64 columns, by a
// warpgroup.  Four rows of a 128-byte block per warp and step: the 16-byte pieces of a row go to the eight
// places that its swizzle gives.
template <typename T, int DP, int ROWS>
__device__ __forceinline__ void copy_long_tile(const Problem& a, const View& x, int head, int pos0, int end, uint32_t to) {
  const int thread = threadIdx.x & 127, piece = thread & 7;
  const T* base = static_cast<const T*>(x.p) + head * x.head;
#pragma unroll 4
  for (int r = thread >> 3; r < ROWS; r += 16) {
    const int pos = pos0 + r;
    const bool real = pos < end;
    const T* from = base + (real ? row_of(a, pos) * x.row : 0);
#pragma unroll
    for (int b = 0; b < DP / 64; ++b) {
      const int column = b * 64 + piece * 8;
      const bool on = real && column < a.dim;
      copy16(to + b * (ROWS * 128) + r * 128 + ((piece ^ (r & 7)) << 4), from + (on ? column : 0), on ? 16 : 0);
    }
  }
}

}  // namespace attention
}  // namespace texb
