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

// Writes columns c0 .. c0 + COLUMNS - 1 of a warp's 32 rows of sums (tensor memory), for fp16 times `factor`, each row
// (lane) its own, to rows of a tensor: through
// `rows`, 32 * COLUMNS * 2 bytes of shared memory that nothing else uses any more, so that a row is written by
// neighbouring lanes.  One row per lane, 16 bytes at a time, touches 32 half sectors per store: the gradients of 8192
// positions, 16 heads of 128 columns, up to 2048 keys take 343.5 us with the forward pass this way and 350 that way.
// The forward pass writes one row per lane: there these stores cost the loop registers (213 us instead of 205 for
// 32768 positions, 8 heads of 128 columns, up to 4096 keys).
template <typename T, int COLUMNS>
__device__ __forceinline__ void store_sums(const Problem& a, const View& x, int head, int pos0, uint32_t sums, int c0,
                                           float factor, unsigned char* rows) {
  constexpr int kPieces = COLUMNS / 8, kMask = kPieces < 8 ? kPieces - 1 : 7;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < COLUMNS; c += 32) {
    float o[32];
    t5::tmem_load32(sums + c0 + c, o);
    t5::tmem_wait_loads();
    if constexpr (kShortRange<T>) {
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] *= factor;
    }
#pragma unroll
    for (int e = 0; e < 32; e += 8) {
      const uint4 piece = {pack2<T>(o[e], o[e + 1]), pack2<T>(o[e + 2], o[e + 3]),
                           pack2<T>(o[e + 4], o[e + 5]), pack2<T>(o[e + 6], o[e + 7])};
      *reinterpret_cast<uint4*>(rows + lane * (COLUMNS * 2) + ((((c + e) / 8) ^ (lane & kMask)) << 4)) = piece;
    }
  }
  __syncwarp();
#pragma unroll 4
  for (int i = lane; i < 32 * kPieces; i += 32) {
    const int r = i / kPieces, piece = i % kPieces, pos = pos0 + r, column = c0 + piece * 8;
    if (pos < a.n && column < a.dim)
      *reinterpret_cast<uint4*>(row_at<T>(a, x, head, pos) + column) =
          *reinterpret_cast<const uint4*>(rows + r * (COLUMNS * 2) + ((piece ^ (r & kMask)) << 4));
  }
  __syncwarp();
}

}  // namespace attention
}  // namespace texb
