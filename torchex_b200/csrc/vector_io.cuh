// Loads and stores of rows of fp32, bf16 or fp16 values, widened to fp32 in registers,
// for the kernels that work on rows of any of the three types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace texb {

template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen<float>(float v) { return v; }
template <> __device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T narrow(float v);  // rounds to nearest even
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

// BYTES bytes of consecutive values of type T, as one access (16, 8, 4 or 2 bytes; the address
// must be a multiple of BYTES).
template <typename T, int BYTES>
struct alignas(BYTES) Chunk {
  static constexpr int kCount = BYTES / int(sizeof(T));
  T v[kCount];
};

template <int BYTES> struct WordOf;
template <> struct WordOf<16> { using type = uint4; };
template <> struct WordOf<8> { using type = uint2; };
template <> struct WordOf<4> { using type = uint32_t; };
template <> struct WordOf<2> { using type = unsigned short; };

template <typename T, int BYTES>
__device__ __forceinline__ Chunk<T, BYTES> load_chunk(const T* p) {
  using W = typename WordOf<BYTES>::type;
  union { W w; Chunk<T, BYTES> c; } u;
  u.w = __ldg(reinterpret_cast<const W*>(p));
  return u.c;
}
// a value that is read once: not kept in the first-level cache
template <typename T, int BYTES>
__device__ __forceinline__ Chunk<T, BYTES> load_chunk_once(const T* p) {
  using W = typename WordOf<BYTES>::type;
  union { W w; Chunk<T, BYTES> c; } u;
  u.w = __ldcs(reinterpret_cast<const W*>(p));
  return u.c;
}
template <typename T, int BYTES>
__device__ __forceinline__ void store_chunk(T* p, const Chunk<T, BYTES>& c) {
  using W = typename WordOf<BYTES>::type;
  union { W w; Chunk<T, BYTES> c; } u;
  u.c = c;
  *reinterpret_cast<W*>(p) = u.w;
}
template <typename T, int BYTES>
__device__ __forceinline__ void store_chunk_once(T* p, const Chunk<T, BYTES>& c) {
  using W = typename WordOf<BYTES>::type;
  union { W w; Chunk<T, BYTES> c; } u;
  u.c = c;
  __stcs(reinterpret_cast<W*>(p), u.w);
}

inline int dtype_bytes(int dtype) { return dtype == TEXB_FLOAT32 ? 4 : 2; }
inline bool dtype_known(int dtype) {
  return dtype == TEXB_FLOAT32 || dtype == TEXB_BFLOAT16 || dtype == TEXB_FLOAT16;
}

}  // namespace texb
