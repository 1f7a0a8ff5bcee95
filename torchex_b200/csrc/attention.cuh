// Softmax attention within segments: what the forward and the backward kernels share.
//
// Rows are walked in segment-sorted order (positions): position p is row perm[p] (or p) of the tensors
// and belongs to segment sid[p], whose positions are offsets[s] .. offsets[s + 1].  A query position i
// sees the keys begin(i) <= j < end(i): those of its segment, up to itself if causal.  A CTA owns a
// tile of consecutive positions, whichever segments they belong to, so that a tile of many short
// segments costs one tile; the mask is two comparisons per score against the row's bounds.
//
//   x_ij = scale q_i.k_j, capped: cap tanh(x / cap), minus slope_h |i - j|
//   p_ij = exp(x_ij - lse_i),  lse_i = log sum_j exp(x_ij),  o_i = sum_j p_ij v_j
//
// A product with a masked probability is 0 only if the other factor is finite.  The matrix
// instructions add up whole tiles, so a NaN or an infinity in a row that a query must not see would
// reach its result.  Rows are therefore looked over first (blocks of kFlag positions are flagged), and
// a tile whose rows meet a flagged block is computed by the plain loops at the end of this file,
// which touch visible rows only.  They add up in another order, with probabilities in 32 bits, so the rows of such a
// tile may differ in the last bits from what they are without the flagged row.  They are also slow: 8192 rows of 16
// heads of 128, segments up to 2048, take 8 (one such row) to 14 ms (all) forward instead of 0.1, and 30 to 35
// backward instead of 0.3.
#pragma once

#include <climits>
#include <type_traits>

#include "vector_io.cuh"

namespace texb {
namespace attention {

constexpr int kBlock = 64;  // positions of a tile
constexpr int kFlag = 16;   // positions of a flag
constexpr float kLog2e = 1.4426950408889634f;

// Rows of 16-bit values of several heads; strides in values, the head dimension is contiguous.
struct View {
  void* p;
  int64_t row, head;
};

struct Problem {
  View q, k, v;              // [n, heads, dim], [n, kv_heads, dim] twice
  const int32_t *sid, *perm, *offsets;
  const float* slopes;       // [heads] or NULL
  int n, segments, heads, kv_heads, dim;
  int causal;
  float scale, cap;          // cap 0: none
  float unit, bend_in, bend_out;  // scale log2(e), 2 scale log2(e) / cap, cap log2(e)
  // forward
  View out;                  // [n, heads, dim]
  View out_low;              // what rounding took from out, for the backward pass; p may be NULL
  float* lse;                // [heads, n] by position, in units of log2; forward may leave it out
  // backward
  View g;                    // gradient of out
  const float* delta;        // [heads, n] by position: scale * g_i . o_i
  View gq, gk, gv;
  // fp16 only, squares of norms: of each row of g, [heads, n]; of the largest finite row of v, and of g (of all heads that
  // share the kv head), of each segment, [kv_heads, n] at the segment's first position
  float *g_size, *v_most, *g_most;
  // flags of blocks with a value that is not finite, [.., ceil(n / kFlag)]; NULL: look for oneself
  const uint8_t *bad_v, *bad_k;  // per kv head
  const uint8_t* bad_q;          // per head: in q or g
  // long kernels: the tiles of queries, and of keys, by falling length of what they walk
  const int32_t *query_order, *key_order;
};

__device__ __forceinline__ int row_of(const Problem& a, int pos) {
  const int r = a.perm ? __ldg(a.perm + pos) : pos;
  return min(max(r, 0), a.n - 1);  // a corrupt plan reads a wrong row, not memory that is not there
}

template <typename T>
__device__ __forceinline__ T* row_at(const Problem& a, const View& x, int head, int pos) {
  return static_cast<T*>(x.p) + row_of(a, pos) * x.row + head * x.head;
}

struct Bounds {
  int begin, end;
  __device__ __forceinline__ bool holds(int p) const { return unsigned(p - begin) < unsigned(end - begin); }  // begin <= end
};
__device__ __forceinline__ Bounds segment_of(const Problem& a, int pos) {
  const int s = min(max(__ldg(a.sid + pos), 0), a.segments - 1);
  const int begin = max(0, __ldg(a.offsets + s));
  return {begin, max(begin, min(a.n, __ldg(a.offsets + s + 1)))};
}
__device__ __forceinline__ int first_of(const Problem& a, int pos) { return min(segment_of(a, pos).begin, a.n - 1); }
// Bounded waits of the kernels for long segments that gave up (part of texb_device_status).
static __device__ int g_wait_timeouts = 0;

// keys that a query sees, and queries that see a key; empty for positions behind the last row
__device__ __forceinline__ Bounds keys_of(const Problem& a, int pos) {
  if (pos >= a.n) return {0, 0};
  Bounds b = segment_of(a, pos);
  if (a.causal) b.end = max(b.begin, min(b.end, pos + 1));
  return b;
}
__device__ __forceinline__ Bounds queries_of(const Problem& a, int pos) {
  if (pos >= a.n) return {0, 0};
  Bounds b = segment_of(a, pos);
  if (a.causal) b.begin = min(b.end, max(b.begin, pos));
  return b;
}

__device__ __forceinline__ float exp2_fast(float x) {  // 2 units in the last place; tiny results become 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float reciprocal_fast(float x) {  // 1 unit in the last place
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The score in units of log2, from the plain product of a query and a key, and its derivative by scale *
// product.  tanh y = 1 - 2 / (exp(2 y) + 1), off by a few 2^-24 whatever y is: the exponential is infinite or 0
// for large |y|, and tanh then +-1.  Where |y| is small, that error is no small part of tanh y (a cap far above the
// scores would lose them), and y - y^3 / 3 is taken: the next term of the series is below 2^-23 of it for |y| < 0.03.
// `slope` is the head's, in units of log2.
struct Score { float x, slope; };
// How scores are formed: scaled (by a positive factor) and nothing else; with a bias by distance, or any factor;
// capped, with or without that.  A template parameter: the choice made per score took a third of the capped kernels' time.
constexpr int kPlain = 0, kBiased = 1, kCapped = 2;
inline int mode_of(const Problem& a) { return a.cap > 0.f ? kCapped : a.slopes || !(a.scale > 0.f) ? kBiased : kPlain; }
template <int MODE>
__device__ __forceinline__ Score score_of(const Problem& a, float product, float slope, float distance) {
  if constexpr (MODE == kPlain) return {product * a.unit, 1.f};
  if constexpr (MODE == kBiased) return {fmaf(-slope, fabsf(distance), product * a.unit), 1.f};
  constexpr float kUnit = 0.34657359f;  // y = z log(2) / 2
  const float z = product * a.bend_in, z2 = z * z;
  const float small = z * fmaf(z2, -1.f / 3.f * kUnit * kUnit * kUnit, kUnit);
  const float large = fmaf(-2.f, reciprocal_fast(exp2_fast(z) + 1.f), 1.f);
  const float t = z2 < 0.0075f ? small : large;
  return {fmaf(-slope, fabsf(distance), a.bend_out * t), fmaf(-t, t, 1.f)};
}
__device__ __forceinline__ Score any_score(const Problem& a, float product, float slope, float distance) {
  return a.cap > 0.f ? score_of<kCapped>(a, product, slope, distance) : score_of<kBiased>(a, product, slope, distance);
}
__device__ __forceinline__ float slope_of(const Problem& a, int head) { return a.slopes ? __ldg(a.slopes + head) * kLog2e : 0.f; }

// ---- matrix instructions on 16-bit fragments -----------------------------------------------------

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(v);
}

// How far probabilities are lifted before they are rounded to T: 2^LIFT times, by subtracting as much less from the
// scores, which costs nothing, and sums of them alike.  fp16's normal numbers end at 2^-14, and below 2^-25 it has none:
// a row of keys that each take 2^-20 of the weight would lose most of it.  Its largest is 65504, so a probability of
// 2^(15 - LIFT) may be lifted; for scores beyond 2^24, whose steps in fp32 are more than 1, it may come out as 2^16 and
// is held at the largest number (a NaN stays one).  bf16 has fp32's exponents.
template <typename T> constexpr bool kShortRange = std::is_same<T, __half>::value;
template <typename T, int LIFT> constexpr float kLifted = kShortRange<T> ? float(LIFT) : 0.f;
template <typename T> __device__ __forceinline__ uint32_t pack_lifted(float lo, float hi) {
  if constexpr (!kShortRange<T>) return pack2<T>(lo, hi);
  uint32_t v;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  return v;
}

// Gradients of scores are lifted in fp16 as well, by the largest power of two, from 1 to 2^100, that keeps what bounds
// them below 2^15: |dS| = P |scale (g v - g o)| <= 2 |scale| |g| |v|, v the largest row of the segment.  They are as
// small as the gradients, which is about g over the length of the segment: for g of 2^-10 and 2048 rows the unlifted
// ones were off by 2 %.  A row has one factor for all that is added up for it, and its sum is divided by it.  Under
// `causal` the largest rows may be ones that are not seen: 2^10 times larger than those that are, they leave fp16's
// normal numbers for gradients down to 2^-18 of their bound, and the factor is never below 1.
__device__ __forceinline__ int gradient_lift(const Problem& a, float g_square, float v_square) {
  const float bound = 2.f * fabsf(a.scale) * sqrtf(g_square) * sqrtf(v_square);
  return min(100, max(0, 14 - (int(__float_as_uint(bound) >> 23) - 127)));
}
// of a row of queries and of a row of keys
__device__ __forceinline__ int query_lift(const Problem& a, int head, int kv, int pos) {
  if (pos >= a.n) return 0;
  return gradient_lift(a, a.g_size[int64_t(head) * a.n + pos], a.v_most[int64_t(kv) * a.n + first_of(a, pos)]);
}
__device__ __forceinline__ int key_lift(const Problem& a, int kv, int pos) {
  if (pos >= a.n) return 0;
  const int64_t at = int64_t(kv) * a.n + first_of(a, pos);
  return gradient_lift(a, a.g_most[at], a.v_most[at]);
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((127 + e) << 23); }  // -126 <= e <= 127
constexpr int kGradientWeights = 15;  // lift of the probabilities of the backward pass: none is above 1

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 4 or 16 bytes to shared memory; `bytes` 0 writes zeros and reads nothing
__device__ __forceinline__ void copy4(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A tile of rows of DP 16-bit values in shared memory (DP: the head dimension padded to 16, 32, 64 or
// 128, columns behind it zero).  16-byte pieces are swizzled so that eight consecutive rows of one
// column of pieces lie in different banks.
template <int DP>
struct Tile {
  static constexpr int kPieces = DP / 8;
  static constexpr int kRowBytes = DP * 2;
  __device__ static __forceinline__ uint32_t at(int row, int piece) {
    constexpr int kShift = DP == 16 ? 2 : DP == 32 ? 1 : 0;
    constexpr int kMask = kPieces < 8 ? kPieces - 1 : 7;
    return uint32_t(row * kRowBytes + ((piece ^ ((row >> kShift) & kMask)) << 4));
  }
};

constexpr int kThreads = 128;

// Copies rows [pos0, pos0 + ROWS) of head `head` into a tile; rows at or behind `end` become zeros.
// The row numbers of the next tile are fetched ahead of it (`rows`), since they come through `perm`.
template <int DP, int ROWS>
struct Loader {
  static constexpr int kPer = (ROWS * (DP / 8) + kThreads - 1) / kThreads;  // pieces of a thread
  int rows[kPer];
  __device__ __forceinline__ void look_up(const Problem& a, int pos0, int end) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int pos = pos0 + (threadIdx.x + i * kThreads) / (DP / 8);
      rows[i] = pos < end ? row_of(a, pos) : -1;
    }
  }
  template <typename T>
  __device__ __forceinline__ void copy(const Problem& a, const View& x, int head, uint32_t to) const {
    const T* base = static_cast<const T*>(x.p) + head * x.head;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = threadIdx.x + i * kThreads;
      if (ROWS * (DP / 8) % kThreads != 0 && c >= ROWS * (DP / 8)) break;
      const int row = c / (DP / 8), piece = c % (DP / 8);
      const bool real = rows[i] >= 0 && piece * 8 < a.dim;
      const T* from = base + (real ? rows[i] * x.row + piece * 8 : 0);
      copy16(to + Tile<DP>::at(row, piece), from, real ? 16 : 0);
    }
  }
};

// A operand: rows row0 .. row0 + 15, columns 16 k .. 16 k + 15 of a tile.
template <int DP>
__device__ __forceinline__ void load_a(uint32_t (&r)[4], uint32_t tile, int row0, int k) {
  const int lane = threadIdx.x & 31;
  ldmatrix4(r, tile + Tile<DP>::at(row0 + (lane & 15), 2 * k + (lane >> 4)));
}
// B operand of a product over columns: rows row0 .. row0 + 15 (two n-tiles: r[0..1], r[2..3]), columns 16 k ...
template <int DP>
__device__ __forceinline__ void load_b(uint32_t (&r)[4], uint32_t tile, int row0, int k) {
  const int lane = threadIdx.x & 31;
  ldmatrix4(r, tile + Tile<DP>::at(row0 + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
}
// B operand of a product over rows: rows row0 .. row0 + 15, columns 16 c .. 16 c + 15 (two n-tiles)
template <int DP>
__device__ __forceinline__ void load_bt(uint32_t (&r)[4], uint32_t tile, int row0, int c) {
  const int lane = threadIdx.x & 31;
  ldmatrix4t(r, tile + Tile<DP>::at(row0 + (lane & 15), 2 * c + (lane >> 4)));
}

// acc [16 x 8 NT] += A (rows a_row0 .. of tile a) times the transpose of NT * 8 rows of tile b
template <typename T, int DP, int NT>
__device__ __forceinline__ void product_rows(float (&acc)[NT][4], uint32_t a, int a_row0, uint32_t b) {
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    uint32_t fa[4];
    load_a<DP>(fa, a, a_row0, k);
#pragma unroll
    for (int t = 0; t < NT; t += 2) {
      uint32_t fb[4];
      load_b<DP>(fb, b, t * 8, k);
      mma16816<T>(acc[t], fa, fb[0], fb[1]);
      mma16816<T>(acc[t + 1], fa, fb[2], fb[3]);
    }
  }
}

// acc [16 x DP] += P (16 x 8 NT, rounded to T) times NT * 8 rows of tile b.  SPLIT: what the rounding takes from P
// is multiplied as well, so that the products are those of some twice as many bits; P then holds gradients
// of scores, otherwise (lifted) probabilities.
template <typename T, int DP, int NT, bool SPLIT = false>
__device__ __forceinline__ void product_probabilities(float (&acc)[DP / 8][4], const float (&p)[NT][4], uint32_t b) {
  auto rest = [](float x) {
    const float high = widen<T>(narrow<T>(x));
    return fabsf(high) < INFINITY ? x - high : 0.f;
  };
#pragma unroll
  for (int k = 0; k < NT / 2; ++k) {
    const float (&x)[4] = p[2 * k], (&y)[4] = p[2 * k + 1];
    auto pack = [](float lo, float hi) { return SPLIT ? pack2<T>(lo, hi) : pack_lifted<T>(lo, hi); };
    const uint32_t fa[4] = {pack(x[0], x[1]), pack(x[2], x[3]), pack(y[0], y[1]), pack(y[2], y[3])};
    uint32_t fr[4];
    if constexpr (SPLIT) {
      fr[0] = pack2<T>(rest(x[0]), rest(x[1]));
      fr[1] = pack2<T>(rest(x[2]), rest(x[3]));
      fr[2] = pack2<T>(rest(y[0]), rest(y[1]));
      fr[3] = pack2<T>(rest(y[2]), rest(y[3]));
    }
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      uint32_t fb[4];
      load_bt<DP>(fb, b, 16 * k, c);
      mma16816<T>(acc[2 * c], fa, fb[0], fb[1]);
      mma16816<T>(acc[2 * c + 1], fa, fb[2], fb[3]);
      if constexpr (SPLIT) {
        mma16816<T>(acc[2 * c], fr, fb[0], fb[1]);
        mma16816<T>(acc[2 * c + 1], fr, fb[2], fb[3]);
      }
    }
  }
}

// Writes the warp's 16 x DP accumulators, times `factor` per row, to rows of a tensor, through the
// warp's own 16 rows of a tile (16-byte stores; the tile's former contents are no longer needed).
// `low`: what rounding those values to T takes from them, instead of the values.
template <typename T, int DP, bool LOW = false>
__device__ __forceinline__ void store_rows(const Problem& a, const View& x, int head, int pos0, const float (&acc)[DP / 8][4],
                                           float factor0, float factor1, unsigned char* tile, int row0) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  auto value = [](float x, float factor) {
    const float y = x * factor;
    return LOW ? y - widen<T>(narrow<T>(y)) : y;
  };
#pragma unroll
  for (int t = 0; t < DP / 8; ++t) {
    const int r = row0 + (lane >> 2);
    *reinterpret_cast<uint32_t*>(tile + Tile<DP>::at(r, t) + (lane & 3) * 4) = pack2<T>(value(acc[t][0], factor0), value(acc[t][1], factor0));
    *reinterpret_cast<uint32_t*>(tile + Tile<DP>::at(r + 8, t) + (lane & 3) * 4) = pack2<T>(value(acc[t][2], factor1), value(acc[t][3], factor1));
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < (16 * (DP / 8) + 31) / 32; ++i) {
    const int c = lane + i * 32;
    const int r = c / (DP / 8), piece = c % (DP / 8), pos = pos0 + r;
    if (r < 16 && pos < a.n && piece * 8 < a.dim) {
      T* to = row_at<T>(a, x, head, pos) + piece * 8;
      *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(tile + Tile<DP>::at(row0 + r, piece));
    }
  }
}

// ---- values that are not finite ------------------------------------------------------------------

// Whether one of eight 16-bit values is infinite or NaN: all bits of an exponent set.
template <typename T> struct ExponentBits;
template <> struct ExponentBits<__nv_bfloat16> { static constexpr uint32_t kMask = 0x7f80u; };
template <> struct ExponentBits<__half> { static constexpr uint32_t kMask = 0x7c00u; };
template <typename T>
__device__ __forceinline__ bool not_finite(const uint4& v) {
  constexpr uint32_t lo = ExponentBits<T>::kMask, hi = lo << 16;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (w[i] & lo) == lo || (w[i] & hi) == hi;
  return bad;
}

// Whether positions [begin, end) of head `head`, or others of the blocks of kFlag that they lie in, hold one: what
// `any_flag` says from the flags of the blocks.  Called by the whole CTA.
template <typename T>
__device__ __forceinline__ bool look_over(const Problem& a, const View& x, int head, int begin, int end) {
  const int pieces = a.dim / 8;
  bool bad = false;
  if (begin < end) {
    begin = begin / kFlag * kFlag;
    end = min(a.n, (end + kFlag - 1) / kFlag * kFlag);
  }
  for (int64_t c = threadIdx.x; c < int64_t(end - begin) * pieces; c += kThreads) {
    const int pos = begin + int(c / pieces);
    bad |= not_finite<T>(*reinterpret_cast<const uint4*>(row_at<T>(a, x, head, pos) + (c % pieces) * 8));
  }
  return __syncthreads_or(bad);
}

// Whether a flagged block meets positions [begin, end); called by the whole CTA.
__device__ __forceinline__ bool any_flag(const Problem& a, const uint8_t* flags, int head, int begin, int end) {
  const int blocks = (a.n + kFlag - 1) / kFlag;
  bool bad = false;
  for (int b = begin / kFlag + threadIdx.x; b < blocks && b * kFlag < end; b += blockDim.x) bad |= flags[int64_t(head) * blocks + b] != 0;
  return __syncthreads_or(bad);
}

// ---- plain loops: only visible rows are touched ---------------------------------------------------
// One warp per row.  32 rows of the other side at a time: a lane computes the product of one of them,
// then the warp adds them up, each lane holding every 32nd column.

constexpr int kColumns = 4;  // columns of a lane: dim <= 128

template <typename T>
__device__ __forceinline__ float dot(const T* x, const T* y, int dim) {
  float s = 0.f;
  for (int d = 0; d < dim; d += 8) {
    const Chunk<T, 16> a = load_chunk<T, 16>(x + d), b = load_chunk<T, 16>(y + d);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(widen<T>(a.v[e]), widen<T>(b.v[e]), s);
  }
  return s;
}

__device__ __forceinline__ float warp_max(float v) {
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = (u > v || u != u) ? u : v;  // a NaN stays
  }
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// acc += sum over the lanes k < count of w_k * row(j0 + k)
template <typename T>
__device__ __forceinline__ void add_weighted(const Problem& a, const View& x, int head, int j0, int count, float w,
                                             float (&acc)[kColumns]) {
  const int lane = threadIdx.x & 31;
  for (int k = 0; k < count; ++k) {
    const float wk = __shfl_sync(0xffffffffu, w, k);
    const T* row = row_at<T>(a, x, head, j0 + k);
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
      if (lane + 32 * c < a.dim) acc[c] = fmaf(wk, widen<T>(row[lane + 32 * c]), acc[c]);
  }
}

template <typename T>
__device__ __forceinline__ void store_columns(const Problem& a, const View& x, int head, int pos, const float (&acc)[kColumns],
                                              float factor) {
  const int lane = threadIdx.x & 31;
  T* row = row_at<T>(a, x, head, pos);
#pragma unroll
  for (int c = 0; c < kColumns; ++c)
    if (lane + 32 * c < a.dim) row[lane + 32 * c] = narrow<T>(acc[c] * factor);
}

template <typename T>
__device__ __noinline__ void plain_forward(const Problem& a, int pos0, int rows, int head) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kv = head / (a.heads / a.kv_heads);
  const float slope = slope_of(a, head);
  for (int i = pos0 + warp; i < min(a.n, pos0 + rows); i += blockDim.x / 32) {
    const Bounds see = keys_of(a, i);
    const T* qi = row_at<T>(a, a.q, head, i);
    float acc[kColumns] = {}, top = -INFINITY, sum = 0.f;
    for (int j0 = see.begin; j0 < see.end; j0 += 32) {
      const int j = j0 + lane;
      const float x = j < see.end ? any_score(a, dot<T>(qi, row_at<T>(a, a.k, kv, j), a.dim), slope, float(i - j)).x : -INFINITY;
      const float top_new = warp_max((x > top || x != x) ? x : top);
      const float base = top_new == -INFINITY ? 0.f : top_new;  // infinitely low scores so far: weight 0, not NaN
      const float w = j < see.end ? exp2f(x - base) : 0.f, shrink = top == -INFINITY ? 0.f : exp2f(top - base);
      sum = sum * shrink + warp_sum(w);
#pragma unroll
      for (int c = 0; c < kColumns; ++c) acc[c] = top == -INFINITY ? 0.f : acc[c] * shrink;
      add_weighted<T>(a, a.v, kv, j0, min(32, see.end - j0), w, acc);
      top = top_new;
    }
    const bool none = see.end <= see.begin;
    store_columns<T>(a, a.out, head, i, acc, none ? 0.f : 1.f / sum);
    if (a.out_low.p) {
#pragma unroll
      for (int c = 0; c < kColumns; ++c) {
        const float y = acc[c] * (none ? 0.f : 1.f / sum);
        acc[c] = y - widen<T>(narrow<T>(y));
      }
      store_columns<T>(a, a.out_low, head, i, acc, 1.f);
    }
    if (a.lse && lane == 0) a.lse[int64_t(head) * a.n + i] = none ? 0.f : top + log2f(sum);
  }
}

struct Pair { float p, ds; };  // probability and gradient of scale * product
template <typename T>
__device__ __forceinline__ Pair pair_of(const Problem& a, const T* qi, const T* kj, const T* vj, const T* gi, int head, int i, int j,
                                        float slope) {
  const Score s = any_score(a, dot<T>(qi, kj, a.dim), slope, float(i - j));
  const float p = exp2f(s.x - a.lse[int64_t(head) * a.n + i]);
  return {p, p * (dot<T>(gi, vj, a.dim) * a.scale - a.delta[int64_t(head) * a.n + i]) * s.slope};
}

template <typename T>
__device__ __noinline__ void plain_query_gradient(const Problem& a, int pos0, int rows, int head) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kv = head / (a.heads / a.kv_heads);
  const float slope = slope_of(a, head);
  for (int i = pos0 + warp; i < min(a.n, pos0 + rows); i += blockDim.x / 32) {
    const Bounds see = keys_of(a, i);
    const T *qi = row_at<T>(a, a.q, head, i), *gi = row_at<T>(a, a.g, head, i);
    float acc[kColumns] = {};
    for (int j0 = see.begin; j0 < see.end; j0 += 32) {
      const int j = j0 + lane;
      float w = 0.f;
      if (j < see.end)
        w = pair_of<T>(a, qi, row_at<T>(a, a.k, kv, j), row_at<T>(a, a.v, kv, j), gi, head, i, j, slope).ds;
      add_weighted<T>(a, a.k, kv, j0, min(32, see.end - j0), w, acc);
    }
    store_columns<T>(a, a.gq, head, i, acc, 1.f);
  }
}

template <typename T>
__device__ __noinline__ void plain_key_gradients(const Problem& a, int pos0, int rows, int kv) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = a.heads / a.kv_heads;
  for (int j = pos0 + warp; j < min(a.n, pos0 + rows); j += blockDim.x / 32) {
    const Bounds seen = queries_of(a, j);
    const T *kj = row_at<T>(a, a.k, kv, j), *vj = row_at<T>(a, a.v, kv, j);
    float acc_k[kColumns] = {}, acc_v[kColumns] = {};
    for (int head = kv * group; head < (kv + 1) * group; ++head) {
      const float slope = slope_of(a, head);
      for (int i0 = seen.begin; i0 < seen.end; i0 += 32) {
        const int i = i0 + lane, count = min(32, seen.end - i0);
        Pair w = {0.f, 0.f};
        if (i < seen.end)
          w = pair_of<T>(a, row_at<T>(a, a.q, head, i), kj, vj, row_at<T>(a, a.g, head, i), head, i, j, slope);
        add_weighted<T>(a, a.g, head, i0, count, w.p, acc_v);
        add_weighted<T>(a, a.q, head, i0, count, w.ds, acc_k);
      }
    }
    store_columns<T>(a, a.gk, kv, j, acc_k, 1.f);
    store_columns<T>(a, a.gv, kv, j, acc_v, 1.f);
  }
}

}  // namespace attention
}  // namespace texb
