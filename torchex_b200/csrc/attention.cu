// Attention within segments: argument checks, workspaces, the pass that looks rows over, and the choice
// of kernel.  The kernels are in attention_forward.cuh and attention_backward.cuh.

#include "attention_long.cuh"

#include <cfloat>
#include <cmath>

namespace texb {
namespace attention {

template <int DP> int forward_by_type(const Problem&, int, int, cudaStream_t);
template <int DP> int backward_by_type(const Problem&, int, int, cudaStream_t);
template <int DP> int long_forward_by_type(const Problem&, int, int, cudaStream_t);
template <int DP> int long_forward_timeouts(int*);
template <int DP> int long_backward_by_type(const Problem&, int, int, cudaStream_t);
template <int DP> int long_backward_timeouts(int*);

bool make_map(CUtensorMap* map, const Problem& a, const View& x, int heads, int box_rows, int dtype) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<Encode>(f);
  }();
  if (!encode || x.row <= 0 || x.head <= 0) return false;
  const cuuint64_t size[3] = {cuuint64_t(a.dim), cuuint64_t(heads), cuuint64_t(a.n)};
  const cuuint64_t stride[2] = {cuuint64_t(x.head) * 2, cuuint64_t(x.row) * 2};
  const cuuint32_t box[3] = {64, 1, cuuint32_t(box_rows)}, step[3] = {1, 1, 1};
  return encode(map, dtype == TEXB_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, x.p, size, stride,
                box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

// How the threads of a CTA share a block of kFlag positions: `lanes` threads walk one row of one head, and the
// rows of as many neighbouring heads as fit are taken together, since they lie side by side in memory (one head
// per CTA reads 256 bytes of every 4 KB).
struct Spread {
  int lanes, heads, rows;  // of a row; heads of a CTA; rows of a pass
};
inline Spread spread_of(int dim, int heads) {
  Spread s = {1, 0, 0};
  while (s.lanes < dim / 8) s.lanes *= 2;
  const int slots = kThreads / s.lanes;
  s.heads = heads < slots ? heads : slots;
  s.rows = slots / s.heads;
  return s;
}

// The order in which the long kernels take their tiles of `rows` positions: by falling length of the rows that a
// tile walks, in 64 classes, so that no long tile begins when the others are done (in order of position a training
// step of packed documents took an eighth longer).  One CTA; which tile of a class comes first does not matter.
struct Order {
  int rows, tiles;
  int32_t *order, *length;  // both [tiles]
};
template <bool KEYS>
__device__ void order_tiles(const Problem& a, const Order& o) {
  constexpr int kClasses = 64;
  __shared__ int s_count[kClasses], s_longest;
  if (threadIdx.x < kClasses) s_count[threadIdx.x] = 0;
  if (threadIdx.x == 0) s_longest = 1;
  __syncthreads();
  int longest = 1;
  for (int t = threadIdx.x; t < o.tiles; t += kThreads) {
    const int pos0 = t * o.rows, last = min(a.n, pos0 + o.rows) - 1;
    const Bounds f = KEYS ? queries_of(a, pos0) : keys_of(a, pos0), l = KEYS ? queries_of(a, last) : keys_of(a, last);
    const int length = max(1, (l.end - f.begin + 63) / 64);
    o.length[t] = length;
    longest = max(longest, length);
  }
  atomicMax(&s_longest, longest);
  __syncthreads();
  auto class_of = [&](int t) { return kClasses - 1 - int(int64_t(o.length[t]) * (kClasses - 1) / s_longest); };
  for (int t = threadIdx.x; t < o.tiles; t += kThreads) atomicAdd(&s_count[class_of(t)], 1);  // its own entries of `length`
  __syncthreads();
  if (threadIdx.x == 0) {
    int before = 0;
    for (int c = 0; c < kClasses; ++c) {
      const int n = s_count[c];
      s_count[c] = before;
      before += n;
    }
  }
  __syncthreads();
  for (int t = threadIdx.x; t < o.tiles; t += kThreads) o.order[atomicAdd(&s_count[class_of(t)], 1)] = t;
}

// Raises a word that holds the bits of a float that is not negative.  The order does not matter: the largest stays.
__device__ __forceinline__ void raise(float* to, float value) {
  if (!(value < INFINITY)) return;  // rows that are not finite
  int* word = reinterpret_cast<int*>(to);
  if (__float_as_int(value) > *static_cast<volatile int*>(word)) atomicMax(word, __float_as_int(value));
}

__device__ __forceinline__ float* word_of(const Problem& a, bool keys, int head, int first) {
  return keys ? a.v_most + int64_t(head) * a.n + first : a.g_most + int64_t(head / (a.heads / a.kv_heads)) * a.n + first;
}

// The flags of the blocks of the values (forward: BACKWARD false, the CTAs along y are groups of kv heads), or, for
// the backward pass, delta_i = scale g_i . o_i and the flags of the queries or gradients of each head (the first
// CTAs along y) and of the keys of each kv head, and for fp16 the sizes of the gradients and values.  Bound by HBM:
// every row is read once.
template <typename T, bool BACKWARD>
__global__ void __launch_bounds__(kThreads)
look_over_kernel(const __grid_constant__ Problem a, Spread q_spread, Spread k_spread, int q_groups, float* __restrict__ delta,
                 uint8_t* __restrict__ bad_q, uint8_t* __restrict__ bad_k, Order queries, Order keys_order) {
  constexpr bool kSized = BACKWARD && kShortRange<T>;
  __shared__ int s_bad[kThreads];  // by head of the CTA
  __shared__ float s_square[kSized ? kFlag * kThreads : 1];  // by row, then by head of the CTA
  const int blocks = (a.n + kFlag - 1) / kFlag;
  if (int(blockIdx.x) >= blocks) {  // one or two CTAs more, for the long kernels
    if (blockIdx.y == 0) order_tiles<false>(a, queries);
    else if (BACKWARD && blockIdx.y == 1) order_tiles<true>(a, keys_order);
    return;
  }
  const int pos0 = blockIdx.x * kFlag, end = min(a.n, pos0 + kFlag);
  const bool keys = !BACKWARD || int(blockIdx.y) >= q_groups;
  const Spread sp = keys ? k_spread : q_spread;
  const int first_head = (keys ? blockIdx.y - q_groups : blockIdx.y) * sp.heads, heads = keys ? a.kv_heads : a.heads;
  const int sub = threadIdx.x & (sp.lanes - 1), slot = threadIdx.x / sp.lanes, mine = slot % sp.heads, head = first_head + mine;
  const bool active = slot < sp.heads * sp.rows && head < heads && sub < a.dim / 8;
  constexpr int kInFlight = 4;  // rows of a thread whose loads are issued together
  s_bad[threadIdx.x] = 0;
  __syncthreads();
  bool bad = false;
  for (int r0 = slot / sp.heads; r0 < kFlag; r0 += sp.rows * kInFlight) {
    uint4 q[kInFlight], g[kInFlight], o[kInFlight], low[kInFlight];
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      q[k] = g[k] = o[k] = low[k] = uint4{0u, 0u, 0u, 0u};
      const int pos = pos0 + r0 + k * sp.rows;
      if (active && pos < end) {
        const int64_t row = row_of(a, pos);
        auto piece = [&](const View& x) {
          return __ldcs(reinterpret_cast<const uint4*>(static_cast<const T*>(x.p) + row * x.row + head * x.head + sub * 8));
        };
        q[k] = piece(!BACKWARD ? a.v : keys ? a.k : a.q);
        if (kSized && keys) g[k] = piece(a.v);
        if (!keys) {
          g[k] = piece(a.g);
          o[k] = piece(a.out);
          if (a.out_low.p) low[k] = piece(a.out_low);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      bad |= not_finite<T>(q[k]) || (!keys && not_finite<T>(g[k]));
      const int pos = pos0 + r0 + k * sp.rows;
      const bool writes = active && sub == 0 && pos < end && r0 + k * sp.rows < kFlag;
      if constexpr (kSized) {
        float square = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = widen<T>(reinterpret_cast<const Chunk<T, 16>&>(g[k]).v[e]);
          square = fmaf(x, x, square);
        }
        for (int x = sp.lanes / 2; x > 0; x >>= 1) square += __shfl_xor_sync(0xffffffffu, square, x);
        if (writes) {
          s_square[(pos - pos0) * sp.heads + mine] = square;
          if (!keys) a.g_size[int64_t(head) * a.n + pos] = square;
        }
      }
      if (keys) continue;
      // out itself is rounded: without the rest, delta's error would reach every dS of the row
      float sum = 0.f;
      const Chunk<T, 16>&gv = reinterpret_cast<const Chunk<T, 16>&>(g[k]), &ov = reinterpret_cast<const Chunk<T, 16>&>(o[k]),
            &lv = reinterpret_cast<const Chunk<T, 16>&>(low[k]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum = fmaf(widen<T>(gv.v[e]), widen<T>(ov.v[e]), sum);
        sum = fmaf(widen<T>(gv.v[e]), widen<T>(lv.v[e]), sum);
      }
      for (int x = sp.lanes / 2; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      if (writes) delta[int64_t(head) * a.n + pos] = sum * a.scale;
    }
  }
  if (bad) s_bad[mine] = 1;
  __syncthreads();
  if (int(threadIdx.x) < sp.heads && first_head + int(threadIdx.x) < heads)
    (keys ? bad_k : bad_q)[int64_t(first_head + threadIdx.x) * blocks + blockIdx.x] = uint8_t(s_bad[threadIdx.x]);
  if constexpr (kSized) {
    const int there = min(sp.heads, heads - first_head), first = first_of(a, pos0);
    if (first == first_of(a, end - 1)) {  // a block within one segment raises each word once
      if (int(threadIdx.x) < there) {
        float most = 0.f;
        for (int r = 0; r < end - pos0; ++r) {
          const float square = s_square[r * sp.heads + threadIdx.x];
          if (square < INFINITY) most = fmaxf(most, square);
        }
        raise(word_of(a, keys, first_head + threadIdx.x, first), most);
      }
    } else {
      for (int i = threadIdx.x; i < (end - pos0) * there; i += kThreads) {
        const int r = i / there, h = i % there;
        raise(word_of(a, keys, first_head + h, first_of(a, pos0 + r)), s_square[r * sp.heads + h]);
      }
    }
  }
}

int check(const Problem& a, int dtype, bool backward) {
  if (dtype != TEXB_BFLOAT16 && dtype != TEXB_FLOAT16)
    return fail(TEXB_ERR_UNSUPPORTED, "segment_attention: bf16 or fp16 only (dtype %d)", dtype);
  if (a.n < 0 || a.segments < 0 || a.heads < 1 || a.kv_heads < 1 || a.dim < 1)
    return fail(TEXB_ERR_INVALID_ARGUMENT, "segment_attention: bad sizes");
  if (a.heads % a.kv_heads != 0)
    return fail(TEXB_ERR_INVALID_ARGUMENT, "segment_attention: %d heads do not share %d key/value heads evenly", a.heads, a.kv_heads);
  if (a.dim % 8 != 0 || a.dim > 128)
    return fail(TEXB_ERR_UNSUPPORTED, "segment_attention: head dimension %d is not a multiple of 8 up to 128", a.dim);
  if (a.heads + a.kv_heads > 65535) return fail(TEXB_ERR_UNSUPPORTED, "segment_attention: too many heads");
  if (!(a.cap >= 0.f && a.cap < INFINITY) || !(fabsf(a.scale) < INFINITY))
    return fail(TEXB_ERR_INVALID_ARGUMENT, "segment_attention: bad scale or softcap");
  // 0 times an infinite factor would be NaN, not a score of 0
  if (a.cap == 0.f && !(fabsf(a.unit) < INFINITY))
    return fail(TEXB_ERR_UNSUPPORTED, "segment_attention: scale %g is out of range", a.scale);
  if (a.cap > 0.f && !(a.cap >= FLT_MIN && fabsf(a.bend_in) < INFINITY && a.bend_out < INFINITY))
    return fail(TEXB_ERR_UNSUPPORTED, "segment_attention: softcap %g is out of range for scale %g", a.cap, a.scale);
  if (a.n == 0) return TEXB_OK;
  if (!a.sid || !a.offsets || a.segments == 0) return fail(TEXB_ERR_INVALID_ARGUMENT, "segment_attention: NULL plan");
  const View* views[] = {&a.q, &a.k, &a.v, &a.out, &a.g, &a.gq, &a.gk, &a.gv};
  if (backward && (!a.gk.p != !a.gv.p)) return fail(TEXB_ERR_INVALID_ARGUMENT, "segment_attention: g_k and g_v are wanted together");
  for (int i = 0; i < (backward ? 8 : 4); ++i) {
    if (!views[i]->p && i >= 5) continue;  // a gradient that is not wanted
    if (!views[i]->p) return fail(TEXB_ERR_INVALID_ARGUMENT, "segment_attention: NULL pointer");
    if (reinterpret_cast<uintptr_t>(views[i]->p) % 16 != 0 || views[i]->row % 8 != 0 || views[i]->head % 8 != 0)
      return fail(TEXB_ERR_UNSUPPORTED, "segment_attention: rows must be 16-byte aligned");
  }
  if (reinterpret_cast<uintptr_t>(a.out_low.p) % 16 != 0) return fail(TEXB_ERR_UNSUPPORTED, "segment_attention: rows must be 16-byte aligned");
  if (backward && !a.lse) return fail(TEXB_ERR_INVALID_ARGUMENT, "segment_attention: the backward pass needs lse");
  return TEXB_OK;
}

inline size_t blocks_of(int64_t n) { return size_t(ceil_div(n, kFlag)); }  // of flags

// Segments short enough that a tile looks at the values of its keys itself instead of a pass of its own
// doing it: at most three tiles of keys.  Either way the same blocks of positions decide, and the kernels are chosen
// without it: whether the host knows the longest segment yet does not show in the results.
constexpr int kShortSegment = 64;

// Whether the 5th-generation tensor cores' kernels are used: where segments are long enough, on average, for tiles of
// 128 rows to be worth it.  Narrow rows are padded to 64 columns there, which takes longer segments to pay.
// Measured on 16 384 rows, 8 heads, training step, general / long kernels in us: dim 128, average 32: 321 / 258,
// 64: 383 / 241, 1024: 2543 / 709; dim 64, 32: 215 / 209, 64: 241 / 205; dim 32, 192: 238 / 221 (causal 169 / 189), 512: 449 / 323
// (280 / 240); dim 16, 512: 311 / 314 (204 / 231), 1024: 562 / 497 (342 / 320).  An average does not see a long segment
// among many short ones: such a batch takes the general kernels for all of its rows.
inline bool long_segments(const Problem& a) {
  const int64_t average = a.dim <= 16 ? 768 : a.dim <= 32 ? 256 : 32;
  return a.n >= a.segments * average;
}

// The forward pass of short segments that do not fill the GPU is latency: tiles of 64 rows start sooner and are more.
// Measured on segments of 32 to 64 rows (48 on average), general / long kernels in us, by rows times heads: dim 64, 1100:
// 13 / 17, 3800: 15 / 25, 15 400: 17 / 27, 30 700: 27 / 27, 61 000: 46 / 44; dim 128, 1100: 17 / 21, 3800: 23 / 27,
// 15 400: 27 / 31, 30 700: 44 / 31.
inline bool long_forward(const Problem& a) {
  return long_segments(a) && (a.n > a.segments * int64_t(64) || int64_t(a.n) * a.heads >= 24576);
}

}  // namespace
}  // namespace attention

int attention_timeouts_impl(int* count) {
  int (*const units[])(int*) = {attention::long_forward_timeouts<64>, attention::long_forward_timeouts<128>,
                                attention::long_backward_timeouts<64>, attention::long_backward_timeouts<128>};
  *count = 0;
  for (auto unit : units) {
    int one = 0;
    const int st = unit(&one);
    if (st != TEXB_OK) return st;
    *count += one;
  }
  return TEXB_OK;
}

namespace attention {
namespace {
struct Workspace {
  uint8_t *flags, *flags_q;  // of values, or keys; of queries and gradients
  float *delta, *g_size, *most;  // most: of the values, then of the gradients
  Order queries, keys;
  size_t bytes;
};
Workspace carve(void* ws, int64_t n, int heads, int kv_heads, bool backward) {
  Workspace w = {};
  const uintptr_t base = align_up(reinterpret_cast<uintptr_t>(ws), 256);
  size_t at = 0;
  auto take = [&](size_t bytes) { void* p = reinterpret_cast<void*>(base + at); at += align_up(bytes, 256); return p; };
  auto order = [&](int rows) {
    const size_t tiles = size_t(ceil_div(n, rows));
    Order o = {rows, int(tiles), nullptr, nullptr};
    o.order = static_cast<int32_t*>(take(tiles * sizeof(int32_t)));
    o.length = static_cast<int32_t*>(take(tiles * sizeof(int32_t)));
    return o;
  };
  w.flags = static_cast<uint8_t*>(take(blocks_of(n) * size_t(kv_heads)));
  w.queries = order(backward ? kLongTile : kLongRows);
  if (backward) {
    w.keys = order(kLongTile);
    w.flags_q = static_cast<uint8_t*>(take(blocks_of(n) * size_t(heads)));
    w.delta = static_cast<float*>(take(size_t(n) * size_t(heads) * sizeof(float)));
    w.g_size = static_cast<float*>(take(size_t(n) * size_t(heads) * sizeof(float)));
    w.most = static_cast<float*>(take(2 * size_t(n) * size_t(kv_heads) * sizeof(float)));
  }
  w.bytes = at + 256;
  return w;
}
}  // namespace
}  // namespace attention

size_t attention_workspace_bytes_impl(int64_t n, int heads, int kv_heads, int backward) {
  if (n < 0 || heads < 1 || kv_heads < 1) return 0;
  return attention::carve(nullptr, n, heads, kv_heads, backward != 0).bytes;
}

namespace attention {
namespace {

View view_of(const void* p, const int64_t* strides) {
  return {const_cast<void*>(p), strides ? strides[0] : 0, strides ? strides[1] : 0};
}

Problem problem_of(const texb_attention_problem& t) {
  Problem a = {};
  a.q = view_of(t.q, t.q_strides);
  a.k = view_of(t.k, t.k_strides);
  a.v = view_of(t.v, t.v_strides);
  const int64_t rows[2] = {int64_t(t.heads) * t.dim, t.dim}, kv_rows[2] = {int64_t(t.kv_heads) * t.dim, t.dim};
  a.out = view_of(t.out, rows);
  a.out_low = view_of(t.out_low, rows);
  a.g = view_of(t.g, t.g_strides);
  a.gq = view_of(t.g_q, rows);
  a.gk = view_of(t.g_k, kv_rows);
  a.gv = view_of(t.g_v, kv_rows);
  a.sid = t.sid;
  a.perm = t.perm;
  a.offsets = t.offsets;
  a.slopes = t.slopes;
  a.n = int(t.n);
  a.segments = int(t.num_segments);
  a.heads = t.heads;
  a.kv_heads = t.kv_heads;
  a.dim = t.dim;
  a.causal = t.causal;
  a.scale = t.scale;
  a.cap = t.softcap;
  a.unit = t.scale * kLog2e;
  a.bend_in = t.softcap > 0.f ? float(2.0 * 1.4426950408889634 * double(t.scale) / double(t.softcap)) : 0.f;
  a.bend_out = t.softcap * kLog2e;
  a.lse = t.lse;
  return a;
}

int check_problem(const texb_attention_problem* t) {
  if (!t) return fail(TEXB_ERR_INVALID_ARGUMENT, "segment_attention: NULL problem");
  if (t->n > INT_MAX - 65536 || t->num_segments > INT_MAX - 65536)
    return fail(TEXB_ERR_UNSUPPORTED, "segment_attention: n and num_segments must be below 2^31 - 65536");
  if (t->n < 0 || t->num_segments < 0) return fail(TEXB_ERR_INVALID_ARGUMENT, "segment_attention: negative size");
  return TEXB_OK;
}

}  // namespace
}  // namespace attention

int attention_forward_impl(const texb_attention_problem* t, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  using namespace attention;
  int st = check_problem(t);
  if (st != TEXB_OK) return st;
  Problem a = problem_of(*t);
  const int dtype = t->dtype;
  st = check(a, dtype, false);
  if (st != TEXB_OK || a.n == 0) return st;
  a.bad_v = nullptr;
  const bool use_long = long_forward(a);
  if (use_long || t->max_count < 0 || t->max_count > kShortSegment) {
    const Workspace w = carve(workspace, a.n, a.heads, a.kv_heads, false);
    if (!workspace || workspace_bytes < w.bytes)
      return fail(TEXB_ERR_WORKSPACE, "segment_attention workspace: need %zu bytes, got %zu", w.bytes, workspace_bytes);
    const Spread ks = spread_of(a.dim, a.kv_heads);
    const dim3 grid(unsigned(blocks_of(a.n)) + (use_long ? 1u : 0u), unsigned(ceil_div(a.kv_heads, ks.heads)));
    auto look = dtype == TEXB_BFLOAT16 ? look_over_kernel<__nv_bfloat16, false> : look_over_kernel<__half, false>;
    look<<<grid, kThreads, 0, stream>>>(a, ks, ks, 0, nullptr, nullptr, w.flags, w.queries, w.queries);
    st = check_launch("attention look_over_kernel");
    if (st != TEXB_OK) return st;
    a.bad_v = w.flags;
    a.query_order = w.queries.order;
  }
  const int mode = mode_of(a);
  if (use_long) {
    if (a.dim <= 64) return long_forward_by_type<64>(a, dtype, mode, stream);
    return long_forward_by_type<128>(a, dtype, mode, stream);
  }
  if (a.dim <= 16) return forward_by_type<16>(a, dtype, mode, stream);
  if (a.dim <= 32) return forward_by_type<32>(a, dtype, mode, stream);
  if (a.dim <= 64) return forward_by_type<64>(a, dtype, mode, stream);
  return forward_by_type<128>(a, dtype, mode, stream);
}

int attention_backward_impl(const texb_attention_problem* t, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  using namespace attention;
  int st = check_problem(t);
  if (st != TEXB_OK) return st;
  Problem a = problem_of(*t);
  const int dtype = t->dtype;
  st = check(a, dtype, true);
  if (st != TEXB_OK || a.n == 0) return st;
  const Workspace w = carve(workspace, a.n, a.heads, a.kv_heads, true);
  if (!workspace || workspace_bytes < w.bytes)
    return fail(TEXB_ERR_WORKSPACE, "segment_attention workspace: need %zu bytes, got %zu", w.bytes, workspace_bytes);
  a.delta = w.delta;
  a.bad_q = w.flags_q;
  a.bad_k = w.flags;
  a.query_order = w.queries.order;
  a.key_order = w.keys.order;
  a.g_size = w.g_size;
  a.v_most = w.most;
  a.g_most = w.most + int64_t(a.n) * a.kv_heads;
  if (dtype == TEXB_FLOAT16) {
    const cudaError_t e = cudaMemsetAsync(w.most, 0, 2 * size_t(a.n) * size_t(a.kv_heads) * sizeof(float), stream);
    if (e != cudaSuccess) return fail(TEXB_ERR_CUDA, "segment_attention: %s", cudaGetErrorString(e));
  }
  const Spread qs = spread_of(a.dim, a.heads), ks = spread_of(a.dim, a.kv_heads);
  const int q_groups = int(ceil_div(a.heads, qs.heads));  // and at least one group of kv heads: two CTAs along y
  const dim3 grid(unsigned(blocks_of(a.n)) + (long_segments(a) ? 1u : 0u), unsigned(q_groups + ceil_div(a.kv_heads, ks.heads)));
  auto look = dtype == TEXB_BFLOAT16 ? look_over_kernel<__nv_bfloat16, true> : look_over_kernel<__half, true>;
  look<<<grid, kThreads, 0, stream>>>(a, qs, ks, q_groups, w.delta, w.flags_q, w.flags, w.queries, w.keys);
  st = check_launch("attention look_over_kernel");
  if (st != TEXB_OK) return st;
  const int mode = mode_of(a);
  if (long_segments(a)) {
    if (a.dim <= 64) return long_backward_by_type<64>(a, dtype, mode, stream);
    return long_backward_by_type<128>(a, dtype, mode, stream);
  }
  if (a.dim <= 16) return backward_by_type<16>(a, dtype, mode, stream);
  if (a.dim <= 32) return backward_by_type<32>(a, dtype, mode, stream);
  if (a.dim <= 64) return backward_by_type<64>(a, dtype, mode, stream);
  return backward_by_type<128>(a, dtype, mode, stream);
}

}  // namespace texb
