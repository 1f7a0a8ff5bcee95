// Rows of a table by token, and the gradient of the table.
//
//   forward : out[t, :] = scale * weight[token_t, :]
//   backward: g_weight[v, :] = scale * sum over {t : token_t = v, v != padding} of g[t, :]
//
// Both are bound by HBM: the forward pass reads every looked-up row and writes n rows, the
// backward pass reads n rows of g and writes all `vocab` rows of the (dense) gradient.  There is
// no arithmetic to speak of and no floating-point atomic: the tokens are sorted (stably, by the
// plan builder's radix sort), so the rows of one token are summed in increasing position, in
// fp32, and rounded once.  For fp32 rows the sum is compensated (error-free additions), as in
// the segment reductions; for 16-bit rows the one rounding to 16 bits at the end is far coarser
// than what plain fp32 additions lose.
//
// A token outside [0, vocab) reads nothing: its output row is zero, it takes no part in the
// gradient, and it is counted (texb_device_status, bad_indices).

#include <climits>

#include "vector_io.cuh"

namespace texb {

int plan_build_impl(const void*, int, int64_t, int64_t, int, int32_t*, int32_t*, int32_t*, int32_t*, void*, size_t,
                    cudaStream_t);
size_t plan_workspace_bytes_impl(int64_t, int64_t, int);

namespace {

static __device__ int g_bad_tokens = 0;

constexpr int kThreads = 256;

// A row is walked by a group of `lanes` lanes (a power of two, at most a warp); every lane holds
// kBlocks accesses of BYTES bytes of a chunk of columns, so that one lane always carries eight
// values whatever the access width.
template <typename T, int BYTES>
struct RowShape {
  static constexpr int kVec = BYTES / int(sizeof(T));
  static constexpr int kBlocks = 8 / kVec;
};

inline int lanes_of(int64_t vectors) {
  int l = 1;
  while (l < 32 && l < vectors) l *= 2;
  return l;
}

// ---- forward -----------------------------------------------------------------------------

template <typename T, int BYTES, typename IdT, bool SCALED>
__global__ void __launch_bounds__(kThreads)
embedding_forward_kernel(const IdT* __restrict__ tokens, int64_t n, const T* __restrict__ weight, int64_t vocab,
                         int dim, float scale, T* __restrict__ out, int lanes, int chunks) {
  constexpr int kVec = RowShape<T, BYTES>::kVec;
  constexpr int kInFlight = 4;  // accesses of a lane before the first store
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t unit = (int64_t(blockIdx.x) * kThreads + threadIdx.x) / lanes;
  if (unit >= n * chunks) return;
  const int64_t t = unit / chunks;
  const int chunk = int(unit - t * chunks);
  const int64_t id = int64_t(tokens[t]);
  const bool ok = id >= 0 && id < vocab;
  if (!ok && chunk == 0 && lane == 0) atomicAdd(&g_bad_tokens, 1);
  const T* src = weight + id * dim;
  T* dst = out + t * dim;
  const int vectors = dim / kVec;
  const int first = chunk * lanes * kInFlight + lane;
  Chunk<T, BYTES> c[kInFlight];
#pragma unroll
  for (int k = 0; k < kInFlight; ++k) {
    const int i = first + k * lanes;
    if (ok && i < vectors) {
      c[k] = load_chunk<T, BYTES>(src + int64_t(i) * kVec);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) c[k].v[e] = narrow<T>(0.f);
    }
  }
#pragma unroll
  for (int k = 0; k < kInFlight; ++k) {
    const int i = first + k * lanes;
    if (i >= vectors) break;
    if constexpr (SCALED) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) c[k].v[e] = narrow<T>(widen<T>(c[k].v[e]) * scale);
    }
    store_chunk<T, BYTES>(dst + int64_t(i) * kVec, c[k]);
  }
}

// ---- backward ----------------------------------------------------------------------------

// Tokens that take part keep their id; the others (padding, out of range) sort behind the table.
template <typename IdT>
__global__ void embedding_keys_kernel(const IdT* __restrict__ tokens, int n, int64_t vocab, int64_t padding,
                                      int32_t* __restrict__ keys) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= n) return;
  const int64_t id = int64_t(tokens[i]);
  const bool ok = id >= 0 && id < vocab;
  if (!ok) atomicAdd(&g_bad_tokens, 1);
  keys[i] = ok && id != padding ? int32_t(id) : int32_t(vocab);
}

template <typename T>
struct Sum {  // running sum of one column: compensated for fp32 rows
  float s = 0.f, c = 0.f;
  __device__ __forceinline__ void add(float v) {
    if constexpr (sizeof(T) == 4) {
      const float t = s + v;
      const float b = t - s;
      c += (s - (t - b)) + (v - b);
      s = t;
    } else {
      s += v;
    }
  }
  __device__ __forceinline__ float total() const {
    if constexpr (sizeof(T) == 4) return isfinite(s) ? s + c : s;  // an infinite sum has no error term
    return s;
  }
};

template <typename T, int BYTES>
__global__ void __launch_bounds__(kThreads)
embedding_backward_rows_kernel(const T* __restrict__ g, const int32_t* __restrict__ perm,
                               const int32_t* __restrict__ offsets, int64_t vocab, int dim, float scale,
                               T* __restrict__ g_weight, int lanes) {
  constexpr int kVec = RowShape<T, BYTES>::kVec;
  constexpr int kBlocks = RowShape<T, BYTES>::kBlocks;
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t v = (int64_t(blockIdx.x) * kThreads + threadIdx.x) / lanes;
  if (v >= vocab) return;
  const int vectors = dim / kVec;
  const int first = blockIdx.y * lanes * kBlocks + lane;
  Sum<T> acc[kBlocks * kVec];
  const int end = offsets[v + 1];
  for (int p = offsets[v]; p < end; ++p) {
    const T* row = g + int64_t(perm[p]) * dim;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const int i = first + b * lanes;
      if (i < vectors) {
        const Chunk<T, BYTES> c = load_chunk_once<T, BYTES>(row + int64_t(i) * kVec);
#pragma unroll
        for (int e = 0; e < kVec; ++e) acc[b * kVec + e].add(widen<T>(c.v[e]));
      }
    }
  }
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const int i = first + b * lanes;
    if (i < vectors) {
      Chunk<T, BYTES> c;
#pragma unroll
      for (int e = 0; e < kVec; ++e) c.v[e] = narrow<T>(acc[b * kVec + e].total() * scale);
      store_chunk<T, BYTES>(g_weight + v * dim + int64_t(i) * kVec, c);
    }
  }
}

// ---- launches ----------------------------------------------------------------------------

// Widest access that every row start and the row length allow.
inline int access_bytes(int elem, int dim, const void* a, const void* b) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | uintptr_t(int64_t(dim) * elem);
  if (bits % 16 == 0) return 16;
  if (bits % 4 == 0) return 4;
  return elem;
}

template <typename T, int BYTES>
int launch_forward(const void* tokens, int id_bytes, int64_t n, const T* weight, int64_t vocab, int dim, float scale,
                   T* out, cudaStream_t stream) {
  const int64_t vectors = dim / RowShape<T, BYTES>::kVec;
  const int lanes = lanes_of(vectors);
  const int chunks = int(ceil_div(vectors, lanes * 4));
  const int64_t blocks = ceil_div(n * chunks, kThreads / lanes);
  if (blocks > INT_MAX) return fail(TEXB_ERR_UNSUPPORTED, "embedding: %lld rows of %d values are too many", (long long)n, dim);
#define TEXB_LAUNCH(ID, SC)                                                                              \
  embedding_forward_kernel<T, BYTES, ID, SC><<<unsigned(blocks), kThreads, 0, stream>>>(                 \
      static_cast<const ID*>(tokens), n, weight, vocab, dim, scale, out, lanes, chunks)
  if (id_bytes == 8) {
    if (scale == 1.f) TEXB_LAUNCH(int64_t, false); else TEXB_LAUNCH(int64_t, true);
  } else {
    if (scale == 1.f) TEXB_LAUNCH(int32_t, false); else TEXB_LAUNCH(int32_t, true);
  }
#undef TEXB_LAUNCH
  return check_launch("embedding_forward_kernel");
}

template <typename T>
int forward_typed(const void* tokens, int id_bytes, int64_t n, const void* weight, int64_t vocab, int dim, float scale,
                  void* out, cudaStream_t stream) {
  const T* w = static_cast<const T*>(weight);
  T* o = static_cast<T*>(out);
  const int bytes = access_bytes(int(sizeof(T)), dim, weight, out);
  if (bytes == 16) return launch_forward<T, 16>(tokens, id_bytes, n, w, vocab, dim, scale, o, stream);
  if (bytes == 4) return launch_forward<T, 4>(tokens, id_bytes, n, w, vocab, dim, scale, o, stream);
  return launch_forward<T, int(sizeof(T))>(tokens, id_bytes, n, w, vocab, dim, scale, o, stream);
}

struct BackwardWorkspace {
  int32_t *keys, *sid, *perm, *offsets, *stats;
  void* sort;
  size_t sort_bytes, bytes;
};

BackwardWorkspace carve_backward(void* ws, int64_t n, int64_t vocab) {
  BackwardWorkspace w;
  const uintptr_t base = align_up(reinterpret_cast<uintptr_t>(ws), 256);
  const size_t rows = align_up(size_t(n) * sizeof(int32_t), 256);
  size_t at = 0;
  auto take = [&](size_t bytes) { void* p = reinterpret_cast<void*>(base + at); at += bytes; return p; };
  w.keys = static_cast<int32_t*>(take(rows));
  w.sid = static_cast<int32_t*>(take(rows));
  w.perm = static_cast<int32_t*>(take(rows));
  w.offsets = static_cast<int32_t*>(take(align_up(size_t(vocab + 2) * sizeof(int32_t), 256)));
  w.stats = static_cast<int32_t*>(take(256));
  w.sort_bytes = plan_workspace_bytes_impl(n, vocab + 1, 0) + 256;
  w.sort = take(w.sort_bytes);
  w.bytes = at + 256;
  return w;
}

template <typename T, int BYTES>
int launch_backward(const T* g, const BackwardWorkspace& w, int64_t vocab, int dim, float scale, T* g_weight,
                    cudaStream_t stream) {
  const int64_t vectors = dim / RowShape<T, BYTES>::kVec;
  const int lanes = lanes_of(vectors);
  const dim3 grid(unsigned(ceil_div(vocab, kThreads / lanes)), unsigned(ceil_div(vectors, lanes * RowShape<T, BYTES>::kBlocks)));
  if (grid.y > 65535u) return fail(TEXB_ERR_UNSUPPORTED, "embedding: rows of %d values are too wide", dim);
  embedding_backward_rows_kernel<T, BYTES><<<grid, kThreads, 0, stream>>>(g, w.perm, w.offsets, vocab, dim, scale,
                                                                          g_weight, lanes);
  return check_launch("embedding_backward_rows_kernel");
}

template <typename T>
int backward_typed(const void* g, const BackwardWorkspace& w, int64_t vocab, int dim, float scale, void* g_weight,
                   cudaStream_t stream) {
  const T* gp = static_cast<const T*>(g);
  T* o = static_cast<T*>(g_weight);
  const int bytes = access_bytes(int(sizeof(T)), dim, g, g_weight);
  if (bytes == 16) return launch_backward<T, 16>(gp, w, vocab, dim, scale, o, stream);
  if (bytes == 4) return launch_backward<T, 4>(gp, w, vocab, dim, scale, o, stream);
  return launch_backward<T, int(sizeof(T))>(gp, w, vocab, dim, scale, o, stream);
}

int check_sizes(int id_bytes, int64_t n, int dtype, int64_t vocab, int dim) {
  if (id_bytes != 4 && id_bytes != 8)
    return fail(TEXB_ERR_INVALID_ARGUMENT, "id_bytes must be 4 or 8, got %d", id_bytes);
  if (!dtype_known(dtype)) return fail(TEXB_ERR_INVALID_ARGUMENT, "embedding: unknown dtype %d", dtype);
  if (n < 0 || vocab < 0 || dim < 1) return fail(TEXB_ERR_INVALID_ARGUMENT, "embedding: bad sizes");
  if (n > INT_MAX - 65536 || vocab > INT_MAX - 65536)
    return fail(TEXB_ERR_UNSUPPORTED, "embedding: tokens and vocab must be below 2^31 - 65536");
  return TEXB_OK;
}

}  // namespace

int embedding_bad_tokens_impl(int* count) {
  const cudaError_t e = cudaMemcpyFromSymbol(count, g_bad_tokens, sizeof(int));
  if (e != cudaSuccess) return fail(TEXB_ERR_CUDA, "device status: %s", cudaGetErrorString(e));
  return TEXB_OK;
}

int embedding_forward_impl(const void* tokens, int id_bytes, int64_t n, const void* weight, int dtype, int64_t vocab,
                           int dim, float scale, void* out, cudaStream_t stream) {
  int st = check_sizes(id_bytes, n, dtype, vocab, dim);
  if (st != TEXB_OK) return st;
  if (n == 0) return TEXB_OK;
  if (!tokens || !out || (vocab > 0 && !weight)) return fail(TEXB_ERR_INVALID_ARGUMENT, "embedding: NULL pointer");
  if (dtype == TEXB_FLOAT32)
    return forward_typed<float>(tokens, id_bytes, n, weight, vocab, dim, scale, out, stream);
  if (dtype == TEXB_BFLOAT16)
    return forward_typed<__nv_bfloat16>(tokens, id_bytes, n, weight, vocab, dim, scale, out, stream);
  return forward_typed<__half>(tokens, id_bytes, n, weight, vocab, dim, scale, out, stream);
}

size_t embedding_backward_workspace_bytes_impl(int64_t n, int64_t vocab, int dim) {
  if (n < 0 || vocab < 0 || dim < 1) return 0;
  return carve_backward(nullptr, n, vocab).bytes;
}

int embedding_backward_impl(const void* tokens, int id_bytes, int64_t n, const void* g, int dtype, int64_t vocab,
                            int dim, float scale, int64_t padding_idx, void* g_weight, void* workspace,
                            size_t workspace_bytes, cudaStream_t stream) {
  int st = check_sizes(id_bytes, n, dtype, vocab, dim);
  if (st != TEXB_OK) return st;
  if (vocab == 0) return TEXB_OK;
  if (!g_weight || (n > 0 && (!tokens || !g))) return fail(TEXB_ERR_INVALID_ARGUMENT, "embedding: NULL pointer");
  const BackwardWorkspace w = carve_backward(workspace, n, vocab);
  if (!workspace || workspace_bytes < w.bytes)
    return fail(TEXB_ERR_WORKSPACE, "embedding workspace: need %zu bytes, got %zu", w.bytes, workspace_bytes);
  if (n > 0) {
    const unsigned blocks = unsigned(ceil_div(n, kThreads));
    if (id_bytes == 8)
      embedding_keys_kernel<int64_t><<<blocks, kThreads, 0, stream>>>(static_cast<const int64_t*>(tokens), int(n), vocab, padding_idx, w.keys);
    else
      embedding_keys_kernel<int32_t><<<blocks, kThreads, 0, stream>>>(static_cast<const int32_t*>(tokens), int(n), vocab, padding_idx, w.keys);
    st = check_launch("embedding_keys_kernel");
    if (st != TEXB_OK) return st;
  }
  st = plan_build_impl(w.keys, 4, n, vocab + 1, 0, w.sid, w.perm, w.offsets, w.stats, w.sort, w.sort_bytes, stream);
  if (st != TEXB_OK) return st;
  if (dtype == TEXB_FLOAT32) return backward_typed<float>(g, w, vocab, dim, scale, g_weight, stream);
  if (dtype == TEXB_BFLOAT16) return backward_typed<__nv_bfloat16>(g, w, vocab, dim, scale, g_weight, stream);
  return backward_typed<__half>(g, w, vocab, dim, scale, g_weight, stream);
}

}  // namespace texb
