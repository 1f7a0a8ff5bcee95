// Rows of a table by token: out[t, :] = scale * weight[token_t, :].
//
// Bound by HBM (every distinct looked-up row is read once -- frequent ones come from L2 -- and n
// rows are written) and, for the few rows of a decoding step, by three dependent trips to memory.
// A group of lanes (a warp for wide rows) copies one chunk of a row with up to four 16-byte loads
// in flight per lane before the first store; wide rows are cut into chunks so that a handful of
// tokens still spreads over the SMs.  Measured: 64 rows of 1024 bf16 values 5.5 us, launch included; 16 384 of
// them out of a table of 32 768 10.6 us.
//
// A token outside [0, vocab) reads nothing: its output row is zero and it is counted
// (texb_device_status, bad_indices).

#include <climits>

#include "embedding.cuh"

namespace texb {

namespace {

static __device__ int g_bad_tokens = 0;

constexpr int kThreads = 256;

template <typename T, int BYTES, typename IdT, bool SCALED>
__global__ void __launch_bounds__(kThreads)
embedding_forward_kernel(const IdT* __restrict__ tokens, int64_t n, const T* __restrict__ weight, int64_t vocab,
                         int dim, float scale, T* __restrict__ out, int lanes, int chunks) {
  constexpr int kVec = Chunk<T, BYTES>::kCount;
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

template <typename T, int BYTES>
int launch_lookup(const void* tokens, int id_bytes, int64_t n, const T* weight, int64_t vocab, int dim, float scale,
                   T* out, cudaStream_t stream) {
  const int64_t vectors = dim / Chunk<T, BYTES>::kCount;
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
int lookup_typed(const void* tokens, int id_bytes, int64_t n, const void* weight, int64_t vocab, int dim, float scale,
                  void* out, cudaStream_t stream) {
  const T* w = static_cast<const T*>(weight);
  T* o = static_cast<T*>(out);
  const int bytes = access_bytes(int(sizeof(T)), dim, weight, out);
  if (bytes == 16) return launch_lookup<T, 16>(tokens, id_bytes, n, w, vocab, dim, scale, o, stream);
  if (bytes == 4) return launch_lookup<T, 4>(tokens, id_bytes, n, w, vocab, dim, scale, o, stream);
  return launch_lookup<T, int(sizeof(T))>(tokens, id_bytes, n, w, vocab, dim, scale, o, stream);
}

}  // namespace

int lookup_bad_tokens_impl(int* count) {
  const cudaError_t e = cudaMemcpyFromSymbol(count, g_bad_tokens, sizeof(int));
  if (e != cudaSuccess) return fail(TEXB_ERR_CUDA, "device status: %s", cudaGetErrorString(e));
  return TEXB_OK;
}

int embedding_forward_impl(const void* tokens, int id_bytes, int64_t n, const void* weight, int dtype, int64_t vocab,
                           int dim, float scale, void* out, cudaStream_t stream) {
  int st = check_embedding_sizes(id_bytes, n, dtype, vocab, dim);
  if (st != TEXB_OK) return st;
  if (n == 0) return TEXB_OK;
  if (!tokens || !out || (vocab > 0 && !weight)) return fail(TEXB_ERR_INVALID_ARGUMENT, "embedding: NULL pointer");
  if (dtype == TEXB_FLOAT32)
    return lookup_typed<float>(tokens, id_bytes, n, weight, vocab, dim, scale, out, stream);
  if (dtype == TEXB_BFLOAT16)
    return lookup_typed<__nv_bfloat16>(tokens, id_bytes, n, weight, vocab, dim, scale, out, stream);
  return lookup_typed<__half>(tokens, id_bytes, n, weight, vocab, dim, scale, out, stream);
}

}  // namespace texb
