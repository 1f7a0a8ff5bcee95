// The 2-norm over a list of tensors, and the tensors scaled down to a largest norm:
//   norm = sqrt(sum over all values x of x^2),   y = x * min(1, max_norm / (norm + 1e-6)).
//
// Bound by HBM: the norm reads every value once, the scaling reads them again and writes them.
// A list is one launch per pass, whatever the number and sizes of its tensors: pointers and sizes
// travel in the kernel's parameters (no copy to the device, so the call can be captured in a
// graph), the tensors are cut into chunks of 16 KB, and one resident wave of CTAs walks the
// chunks with 64 bytes of loads in flight per thread.  The second pass walks them from the last to the first,
// so that what the first pass read last still comes from L2, and stores past it; it reads the coefficient's
// partial sums itself, which saves a launch, and leaves tensors that are scaled in place alone when the
// coefficient is 1.  Measured: 100 M bf16 values in 60 tensors, read twice and written once, 104 us (5.8 TB/s of
// all bytes moved); 400 M into fp32 559 us; 60 000 values 10.6 us, which is the two launches.
//
// The squares of eight values are added in fp32, everything above that in fp64: the result is
// within a few 2^-24 of the exact norm whatever the number of values.  A group of eight whose sum
// leaves the range where fp32 squares lose nothing (tiny, huge, infinite, NaN) is added again in
// fp64, so a norm overflows only where it cannot be held in fp32.  There are no atomics: partial
// sums are added in a fixed order, and every CTA arrives at the same coefficient.

#include <climits>
#include <cmath>

#include "vector_io.cuh"

namespace texb {
namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 8;              // squares that are added in fp32
constexpr int kInFlight = 64;          // bytes of loads of a thread before the first is used (128: larger chunks,
                                       // an eighth slower for 100 M values, as the last chunks leave SMs idle)
constexpr int kChunkBytes = kThreads * kInFlight;
inline int64_t chunk_values(int dtype) { return kChunkBytes / dtype_bytes(dtype); }
constexpr int kCtasPerSm = 4;
constexpr int kWave = 148 * kCtasPerSm;

// How a tensor is read and written: its types, and whether rows of eight values are aligned.
constexpr int kTypeBits = 2;
constexpr int kWide = 1 << (2 * kTypeBits);
inline uint8_t kind_of(int in, int out, bool wide) { return uint8_t(in | out << kTypeBits | (wide ? kWide : 0)); }

// One launch's share of the list.  `capacity` is chosen by the length of the list: the parameters
// are copied at every launch.
template <int CAPACITY>
struct List {
  const void* in[CAPACITY];
  void* out[CAPACITY];
  int64_t size[CAPACITY];
  uint32_t chunk_end[CAPACITY];  // chunks of tensors 0 .. i
  uint8_t kind[CAPACITY];
  int count;
  uint32_t chunks;
};
constexpr int kSmall = 64, kMedium = 256, kLarge = 1024;
static_assert(sizeof(List<kLarge>) <= 32000, "kernel parameters are limited to 32 764 bytes");

template <int CAPACITY>
__device__ __forceinline__ int tensor_of(const List<CAPACITY>& l, uint32_t chunk) {
  int lo = 0, hi = l.count - 1;  // the first tensor whose chunks end behind `chunk`
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (l.chunk_end[mid] > chunk) hi = mid; else lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ void add_squares(const float (&v)[kGroup], double& sum) {
  float s = v[0] * v[0];
#pragma unroll
  for (int e = 1; e < kGroup; ++e) s = fmaf(v[e], v[e], s);
  if (s > 1e-28f && s < INFINITY) {  // squares that underflowed are below 1e-45
    sum += double(s);
    return;
  }
  uint32_t bits = 0u;
#pragma unroll
  for (int e = 0; e < kGroup; ++e) bits |= __float_as_uint(v[e]) << 1;
  if (bits == 0u) return;  // zeros, as in the gradient of a table
#pragma unroll
  for (int e = 0; e < kGroup; ++e) sum = fma(double(v[e]), double(v[e]), sum);
}

// `wide`: p is aligned to 16 bytes.  A full chunk is read 16 bytes per lane, neighbouring lanes side by side.
template <typename T>
__device__ __forceinline__ void square_chunk(const T* p, int count, bool wide, double& sum) {
  constexpr int kPer = 16 / int(sizeof(T)), kLoads = kInFlight / 16, kLoadsPerGroup = kGroup / kPer;
  float v[kGroup];
  if (wide && count == kThreads * kLoads * kPer) {
    Chunk<T, 16> c[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) c[k] = load_chunk<T, 16>(p + (k * kThreads + int(threadIdx.x)) * kPer);
#pragma unroll
    for (int k = 0; k < kLoads; k += kLoadsPerGroup) {
#pragma unroll
      for (int e = 0; e < kGroup; ++e) v[e] = widen<T>(c[k + e / kPer].v[e % kPer]);
      add_squares(v, sum);
    }
    return;
  }
  // the end of a tensor, or one that begins anywhere: single values, eight in flight
  for (int i = threadIdx.x; i < count; i += kThreads * kGroup) {
#pragma unroll
    for (int e = 0; e < kGroup; ++e) v[e] = i + e * kThreads < count ? widen<T>(__ldg(p + i + e * kThreads)) : 0.f;
    add_squares(v, sum);
  }
}

// The sum over the CTA, in every thread, always in the same order.
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double s_warp[kThreads / 32];
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = v;
  __syncthreads();
  double total = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) total += s_warp[w];
  return total;
}

template <int CAPACITY>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
square_sums_kernel(const __grid_constant__ List<CAPACITY> list, double* __restrict__ partial) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  double sum = 0.0;
  for (uint32_t c = blockIdx.x; c < list.chunks; c += gridDim.x) {
    const int t = tensor_of(list, c);
    const int in = list.kind[t] & ((1 << kTypeBits) - 1);
    const int chunk = kChunkBytes / (in == TEXB_FLOAT32 ? 4 : 2);
    const int64_t at = int64_t(c - (t > 0 ? list.chunk_end[t - 1] : 0u)) * chunk;
    const int count = int(min(int64_t(chunk), list.size[t] - at));
    const bool wide = list.kind[t] & kWide;
    switch (in) {
      case TEXB_FLOAT32: square_chunk<float>(static_cast<const float*>(list.in[t]) + at, count, wide, sum); break;
      case TEXB_BFLOAT16: square_chunk<__nv_bfloat16>(static_cast<const __nv_bfloat16*>(list.in[t]) + at, count, wide, sum); break;
      default: square_chunk<__half>(static_cast<const __half*>(list.in[t]) + at, count, wide, sum); break;
    }
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

__device__ __forceinline__ float norm_of(const double* __restrict__ partial, int partials) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < partials; i += kThreads) sum += partial[i];
  return float(sqrt(block_sum(sum)));
}

__global__ void __launch_bounds__(kThreads)
norm_kernel(const double* __restrict__ partial, int partials, float* __restrict__ norm_out) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float norm = norm_of(partial, partials);
  if (threadIdx.x == 0) norm_out[0] = norm;
}

// Loads and stores run over the same values per lane, at most 16 bytes of either: 16-bit values into fp32
// ones are read 8 bytes per lane, so that neighbouring lanes store side by side (stores of 32 bytes per
// lane as two halves took 517 us instead of 418 for 400 M values).
template <typename In, typename Out>
__device__ __forceinline__ void scale_chunk(const In* p, Out* q, int count, bool wide, float coef) {
  constexpr int kPer = 16 / int(sizeof(Out) > sizeof(In) ? sizeof(Out) : sizeof(In));
  constexpr int kBytes = kPer * int(sizeof(In)), kLoads = kInFlight / kBytes;
  if (wide && count == kThreads * kLoads * kPer) {
    Chunk<In, kBytes> c[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) c[k] = load_chunk_once<In, kBytes>(p + (k * kThreads + int(threadIdx.x)) * kPer);
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      Chunk<Out, kPer * int(sizeof(Out))> o;
#pragma unroll
      for (int e = 0; e < kPer; ++e) o.v[e] = narrow<Out>(widen<In>(c[k].v[e]) * coef);
      store_chunk_once<Out, kPer * int(sizeof(Out))>(q + (k * kThreads + int(threadIdx.x)) * kPer, o);
    }
    return;
  }
  for (int i = threadIdx.x; i < count; i += kThreads * kGroup) {
    In v[kGroup];
#pragma unroll
    for (int e = 0; e < kGroup; ++e)
      if (i + e * kThreads < count) v[e] = __ldcs(p + i + e * kThreads);
#pragma unroll
    for (int e = 0; e < kGroup; ++e)
      if (i + e * kThreads < count) q[i + e * kThreads] = narrow<Out>(widen<In>(v[e]) * coef);
  }
}

template <int CAPACITY>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
scale_kernel(const __grid_constant__ List<CAPACITY> list, const double* __restrict__ partial, int partials, float max_norm,
             float* __restrict__ norm_out) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float norm = norm_of(partial, partials);
  if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = norm;
  float coef = __fdiv_rn(max_norm, norm + 1e-6f);
  coef = coef >= 1.f ? 1.f : coef;  // a NaN norm makes every value NaN
  for (uint32_t k = blockIdx.x; k < list.chunks; k += gridDim.x) {
    const uint32_t c = list.chunks - 1 - k;
    const int t = tensor_of(list, c);
    if (coef == 1.f && list.in[t] == list.out[t]) continue;
    const int in = list.kind[t] & ((1 << kTypeBits) - 1);
    const int chunk = kChunkBytes / (in == TEXB_FLOAT32 ? 4 : 2);
    const int64_t at = int64_t(c - (t > 0 ? list.chunk_end[t - 1] : 0u)) * chunk;
    const int count = int(min(int64_t(chunk), list.size[t] - at));
    const bool wide = list.kind[t] & kWide;
#define TEXB_SCALE(In, Out) \
  scale_chunk<In, Out>(static_cast<const In*>(list.in[t]) + at, static_cast<Out*>(list.out[t]) + at, count, wide, coef)
    switch (list.kind[t] & (kWide - 1)) {
      case TEXB_FLOAT32 | TEXB_FLOAT32 << kTypeBits: TEXB_SCALE(float, float); break;
      case TEXB_BFLOAT16 | TEXB_BFLOAT16 << kTypeBits: TEXB_SCALE(__nv_bfloat16, __nv_bfloat16); break;
      case TEXB_FLOAT16 | TEXB_FLOAT16 << kTypeBits: TEXB_SCALE(__half, __half); break;
      case TEXB_BFLOAT16 | TEXB_FLOAT32 << kTypeBits: TEXB_SCALE(__nv_bfloat16, float); break;
      default: TEXB_SCALE(__half, float); break;
    }
#undef TEXB_SCALE
  }
}

// ---- launches --------------------------------------------------------------------------------

template <typename K, typename... Args>
int launch(const char* what, K kernel, unsigned grid, cudaStream_t stream, bool dependent, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return fail(TEXB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

struct Request {
  int count;
  const void* const* in;
  const int64_t* sizes;
  const int* dtypes;
  void* const* out;       // NULL: only the norm is wanted
  const int* out_dtypes;
};

inline unsigned wave(uint32_t chunks) { return chunks < unsigned(kWave) ? (chunks > 0 ? chunks : 1u) : unsigned(kWave); }

// Fills the share of the list that begins at tensor `first`; returns the tensor behind it.  A share
// ends at the capacity, or where its chunks would no longer fit 32 bits.
template <int CAPACITY>
int fill(const Request& r, int first, List<CAPACITY>& l) {
  l.count = 0;
  l.chunks = 0;
  int i = first;
  for (; i < r.count && l.count < CAPACITY; ++i) {
    if (r.sizes[i] == 0) continue;
    const int64_t chunks = ceil_div(r.sizes[i], chunk_values(r.dtypes[i]));
    if (int64_t(l.chunks) + chunks > INT_MAX) break;
    const int out_dtype = r.out ? r.out_dtypes[i] : r.dtypes[i];
    void* out = r.out ? r.out[i] : nullptr;
    const bool wide = reinterpret_cast<uintptr_t>(r.in[i]) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    l.in[l.count] = r.in[i];
    l.out[l.count] = out;
    l.size[l.count] = r.sizes[i];
    l.chunks += uint32_t(chunks);
    l.chunk_end[l.count] = l.chunks;
    l.kind[l.count] = kind_of(r.dtypes[i], out_dtype, wide);
    ++l.count;
  }
  return i;
}

template <int CAPACITY>
int run(const Request& r, float max_norm, double* partial, float* norm_out, cudaStream_t stream) {
  List<CAPACITY> l;
  int partials = 0, launches = 0;
  for (int at = 0; at < r.count || launches == 0; ++launches) {
    at = fill(r, at, l);
    const unsigned grid = wave(l.chunks);
    const int st = launch("square_sums_kernel", square_sums_kernel<CAPACITY>, grid, stream, false, l, partial + partials);
    if (st != TEXB_OK) return st;
    partials += int(grid);
  }
  if (!r.out) return launch("norm_kernel", norm_kernel, 1u, stream, launches == 1, partial, partials, norm_out);
  float* first_norm = norm_out;
  for (int at = 0, k = 0; k < launches; ++k) {
    if (launches > 1) at = fill(r, at, l);
    // only the launch right behind the sums of a single share may be placed early: the scaling of one
    // share must not start before the sums of all are complete
    const int st = launch("scale_kernel", scale_kernel<CAPACITY>, wave(l.chunks), stream, launches == 1, l, partial, partials,
                          max_norm, first_norm);
    if (st != TEXB_OK) return st;
    first_norm = nullptr;
  }
  return TEXB_OK;
}

int check(const Request& r, const float* norm_out, const void* workspace, size_t workspace_bytes) {
  if (r.count < 0) return fail(TEXB_ERR_INVALID_ARGUMENT, "grad_norm: negative count");
  if (!norm_out || (r.count > 0 && (!r.in || !r.sizes || !r.dtypes)))
    return fail(TEXB_ERR_INVALID_ARGUMENT, "grad_norm: NULL pointer");
  for (int i = 0; i < r.count; ++i) {
    if (r.sizes[i] < 0) return fail(TEXB_ERR_INVALID_ARGUMENT, "grad_norm: tensor %d has a negative size", i);
    if (!dtype_known(r.dtypes[i])) return fail(TEXB_ERR_INVALID_ARGUMENT, "grad_norm: tensor %d has an unknown dtype", i);
    if (r.sizes[i] / chunk_values(r.dtypes[i]) >= INT_MAX) return fail(TEXB_ERR_UNSUPPORTED, "grad_norm: tensor %d is too large", i);
    if (r.sizes[i] > 0 && !r.in[i]) return fail(TEXB_ERR_INVALID_ARGUMENT, "grad_norm: tensor %d is NULL", i);
    if (!r.out) continue;
    if (r.sizes[i] > 0 && !r.out[i]) return fail(TEXB_ERR_INVALID_ARGUMENT, "clip_grads: output %d is NULL", i);
    if (r.out_dtypes[i] != r.dtypes[i] && r.out_dtypes[i] != TEXB_FLOAT32)
      return fail(TEXB_ERR_UNSUPPORTED, "clip_grads: output %d must have its input's dtype or float32", i);
    if (r.out[i] == r.in[i] && r.out_dtypes[i] != r.dtypes[i] && r.sizes[i] > 0)
      return fail(TEXB_ERR_INVALID_ARGUMENT, "clip_grads: output %d is in place but of another dtype", i);
  }
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 8 != 0 || workspace_bytes < texb_grad_norm_workspace_bytes(r.count))
    return fail(TEXB_ERR_WORKSPACE, "grad_norm workspace: need %zu bytes aligned to 8, got %zu",
                texb_grad_norm_workspace_bytes(r.count), workspace_bytes);
  return TEXB_OK;
}

int run_any(const Request& r, float max_norm, void* workspace, float* norm_out, cudaStream_t stream) {
  double* partial = static_cast<double*>(workspace);
  if (r.count <= kSmall) return run<kSmall>(r, max_norm, partial, norm_out, stream);
  if (r.count <= kMedium) return run<kMedium>(r, max_norm, partial, norm_out, stream);
  return run<kLarge>(r, max_norm, partial, norm_out, stream);
}

}  // namespace

size_t grad_norm_workspace_bytes_impl(int count) {
  if (count < 0) return 0;
  // one partial sum per CTA of every launch; a tensor of 2^45 values could end a share of the list early
  return size_t(kWave) * sizeof(double) * (size_t(count) / kSmall + 2) * 2;
}

int grad_norm_impl(int count, const void* const* grads, const int64_t* sizes, const int* dtypes, float* norm_out,
                   void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  const Request r = {count, grads, sizes, dtypes, nullptr, nullptr};
  const int st = check(r, norm_out, workspace, workspace_bytes);
  return st == TEXB_OK ? run_any(r, 0.f, workspace, norm_out, stream) : st;
}

int clip_grads_impl(int count, const void* const* grads, const int64_t* sizes, const int* dtypes, void* const* outs,
                    const int* out_dtypes, float max_norm, float* norm_out, void* workspace, size_t workspace_bytes,
                    cudaStream_t stream) {
  static void* const kNoOut = nullptr;
  static const int kNoType = 0;
  if (count > 0 && (!outs || !out_dtypes)) return fail(TEXB_ERR_INVALID_ARGUMENT, "clip_grads: NULL pointer");
  if (!(max_norm >= 0.f)) return fail(TEXB_ERR_INVALID_ARGUMENT, "clip_grads: max_norm must not be negative");
  const Request r = {count, grads, sizes, dtypes, count > 0 ? outs : &kNoOut, count > 0 ? out_dtypes : &kNoType};
  const int st = check(r, norm_out, workspace, workspace_bytes);
  return st == TEXB_OK ? run_any(r, max_norm, workspace, norm_out, stream) : st;
}

}  // namespace texb
