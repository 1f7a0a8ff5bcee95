// Forward kernel of the attention within segments; instantiated by the attention_forward_*.cu files.
//
// A CTA of four warps owns 64 query positions of one head, 16 per warp, and walks the keys its rows
// see in tiles of 64 (32 for narrow rows): scores, running maximum and sum (in units of log2), and the product with the
// values stay in registers; keys and values are copied ahead (cp.async, two to four stages).  A warp
// passes over tiles that none of its 16 rows see, which is what keeps a tile of many short segments
// cheap, and over the mask where all of its rows see the whole tile.  Probabilities are rounded to the
// type of the values before the second product, which the matrix instructions require: half a step
// of that type each (2^-8 for bf16, 2^-11 for fp16), averaged over the keys.
// Bound: instruction issue (masks and exponentials; for heads of 16 columns there are eight multiply-adds to each).
// Measured: 20 000 rows, 8 heads of 16, segments up to 128: 30 us, issue slots 58 % busy.
#pragma once

#include "attention.cuh"

namespace texb {
namespace attention {

template <typename T, int DP>
struct ForwardMemory {
  static constexpr int kStages = DP <= 32 ? 4 : 2;  // narrow rows: most keys of a tile of short segments at once
  static constexpr int kKeys = DP <= 32 ? 32 : 64;  // of a stage; fewer where most of a tile of 64 would be masked
  static constexpr int kQ = 0, kQueries = kBlock * DP * 2;
  static constexpr int kTile = kKeys * DP * 2;
  static constexpr int kK = kQueries, kV = kK + kStages * kTile;
  static constexpr int kBytes = kQueries + 2 * kStages * kTile;
};

template <typename T, int DP, int MODE>
__global__ void __launch_bounds__(kThreads, DP <= 32 ? 6 : 1) forward_kernel(const __grid_constant__ Problem a) {
  extern __shared__ __align__(128) unsigned char smem[];
  using M = ForwardMemory<T, DP>;
  const int head = blockIdx.y, kv = head / (a.heads / a.kv_heads);
  const int pos0 = blockIdx.x * kBlock, last = min(a.n, pos0 + kBlock) - 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first_key = keys_of(a, pos0).begin, end_key = keys_of(a, last).end;

  const uint32_t base = smem_u32(smem), sq = base + M::kQ;
  constexpr int S = M::kStages, N = M::kKeys;
  Loader<DP, kBlock> queries;
  Loader<DP, N> ahead[S - 1], loader;
  queries.look_up(a, pos0, last + 1);
#pragma unroll
  for (int t = 0; t < S - 1; ++t) ahead[t].look_up(a, first_key + t * N, end_key);
  queries.template copy<T>(a, a.q, head, sq);
#pragma unroll
  for (int t = 0; t < S - 1; ++t) {
    if (first_key + t * N < end_key) {
      ahead[t].template copy<T>(a, a.k, kv, base + M::kK + t * M::kTile);
      ahead[t].template copy<T>(a, a.v, kv, base + M::kV + t * M::kTile);
    }
    commit_copies();
  }
  loader.look_up(a, first_key + (S - 1) * N, end_key);
  // looked at while the first rows are on their way
  const bool bad = a.bad_v ? any_flag(a, a.bad_v, kv, first_key, end_key) : look_over<T>(a, a.v, kv, first_key, end_key);
  if (bad) {
    wait_copies<0>();
    plain_forward<T>(a, pos0, kBlock, head);
    return;
  }

  const int row0 = warp * 16, i0 = pos0 + row0 + (lane >> 2), i1 = i0 + 8;
  const Bounds see0 = keys_of(a, i0), see1 = keys_of(a, i1);
  // of the warp's rows: the first key and the end of what any of them sees, and of what all of them see
  const int warp_begin = keys_of(a, pos0 + row0).begin, warp_last = min(last, pos0 + row0 + 15);
  const Bounds tail = pos0 + row0 <= last ? keys_of(a, warp_last) : Bounds{0, 0};
  const int warp_end = tail.end;
  const int all_begin = tail.begin, all_end = pos0 + row0 + 15 <= last ? keys_of(a, pos0 + row0).end : 0;
  const float slope = MODE != kPlain ? slope_of(a, head) : 0.f;

  constexpr float kLift = kLifted<T, 15>;  // no probability is above 1
  float out[DP / 8][4] = {};
  float top0 = -INFINITY, top1 = -INFINITY, sum0 = 0.f, sum1 = 0.f;
  int stage = 0;
  for (int j0 = first_key; j0 < end_key; j0 += N) {
    wait_copies<S - 2>();
    __syncthreads();  // this tile is there, and the stage of the last one is free
    if (j0 + (S - 1) * N < end_key) {
      const int free = stage == 0 ? S - 1 : stage - 1;
      loader.template copy<T>(a, a.k, kv, base + M::kK + free * M::kTile);
      loader.template copy<T>(a, a.v, kv, base + M::kV + free * M::kTile);
    }
    commit_copies();
    loader.look_up(a, j0 + S * N, end_key);
    if (j0 + N > warp_begin && j0 < warp_end) {
      constexpr int NT = N / 8;
      float s[NT][4] = {};
      product_rows<T, DP, NT>(s, sq, row0, base + M::kK + stage * M::kTile);
      const bool whole = j0 >= all_begin && j0 + N <= all_end;
      float top0_new = top0, top1_new = top1;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = j0 + t * 8 + (lane & 3) * 2 + e;
          s[t][e] = score_of<MODE>(a, s[t][e], slope, float(i0 - j)).x;
          s[t][2 + e] = score_of<MODE>(a, s[t][2 + e], slope, float(i1 - j)).x;
          if (!whole) {
            if (!see0.holds(j)) s[t][e] = -INFINITY;
            if (!see1.holds(j)) s[t][2 + e] = -INFINITY;
          }
          top0_new = fmaxf(top0_new, s[t][e]);
          top1_new = fmaxf(top1_new, s[t][2 + e]);
        }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        top0_new = fmaxf(top0_new, __shfl_xor_sync(0xffffffffu, top0_new, o));
        top1_new = fmaxf(top1_new, __shfl_xor_sync(0xffffffffu, top1_new, o));
      }
      // no visible key so far: subtract 0, so that the weights become 0 and not NaN
      const float base0 = top0_new == -INFINITY ? 0.f : top0_new, base1 = top1_new == -INFINITY ? 0.f : top1_new;
      const float less0 = base0 - kLift, less1 = base1 - kLift;
      const float shrink0 = exp2_fast(top0 - base0), shrink1 = exp2_fast(top1 - base1);
      top0 = top0_new;
      top1 = top1_new;
      sum0 *= shrink0;
      sum1 *= shrink1;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[t][e] = exp2_fast(s[t][e] - less0);
          s[t][2 + e] = exp2_fast(s[t][2 + e] - less1);
          sum0 += s[t][e];
          sum1 += s[t][2 + e];
        }
      }
#pragma unroll
      for (int t = 0; t < DP / 8; ++t) {
        out[t][0] *= shrink0;
        out[t][1] *= shrink0;
        out[t][2] *= shrink1;
        out[t][3] *= shrink1;
      }
      product_probabilities<T, DP, NT>(out, s, base + M::kV + stage * M::kTile);
    }
    stage = stage + 1 == S ? 0 : stage + 1;
  }
  wait_copies<0>();
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    sum0 += __shfl_xor_sync(0xffffffffu, sum0, o);
    sum1 += __shfl_xor_sync(0xffffffffu, sum1, o);
  }
  // a row sees itself, so only rows behind the last position have an empty sum
  const bool none0 = see0.end <= see0.begin, none1 = see1.end <= see1.begin;
  if (a.lse && (lane & 3) == 0) {
    if (i0 < a.n) a.lse[int64_t(head) * a.n + i0] = none0 ? 0.f : top0 - kLift + log2f(sum0);
    if (i1 < a.n) a.lse[int64_t(head) * a.n + i1] = none1 ? 0.f : top1 - kLift + log2f(sum1);
  }
  const float factor0 = none0 ? 0.f : 1.f / sum0, factor1 = none1 ? 0.f : 1.f / sum1;
  store_rows<T, DP>(a, a.out, head, pos0 + row0, out, factor0, factor1, smem + M::kQ, row0);
  if (a.out_low.p) store_rows<T, DP, true>(a, a.out_low, head, pos0 + row0, out, factor0, factor1, smem + M::kQ, row0);
}

template <typename T, int DP, int MODE>
int launch_forward(const Problem& a, cudaStream_t stream) {
  auto kernel = forward_kernel<T, DP, MODE>;
  constexpr int bytes = ForwardMemory<T, DP>::kBytes;
  if (bytes > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return fail(TEXB_ERR_CUDA, "attention forward_kernel: %s", cudaGetErrorString(e));
  }
  const dim3 grid(unsigned((a.n + kBlock - 1) / kBlock), unsigned(a.heads));
  kernel<<<grid, kThreads, bytes, stream>>>(a);
  return check_launch("attention forward_kernel");
}

template <int DP>
int forward_by_type(const Problem& a, int dtype, int mode, cudaStream_t stream) {
  const bool bf16 = dtype == TEXB_BFLOAT16;
  if (mode == kCapped) return bf16 ? launch_forward<__nv_bfloat16, DP, kCapped>(a, stream) : launch_forward<__half, DP, kCapped>(a, stream);
  if (mode == kBiased) return bf16 ? launch_forward<__nv_bfloat16, DP, kBiased>(a, stream) : launch_forward<__half, DP, kBiased>(a, stream);
  return bf16 ? launch_forward<__nv_bfloat16, DP, kPlain>(a, stream) : launch_forward<__half, DP, kPlain>(a, stream);
}

}  // namespace attention
}  // namespace texb
