// Backward kernels of the attention within segments; instantiated by the attention_backward_*.cu files.
//
// The probabilities are computed again from the scores and the log-sums of the forward pass.  Two
// kernels, so that every gradient is summed by one CTA in a fixed order (no atomics, the same bits
// every time), at the price of computing the scores twice:
//   queries: as the forward kernel, 64 query positions of one head against the keys they see;
//   keys   : 64 key positions of one kv head against the queries that see them, of all query heads
//            that share it -- the gradient of a shared key or value is one sum.
// P is rounded to the inputs' type before its product (half a step); dS goes in as two such values, which costs
// little here and halves the squared error of gq and gk:
//   dS = P (scale g v - delta) x (derivative of the capped score), delta = scale g o,  gq = dS k, gk = dS^T q, gv = P^T g.
// In fp16 both are lifted first (attention.cuh), so that values far below its smallest normal number keep their bits.
// A masked pair's dS is set to 0, not multiplied by 0: its g v may be infinite.
// Bound as the forward kernel.  Measured: 20 000 rows, 8 heads of 16, segments up to 128: 31 us for the queries, 42
// for the keys and values; 33 and 47 in fp16.
#pragma once

#include "attention.cuh"

namespace texb {
namespace attention {

template <int DP>
struct QueryMemory {
  static constexpr int kStages = DP <= 32 ? 4 : 2, kKeys = DP <= 32 ? 32 : 64;
  static constexpr int kQueries = kBlock * DP * 2, kTile = kKeys * DP * 2;
  static constexpr int kQ = 0, kG = kQueries, kK = 2 * kQueries, kV = kK + kStages * kTile;
  static constexpr int kBytes = 2 * kQueries + 2 * kStages * kTile;
};

template <typename T, int DP, int MODE>
__global__ void __launch_bounds__(kThreads, DP <= 32 ? 6 : 1) query_gradient_kernel(const __grid_constant__ Problem a) {
  extern __shared__ __align__(128) unsigned char smem[];
  using M = QueryMemory<DP>;
  const int head = blockIdx.y, kv = head / (a.heads / a.kv_heads);
  const int pos0 = blockIdx.x * kBlock, last = min(a.n, pos0 + kBlock) - 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first_key = keys_of(a, pos0).begin, end_key = keys_of(a, last).end;
  const uint32_t base = smem_u32(smem);
  constexpr int S = M::kStages, N = M::kKeys;
  Loader<DP, kBlock> queries;
  Loader<DP, N> ahead[S - 1], loader;
  queries.look_up(a, pos0, last + 1);
#pragma unroll
  for (int t = 0; t < S - 1; ++t) ahead[t].look_up(a, first_key + t * N, end_key);
  queries.template copy<T>(a, a.q, head, base + M::kQ);
  queries.template copy<T>(a, a.g, head, base + M::kG);
#pragma unroll
  for (int t = 0; t < S - 1; ++t) {
    if (first_key + t * N < end_key) {
      ahead[t].template copy<T>(a, a.k, kv, base + M::kK + t * M::kTile);
      ahead[t].template copy<T>(a, a.v, kv, base + M::kV + t * M::kTile);
    }
    commit_copies();
  }
  loader.look_up(a, first_key + (S - 1) * N, end_key);
  if (any_flag(a, a.bad_k, kv, first_key, end_key)) {  // looked at while the first rows are on their way
    wait_copies<0>();
    plain_query_gradient<T>(a, pos0, kBlock, head);
    return;
  }

  const int row0 = warp * 16, i0 = pos0 + row0 + (lane >> 2), i1 = i0 + 8;
  const Bounds see0 = keys_of(a, i0), see1 = keys_of(a, i1);
  const int warp_begin = keys_of(a, pos0 + row0).begin, warp_last = min(last, pos0 + row0 + 15);
  const int warp_end = pos0 + row0 <= last ? keys_of(a, warp_last).end : 0;
  const float slope = MODE != kPlain ? slope_of(a, head) : 0.f;
  const int64_t place = int64_t(head) * a.n;
  const float lse0 = i0 < a.n ? a.lse[place + i0] : 0.f, lse1 = i1 < a.n ? a.lse[place + i1] : 0.f;
  int lift0 = 0, lift1 = 0;
  if constexpr (kShortRange<T>) {
    lift0 = query_lift(a, head, kv, i0);
    lift1 = query_lift(a, head, kv, i1);
  }
  const float up0 = power_of_two(lift0), up1 = power_of_two(lift1), scale0 = a.scale * up0, scale1 = a.scale * up1;
  const float delta0 = i0 < a.n ? a.delta[place + i0] * up0 : 0.f, delta1 = i1 < a.n ? a.delta[place + i1] * up1 : 0.f;

  float gq[DP / 8][4] = {};
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
      float s[NT][4] = {}, dp[NT][4] = {};
      product_rows<T, DP, NT>(s, base + M::kQ, row0, base + M::kK + stage * M::kTile);
      product_rows<T, DP, NT>(dp, base + M::kG, row0, base + M::kV + stage * M::kTile);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = j0 + t * 8 + (lane & 3) * 2 + e;
          const Score x0 = score_of<MODE>(a, s[t][e], slope, float(i0 - j)), x1 = score_of<MODE>(a, s[t][2 + e], slope, float(i1 - j));
          const float d0 = exp2_fast(x0.x - lse0) * fmaf(dp[t][e], scale0, -delta0) * x0.slope;
          const float d1 = exp2_fast(x1.x - lse1) * fmaf(dp[t][2 + e], scale1, -delta1) * x1.slope;
          dp[t][e] = see0.holds(j) ? d0 : 0.f;
          dp[t][2 + e] = see1.holds(j) ? d1 : 0.f;
        }
      }
      product_probabilities<T, DP, NT, true>(gq, dp, base + M::kK + stage * M::kTile);
    }
    stage = stage + 1 == S ? 0 : stage + 1;
  }
  wait_copies<0>();
  __syncwarp();
  store_rows<T, DP>(a, a.gq, head, pos0 + row0, gq, power_of_two(-lift0), power_of_two(-lift1), smem + M::kQ, row0);
}

// Queries per step of the key kernel: 32 for the widest rows, whose two accumulators of 64 registers
// leave no room for more.
template <int DP>
struct KeyMemory {
  static constexpr int kRows = DP == 128 ? 32 : 64;
  static constexpr int kTile = kBlock * DP * 2, kStep = kRows * DP * 2;
  static constexpr int kStages = DP <= 32 ? 4 : 2;  // of queries and gradients
  static constexpr int kK = 0, kV = kTile, kQ = 2 * kTile, kG = kQ + kStages * kStep;
  static constexpr int kLse = kG + kStages * kStep, kDelta = kLse + kStages * kRows * 4;
  static constexpr int kBytes = kDelta + kStages * kRows * 4;
};

template <typename T, int DP, int MODE>
__global__ void __launch_bounds__(kThreads, DP <= 32 ? 4 : 1) key_gradients_kernel(const __grid_constant__ Problem a) {
  extern __shared__ __align__(128) unsigned char smem[];
  using M = KeyMemory<DP>;
  constexpr int R = M::kRows, NT = R / 8;
  const int kv = blockIdx.y, group = a.heads / a.kv_heads;
  const int pos0 = blockIdx.x * kBlock, last = min(a.n, pos0 + kBlock) - 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first_query = queries_of(a, pos0).begin, end_query = queries_of(a, last).end;
  const uint32_t base = smem_u32(smem);
  {
    Loader<DP, kBlock> keys;
    keys.look_up(a, pos0, last + 1);
    keys.template copy<T>(a, a.k, kv, base + M::kK);
    keys.template copy<T>(a, a.v, kv, base + M::kV);
  }
  float* s_lse = reinterpret_cast<float*>(smem + M::kLse);
  float* s_delta = reinterpret_cast<float*>(smem + M::kDelta);
  constexpr int S = M::kStages;
  auto fetch = [&](const Loader<DP, R>& rows, int head, int q0, int stage) {
    rows.template copy<T>(a, a.q, head, base + M::kQ + stage * M::kStep);
    rows.template copy<T>(a, a.g, head, base + M::kG + stage * M::kStep);
    for (int r = threadIdx.x; r < R; r += kThreads) {
      const bool real = q0 + r < end_query;
      const int64_t at = int64_t(head) * a.n + (real ? q0 + r : 0);
      copy4(smem_u32(s_lse + stage * R + r), a.lse + at, real ? 4 : 0);
      copy4(smem_u32(s_delta + stage * R + r), a.delta + at, real ? 4 : 0);
    }
  };
  const int steps = (end_query - first_query + R - 1) / R, total = steps * group;
  // the steps of the first head, then of the next: what is fetched next, and its rows, looked up a step ahead
  int fetch_step = 0, fetch_head = kv * group;
  auto advance = [&] {
    if (++fetch_step == steps) {
      fetch_step = 0;
      ++fetch_head;
    }
  };
  Loader<DP, R> ahead[S - 1], loader;
#pragma unroll
  for (int t = 0; t < S - 1; ++t) ahead[t].look_up(a, first_query + (steps > 0 ? t % steps : 0) * R, end_query);
#pragma unroll
  for (int t = 0; t < S - 1; ++t) {
    if (t < total) {
      fetch(ahead[t], fetch_head, first_query + fetch_step * R, t);
      advance();
    }
    commit_copies();
  }
  loader.look_up(a, first_query + fetch_step * R, end_query);
  bool bad = false;  // looked at while the first rows are on their way
  for (int h = kv * group; h < (kv + 1) * group; ++h) bad |= any_flag(a, a.bad_q, h, first_query, end_query);
  if (bad) {
    wait_copies<0>();
    plain_key_gradients<T>(a, pos0, kBlock, kv);
    return;
  }

  const int row0 = warp * 16, j0 = pos0 + row0 + (lane >> 2), j1 = j0 + 8;
  const Bounds seen0 = queries_of(a, j0), seen1 = queries_of(a, j1);
  const int warp_begin = pos0 + row0 <= last ? queries_of(a, pos0 + row0).begin : INT_MAX;
  const int warp_end = pos0 + row0 <= last ? queries_of(a, min(last, pos0 + row0 + 15)).end : 0;

  constexpr float kLift = kLifted<T, kGradientWeights>;
  int lift0 = 0, lift1 = 0;
  float up0 = 1.f, up1 = 1.f;  // of the gradients of scores, whose probabilities are lifted already
  if constexpr (kShortRange<T>) {
    lift0 = key_lift(a, kv, j0);
    lift1 = key_lift(a, kv, j1);
    up0 = power_of_two(lift0 - kGradientWeights);
    up1 = power_of_two(lift1 - kGradientWeights);
  }
  float gk[DP / 8][4] = {}, gv[DP / 8][4] = {};
  int stage = 0, head = kv * group, step = 0;
  for (int it = 0; it < total; ++it) {
    const int q0 = first_query + step * R;
    wait_copies<S - 2>();
    __syncthreads();  // this step's rows are there, and the stage of the last one is free
    if (it + S - 1 < total) {
      fetch(loader, fetch_head, first_query + fetch_step * R, stage == 0 ? S - 1 : stage - 1);
      advance();
    }
    commit_copies();
    loader.look_up(a, first_query + fetch_step * R, end_query);
    if (q0 + R > warp_begin && q0 < warp_end) {
      const float slope = MODE != kPlain ? slope_of(a, head) : 0.f;
      const uint32_t tq = base + M::kQ + stage * M::kStep, tg = base + M::kG + stage * M::kStep;
      float p[NT][4] = {}, ds[NT][4] = {};
      product_rows<T, DP, NT>(p, base + M::kK, row0, tq);
      product_rows<T, DP, NT>(ds, base + M::kV, row0, tg);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = t * 8 + (lane & 3) * 2 + e, i = q0 + r;
          const float lse = s_lse[stage * R + r] - kLift, delta = s_delta[stage * R + r];
          const Score x0 = score_of<MODE>(a, p[t][e], slope, float(i - j0)), x1 = score_of<MODE>(a, p[t][2 + e], slope, float(i - j1));
          const bool on0 = seen0.holds(i), on1 = seen1.holds(i);
          p[t][e] = on0 ? exp2_fast(x0.x - lse) : 0.f;
          p[t][2 + e] = on1 ? exp2_fast(x1.x - lse) : 0.f;
          ds[t][e] = on0 ? p[t][e] * fmaf(ds[t][e], a.scale, -delta) * x0.slope * up0 : 0.f;
          ds[t][2 + e] = on1 ? p[t][2 + e] * fmaf(ds[t][2 + e], a.scale, -delta) * x1.slope * up1 : 0.f;
        }
      }
      product_probabilities<T, DP, NT>(gv, p, tg);
      product_probabilities<T, DP, NT, true>(gk, ds, tq);
    }
    stage = stage + 1 == S ? 0 : stage + 1;
    if (++step == steps) {
      step = 0;
      ++head;
    }
  }
  wait_copies<0>();
  __syncthreads();  // the key tiles are written over below, by warps that read only their own rows of them
  constexpr float kUnlift = kShortRange<T> ? 1.f / (1 << kGradientWeights) : 1.f;
  store_rows<T, DP>(a, a.gk, kv, pos0 + row0, gk, power_of_two(-lift0), power_of_two(-lift1), smem + M::kK, row0);
  store_rows<T, DP>(a, a.gv, kv, pos0 + row0, gv, kUnlift, kUnlift, smem + M::kV, row0);
}

template <typename K>
int prepare_kernel(K kernel, int bytes, const char* what) {
  if (bytes <= 48 * 1024) return TEXB_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  return e == cudaSuccess ? TEXB_OK : fail(TEXB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

template <typename T, int DP, int MODE>
int launch_backward(const Problem& a, cudaStream_t stream) {
  const unsigned tiles = unsigned((a.n + kBlock - 1) / kBlock);
  auto queries = query_gradient_kernel<T, DP, MODE>;
  auto keys = key_gradients_kernel<T, DP, MODE>;
  int st = prepare_kernel(queries, QueryMemory<DP>::kBytes, "attention query_gradient_kernel");
  if (st == TEXB_OK) st = prepare_kernel(keys, KeyMemory<DP>::kBytes, "attention key_gradients_kernel");
  if (st != TEXB_OK) return st;
  if (a.gq.p) {
    queries<<<dim3(tiles, unsigned(a.heads)), kThreads, QueryMemory<DP>::kBytes, stream>>>(a);
    st = check_launch("attention query_gradient_kernel");
  }
  if (st != TEXB_OK || !a.gk.p) return st;
  keys<<<dim3(tiles, unsigned(a.kv_heads)), kThreads, KeyMemory<DP>::kBytes, stream>>>(a);
  return check_launch("attention key_gradients_kernel");
}

template <int DP>
int backward_by_type(const Problem& a, int dtype, int mode, cudaStream_t stream) {
  const bool bf16 = dtype == TEXB_BFLOAT16;
  if (mode == kCapped) return bf16 ? launch_backward<__nv_bfloat16, DP, kCapped>(a, stream) : launch_backward<__half, DP, kCapped>(a, stream);
  if (mode == kBiased) return bf16 ? launch_backward<__nv_bfloat16, DP, kBiased>(a, stream) : launch_backward<__half, DP, kBiased>(a, stream);
  return bf16 ? launch_backward<__nv_bfloat16, DP, kPlain>(a, stream) : launch_backward<__half, DP, kPlain>(a, stream);
}

}  // namespace attention
}  // namespace texb
