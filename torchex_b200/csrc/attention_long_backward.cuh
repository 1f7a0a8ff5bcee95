// Backward kernel of the attention within segments for long segments, on the 5th-generation tensor cores.
//
// One kernel in two forms, as the general one (attention_backward.cuh):
//   queries (KEYS false): a CTA owns 128 query positions of a head and walks the keys they see;
//   keys    (KEYS true) : a CTA owns 128 key positions of a kv head and walks the queries that see them, for all
//                         query heads that share it.
// Its own rows -- queries and gradients, or keys and values -- stay in shared memory, the rows of the other side
// ("the stream") pass through it 64 at a time, in four stages.  For a tile of the stream
//   S = own1 stream1^T,  G = own2 stream2^T,  P = exp(S - lse),  dS = P (G - delta) scale slope,
//   queries: g_q += dS K;   keys: g_v += P^T g, g_k += dS^T Q   (S and G transposed: rows are keys),
// all in tensor memory: two buffers of 64 + 64 columns for S and G, over which P and dS are written in 16 bits, and
// the sums.  In fp16 both are lifted by powers of two first (attention.cuh).  Two warpgroups take the tiles in turn,
// one row per thread; warps 8 to 11 copy rows, one thread of warp 12 issues all products, those of one buffer while the
// other one's exponentials are taken.
// Bound: matrix products.  A tile of 64 takes 390 cycles for each of S and G (an operand of 64 rows runs at three
// quarters of the rate of one of 128, for which tensor memory has no room) and 262 for each sum.
// Measured with cold caches: 8192 rows, 16 heads that share 4, of 128 columns, up to 2048 keys, causal, 118 us for the
// queries and 120 for the keys and values; the tensor pipe is 36 and 52 % busy over the launch.  With warm caches
// 104 and 105 in bf16, 106 and 109 in fp16, whose lifted gradients take a product more in the keys' form.
#pragma once

#include "attention_long.cuh"

namespace texb {
namespace attention {

template <int DP>
struct LongBackwardMemory {
  static constexpr int kRows = 64, kStages = 4;
  static constexpr int kOwn = kLongTile * DP * 2, kPart = kRows * DP * 2;
  static constexpr int kOwn1 = 0, kOwn2 = kOwn, kStream = 2 * kOwn;  // a stage: stream1, then stream2
  static constexpr int kLse = kStream + kStages * 2 * kPart;         // keys only: [stages][lse, delta][kRows]
  static constexpr int kBarriers = kLse + kStages * 2 * kRows * 4;
  static constexpr int kBytes = kBarriers + 128 + 1024;  // and room to align the start to 1024 bytes
  static constexpr int kScores = 0, kSums = 256, kColumns = 512;  // tensor memory
};

template <typename T, int DP, int MODE, bool KEYS>
__global__ void __launch_bounds__(kLongThreads, 1)
long_backward_kernel(const __grid_constant__ Problem a, const __grid_constant__ Maps maps) {
  extern __shared__ unsigned char raw[];
  using M = LongBackwardMemory<DP>;
  constexpr int N = M::kRows, S = M::kStages;
  unsigned char* smem = raw + ((1024 - (t5::smem_u32(raw) & 1023)) & 1023);
  __shared__ uint32_t s_tmem;
  __shared__ int s_dead;
  const uint32_t base = t5::smem_u32(smem);
  auto bar = [&](int i) { return base + M::kBarriers + i * 8; };
  enum { kOwnFull = 0, kFull = 1, kEmpty = kFull + S, kScoresFull = kEmpty + S, kWeightsFull = kScoresFull + 2, kDone = kWeightsFull + 2,
         kSettle = kDone + 1 };
  static_assert((kSettle + 1) * 8 <= 128, "room for the barriers");
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  if (threadIdx.x == 0) {
    s_dead = 0;
    t5::barrier_init(bar(kOwnFull), maps.used ? 1 : 4);
    for (int s = 0; s < S; ++s) {
      t5::barrier_init(bar(kFull + s), maps.used ? (KEYS ? 2 : 1) : 4);
      t5::barrier_init(bar(kEmpty + s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      t5::barrier_init(bar(kScoresFull + b), 1);
      t5::barrier_init(bar(kWeightsFull + b), 4);
    }
    t5::barrier_init(bar(kDone), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) t5::tmem_alloc(t5::smem_u32(&s_tmem), M::kColumns);
  const int group = a.heads / a.kv_heads;
  // the heads of a tile side by side, since they share rows; the longest tiles first
  const int own_heads = KEYS ? a.kv_heads : a.heads, own_head = blockIdx.x % own_heads;
  const int kv = KEYS ? own_head : own_head / group;
  const int pos0 = __ldg((KEYS ? a.key_order : a.query_order) + blockIdx.x / own_heads) * kLongTile;
  const int last = min(a.n, pos0 + kLongTile) - 1;
  auto seen_by = [&](int pos) { return KEYS ? queries_of(a, pos) : keys_of(a, pos); };
  const Bounds head_bounds = seen_by(pos0), tail_bounds = seen_by(last);
  const int first = head_bounds.begin, end = tail_bounds.end;
  // positions that all rows see: between the last beginning and the first end
  const int all_begin = tail_bounds.begin, all_end = head_bounds.end;
  const int steps = max(0, (end - first + N - 1) / N);  // tiles of one head's stream
  const int heads = KEYS ? group : 1, total = steps * heads;
  t5::fence_before_sync();
  __syncthreads();
  t5::fence_after_sync();
  volatile int* dead = &s_dead;

  // Rows in segment order are fetched by the copy engine, the CTA's own and the first of the stream before
  // anything else.
  auto stream_head = [&](int h) { return KEYS ? kv * group + h : kv; };
  auto part = [&](int stage, int which) { return base + M::kStream + (stage * 2 + which) * M::kPart; };
  auto box = [&](const CUtensorMap& map, uint32_t to, int rows, int full, int h, int pos) {
#pragma unroll
    for (int b = 0; b < DP / 64; ++b) t5::copy_box(to + b * (rows * 128), &map, bar(full), b * 64, h, pos);
  };
  auto fetch = [&](int u, int step, int head) {
    const int stage = u % S;
    t5::barrier_arrive_expect(bar(kFull + stage), 2 * M::kPart);
    box(KEYS ? maps.q : maps.k, part(stage, 0), N, kFull + stage, stream_head(head), first + step * N);
    box(KEYS ? maps.g : maps.v, part(stage, 1), N, kFull + stage, stream_head(head), first + step * N);
  };
  const int early = min(total, S);
  if (maps.used && warp == 8 && t5::elect_one() && total > 0) {
    t5::barrier_arrive_expect(bar(kOwnFull), 2 * M::kOwn);
    box(KEYS ? maps.k : maps.q, base + M::kOwn1, kLongTile, kOwnFull, own_head, pos0);
    box(KEYS ? maps.v : maps.g, base + M::kOwn2, kLongTile, kOwnFull, own_head, pos0);
    for (int u = 0; u < early; ++u) fetch(u, u % steps, u / steps);
  }
  bool bad = false;
  const int looked = steps > 0 ? min(a.n, first + steps * N) : first;  // tiles are copied whole
  if (KEYS) {
    for (int h = 0; h < heads; ++h) bad |= any_flag(a, a.bad_q, kv * group + h, first, looked);
  } else {
    bad = any_flag(a, a.bad_k, kv, first, looked);
  }
  if (bad || total == 0) {
    if (maps.used && warp == 8 && t5::elect_one() && total > 0) {  // nothing may be under way when this memory is given up
      t5::barrier_wait(bar(kOwnFull), 0, dead);
      for (int u = 0; u < early; ++u) {
        if (KEYS) t5::barrier_arrive(bar(kFull + u));  // in place of lse and delta
        t5::barrier_wait(bar(kFull + u), 0, dead);
      }
    }
    __syncthreads();
    if (warp == 12) t5::tmem_free(__shfl_sync(0xffffffffu, s_tmem, 0), M::kColumns);
    if (total == 0) return;  // a plan without the row itself in its segment
    if (KEYS) plain_key_gradients<T>(a, pos0, kLongTile, kv);
    else plain_query_gradient<T>(a, pos0, kLongTile, own_head);
    return;
  }
  const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
  const float* s_lse = reinterpret_cast<const float*>(smem + M::kLse);

  if (warp < 8) {  // ---- probabilities and gradients of scores
    const int buffer = warp >> 2, row = threadIdx.x & 127, pos = pos0 + row;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t scores = tmem + lanes + M::kScores + buffer * 2 * N, products = scores + N;
    const Bounds see = seen_by(pos);
    float row_lse = 0.f, row_delta = 0.f;
    if (!KEYS && pos < a.n) {
      row_lse = a.lse[int64_t(own_head) * a.n + pos];
      row_delta = a.delta[int64_t(own_head) * a.n + pos];
    }
    // fp16: the row's factors.  The probabilities of the keys' form are lifted, and so are the gradients that they enter.
    constexpr float kLift = KEYS ? kLifted<T, kGradientWeights> : 0.f;
    int lift = 0;
    float2 up = {1.f, 1.f};
    if constexpr (kShortRange<T>) {
      lift = KEYS ? key_lift(a, kv, pos) : query_lift(a, own_head, kv, pos);
      up.x = up.y = power_of_two(lift - (KEYS ? kGradientWeights : 0));
      if (!KEYS) row_delta *= up.x;
    }
    const float own_scale = KEYS ? a.scale : a.scale * up.x;
    const float2 unit = {a.unit, a.unit}, scale = {own_scale, own_scale};
    int step = buffer, head = 0;  // of tile u = buffer, buffer + 2, ...
    while (step >= steps) {
      step -= steps;
      ++head;
    }
    for (int u = buffer; u < total; u += 2) {
      const int p0 = first + step * N, stage = u % S;
      const float slope = MODE != kPlain ? slope_of(a, KEYS ? kv * group + head : own_head) : 0.f;
      if (KEYS) t5::warp_wait(bar(kFull + stage), (u / S) & 1, dead);  // lse and delta of the tile's queries
      t5::warp_wait(bar(kScoresFull + buffer), (u >> 1) & 1, dead);
      const float* lse = s_lse + stage * 2 * N;
      const float* delta = lse + N;
      const bool whole = p0 >= all_begin && p0 + N <= all_end;
      const unsigned from = unsigned(see.begin - p0), count = unsigned(see.end - see.begin);
#pragma unroll
      for (int c = 0; c < N; c += 32) {
        float s[32], g[32];
        uint32_t p16[16], d16[16];
        t5::tmem_load32(scores + c, s);
        t5::tmem_load32(products + c, g);
        t5::tmem_wait_loads();
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          float4 l4, d4;
          if (KEYS) {
            l4 = *reinterpret_cast<const float4*>(lse + c + e);
            d4 = *reinterpret_cast<const float4*>(delta + c + e);
          } else {
            l4 = {row_lse, row_lse, row_lse, row_lse};
            d4 = {row_delta, row_delta, row_delta, row_delta};
          }
#pragma unroll
          for (int h = 0; h < 4; h += 2) {
            const int k = e + h;
            const float2 l = h ? float2{l4.z, l4.w} : float2{l4.x, l4.y}, d = h ? float2{d4.z, d4.w} : float2{d4.x, d4.y};
            float2 x, bend = {1.f, 1.f};
            if constexpr (MODE != kPlain) {
              const float away = float(pos - p0) - float(c + k);
              const Score x0 = score_of<MODE>(a, s[k], slope, away), x1 = score_of<MODE>(a, s[k + 1], slope, away - 1.f);
              x = {x0.x - (l.x - kLift), x1.x - (l.y - kLift)};
              bend = {x0.slope, x1.slope};
            } else {
              x = t5::fma2({s[k], s[k + 1]}, unit, kLift > 0.f ? float2{kLift - l.x, kLift - l.y} : float2{-l.x, -l.y});
            }
            float2 p = {exp2_fast(x.x), exp2_fast(x.y)};
            float2 ds = t5::mul2(p, t5::fma2({g[k], g[k + 1]}, scale, {-d.x, -d.y}));
            if constexpr (MODE != kPlain) ds = t5::mul2(ds, bend);
            if constexpr (KEYS && kShortRange<T>) ds = t5::mul2(ds, up);
            if (!whole) {  // set, not multiplied: a masked pair's product may be infinite
              const bool on0 = unsigned(c + k) - from < count, on1 = unsigned(c + k + 1) - from < count;
              p = {on0 ? p.x : 0.f, on1 ? p.y : 0.f};
              ds = {on0 ? ds.x : 0.f, on1 ? ds.y : 0.f};
            }
            if (KEYS) p16[k / 2] = pack_lifted<T>(p.x, p.y);
            d16[k / 2] = pack2<T>(ds.x, ds.y);
          }
        }
        if (KEYS) t5::tmem_store16(scores + c / 2, p16);
        t5::tmem_store16(products + c / 2, d16);
      }
      t5::tmem_wait_stores();
      t5::fence_before_sync();
      t5::warp_arrive(bar(kWeightsFull + buffer));
      step += 2;
      while (step >= steps && head < heads) {
        step -= steps;
        ++head;
      }
    }
    // the sums: one warpgroup writes the keys' gradient, the other the values', or each half of the queries'
    t5::warp_wait(bar(kDone), 0, dead);
    // all products are done: the CTA's own rows in shared memory are free
    constexpr int kWritten = KEYS ? DP : DP / 2;
    unsigned char* rows = smem + (buffer ? M::kOwn2 : M::kOwn1) + (warp & 3) * (32 * kWritten * 2);
    const View& view = !KEYS ? a.gq : buffer ? a.gv : a.gk;
    store_sums<T, kWritten>(a, view, own_head, pos0 + (warp & 3) * 32, tmem + lanes + M::kSums + (KEYS ? buffer * DP : 0),
                            KEYS ? 0 : buffer * kWritten, power_of_two(KEYS && buffer ? -kGradientWeights : -lift), rows);
  } else if (warp < 12) {  // ---- copies
    const View &own1 = KEYS ? a.k : a.q, &own2 = KEYS ? a.v : a.g, &stream1 = KEYS ? a.q : a.k, &stream2 = KEYS ? a.g : a.v;
    if (maps.used) {
      if (warp == 8 && t5::elect_one()) {
        int step = early % steps, head = early / steps;
        for (int u = early; u < total; ++u) {
          t5::barrier_wait(bar(kEmpty + u % S), (u / S - 1) & 1, dead);
          fetch(u, step, head);
          if (++step == steps) {
            step = 0;
            ++head;
          }
        }
      } else if (KEYS && warp == 9) {  // lse and delta of the stream's queries
        const int lane = threadIdx.x & 31;
        int step = 0, head = 0;
        for (int u = 0; u < total; ++u) {
          const int stage = u % S;
          float v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int q = first + step * N + (k & 1) * 32 + lane;
            const float* from = k < 2 ? a.lse : a.delta;
            v[k] = q < end ? __ldg(from + int64_t(kv * group + head) * a.n + q) : 0.f;
          }
          if (u >= S) t5::warp_wait(bar(kEmpty + stage), (u / S - 1) & 1, dead);
          float* to = reinterpret_cast<float*>(smem + M::kLse) + stage * 2 * N;
#pragma unroll
          for (int k = 0; k < 4; ++k) to[(k >> 1) * N + (k & 1) * 32 + lane] = v[k];
          t5::warp_arrive(bar(kFull + stage));
          if (++step == steps) {
            step = 0;
            ++head;
          }
        }
      }
    } else {
      constexpr int kLag = 2;  // tiles under way
      auto announce = [&](int u) {
        t5::fence_copies();
        if (u == 0) t5::warp_arrive(bar(kOwnFull));
        t5::warp_arrive(bar(kFull + u % S));
      };
      copy_long_tile<T, DP, kLongTile>(a, own1, own_head, pos0, a.n, base + M::kOwn1);
      copy_long_tile<T, DP, kLongTile>(a, own2, own_head, pos0, a.n, base + M::kOwn2);
      int step = 0, head = 0;
      for (int u = 0; u < total; ++u) {
        const int stage = u % S, p0 = first + step * N;
        if (u >= S) t5::warp_wait(bar(kEmpty + stage), (u / S - 1) & 1, dead);
        copy_long_tile<T, DP, N>(a, stream1, stream_head(head), p0, end, part(stage, 0));
        copy_long_tile<T, DP, N>(a, stream2, stream_head(head), p0, end, part(stage, 1));
        if (KEYS) {
          const int t = threadIdx.x & 127, q = p0 + (t & (N - 1));
          const float* from = t < N ? a.lse : a.delta;
          copy4(base + M::kLse + (stage * 2 * N + t) * 4, from + (q < end ? int64_t(kv * group + head) * a.n + q : 0), q < end ? 4 : 0);
        }
        commit_copies();
        if (u >= kLag) {
          wait_copies<kLag>();
          announce(u - kLag);
        }
        if (++step == steps) {
          step = 0;
          ++head;
        }
      }
      wait_copies<0>();
      for (int late = max(0, total - kLag); late < total; ++late) announce(late);
    }
  } else if (warp == 12 && t5::elect_one()) {  // ---- products
    constexpr uint32_t score_instr = t5::instruction<T>(128, N, false), sum_instr = t5::instruction<T>(128, DP, true);
    auto scores_of = [&](int u) { return tmem + M::kScores + (u & 1) * 2 * N; };
    auto score = [&](int u) {
      t5::barrier_wait(bar(kFull + u % S), (u / S) & 1, dead);
      t5::fence_after_sync();
      t5::multiply_columns<DP>(scores_of(u), base + M::kOwn1, kLongTile, part(u % S, 0), N, score_instr);
      t5::multiply_columns<DP>(scores_of(u) + N, base + M::kOwn2, kLongTile, part(u % S, 1), N, score_instr);
      t5::commit(bar(kScoresFull + (u & 1)));
    };
    t5::barrier_wait(bar(kOwnFull), 0, dead);
    for (int u = 0; u < min(2, total); ++u) score(u);
    for (int u = 0; u < total; ++u) {
      t5::barrier_wait(bar(kWeightsFull + (u & 1)), (u >> 1) & 1, dead);
      t5::fence_after_sync();
      if (KEYS) t5::multiply_rows<N>(tmem + M::kSums + DP, scores_of(u), part(u % S, 1), sum_instr, u > 0);
      t5::multiply_rows<N>(tmem + M::kSums, scores_of(u) + N, part(u % S, 0), sum_instr, u > 0);
      if (u + S < total) t5::commit(bar(kEmpty + u % S));  // only stages that are filled again
      if (u + 1 == total) t5::commit(bar(kDone));
      // products are done in the order of their issue: new scores may overwrite what these sums read
      if (u + 2 < total) score(u + 2);
    }
  }
  t5::fence_before_sync();
  __syncthreads();
  if (s_dead) t5::settle(bar(kSettle), warp == 12 && t5::elect_one(), &g_wait_timeouts);
  __syncthreads();
  t5::fence_after_sync();
  if (warp == 12) t5::tmem_free(tmem, M::kColumns);
}

template <typename T, int DP, int MODE, bool KEYS>
int launch_long_backward(const Problem& a, int dtype, cudaStream_t stream) {
  auto kernel = long_backward_kernel<T, DP, MODE, KEYS>;
  using M = LongBackwardMemory<DP>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, M::kBytes);
  if (e != cudaSuccess) return fail(TEXB_ERR_CUDA, "attention long_backward_kernel: %s", cudaGetErrorString(e));
  Maps maps = {};
  const int query_rows = KEYS ? M::kRows : kLongTile, key_rows = KEYS ? kLongTile : M::kRows;
  maps.used = a.perm == nullptr && make_map(&maps.q, a, a.q, a.heads, query_rows, dtype) && make_map(&maps.g, a, a.g, a.heads, query_rows, dtype) &&
              make_map(&maps.k, a, a.k, a.kv_heads, key_rows, dtype) && make_map(&maps.v, a, a.v, a.kv_heads, key_rows, dtype);
  const int64_t grid = ceil_div(a.n, kLongTile) * (KEYS ? a.kv_heads : a.heads);
  if (grid > INT_MAX) return fail(TEXB_ERR_UNSUPPORTED, "segment_attention: too many rows and heads");
  kernel<<<unsigned(grid), kLongThreads, M::kBytes, stream>>>(a, maps);
  return check_launch("attention long_backward_kernel");
}

template <typename T, int DP, int MODE>
int launch_long_backward_both(const Problem& a, int dtype, cudaStream_t stream) {
  const int st = a.gq.p ? launch_long_backward<T, DP, MODE, false>(a, dtype, stream) : TEXB_OK;
  return st == TEXB_OK && a.gk.p ? launch_long_backward<T, DP, MODE, true>(a, dtype, stream) : st;
}

template <int DP>
int long_backward_by_type(const Problem& a, int dtype, int mode, cudaStream_t stream) {
  const bool bf16 = dtype == TEXB_BFLOAT16;
  if (mode == kCapped) return bf16 ? launch_long_backward_both<__nv_bfloat16, DP, kCapped>(a, dtype, stream) : launch_long_backward_both<__half, DP, kCapped>(a, dtype, stream);
  if (mode == kBiased) return bf16 ? launch_long_backward_both<__nv_bfloat16, DP, kBiased>(a, dtype, stream) : launch_long_backward_both<__half, DP, kBiased>(a, dtype, stream);
  return bf16 ? launch_long_backward_both<__nv_bfloat16, DP, kPlain>(a, dtype, stream) : launch_long_backward_both<__half, DP, kPlain>(a, dtype, stream);
}

// Waits that gave up in this unit's kernels since the library was loaded.
template <int DP>
int long_backward_timeouts(int* count) {
  const cudaError_t e = cudaMemcpyFromSymbol(count, g_wait_timeouts, sizeof(int));
  return e == cudaSuccess ? TEXB_OK : fail(TEXB_ERR_CUDA, "device status: %s", cudaGetErrorString(e));
}

}  // namespace attention
}  // namespace texb
