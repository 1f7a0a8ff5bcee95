// Forward kernel of the attention within segments for long segments, on the 5th-generation tensor cores.
//
// A CTA owns 256 query positions of one head, as two tiles of 128, and walks the keys they see in tiles of 64.
// Scores and outputs live in tensor memory (two buffers of 64 columns of scores and DP columns of outputs for each
// query tile), queries, keys and values in shared memory (keys and values in four stages each).  Sixteen warps:
//   0-3, 4-7 : softmax of query tile 0 and 1, one row per thread.  A thread reads its row of scores, and
//              writes its probabilities over them in 16 bits, where the second product takes them from;
//   8-11     : copies of rows into shared memory: rows that lie in segment order by the copy engine, a tile
//              of 64 columns at a time (one thread); rows that come through the plan's permutation 16 bytes at a
//              time, by all four warps;
//   12, 13   : one thread each issues the products of query tile 0 and 1.
// While the softmax works on one buffer of scores, the products of the other one run (with one buffer of 128 columns
// per query tile the softmax waited 1600 of every 4300 cycles for the products between two of its tiles).
// The outputs are rescaled only when a row's maximum has grown by more than 2^8 (the sums carry the stale
// maximum until then: probabilities up to 2^8 lose nothing in fp32 sums), which is rare after the first tiles; the
// technique is a published one.
// Bound: products and exponentials together.  For 128 x 128 scores of 128 columns the products take some 1280 cycles of
// an SM (768 for the scores, in tiles of 64 columns at three quarters of the full rate, 512 for the outputs), the
// exponentials 1024.  Measured: 32 768 rows, 8 heads of 128, up to 4096 keys, causal, 208 us on the same inputs again
// and again, 229 on new ones (a floor of 105 for the products alone); over the launch the tensor pipe is 46 % busy and
// the special function pipe 50 %.
#pragma once

#include "attention_long.cuh"

namespace texb {
namespace attention {

constexpr float kStale = 8.f;  // growth of a row's maximum, in units of log2, that is left unscaled
// Scores, in the same units, beyond which a query tile is computed again by the plain loops.  `top` is a rounded product,
// and one rounding of s unit - top leaves what that took from it: all weights of a row have it in common, but it is half
// a step of the score, 1 at 2^24 and 64 at 2^30, and takes the lifted weights out of fp16, or those of bf16 out of fp32.
// (A second rounding in the loop for such scores, behind a branch, took 216 us instead of 206 for all others.)
template <typename T> constexpr float kLargeScore = kShortRange<T> ? 16777216.f : 1073741824.f;

template <int DP>
struct LongForwardMemory {
  static constexpr int kKeys = 64, kStages = 4;
  static constexpr int kTile = kLongTile * DP * 2, kStage = kKeys * DP * 2;
  static constexpr int kQ = 0, kK = 2 * kTile, kV = kK + kStages * kStage;
  static constexpr int kBarriers = kV + kStages * kStage;
  static constexpr int kBytes = kBarriers + 256 + 1024;  // and room to align the start to 1024 bytes
  static constexpr int kScores = 0, kOut = 4 * kKeys, kColumns = 512;  // tensor memory
};

struct LongRange {  // of a query tile: the tiles of keys that some row sees, and those that all rows see
  int begin, end, all_begin, all_end;
};
__device__ __forceinline__ LongRange range_of(const Problem& a, int pos0) {
  if (pos0 >= a.n) return {INT_MAX, 0, INT_MAX, 0};
  const int last = min(a.n, pos0 + kLongTile) - 1;
  const Bounds f = keys_of(a, pos0), l = keys_of(a, last);
  return {f.begin, l.end, l.begin, f.end};
}

template <typename T, int DP, int MODE>
__global__ void __launch_bounds__(kLongThreads, 1)
long_forward_kernel(const __grid_constant__ Problem a, const __grid_constant__ Maps maps) {
  extern __shared__ unsigned char raw[];
  using M = LongForwardMemory<DP>;
  constexpr int N = M::kKeys, S = M::kStages;
  unsigned char* smem = raw + ((1024 - (t5::smem_u32(raw) & 1023)) & 1023);
  __shared__ uint32_t s_tmem;
  __shared__ int s_dead, s_large;
  const uint32_t base = t5::smem_u32(smem);
  auto bar = [&](int i) { return base + M::kBarriers + i * 8; };
  // barriers by stage: keys full, keys empty, values full, values empty; by query tile and buffer: scores full,
  // probabilities full, outputs done
  enum { kQueries = 0, kKeysFull = 1, kKeysEmpty = kKeysFull + S, kValuesFull = kKeysEmpty + S, kValuesEmpty = kValuesFull + S,
         kScoresFull = kValuesEmpty + S, kWeightsFull = kScoresFull + 4, kDone = kWeightsFull + 4, kSettle = kDone + 4 };
  static_assert((kSettle + 2) * 8 <= 256, "room for the barriers");
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform, and known to be
  if (threadIdx.x == 0) {
    s_dead = s_large = 0;
    const int copiers = maps.used ? 1 : 4;
    t5::barrier_init(bar(kQueries), copiers);
    for (int s = 0; s < S; ++s) {
      t5::barrier_init(bar(kKeysFull + s), copiers);
      t5::barrier_init(bar(kKeysEmpty + s), 2);
      t5::barrier_init(bar(kValuesFull + s), copiers);
      t5::barrier_init(bar(kValuesEmpty + s), 2);
    }
    for (int s = 0; s < 4; ++s) {
      t5::barrier_init(bar(kScoresFull + s), 1);
      t5::barrier_init(bar(kWeightsFull + s), 4);
      t5::barrier_init(bar(kDone + s), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) t5::tmem_alloc(t5::smem_u32(&s_tmem), M::kColumns);
  // the heads of a tile side by side, since they share keys and values; the longest tiles first
  const int head = blockIdx.x % a.heads, kv = head / (a.heads / a.kv_heads);
  const int pos0 = __ldg(a.query_order + blockIdx.x / a.heads) * kLongRows;
  const LongRange range[2] = {range_of(a, pos0), range_of(a, pos0 + kLongTile)};
  const int first_key = range[0].begin, end_key = max(range[0].end, range[1].end);
  const int tiles = max(0, (end_key - first_key + N - 1) / N);
  t5::fence_before_sync();
  __syncthreads();
  t5::fence_after_sync();
  volatile int* dead = &s_dead;

  // Rows in segment order are fetched by the copy engine: item 0 queries and keys of tile 0, item 2 j + 1 values of
  // tile j, item 2 j keys of tile j.  The first of them before anything else.
  const int items = 2 * tiles, early = min(items, 2 * S);
  auto fetch = [&](int item) {
    const int j = item >> 1, stage = j % S, pos = first_key + j * N, full = (item & 1 ? kValuesFull : kKeysFull) + stage;
    auto box = [&](const CUtensorMap& map, uint32_t to, int rows, int arrival, int h, int p) {
#pragma unroll
      for (int b = 0; b < DP / 64; ++b) t5::copy_box(to + b * (rows * 128), &map, bar(arrival), b * 64, h, p);
    };
    if (item == 0) {
      t5::barrier_arrive_expect(bar(kQueries), 2 * M::kTile);
      for (int t = 0; t < 2; ++t) box(maps.q, base + M::kQ + t * M::kTile, kLongTile, kQueries, head, pos0 + t * kLongTile);
    }
    t5::barrier_arrive_expect(bar(full), M::kStage);
    if (item & 1) box(maps.v, base + M::kV + stage * M::kStage, N, full, kv, pos);
    else box(maps.k, base + M::kK + stage * M::kStage, N, full, kv, pos);
  };
  if (maps.used && warp == 8 && t5::elect_one())
    for (int item = 0; item < early; ++item) fetch(item);
  // boxes are copied whole: the last one may hold rows behind the last key, which must be finite as well
  if (any_flag(a, a.bad_v, kv, first_key, tiles > 0 ? min(a.n, first_key + tiles * N) : first_key) || tiles == 0) {
    if (maps.used && warp == 8 && t5::elect_one() && tiles > 0) {  // nothing may be under way when this memory is given up
      t5::barrier_wait(bar(kQueries), 0, dead);
      for (int item = 0; item < early; ++item) t5::barrier_wait(bar((item & 1 ? kValuesFull : kKeysFull) + (item >> 1)), 0, dead);
    }
    __syncthreads();
    if (warp == 12) t5::tmem_free(__shfl_sync(0xffffffffu, s_tmem, 0), M::kColumns);
    if (tiles > 0) plain_forward<T>(a, pos0, kLongRows, head);  // (no tiles: a plan without the row itself in its segment)
    return;
  }
  const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
  // This warp's query tile, and the tiles of keys that some row of it sees: from `from` on, before `until`.  In
  // registers: looked up by an index in the loops below they took 400 cycles of every 2000.
  const int w = warp < 8 ? warp >> 2 : warp & 1;
  const LongRange mine = w ? range[1] : range[0];
  const int from_tile = mine.end > mine.begin ? (mine.begin - first_key) / N : 0;
  const int until_tile = mine.end > mine.begin ? (mine.end - first_key + N - 1) / N : 0;

  if (warp < 8) {  // ---- softmax
    const int row = threadIdx.x & 127, i = pos0 + w * kLongTile + row;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t sums = tmem + lanes + M::kOut + w * DP;
    const Bounds see = keys_of(a, i);
    constexpr float kLift = kLifted<T, 7>;  // the largest probability is 2^kStale
    const float unit = a.unit, slope = MODE != kPlain ? slope_of(a, head) : 0.f;
    float top = -INFINITY;  // in units of log2
    float2 sum = {0.f, 0.f};
    int done = 0;           // tiles of this query tile so far
    for (int j = from_tile; j < until_tile; ++j) {
      const int buffer = 2 * w + (done & 1);
      const uint32_t scores = tmem + lanes + M::kScores + buffer * N;
      t5::warp_wait(bar(kScoresFull + buffer), (done >> 1) & 1, dead);
      float s[N];
#pragma unroll
      for (int c = 0; c < N; c += 32) t5::tmem_load32(scores + c, reinterpret_cast<float(&)[32]>(s[c]));
      t5::tmem_wait_loads();
      const int j0 = first_key + j * N;
      if constexpr (MODE != kPlain) {
#pragma unroll
        for (int c = 0; c < N; ++c) s[c] = score_of<MODE>(a, s[c], slope, float(i - j0) - float(c)).x;
      }
      if (!(j0 >= mine.all_begin && j0 + N <= mine.all_end)) {
        const unsigned from = unsigned(see.begin - j0), count = unsigned(see.end - see.begin);
#pragma unroll
        for (int c = 0; c < N; ++c) s[c] = unsigned(c) - from < count ? s[c] : -INFINITY;
      }
      float most[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int c = 4; c + 1 < N; c += 2) most[(c >> 1) & 3] = t5::max3(most[(c >> 1) & 3], s[c], s[c + 1]);
      float now = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
      if constexpr (MODE == kPlain) now *= unit;  // the scale is positive here
      if (done == 0) {
        top = now;
      } else if (__any_sync(0xffffffffu, now > top + kStale)) {
        // rescale this warp's rows: the product that last added to them must be done
        const int last = done - 1;
        t5::warp_wait(bar(kDone + 2 * w + (last & 1)), (last >> 1) & 1, dead);
        const float next = fmaxf(top, now);
        const float shrink = next == -INFINITY ? 1.f : exp2_fast(top - next);
        top = next;
        sum.x *= shrink;
        sum.y *= shrink;
#pragma unroll
        for (int c = 0; c < DP; c += 16) {
          float o[16];
          t5::tmem_load16(sums + c, o);
          t5::tmem_wait_loads();
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] *= shrink;
          t5::tmem_store16(sums + c, reinterpret_cast<const uint32_t*>(o));
        }
      }
      const float less = (top == -INFINITY ? 0.f : top) - kLift;  // a row without a visible key so far: weights 0, not NaN
      const float2 factor = {MODE != kPlain ? 1.f : unit, MODE != kPlain ? 1.f : unit}, shift = {-less, -less};
      float2 part[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
      for (int c = 0; c < N; c += 32) {
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 x = t5::fma2({s[c + e], s[c + e + 1]}, factor, shift);
          const float2 y = {exp2_fast(x.x), exp2_fast(x.y)};
          part[(e >> 1) & 1] = t5::add2(part[(e >> 1) & 1], y);
          p[e / 2] = pack_lifted<T>(y.x, y.y);
        }
        t5::tmem_store16(scores + c / 2, p);
      }
      sum = t5::add2(sum, t5::add2(part[0], part[1]));
      t5::tmem_wait_stores();
      t5::fence_before_sync();
      t5::warp_arrive(bar(kWeightsFull + buffer));
      ++done;
    }
    if (done > 0) {
      const int last = done - 1;  // products are done in order: the last one means all
      t5::warp_wait(bar(kDone + 2 * w + (last & 1)), (last >> 1) & 1, dead);
      const bool there = i < a.n;
      if (MODE == kPlain && fabsf(top) > kLargeScore<T> && fabsf(top) < INFINITY) s_large = 1;
      const float total = sum.x + sum.y, factor = see.end > see.begin ? 1.f / total : 0.f;
      if (there && a.lse) a.lse[int64_t(head) * a.n + i] = see.end > see.begin ? top - kLift + log2f(total) : 0.f;
      T* to = row_at<T>(a, a.out, head, min(i, a.n - 1));
      T* low = a.out_low.p ? row_at<T>(a, a.out_low, head, min(i, a.n - 1)) : nullptr;
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        float o[32];
        t5::tmem_load32(sums + c, o);
        t5::tmem_wait_loads();
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (there && c + e < a.dim) {
            Chunk<T, 16> high, rest;
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const float y = o[e + x] * factor;
              high.v[x] = narrow<T>(y);
              rest.v[x] = narrow<T>(y - widen<T>(high.v[x]));
            }
            store_chunk<T, 16>(to + c + e, high);
            if (low) store_chunk<T, 16>(low + c + e, rest);
          }
        }
      }
    }
  } else if (warp < 12) {  // ---- copies: queries and the first keys, then values and keys in turn
    auto announce = [&](int item) {
      t5::fence_copies();
      if (item == 0) t5::warp_arrive(bar(kQueries));
      t5::warp_arrive(bar((item & 1 ? kValuesFull : kKeysFull) + (item >> 1) % S));
    };
    if (maps.used && warp == 8 && t5::elect_one()) {
      for (int item = early; item < items; ++item) {
        const int j = item >> 1;
        t5::barrier_wait(bar((item & 1 ? kValuesEmpty : kKeysEmpty) + j % S), (j / S - 1) & 1, dead);
        fetch(item);
      }
    }
    constexpr int kLag = 4;  // items under way
    for (int item = maps.used ? items : 0; item < items; ++item) {
      const int j = item >> 1, stage = j % S, pos = first_key + j * N;
      if (j >= S) t5::warp_wait(bar((item & 1 ? kValuesEmpty : kKeysEmpty) + stage), (j / S - 1) & 1, dead);
      if (item == 0) {
        for (int t = 0; t < 2; ++t) copy_long_tile<T, DP, kLongTile>(a, a.q, head, pos0 + t * kLongTile, a.n, base + M::kQ + t * M::kTile);
      }
      if (item & 1) copy_long_tile<T, DP, N>(a, a.v, kv, pos, end_key, base + M::kV + stage * M::kStage);
      else copy_long_tile<T, DP, N>(a, a.k, kv, pos, end_key, base + M::kK + stage * M::kStage);
      commit_copies();
      if (item >= kLag) {
        wait_copies<kLag>();
        announce(item - kLag);
      }
    }
    if (!maps.used) {
      wait_copies<0>();
      for (int late = max(0, items - kLag); late < items; ++late) announce(late);
    }
  } else {
    if (warp < 14 && t5::elect_one()) {  // ---- products
      constexpr uint32_t score_instr = t5::instruction<T>(128, N, false), out_instr = t5::instruction<T>(128, DP, true);
      const uint32_t sums = tmem + M::kOut + w * DP;
      int scored = 0, done = 0;
      auto buffer_of = [&](int count) { return tmem + M::kScores + (2 * w + (count & 1)) * N; };
      // Scores of tile j.  The keys' stage is given back in any case, if it is filled again: nothing may arrive at
      // a barrier that nobody waits for any more.
      auto score = [&](int j) {
        t5::barrier_wait(bar(kKeysFull + j % S), (j / S) & 1, dead);
        t5::fence_after_sync();
        if (j >= from_tile && j < until_tile) {
          t5::multiply_columns<DP>(buffer_of(scored), base + M::kQ + w * M::kTile, kLongTile, base + M::kK + (j % S) * M::kStage, N, score_instr);
          t5::commit(bar(kScoresFull + 2 * w + (scored & 1)));
          ++scored;
        }
        if (j + S < tiles) t5::commit(bar(kKeysEmpty + j % S));
      };
      t5::barrier_wait(bar(kQueries), 0, dead);
      for (int j = 0; j < min(2, tiles); ++j) score(j);
      for (int j = 0; j < tiles; ++j) {
        t5::barrier_wait(bar(kValuesFull + j % S), (j / S) & 1, dead);
        if (j >= from_tile && j < until_tile) {
          t5::barrier_wait(bar(kWeightsFull + 2 * w + (done & 1)), (done >> 1) & 1, dead);
          t5::fence_after_sync();
          t5::multiply_rows<N>(sums, buffer_of(done), base + M::kV + (j % S) * M::kStage, out_instr, done > 0);
          t5::commit(bar(kDone + 2 * w + (done & 1)));
          ++done;
        }
        if (j + S < tiles) t5::commit(bar(kValuesEmpty + j % S));
        // products of one thread are done in the order of their issue: the scores may overwrite the probabilities
        if (j + 2 < tiles) score(j + 2);
      }
    }
  }
  // All products and copies have been waited for, except after a wait that gave up: then what is still under
  // way must end within the memory that this CTA holds.
  t5::fence_before_sync();
  __syncthreads();
  if (s_dead) t5::settle(bar(kSettle + (warp & 1)), (warp == 12 || warp == 13) && t5::elect_one(), &g_wait_timeouts);
  __syncthreads();
  t5::fence_after_sync();
  if (warp == 12) t5::tmem_free(tmem, M::kColumns);
  if (MODE == kPlain && s_large) plain_forward<T>(a, pos0, kLongRows, head);
}

template <typename T, int DP, int MODE>
int launch_long_forward(const Problem& a, int dtype, cudaStream_t stream) {
  auto kernel = long_forward_kernel<T, DP, MODE>;
  constexpr int bytes = LongForwardMemory<DP>::kBytes;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(TEXB_ERR_CUDA, "attention long_forward_kernel: %s", cudaGetErrorString(e));
  Maps maps = {};
  constexpr int keys = LongForwardMemory<DP>::kKeys;
  maps.used = a.perm == nullptr && make_map(&maps.q, a, a.q, a.heads, kLongTile, dtype) && make_map(&maps.k, a, a.k, a.kv_heads, keys, dtype) &&
              make_map(&maps.v, a, a.v, a.kv_heads, keys, dtype);
  const int64_t grid = ceil_div(a.n, kLongRows) * a.heads;
  if (grid > INT_MAX) return fail(TEXB_ERR_UNSUPPORTED, "segment_attention: too many rows and heads");
  kernel<<<unsigned(grid), kLongThreads, bytes, stream>>>(a, maps);
  return check_launch("attention long_forward_kernel");
}

template <int DP>
int long_forward_by_type(const Problem& a, int dtype, int mode, cudaStream_t stream) {
  const bool bf16 = dtype == TEXB_BFLOAT16;
  if (mode == kCapped) return bf16 ? launch_long_forward<__nv_bfloat16, DP, kCapped>(a, dtype, stream) : launch_long_forward<__half, DP, kCapped>(a, dtype, stream);
  if (mode == kBiased) return bf16 ? launch_long_forward<__nv_bfloat16, DP, kBiased>(a, dtype, stream) : launch_long_forward<__half, DP, kBiased>(a, dtype, stream);
  return bf16 ? launch_long_forward<__nv_bfloat16, DP, kPlain>(a, dtype, stream) : launch_long_forward<__half, DP, kPlain>(a, dtype, stream);
}

// Waits that gave up in this unit's kernels since the library was loaded.
template <int DP>
int long_forward_timeouts(int* count) {
  const cudaError_t e = cudaMemcpyFromSymbol(count, g_wait_timeouts, sizeof(int));
  return e == cudaSuccess ? TEXB_OK : fail(TEXB_ERR_CUDA, "device status: %s", cudaGetErrorString(e));
}

}  // namespace attention
}  // namespace texb
