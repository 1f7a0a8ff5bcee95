// Forward kernel of the attention within segments for long segments, on the 5th-generation tensor cores.
//
// A CTA owns 256 query positions of one head, as two tiles of 128, and walks the keys they see in tiles of
// 128.  Scores and outputs live in tensor memory (2 x 128 columns of scores, 2 x DP of outputs), queries,
// keys and values in shared memory (keys and values in two stages each).  Sixteen warps:
//   0-3, 4-7 : softmax of query tile 0 and 1, one row per thread.  A thread reads its row of scores, and
//              writes its probabilities over them in 16 bits, where the second product takes them from;
//   8-11     : copies of rows into shared memory: rows that lie in segment order by the copy engine, a tile
//              of 64 columns by 128 rows at a time (one thread); rows that come through the plan's permutation
//              16 bytes at a time, by all four warps;
//   12, 13   : one thread each issues the products of query tile 0 and 1.  While one tile's softmax runs, the
//              other tile's products do.
// The outputs are rescaled only when a row's maximum has grown by more than 2^8 (the sums carry the stale
// maximum until then: probabilities up to 2^8 lose nothing in fp32 sums), which is rare after the first tiles.
// Bound: exponentials.  128 x 128 of them take 1024 cycles of an SM, the two products of that tile 512 at
// the tensor cores' nominal rate.
#pragma once

#include "attention_long.cuh"

namespace texb {
namespace attention {

constexpr float kStale = 8.f;  // growth of a row's maximum, in units of log2, that is left unscaled

template <int DP>
struct LongForwardMemory {
  static constexpr int kTile = kLongTile * DP * 2;
  static constexpr int kQ = 0, kK = 2 * kTile, kV = 4 * kTile;
  static constexpr int kBarriers = 6 * kTile;
  static constexpr int kBytes = kBarriers + 256 + 1024;  // and room to align the start to 1024 bytes
  static constexpr int kScores = 0, kOut = 2 * kLongTile, kColumns = 512;  // tensor memory
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

template <typename T, int DP, bool GENERAL>
__global__ void __launch_bounds__(kLongThreads, 1)
long_forward_kernel(const __grid_constant__ Problem a, const __grid_constant__ Maps maps) {
  extern __shared__ unsigned char raw[];
  using M = LongForwardMemory<DP>;
  unsigned char* smem = raw + ((1024 - (t5::smem_u32(raw) & 1023)) & 1023);
  __shared__ uint32_t s_tmem;
  __shared__ int s_dead;
  const int head = blockIdx.y, kv = head / (a.heads / a.kv_heads);
  // the last tiles of a causal segment see the most keys: begin with them
  const int pos0 = (a.causal ? gridDim.x - 1 - blockIdx.x : blockIdx.x) * kLongRows;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform, and known to be
  const LongRange range[2] = {range_of(a, pos0), range_of(a, pos0 + kLongTile)};
  const int first_key = range[0].begin, end_key = max(range[0].end, range[1].end);
  const int tiles = (end_key - first_key + kLongTile - 1) / kLongTile;
  // boxes are copied whole: the last one may hold rows behind the last key, which must be finite as well
  if (any_flag(a, a.bad_v, kv, first_key, min(a.n, first_key + tiles * kLongTile))) {
    plain_forward<T>(a, pos0, kLongRows, head);
    return;
  }
  const uint32_t base = t5::smem_u32(smem);
  auto bar = [&](int i) { return base + M::kBarriers + i * 8; };
  // barriers: 0 queries full; 1-2 keys full, 3-4 keys empty, 5-6 values full, 7-8 values empty (by stage);
  // 9-10 scores full, 11-12 probabilities full, 13-14 outputs done (by query tile)
  if (threadIdx.x == 0) {
    s_dead = 0;
    const int copiers = maps.used ? 1 : 128;
    t5::barrier_init(bar(0), copiers);
    for (int s = 0; s < 2; ++s) {
      t5::barrier_init(bar(1 + s), copiers);
      t5::barrier_init(bar(3 + s), 2);
      t5::barrier_init(bar(5 + s), copiers);
      t5::barrier_init(bar(7 + s), 2);
      t5::barrier_init(bar(9 + s), 1);
      t5::barrier_init(bar(11 + s), 128);
      t5::barrier_init(bar(13 + s), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) t5::tmem_alloc(t5::smem_u32(&s_tmem), M::kColumns);
  t5::fence_before_sync();
  __syncthreads();
  t5::fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
  volatile int* dead = &s_dead;
  auto sees = [&](int w, int j) {  // whether query tile w sees some key of tile j
    const int j0 = first_key + j * kLongTile;
    return j < tiles && j0 < range[w].end && j0 + kLongTile > range[w].begin;
  };

  if (warp < 8) {  // ---- softmax
    t5::more_registers<184>();
    const int w = warp >> 2, row = threadIdx.x & 127, i = pos0 + w * kLongTile + row;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t scores = tmem + lanes + M::kScores + w * kLongTile, sums = tmem + lanes + M::kOut + w * DP;
    const Bounds see = keys_of(a, i);
    const float unit = a.unit, slope = GENERAL ? slope_of(a, head) : 0.f;
    float top = -INFINITY, sum = 0.f;  // in units of log2
    int done = 0;                      // tiles of this query tile so far
    bool alive = true;
    for (int j = 0; j < tiles; ++j) {
      if (!sees(w, j)) continue;
      alive = __all_sync(0xffffffffu, t5::barrier_wait(bar(9 + w), done & 1, dead));
      if (!alive) break;
      t5::fence_after_sync();
      float s[kLongTile];
#pragma unroll
      for (int c = 0; c < kLongTile; c += 32) t5::tmem_load32(scores + c, reinterpret_cast<float(&)[32]>(s[c]));
      t5::tmem_wait_loads();
      const int j0 = first_key + j * kLongTile;
      if constexpr (GENERAL) {
#pragma unroll
        for (int c = 0; c < kLongTile; ++c) s[c] = score_of<true>(a, s[c], slope, float(i - j0) - float(c)).x;
      }
      if (!(j0 >= range[w].all_begin && j0 + kLongTile <= range[w].all_end && pos0 + (w + 1) * kLongTile <= a.n)) {
        const int from = see.begin - j0, to = see.end - j0;
#pragma unroll
        for (int c = 0; c < kLongTile; ++c) s[c] = c >= from && c < to ? s[c] : -INFINITY;
      }
      float most[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int c = 4; c < kLongTile; ++c) most[c & 3] = fmaxf(most[c & 3], s[c]);
      float now = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
      if constexpr (!GENERAL) now *= unit;  // the scale is positive here
      if (done == 0) {
        top = now;
      } else if (__any_sync(0xffffffffu, now > top + kStale)) {
        // rescale this warp's rows: the product that last added to them must be done
        alive = __all_sync(0xffffffffu, t5::barrier_wait(bar(13 + w), (done - 1) & 1, dead));
        if (!alive) break;
        t5::fence_after_sync();
        const float next = fmaxf(top, now);
        const float shrink = next == -INFINITY ? 1.f : exp2_fast(top - next);
        top = next;
        sum *= shrink;
#pragma unroll
        for (int c = 0; c < DP; c += 16) {  // 16 at a time: the row of scores is in registers as well
          float o[16];
          t5::tmem_load16(sums + c, o);
          t5::tmem_wait_loads();
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] *= shrink;
          t5::tmem_store16(sums + c, reinterpret_cast<const uint32_t*>(o));
        }
      }
      const float less = top == -INFINITY ? 0.f : top;  // a row without a visible key so far: weights 0, not NaN
      float part[4] = {};
#pragma unroll
      for (int c = 0; c < kLongTile; c += 32) {
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float x0 = exp2_fast(GENERAL ? s[c + e] - less : fmaf(s[c + e], unit, -less));
          const float x1 = exp2_fast(GENERAL ? s[c + e + 1] - less : fmaf(s[c + e + 1], unit, -less));
          part[e & 2] += x0;
          part[(e & 2) + 1] += x1;
          p[e / 2] = pack2<T>(x0, x1);
        }
        t5::tmem_store16(scores + c / 2, p);
      }
      sum += (part[0] + part[1]) + (part[2] + part[3]);
      t5::tmem_wait_stores();
      t5::fence_before_sync();
      t5::barrier_arrive(bar(11 + w));
      ++done;
    }
    if (done > 0 && alive) {
      alive = __all_sync(0xffffffffu, t5::barrier_wait(bar(13 + w), (done - 1) & 1, dead));
      t5::fence_after_sync();
      if (alive) {
        const bool there = i < a.n;
        const float factor = see.end > see.begin ? 1.f / sum : 0.f;
        if (there && a.lse) a.lse[int64_t(head) * a.n + i] = see.end > see.begin ? top + log2f(sum) : 0.f;
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
    }
  } else if (warp < 12) {  // ---- copies: queries and the first keys, then values and keys in turn
    t5::fewer_registers<72>();
    // item 0: queries and keys of tile 0; item 2 j + 1: values of tile j; item 2 j: keys of tile j
    auto announce = [&](int item) {
      t5::fence_copies();
      if (item == 0) t5::barrier_arrive(bar(0));
      t5::barrier_arrive(bar((item & 1 ? 5 : 1) + ((item >> 1) & 1)));
    };
    const int items = 2 * tiles;
    bool alive = true;
    if (maps.used) {
      if (warp == 8 && t5::elect_one()) {
        auto box = [&](const CUtensorMap& map, uint32_t to, int full, int h, int pos) {
#pragma unroll
          for (int b = 0; b < DP / 64; ++b) t5::copy_box(to + b * (kLongTile * 128), &map, bar(full), b * 64, h, pos);
        };
        for (int item = 0; item < items; ++item) {
          const int j = item >> 1, stage = j & 1, pos = first_key + j * kLongTile, full = (item & 1 ? 5 : 1) + stage;
          if (j >= 2 && !t5::barrier_wait(bar((item & 1 ? 7 : 3) + stage), ((j >> 1) - 1) & 1, dead)) break;
          if (item == 0) {
            t5::barrier_arrive_expect(bar(0), 2 * M::kTile);
            box(maps.q, base + M::kQ, 0, head, pos0);
            box(maps.q, base + M::kQ + M::kTile, 0, head, pos0 + kLongTile);
          }
          t5::barrier_arrive_expect(bar(full), M::kTile);
          if (item & 1) box(maps.v, base + M::kV + stage * M::kTile, full, kv, pos);
          else box(maps.k, base + M::kK + stage * M::kTile, full, kv, pos);
        }
      }
    }
    for (int item = maps.used ? items : 0; item < items; ++item) {
      const int j = item >> 1, stage = j & 1, pos = first_key + j * kLongTile;
      if (j >= 2) {
        alive = __all_sync(0xffffffffu, t5::barrier_wait(bar((item & 1 ? 7 : 3) + stage), ((j >> 1) - 1) & 1, dead));
        if (!alive) break;
      }
      if (item == 0) {
        copy_long_tile<T, DP>(a, a.q, head, pos0, a.n, base + M::kQ);
        copy_long_tile<T, DP>(a, a.q, head, pos0 + kLongTile, a.n, base + M::kQ + M::kTile);
      }
      if (item & 1) copy_long_tile<T, DP>(a, a.v, kv, pos, end_key, base + M::kV + stage * M::kTile);
      else copy_long_tile<T, DP>(a, a.k, kv, pos, end_key, base + M::kK + stage * M::kTile);
      commit_copies();
      if (item >= 2) {
        wait_copies<2>();
        announce(item - 2);
      }
    }
    if (alive && !maps.used) {
      wait_copies<0>();
      for (int late = max(0, items - 2); late < items; ++late) announce(late);
    }
    wait_copies<0>();
  } else {
    t5::fewer_registers<72>();
    if (warp < 14 && t5::elect_one()) {  // ---- products
      constexpr uint32_t score_instr = t5::instruction<T>(128, kLongTile, false), out_instr = t5::instruction<T>(128, DP, true);
      const int w = warp - 12;
      const uint32_t scores = tmem + M::kScores + w * kLongTile, sums = tmem + M::kOut + w * DP;
      int done = 0;
      // Scores of tile j.  Either way the keys' stage is given back, if it is filled again: nothing may arrive at
      // a barrier that nobody waits for any more.
      auto score = [&](int j) {
        if (!t5::barrier_wait(bar(1 + (j & 1)), (j >> 1) & 1, dead)) return false;
        t5::fence_after_sync();
        if (sees(w, j)) {
          t5::multiply_columns<DP>(scores, base + M::kQ + w * M::kTile, kLongTile, base + M::kK + (j & 1) * M::kTile, kLongTile, score_instr);
          t5::commit(bar(9 + w));
        }
        if (j + 2 < tiles) t5::commit(bar(3 + (j & 1)));
        return true;
      };
      bool alive = tiles == 0 || (t5::barrier_wait(bar(0), 0, dead) && score(0));
      for (int j = 0; alive && j < tiles; ++j) {
        alive = t5::barrier_wait(bar(5 + (j & 1)), (j >> 1) & 1, dead);
        if (alive && sees(w, j)) {
          alive = t5::barrier_wait(bar(11 + w), done & 1, dead);
          if (!alive) break;
          t5::fence_after_sync();
          t5::multiply_rows<kLongTile>(sums, scores, base + M::kV + (j & 1) * M::kTile, out_instr, done > 0);
          t5::commit(bar(13 + w));
          ++done;
        }
        if (!alive) break;
        if (j + 2 < tiles) t5::commit(bar(7 + (j & 1)));
        // products of one thread are done in the order of their issue: the scores may overwrite the probabilities
        if (j + 1 < tiles) alive = score(j + 1);
      }
    }
  }
  // All products and copies have been waited for, except after a wait that gave up: then what is still under
  // way ends within the memory that this CTA holds.
  t5::fence_before_sync();
  __syncthreads();
  if (s_dead) t5::settle(bar(15 + (warp & 1)), (warp == 12 || warp == 13) && t5::elect_one(), &g_wait_timeouts);
  __syncthreads();
  t5::fence_after_sync();
  if (warp == 12) t5::tmem_free(tmem, M::kColumns);
}

template <typename T, int DP, bool GENERAL>
int launch_long_forward(const Problem& a, int dtype, cudaStream_t stream) {
  auto kernel = long_forward_kernel<T, DP, GENERAL>;
  constexpr int bytes = LongForwardMemory<DP>::kBytes;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(TEXB_ERR_CUDA, "attention long_forward_kernel: %s", cudaGetErrorString(e));
  Maps maps = {};
  maps.used = a.perm == nullptr && make_map(&maps.q, a, a.q, a.heads, kLongTile, dtype) && make_map(&maps.k, a, a.k, a.kv_heads, kLongTile, dtype) &&
              make_map(&maps.v, a, a.v, a.kv_heads, kLongTile, dtype);
  const dim3 grid(unsigned((a.n + kLongRows - 1) / kLongRows), unsigned(a.heads));
  kernel<<<grid, kLongThreads, bytes, stream>>>(a, maps);
  return check_launch("attention long_forward_kernel");
}

template <int DP>
int long_forward_by_type(const Problem& a, int dtype, bool general, cudaStream_t stream) {
  if (dtype == TEXB_BFLOAT16)
    return general ? launch_long_forward<__nv_bfloat16, DP, true>(a, dtype, stream)
                   : launch_long_forward<__nv_bfloat16, DP, false>(a, dtype, stream);
  return general ? launch_long_forward<__half, DP, true>(a, dtype, stream) : launch_long_forward<__half, DP, false>(a, dtype, stream);
}

// Waits that gave up in this unit's kernels since the library was loaded.
template <int DP>
int long_forward_timeouts(int* count) {
  const cudaError_t e = cudaMemcpyFromSymbol(count, g_wait_timeouts, sizeof(int));
  return e == cudaSuccess ? TEXB_OK : fail(TEXB_ERR_CUDA, "device status: %s", cudaGetErrorString(e));
}

}  // namespace attention
}  // namespace texb
