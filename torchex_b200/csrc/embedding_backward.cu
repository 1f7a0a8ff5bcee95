// Gradient of a table of rows by token:
//   g_weight[v, :] = scale * sum over {t : token_t = v, v != padding} of g[t, :]
// for every row v of the table, rows without a token being 0.
//
// Bound by HBM: n rows of g are read once and `vocab` rows written once.  There is no
// floating-point atomic, so the result is the same bits every time:
//
//   1. The tokens are sorted, stably, with their positions as payload.  Up to 131 072 tokens
//      stay on chip for that: one cluster of up to eight CTAs keeps them in registers, and each
//      digit pass moves them through distributed shared memory -- one launch, no trip to HBM
//      between passes.  The rest of the same grid meanwhile writes the zero rows: each CTA marks
//      the tokens that fall into its part of the table in shared memory and clears the rows
//      nobody asked for, so the larger part of a sparse gradient is written while the sort runs.
//      More tokens take the plan builder's multi-launch sort, and a kernel that looks every row
//      up in the sorted tokens clears the others.
//   2. Tiles of consecutive sorted positions are walked by one group of lanes each, three batches
//      of eight rows of g (four of fp32) in flight whatever the lengths of the runs.  A run that begins and ends inside its
//      tile is written at once; the parts of the others go to two slots per tile, in fp32.
//   3. Where a run first crosses a tile boundary, one group adds its parts in order; runs of
//      many tiles (padding that is not excluded, very frequent tokens) are added by all
//      warps of a CTA.
//
// Measured, sort and clear / sums / joins: 16 384 tokens of a Zipf distribution, table of 32 768 rows of 1024 bf16
// values: 17 / 17 / 6 us; 9973 tokens, 50 021 rows of 515 fp32 values (4-byte accesses): 22 / 21 / 10 us.
//
// Sums of 16-bit rows are plain fp32 sums: the one rounding at the end is coarser than what the
// additions lose.  Sums of fp32 rows carry an error-free correction term through every addition,
// as in the segment reductions.

#include <cooperative_groups.h>

#include <atomic>

#include "embedding.cuh"

namespace cg = cooperative_groups;

namespace texb {

int sort_keys_impl(const int32_t*, int64_t, int64_t, int32_t*, int32_t*, void*, size_t, cudaStream_t);
size_t plan_workspace_bytes_impl(int64_t, int64_t, int);

namespace {

static __device__ int g_bad_tokens = 0;

// Key of a token: its id, or `vocab` for those that take no part (they sort behind the table).
template <typename IdT>
__device__ __forceinline__ uint32_t key_of(IdT token, int64_t vocab, int64_t padding, bool count) {
  const int64_t id = int64_t(token);
  const bool ok = id >= 0 && id < vocab;
  if (!ok && count) atomicAdd(&g_bad_tokens, 1);
  return ok && id != padding ? uint32_t(id) : uint32_t(vocab);
}

// ---- clearing rows ------------------------------------------------------------------------

// Row v of a table of rows of `row_words` words of type W, cleared by `lanes` lanes: 16 bytes at a time
// between the words in front of the first 16-byte boundary and those behind the last.
template <typename W>
__device__ __forceinline__ void clear_row(W* table, int64_t v, int64_t row_words, int lane, int lanes) {
  W* row = table + v * row_words;
  constexpr int kPer = 16 / int(sizeof(W));
  const int64_t head = min(row_words, int64_t((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / int64_t(sizeof(W)));
  const int64_t wide = (row_words - head) / kPer;
  uint4* body = reinterpret_cast<uint4*>(row + head);
  for (int64_t i = lane; i < wide; i += lanes) body[i] = uint4{};
  if constexpr (kPer > 1) {
    for (int64_t i = lane; i < head; i += lanes) row[i] = W{};
    for (int64_t i = head + wide * kPer + lane; i < row_words; i += lanes) row[i] = W{};
  }
}

// ---- sort of up to 131 072 tokens, and the zero rows, in one launch ------------------------------

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxItems = 16;              // tokens of a thread
constexpr int kMaxCluster = 8;             // the portable cluster size
constexpr int kMaxSorted = kMaxCluster * kSortThreads * kMaxItems;
constexpr int kMaxDigitBits = 9;
constexpr int kMaxBins = 1 << kMaxDigitBits;
constexpr int64_t kMarkBits = int64_t(1) << 19;  // rows of the table that a clearing CTA marks at a time (64 KB)

struct SortLayout {  // shared memory of a sorting CTA, in bytes
  static constexpr int kCounts = 0;                                       // uint16 [kSortWarps][kMaxBins]
  static constexpr int kTotals = kCounts + kSortWarps * kMaxBins * 2;     // uint32 [kMaxCluster][kMaxBins]
  static constexpr int kBase = kTotals + kMaxCluster * kMaxBins * 4;      // uint32 [kMaxBins]
  static constexpr int kScan = kBase + kMaxBins * 4;                      // uint32 [32]
  static constexpr int kItems = kScan + 128;                              // uint2 [items of the CTA]
};

// Sum of `v` over the threads before this one.  All threads of the CTA call it; values beyond the first
// 512 threads must be 0 (only their sum over 16 warps is needed).
__device__ __forceinline__ uint32_t exclusive_scan(uint32_t v, uint32_t* scan) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t incl = v;
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  __syncthreads();  // the last call's readers are done
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  uint32_t before = incl - v;
  for (int w = 0; w < min(warp, kMaxBins / 32); ++w) before += scan[w];
  return before;
}

// Cluster 0 sorts; CTAs of the other clusters clear the rows of the table without a token.
// items: tokens per thread (a power of two); digit_bits * passes covers the keys 0 .. vocab.
template <typename IdT, typename W>
__global__ void __launch_bounds__(kSortThreads, 1)
sort_and_clear_kernel(const IdT* __restrict__ tokens, int n, int64_t vocab, int64_t padding, int items, int digit_bits,
                      int passes, int32_t* __restrict__ sid, int32_t* __restrict__ perm, W* __restrict__ table,
                      int64_t row_words, int lanes) {
  extern __shared__ __align__(16) unsigned char smem[];
  const cg::cluster_group cluster = cg::this_cluster();
  const int ranks = int(cluster.num_blocks());

  if (int(blockIdx.x) >= ranks) {
    // ---- clear: every cluster has an even share of the table's rows, every CTA of it a part of the
    // share.  The CTAs divide the tokens, and mark those of the share in the memory of the CTA that has
    // the row (each CTA reading all tokens took 30 us for 131 072).
    constexpr int kScan = 8;
    uint32_t* marks = reinterpret_cast<uint32_t*>(smem);
    const int64_t shares = gridDim.x / ranks - 1, which = blockIdx.x / ranks - 1;
    const int me = int(cluster.block_rank());
    const int64_t end = vocab * (which + 1) / shares;
    for (int64_t lo = vocab * which / shares; lo < end; lo += ranks * kMarkBits) {
      const int64_t hi = min(end, lo + ranks * kMarkBits);
      const int64_t part = (hi - lo + ranks - 1) / ranks;  // rows of a CTA, at most kMarkBits
      for (int i = threadIdx.x; i < int((part + 31) / 32); i += kSortThreads) marks[i] = 0u;
      cluster.sync();
      for (int i0 = me * kSortThreads + threadIdx.x; i0 < n; i0 += ranks * kSortThreads * kScan) {
        IdT token[kScan];  // all loads of a batch before the first mark
#pragma unroll
        for (int k = 0; k < kScan; ++k)
          if (i0 + k * ranks * kSortThreads < n) token[k] = __ldg(tokens + i0 + k * ranks * kSortThreads);
#pragma unroll
        for (int k = 0; k < kScan; ++k) {
          if (i0 + k * ranks * kSortThreads >= n) break;
          const int64_t key = key_of<IdT>(token[k], vocab, padding, false);
          if (key >= lo && key < hi) {
            const int owner = int((key - lo) / part), place = int((key - lo) - owner * part);
            volatile uint32_t* word = cluster.map_shared_rank(marks + (place >> 5), owner);
            // a frequent token is marked once, not by a queue of atomics on one word
            if (!(*word >> (place & 31) & 1u)) atomicOr(const_cast<uint32_t*>(word), 1u << (place & 31));
          }
        }
      }
      cluster.sync();  // all marks are there; and, behind it, nobody touches another CTA's memory before the next round's first barrier
      const int64_t first = lo + me * part, last = min(hi, first + part);
      for (int64_t v = first + threadIdx.x / lanes; v < last; v += kSortThreads / lanes)
        if (!(marks[(v - first) >> 5] >> ((v - first) & 31) & 1u)) clear_row(table, v, row_words, threadIdx.x & (lanes - 1), lanes);
      __syncthreads();
    }
    return;
  }

  // ---- sort.  Item k of lane l of warp w of CTA c is token ((c * 32 + w) * items + k) * 32 + l,
  // so (c, w, k, l) order is token order, and every pass keeps it for equal digits.
  uint16_t(*counts)[kMaxBins] = reinterpret_cast<uint16_t(*)[kMaxBins]>(smem + SortLayout::kCounts);
  uint32_t(*totals)[kMaxBins] = reinterpret_cast<uint32_t(*)[kMaxBins]>(smem + SortLayout::kTotals);
  uint32_t* base = reinterpret_cast<uint32_t*>(smem + SortLayout::kBase);
  uint32_t* scan = reinterpret_cast<uint32_t*>(smem + SortLayout::kScan);
  uint2* buffer = reinterpret_cast<uint2*>(smem + SortLayout::kItems);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = int(cluster.block_rank());
  const int per_cta = kSortThreads * items;  // a power of two
  const int shift_cta = 31 - __clz(per_cta);
  const int bins = 1 << digit_bits;
  const int mine = warp * items * 32 + lane;  // place of item 0 of this lane in the CTA's share
  const uint32_t before_me = (1u << lane) - 1u;
  const int share = max(0, min(per_cta, n - rank * per_cta));  // tokens of this CTA: all but the last ones have per_cta

  uint2 item[kMaxItems];  // (key, position)
#pragma unroll
  for (int k = 0; k < kMaxItems; ++k) {
    const int at = rank * per_cta + mine + k * 32;
    if (k < items && at < n) item[k] = make_uint2(key_of<IdT>(tokens[at], vocab, padding, true), uint32_t(at));
  }
  cluster.sync();  // every CTA of the cluster runs before the first write into another one's memory
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * digit_bits;
    for (int i = threadIdx.x; i < kSortWarps * kMaxBins / 2; i += kSortThreads) reinterpret_cast<uint32_t*>(&counts[0][0])[i] = 0u;
    __syncthreads();
    uint32_t order[kMaxItems];  // items of the same digit before this one in its warp
#pragma unroll
    for (int k = 0; k < kMaxItems; ++k) {
      if (k < items) {
        const bool valid = mine + k * 32 < share;
        const uint32_t d = (item[k].x >> shift) & (bins - 1);
        uint32_t peers = __ballot_sync(0xffffffffu, valid);  // match.any took 1.6 times as long as nine ballots
#pragma unroll
        for (int b = 0; b < kMaxDigitBits; ++b) {
          const bool one = (d >> b) & 1u;
          const uint32_t ones = __ballot_sync(0xffffffffu, one);
          peers &= one ? ones : ~ones;
        }
        uint32_t seen = 0u;
        if (valid) seen = counts[warp][d];
        __syncwarp();
        if (valid && (peers & before_me) == 0u) counts[warp][d] = uint16_t(seen + __popc(peers));
        __syncwarp();
        order[k] = seen + __popc(peers & before_me);
      }
    }
    __syncthreads();
    // counts become prefixes over the CTA's warps; the CTA's totals go to every CTA of the cluster
    const int d = threadIdx.x;
    uint32_t run = 0u;
    if (d < bins) {
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = counts[w][d];
        counts[w][d] = uint16_t(run);
        run += c;
      }
      for (int r = 0; r < ranks; ++r) cluster.map_shared_rank(&totals[rank][d], r)[0] = run;
    }
    cluster.sync();
    // place of this CTA's first item of each digit: all items of smaller digits, and those of this
    // digit in earlier CTAs
    uint32_t all = 0u, earlier = 0u;
    if (d < bins) {
      for (int r = 0; r < ranks; ++r) {
        const uint32_t t = totals[r][d];
        earlier += r < rank ? t : 0u;
        all += t;
      }
    }
    const uint32_t start = exclusive_scan(all, scan);
    if (d < bins) base[d] = start + earlier;
    __syncthreads();
    // Straight to their places in the cluster's memory.  Putting the share into digit order in the CTA's own
    // memory first, so that these stores run along consecutive words, took longer: 25 us instead of 23 for the
    // whole gradient of 1024 tokens (32768 rows of 8 columns), 79 instead of 75 for 131072 (131072 rows of 8).
#pragma unroll
    for (int k = 0; k < kMaxItems; ++k) {
      if (k < items && mine + k * 32 < share) {
        const uint32_t dg = (item[k].x >> shift) & (bins - 1);
        const uint32_t to = base[dg] + counts[warp][dg] + order[k];  // < n <= ranks * per_cta
        cluster.map_shared_rank(buffer, to >> shift_cta)[to & (per_cta - 1)] = item[k];
      }
    }
    cluster.sync();
    // after the last pass nobody writes into another CTA's memory any more, so no CTA has to wait
    // for the others' reads before it ends
#pragma unroll
    for (int k = 0; k < kMaxItems; ++k)
      if (k < items && mine + k * 32 < share) item[k] = buffer[mine + k * 32];
  }
#pragma unroll
  for (int k = 0; k < kMaxItems; ++k) {
    const int at = rank * per_cta + mine + k * 32;
    if (k < items && at < n) {
      sid[at] = int32_t(item[k].x);
      perm[at] = int32_t(item[k].y);
    }
  }
}

// ---- more tokens: keys for the plan builder's sort, and the zero rows by search --------------------

constexpr int kThreads = 256;

template <typename IdT>
__global__ void token_keys_kernel(const IdT* __restrict__ tokens, int n, int64_t vocab, int64_t padding,
                                  int32_t* __restrict__ keys) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i < n) keys[i] = int32_t(key_of<IdT>(tokens[i], vocab, padding, true));
}

// One warp per 32 rows: each lane searches one row in the sorted tokens, then the warp clears
// those that are not there.
template <typename W>
__global__ void __launch_bounds__(kThreads)
clear_absent_rows_kernel(const int32_t* __restrict__ sid, int n, int64_t vocab, W* __restrict__ table, int64_t row_words,
                         int lanes) {
  const int lane = threadIdx.x & 31;
  const int64_t v0 = (int64_t(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32) * 32;
  if (v0 >= vocab) return;
  const int64_t v = v0 + lane;
  int lo = 0, hi = n;  // sid[i] < v for i < lo, sid[i] >= v for i >= hi
  while (lo < hi) {
    const int mid = lo + ((hi - lo) >> 1);
    if (__ldg(sid + mid) < v) lo = mid + 1; else hi = mid;
  }
  const bool absent = v < vocab && (lo == n || __ldg(sid + lo) != v);
  const uint32_t todo = __ballot_sync(0xffffffffu, absent);
  const int step = 32 / lanes, sub = lane / lanes;
  for (int r = sub; r < 32; r += step)
    if (todo >> r & 1u) clear_row(table, v0 + r, row_words, lane & (lanes - 1), lanes);
}

// ---- sums ------------------------------------------------------------------------------------

template <typename T>
struct Sum {  // running sum of one column
  static constexpr bool kExact = sizeof(T) == 4;
  static constexpr int kPlanes = kExact ? 2 : 1;
  float s, c;
  __device__ __forceinline__ void clear() { s = 0.f; c = 0.f; }
  __device__ __forceinline__ void add(float v) {
    if constexpr (kExact) {
      const float t = s + v;
      const float b = t - s;
      c += (s - (t - b)) + (v - b);
      s = t;
    } else {
      s += v;
    }
  }
  __device__ __forceinline__ void add(const Sum& o) {
    add(o.s);
    if constexpr (kExact) c += o.c;
  }
  __device__ __forceinline__ float total() const {
    if constexpr (kExact) return isfinite(s) ? s + c : s;  // an infinite or NaN sum has no error term
    return s;
  }
};

// A lane holds kBlocks accesses of BYTES bytes of a chunk of columns: eight values, whatever the
// width of the access.  Its ring in shared memory holds kStages batches of kBatch rows, 384 bytes.
constexpr int kSumThreads = 128;
template <typename T, int BYTES>
struct Shape {
  static constexpr int kVec = BYTES / int(sizeof(T));
  static constexpr int kBlocks = 8 / kVec;
  static constexpr int kColumns = 8;
  static constexpr int kStages = 3;
  static constexpr int kBatch = 16 / int(sizeof(T));
};

struct Tiles {
  int n;              // sorted positions
  int tile;           // positions of a tile
  int dim, lanes;     // columns; lanes of a group
  int64_t vocab;
  float scale;
  float* slots;       // [tiles][2][planes][padded columns]: the part of the run that comes from the left, and of the
                      // one that begins here and goes on to the right
  int64_t slot_words; // words of one slot
};

// Columns of this lane: access b covers columns (first + b * lanes) * kVec ...
template <typename T, int BYTES>
__device__ __forceinline__ void store_slot(const Tiles& t, int64_t slot, int first, const Sum<T>* acc) {
  using S = Shape<T, BYTES>;
  float* p = t.slots + slot * t.slot_words;
  const int vectors = t.dim / S::kVec;
#pragma unroll
  for (int b = 0; b < S::kBlocks; ++b) {
    const int i = first + b * t.lanes;
    if (i < vectors) {
#pragma unroll
      for (int e = 0; e < S::kVec; ++e) {
        p[int64_t(i) * S::kVec + e] = acc[b * S::kVec + e].s;
        if constexpr (Sum<T>::kExact) p[t.dim + int64_t(i) * S::kVec + e] = acc[b * S::kVec + e].c;
      }
    }
  }
}

template <typename T, int BYTES>
__device__ __forceinline__ void add_slot(const Tiles& t, int64_t slot, int first, Sum<T>* acc) {
  using S = Shape<T, BYTES>;
  const float* p = t.slots + slot * t.slot_words;
  const int vectors = t.dim / S::kVec;
#pragma unroll
  for (int b = 0; b < S::kBlocks; ++b) {
    const int i = first + b * t.lanes;
    if (i < vectors) {
#pragma unroll
      for (int e = 0; e < S::kVec; ++e) {
        Sum<T> o;
        o.s = p[int64_t(i) * S::kVec + e];
        o.c = 0.f;
        if constexpr (Sum<T>::kExact) o.c = p[t.dim + int64_t(i) * S::kVec + e];
        acc[b * S::kVec + e].add(o);
      }
    }
  }
}

template <typename T, int BYTES>
__device__ __forceinline__ void store_row(const Tiles& t, T* g_weight, int64_t v, int first, const Sum<T>* acc) {
  using S = Shape<T, BYTES>;
  const int vectors = t.dim / S::kVec;
#pragma unroll
  for (int b = 0; b < S::kBlocks; ++b) {
    const int i = first + b * t.lanes;
    if (i < vectors) {
      Chunk<T, BYTES> c;
#pragma unroll
      for (int e = 0; e < S::kVec; ++e) c.v[e] = narrow<T>(acc[b * S::kVec + e].total() * t.scale);
      store_chunk<T, BYTES>(g_weight + v * t.dim + int64_t(i) * S::kVec, c);
    }
  }
}

__device__ __forceinline__ uint32_t smem_address(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

// One access of a row of g into the lane's ring.  Rows of an odd number of 16-bit values have no
// 4-byte alignment to copy by, and go through registers.
template <typename T, int BYTES>
__device__ __forceinline__ void fetch(Chunk<T, BYTES>* to, const T* from) {
  if constexpr (BYTES == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_address(to)), "l"(from) : "memory");
  } else if constexpr (BYTES == 4) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_address(to)), "l"(from) : "memory");
  } else {
    *to = load_chunk_once<T, BYTES>(from);
  }
}

// One group of lanes per (tile, chunk of columns).  The rows of g go through a ring in shared memory,
// three batches deep, in which every lane reads only what it copied itself -- so the copies need no
// barrier, and a run's end does not hold back the loads behind it.  Walking the rows of a batch is a
// loop, not unrolled: eight copies of the code that closes a run (division of the work between row and
// slot, stores) overflowed the instruction cache: 27 us instead of 16 for 16 384 rows of 1024.
template <typename T, int BYTES>
__global__ void __launch_bounds__(kSumThreads)
sum_tiles_kernel(const T* __restrict__ g, const int32_t* __restrict__ sid, const int32_t* __restrict__ perm, Tiles t,
                 T* __restrict__ g_weight) {
  using S = Shape<T, BYTES>;
  using Access = Chunk<T, BYTES>;
  __shared__ Access ring[S::kStages][S::kBatch][S::kBlocks][kSumThreads];
  const int lane = threadIdx.x & (t.lanes - 1);
  const int64_t tile = (int64_t(blockIdx.x) * kSumThreads + threadIdx.x) / t.lanes;
  const int64_t begin = tile * t.tile;
  if (begin >= t.n) return;
  const int end = int(min(int64_t(t.n), begin + t.tile));
  const int vectors = t.dim / S::kVec;
  const int first = blockIdx.y * t.lanes * S::kBlocks + lane;
  const int vocab = int(t.vocab);
  const int before = begin > 0 ? __ldg(sid + begin - 1) : -1;

  // Keys and rows of a batch; positions behind the tile or without a table row have row -1.
  int next_key[S::kBatch], next_row[S::kBatch];
  auto load_places = [&](int p0) {
#pragma unroll
    for (int u = 0; u < S::kBatch; ++u) {
      next_key[u] = p0 + u < end ? __ldg(sid + p0 + u) : vocab;
      next_row[u] = p0 + u < end ? __ldg(perm + p0 + u) : -1;
    }
  };
  auto fetch_batch = [&](int stage) {
#pragma unroll
    for (int u = 0; u < S::kBatch; ++u) {
      if (next_key[u] < vocab) {
        const T* row = g + int64_t(next_row[u]) * t.dim;
#pragma unroll
        for (int b = 0; b < S::kBlocks; ++b) {
          const int i = first + b * t.lanes;
          if (i < vectors) fetch<T, BYTES>(&ring[stage][u][b][threadIdx.x], row + int64_t(i) * S::kVec);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int p_load = int(begin);
#pragma unroll
  for (int st = 0; st < S::kStages - 1; ++st) {
    load_places(p_load);
    fetch_batch(st);
    p_load += S::kBatch;
  }
  load_places(p_load);

  int run = __ldg(sid + begin);
  bool from_left = before == run;
  Sum<T> acc[S::kColumns];
#pragma unroll
  for (int k = 0; k < S::kColumns; ++k) acc[k].clear();
  int stage = 0, load_stage = S::kStages - 1;
  for (int p0 = int(begin); p0 < end && run < vocab; p0 += S::kBatch) {
    fetch_batch(load_stage);
    p_load += S::kBatch;
    load_places(p_load);
    load_stage = load_stage + 1 == S::kStages ? 0 : load_stage + 1;
    asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
#pragma unroll 1
    for (int u = 0; u < S::kBatch && p0 + u < end; ++u) {
      const int key = __ldg(sid + p0 + u);
      if (key != run) {  // the run before this position ends inside the tile
        if (from_left) store_slot<T, BYTES>(t, 2 * tile, first, acc);
        else store_row<T, BYTES>(t, g_weight, run, first, acc);
#pragma unroll
        for (int k = 0; k < S::kColumns; ++k) acc[k].clear();
        run = key;
        from_left = false;
        if (run >= vocab) break;
      }
#pragma unroll
      for (int b = 0; b < S::kBlocks; ++b) {
        const Access c = ring[stage][u][b][threadIdx.x];
#pragma unroll
        for (int e = 0; e < S::kVec; ++e) acc[b * S::kVec + e].add(widen<T>(c.v[e]));
      }
    }
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (run >= vocab) return;
  if (from_left) store_slot<T, BYTES>(t, 2 * tile, first, acc);
  else if (end < t.n && __ldg(sid + end) == run) store_slot<T, BYTES>(t, 2 * tile + 1, first, acc);
  else store_row<T, BYTES>(t, g_weight, run, first, acc);
}

// Runs that cross tile boundaries.  One group of lanes per (boundary, chunk); only the first
// boundary of a run has work.  Runs of more than kShortChain tiles are added by the whole CTA.
constexpr int kShortChain = 8;
constexpr int kJoinThreads = 128;

template <typename T, int BYTES>
__global__ void __launch_bounds__(kJoinThreads)
join_runs_kernel(const int32_t* __restrict__ sid, Tiles t, T* __restrict__ g_weight) {
  using S = Shape<T, BYTES>;
  __shared__ float s_part[kJoinThreads * S::kColumns * Sum<T>::kPlanes];
  __shared__ int s_long[kJoinThreads], s_longs;  // boundaries where a long run begins
  const int lane = threadIdx.x & (t.lanes - 1), group = threadIdx.x / t.lanes, groups = kJoinThreads / t.lanes;
  const int tiles = int((int64_t(t.n) + t.tile - 1) / t.tile);
  const int boundary = int(blockIdx.x) * groups + group + 1;  // between tiles boundary - 1 and boundary
  const int first = blockIdx.y * t.lanes * S::kBlocks + lane;
  if (threadIdx.x == 0) s_longs = 0;
  __syncthreads();
  auto key_at = [&](int64_t tile) { return __ldg(sid + tile * t.tile); };
  Sum<T> acc[S::kColumns];
#pragma unroll
  for (int k = 0; k < S::kColumns; ++k) acc[k].clear();
  if (boundary < tiles) {
    const int64_t p = int64_t(boundary) * t.tile;
    const int v = __ldg(sid + p), left = __ldg(sid + p - 1);
    const int before = p > t.tile ? __ldg(sid + p - t.tile - 1) : -1;
    int more = 0;  // tiles behind this one that the run reaches, up to kShortChain
#pragma unroll
    for (int k = 1; k <= kShortChain; ++k) more += boundary + k < tiles && key_at(boundary + k) == v;
    if (v < t.vocab && left == v && before != v) {
      if (more == kShortChain) {
        if (lane == 0) s_long[atomicAdd(&s_longs, 1)] = boundary;
      } else {
        add_slot<T, BYTES>(t, 2 * int64_t(boundary - 1) + 1, first, acc);
        for (int k = 0; k <= more; ++k) add_slot<T, BYTES>(t, 2 * int64_t(boundary + k), first, acc);
        store_row<T, BYTES>(t, g_weight, v, first, acc);
      }
    }
  }
  __syncthreads();
  const int longs = s_longs;
  for (int q = 0; q < longs; ++q) {  // in any order: each is a row of its own
    const int b0 = s_long[q];
    const int u = key_at(b0);
    int64_t lo = b0, hi = tiles;  // the run reaches tile lo, not hi
    while (hi - lo > 1) {         // kJoinThreads probes at a time
      const int64_t step = (hi - lo + kJoinThreads - 1) / kJoinThreads, at = lo + step * (threadIdx.x + 1);
      const int reached = __syncthreads_count(at < hi && key_at(at) == u);
      hi = min(hi, lo + step * (reached + 1));
      lo += step * reached;
    }
    // group k adds an even, consecutive share of the run's parts; the shares are added pairwise
    const int64_t count = hi - b0, from = b0 + count * group / groups, to = b0 + count * (group + 1) / groups;
#pragma unroll
    for (int k = 0; k < S::kColumns; ++k) acc[k].clear();
    if (group == 0) add_slot<T, BYTES>(t, 2 * int64_t(b0 - 1) + 1, first, acc);
#pragma unroll 4
    for (int64_t b = from; b < to; ++b) add_slot<T, BYTES>(t, 2 * b, first, acc);
    for (int half = groups / 2; half > 0; half /= 2) {
      if (group >= half && group < 2 * half) {
#pragma unroll
        for (int k = 0; k < S::kColumns; ++k) {
          s_part[k * kJoinThreads + threadIdx.x] = acc[k].s;
          if constexpr (Sum<T>::kExact) s_part[(S::kColumns + k) * kJoinThreads + threadIdx.x] = acc[k].c;
        }
      }
      __syncthreads();
      if (group < half) {
        const int other = threadIdx.x + half * t.lanes;
#pragma unroll
        for (int k = 0; k < S::kColumns; ++k) {
          Sum<T> part;
          part.s = s_part[k * kJoinThreads + other];
          part.c = 0.f;
          if constexpr (Sum<T>::kExact) part.c = s_part[(S::kColumns + k) * kJoinThreads + other];
          acc[k].add(part);
        }
      }
      __syncthreads();
    }
    if (group == 0) store_row<T, BYTES>(t, g_weight, u, first, acc);
  }
}

// ---- launches --------------------------------------------------------------------------------

// Positions of a tile: 128 where that still gives some 380 threads per SM a tile, less for fewer
// tokens or narrower rows, down to 8.  Larger tiles mean fewer partial sums through HBM (up to two
// fp32 rows per tile), smaller ones more rows in flight.  A batch that fits one tile takes one, which saves
// joining them, a launch: what a small step costs is its launches.
inline int tile_positions(int64_t n, int dim) {
  if (n <= 128) return 128;
  const int64_t threads = ceil_div(dim, 8);  // eight values per lane
  int tile = 128;
  while (tile > 8 && ceil_div(n, tile) * threads < 148 * 384) tile /= 2;
  return tile;
}

struct Workspace {
  int32_t *sid, *perm, *keys;
  float* slots;
  void* sort;
  size_t sort_bytes, bytes;
  int tile;
};

Workspace carve(void* ws, int64_t n, int dim, int dtype) {
  Workspace w;
  const uintptr_t base = align_up(reinterpret_cast<uintptr_t>(ws), 256);
  const size_t rows = align_up(size_t(n) * sizeof(int32_t), 256);
  const bool on_chip = n <= kMaxSorted;
  size_t at = 0;
  auto take = [&](size_t bytes) { void* p = reinterpret_cast<void*>(base + at); at += align_up(bytes, 256); return p; };
  w.tile = tile_positions(n, dim);
  w.sid = static_cast<int32_t*>(take(rows));
  w.perm = static_cast<int32_t*>(take(rows));
  w.keys = static_cast<int32_t*>(take(on_chip ? 0 : rows));
  w.slots = static_cast<float*>(take(size_t(ceil_div(n, w.tile)) * 2 * size_t(dim) * (dtype == TEXB_FLOAT32 ? 8 : 4)));
  w.sort_bytes = on_chip ? 0 : plan_workspace_bytes_impl(n, 0, 0) + 256;
  w.sort = take(w.sort_bytes);
  w.bytes = at + 256;
  return w;
}

// Clusters of `ranks` CTAs of the kernel that fit the current device at once; asked once per device
// and shape (the query takes longer than a launch).
template <typename K>
int resident_clusters(K kernel, const cudaLaunchConfig_t& cfg, int ranks, int items) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices][kMaxCluster + 1][kMaxItems + 1];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kDevices) device = -1;
  if (device >= 0) {
    const int v = known[device][ranks][items].load(std::memory_order_relaxed);
    if (v > 0) return v;
  }
  // the largest shared memory that any shape asks for: the attribute stays with the kernel
  constexpr int kMost = SortLayout::kItems + kSortThreads * kMaxItems * int(sizeof(uint2));
  static_assert(kMost >= kMarkBits / 8, "the marks fit as well");
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost) != cudaSuccess) return 0;
  int count = 0;
  if (cudaOccupancyMaxActiveClusters(&count, kernel, &cfg) != cudaSuccess || count < 2) {
    (void)cudaGetLastError();
    count = 2;
  }
  if (device >= 0) known[device][ranks][items].store(count, std::memory_order_relaxed);
  return count;
}

template <typename IdT, typename W>
int launch_sort_and_clear(const IdT* tokens, int64_t n, int64_t vocab, int64_t padding, const Workspace& w, W* table,
                          int64_t row_words, cudaStream_t stream) {
  int ranks = 1;
  while (ranks < kMaxCluster && n > int64_t(ranks) * kSortThreads * 2) ranks *= 2;
  int items = 1;
  while (int64_t(ranks) * kSortThreads * items < n) items *= 2;
  int bits = 0;
  while (vocab >> bits) ++bits;  // keys 0 .. vocab
  const int passes = n > 1 ? int(ceil_div(bits, kMaxDigitBits)) : 0;
  const int digit_bits = passes ? int(ceil_div(bits, passes)) : 1;
  const int lanes = lanes_of(row_words);
  // for the items of a sorting CTA or the marks of a clearing one, whatever the table: the number of clusters that fit is
  // remembered by ranks and items
  size_t smem = SortLayout::kItems + size_t(kSortThreads) * items * sizeof(uint2);
  if (smem < size_t(kMarkBits / 8)) smem = size_t(kMarkBits / 8);
  cudaError_t e = cudaSuccess;
  auto kernel = sort_and_clear_kernel<IdT, W>;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(ranks);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // Clearing CTAs: at least 64 KB of table each, and no more than run beside the sort at once -- a
  // cluster that had to wait for a free one starts when the others end (239 us instead of 143 for 0.7 GB).
  int64_t workers = ceil_div(vocab * row_words * int64_t(sizeof(W)), 65536);
  cfg.gridDim = dim3(unsigned(ranks) * 2);
  const int clusters = resident_clusters(kernel, cfg, ranks, items);
  if (clusters == 0) return check_launch("sort_and_clear_kernel");
  const int64_t room = int64_t(clusters - 1) * ranks;
  workers = workers < 1 ? 1 : workers;
  workers = int64_t(align_up(size_t(workers), size_t(ranks)));
  if (workers > room) workers = room;
  cfg.gridDim = dim3(unsigned(ranks + workers));
  e = cudaLaunchKernelEx(&cfg, kernel, tokens, int(n), vocab, padding, items, digit_bits, passes, w.sid, w.perm, table,
                         row_words, lanes);
  if (e != cudaSuccess) return fail(TEXB_ERR_CUDA, "sort_and_clear_kernel: %s", cudaGetErrorString(e));
  return check_launch("sort_and_clear_kernel");
}

// W: the widest word that the table's rows allow.
template <typename IdT, typename W>
int sort_tokens(const IdT* tokens, int64_t n, int64_t vocab, int64_t padding, const Workspace& w, void* g_weight,
                int64_t row_bytes, cudaStream_t stream) {
  W* table = static_cast<W*>(g_weight);
  const int64_t row_words = row_bytes / int64_t(sizeof(W));
  if (n <= kMaxSorted) return launch_sort_and_clear<IdT, W>(tokens, n, vocab, padding, w, table, row_words, stream);
  token_keys_kernel<IdT><<<unsigned(ceil_div(n, kThreads)), kThreads, 0, stream>>>(tokens, int(n), vocab, padding, w.keys);
  int st = check_launch("token_keys_kernel");
  if (st == TEXB_OK) st = sort_keys_impl(w.keys, n, vocab + 1, w.sid, w.perm, w.sort, w.sort_bytes, stream);
  if (st != TEXB_OK) return st;
  clear_absent_rows_kernel<W><<<unsigned(ceil_div(vocab, kThreads)), kThreads, 0, stream>>>(
      w.sid, int(n), vocab, table, row_words, lanes_of(row_words));
  return check_launch("clear_absent_rows_kernel");
}

template <typename IdT>
int sort_tokens_any(const void* tokens, int64_t n, int64_t vocab, int64_t padding, const Workspace& w, void* g_weight,
                    int64_t row_bytes, cudaStream_t stream) {
  const IdT* tok = static_cast<const IdT*>(tokens);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(g_weight) | uintptr_t(row_bytes);
  if (bits % 16 == 0) return sort_tokens<IdT, uint4>(tok, n, vocab, padding, w, g_weight, row_bytes, stream);
  if (bits % 4 == 0) return sort_tokens<IdT, uint32_t>(tok, n, vocab, padding, w, g_weight, row_bytes, stream);
  return sort_tokens<IdT, unsigned short>(tok, n, vocab, padding, w, g_weight, row_bytes, stream);
}

template <typename T, int BYTES>
int launch_sums(const T* g, const Workspace& w, int64_t n, int64_t vocab, int dim, float scale, T* g_weight,
                cudaStream_t stream) {
  using S = Shape<T, BYTES>;
  const int64_t vectors = dim / S::kVec;
  Tiles t;
  t.n = int(n);
  t.tile = w.tile;
  t.dim = dim;
  t.lanes = lanes_of(vectors);
  t.vocab = vocab;
  t.scale = scale;
  t.slots = w.slots;
  t.slot_words = int64_t(dim) * Sum<T>::kPlanes;
  const int64_t tiles = ceil_div(n, w.tile);
  static_assert(kSumThreads == kJoinThreads, "one grid for both kernels");
  const dim3 grid(unsigned(ceil_div(tiles, kSumThreads / t.lanes)), unsigned(ceil_div(vectors, t.lanes * S::kBlocks)));
  if (grid.y > 65535u) return fail(TEXB_ERR_UNSUPPORTED, "embedding: rows of %d values are too wide", dim);
  sum_tiles_kernel<T, BYTES><<<grid, kSumThreads, 0, stream>>>(g, w.sid, w.perm, t, g_weight);
  const int st = check_launch("sum_tiles_kernel");
  if (st != TEXB_OK || tiles == 1) return st;
  join_runs_kernel<T, BYTES><<<grid, kJoinThreads, 0, stream>>>(w.sid, t, g_weight);
  return check_launch("join_runs_kernel");
}

template <typename T>
int launch_sums_any(const void* g, const Workspace& w, int64_t n, int64_t vocab, int dim, float scale, void* g_weight,
                    cudaStream_t stream) {
  const T* gp = static_cast<const T*>(g);
  T* o = static_cast<T*>(g_weight);
  const int bytes = access_bytes(int(sizeof(T)), dim, g, g_weight);
  if (bytes == 16) return launch_sums<T, 16>(gp, w, n, vocab, dim, scale, o, stream);
  if (bytes == 4) return launch_sums<T, 4>(gp, w, n, vocab, dim, scale, o, stream);
  return launch_sums<T, int(sizeof(T))>(gp, w, n, vocab, dim, scale, o, stream);
}

}  // namespace

int table_grad_bad_tokens_impl(int* count) {
  const cudaError_t e = cudaMemcpyFromSymbol(count, g_bad_tokens, sizeof(int));
  if (e != cudaSuccess) return fail(TEXB_ERR_CUDA, "device status: %s", cudaGetErrorString(e));
  return TEXB_OK;
}

size_t embedding_backward_workspace_bytes_impl(int64_t n, int64_t vocab, int dim) {
  if (n < 0 || vocab < 0 || dim < 1) return 0;
  return carve(nullptr, n, dim, TEXB_FLOAT32).bytes;
}

int embedding_backward_impl(const void* tokens, int id_bytes, int64_t n, const void* g, int dtype, int64_t vocab,
                            int dim, float scale, int64_t padding_idx, void* g_weight, void* workspace,
                            size_t workspace_bytes, cudaStream_t stream) {
  int st = check_embedding_sizes(id_bytes, n, dtype, vocab, dim);
  if (st != TEXB_OK) return st;
  if (vocab == 0) return TEXB_OK;
  if (!g_weight || (n > 0 && (!tokens || !g))) return fail(TEXB_ERR_INVALID_ARGUMENT, "embedding: NULL pointer");
  const Workspace w = carve(workspace, n, dim, dtype);
  if (!workspace || workspace_bytes < w.bytes)
    return fail(TEXB_ERR_WORKSPACE, "embedding workspace: need %zu bytes, got %zu", w.bytes, workspace_bytes);
  const int64_t row_bytes = int64_t(dim) * dtype_bytes(dtype);
  st = id_bytes == 8 ? sort_tokens_any<int64_t>(tokens, n, vocab, padding_idx, w, g_weight, row_bytes, stream)
                     : sort_tokens_any<int32_t>(tokens, n, vocab, padding_idx, w, g_weight, row_bytes, stream);
  if (st != TEXB_OK || n == 0) return st;
  if (dtype == TEXB_FLOAT32) return launch_sums_any<float>(g, w, n, vocab, dim, scale, g_weight, stream);
  if (dtype == TEXB_BFLOAT16) return launch_sums_any<__nv_bfloat16>(g, w, n, vocab, dim, scale, g_weight, stream);
  return launch_sums_any<__half>(g, w, n, vocab, dim, scale, g_weight, stream);
}

}  // namespace texb
