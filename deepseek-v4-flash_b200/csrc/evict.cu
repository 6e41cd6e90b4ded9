// evict.cu -- bounding a paged latent cache, and ending a drafting step: the
// tokens to keep by their accumulated attention weight, and the move of kept
// rows to the front of a sequence.  No counterpart in the reference.
//
//  * tree_mask: the ancestors of each node of a draft tree (and itself).
//  * evict_select: of a sequence's len tokens the first n_first, the last
//    n_recent and those of the largest weight sums, budget in all, in position
//    order; among equal sums the lowest positions.
//  * keep_rows: row start + keep[i] of a sequence to row start + i, for i in
//    order, through the block table (in place, or into another cache).
//  * keep_sums: the same move of the sequence's weight sums, 0 behind them.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "kernels.h"

namespace qcau {
namespace {

// ---------------------------------------------------------------- tree mask

// One warp per node: its row is cleared, then its chain of parents marked.
// The walk is at most t steps, since a parent comes before its children.
__global__ void __launch_bounds__(256) tree_mask_kernel(const int32_t* parents, uint8_t* mask,
                                                        int64_t nodes, int s, int* err) {
  const int lane = threadIdx.x & 31;
  const int64_t node = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (node >= nodes) return;
  const int t = (int)(node % s);
  const int32_t* par = parents + (node - t);
  uint8_t* row = mask + node * s;
  for (int j = lane; j < s; j += 32) row[j] = 0;
  __syncwarp();
  if (lane == 0) {
    int at = t;
    while (at >= 0) {
      row[at] = 1;
      const int up = par[at];
      if (up >= at || up < -1) {  // not a tree in topological order
        raise_dev_error(err, QCAU_DEVERR_INDEX);
        break;
      }
      at = up;
    }
  }
}

// ---------------------------------------------------------------- selection

constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;

// Order-preserving unsigned key of a weight sum: larger sum, larger key; -0
// equals +0, NaN is above +infinity.  0 and 0xffffffff belong to no sum.
__device__ __forceinline__ uint32_t sum_key(float x) {
  if (x != x) return 0xfffffffeu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int kBins = 2048;

struct SelShared {
  int hist[3][kBins];            // one per digit, all cleared at the start
  uint32_t count[32 * kSelWarps];  // kept-token counts per (j, warp): above the bar | at it << 16
  uint32_t scan[2][kSelWarps];
  int pick[3];
  uint32_t total;                // this block's kept-token counts, packed as `count`
};

// Word of the same shared variable in block `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_u32(const void* p, int rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ int2 peer_int2(const void* p, int rank) {
  int2 v;
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];"
               : "=r"(v.x), "=r"(v.y)
               : "r"(mapa_shared(smem_u32(p), rank))
               : "memory");
  return v;
}

__device__ __forceinline__ void select_clear(SelShared* sh) {
  for (int i = threadIdx.x; i < 3 * kBins; i += kSelThreads) (&sh->hist[0][0])[i] = 0;
}

struct Bar {
  uint32_t key;  // tokens above it are kept,
  bool tied;     // and as many at it as still fit (false: none)
};

// The bar that `budget` of more keys than that pass: three
// digits of 11, 11 and 10 bits from the top, a histogram of the keys that share
// the digits so far, and the bin that holds the budget-th key.  A bin that ends
// exactly there ends the search.  visit(f) calls f(key) for each of the thread's
// keys (0: none).  Starts behind select_clear and a barrier; a digit costs three
// barriers, which is most of its time after the first.  The `blocks` blocks of a
// cluster add up their histograms, each for itself.
template <typename Visit>
__device__ __forceinline__ Bar select_bar(SelShared* sh, int budget, int blocks, Visit visit) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t prefix = 0, known = 0;
  int want = budget;
#pragma unroll 1
  for (int digit = 0; digit < 3; digit++) {
    const int width = digit < 2 ? 11 : 10, shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
    int* hist = sh->hist[digit];
    visit([&](uint32_t k) {
      if (k != 0 && (k & known) == prefix)
        atomicAdd(&hist[(k >> shift) & ((1u << width) - 1u)], 1);
    });
    // thread i owns bins 2047 - 2i and 2046 - 2i
    int h0 = 0, h1 = 0;
    if (blocks > 1) {
      cluster_sync();
      for (int r = 0; r < blocks; r++) {
        const int2 h = peer_int2(&hist[kBins - 2 - 2 * tid], r);
        h0 += h.y;
        h1 += h.x;
      }
    } else {
      __syncthreads();
      const int2 h = *reinterpret_cast<const int2*>(&hist[kBins - 2 - 2 * tid]);
      h0 = h.y;
      h1 = h.x;
    }
    int inc = h0 + h1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    if (lane == 31) sh->scan[digit & 1][warp] = inc;
    __syncthreads();
    const int above = (int)__reduce_add_sync(0xffffffffu, lane < warp ? sh->scan[digit & 1][lane] : 0u) +
                      inc - h0 - h1;
    if (above < want && want <= above + h0 + h1) {
      const bool second = want > above + h0;
      sh->pick[0] = kBins - 1 - 2 * tid - (second ? 1 : 0);
      sh->pick[1] = above + (second ? h0 : 0);
      sh->pick[2] = above + h0 + (second ? h1 : 0);
    }
    __syncthreads();
    prefix |= (uint32_t)sh->pick[0] << shift;
    known |= ((1u << width) - 1u) << shift;
    if (sh->pick[2] == want) return {prefix - 1, false};
    want -= sh->pick[1];
  }
  return {prefix, true};
}

// A cluster of `blocks` blocks per sequence, its keys in registers: value j of
// thread i of block r is token (r V + j) * 1024 + i.  One read of the sums (all
// loads in flight at once, past the length they read the last sum again);
// select_bar works on the registers and shared-memory histograms (kCluster: more than
// one block); then each kept
// token's place is the number of kept tokens before it, from ballots, one scan over
// (j, warp) and the totals of the blocks before.  Bound by the instructions of one
// SM (16384 sums in one block: 10 us) and, split further, by latencies.
template <int V, bool kCluster>
__global__ void __launch_bounds__(kSelThreads)
    evict_select_kernel(qcau_select_args p, int cluster, int* err) {
  const int blocks = kCluster ? cluster : 1;
  __shared__ __align__(16) SelShared shared;
  SelShared* sh = &shared;
  select_clear(sh);
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();  // the move of the rows may be launched; it waits
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.x / blocks, rank = blockIdx.x % blocks;
  const int max_len = (int)p.max_seqlen, budget = (int)p.budget;
  const int n_first = (int)p.n_first, n_recent = (int)p.n_recent;
  const int token0 = rank * V * kSelThreads + tid;
  int len = p.seqlens[b];
  const float* src = p.sums + b * p.sums_stride;
  float x[V];
#pragma unroll
  for (int j = 0; j < V; j++) x[j] = src[min(token0 + j * kSelThreads, max_len - 1)];
  if (len < 0 || len > max_len) {
    if (tid == 0) raise_dev_error(err, QCAU_DEVERR_INDEX);
    len = min(max(len, 0), max_len);
  }
  // the always-kept tokens rank above every sum
  uint32_t key[V];
#pragma unroll
  for (int j = 0; j < V; j++) {
    const int i = token0 + j * kSelThreads;
    key[j] = i >= len ? 0u : i < n_first || i >= len - n_recent ? 0xffffffffu : sum_key(x[j]);
  }
  const int count = min(len, budget);
  Bar bar = {1, false};  // every token's key is above it
  __syncthreads();
  if (len > budget)  // the same in all blocks of the cluster
    bar = select_bar(sh, budget, blocks, [&](auto f) {
#pragma unroll
      for (int j = 0; j < V; j++) f(key[j]);
    });
  // tokens above the bar and at it, per (j, warp)
#pragma unroll
  for (int j = 0; j < V; j++) {
    const unsigned g = __ballot_sync(0xffffffffu, key[j] > bar.key);
    const unsigned e = bar.tied ? __ballot_sync(0xffffffffu, key[j] == bar.key) : 0;
    if (lane == 0) sh->count[j * kSelWarps + warp] = __popc(g) | __popc(e) << 16;
  }
  __syncthreads();
  // exclusive prefix sums over the V * 32 entries in token order, both counts at
  // once (at most 32768 tokens: no carry between the halves)
  const uint32_t mine = tid < V * kSelWarps ? sh->count[tid] : 0u;
  uint32_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) sh->scan[0][warp] = inc;
  __syncthreads();
  const uint32_t sums = sh->scan[0][lane];
  const uint32_t total = __reduce_add_sync(0xffffffffu, sums);
  if (tid < V * kSelWarps)
    sh->count[tid] = inc - mine + __reduce_add_sync(0xffffffffu, lane < warp ? sums : 0u);
  int total_gt = (int)(total & 0xffffu), prior_gt = 0, prior_eq = 0;
  // behind the barrier all sums of this sequence are read: sums_out may be sums
  if (blocks > 1) {
    if (tid == 0) sh->total = total;
    cluster_sync();
    total_gt = 0;
    for (int r = 0; r < blocks; r++) {
      const uint32_t t = peer_u32(&sh->total, r);
      total_gt += (int)(t & 0xffffu);
      if (r < rank) {
        prior_gt += (int)(t & 0xffffu);
        prior_eq += (int)(t >> 16);
      }
    }
    cluster_arrive();  // no block leaves while another reads its shared memory
  } else {
    __syncthreads();
  }
  const int ties = count - total_gt;  // of the tokens at the bar, the first ones
  int32_t* kp = p.keep + (int64_t)b * budget;
  float* out = p.sums_out ? p.sums_out + b * p.out_stride : nullptr;
#pragma unroll
  for (int j = 0; j < V; j++) {
    const uint32_t k = key[j], before = sh->count[j * kSelWarps + warp];
    const unsigned g = __ballot_sync(0xffffffffu, k > bar.key);
    const unsigned lt = (1u << lane) - 1u;
    int pos = prior_gt + (int)(before & 0xffffu) + __popc(g & lt);
    bool kept = k > bar.key;
    if (bar.tied) {
      const unsigned e = __ballot_sync(0xffffffffu, k == bar.key);
      const int before_eq = prior_eq + (int)(before >> 16) + __popc(e & lt);
      pos += min(before_eq, ties);
      kept = kept || (k == bar.key && before_eq < ties);
    }
    if (kept) {
      kp[pos] = token0 + j * kSelThreads;
      if (out) out[pos] = x[j];
    }
  }
  const int step = blocks * kSelThreads, at = rank * kSelThreads + tid;
  for (int i = count + at; i < budget; i += step) kp[i] = -1;
  if (out)
    for (int i = count + at; i < max_len; i += step) out[i] = 0.f;
  if (at == 0) p.counts[b] = count;
  if (blocks > 1) cluster_wait();
}

// Sequences longer than the registers hold: the sums are read again (from L2) for
// each digit, and the kept tokens are written chunk by chunk in token order, so
// that sums_out may be sums here too (a token moves to its own place or an
// earlier one).
__global__ void __launch_bounds__(kSelThreads)
    evict_select_long_kernel(qcau_select_args p, int* err) {
  __shared__ __align__(16) SelShared shared;
  SelShared* sh = &shared;
  select_clear(sh);
  __syncthreads();
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
  const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int max_len = (int)p.max_seqlen, budget = (int)p.budget;
  const int n_first = (int)p.n_first, n_recent = (int)p.n_recent;
  int len = p.seqlens[b];
  if (len < 0 || len > max_len) {
    if (tid == 0) raise_dev_error(err, QCAU_DEVERR_INDEX);
    len = min(max(len, 0), max_len);
  }
  const float* src = p.sums + b * p.sums_stride;
  const int count = min(len, budget);
  auto rank_key = [&](int i, float x) {
    return i < n_first || i >= len - n_recent ? 0xffffffffu : sum_key(x);
  };
  uint32_t bar = 1;
  int total_gt = len;  // tokens above the bar
  if (len > budget) {
    bar = select_bar(sh, budget, 1, [&](auto f) {
#pragma unroll 8
      for (int i = tid; i < len; i += kSelThreads) f(rank_key(i, src[i]));
    }).key;  // (not tied: as many are above it as are kept)
    int n = 0;
#pragma unroll 8
    for (int i = tid; i < len; i += kSelThreads) n += rank_key(i, src[i]) > bar;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) sh->scan[1][warp] = n;
    __syncthreads();
    total_gt = (int)__reduce_add_sync(0xffffffffu, sh->scan[1][lane]);
    __syncthreads();
  }
  const int ties = count - total_gt;
  int32_t* kp = p.keep + (int64_t)b * budget;
  float* out = p.sums_out ? p.sums_out + b * p.out_stride : nullptr;
  int done_gt = 0, done_eq = 0;
  for (int i0 = 0; i0 < len; i0 += kSelThreads) {
    const int i = i0 + tid;
    const float x = i < len ? src[i] : 0.f;
    const uint32_t k = i < len ? rank_key(i, x) : 0u;
    const unsigned bg = __ballot_sync(0xffffffffu, k > bar), be = __ballot_sync(0xffffffffu, k == bar);
    if (lane == 0) {
      sh->scan[0][warp] = __popc(bg);
      sh->scan[1][warp] = __popc(be);
    }
    __syncthreads();  // the chunk is read before any of it is overwritten
    const int sg = sh->scan[0][lane], se = sh->scan[1][lane];
    const unsigned lt = (1u << lane) - 1u;
    const int before_eq = done_eq + __reduce_add_sync(0xffffffffu, lane < warp ? se : 0) + __popc(be & lt);
    const int pos = done_gt + __reduce_add_sync(0xffffffffu, lane < warp ? sg : 0) + __popc(bg & lt) +
                    min(before_eq, ties);
    if (k > bar || (k == bar && before_eq < ties)) {
      kp[pos] = i;
      if (out) out[pos] = x;
    }
    done_gt += __reduce_add_sync(0xffffffffu, sg);
    done_eq += __reduce_add_sync(0xffffffffu, se);
    __syncthreads();  // the counts are read before the next chunk's are written
  }
  for (int i = count + tid; i < budget; i += kSelThreads) kp[i] = -1;
  if (out)
    for (int i = count + tid; i < max_len; i += kSelThreads) out[i] = 0.f;
  if (tid == 0) p.counts[b] = count;
}

// ---------------------------------------------------------------- row moves

constexpr int kKeepThreads = 256;
constexpr int kKeepLoads = 8;  // 16-byte loads in flight per thread
constexpr int64_t kKeepSlots = 4 * 148;  // blocks that run at once

// Where the rows of sequence b go, and how many; refused: not within the block table.
struct KeepRange {
  int start, count;
  bool refused;
};
__device__ __forceinline__ KeepRange keep_range(const qcau_keep_args& p, int b) {
  KeepRange r;
  r.start = p.start ? p.start[b] : 0;
  r.count = p.counts[b];
  const int room = (int)(p.dst_max_pages * p.page_size);
  r.refused = r.count < 0 || r.count > p.k || r.start < 0 || r.start > room - r.count;
  return r;
}

// A cluster of `spread` blocks moves one column slice of UNITS x 16 bytes (0:
// whole rows) of all kept rows of sequence b, in order, spread x some rows a turn:
// keep is strictly ascending, so row start + i comes from itself or from a later
// row, and a turn overwrites only rows that this turn or an earlier one has read.
// So the move is in place with one barrier a turn (between a turn's loads and its
// stores), needs no other buffer, and clusters never wait for one another.  The
// addresses (two dependent table lookups) are made while the turn before is read,
// and four blocks an SM overlap one another's loads and stores (turns double-
// buffered in registers, at two blocks an SM, took 92 us for 33 x 4096 rows of 576
// values against 62, and 14 against 9 for 8192 rows of one sequence).  Bound by
// HBM: 4 d bytes a row moved (32 x 4096 rows: 60 us, 5.0 TB/s; 128 x 1024: 57 us, 5.3;
// random or consecutive rows, in place or not).
template <int UNITS>
__global__ void __launch_bounds__(kKeepThreads, UNITS ? 4 : 1) keep_rows_kernel(qcau_keep_args p, int spread, int* err) {
  constexpr int U = kKeepLoads;
  constexpr int kMaxRows = UNITS ? kKeepThreads * U / UNITS : 128;
  __shared__ int from[2][kMaxRows], to[2][kMaxRows];  // cache rows, or -1
  cudaGridDependencySynchronize();
  const int b = blockIdx.y, tid = threadIdx.x;
  const int row_units = (int)(p.d / 8);
  const int units = UNITS ? UNITS : row_units;             // of this block's slice
  const int rows = UNITS ? kMaxRows : min(kMaxRows, kKeepThreads * U / row_units);  // a turn
  const int unit0 = UNITS ? blockIdx.x / spread * UNITS : 0;
  const int share = blockIdx.x % spread;  // this block's rows of a turn
  const KeepRange range = keep_range(p, b);
  const int start = range.start, count = range.refused ? 0 : range.count;
  const int page = (int)p.page_size, room = (int)(p.max_pages * p.page_size);
  bool bad = range.refused;
  const int32_t* keep = p.keep + b * p.keep_stride;
  const int32_t* stab = p.block_table + b * p.max_pages;
  const int32_t* dtab = p.dst_table + b * p.dst_max_pages;
  const bool same = p.cache == p.dst_cache && p.block_table == p.dst_table;
  // the addresses of a turn's rows: both lookups of all of a thread's rows at a time
  constexpr int kPlaces = (kMaxRows + kKeepThreads - 1) / kKeepThreads;
  auto place = [&](int turn) {
    const int i0 = (turn * spread + share) * rows;
    int k[kPlaces], before[kPlaces], f[kPlaces], t[kPlaces], f_at[kPlaces], t_at[kPlaces];
#pragma unroll
    for (int j = 0; j < kPlaces; j++) {
      const int r = tid + j * kKeepThreads, i = i0 + r;
      const bool live = r < rows && i < count;
      k[j] = live ? keep[i] : -1;
      before[j] = live && i > 0 ? keep[i - 1] : -1;
    }
#pragma unroll
    for (int j = 0; j < kPlaces; j++) {
      const int r = tid + j * kKeepThreads, i = i0 + r;
      f[j] = t[j] = -1;
      f_at[j] = t_at[j] = 0;
      if (r < rows && i < count) {
        // ascending: behind its predecessor, hence never before its own place
        if (k[j] < i || k[j] <= before[j] || k[j] >= room - start) {
          bad = true;
        } else if (!(same && k[j] == i)) {
          const unsigned at = start + k[j], row = start + i, fp = at / (unsigned)page, tp = row / (unsigned)page;
          f[j] = stab[fp];
          t[j] = dtab[tp];
          f_at[j] = at - fp * page;
          t_at[j] = row - tp * page;
          bad = bad || f[j] < 0 || t[j] < 0;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kPlaces; j++) {
      const int r = tid + j * kKeepThreads;
      if (f[j] >= p.num_pages || t[j] >= p.dst_num_pages) bad = true;
      const bool move = f[j] >= 0 && t[j] >= 0 && f[j] < p.num_pages && t[j] < p.dst_num_pages;
      if (r < rows) {
        from[turn & 1][r] = move ? f[j] * page + f_at[j] : -1;
        to[turn & 1][r] = move ? t[j] * page + t_at[j] : -1;
      }
    }
  };
  const uint4* src = reinterpret_cast<const uint4*>(p.cache);
  uint4* dst = reinterpret_cast<uint4*>(p.dst_cache);
  struct Turn {
    uint4 v[U];
    int t[U];
  };
  // unit u of this thread: row (u * 256 + tid) / units of the turn
  int row_of[U], unit_of[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int x = u * kKeepThreads + tid;
    row_of[u] = x / units;
    unit_of[u] = unit0 + x % units;
  }
  auto load = [&](int turn, Turn& w) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      w.t[u] = -1;
      if (row_of[u] < rows) {
        const int f = from[turn & 1][row_of[u]];
        w.t[u] = to[turn & 1][row_of[u]];
        if (f >= 0) w.v[u] = src[(int64_t)f * row_units + unit_of[u]];
      }
    }
  };
  auto store = [&](const Turn& w) {
#pragma unroll
    for (int u = 0; u < U; u++)
      if (w.t[u] >= 0) dst[(int64_t)w.t[u] * row_units + unit_of[u]] = w.v[u];
  };
  const int turns = (count + rows * spread - 1) / (rows * spread);
  auto barrier = [&]() {
    if (spread > 1)
      cluster_sync();
    else
      __syncthreads();
  };
  if (turns > 0) {
    Turn w;
    place(0);
    __syncthreads();
    for (int turn = 0; turn < turns; turn++) {
      load(turn, w);
      if (turn + 1 < turns) place(turn + 1);
      barrier();
      store(w);
    }
  }
  if (bad) raise_dev_error(err, QCAU_DEVERR_INDEX);
  if (p.lens_out && blockIdx.x == 0) {
    __syncthreads();  // start and counts, either of which lens_out may be, are read
    if (tid == 0 && !range.refused) p.lens_out[b] = start + count;
  }
}

constexpr int kSumThreads = 1024;

// The weight sums of the rows that keep_rows moves, one block a sequence: sum start +
// keep[i] to place start + i, then 0 from the last kept one to the row's end.  In place:
// keep is strictly ascending, so a chunk of i reads at or behind the places that it
// writes, and the barrier between its loads and its stores is all that is needed.
// Bound by latency at a drafting step's few nodes (1 to 3 us on top of the rows' move,
// sequences of up to 32768 positions), then by one SM's stores of zeros, 4 bytes a
// position (9 us for one of 131072, 10 for 32 of them).
__global__ void __launch_bounds__(kSumThreads)
    keep_sums_kernel(qcau_keep_args p, float* sums, int64_t stride, int64_t positions, int* err) {
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();  // the move of the rows may be launched; it waits
  const int b = blockIdx.x, tid = threadIdx.x, n = (int)positions;
  const KeepRange range = keep_range(p, b);
  if (range.refused) return;  // keep_rows raises the error
  const int start = range.start, count = range.count;
  const int32_t* keep = p.keep + b * p.keep_stride;
  float* row = sums + b * stride;
  bool bad = false;
  for (int i0 = 0; i0 < count; i0 += kSumThreads) {
    const int i = i0 + tid;
    bool move = false;
    float x = 0.f;
    if (i < count) {
      const int k = keep[i], before = i > 0 ? keep[i - 1] : -1;
      // what keep_rows moves, and within the row of sums
      move = k >= i && k > before && k < n - start;
      bad = bad || !move;
      if (move) x = row[start + k];
    }
    __syncthreads();
    if (move) row[start + i] = x;
  }
  __syncthreads();  // the sums are read: the rest may be cleared
  for (int i = start + count + tid; i < n; i += kSumThreads) row[i] = 0.f;
  if (bad) raise_dev_error(err, QCAU_DEVERR_INDEX);
}

// lens_out where it is start or counts, which all the blocks of a sequence read.
__global__ void __launch_bounds__(256) keep_lens_kernel(qcau_keep_args p) {
  cudaGridDependencySynchronize();
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b >= p.b) return;
  const KeepRange r = keep_range(p, b);
  if (!r.refused) p.lens_out[b] = r.start + r.count;
}

}  // namespace

cudaError_t launch_tree_mask(const int32_t* parents, uint8_t* mask, int64_t b, int64_t s,
                             cudaStream_t st) {
  tree_mask_kernel<<<(unsigned)((b * s + 7) / 8), 256, 0, st>>>(parents, mask, b * s, (int)s,
                                                               device_error_word());
  return cudaGetLastError();
}

cudaError_t launch_evict_select(const qcau_select_args& a, cudaStream_t st) {
  int* err = device_error_word();
  // one block up to 8192 sums (7.5 us against 7.8 in two); then clusters of up to 8
  // blocks of 4096, one block per SM in all (one sequence of 16384: 8.5 us, 11.1 in one
  // block; of 32768: 11.6, 23.1); fuller ones for more sequences or longer ones (of
  // 131072: 17.3 us, 174 where the sums are read again for each digit)
  int64_t blocks = 1;
  if (a.max_seqlen > 8 * kSelThreads)
    while (blocks < 8 && blocks * 4 * kSelThreads < a.max_seqlen && 2 * blocks * a.b <= 148) blocks *= 2;
  while (blocks < 8 && blocks * 32 * kSelThreads < a.max_seqlen) blocks *= 2;
  const int64_t values = (a.max_seqlen + blocks * kSelThreads - 1) / (blocks * kSelThreads);
  auto run = [&](auto single, auto clustered) {
    return launch_early(blocks > 1 ? clustered : single, dim3((unsigned)(a.b * blocks)),
                        (unsigned)blocks, kSelThreads, 0, st, a, (int)blocks, err);
  };
  if (values <= 4) return run(evict_select_kernel<4, false>, evict_select_kernel<4, true>);
  if (values <= 8) return run(evict_select_kernel<8, false>, evict_select_kernel<8, true>);
  if (values <= 16) return run(evict_select_kernel<16, false>, evict_select_kernel<16, true>);
  if (values <= 32) return run(evict_select_kernel<32, false>, evict_select_kernel<32, true>);
  return launch_early(evict_select_long_kernel, dim3((unsigned)a.b), 1, kSelThreads, 0, st, a, err);
}

cudaError_t launch_keep_sums(const qcau_keep_args& a, float* sums, int64_t stride, int64_t positions,
                             cudaStream_t st) {
  return launch_early(keep_sums_kernel, dim3((unsigned)a.b), 1, kSumThreads, 0, st, a, sums, stride, positions,
                      device_error_word());
}

cudaError_t launch_keep_rows(const qcau_keep_args& a, cudaStream_t st) {
  int* err = device_error_word();
  const int64_t units = a.d / 8;  // 16-byte units of a row
  const bool late = a.lens_out && (a.lens_out == a.start || a.lens_out == a.counts);
  auto run = [&](auto kernel, int64_t slices, int64_t spread) {
    const bool two = late && slices * spread > 1;
    qcau_keep_args rows = a;
    if (two) rows.lens_out = nullptr;
    cudaError_t e = launch_early(kernel, dim3((unsigned)(slices * spread), (unsigned)a.b), (unsigned)spread,
                                 kKeepThreads, 0, st, rows, (int)spread, err);
    if (e != cudaSuccess || !two) return e;
    return launch_early(keep_lens_kernel, dim3((unsigned)((a.b + 255) / 256)), 1, 256, 0, st, a);
  };
  // few rows (a commit): a block takes whole rows, up to 28 of 576 values a turn
  if (a.k <= 64 && units <= kKeepThreads) return run(keep_rows_kernel<0>, 1, 1);
  // Slices of 128 bytes or narrower (down to a 32-byte sector), in clusters of up to
  // 8 blocks: the pair with the least estimated time (us) from B200 timings of 1 to
  // 128 sequences: waves of four blocks per SM, each 6 us of set-up (2 more in a
  // cluster) and 2 us a turn; and not below the bytes at 5.4 TB/s (less in fewer than
  // 360 blocks, a quarter more time in slices under 128 bytes) and a last wave.
  const double bytes_us = (double)a.b * (double)a.k * (double)a.d * 4 / 5.4e6;
  int64_t width = 0, spread = 1;
  double best = 1e300;
  for (int64_t w = 8; w >= 2; w /= 2) {
    if (units % w) continue;
    const int64_t turns = (a.k * w + kKeepThreads * kKeepLoads - 1) / (kKeepThreads * kKeepLoads);
    for (int64_t n = 1; n <= 8 && n <= turns; n++) {
      const int64_t blocks = a.b * (units / w) * n, waves = (blocks + kKeepSlots - 1) / kKeepSlots;
      const double wave = 6 + (n > 1 ? 2 : 0) + 2.0 * (double)((turns + n - 1) / n);
      const double us = std::max((double)waves * wave,
                                 bytes_us * (w == 8 ? 1.0 : 1.25) *
                                         std::sqrt(std::max(1.0, 360.0 / (double)blocks)) +
                                     (waves > 1 ? wave : 0.0));
      if (us < best) {
        best = us;
        width = w;
        spread = n;
      }
    }
  }
  if (width == 8) return run(keep_rows_kernel<8>, units / 8, spread);
  if (width == 4) return run(keep_rows_kernel<4>, units / 4, spread);
  return run(keep_rows_kernel<2>, units / 2, spread);
}

}  // namespace qcau
