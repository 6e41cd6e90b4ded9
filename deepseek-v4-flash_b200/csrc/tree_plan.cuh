// tree_plan.cuh -- the lengths of a batch of draft trees over a paged cache,
// and the cut of their tiles into one range per CTA pair, shared by the tree
// attention and the attention weight sums.
//
// The query rows of a sequence (its n nodes x h heads) form groups of
// kGroupRows; a (sequence, group) row has one tile per kTile cached tokens.
// The tiles of all rows, laid end to end at the batch's own lengths (read on
// the device, so a ragged batch is balanced too), are cut into equal ranges.  In
// long ranges a row takes `row_cost` places in front of its tiles, for its Q
// load and its epilogue, which its tiles do not hide.
// In the team schedule the tiles of the sequences are cut instead, and each of
// a team's `groups` pairs runs one group over the team's range.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace qcau {

constexpr int kTreePairs = 74;  // CTA pairs of a B200 (148 SMs)
constexpr int kTreeMinTiles = 1;
// 32 sequences x up to 8 nodes x 128 heads, ragged: 132.6 us with 0, 126.6 with 1,
// 124.7 with 2, 124.8 with 3.
constexpr int kTreeRowCost = 2;

// The tensor core truncates an accumulator to fp32 at every MMA step, towards
// zero: scores come out short by a share that grows with the steps of their chain,
// half an ulp of the running sum a step on average.  Measured (16384 tokens, rows
// of standard deviations 1.7 and 4.3): 1.3e-7 of a score in chains of 9 steps,
// 2.4e-7 in chains of 18, with about as much scatter.  The softmax scale takes the
// mean back.
constexpr float kTruncPerStep = 1.35e-8f;

struct TreeShape {
  const int32_t* table;      // [b, max_pages]
  const int32_t* seqlens;    // [b], the drafted tokens included
  const int32_t* tree_lens;  // [b], or nullptr: s nodes each
  const uint8_t* mask;       // [b or 1, s, s] or nullptr (a chain)
  int* err;
  int64_t max_pages, num_pages, mask_stride;
  int b, s, h, max_len;
  int page_blocks;  // 64-token blocks of a page
  int groups;       // groups of a sequence at s nodes
  int team;         // 1: the team schedule may be used
  int min_tiles;    // tiles of a range, at least
  int row_cost;     // what starting a row costs, in tiles (long ranges only)
};

// Host side (attn_tree_sm100.cu): CTA pairs of a launch, and its shape.
int64_t tree_pairs(const TreeArgs& a, int group_rows, int tile);
TreeShape tree_shape(const TreeArgs& a, int group_rows, int64_t pairs);

// The kernel's cut of the work: rows of a group, tokens of a tile (both constants,
// so that what every role computes before its first load has no division by them).
template <int kRows, int kTokens>
struct TreeCut {
  static constexpr int kGroupRows = kRows, kTile = kTokens;
};

struct TreeSeq {
  int len, n, tiles, groups;
};

// Lengths of one sequence.  What the caller's arrays may not hold (a length
// past max_len, more nodes than tokens or than s) is cut to what they may.  A
// sequence of no tokens, an idle slot of the cache, has no nodes where none are given.
template <typename Cut>
__device__ __forceinline__ TreeSeq tree_seq(const TreeShape& p, int b) {
  TreeSeq q;
  const int len = p.seqlens[b], n = p.tree_lens ? p.tree_lens[b] : len == 0 ? 0 : p.s;
  q.len = min(max(len, 0), p.max_len);
  q.n = min(min(max(n, 0), p.s), q.len);
  if (q.len != len || q.n != n) raise_dev_error(p.err, QCAU_DEVERR_INDEX);
  q.groups = (q.n * p.h + Cut::kGroupRows - 1) / Cut::kGroupRows;
  q.tiles = q.n > 0 ? (q.len + Cut::kTile - 1) / Cut::kTile : 0;
  return q;
}

// One piece of work: tiles [t_begin, t_end) of group g of sequence b.
struct TreePiece {
  int b, g, t_begin, t_end;
  int row0;  // the place of the row's first tile in the list of all rows
  TreeSeq q;
};

// A pair's walk over its range of places [x, x_end).  Every role of the pair
// takes the same walk.
struct TreeCursor {
  int b, first;  // current sequence and its first place in the list
  int x, x_end;
  int extra;     // places in front of a row's tiles
  int group;     // team schedule: this pair's group; else -1
};

struct TreeRange {
  TreeCursor start;
  int nranges, range, total;
  int tsize;  // pairs between a range and the next one of the same group
};

struct TreePlanShared {
  long long sum_rows[8], sum_seqs[8];  // per warp (up to 8): tiles of all rows, of all sequences
  int num_rows[8], num_seqs[8];        // per warp: rows, sequences that have tiles
  int scan[8];                         // per warp: tiles of a run of sequences
  int start_b, start_tile;             // first sequence of the range, and its first tile
};

template <typename Cut>
__device__ __forceinline__ bool tree_piece(const TreeShape& p, TreeCursor& c, TreePiece& u) {
  while (c.x < c.x_end && c.b < p.b) {
    u.q = tree_seq<Cut>(p, c.b);
    const int rows = c.group >= 0 ? 1 : u.q.groups, places = u.q.tiles + c.extra;
    if (u.q.tiles == 0 || c.x >= c.first + places * rows) {
      c.first += u.q.tiles == 0 ? 0 : places * rows;
      c.b++;
      continue;
    }
    const int k = (c.x - c.first) / places;
    u.b = c.b;
    u.g = c.group >= 0 ? c.group : k;
    u.row0 = c.first + k * places + c.extra;
    u.t_begin = max(c.x - u.row0, 0);
    u.t_end = min(u.q.tiles, c.x_end - u.row0);
    c.x = min(u.row0 + u.q.tiles, c.x_end);
    // a range that ends in front of a row's tiles leaves the row to the next one, and
    // a team's pair past the sequence's groups has nothing to do
    if (u.t_end > u.t_begin && u.g < u.q.groups) return true;
  }
  return false;
}

// First half of the plan, before a barrier of the CTA: the batch's tiles.
template <typename Cut>
__device__ __forceinline__ void tree_plan_sums(const TreeShape& p, TreePlanShared* sh) {
  long long rows = 0, seqs = 0;
  int nrows = 0, nseqs = 0;
  for (int i = threadIdx.x; i < p.b; i += blockDim.x) {
    const TreeSeq q = tree_seq<Cut>(p, i);
    rows += (long long)q.tiles * q.groups;
    seqs += q.tiles;
    nrows += q.groups;
    nseqs += q.tiles > 0 ? 1 : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    rows += __shfl_xor_sync(0xffffffffu, rows, o);
    seqs += __shfl_xor_sync(0xffffffffu, seqs, o);
  }
  nrows = __reduce_add_sync(0xffffffffu, nrows);
  nseqs = __reduce_add_sync(0xffffffffu, nseqs);
  if ((threadIdx.x & 31) == 0) {
    sh->sum_rows[threadIdx.x >> 5] = rows;
    sh->sum_seqs[threadIdx.x >> 5] = seqs;
    sh->num_rows[threadIdx.x >> 5] = nrows;
    sh->num_seqs[threadIdx.x >> 5] = nseqs;
  }
  if (threadIdx.x == 0) {
    sh->start_b = p.b;
    sh->start_tile = 0;
  }
}

// First place of range i: floor(i total / nranges), in 32 bits (nranges is small).
__device__ __forceinline__ int tree_cut(const TreeRange& r, int i) {
  const int q = r.total / r.nranges, rem = r.total - q * r.nranges;
  return i * q + i * rem / r.nranges;
}

// The range that place x belongs to: the largest i with tree_cut(i) <= x.
__device__ __forceinline__ int tree_range_of(const TreeRange& r, int x) {
  return (int)(((int64_t)(x + 1) * r.nranges - 1) / r.total);
}

// Second half, after that barrier (all threads of the CTA): this pair's range.
// Every CTA sums the same lengths, so all take one plan.
template <typename Cut>
__device__ __forceinline__ TreeRange tree_plan_range(const TreeShape& p, TreePlanShared* sh,
                                                     int pair, int npairs) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nwarps = blockDim.x >> 5;
  long long rows = 0, seqs = 0;
  int nrows = 0, nseqs = 0;
  for (int w = 0; w < nwarps; w++) {
    rows += sh->sum_rows[w];
    seqs += sh->sum_seqs[w];
    nrows += sh->num_rows[w];
    nseqs += sh->num_seqs[w];
  }
  TreeRange r;
  // a team runs every group on every sequence's tiles: not worth it where the
  // trees' own sizes leave a tenth of them empty
  const bool team = p.team && rows * 10 >= seqs * p.groups * 9;
  r.tsize = team ? p.groups : 1;
  r.total = (int)(team ? seqs : rows);
  r.nranges = max(1, min(npairs / r.tsize, r.total / p.min_tiles));
  // ranges of 8 tiles or more: the rows' starts count too
  const int extra = r.total >= 8 * r.nranges ? p.row_cost : 0;
  r.total += extra * (team ? nseqs : nrows);
  r.start.extra = extra;
  r.range = pair / r.tsize;
  const bool busy = r.range < r.nranges;
  r.start.x = busy ? tree_cut(r, r.range) : 0;
  r.start.x_end = busy ? tree_cut(r, r.range + 1) : 0;
  r.start.group = team ? pair % r.tsize : -1;
  r.start.b = 0;
  r.start.first = 0;
  if (p.b > 1) {
    // the sequence that place start.x belongs to: prefix sums of a block's worth of sequences
    int before = 0;
    for (int b0 = 0; b0 < p.b; b0 += blockDim.x) {
      const int i = b0 + threadIdx.x;
      int w = 0;
      if (i < p.b) {
        const TreeSeq q = tree_seq<Cut>(p, i);
        w = q.tiles > 0 ? (q.tiles + extra) * (team ? 1 : q.groups) : 0;
      }
      int inc = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (lane == 31) sh->scan[warp] = inc;
      __syncthreads();
      int prior = before, all = before;
      for (int k = 0; k < nwarps; k++) {
        if (k < warp) prior += sh->scan[k];
        all += sh->scan[k];
      }
      const int lo = prior + inc - w;
      if (w > 0 && lo <= r.start.x && r.start.x < lo + w) {
        sh->start_b = i;
        sh->start_tile = lo;
      }
      __syncthreads();
      before = all;
      if (before > r.start.x) break;
    }
    r.start.b = sh->start_b;
    r.start.first = sh->start_tile;
  }
  return r;
}

// Physical 64-token block of block `blk` of sequence b.  A block past the
// sequence's end holds masked tokens only: any block of the sequence does.
__device__ __forceinline__ int tree_block(const TreeShape& p, const TreePiece& u, int blk) {
  const int used = (u.q.len + 63) / 64;
  if (blk >= used) blk = used - 1;
  // pages of one block, the usual ones, need no division
  const int page = p.page_blocks == 1 ? blk : blk / p.page_blocks;
  const int64_t e = p.table[(int64_t)u.b * p.max_pages + page];
  if (e < 0 || e >= p.num_pages) {
    raise_dev_error(p.err, QCAU_DEVERR_INDEX);
    return 0;
  }
  return (int)(e * p.page_blocks + blk - page * p.page_blocks);
}

// All lanes wait; the warp agrees on the outcome (timeouts are per lane).
__device__ __forceinline__ bool tree_warp_wait(uint64_t* bar, uint32_t parity,
                                               volatile int* abort) {
  const bool ok = mbar_wait<true>(bar, parity, abort);
  return __all_sync(0xffffffffu, ok);
}

}  // namespace qcau
