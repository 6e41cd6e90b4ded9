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
// 32 sequences x up to 8 nodes x 128 heads, ragged: 132.6 us with 0, 126.6 with 1,
// 124.7 with 2, 124.8 with 3.
constexpr int kTreeRowCost = 2;

// The tensor core truncates an accumulator to fp32 at every MMA step, towards
// zero: scores come out short by a share that grows with the steps of their chain.
// Measured (slope of a score's error over the score, sequences of one token, 64 scales;
// per step): queries independent of their token 0.95e-8 in chains of 9 steps, 1.1e-8 of
// 18, 1.26e-8 of 32 and 36; queries that lean towards it, whose large scores carry a
// softmax, 1.68e-8 in all of them.  The softmax scale takes a value between the two
// back, which leaves a third or less.  It is a mean: a score whose partial sums cancel
// lost nothing in proportion to itself, and is moved by it all the same (under 5e-7 of
// the score).
constexpr double kTruncPerStep = 1.35e-8;

// What a score q . k is multiplied by: softmax scale x log2(e), with the mean share back
// that it lost in chains of `steps` MMAs of 16 dims (the last one shorter where d / 16 is
// no multiple).  Of chains that a score is the sum of, each lost by its own steps of its
// own share, steps over all steps: their mean is that of the squares.  In 64 bits,
// rounded once: the shares are a few ulps of the scale.
inline float tree_score_scale(float scale, double log2e, int64_t d_qk, int steps) {
  const int64_t all = d_qk / 16, rest = all % steps;
  const double mean = (double)(all / steps * steps * steps + rest * rest) / (double)all;
  return (float)((double)scale * log2e * (1.0 + kTruncPerStep * mean));
}

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
  TreeSeq q;     // the current sequence
  int x, x_end;
  int extra;     // places in front of a row's tiles
  int group;     // team schedule: this pair's group; else -1
};

struct TreeRange {
  TreeCursor start;
  int nranges, range, total;
  int tsize;  // pairs between a range and the next one of the same group
};

struct TreePlanShared {  // batches of more than 32 sequences
  int4 sums[8];              // per warp (up to 8): tiles of all rows, of all sequences; rows, sequences
  int scan[8];               // per warp: places of a run of sequences
  int start_b, start_first;  // first sequence of the range, and its first place
  TreeSeq start;
};

template <typename Cut>
__device__ __forceinline__ bool tree_piece(const TreeShape& p, TreeCursor& c, TreePiece& u) {
  while (c.x < c.x_end && c.b < p.b) {
    u.q = c.q;
    const int rows = c.group >= 0 ? 1 : u.q.groups, places = u.q.tiles + c.extra;
    if (u.q.tiles == 0 || c.x >= c.first + places * rows) {
      c.first += u.q.tiles == 0 ? 0 : places * rows;
      if (++c.b < p.b) c.q = tree_seq<Cut>(p, c.b);
      continue;
    }
    const int k = rows == 1 ? 0 : (int)((unsigned)(c.x - c.first) / (unsigned)places);
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

// floor(x / n) of small numbers, n <= kTreePairs and x < 2^14: (x + 1/2) / n is at
// least 1/148 from an integer, far more than its rounding.
__device__ __forceinline__ int tree_div_small(int x, float inv_n) {
  return (int)(((float)x + 0.5f) * inv_n);
}

// First place of range i: floor(i total / nranges), in 32 bits (nranges is small).
__device__ __forceinline__ int tree_cut(int total, int nranges, int i) {
  const int q = (unsigned)total / (unsigned)nranges, rem = total - q * nranges;
  return i * q + tree_div_small(i * rem, __fdividef(1.f, (float)nranges));
}

// The range that place x belongs to: the largest i with tree_cut(i) <= x.
__device__ __forceinline__ int tree_range_of(const TreeRange& r, int x) {
  // off by one at most
  int i = min((int)((float)x * (float)r.nranges / (float)r.total), r.nranges - 1);
  if (tree_cut(r.total, r.nranges, i) > x) return i - 1;
  if (i + 1 < r.nranges && tree_cut(r.total, r.nranges, i + 1) <= x) i++;
  return i;
}

// The cut of a batch of `rows` tiles (of `seqs` sequences' tiles; nrows rows of nseqs
// sequences that have tiles): this pair's range, but for its first sequence.
__device__ __forceinline__ TreeRange tree_plan_cut(const TreeShape& p, int rows, int seqs, int nrows, int nseqs,
                                                   int pair, int npairs) {
  TreeRange r;
  // a team runs every group on every sequence's tiles: not worth it where the
  // trees' own sizes leave a tenth of them empty
  const bool team = p.team && (int64_t)rows * 10 >= (int64_t)seqs * p.groups * 9;
  r.tsize = team ? p.groups : 1;
  r.total = team ? seqs : rows;
  r.range = team ? pair / p.groups : pair;
  r.start.group = team ? pair - r.range * p.groups : -1;
  r.nranges = max(1, min(team ? npairs / p.groups : npairs, r.total));
  // ranges of 8 tiles or more: the rows' starts count too
  const int extra = r.total >= 8 * r.nranges ? p.row_cost : 0;
  r.total += extra * (team ? nseqs : nrows);
  r.start.extra = extra;
  const bool busy = r.range < r.nranges;
  r.start.x = busy ? tree_cut(r.total, r.nranges, r.range) : 0;
  r.start.x_end = busy ? tree_cut(r.total, r.nranges, r.range + 1) : 0;
  return r;
}

// Places of a sequence in the list.
__device__ __forceinline__ int tree_places(const TreeRange& r, const TreeSeq& q) {
  return q.tiles > 0 ? (q.tiles + r.start.extra) * (r.start.group >= 0 ? 1 : q.groups) : 0;
}

__device__ __forceinline__ int warp_scan(int x) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, x, o);
    if ((threadIdx.x & 31) >= o) x += v;
  }
  return x;
}

// This pair's range (all threads of the CTA).  Every CTA sums the same lengths, so
// all take one plan.
//
// A short call waits for the plan alone, so it goes without what can be spared:
// divisions (a handful of them was half a microsecond), a second read of the
// lengths and, up to 32 sequences, barriers: each warp plans for itself (a tree of one
// sequence 13.8 -> 13.4 us, weight sums of one 6.1 -> 5.9).
template <typename Cut>
__device__ __forceinline__ TreeRange tree_plan(const TreeShape& p, TreePlanShared* sh, int pair, int npairs) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nwarps = blockDim.x >> 5;
  if (p.b <= 32) {
    TreeSeq q{};
    if (lane < p.b) q = tree_seq<Cut>(p, lane);
    const int rows = __reduce_add_sync(0xffffffffu, q.tiles * q.groups);
    const int seqs = __reduce_add_sync(0xffffffffu, q.tiles);
    const int nrows = __reduce_add_sync(0xffffffffu, q.groups);
    TreeRange r = tree_plan_cut(p, rows, seqs, nrows, __popc(__ballot_sync(0xffffffffu, q.tiles > 0)), pair, npairs);
    const int w = tree_places(r, q), lo = p.b > 1 ? warp_scan(w) - w : 0;
    const unsigned at = __ballot_sync(0xffffffffu, lo <= r.start.x && r.start.x < lo + w);
    const int i = at ? __ffs(at) - 1 : 0;
    r.start.b = at ? i : p.b;
    r.start.first = __shfl_sync(0xffffffffu, lo, i);
    r.start.q.len = __shfl_sync(0xffffffffu, q.len, i);
    r.start.q.n = __shfl_sync(0xffffffffu, q.n, i);
    r.start.q.tiles = __shfl_sync(0xffffffffu, q.tiles, i);
    r.start.q.groups = __shfl_sync(0xffffffffu, q.groups, i);
    return r;
  }
  int rows = 0, seqs = 0, nrows = 0, nseqs = 0;
  for (int i = tid; i < p.b; i += blockDim.x) {
    const TreeSeq q = tree_seq<Cut>(p, i);
    rows += q.tiles * q.groups;
    seqs += q.tiles;
    nrows += q.groups;
    nseqs += q.tiles > 0 ? 1 : 0;
  }
  rows = __reduce_add_sync(0xffffffffu, rows);
  seqs = __reduce_add_sync(0xffffffffu, seqs);
  nrows = __reduce_add_sync(0xffffffffu, nrows);
  nseqs = __reduce_add_sync(0xffffffffu, nseqs);
  if (lane == 0) sh->sums[warp] = make_int4(rows, seqs, nrows, nseqs);
  if (tid == 0) {
    sh->start_b = p.b;
    sh->start_first = 0;
    sh->start = TreeSeq{};
  }
  __syncthreads();
  rows = seqs = nrows = nseqs = 0;
  for (int w = 0; w < nwarps; w++) {
    rows += sh->sums[w].x;
    seqs += sh->sums[w].y;
    nrows += sh->sums[w].z;
    nseqs += sh->sums[w].w;
  }
  TreeRange r = tree_plan_cut(p, rows, seqs, nrows, nseqs, pair, npairs);
  // the sequence that place start.x belongs to: prefix sums of a block's worth of sequences
  int before = 0;
  for (int b0 = 0; b0 < p.b; b0 += blockDim.x) {
    const int i = b0 + tid;
    TreeSeq q{};
    if (i < p.b) q = tree_seq<Cut>(p, i);
    const int w = tree_places(r, q), inc = warp_scan(w);
    if (lane == 31) sh->scan[warp] = inc;
    __syncthreads();
    int prior = before, all = before;
    for (int k = 0; k < nwarps; k++) {
      if (k < warp) prior += sh->scan[k];
      all += sh->scan[k];
    }
    const int lo = prior + inc - w;
    if (lo <= r.start.x && r.start.x < lo + w) {
      sh->start_b = i;
      sh->start_first = lo;
      sh->start = q;
    }
    __syncthreads();
    before = all;
    if (before > r.start.x) break;
  }
  r.start.b = sh->start_b;
  r.start.first = sh->start_first;
  r.start.q = sh->start;
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
