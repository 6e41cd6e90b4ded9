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
#include <algorithm>

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

__device__ __forceinline__ float key_sum(uint32_t k) {
  return __uint_as_float(k == 0xfffffffeu ? 0x7fc00000u : k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct SelShared {
  int part[2][3][kSelWarps];  // per warp: counts of a step's three candidates
  int gt[32 * kSelWarps], eq[32 * kSelWarps];
  int scan[2][kSelWarps];
};

// One block per sequence, its keys in registers: value j of thread i is token
// j * 1024 + i.  The budget-th largest key is built from the top, two bits a
// step (three counts, one barrier), and as soon as exactly `budget` keys reach
// the candidate the search ends: the rest of the bits cannot change the set.  A
// step costs a few compares a value and one block-wide sum, so the time is that of
// the loads plus about a microsecond; a histogram per digit reads no more but
// serialises on the few leading digits that positive sums share.  Then each
// kept token's place is the number of kept tokens before it, from ballots and
// one scan over (j, warp).
template <int V>
__global__ void __launch_bounds__(kSelThreads)
    evict_select_kernel(const float* sums, int64_t sums_stride, const int32_t* seqlens,
                        int32_t* keep, int32_t* counts, float* sums_out, int64_t out_stride,
                        int max_len, int budget, int n_first, int n_recent, int* err) {
  extern __shared__ uint8_t smem_raw[];
  SelShared* sh = reinterpret_cast<SelShared*>(smem_raw);
  const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int len = seqlens[b];
  if (len < 0 || len > max_len) {
    if (tid == 0) raise_dev_error(err, QCAU_DEVERR_INDEX);
    len = min(max(len, 0), max_len);
  }
  const float* src = sums + b * sums_stride;
  uint32_t key[V];
#pragma unroll
  for (int j = 0; j < V; j++) {
    const int i = j * kSelThreads + tid;
    key[j] = i < len ? sum_key(src[i]) : 0u;
  }
  const int count = min(len, budget);
  // the always-kept tokens rank above every sum
  auto rank_key = [&](int j) {
    const int i = j * kSelThreads + tid;
    return i < len && (i < n_first || i >= len - n_recent) ? 0xffffffffu : key[j];
  };
  uint32_t bar = 1;  // every token has a key of at least 1
  if (len > budget) {
    bar = 0;
    for (int step = 0; step < 16; step++) {
      const int shift = 30 - 2 * step;
      int n1 = 0, n2 = 0, n3 = 0;
      const uint32_t c1 = bar | (1u << shift), c2 = bar | (2u << shift), c3 = bar | (3u << shift);
#pragma unroll
      for (int j = 0; j < V; j++) {
        const uint32_t k = rank_key(j);
        n1 += k >= c1;
        n2 += k >= c2;
        n3 += k >= c3;
      }
      n1 = __reduce_add_sync(0xffffffffu, n1);
      n2 = __reduce_add_sync(0xffffffffu, n2);
      n3 = __reduce_add_sync(0xffffffffu, n3);
      if (lane == 0) {
        sh->part[step & 1][0][warp] = n1;
        sh->part[step & 1][1][warp] = n2;
        sh->part[step & 1][2][warp] = n3;
      }
      __syncthreads();
      n1 = __reduce_add_sync(0xffffffffu, sh->part[step & 1][0][lane]);
      n2 = __reduce_add_sync(0xffffffffu, sh->part[step & 1][1][lane]);
      n3 = __reduce_add_sync(0xffffffffu, sh->part[step & 1][2][lane]);
      bar = n3 >= budget ? c3 : n2 >= budget ? c2 : n1 >= budget ? c1 : bar;
      if (n1 == budget || n2 == budget || n3 == budget) break;
    }
  }
  // tokens above the bar and at it, per (j, warp)
#pragma unroll
  for (int j = 0; j < V; j++) {
    const uint32_t k = rank_key(j);
    const unsigned g = __ballot_sync(0xffffffffu, k > bar), e = __ballot_sync(0xffffffffu, k == bar);
    if (lane == 0) {
      sh->gt[j * kSelWarps + warp] = __popc(g);
      sh->eq[j * kSelWarps + warp] = __popc(e);
    }
  }
  __syncthreads();
  // exclusive prefix sums over the V * 32 entries in token order: thread i owns
  // V / 32 (at least 1) of them
  constexpr int kPer = V * kSelWarps > kSelThreads ? V * kSelWarps / kSelThreads : 1;
  int g[kPer], e[kPer], gs = 0, es = 0;
#pragma unroll
  for (int k = 0; k < kPer; k++) {
    const int i = tid * kPer + k;
    g[k] = i < V * kSelWarps ? sh->gt[i] : 0;
    e[k] = i < V * kSelWarps ? sh->eq[i] : 0;
    gs += g[k];
    es += e[k];
  }
  int gi = gs, ei = es;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, gi, o), y = __shfl_up_sync(0xffffffffu, ei, o);
    if (lane >= o) {
      gi += x;
      ei += y;
    }
  }
  if (lane == 31) {
    sh->scan[0][warp] = gi;
    sh->scan[1][warp] = ei;
  }
  __syncthreads();
  const int sg = sh->scan[0][lane], se = sh->scan[1][lane];
  const int total_gt = __reduce_add_sync(0xffffffffu, sg);
  int gx = gi - gs + __reduce_add_sync(0xffffffffu, lane < warp ? sg : 0);
  int ex = ei - es + __reduce_add_sync(0xffffffffu, lane < warp ? se : 0);
#pragma unroll
  for (int k = 0; k < kPer; k++) {
    const int i = tid * kPer + k;
    if (i < V * kSelWarps) {
      sh->gt[i] = gx;
      sh->eq[i] = ex;
    }
    gx += g[k];
    ex += e[k];
  }
  const int ties = count - total_gt;  // of the tokens at the bar, the first ones
  __syncthreads();  // the values of this sequence are all read: sums_out may be sums
  int32_t* kp = keep + (int64_t)b * budget;
  float* out = sums_out ? sums_out + b * out_stride : nullptr;
#pragma unroll
  for (int j = 0; j < V; j++) {
    const uint32_t k = rank_key(j);
    const unsigned bg = __ballot_sync(0xffffffffu, k > bar), be = __ballot_sync(0xffffffffu, k == bar);
    const unsigned lt = (1u << lane) - 1u;
    const int before_eq = sh->eq[j * kSelWarps + warp] + __popc(be & lt);
    const int pos = sh->gt[j * kSelWarps + warp] + __popc(bg & lt) + min(before_eq, ties);
    if (k > bar || (k == bar && before_eq < ties)) {
      kp[pos] = j * kSelThreads + tid;
      if (out) out[pos] = key_sum(key[j]);
    }
  }
  for (int i = count + tid; i < budget; i += kSelThreads) kp[i] = -1;
  if (out)
    for (int i = count + tid; i < max_len; i += kSelThreads) out[i] = 0.f;
  if (tid == 0) counts[b] = count;
}

// Sequences longer than the registers hold: the keys are read again for each of
// three 11-bit digits (a shared-memory histogram, the same key and order), and
// the kept tokens are written chunk by chunk in token order, so that sums_out
// may be sums here too (a token moves to its own place or an earlier one).
constexpr int kBins = 2048;

__global__ void __launch_bounds__(kSelThreads)
    evict_select_long_kernel(const float* sums, int64_t sums_stride, const int32_t* seqlens,
                             int32_t* keep, int32_t* counts, float* sums_out, int64_t out_stride,
                             int max_len, int budget, int n_first, int n_recent, int* err) {
  __shared__ int hist[kBins];
  __shared__ int scan[2][kSelWarps];
  __shared__ int pick[2];
  const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int len = seqlens[b];
  if (len < 0 || len > max_len) {
    if (tid == 0) raise_dev_error(err, QCAU_DEVERR_INDEX);
    len = min(max(len, 0), max_len);
  }
  const float* src = sums + b * sums_stride;
  const int count = min(len, budget);
  auto rank_key = [&](int i, float x) {
    return i < n_first || i >= len - n_recent ? 0xffffffffu : sum_key(x);
  };
  uint32_t bar = 1;
  int total_gt = len;  // tokens above the bar
  if (len > budget) {
    uint32_t prefix = 0, known = 0;  // the bar's leading bits
    int want = budget;
    for (int digit = 0; digit < 3; digit++) {
      const int width = digit < 2 ? 11 : 10, shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
      for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int i0 = 0; i0 < len; i0 += kSelThreads) {
        const int i = i0 + tid;
        const uint32_t k = i < len ? rank_key(i, src[i]) : 0u;
        const bool in = i < len && (k & known) == prefix;
        // lanes with the same digit add once
        const uint32_t d = in ? (k >> shift) & ((1u << width) - 1u) : kBins;
        const unsigned same = __match_any_sync(0xffffffffu, d);
        if (in && lane == __ffs(same) - 1) atomicAdd(&hist[d], __popc(same));
      }
      __syncthreads();
      // the digit whose bin holds the want-th key from the top: thread i owns
      // bins 2047 - 2i and 2046 - 2i
      const int h0 = hist[kBins - 1 - 2 * tid], h1 = hist[kBins - 2 - 2 * tid];
      int inc = h0 + h1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
      }
      if (lane == 31) scan[0][warp] = inc;
      __syncthreads();
      const int prior = __reduce_add_sync(0xffffffffu, lane < warp ? scan[0][lane] : 0);
      const int above = prior + inc - h0 - h1;
      if (above < want && want <= above + h0 + h1) {
        const bool second = want > above + h0;
        pick[0] = kBins - 1 - 2 * tid - (second ? 1 : 0);
        pick[1] = above + (second ? h0 : 0);
      }
      __syncthreads();
      prefix |= (uint32_t)pick[0] << shift;
      known |= ((1u << width) - 1u) << shift;
      want -= pick[1];
      __syncthreads();
    }
    bar = prefix;
    total_gt = budget - want;
  }
  const int ties = count - total_gt;
  int32_t* kp = keep + (int64_t)b * budget;
  float* out = sums_out ? sums_out + b * out_stride : nullptr;
  int done_gt = 0, done_eq = 0;
  for (int i0 = 0; i0 < len; i0 += kSelThreads) {
    const int i = i0 + tid;
    const float x = i < len ? src[i] : 0.f;
    const uint32_t k = i < len ? rank_key(i, x) : 0u;
    const unsigned bg = __ballot_sync(0xffffffffu, k > bar), be = __ballot_sync(0xffffffffu, k == bar);
    if (lane == 0) {
      scan[0][warp] = __popc(bg);
      scan[1][warp] = __popc(be);
    }
    __syncthreads();  // the chunk is read before any of it is overwritten
    const int sg = scan[0][lane], se = scan[1][lane];
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
  if (tid == 0) counts[b] = count;
}

// ---------------------------------------------------------------- row moves

constexpr int kKeepThreads = 256;

// Block (slice, b) moves one column slice of UNITS x 16 bytes of all kept rows
// of sequence b, in order, `kRows` rows a turn: keep is strictly ascending, so
// row start + i comes from itself or from a later row, and a turn overwrites
// only rows that this turn or an earlier one has read.  So the move is in place
// with one barrier a turn (between a turn's loads and its stores), needs no other
// buffer, and blocks never wait for one another.  Each thread has U 16-byte loads in
// flight; the addresses of the next turn (two dependent table lookups) are made
// while this turn's rows arrive.  Bound by HBM: 4 d bytes a row moved.
template <int UNITS, int U>
__global__ void __launch_bounds__(kKeepThreads) keep_rows_kernel(KeepArgs p, int* err) {
  constexpr int kStep = kKeepThreads / UNITS;  // rows of one load
  constexpr int kRows = kStep * U;             // rows of a turn
  __shared__ int64_t from[2][kRows], to[2][kRows];  // row offsets in 16-byte units, or -1
  const int b = blockIdx.y, tid = threadIdx.x;
  const int unit = blockIdx.x * UNITS + tid % UNITS;
  const int row_units = (int)(p.d / 8);
  const int start = p.start ? p.start[b] : 0, page = (int)p.page_size;
  const int room = (int)(p.max_pages * p.page_size), dst_room = (int)(p.dst_max_pages * p.page_size);
  int count = p.counts[b];
  const bool refused = count < 0 || count > p.k || start < 0 || start > dst_room - count;
  bool bad = refused;
  if (refused) count = 0;
  const int32_t* keep = p.keep + b * p.keep_stride;
  const int32_t* stab = p.table + b * p.max_pages;
  const int32_t* dtab = p.dst_table + b * p.dst_max_pages;
  const bool same = p.cache == p.dst && p.table == p.dst_table;
  auto place = [&](int turn) {
    for (int r = tid; r < kRows; r += kKeepThreads) {
      const int i = turn * kRows + r;
      int64_t f = -1, t = -1;
      if (i < count) {
        const int k = keep[i], at = start + k, row = start + i;
        // ascending: behind its predecessor, hence never before its own place
        if (k < i || (i > 0 && k <= keep[i - 1]) || k >= room - start) {
          bad = true;
        } else if (!(same && k == i)) {
          const int64_t sp = stab[at / page], dp = dtab[row / page];
          if (sp < 0 || sp >= p.num_pages || dp < 0 || dp >= p.dst_num_pages) {
            bad = true;
          } else {
            f = (sp * page + at % page) * row_units;
            t = (dp * page + row % page) * row_units;
          }
        }
      }
      from[turn & 1][r] = f;
      to[turn & 1][r] = t;
    }
  };
  const uint4* src = reinterpret_cast<const uint4*>(p.cache);
  uint4* dst = reinterpret_cast<uint4*>(p.dst);
  const int turns = (count + kRows - 1) / kRows;
  if (turns > 0) place(0);
  __syncthreads();
  for (int turn = 0; turn < turns; turn++) {
    uint4 v[U];
    int64_t t[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int r = u * kStep + tid / UNITS;
      const int64_t f = from[turn & 1][r];
      t[u] = to[turn & 1][r];
      if (f >= 0) v[u] = src[f + unit];
    }
    if (turn + 1 < turns) place(turn + 1);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; u++)
      if (t[u] >= 0) dst[t[u] + unit] = v[u];
  }
  if (bad) raise_dev_error(err, QCAU_DEVERR_INDEX);
  if (p.lens_out && !refused && blockIdx.x == 0 && tid == 0) p.lens_out[b] = start + count;
}

}  // namespace

cudaError_t launch_tree_mask(const int32_t* parents, uint8_t* mask, int64_t b, int64_t s,
                             cudaStream_t st) {
  tree_mask_kernel<<<(unsigned)((b * s + 7) / 8), 256, 0, st>>>(parents, mask, b * s, (int)s,
                                                               device_error_word());
  return cudaGetLastError();
}

cudaError_t launch_evict_select(const float* sums, int64_t sums_stride, const int32_t* seqlens,
                                int32_t* keep, int32_t* counts, float* sums_out,
                                int64_t out_stride, int64_t b, int64_t max_len, int64_t budget,
                                int64_t n_first, int64_t n_recent, cudaStream_t st) {
  auto run = [&](auto kernel, size_t smem) {
    kernel<<<(unsigned)b, kSelThreads, smem, st>>>(sums, sums_stride, seqlens, keep, counts,
                                                  sums_out, out_stride, (int)max_len, (int)budget,
                                                  (int)n_first, (int)n_recent, device_error_word());
    return cudaGetLastError();
  };
  if (max_len <= 4 * kSelThreads) return run(evict_select_kernel<4>, sizeof(SelShared));
  if (max_len <= 16 * kSelThreads) return run(evict_select_kernel<16>, sizeof(SelShared));
  if (max_len <= 32 * kSelThreads) return run(evict_select_kernel<32>, sizeof(SelShared));
  return run(evict_select_long_kernel, 0);
}

cudaError_t launch_keep_rows(const KeepArgs& a, cudaStream_t st) {
  int* err = device_error_word();
  const int64_t units = a.d / 8;  // 16-byte units of a row
  // 128-byte slices, narrower ones (down to a 32-byte sector) while the blocks
  // leave SMs idle
  if (units % 8 == 0 && a.b * (units / 8) >= 148)
    keep_rows_kernel<8, 8><<<dim3((unsigned)(units / 8), (unsigned)a.b), kKeepThreads, 0, st>>>(a, err);
  else if (units % 4 == 0 && a.b * (units / 4) >= 148)
    keep_rows_kernel<4, 8><<<dim3((unsigned)(units / 4), (unsigned)a.b), kKeepThreads, 0, st>>>(a, err);
  else
    keep_rows_kernel<2, 8><<<dim3((unsigned)(units / 2), (unsigned)a.b), kKeepThreads, 0, st>>>(a, err);
  return cudaGetLastError();
}

}  // namespace qcau
