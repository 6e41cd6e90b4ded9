// attn_weights_sm100.cu -- the attention weight every cached token received,
// summed over the query tokens and heads of a step (what decides which tokens a
// bounded cache keeps).  No counterpart in the reference.
//
//   w[p] = sum over the rows r = (token t, head) that see p of
//          e^(scale * q[r] . k[p] - lse[r])
// with the log-sum-exps of the attention that ran before: the scores are made
// again (2 d FLOP per row and token) rather than kept by the attention, whose
// running maximum is not final while it has them, and whose fp32 scores would
// be 512 bytes a token and 128 rows against the 1152 bytes of reading K again.
//
// The tokens are the MMAs' M and the query rows the N, resident in shared
// memory while K streams past: a token is one TMEM lane and its rows lie along
// the columns, so its sum needs no shuffles, one thread adds it up in registers
// and one thread owns the result: no atomics, the same bits each time.  A
// sequence with more rows than a group leaves one partial sum per group and
// token (4 bytes against the 2 d bytes of its K row), added in group order by
// weights_combine.
//
// Up to 128 rows (a decode step) HBM bounds it: 1152 bytes a token.  There M is
// 256 (128 tokens per CTA: two 64-token blocks) and N 64 or 128: at M = 128 and
// N = 128 a CTA reads as many operand bytes per MMA as shared memory delivers in
// its time, and the MMAs took longer than the loads (B200, 32 x 16384 tokens x
// 128 heads: 117 us, 98.6 us with a third of them).  The M operand of 128 tokens
// is two boxes of 64 tokens x 3 chunks laid out [8 rows][chunk][8 groups], which
// makes its 8-row groups 3 KB apart across both.  With more rows, N is 256
// (K is read half as often, from L2, and N = 256 needs fewer operand bytes) and
// M 128: Q takes 147 KB, and 72 KB of ring hold one 128-token tile.
//
// Schedule: tree_plan.cuh.  Warp 0 TMA producer, warp 1 TMEM allocator and MMA
// issuer (pair leader), warps 2-5 the epilogue.
// Every wait is bounded; a timeout raises QCAU_DEVERR_TIMEOUT, drains the
// copies in flight, frees TMEM and returns.
#include "common.cuh"
#include "kernels.h"
#include "tree_plan.cuh"

namespace qcau {
namespace {

constexpr int kThreads = 192;
constexpr int kBlockBox = 24576;  // 64 tokens x 3 chunks of 64 dims
constexpr int kBoxes = 3;         // stages of a tile: 9 chunks (8: the last stage ends in zeros)
constexpr float kLog2e = 1.4426950408889634f;

// N rows of a group (64, 128 or 256): half of them in each CTA's shared memory.
template <int N>
struct WeightsCfg {
  static constexpr int kBlocks = N == 256 ? 1 : 2;  // 64-token blocks per CTA and tile
  static constexpr int kTile = 128 * kBlocks;       // tokens of a pair's tile (MMA M)
  static constexpr int kStage = kBlocks * kBlockBox;
  static constexpr int kStages = 3;
  static_assert(kStages == kBoxes, "Q's thirds are released by the stages of one tile");
  static constexpr int kQChunk = N / 2 * 128;  // N/2 rows x 64 dims bf16
  static constexpr int kQBox = 3 * kQChunk;
  // TMEM: M = 128 puts a token's first N/2 columns in lanes 0-63 and the rest in
  // lanes 64-127; M = 256 all N in its one lane
  static constexpr int kCols = N == 256 ? 128 : N;
  // accumulation chains of a score (see the issuer): as many as TMEM holds twice
  static constexpr int kChains = N == 64 ? 4 : 2;
  static constexpr int kSteps = 36 / kChains;  // MMAs of 16 dims in a chain
  static constexpr uint32_t kBufCols = kChains * kCols;
  static constexpr uint32_t kTmemCols = 2 * kBufCols;
};

template <int N>
struct WeightsShared {
  uint64_t kfull[WeightsCfg<N>::kStages], kempty[WeightsCfg<N>::kStages];
  uint64_t s_full[2], s_free[2];
  uint64_t xbar[2][4];  // M = 128: halves of a token's sum handed over: 2 warp pairs x 4 buffers
  float xsum[4][64];
  // per epilogue warp: -lse * log2e of its columns, read as 16-byte vectors
  alignas(16) float neg[4][WeightsCfg<N>::kCols];
  uint32_t tmem_base;
  int abort;
  TreePlanShared plan;
};

template <int N>
constexpr size_t weights_smem() {
  using C = WeightsCfg<N>;
  return 1024 + 9 * (size_t)C::kQChunk + (size_t)C::kStages * C::kStage + sizeof(WeightsShared<N>);
}
static_assert(weights_smem<256>() <= 232448 && weights_smem<128>() <= 232448 &&
                  weights_smem<64>() <= 232448,
              "shared memory budget");

struct WeightsParams {
  TreeShape sh;      // groups of N rows
  const float* lse;  // [b, s, h]
  float* sums;       // [b, sums_stride]
  float* part;       // [groups][b][part_stride] when groups > 1
  int64_t sums_stride, part_stride;
  int accumulate, chunks;
  float score_scale;  // log2 units
};

template <int N>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    attn_weights_sm100_kernel(const __grid_constant__ CUtensorMap tm_q,
                              const __grid_constant__ CUtensorMap tm_k, WeightsParams p) {
  using C = WeightsCfg<N>;
  using Cut = TreeCut<N, C::kTile>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  uint8_t* sQ = smem_raw + pad;
  uint8_t* sK = sQ + 9 * C::kQChunk;
  WeightsShared<N>* sh = reinterpret_cast<WeightsShared<N>*>(sK + (size_t)C::kStages * C::kStage);
  volatile int* abort = &sh->abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; i++) {
      mbar_init(&sh->kfull[i], 1);
      mbar_init(&sh->kempty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&sh->s_full[i], 1);
      mbar_init(&sh->s_free[i], 8);
      for (int k = 0; k < 4; k++) mbar_init(&sh->xbar[i][k], 1);
    }
    sh->abort = 0;
    fence_barrier_init();
  }
  if (threadIdx.x == 32) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
  }
  if (warp == 1) tmem_alloc<2>(&sh->tmem_base, C::kTmemCols);
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  cudaGridDependencySynchronize();
  const TreeRange range = tree_plan<Cut>(p.sh, &sh->plan, pair, npairs);

  if (warp == 0) {
    // ------------------------------------------------ producer (both CTAs)
    if (lane == 0) {
      int last_use[C::kStages];
      for (int i = 0; i < C::kStages; i++) last_use[i] = -1;
      int n = 0;  // stages issued
      bool ok = true;
      TreeCursor c = range.start;
      TreePiece u;
      while (ok && tree_piece<Cut>(p.sh, c, u)) {
        for (int t = u.t_begin; t < u.t_end && ok; t++) {
          int blk[C::kBlocks];
#pragma unroll
          for (int j = 0; j < C::kBlocks; j++)
            blk[j] = tree_block(p.sh, u, (2 * t + (int)rank) * C::kBlocks + j);
          for (int i = 0; i < kBoxes; i++, n++) {
            const int slot = n % C::kStages, use = n / C::kStages;
            if (!(ok = mbar_wait(&sh->kempty[slot], (use & 1) ^ 1, abort))) break;
            // a piece's first tile brings its Q (rows past the sequence's: zeros) along,
            // the stage's three chunks at a time: the MMAs that freed the stage were the
            // last to read the previous piece's (a ring holds one tile)
            const bool with_q = t == u.t_begin;
            if (leader) mbar_arrive_expect_tx(&sh->kfull[slot], 2 * (C::kStage + (with_q ? C::kQBox : 0)));
            last_use[slot] = use;
            const uint32_t bar = mapa_shared(smem_u32(&sh->kfull[slot]), 0);
            if (with_q)
              tma_load_4d_pair(sQ + i * C::kQBox, &tm_q, bar, 0, u.g * N + N / 2 * (int)rank, 3 * i, u.b);
#pragma unroll
            for (int j = 0; j < C::kBlocks; j++)
              tma_load_5d_pair(sK + (size_t)slot * C::kStage + j * kBlockBox, &tm_k, bar, 0, 0, 3 * i,
                               0, blk[j]);
          }
        }
      }
      if (*abort && leader) {
        // the leader's full barriers count both CTAs' copies: drain them all
        volatile int never = 0;
        for (int i = 0; i < C::kStages; i++)
          if (last_use[i] >= 0) mbar_wait<true>(&sh->kfull[i], last_use[i] & 1, &never);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer (pair leader)
    if (leader && lane == 0) {
      const uint32_t idesc = make_idesc(C::kTile, N, kFmtBF16, kFmtBF16, false, false);
      const uint64_t k_desc = make_sdesc(smem_u32(sK), 16, 3 * 1024);
      const uint64_t q_desc = make_sdesc(smem_u32(sQ), 16, 1024);
      int n = 0, gt = 0;  // stages, tiles
      uint64_t* last_bar = nullptr;
      int last_phase = 0;
      bool ok = true;
      TreeCursor c = range.start;
      TreePiece u;
      while (ok && tree_piece<Cut>(p.sh, c, u)) {
        for (int t = u.t_begin; t < u.t_end && ok; t++, gt++) {
          const int sb = gt & 1;
          if (gt >= 2 && !(ok = mbar_wait<true>(&sh->s_free[sb], ((gt >> 1) - 1) & 1, abort)))
            break;
          tc_fence_after();
#pragma unroll
          for (int g = 0; g < kBoxes; g++, n++) {
            const int slot = n % C::kStages, use = n / C::kStages;
            if (!(ok = mbar_wait(&sh->kfull[slot], use & 1, abort))) break;
            // chunk 3g + i: A = this CTA's tokens, B = its N/2 query rows.  The
            // exponential turns what a score loses in truncated sums (kTruncPerStep)
            // into a share of the weight: 18 * 4.9e-7 for a token with x = 18 and one
            // chain of 36 steps.  kChains accumulators of kSteps steps each, added in
            // registers with rounding, divide it by kChains; the scale takes the mean
            // of the rest back
            const uint64_t kg = k_desc + (uint64_t)((slot * C::kStage) >> 4);
            const uint64_t qg = q_desc + (uint64_t)((3 * g * C::kQChunk) >> 4);
#pragma unroll
            for (int i = 0; i < 3; i++) {
              if (3 * g + i >= p.chunks) break;
#pragma unroll
              for (int kk = 0; kk < 4; kk++) {
                const int step = 12 * g + 4 * i + kk;
                mma_bf16_pair(tmem + sb * C::kBufCols + step / C::kSteps * C::kCols,
                              kg + (uint64_t)((i * 1024 + kk * 32) >> 4),
                              qg + (uint64_t)((i * C::kQChunk + kk * 32) >> 4), idesc,
                              step % C::kSteps != 0 ? 1u : 0u);
              }
            }
            tc_commit_pair(&sh->kempty[slot], 3);
            last_bar = &sh->kempty[slot];
            last_phase = use & 1;
          }
          if (ok) {
            tc_commit_pair(&sh->s_full[sb], 3);
            last_bar = &sh->s_full[sb];
            last_phase = (gt >> 1) & 1;
          }
        }
      }
      if (*abort && last_bar != nullptr) {
        // the MMAs issued so far finish before TMEM and the slots go away
        volatile int never = 0;
        mbar_wait<true>(last_bar, last_phase, &never);
      }
    }
  } else {
    // ------------------------------------------------ epilogue (warps 2-5)
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;  // TMEM lane
    constexpr bool kSplit = C::kCols < N;  // a token's columns in two lanes
    const int hl = kSplit ? row & 63 : row, half = kSplit ? row >> 6 : 0;
    const int et = threadIdx.x - 64;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const float sl2 = p.score_scale;
    const uint32_t s_free_l[2] = {mapa_shared(smem_u32(&sh->s_free[0]), 0),
                                  mapa_shared(smem_u32(&sh->s_free[1]), 0)};
    const int64_t seq_rows = (int64_t)p.sh.s * p.sh.h;
    float* neg = sh->neg[warp - 2];

    cudaTriggerProgrammaticLaunchCompletion();  // the next kernel may be launched; it waits for this grid
    // positions that no token of the step can see: zero, unless sums are added to
    if (!p.accumulate)
      for (int b = blockIdx.x; b < p.sh.b; b += gridDim.x) {
        const TreeSeq q = tree_seq<Cut>(p.sh, b);
        for (int i = (q.n > 0 ? q.len : 0) + et; i < p.sh.max_len; i += 128)
          p.sums[b * p.sums_stride + i] = 0.f;
      }

    int gt = 0;
    bool ok = true;
    TreeCursor c = range.start;
    TreePiece u;
    while (ok && tree_piece<Cut>(p.sh, c, u)) {
      const int base = u.q.len - u.q.n;
      const int col0 = u.g * N + half * C::kCols;  // first row of this thread's columns
      const int ncol = min(max(u.q.n * p.sh.h - col0, 0), C::kCols);
      __syncwarp();
      for (int i = lane; i < C::kCols; i += 32)
        neg[i] = i < ncol ? -kLog2e * p.lse[u.b * seq_rows + col0 + i] : 0.f;
      __syncwarp();
      const uint8_t* mask = p.sh.mask ? p.sh.mask + u.b * p.sh.mask_stride : nullptr;
      const bool direct = u.q.groups == 1;
      float* out = direct ? p.sums + u.b * p.sums_stride
                          : p.part + ((int64_t)u.g * p.sh.b + u.b) * p.part_stride;
      for (int t = u.t_begin; t < u.t_end && ok; t++, gt++) {
        const int sb = gt & 1, xb = gt & 3;
        const int tok0 = t * C::kTile + (int)rank * (C::kTile / 2), tok = tok0 + hl;
        // columns (rows of the sequence) that see this token
        const bool full = tok0 + C::kTile / 2 <= base && ncol == C::kCols;
        uint32_t bits[C::kCols / 32];
        if (!full) {
#pragma unroll
          for (int k = 0; k < C::kCols / 32; k++) bits[k] = 0;
          auto set = [&](int c0, int c1) {  // columns [c0, c1)
#pragma unroll
            for (int k = 0; k < C::kCols / 32; k++) {
              const int lo = max(c0 - 32 * k, 0), hi = min(c1 - 32 * k, 32);
              if (lo < hi) bits[k] |= (hi - lo == 32 ? 0xffffffffu : ((1u << (hi - lo)) - 1u) << lo);
            }
          };
          if (tok < base) {
            set(0, ncol);
          } else if (tok < u.q.len && ncol > 0) {
            const int j = tok - base, t_end = (col0 + ncol - 1) / p.sh.h;
            // the masks of several nodes are read together (13 trees of 60 nodes x 1 head
            // x 4361 tokens: 17.7 us, 27.4 one by one); groups of 256 rows, mostly of many
            // heads a node, have few nodes (47 trees of 23 nodes x 128 heads x 256 tokens:
            // 57.6 us with 4 at a time, 60.5 with 8)
            constexpr int kNodes = kSplit ? 4 : 8;
            for (int n0 = col0 / p.sh.h; n0 <= t_end; n0 += kNodes) {
              uint8_t m[kNodes];
#pragma unroll
              for (int i = 0; i < kNodes; i++) {
                const int node = min(n0 + i, t_end);
                m[i] = j <= node;  // a chain
                if (mask) m[i] = mask[(int64_t)node * p.sh.s + j];
              }
#pragma unroll
              for (int i = 0; i < kNodes; i++) {
                const int node = n0 + i;
                if (node <= t_end && m[i]) set(max(node * p.sh.h - col0, 0), min((node + 1) * p.sh.h - col0, ncol));
              }
            }
          }
        }
        if (!(ok = tree_warp_wait(&sh->s_full[sb], (gt >> 1) & 1, abort))) break;
        tc_fence_after();
        const uint32_t s_addr = tmem + lane_base + sb * C::kBufCols;
        const uint64_t sc2 = f2_pack(sl2, sl2);
        uint64_t acc[4];
#pragma unroll
        for (int k = 0; k < 4; k++) acc[k] = f2_pack(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < C::kCols / 16; k++) {  // 16 columns at a time
          float v[C::kChains][16];
#pragma unroll
          for (int c = 0; c < C::kChains; c++) tmem_ld16(s_addr + c * C::kCols + 16 * k, v[c]);
#pragma unroll
          for (int c = 0; c < C::kChains; c++) tmem_ld_wait_regs16(v[c]);
          if (k == C::kCols / 16 - 1) {  // all scores are read: the S buffer is free
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(s_free_l[sb]);
          }
          const ulonglong2* n2 = reinterpret_cast<const ulonglong2*>(neg + 16 * k);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const ulonglong2 ng = n2[i];
            uint64_t s01 = f2_pack(v[0][4 * i], v[0][4 * i + 1]);
            uint64_t s23 = f2_pack(v[0][4 * i + 2], v[0][4 * i + 3]);
#pragma unroll
            for (int c = 1; c < C::kChains; c++) {
              s01 = f2_add(s01, f2_pack(v[c][4 * i], v[c][4 * i + 1]));
              s23 = f2_add(s23, f2_pack(v[c][4 * i + 2], v[c][4 * i + 3]));
            }
            float x0, x1, x2, x3;
            f2_unpack(f2_fma(s01, sc2, ng.x), x0, x1);
            f2_unpack(f2_fma(s23, sc2, ng.y), x2, x3);
            float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
            float p2 = ex2_approx(x2), p3 = ex2_approx(x3);
            if (!full) {  // a selection, not a product: unseen scores may be NaN
              const uint32_t m = bits[k / 2] >> (16 * (k & 1) + 4 * i);
              p0 = m & 1u ? p0 : 0.f;
              p1 = m & 2u ? p1 : 0.f;
              p2 = m & 4u ? p2 : 0.f;
              p3 = m & 8u ? p3 : 0.f;
            }
            acc[(2 * i) & 3] = f2_add(acc[(2 * i) & 3], f2_pack(p0, p1));
            acc[(2 * i + 1) & 3] = f2_add(acc[(2 * i + 1) & 3], f2_pack(p2, p3));
          }
        }
        float a0, a1;
        f2_unpack(f2_add(f2_add(acc[0], acc[1]), f2_add(acc[2], acc[3])), a0, a1);
        float w = a0 + a1;
        bool owner = true;
        if constexpr (kSplit) {
          // the token's other half of the columns.  Buffer xb is written again
          // four tiles on, after an s_full that needs this warp pair's reader to
          // have released S two tiles later than this one
          owner = half == 0;
          if (!owner) {
            sh->xsum[xb][hl] = w;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->xbar[quarter & 1][xb]);
          } else {
            if (!(ok = tree_warp_wait(&sh->xbar[quarter & 1][xb], (gt >> 2) & 1, abort))) break;
            w += sh->xsum[xb][hl];
          }
        }
        if (owner && tok < u.q.len) out[tok] = direct && p.accumulate ? out[tok] + w : w;
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<2>(tmem, C::kTmemCols);
  }
  if (threadIdx.x == 0 && *abort) raise_dev_error(p.sh.err, QCAU_DEVERR_TIMEOUT);
}

// The groups' partial sums of a token, in group order.
// (Only groups of 256 rows leave several.)
__global__ void __launch_bounds__(256) weights_combine_kernel(WeightsParams p) {
  using Cut = TreeCut<256, WeightsCfg<256>::kTile>;
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
  const int b = blockIdx.y, tok = blockIdx.x * 256 + threadIdx.x;
  const TreeSeq q = tree_seq<Cut>(p.sh, b);
  if (q.groups < 2 || tok >= q.len) return;
  float w = 0.f;
#pragma unroll 8
  for (int g = 0; g < q.groups; g++) w += p.part[((int64_t)g * p.sh.b + b) * p.part_stride + tok];
  float* out = p.sums + b * p.sums_stride + tok;
  *out = p.accumulate ? *out + w : w;
}

// Rows of a group: all the rows in one group up to 256, so that K is read once.
int weights_group(const TreeArgs& a) {
  const int64_t rows = a.s * a.h;
  return rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
}

template <int N>
cudaError_t run_weights(const TreeArgs& a, const WeightsParams& p, const CUtensorMap& tq,
                        const CUtensorMap& tk, int64_t pairs, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem((const void*)attn_weights_sm100_kernel<N>, weights_smem<N>(), done);
  if (e != cudaSuccess) return e;
  return launch_early(attn_weights_sm100_kernel<N>, dim3((unsigned)(2 * pairs)), 1, kThreads,
                      weights_smem<N>(), st, tq, tk, p);
}

}  // namespace

size_t attn_weights_workspace(const TreeArgs& a) {
  const int n = weights_group(a);
  const int64_t groups = (a.s * a.h + n - 1) / n;
  return groups > 1 ? (size_t)groups * a.b * ((a.max_len + 3) / 4 * 4) * 4 : 0;
}

cudaError_t launch_attn_weights_sm100(const TreeArgs& a, void* ws, cudaStream_t st) {
  const int n = weights_group(a);
  const int tile = n == 256 ? WeightsCfg<256>::kTile : WeightsCfg<128>::kTile;
  const int64_t rows = a.s * a.h, pairs = tree_pairs(a, n, tile);
  CUtensorMap tq, tk;
  {
    // Q as [b][chunks][rows][64 values]: three chunks of a CTA's rows in a box
    const uint64_t row = (uint64_t)a.d_qk * 2;
    const uint64_t dims[4] = {64, (uint64_t)rows, (uint64_t)(a.d_qk / 64), (uint64_t)a.b};
    const uint64_t strides[3] = {row, 128, (uint64_t)rows * row};
    const uint32_t box[4] = {64, (uint32_t)n / 2, 3, 1};
    if (!make_tmap(&tq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, a.q, dims, strides, box,
                   CU_TENSOR_MAP_SWIZZLE_128B))
      return cudaErrorInvalidValue;
  }
  {
    // the cache as [64-token blocks][groups of 8 tokens][chunks][8 tokens][64 values]
    const uint64_t row = (uint64_t)a.d_qk * 2;
    const uint64_t dims[5] = {64, 8, (uint64_t)(a.d_qk / 64), 8,
                              (uint64_t)(a.num_pages * (a.page_size / 64))};
    const uint64_t strides[4] = {row, 128, 8 * row, 64 * row};
    const uint32_t box[5] = {64, 8, 3, 8, 1};
    if (!make_tmap(&tk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, a.cache, dims, strides, box,
                   CU_TENSOR_MAP_SWIZZLE_128B))
      return cudaErrorInvalidValue;
  }
  WeightsParams p{};
  p.sh = tree_shape(a, n, pairs);
  // a row's start hides behind the K stream (64 x 4000 tokens x 64 heads: 41.8 us against
  // 43.2 with a cost of 2 tiles; 4 x 16 nodes x 64 heads x 8000: 38.3, 39.7 with 1)
  p.sh.row_cost = 0;
  p.lse = a.lse;
  p.sums = a.sums;
  p.sums_stride = a.sums_stride;
  p.part = reinterpret_cast<float*>(ws);
  p.part_stride = (a.max_len + 3) / 4 * 4;
  p.accumulate = a.accumulate;
  p.chunks = (int)(a.d_qk / 64);
  // (log2(e) as the kernel has it for the log-sum-exps: its rounding leaves the difference)
  p.score_scale = tree_score_scale(a.scale, kLog2e, a.d_qk,
                                   n == 256   ? WeightsCfg<256>::kSteps
                                   : n == 128 ? WeightsCfg<128>::kSteps
                                              : WeightsCfg<64>::kSteps);
  cudaError_t e = n == 256   ? run_weights<256>(a, p, tq, tk, pairs, st)
                  : n == 128 ? run_weights<128>(a, p, tq, tk, pairs, st)
                             : run_weights<64>(a, p, tq, tk, pairs, st);
  if (e != cudaSuccess || p.sh.groups == 1) return e;
  return launch_early(weights_combine_kernel,
                      dim3((unsigned)((a.max_len + 255) / 256), (unsigned)a.b), 1, 256, 0, st,
                      p);
}

}  // namespace qcau
