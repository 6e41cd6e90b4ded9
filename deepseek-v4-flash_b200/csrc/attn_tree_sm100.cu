// attn_tree_sm100.cu -- tcgen05 two-CTA attention of a tree of drafted tokens
// over a paged latent cache that already holds their rows (verification in
// speculative decoding).  No counterpart in the reference.
//
//   x[r, p]  = scale * q[r] . k[p]          r = (node t, head), p a cached token
//   lse[r]   = log(sum over the p that t sees of e^x[r, p]  +  e^sink[head])
//   o[r]     = sum e^(x[r, p] - lse[r]) v[p],  v[p] = k[p][:512]
// A sequence of len tokens ends with its n nodes: node t is token base + t,
// base = len - n; it sees every token before base, and token base + j when
// mask[t][j] is set (no mask: j <= t).
//
// All rows of a sequence share its cache, so the s * h query rows are laid end
// to end and cut into groups of 128 (the MMAs' M): 16 heads x 8 nodes fill a
// group as 128 heads of one node do, and a head count that divides nothing
// (5, 48) costs one partly filled group at the end, not padding per node.
// The pair's tile pipeline is the decode kernel's (attn_decode_sm100.cu): CTA
// r of the pair owns rows [64 r, 64 r + 64) of the group, tiles of 128 tokens,
// QK 128 x 128 x d, P rounded to bf16 at the exact running max of each tile
// (the denominator is summed from the fp32 P), PV 128 x 256 x 128 twice.  (A
// maximum raised only past 2^8 spares most rescales of O, 5 % of the time, but
// the largest P is then no exact 1: errors of 2.0e-3 against 1.7e-3 of the
// output's norm at 16 x 64 nodes x 16 heads x 32768 tokens.)
//
// Schedule: the tiles of all (sequence, group) rows, laid end to end at the
// batch's own lengths (read on the device: a ragged batch is balanced too),
// are cut into one equal range per CTA pair.  A row inside a range is
// normalised and written by the pair itself; a range has at most two pieces of
// rows that others share (its first and its last), whose softmax state and fp32
// O go to the pair's two slots, and tree_combine merges them.  So the partials
// are 2 x 128 rows a pair whatever the batch.  When the groups of a sequence
// fill the pairs evenly (teams of `groups` pairs), a team takes one range of
// the sequences' tiles and each of its pairs one group: the pairs read the same
// K and V tiles at the same time, which then come from L2.
//
// Rows of V that no query may see are zeroed in shared memory before the MMAs
// read them (0 * NaN would reach every row): tokens past the sequence's end,
// left over in its last page; and among the drafted tokens' rows, which only
// their descendants see, values that are not finite.
// Every wait is bounded; a timeout raises QCAU_DEVERR_TIMEOUT, drains the
// copies in flight, frees TMEM and returns.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "tree_plan.cuh"

namespace qcau {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 128;            // tokens per tile (two blocks of 64, one per CTA for K)
using Cut = TreeCut<128, kTile>;
constexpr int kKSlot = 24576;         // this CTA's 64 tokens x 3 chunks of 64 dims (one box)
constexpr int kKSlots = 3;            // 9 chunks = 576 dims (8 = 512: the last box ends in zeros)
constexpr int kVSlot = 32768;         // 64 tokens x this CTA's 256 dims (4 chunks, one box)
constexpr int kVSlots = 2;            // the tile's two blocks
constexpr int kQBox = 3 * 8192;       // 64 rows x 3 chunks
constexpr int kQBytes = 3 * kQBox;    // 64 rows x 576 bf16
constexpr int kPBytes = 2 * 8192;     // 64 rows x 128 tokens bf16 (2 chunks of 64 tokens)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

constexpr uint32_t kTmemO = 0;        // 2 accumulators x 128 columns
constexpr uint32_t kTmemS = 256;      // 2 buffers x 64 columns
constexpr uint32_t kTmemCols = 512;

struct TreeShared {
  uint64_t kfull[kKSlots];   // leader: K slot (and a third of a new piece's Q) landed in both CTAs
  uint64_t kempty[kKSlots];  // both: K slot consumed by QK (the last slot: s_full)
  uint64_t vfull[kVSlots];   // leader: V slot ready in both CTAs
  uint64_t vempty[kVSlots];  // both: V slot consumed by PV (the last slot: p_free)
  uint64_t vtail;            // local: a V slot that is cleaned before use has landed
  uint64_t s_full[2];        // both: S(t) ready
  uint64_t s_free[2];        // leader: the 8 softmax warps have read S(t)
  uint64_t p_full;           // leader: the 8 softmax warps wrote P(t) / corrected O
  uint64_t p_free;           // both: PV(t) done with P and O
  uint64_t o_full;           // both: last PV of the piece done
  uint64_t o_free;           // leader: the 8 epilogue warps have read O
  uint64_t xbar[2];          // local: the 4 softmax warps exchanged tile maxima
  uint64_t lbar;             // local: denominator exchange
  float xmax[2][128];
  float xsum[128];
  uint32_t tmem_base;
  int abort;
  TreePlanShared plan;
};

constexpr size_t kSmemBytes = 1024 + kQBytes + kPBytes + (size_t)kKSlots * kKSlot +
                              (size_t)kVSlots * kVSlot + sizeof(TreeShared);
static_assert(kSmemBytes <= 232448, "shared memory budget");

struct TreeParams {
  TreeShape sh;        // groups of 128 rows
  __nv_bfloat16* out;  // [b, s, h, 512]
  float* lse;          // [b, s, h] or nullptr
  const float* sink;   // [h] or nullptr
  int chunks;          // 64-value chunks of a row: 9 or 8
  float score_scale;   // log2 units
  float* part_o;   // [pairs][2][128][512]
  float* part_ml;  // [pairs][2][128][2]: max (log2 units), sum
  int4* desc;      // [pairs]: the row whose pieces start at this pair {b or -1, group, rows of
                   // the sequence, pieces | pairs between pieces << 16}
};

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

// The weight of O and the log-sum-exp of a row whose scores have the maximum m
// (log2 units) and the sum l relative to it, with the sink's term: both are
// taken relative to the larger of m and the sink, so neither overflows.
__device__ __forceinline__ void tree_norm(float m, float l, float sink, float& inv, float& lse) {
  const float sk = sink * kLog2e;
  const float top = fmaxf(m, sk);
  if (top == -INFINITY && l == 0.f) {  // nothing seen and no sink
    inv = 0.f;
    lse = -INFINITY;
    return;
  }
  const float wm = m == -INFINITY ? 0.f : exp2f(m - top);
  const float den = l * wm + (sk == top ? 1.f : exp2f(sk - top));  // (an infinite sink: 1)
  inv = den > 0.f || den != den ? wm / den : 0.f;
  lse = (top + log2f(den)) * kLn2;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    attn_tree_sm100_kernel(const __grid_constant__ CUtensorMap tm_q,
                           const __grid_constant__ CUtensorMap tm_k,
                           const __grid_constant__ CUtensorMap tm_v, TreeParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  uint8_t* sQ = smem_raw + pad;
  uint8_t* sP = sQ + kQBytes;
  uint8_t* sK = sP + kPBytes;
  uint8_t* sV = sK + (size_t)kKSlots * kKSlot;
  TreeShared* sh = reinterpret_cast<TreeShared*>(sV + (size_t)kVSlots * kVSlot);
  volatile int* abort = &sh->abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kKSlots; i++) {
      mbar_init(&sh->kfull[i], 1);
      mbar_init(&sh->kempty[i], 1);
    }
    for (int i = 0; i < kVSlots; i++) {
      mbar_init(&sh->vfull[i], 2);
      mbar_init(&sh->vempty[i], 1);
    }
    mbar_init(&sh->vtail, 1);
    for (int i = 0; i < 2; i++) {
      mbar_init(&sh->s_full[i], 1);
      mbar_init(&sh->s_free[i], 8);
      mbar_init(&sh->xbar[i], 4);
    }
    mbar_init(&sh->p_full, 8);
    mbar_init(&sh->p_free, 1);
    mbar_init(&sh->o_full, 1);
    mbar_init(&sh->o_free, 8);
    mbar_init(&sh->lbar, 4);
    sh->abort = 0;
    fence_barrier_init();
  }
  if (threadIdx.x == 32) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 1) tmem_alloc<2>(&sh->tmem_base, kTmemCols);
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  cudaGridDependencySynchronize();
  const TreeRange range = tree_plan<Cut>(p.sh, &sh->plan, pair, npairs);

  if (warp == 0) {
    // ------------------------------------------------ Q and K producer (both CTAs)
    if (lane == 0) {
      int last_use[kKSlots];
      for (int i = 0; i < kKSlots; i++) last_use[i] = -1;
      int gt = 0;  // tiles
      bool ok = true;
      TreeCursor c = range.start;
      TreePiece u;
      while (ok && tree_piece<Cut>(p.sh, c, u)) {
        for (int t = u.t_begin; t < u.t_end && ok; t++, gt++) {
          const int blk = tree_block(p.sh, u, 2 * t + (int)rank);
          for (int i = 0; i < kKSlots; i++) {
            // the tile's last box is released by the tile's completion commit
            if (i == kKSlots - 1) {
              if (gt > 0 && !(ok = mbar_wait(&sh->s_full[(gt - 1) & 1], ((gt - 1) >> 1) & 1, abort)))
                break;
            } else if (!(ok = mbar_wait(&sh->kempty[i], (gt & 1) ^ 1, abort))) {
              break;
            }
            // a piece's first tile brings its Q (rows past the sequence's: zeros) along,
            // the box's three chunks at a time: the MMAs that freed the slot were the
            // last to read the previous piece's
            const bool with_q = t == u.t_begin;
            const uint32_t bar = mapa_shared(smem_u32(&sh->kfull[i]), 0);
            if (leader) mbar_arrive_expect_tx(&sh->kfull[i], 2 * (kKSlot + (with_q ? kQBox : 0)));
            last_use[i] = gt;
            if (with_q)
              tma_load_4d_pair(sQ + i * kQBox, &tm_q, bar, 0, u.g * 128 + 64 * (int)rank, 3 * i, u.b);
            tma_load_4d_pair(sK + i * kKSlot, &tm_k, bar, 0, 0, 3 * i, blk);
          }
        }
      }
      if (*abort && leader) {
        // the leader's full barriers count both CTAs' copies: drain them all
        volatile int never = 0;
        for (int i = 0; i < kKSlots; i++)
          if (last_use[i] >= 0) mbar_wait<true>(&sh->kfull[i], last_use[i] & 1, &never);
      }
    }
  } else if (warp == 6) {
    // ------------------------------------------------ V producer (both CTAs, the whole warp)
    int last_use[kVSlots];
    for (int i = 0; i < kVSlots; i++) last_use[i] = -1;
    int gt = 0, tails = 0;
    bool ok = true;
    TreeCursor c = range.start;
    TreePiece u;
    while (ok && tree_piece<Cut>(p.sh, c, u)) {
      const int base = u.q.len - u.q.n;
      for (int t = u.t_begin; t < u.t_end && ok; t++, gt++) {
#pragma unroll
        for (int i = 0; i < kVSlots; i++) {
          if (i == kVSlots - 1) {
            if (gt > 0 && !(ok = tree_warp_wait(&sh->p_free, (gt - 1) & 1, abort))) break;
          } else if (!(ok = tree_warp_wait(&sh->vempty[i], (gt & 1) ^ 1, abort))) {
            break;
          }
          const int tok0 = t * kTile + 64 * i;
          uint8_t* slot = sV + i * kVSlot;
          const uint32_t full_l = mapa_shared(smem_u32(&sh->vfull[i]), 0);
          const bool tail = tok0 + 64 > base;
          last_use[i] = gt;
          if (lane == 0) {
            const int blk = tree_block(p.sh, u, 2 * t + i);
            uint32_t bar = full_l;
            if (tail) {
              mbar_arrive_expect_tx(&sh->vtail, kVSlot);
              bar = mapa_shared(smem_u32(&sh->vtail), rank);
            } else if (leader) {
              mbar_arrive_expect_tx(&sh->vfull[i], 2 * kVSlot);
            } else {
              mbar_arrive_remote(full_l);
            }
            tma_load_4d_pair(slot, &tm_v, bar, 0, 0, 4 * (int)rank, blk);
          }
          __syncwarp();
          if (!tail) continue;
          // drafted tokens and the rest of the block: lane = 16 bytes of a
          // row's four 128-byte chunks (the swizzle stays inside a row)
          if (!(ok = tree_warp_wait(&sh->vtail, tails & 1, abort))) {
            volatile int never = 0;
            tree_warp_wait(&sh->vtail, tails & 1, &never);
            break;
          }
          tails++;
          uint8_t* at = slot + (lane >> 3) * 8192 + (lane & 7) * 16;
          const int live_end = min(64, u.q.len - tok0);
#pragma unroll 8
          for (int r = max(0, base - tok0); r < live_end; r++) {
            uint4 v = *reinterpret_cast<const uint4*>(at + r * 128);
            uint32_t* w = reinterpret_cast<uint32_t*>(&v);
            uint32_t bad = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) bad |= (w[k] & 0x7f807f80u) + 0x00800080u;
            if (bad & 0x80008000u) {  // an exponent of all ones: infinity or NaN
#pragma unroll
              for (int k = 0; k < 4; k++) {
                if ((w[k] & 0x7f80u) == 0x7f80u) w[k] &= 0xffff0000u;
                if ((w[k] & 0x7f800000u) == 0x7f800000u) w[k] &= 0x0000ffffu;
              }
              *reinterpret_cast<uint4*>(at + r * 128) = v;
            }
          }
          for (int r = max(0, live_end); r < 64; r++)
            *reinterpret_cast<uint4*>(at + r * 128) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(full_l);
        }
      }
    }
    if (*abort && leader && lane == 0) {
      volatile int never = 0;
      for (int i = 0; i < kVSlots; i++)
        if (last_use[i] >= 0) mbar_wait<true>(&sh->vfull[i], last_use[i] & 1, &never);
    }
  } else if (warp == 1 || warp == 7) {
    // ------------------------------------------------ MMA issuers (pair leader)
    if (leader && lane == 0) {
      const uint32_t q_addr = smem_u32(sQ), p_addr = smem_u32(sP);
      const uint32_t k_addr = smem_u32(sK), v_addr = smem_u32(sV);
      uint64_t* last_bar = nullptr;  // barrier of the last commit, for the drain
      int last_phase = 0;
      bool ok = true;
      TreeCursor cur = range.start;
      TreePiece u;
      if (warp == 1) {
        const uint32_t idesc_qk = make_idesc(128, 128, kFmtBF16, kFmtBF16, false, false);
        const uint64_t q_desc = make_sdesc(q_addr, 16, 1024), k_desc = make_sdesc(k_addr, 16, 1024);
        int gt = 0;  // tiles
        while (ok && tree_piece<Cut>(p.sh, cur, u)) {
          for (int t = u.t_begin; t < u.t_end && ok; t++, gt++) {
            const int sb = gt & 1;
            if (gt >= 2 && !(ok = mbar_wait<true>(&sh->s_free[sb], ((gt >> 1) - 1) & 1, abort)))
              break;
            tc_fence_after();
            for (int g = 0; g < kKSlots; g++) {
              if (!(ok = mbar_wait(&sh->kfull[g], gt & 1, abort))) break;
              // chunk 3g + c: 4 MMAs of 16 dims, B = this CTA's 64 tokens (N = 128)
              const uint64_t qg = q_desc + (uint64_t)((3 * g * 8192) >> 4);
              const uint64_t kg = k_desc + (uint64_t)((g * kKSlot) >> 4);
#pragma unroll
              for (int c = 0; c < 3; c++) {
                if (3 * g + c >= p.chunks) break;
#pragma unroll
                for (int kk = 0; kk < 4; kk++)
                  mma_bf16_pair(tmem + kTmemS + sb * 64, qg + (uint64_t)((c * 8192 + kk * 32) >> 4),
                                kg + (uint64_t)((c * 8192 + kk * 32) >> 4), idesc_qk,
                                (g | c | kk) != 0 ? 1u : 0u);
              }
              if (g + 1 < kKSlots) {  // the last box is released by s_full
                tc_commit_pair(&sh->kempty[g], 3);
                last_bar = &sh->kempty[g];
                last_phase = gt & 1;
              }
            }
            if (ok) {
              tc_commit_pair(&sh->s_full[sb], 3);
              last_bar = &sh->s_full[sb];
              last_phase = (gt >> 1) & 1;
            }
          }
        }
      } else {
        const uint32_t idesc_pv = make_idesc(128, 256, kFmtBF16, kFmtBF16, false, true);
        const uint64_t p_desc = make_sdesc(p_addr, 16, 1024), v_desc = make_sdesc(v_addr, 8192, 1024);
        int gt = 0, nu = 0;
        while (ok && tree_piece<Cut>(p.sh, cur, u)) {
          // the first PV of a piece overwrites O: the previous epilogue has read it
          if (nu > 0 && !(ok = mbar_wait<true>(&sh->o_free, (nu - 1) & 1, abort))) break;
          for (int t = u.t_begin; t < u.t_end && ok; t++, gt++) {
            if (!(ok = mbar_wait<true>(&sh->p_full, gt & 1, abort))) break;
            tc_fence_after();
            for (int pg = 0; pg < kVSlots; pg++) {
              if (!(ok = mbar_wait(&sh->vfull[pg], gt & 1, abort))) break;
              // PV MMA j takes chunks 2j, 2j+1 of each CTA's slot: its output
              // columns are dims 256r + 128j + [0, 128) of CTA r's half
#pragma unroll
              for (int j = 0; j < 2; j++)
#pragma unroll
                for (int kk = 0; kk < 4; kk++) {
                  const uint64_t ad = p_desc + (uint64_t)((pg * 8192 + kk * 32) >> 4);
                  const uint64_t bd =
                      v_desc + (uint64_t)((pg * kVSlot + j * 16384 + kk * 2048) >> 4);
                  mma_bf16_pair(tmem + kTmemO + j * 128, ad, bd, idesc_pv,
                                (t > u.t_begin || pg > 0 || kk > 0) ? 1u : 0u);
                }
              if (pg + 1 < kVSlots) {  // the last block is released by p_free
                tc_commit_pair(&sh->vempty[pg], 3);
                last_bar = &sh->vempty[pg];
                last_phase = gt & 1;
              }
            }
            if (ok) {
              tc_commit_pair(&sh->p_free, 3);
              last_bar = &sh->p_free;
              last_phase = gt & 1;
            }
          }
          if (ok) tc_commit_pair(&sh->o_full, 3);
          nu++;
        }
      }
      if (*abort && last_bar != nullptr) {
        // the MMAs issued so far finish before TMEM and the slots go away
        volatile int never = 0;
        mbar_wait<true>(last_bar, last_phase, &never);
      }
    }
  } else {
    // ------------------------------------------------ softmax / correction / epilogue
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;  // TMEM lane
    const int hl = row & 63, half = row >> 6;
    const int et = threadIdx.x - 64;      // 0..127 over warps 2-5
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const float sl2 = p.score_scale;
    const uint32_t s_free_l[2] = {mapa_shared(smem_u32(&sh->s_free[0]), 0),
                                  mapa_shared(smem_u32(&sh->s_free[1]), 0)};
    const uint32_t p_full_l = mapa_shared(smem_u32(&sh->p_full), 0);
    const uint32_t o_free_l = mapa_shared(smem_u32(&sh->o_free), 0);

    cudaTriggerProgrammaticLaunchCompletion();  // the merge may be launched; it waits for this grid
    // the rows of nodes that a sequence does not have: zero, log-sum-exp -inf
    const int64_t seq_rows = (int64_t)p.sh.s * p.sh.h;
    // (CTA c: sequence c mod b, together with the other CTAs of that sequence)
    const int parts = max((int)gridDim.x / p.sh.b, 1), part = blockIdx.x / p.sh.b;
    for (int b = blockIdx.x % p.sh.b; b < p.sh.b && part < parts; b += gridDim.x) {
      const int64_t r0 = (int64_t)tree_seq<Cut>(p.sh, b).n * p.sh.h;
      uint4* o = reinterpret_cast<uint4*>(p.out + ((int64_t)b * seq_rows + r0) * 512);
      for (int64_t i = part * 128 + et; i < (seq_rows - r0) * 64; i += parts * 128)
        o[i] = make_uint4(0u, 0u, 0u, 0u);
      if (p.lse)
        for (int64_t i = r0 + part * 128 + et; i < seq_rows; i += parts * 128)
          p.lse[b * seq_rows + i] = -INFINITY;
    }

    int4 owner = make_int4(-1, 0, 0, 0);
    int gt = 0, nu = 0;  // tiles, pieces
    bool ok = true;
    TreeCursor c = range.start;
    TreePiece u;
    while (ok && tree_piece<Cut>(p.sh, c, u)) {
      const int base = u.q.len - u.q.n;
      const int my_row = u.g * 128 + (int)rank * 64 + hl;  // row of the sequence
      const bool mine = my_row < u.q.n * p.sh.h;
      const int my_t = mine ? my_row / p.sh.h : -1;
      const uint8_t* mask = p.sh.mask ? p.sh.mask + u.b * p.sh.mask_stride : nullptr;
      float m_run = -INFINITY, l_run = 0.f;
      for (int t = u.t_begin; t < u.t_end && ok; t++, gt++) {
        const int sb = gt & 1;
        const uint32_t s_addr = tmem + lane_base + kTmemS + sb * 64;
        const int tok0 = t * kTile + half * 64;
        // which of the half tile's 64 tokens this thread's row sees
        const bool full = tok0 + 64 <= base;
        uint32_t bits[2] = {0xffffffffu, 0xffffffffu};
        if (!full) {
          // A ballot pair per node among the warp's rows; the masks of two nodes are read
          // together, from a valid address wherever the token lies, so that no branch
          // parts the loads (one tree of 64 nodes x 1 head x 2000 tokens: 16.4 us, 23.5
          // one by one)
          constexpr int kNodes = 2;
          const int j0 = tok0 + lane - base, j1 = j0 + 32;  // this lane's two tokens, as nodes
          const bool live0 = j0 < u.q.n, live1 = j1 < u.q.n;
          unsigned left = __ballot_sync(0xffffffffu, mine);
          bits[0] = bits[1] = 0;
          while (left) {
            unsigned same[kNodes];
            uint8_t m0[kNodes], m1[kNodes];
#pragma unroll
            for (int k = 0; k < kNodes; k++) {
              const int node = __shfl_sync(0xffffffffu, my_t, left ? __ffs(left) - 1 : 0);
              same[k] = left & __ballot_sync(0xffffffffu, my_t == node);
              left &= ~same[k];
              m0[k] = j0 <= node;  // a chain
              m1[k] = j1 <= node;
              if (mask) {
                const uint8_t* row = mask + (int64_t)max(node, 0) * p.sh.s;
                m0[k] = row[min(max(j0, 0), p.sh.s - 1)];
                m1[k] = row[min(max(j1, 0), p.sh.s - 1)];
              }
            }
#pragma unroll
            for (int k = 0; k < kNodes; k++) {
              const unsigned b0 = __ballot_sync(0xffffffffu, live0 && (j0 < 0 || m0[k] != 0));
              const unsigned b1 = __ballot_sync(0xffffffffu, live1 && (j1 < 0 || m1[k] != 0));
              if (same[k] >> lane & 1u) {
                bits[0] = b0;
                bits[1] = b1;
              }
            }
          }
        }
        if (!(ok = tree_warp_wait(&sh->s_full[sb], (gt >> 1) & 1, abort))) break;
        tc_fence_after();
        // this thread's 64 scores into registers; the S buffer is then free
        float v[64];
#pragma unroll
        for (int k = 0; k < 2; k++)
          tmem_ld32(s_addr + k * 32, *reinterpret_cast<float(*)[32]>(v + 32 * k));
#pragma unroll
        for (int k = 0; k < 2; k++) tmem_ld_wait_regs(v + 32 * k);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(s_free_l[sb]);
        // pass 1: tile max; unseen scores (of stale or unfinished rows) become -inf
        if (!full) {
#pragma unroll
          for (int i = 0; i < 64; i++)
            if (!((bits[i >> 5] >> (i & 31)) & 1u)) v[i] = -INFINITY;
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // four chains: latency
#pragma unroll
        for (int i = 0; i < 64; i++) m4[i & 3] = fmaxf(m4[i & 3], v[i]);
        const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * sl2;
        sh->xmax[sb][row] = mx;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->xbar[sb]);
        if (!(ok = tree_warp_wait(&sh->xbar[sb], (gt >> 1) & 1, abort))) break;
        const float tmax = fmaxf(mx, sh->xmax[sb][row ^ 64]);
        float alpha = 1.f;
        bool resc = false;
        if (m_run == -INFINITY) {
          m_run = tmax;  // nothing seen yet: O holds zeros (or PV starts a fresh accumulator)
        } else if (tmax > m_run) {
          alpha = exp2f(m_run - tmax);
          m_run = tmax;
          resc = true;
        }
        // pass 2 into registers: P = 2^(s*scale*log2e - m) as bf16 pairs; the
        // row sum is over the unrounded values
        const float m_use = m_run == -INFINITY ? 0.f : m_run;
        const uint64_t sc2 = f2_pack(sl2, sl2), nm2 = f2_pack(-m_use, -m_use);
        uint64_t sum2[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
        uint32_t pk[32];
#pragma unroll
        for (int i = 0; i < 32; i++) {
          float x0, x1;
          f2_unpack(f2_fma(f2_pack(v[2 * i], v[2 * i + 1]), sc2, nm2), x0, x1);
          const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
          sum2[i & 1] = f2_add(sum2[i & 1], f2_pack(p0, p1));
          pk[i] = pack_bf16(p0, p1);
        }
        float ps0, ps1;
        f2_unpack(f2_add(sum2[0], sum2[1]), ps0, ps1);
        // P(t) reuses the buffer of P(t-1), and O holds tiles < t, once PV(t-1) is done
        if (gt >= 1 && !(ok = tree_warp_wait(&sh->p_free, (gt - 1) & 1, abort))) break;
        // 64 tokens = one 128-byte row (chunk `half`) of eight swizzled 16-byte units
        uint8_t* pbase = sP + half * 8192 + hl * 128;
#pragma unroll
        for (int k = 0; k < 8; k++)
          *reinterpret_cast<uint4*>(pbase + ((k ^ (hl & 7)) << 4)) =
              make_uint4(pk[4 * k], pk[4 * k + 1], pk[4 * k + 2], pk[4 * k + 3]);
        l_run = l_run * alpha + (ps0 + ps1);
        if (__any_sync(0xffffffffu, resc)) {
          // rescale this warp's rows of O (PV(t-1) is complete)
          tc_fence_after();
#pragma unroll 1
          for (int c0 = 0; c0 < 8; c0 += 4) {
            float o[4][32];
            const uint32_t ta = tmem + lane_base + kTmemO + c0 * 32;
#pragma unroll
            for (int k = 0; k < 4; k++) tmem_ld32(ta + k * 32, o[k]);
#pragma unroll
            for (int k = 0; k < 4; k++) tmem_ld_wait_regs(o[k]);
#pragma unroll
            for (int k = 0; k < 4; k++) {
#pragma unroll
              for (int i = 0; i < 32; i++) o[k][i] *= alpha;
              tmem_st32(ta + k * 32, o[k]);
            }
          }
          tmem_st_wait();
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(p_full_l);
      }
      if (ok) ok = tree_warp_wait(&sh->o_full, nu & 1, abort);
      sh->xsum[row] = l_run;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->lbar);
      if (ok) ok = tree_warp_wait(&sh->lbar, nu & 1, abort);
      if (ok) {
        tc_fence_after();
        const float l_tot = l_run + sh->xsum[row ^ 64];
        const bool first = u.t_begin == 0, last = u.t_end == u.q.tiles;
        // A thread holds 256 dims of one row; stored as they are, every store of a
        // warp would touch 32 lines (5300 cycles for bf16, 10200 for fp32).  So
        // each warp turns 32 rows x 128 bytes at a time in its own 4 KB of the P
        // buffer, which its last PV has left: 16-byte units swizzled within rows
        uint8_t* stage = sP + quarter * 4096;
        const int warp_row = u.g * 128 + (int)rank * 64 + (quarter & 1) * 32;
        const int live = u.q.n * p.sh.h - warp_row;  // rows of this warp that exist
        auto put = [&](int k, uint4 v) {
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((k ^ (lane & 7)) << 4)) = v;
        };
        // 128 bytes of each row, from the stage to dst + row * stride
        auto turn = [&](uint8_t* dst, int stride) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int r = 4 * i + (lane >> 3), k = lane & 7;
            const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + ((k ^ (r & 7)) << 4));
            if (r < live) *reinterpret_cast<uint4*>(dst + (int64_t)r * stride + k * 16) = v;
          }
          __syncwarp();
        };
        if (first && last) {
          // the whole row: normalise and write it
          float inv, lse;
          tree_norm(m_run, l_tot, mine && p.sink ? p.sink[my_row % p.sh.h] : -INFINITY, inv, lse);
          const int64_t orow = u.b * seq_rows + my_row;
          uint8_t* po = reinterpret_cast<uint8_t*>(p.out + (u.b * seq_rows + warp_row) * 512 + 256 * half);
#pragma unroll 1
          for (int c = 0; c < 4; c += 2) {  // 2 x 64 dims, loaded together
            float v[2][64];
#pragma unroll
            for (int k = 0; k < 4; k++)
              tmem_ld32(tmem + lane_base + kTmemO + 64 * c + 32 * k,
                        *reinterpret_cast<float(*)[32]>(&v[0][0] + 32 * k));
#pragma unroll
            for (int k = 0; k < 4; k++) tmem_ld_wait_regs(&v[0][0] + 32 * k);
#pragma unroll
            for (int j = 0; j < 2; j++) {
#pragma unroll
              for (int k = 0; k < 8; k++)
                put(k, make_uint4(pack_bf16(v[j][8 * k] * inv, v[j][8 * k + 1] * inv),
                                  pack_bf16(v[j][8 * k + 2] * inv, v[j][8 * k + 3] * inv),
                                  pack_bf16(v[j][8 * k + 4] * inv, v[j][8 * k + 5] * inv),
                                  pack_bf16(v[j][8 * k + 6] * inv, v[j][8 * k + 7] * inv)));
              turn(po + 128 * (c + j), 1024);
            }
          }
          if (p.lse && half == 0 && mine) p.lse[orow] = lse;
        } else {
          // a piece: its state and unnormalised O (fp32) to slot 1 when the row
          // starts here, else to slot 0
          const int64_t prow0 = ((int64_t)pair * 2 + (first ? 1 : 0)) * 128 + rank * 64;
          uint8_t* po = reinterpret_cast<uint8_t*>(p.part_o + (prow0 + (quarter & 1) * 32) * 512 + 256 * half);
#pragma unroll 1
          for (int c = 0; c < 8; c += 4) {  // 4 x 32 dims, loaded together
            float v[4][32];
#pragma unroll
            for (int j = 0; j < 4; j++) tmem_ld32(tmem + lane_base + kTmemO + (c + j) * 32, v[j]);
#pragma unroll
            for (int j = 0; j < 4; j++) tmem_ld_wait_regs(v[j]);
#pragma unroll
            for (int j = 0; j < 4; j++) {
#pragma unroll
              for (int k = 0; k < 8; k++)
                put(k, make_uint4(__float_as_uint(v[j][4 * k]), __float_as_uint(v[j][4 * k + 1]),
                                  __float_as_uint(v[j][4 * k + 2]), __float_as_uint(v[j][4 * k + 3])));
              turn(po + 128 * (c + j), 2048);
            }
          }
          if (half == 0)
            *reinterpret_cast<float2*>(p.part_ml + (prow0 + hl) * 2) = make_float2(m_run, l_tot);
          if (first) {
            const int last_range = tree_range_of(range, u.row0 + u.q.tiles - 1);
            owner = make_int4(u.b, u.g, u.q.n * p.sh.h,
                              (last_range - range.range + 1) | range.tsize << 16);
          }
        }
      }
      // O is read: the next piece's first PV may overwrite it
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(o_free_l);
      nu++;
    }
    if (leader && et == 0) p.desc[pair] = ok ? owner : make_int4(-1, 0, 0, 0);
  }

  __syncwarp();
  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<2>(tmem, kTmemCols);
  }
  if (threadIdx.x == 0 && *abort) raise_dev_error(p.sh.err, QCAU_DEVERR_TIMEOUT);
}

// Merge of the rows that several ranges share: M = max m_i, L = sum l_i 2^(m_i - M),
// O = sum O_i 2^(m_i - M), then the sink and the normalisation.  2 KB a row and
// piece, from L2: 44 MB for 74 groups of 128 rows of two or three pieces.
//
// Many groups: block (pair, j) takes rows [8 j, 8 j + 8) of the group whose pieces
// start at that pair, one warp a row, two pieces at a time so that four blocks fit an
// SM (23 sequences of 13 nodes x 64 heads x 1536: 83.6 us, 85.7 with four at a time
// and two blocks).
constexpr int kMaxPieces = 96;  // at least kTreePairs
static_assert(kMaxPieces >= kTreePairs, "a row's pieces fit the merge");

__global__ void __launch_bounds__(256, 4) tree_combine_kernel(TreeParams p) {
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
  const int pair = blockIdx.x, lane = threadIdx.x & 31;
  const int4 own = p.desc[pair];
  const int local = blockIdx.y * 8 + (threadIdx.x >> 5);
  const int row = own.y * 128 + local, pieces = own.w & 0xffff, step = own.w >> 16;
  if (own.x < 0 || row >= own.z) return;
  auto slot = [&](int i) -> int64_t {
    return ((int64_t)(pair + i * step) * 2 + (i == 0 ? 1 : 0)) * 128 + local;
  };
  float4 f[2][4];
  auto load = [&](int i0) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const float4* src = reinterpret_cast<const float4*>(p.part_o + slot(i0 + j) * 512) + lane;
#pragma unroll
      for (int k = 0; k < 4; k++)
        f[j][k] = i0 + j < pieces ? src[32 * k] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  float2 ml[kMaxPieces / 32];
#pragma unroll
  for (int r = 0; r < kMaxPieces / 32; r++)
    ml[r] = 32 * r + lane < pieces
                ? *reinterpret_cast<const float2*>(p.part_ml + slot(32 * r + lane) * 2)
                : make_float2(-INFINITY, 0.f);
  load(0);
  float M = -INFINITY;
#pragma unroll
  for (int r = 0; r < kMaxPieces / 32; r++) M = fmaxf(M, ml[r].x);
  M = warp_max(M);
  float w[kMaxPieces / 32], L = 0.f;
#pragma unroll
  for (int r = 0; r < kMaxPieces / 32; r++) {
    w[r] = ml[r].x == -INFINITY ? 0.f : exp2f(ml[r].x - M);
    L = fmaf(ml[r].y, w[r], L);
  }
  L = warp_sum(L);
  float a[16];
#pragma unroll
  for (int j = 0; j < 16; j++) a[j] = 0.f;
  for (int i0 = 0; i0 < pieces; i0 += 2) {
    if (i0 > 0) load(i0);
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int i = i0 + j;  // past the pieces: weight 0 of zeros
      const float wr = i < 32 ? w[0] : i < 64 ? w[1] : w[2];
      const float wi = __shfl_sync(0xffffffffu, wr, i & 31);
#pragma unroll
      for (int k = 0; k < 4; k++) {
        a[4 * k] = fmaf(f[j][k].x, wi, a[4 * k]);
        a[4 * k + 1] = fmaf(f[j][k].y, wi, a[4 * k + 1]);
        a[4 * k + 2] = fmaf(f[j][k].z, wi, a[4 * k + 2]);
        a[4 * k + 3] = fmaf(f[j][k].w, wi, a[4 * k + 3]);
      }
    }
  }
  float inv, lse;
  tree_norm(M, L, p.sink ? p.sink[row % p.sh.h] : -INFINITY, inv, lse);
  const int64_t orow = (int64_t)own.x * p.sh.s * p.sh.h + row;
  uint2* out = reinterpret_cast<uint2*>(p.out + orow * 512) + lane;
#pragma unroll
  for (int k = 0; k < 4; k++)
    out[32 * k] = make_uint2(pack_bf16(a[4 * k] * inv, a[4 * k + 1] * inv),
                             pack_bf16(a[4 * k + 2] * inv, a[4 * k + 3] * inv));
  if (p.lse && lane == 0) p.lse[orow] = lse;
}

// Few groups (one sequence, or some short trees), whose rows are cut into many pieces:
// every warp finds the shared rows in the descriptors, and rows go to as many of a
// block's warps as leave the blocks busy, all 8 for one group, which share out the
// row's pieces and read four at a time.
constexpr int kFewBlocks = 2 * 148;  // that run at once

__global__ void __launch_bounds__(256, 2) tree_combine_few_kernel(TreeParams p, int npairs) {
  constexpr int kFlight = 4;
  __shared__ __align__(16) float so[8][512];
  __shared__ float2 sml[8];
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the shared rows, pair by pair: this lane's three pairs and their places in the list
  static_assert(kTreePairs <= 96, "three descriptors a lane");
  int4 own[3];
  int first[3], rows[3], total = 0;
#pragma unroll
  for (int k = 0; k < 3; k++)
    own[k] = 32 * k + lane < npairs ? p.desc[32 * k + lane] : make_int4(-1, 0, 0, 0);
#pragma unroll
  for (int k = 0; k < 3; k++) {
    rows[k] = own[k].x >= 0 ? min(own[k].z - own[k].y * 128, 128) : 0;
    const int inc = warp_scan(rows[k]);
    first[k] = total + inc - rows[k];
    total += __shfl_sync(0xffffffffu, inc, 31);
  }
  int split = 8;  // warps of a row
  while (split > 1 && total * split > (int)gridDim.x * 8) split >>= 1;
  const int part = warp & (split - 1), per_block = 8 / split;
  for (int item0 = blockIdx.x * per_block; item0 < total; item0 += gridDim.x * per_block) {
    const int item = item0 + warp / split;
    int pair = -1, b = 0, g = 0, pieces = 0, step = 0, local = 0;
#pragma unroll
    for (int k = 0; k < 3; k++) {
      const unsigned at = __ballot_sync(0xffffffffu, first[k] <= item && item < first[k] + rows[k]);
      if (at) {
        const int l = __ffs(at) - 1;
        pair = 32 * k + l;
        b = __shfl_sync(0xffffffffu, own[k].x, l);
        g = __shfl_sync(0xffffffffu, own[k].y, l);
        const int w = __shfl_sync(0xffffffffu, own[k].w, l);
        pieces = w & 0xffff;
        step = w >> 16;
        local = item - __shfl_sync(0xffffffffu, first[k], l);
      }
    }
    const int row = g * 128 + local;
    const float sink = pair >= 0 && p.sink ? p.sink[row % p.sh.h] : -INFINITY;
    float M = -INFINITY, L = 0.f, a[16];
#pragma unroll
    for (int j = 0; j < 16; j++) a[j] = 0.f;
    for (int i0 = part; i0 < pieces; i0 += kFlight * split) {
      float m[kFlight], l[kFlight];
      float4 f[kFlight][4];
      float top = M;
#pragma unroll
      for (int j = 0; j < kFlight; j++) {
        // (past the last piece: that one again, at no weight, so that no branch parts the loads)
        const int i = min(i0 + j * split, pieces - 1);
        const int64_t slot = ((int64_t)(pair + i * step) * 2 + (i == 0 ? 1 : 0)) * 128 + local;
        const float4* src = reinterpret_cast<const float4*>(p.part_o + slot * 512) + lane;
        const float2 ml = reinterpret_cast<const float2*>(p.part_ml)[slot];
        m[j] = i0 + j * split < pieces ? ml.x : -INFINITY;
        l[j] = ml.y;
#pragma unroll
        for (int k = 0; k < 4; k++) f[j][k] = src[32 * k];
      }
#pragma unroll
      for (int j = 0; j < kFlight; j++) top = fmaxf(top, m[j]);
      const float w = M == -INFINITY ? 0.f : exp2f(M - top);
      M = top;
      L *= w;
#pragma unroll
      for (int j = 0; j < 16; j++) a[j] *= w;
#pragma unroll
      for (int j = 0; j < kFlight; j++) {
        if (i0 + j * split >= pieces) break;
        const float wj = m[j] == -INFINITY ? 0.f : exp2f(m[j] - top);
        L = fmaf(l[j], wj, L);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          a[4 * k] = fmaf(f[j][k].x, wj, a[4 * k]);
          a[4 * k + 1] = fmaf(f[j][k].y, wj, a[4 * k + 1]);
          a[4 * k + 2] = fmaf(f[j][k].z, wj, a[4 * k + 2]);
          a[4 * k + 3] = fmaf(f[j][k].w, wj, a[4 * k + 3]);
        }
      }
    }
    const int64_t orow = (int64_t)b * p.sh.s * p.sh.h + row;
    uint2* out = reinterpret_cast<uint2*>(p.out + orow * 512);
    float inv, lse;
    if (split == 1) {
      if (pair < 0) continue;
      tree_norm(M, L, sink, inv, lse);
#pragma unroll
      for (int k = 0; k < 4; k++)
        out[lane + 32 * k] = make_uint2(pack_bf16(a[4 * k] * inv, a[4 * k + 1] * inv),
                                        pack_bf16(a[4 * k + 2] * inv, a[4 * k + 3] * inv));
    } else {
      // the row's warps, of which each then adds up its share of the dims
#pragma unroll
      for (int k = 0; k < 4; k++)
        reinterpret_cast<float4*>(so[warp])[lane + 32 * k] = make_float4(a[4 * k], a[4 * k + 1], a[4 * k + 2], a[4 * k + 3]);
      if (lane == 0) sml[warp] = make_float2(M, L);
      __syncthreads();
      const int w0 = warp - part;
      const float2 ml = lane < split ? sml[w0 + lane] : make_float2(-INFINITY, 0.f);
      M = warp_max(ml.x);
      const float w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M);
      L = warp_sum(ml.y * w);
      float wj[8];
#pragma unroll
      for (int j = 0; j < 8; j++) wj[j] = __shfl_sync(0xffffffffu, w, j);
      tree_norm(M, L, sink, inv, lse);
      const int units = 128 / split;
      for (int u = part * units + lane; pair >= 0 && u < (part + 1) * units; u += 32) {
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          if (j >= split) break;
          const float4 x = reinterpret_cast<const float4*>(so[w0 + j])[u];
          o.x = fmaf(x.x, wj[j], o.x);
          o.y = fmaf(x.y, wj[j], o.y);
          o.z = fmaf(x.z, wj[j], o.z);
          o.w = fmaf(x.w, wj[j], o.w);
        }
        out[u] = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
      }
      __syncthreads();
    }
    if (p.lse && pair >= 0 && part == 0 && lane == 0) p.lse[orow] = lse;
  }
}

}  // namespace

// As many pairs as there can be tiles, up to one per two SMs.
int64_t tree_pairs(const TreeArgs& a, int group_rows, int tile) {
  const int64_t groups = (a.s * a.h + group_rows - 1) / group_rows;
  const int64_t tiles = a.b * groups * ((a.max_len + tile - 1) / tile);
  return tiles < 1 ? 1 : (tiles < kTreePairs ? tiles : kTreePairs);
}

TreeShape tree_shape(const TreeArgs& a, int group_rows, int64_t pairs) {
  TreeShape p{};
  p.table = a.block_table;
  p.seqlens = a.seqlens;
  p.tree_lens = a.tree_lens;
  p.mask = a.mask;
  p.err = device_error_word();
  p.max_pages = a.max_pages;
  p.num_pages = a.num_pages;
  p.mask_stride = a.mask_stride;
  p.b = (int)a.b;
  p.s = (int)a.s;
  p.h = (int)a.h;
  p.max_len = (int)a.max_len;
  p.page_blocks = (int)(a.page_size / 64);
  p.groups = (int)((a.s * a.h + group_rows - 1) / group_rows);
  // teams of `groups` pairs when they leave at most 4 of the 74 pairs idle
  p.team = p.groups > 1 && pairs == kTreePairs &&
           kTreePairs / p.groups * p.groups >= kTreePairs - 4;
  p.row_cost = kTreeRowCost;
  return p;
}

size_t attn_tree_workspace(const TreeArgs& a) {
  return (size_t)tree_pairs(a, Cut::kGroupRows, kTile) * (2 * 128 * (512 + 2) * 4 + 16);
}

cudaError_t launch_attn_tree_sm100(const TreeArgs& a, void* ws, cudaStream_t st) {
  const int64_t rows = a.s * a.h;
  const int64_t pairs = tree_pairs(a, Cut::kGroupRows, kTile);
  CUtensorMap tq, tk, tv;
  {
    // Q as [b][chunks][rows][64 values]: three chunks of a CTA's 64 rows in a box
    const uint64_t row = (uint64_t)a.d_qk * 2;
    const uint64_t dims[4] = {64, (uint64_t)rows, (uint64_t)(a.d_qk / 64), (uint64_t)a.b};
    const uint64_t strides[3] = {row, 128, (uint64_t)rows * row};
    const uint32_t box[4] = {64, 64, 3, 1};
    if (!make_tmap(&tq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, a.q, dims, strides, box,
                   CU_TENSOR_MAP_SWIZZLE_128B))
      return cudaErrorInvalidValue;
  }
  // K and V: the cache as [64-token blocks][64 tokens][chunks][64 values], so
  // that one box carries several chunks of a block
  const int64_t blocks = a.num_pages * (a.page_size / 64);
  const uint64_t dims[4] = {64, 64, (uint64_t)(a.d_qk / 64), (uint64_t)blocks};
  const uint64_t strides[3] = {(uint64_t)a.d_qk * 2, 128, (uint64_t)a.d_qk * 128};
  const uint32_t kbox[4] = {64, 64, 3, 1}, vbox[4] = {64, 64, 4, 1};
  if (!make_tmap(&tk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, a.cache, dims, strides, kbox,
                 CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tmap(&tv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, a.cache, dims, strides, vbox,
                 CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  TreeParams p{};
  p.sh = tree_shape(a, Cut::kGroupRows, pairs);
  p.out = reinterpret_cast<__nv_bfloat16*>(a.o);
  p.lse = a.lse;
  p.sink = a.sink;
  p.chunks = (int)(a.d_qk / 64);
  p.score_scale = tree_score_scale(a.scale, 1.4426950408889634, a.d_qk, (int)(a.d_qk / 16));  // one chain
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_ml = p.part_o + (size_t)pairs * 2 * 128 * 512;
  p.desc = reinterpret_cast<int4*>(p.part_ml + (size_t)pairs * 2 * 128 * 2);
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem((const void*)attn_tree_sm100_kernel, kSmemBytes, done);
  if (e != cudaSuccess) return e;
  e = launch_early(attn_tree_sm100_kernel, dim3((unsigned)(2 * pairs)), 1, kThreads, kSmemBytes, st,
                   tq, tk, tv, p);
  if (e != cudaSuccess || pairs == 1) return e;  // one pair: no row is shared
  // the merge by how many groups share the pairs (one sequence of 8 nodes x 16 heads x 8192:
  // 18.5 us with the merge of few groups, 28.6 with the other; of 23 sequences of up to 7
  // groups, 512 wide, 56.4 and 54.0)
  const int64_t groups = a.b * p.sh.groups;
  if (4 * groups > pairs)
    return launch_early(tree_combine_kernel, dim3((unsigned)pairs, 16), 1, 256, 0, st, p);
  const int64_t shared_rows = groups * std::min<int64_t>(rows, 128);  // at most a row a block
  return launch_early(tree_combine_few_kernel, dim3((unsigned)std::min<int64_t>(shared_rows, kFewBlocks)), 1,
                      256, 0, st, p, (int)pairs);
}

}  // namespace qcau
