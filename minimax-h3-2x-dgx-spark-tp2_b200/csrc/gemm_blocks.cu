// Block-scaled FP8 products on the 5th-generation tensor cores:
//   y[m, n] = out( sum_j sa[m, j] * sb[n / 128, j] * sum_{k in block j} a[m, k] * w[n, k] )  (+ bias[n])
// with e4m3 operands and one fp32 scale per row of a and 128 values of K, and per 128 x 128 tile of w; dense, or grouped
// by expert (rows offsets[e] .. offsets[e+1] of a use w[e], read on the device: no host copy of the sizes).
//
// The scales change every 128 values of K, so the tensor core's accumulator holds one block's product only: each
// K step of 128 is its own accumulator in TMEM, and the epilogue warps add it, scaled, to fp32 running sums in
// registers while the next step's MMAs fill another TMEM buffer.  Both forms below are that loop:
//
//   wide    (many rows): CTA pairs with 2-SM MMAs over 256 rows x 256 columns, or single CTAs over 128 x 256.  Thread = output
//           row, so sa * sb is one scalar per thread and step and the promotion costs one FMA per element: 8 warps x 128 FMAs
//           per 512 tensor cycles.  128 running sums per thread, two 256-column TMEM buffers.
//   narrow  (few rows): the operands swapped, D^T = w a^T: 128 weight rows x NT tokens (NT = 16, 32 or 64) per CTA, so that
//           a tile streams the weight once with no tensor work on absent rows.
//
// Where the tiles are few, K is split over a cluster of CTAs that add their sums through distributed shared memory in the
// order of K (the result does not depend on timing).
//
// What bounds them.  Wide, 62,496 x 15,360 x 5,120: 5.0 to 5.4 ms, 1.9 PFLOP/s, at the power cap (about 1.5 GHz); the tensor
// pipe alone would take 512 cycles a step, a step takes about 1,000.  A TMEM buffer goes round between the MMAs, the eight
// epilogue warps (of both SMs) and back: 512 cycles of MMAs, then commit, TMEM reads under the additions and the arrival,
// 1,200 more where the other SM is part of it, and 512 columns hold only two buffers.  Half as wide buffers, four of them:
// 6.1 ms (twice the handshakes).  Sixteen epilogue warps of 64 columns: 7.7 ms.  Two additions per instruction (fma.rn.f32x2):
// fewer cycles alone, more here.  Single CTAs have no cross-SM handshake, but 48 KB a step and SM to fetch for 32, at
// the same speed: 777 x 5,120 x 13,824 65 us; with a third of the loads left out 60, with most of the additions left out 60,
// with both 56.  Spinning waits and L2 prefetches ahead of the ring gain nothing.  Narrow: the weight's bytes, and at one row
// the start and end of a call: 1 x 15,360 x 5,120 16.4 us (12.2 at copy speed), 1 x 5,120 x 5,120 8.5 (4.1).
//
// Spills (-Xptxas -v: 132 bytes in the pair form, 116 in the single one, 16 in narrow<64>) lie outside the loop over K: the local
// loads and stores of a launch are the same for twice the K.  With K in parts pairs have five loads and a store a step and
// epilogue warp in it, single CTAs two and one.
//
// Every wait is bounded (common.cuh); no TMA multicast.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "common.cuh"

namespace h3b {
namespace {

constexpr int BLK = 128;
constexpr int MAX_DEVICES = 64;

struct Params {
  int64_t T, N;       // rows of a, rows of w (of one expert)
  int num_kb;         // 128-value blocks of K
  int num_nb;         // column tiles (256 wide, or 128 weight rows narrow)
  int split;          // CTAs (wide: pairs of CTAs) of a cluster that share a tile, each with a part of K
  int experts;        // groups; dense: 1 without offsets
  const void* offsets;
  int off64;          // offsets are int64 (else int32)
  const float* sa;
  int64_t sa_row, sa_blk;
  const float* sb;
  int64_t sb_exp, sb_row, sb_blk;
  const __nv_bfloat16* bias;
  uint16_t* y;
  int64_t ldy;
  int out_f16;
  int tma_out;        // wide: whole slices leave through TMA stores
  int y_align;        // rows of y are aligned to this many bytes: 16, 8, 4 or 2
  WaitCtl wc;
};

__device__ __forceinline__ int64_t group_bound(const Params& p, int e) {
  return p.off64 ? static_cast<const int64_t*>(p.offsets)[e]
                 : static_cast<int64_t>(static_cast<const int32_t*>(p.offsets)[e]);
}

__device__ __forceinline__ uint16_t to_out(float v, int f16) {
  return f16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}
__device__ __forceinline__ uint32_t to_out2(float lo, float hi, int f16) {
  return static_cast<uint32_t>(to_out(lo, f16)) | (static_cast<uint32_t>(to_out(hi, f16)) << 16);
}

// four columns n .. n + 3 of y at element `at`, with the bias: those below N
__device__ __forceinline__ void store4(const Params& p, int64_t at, int64_t n, float (&v)[4]) {
  if (p.bias != nullptr) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < p.N) v[j] += __bfloat162float(p.bias[n + j]);
  }
  const uint32_t lo = to_out2(v[0], v[1], p.out_f16), hi = to_out2(v[2], v[3], p.out_f16);
  uint16_t* dst = p.y + at;
  if (p.y_align >= 8 && n + 4 <= p.N) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
  } else if (p.y_align >= 4 && n + 4 <= p.N) {
    reinterpret_cast<uint32_t*>(dst)[0] = lo;
    reinterpret_cast<uint32_t*>(dst)[1] = hi;
  } else {
    const uint32_t w[2] = {lo, hi};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < p.N) dst[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
  }
}

// Walk over the row tiles of the groups in order.  `before`: tiles of the experts below e0.  find() places tile t
// (non-decreasing over calls) with the whole warp: 32 experts' bounds per step and a shuffle scan.  A group whose bounds
// are not 0 <= lo <= hi <= T has no tiles, and `bad` is set.  From then on a group's rows start at `reach` at the earliest, the
// largest end before it: no row is in two groups, so that there are never more tiles than the launch has counted on.
// (While no bound is bad they are in order, and lo is `reach`.)
template <int ROWS>
struct Walk {
  int e0 = 0;
  int64_t before = 0;
  bool bad = false;    // the same for the whole warp
  int reach = 0;       // of the experts below e0
  int e;               // the tile found: expert, its rows [lo, hi), row blocks and the tile's index within the expert
  int64_t lo, hi;
  int blocks, r;
  __device__ __forceinline__ bool find(const Params& p, int64_t t, int per_block) {
    const int lane = threadIdx.x & 31;
    while (e0 < p.experts) {
      int64_t l = 0, h = 0;
      bool wrong = false;
      if (e0 + lane < p.experts) {
        if (p.offsets == nullptr) {
          h = p.T;
        } else {
          l = group_bound(p, e0 + lane);
          h = group_bound(p, e0 + lane + 1);
          wrong = l < 0 || h < l || h > p.T;
          if (wrong) l = h = 0;
        }
      }
      const int last = static_cast<int>(h);  // at most T, which is below 2^31
      bad |= __any_sync(0xffffffffu, wrong);
      if (bad) {
        int most = max(last, reach);  // of the groups up to this lane's, then before it
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, most, o);
          if (lane >= o) most = max(most, up);
        }
        most = __shfl_up_sync(0xffffffffu, most, 1);
        if (lane == 0) most = reach;
        l = l > most ? l : most;
        h = h > l ? h : l;
      }
      const int mine = static_cast<int>((h - l + ROWS - 1) / ROWS);
      int64_t sum = static_cast<int64_t>(mine) * per_block;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      const int64_t total = __shfl_sync(0xffffffffu, sum, 31);
      if (t < before + total) {
        const int64_t rel = t - before;
        const int src = __ffs(__ballot_sync(0xffffffffu, sum > rel)) - 1;
        e = e0 + src;
        lo = __shfl_sync(0xffffffffu, l, src);
        hi = __shfl_sync(0xffffffffu, h, src);
        blocks = __shfl_sync(0xffffffffu, mine, src);
        r = static_cast<int>(rel - (__shfl_sync(0xffffffffu, sum, src) - static_cast<int64_t>(blocks) * per_block));
        return true;
      }
      before += total;
      e0 += 32;
      reach = max(reach, __reduce_max_sync(0xffffffffu, last));
    }
    return false;
  }
};

// whether this cluster starts: the status word as its first CTA read it (so that all its CTAs take the same way).
// Call between two cluster-wide barriers that keep the first CTA's shared memory alive.
__device__ __forceinline__ bool cluster_flag(uint32_t flag_smem) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(flag_smem, 0)) : "memory");
  return v != 0;
}

// A wait of this CTA has given up, so its sums are not whole: every CTA of the cluster (they add each other's) is told, and
// stores nothing.  `flag`: cleared before the cluster's first barrier, read behind one that follows this.
__device__ __forceinline__ void give_up(uint32_t flag_smem, int ctas) {
  for (int r = 0; r < ctas; ++r)
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_shared(flag_smem, static_cast<uint32_t>(r))), "r"(1u)
                 : "memory");
}

// ---------------------------------------------------------------------------------------------------------------
// wide: 256 x 256 tiles by CTA pairs or 128 x 256 by single CTAs, running sums in registers
// ---------------------------------------------------------------------------------------------------------------
namespace wide {

constexpr int BM = 128, BN = 256;
// a stage: 128 rows of a, and of w its half of the pair's 256 rows or (one CTA) all of them, 128 bytes each
__host__ __device__ constexpr int stages(bool pair) { return pair ? 6 : 4; }
__host__ __device__ constexpr int stage_bytes(bool pair) { return (BM + (pair ? BN / 2 : BN)) * BLK; }
constexpr int RING_BYTES = stages(true) * stage_bytes(true);
static_assert(RING_BYTES == stages(false) * stage_bytes(false), "the rings take the same room");
constexpr int EPI_WARPS = 8, FIRST_EPI = 4, THREADS = 32 * (FIRST_EPI + EPI_WARPS);
// Clusters of 8 CTAs at most: 4 parts for pairs.  What a round of tiles takes besides its steps, in steps: with 7 or less, 512
// x 5,120 x 5,120 goes to 2 rounds in parts, 37 us for 26; at 28 nothing measured changed.  Without parts 256 x 1,024 x 13,824
// takes 53 us for 21, 256 x 5,120 x 13,824 57 for 33
constexpr int MAX_SPLIT = 8, ROUND_COST = 14;
constexpr int WARP_STAGING = 32 * 128;              // 32 rows x 64 columns of 16-bit output
constexpr int SMEM = RING_BYTES + 1024 + 1024 + EPI_WARPS * WARP_STAGING;
static_assert(SMEM <= 232448, "shared memory");
// row blocks that share a column block's w tile in L2, as in the per-token product (4 and 8 measure the same, 32 takes 3 %
// longer at 8,192 x 15,360 x 5,120)
constexpr int GROUP_M = 16;

// tile r of a group of `blocks` row blocks -> (row block, column block)
__device__ __forceinline__ void coords(int r, int blocks, int num_nb, int& mb, int& nb) {
  const int in_group = GROUP_M * num_nb;
  const int g = r / in_group, first = g * GROUP_M;
  const int size = min(blocks - first, GROUP_M);
  const int q = r - g * in_group;
  mb = first + q % size;
  nb = q / size;
}

// SPLIT: clusters of p.split pairs take a tile each, every pair a part of K
template <bool PAIR, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1)
    kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
           const __grid_constant__ CUtensorMap tmY, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int STAGES = stages(PAIR), STAGE_BYTES = stage_bytes(PAIR), CTAS = PAIR ? 2 : 1;
  constexpr uint32_t IDESC = idesc_make(FMT_E4M3, FMT_E4M3, 0, CTAS * BM, BN);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + RING_BYTES);
  // bars: full[STAGES], used[STAGES], tempty[2], done; then the TMEM address, the start and give-up flags.  used[s]: the MMAs of
  // the step in stage s are complete, which frees the stage for the producer and hands the step's accumulator to the
  // epilogue (one commit per step for both)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 3);
  uint32_t* start_flag = tmem_slot + 1;
  volatile uint32_t* gave_up = start_flag + 1;
  uint8_t* staging = smem + RING_BYTES + 1024;
  const uint32_t smem0 = smem_u32(smem), bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto used_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto tempty_bar = [&](int b) { return bar0 + 8u * (2 * STAGES + b); };
  const uint32_t done_bar = bar0 + 8u * (2 * STAGES + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR || SPLIT ? cluster_ctarank() : 0u;
  const int crank = PAIR ? static_cast<int>(rank & 1u) : 0;  // 0: the pair's leader (issues the MMAs)
  const int part = SPLIT ? static_cast<int>(rank / CTAS) : 0;  // the part of K: steps [kb0, kb1)
  const uint32_t leader = static_cast<uint32_t>(part * CTAS);
  const int kb0 = SPLIT ? static_cast<int>(static_cast<int64_t>(p.num_kb) * part / p.split) : 0;
  const int kb1 = SPLIT ? static_cast<int>(static_cast<int64_t>(p.num_kb) * (part + 1) / p.split) : p.num_kb;
  const uint16_t pair_mask = static_cast<uint16_t>(3u << leader);
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(used_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) mbar_init(tempty_bar(b), CTAS * EPI_WARPS);  // every epilogue warp (of both CTAs)
    mbar_init(done_bar, 2);
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmW);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(smem_u32(tmem_slot), 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), 512);
      tmem_relinquish();
    }
  }
  pdl_wait();
  if (threadIdx.x == 0) {
    *start_flag = status_bad(p.wc) ? 0u : 1u;
    *gave_up = 0u;
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  // no pdl_launch in this form: with the next kernel starting as CTAs leave, an FFN chain of 256 rows takes 92 us for 89
  const uint32_t tmem_base = *tmem_slot;
  const bool start = cluster_flag(smem_u32(start_flag));  // of the cluster's first CTA
  const int first_tile = static_cast<int>(cluster_id_x()), tile_step = static_cast<int>(cluster_count_x());
  // parts of K: a cluster takes one tile, and the last find only looks for bad bounds
  auto next_tile = [&](int64_t t) { return SPLIT ? INT64_MAX : t + tile_step; };
  Walk<CTAS * BM> walk;
  bool ok = true;  // no wait of this thread's role has given up

  if (warp < FIRST_EPI) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (start && warp == 0) {
      // ---------------- TMA producer (both CTAs; stages complete on the leader's full barrier) ----------------
      const uint32_t lead_full0 = mapa_shared(full_bar(0), leader);
      int stage = 0;
      uint32_t phase = 0;
      uint32_t loaded = 0, last = 0;  // per stage: loaded at all, parity of its last load
      for (int64_t t = first_tile; ok && walk.find(p, t, p.num_nb); t = next_tile(t)) {
        int mb, nb;
        coords(walk.r, walk.blocks, p.num_nb, mb, nb);
        const int arow = static_cast<int>(walk.lo) + (CTAS * mb + crank) * BM;
        const int wrow = nb * BN + crank * BM;
        if (lane == 0) {
          for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait_inline(used_bar(stage), phase ^ 1u, p.wc)) {
              ok = false;
              break;
            }
            const uint32_t sA = smem0 + stage * STAGE_BYTES;
            if (crank == 0) mbar_arrive_expect_tx(full_bar(stage), CTAS * STAGE_BYTES);
            if constexpr (PAIR) {
              tma_load_2d_pair(sA, &tmA, lead_full0 + 8u * stage, kb * BLK, arow);
              tma_load_3d_pair(sA + BM * BLK, &tmW, lead_full0 + 8u * stage, kb * BLK, wrow, walk.e);
            } else {
              tma_load_2d(sA, &tmA, full_bar(stage), kb * BLK, arow);
              tma_load_3d(sA + BM * BLK, &tmW, full_bar(stage), kb * BLK, wrow, walk.e);
              tma_load_3d(sA + 2 * BM * BLK, &tmW, full_bar(stage), kb * BLK, wrow + BM, walk.e);
            }
            loaded |= 1u << stage;
            last = (last & ~(1u << stage)) | (phase << stage);
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
      }
      // drain: no TMA write may be in flight into shared memory that the CTA is about to give up.  The leader sees
      // both CTAs' bytes on its full barriers; the partner's last load of a stage has landed once the leader's MMAs
      // consumed it.
      if (lane == 0) {
        for (int s = 0; s < STAGES; ++s) {
          if (!(loaded >> s & 1u)) continue;
          const uint32_t bar = crank == 0 ? full_bar(s) : used_bar(s), par = last >> s & 1u;
          const uint64_t t0 = globaltimer();
          while (!mbar_try_wait(bar, par) && globaltimer() - t0 < p.wc.timeout) {
          }
        }
      }
    } else if (start && (warp == 1 || warp == 2)) {
      if (crank == 0) {
        // ---------------- MMA issuers (the leader only): one accumulator per 128-value step of K ----------------
        // Two warps take the steps in turn, each with a TMEM buffer of its own: a thread that issues MMAs is held while
        // the tensor pipe is busy, and its waits and commits (~350 cycles a step) would leave the pipe idle.
        const int b = warp - 1;
        uint32_t it = 0;  // steps before this tile
        for (int64_t t = first_tile; ok && walk.find(p, t, p.num_nb); t = next_tile(t), it += kb1 - kb0) {
          if (lane == 0) {
            for (uint32_t i = it + ((it ^ b) & 1u); i < it + (kb1 - kb0); i += 2) {
              const uint32_t round = i / STAGES, stage = i - round * STAGES;
              if (!mbar_wait_inline(full_bar(stage), round & 1u, p.wc) ||
                  !mbar_wait_inline(tempty_bar(b), ((i >> 1) & 1u) ^ 1u, p.wc)) {
                ok = false;
                break;
              }
              tc_fence_after();
              const uint32_t sA = smem0 + stage * STAGE_BYTES;
              const uint64_t adesc = sdesc_sw128(sA, 16, 1024), bdesc = sdesc_sw128(sA + BM * BLK, 16, 1024);
#pragma unroll
              for (int kk = 0; kk < BLK / 32; ++kk) {
                const uint32_t d = tmem_base + static_cast<uint32_t>(b * BN);
                if constexpr (PAIR)
                  umma_f8_ss_pair(d, adesc + 2u * kk, bdesc + 2u * kk, IDESC, kk != 0);
                else
                  umma_f8_ss(d, adesc + 2u * kk, bdesc + 2u * kk, IDESC, kk != 0);
              }
              if constexpr (PAIR)
                umma_commit_pair_mc(used_bar(stage), pair_mask);
              else
                umma_commit(used_bar(stage));
            }
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
        }
        if (lane == 0) {  // every issued MMA completes before TMEM is released
          if constexpr (PAIR)
            umma_commit_pair(done_bar);
          else
            umma_commit(done_bar);
          const uint64_t t0 = globaltimer();
          while (!mbar_try_wait(done_bar, 0) && globaltimer() - t0 < p.wc.timeout) {
          }
        }
      }
    }
    if constexpr (SPLIT) {  // the barriers of the epilogue's end phase
      __syncwarp();
      __syncthreads();
      cluster_sync();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    if (start) {
      // ---------------- epilogue warps: 32 rows x 128 columns of running sums each ----------------
      const int sub = warp & 3, half = (warp - FIRST_EPI) >> 2;
      const uint32_t tmine = tmem_base + (static_cast<uint32_t>(sub * 32) << 16) + static_cast<uint32_t>(half * 128);
      const uint32_t lead_tempty0 = mapa_shared(tempty_bar(0), leader);
      uint4* stg = reinterpret_cast<uint4*>(staging + (warp - FIRST_EPI) * WARP_STAGING);
      uint32_t it = 0, phase = 0;
      int stage = 0;
      bool have = false;
      float acc[128];
      int mb = 0, nb = 0;
      int64_t m0 = 0, n0 = 0;  // the warp's first row and column
      const float *sap = p.sa, *sbp = p.sb;
      // the scales of the next two steps are on their way while a step is added; pairs ask for those of the next tile while one
      // is stored (8,192 x 15,360 x 5,120 705 us for 717 in long runs; single CTAs, short of registers, lose 1 %)
      float sa0 = 0.0f, sb0 = 0.0f, sa1 = 0.0f, sb1 = 0.0f;
      auto find = [&](int64_t t) {
        if (!walk.find(p, t, p.num_nb)) return false;
        coords(walk.r, walk.blocks, p.num_nb, mb, nb);
        m0 = walk.lo + (CTAS * mb + crank) * BM + sub * 32;
        n0 = static_cast<int64_t>(nb) * BN + half * 128;
        sap = p.sa + (m0 + lane < walk.hi ? m0 + lane : walk.lo) * p.sa_row;
        sbp = p.sb + walk.e * p.sb_exp + (n0 < p.N ? n0 / BLK : 0) * p.sb_row;
        sa0 = sap[kb0 * p.sa_blk];
        sb0 = sbp[kb0 * p.sb_blk];
        if (kb0 + 1 < kb1) {
          sa1 = sap[(kb0 + 1) * p.sa_blk];
          sb1 = sbp[(kb0 + 1) * p.sb_blk];
        }
        return true;
      };
      int64_t t = first_tile;
      bool more = find(t);
      while (more) {
#pragma unroll
        for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
#pragma unroll 1
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const float s = sa0 * sb0;
          sa0 = sa1;
          sb0 = sb1;
          if (kb + 2 < kb1) {
            sa1 = sap[(kb + 2) * p.sa_blk];
            sb1 = sbp[(kb + 2) * p.sb_blk];
          }
          const int b = it & 1;
          if (!__all_sync(0xffffffffu, mbar_wait_inline(used_bar(stage), phase, p.wc))) {
            ok = false;  // for the whole warp: the TMEM loads below need all of it
            break;
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
          tc_fence_after();
          const uint32_t tcur = tmine + static_cast<uint32_t>(b * BN);
          // 32-column slices, two ahead: the buffer is read (and given back) after half of the additions
          uint32_t ra[32], rb[32];
          auto add = [&](const uint32_t (&r)[32], int c) {
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[c + i] = fmaf(__uint_as_float(r[i]), s, acc[c + i]);
          };
          tmem_ld32(tcur, ra);
          tmem_ld32(tcur + 32, rb);
          tmem_ld_wait();
          reg_fence(ra);
          reg_fence(rb);
          add(ra, 0);
          tmem_ld32(tcur + 64, ra);
          add(rb, 32);
          tmem_ld32(tcur + 96, rb);
          tmem_ld_wait();
          reg_fence(ra);
          reg_fence(rb);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (PAIR)
              mbar_arrive_cluster_relaxed(lead_tempty0 + 8u * b);
            else
              mbar_arrive(tempty_bar(b));
          }
          add(ra, 64);
          add(rb, 96);
        }
        if (!ok) break;
        if constexpr (SPLIT) {  // there is a cluster for every tile
          have = true;
          break;
        }
        const int64_t m_at = m0, n_at = n0, hi = walk.hi;
        t = next_tile(t);
        if constexpr (PAIR) more = find(t);
        if (p.bias != nullptr) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (n_at + i < p.N) acc[i] += __bfloat162float(p.bias[n_at + i]);
        }
        // two halves of 64 columns through the warp's staging: 32 rows x 128 bytes in the 128-byte swizzle
        const bool whole = p.tma_out && m_at + 32 <= hi;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (p.tma_out && lane == 0) bulk_wait_read0();
          __syncwarp();
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const float* v = acc + 64 * h + 8 * g;
            stg[lane * 8 + (g ^ (lane & 7))] = make_uint4(to_out2(v[0], v[1], p.out_f16), to_out2(v[2], v[3], p.out_f16),
                                                          to_out2(v[4], v[5], p.out_f16), to_out2(v[6], v[7], p.out_f16));
          }
          const int64_t nh = n_at + 64 * h;
          // a TMA store ends at the map's edge rounded up to 16 bytes: slices across an odd edge leave row by row
          if (whole && (nh + 64 <= p.N || p.N % 8 == 0)) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && nh < p.N) {
              tma_store_2d(&tmY, smem_u32(stg), static_cast<int32_t>(nh), static_cast<int32_t>(m_at));
              bulk_commit();
            }
          } else {
            __syncwarp();
            if (p.y_align == 16) {
#pragma unroll 1
              for (int i = lane; i < 32 * 8; i += 32) {
                const int r = i >> 3, g = i & 7;
                const int64_t m = m_at + r, n = nh + 8 * g;
                if (m >= hi || n >= p.N) continue;
                const uint4 val = stg[r * 8 + (g ^ (r & 7))];
                uint16_t* dst = p.y + m * p.ldy + n;
                if (n + 8 <= p.N) {
                  *reinterpret_cast<uint4*>(dst) = val;
                } else {
                  const uint32_t w[4] = {val.x, val.y, val.z, val.w};
#pragma unroll
                  for (int e2 = 0; e2 < 8; ++e2)
                    if (n + e2 < p.N) dst[e2] = static_cast<uint16_t>(w[e2 >> 1] >> (16 * (e2 & 1)));
                }
              }
            } else {
              // a row per instruction, two columns a lane: from the row's first column, or from its second where only that one
              // is 4-byte aligned: 30,000 x 5,001 x 64 in 275 us (a value a lane: 308; eight values a lane, one by one: 546)
              const int left = static_cast<int>(p.N - nh < 64 ? p.N - nh : 64), c = 2 * lane;
              const int rows = static_cast<int>(hi - m_at < 32 ? hi - m_at : 32);
              uint16_t* dst = p.y + m_at * p.ldy + nh + c;
#pragma unroll 4
              for (int r = 0; r < rows; ++r, dst += p.ldy) {
                const uint32_t val = reinterpret_cast<const uint32_t*>(stg)[(r * 8 + (lane >> 2 ^ (r & 7))) * 4 + (lane & 3)];
                if ((reinterpret_cast<uintptr_t>(dst) & 2u) == 0) {  // the same for all lanes
                  if (c + 2 <= left)
                    *reinterpret_cast<uint32_t*>(dst) = val;
                  else if (c < left)
                    *dst = static_cast<uint16_t>(val);
                } else {
                  const uint32_t next = __shfl_down_sync(0xffffffffu, val, 1);
                  if (c + 3 <= left)
                    *reinterpret_cast<uint32_t*>(dst + 1) = __byte_perm(val, next, 0x5432);
                  else if (c + 1 < left)
                    dst[1] = static_cast<uint16_t>(val >> 16);
                  if (lane == 0 && left > 0) *dst = static_cast<uint16_t>(val);
                }
              }
            }
            __syncwarp();
          }
        }
        if constexpr (!PAIR) more = find(t);
      }
      if (p.tma_out && lane == 0) bulk_wait_all0();  // this warp's TMA stores are complete before the CTA leaves
      if constexpr (SPLIT) {
        // the parts' sums through the idle rings, [64][128 rows][4 columns] fp32 each; part r adds and stores the groups
        // r, r + split, ... of 16 columns, the parts in the order of K.  (Lanes along the columns of a row instead, for wider
        // stores: 100 x 5,120 x 5,120 in 23.4 us for 15.9, the reads of other CTAs' memory want lanes side by side)
        __syncthreads();  // every load has landed and every MMA has read the ring
        float4* sums = reinterpret_cast<float4*>(smem);
        if (!ok && lane == 0) give_up(smem_u32(start_flag + 1), CTAS * p.split);
        if (have) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            sums[(half * 32 + i) * BM + sub * 32 + lane] =
                make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
        }
        __syncwarp();
        cluster_sync();
        const int64_t m0 = walk.lo + (CTAS * mb + crank) * BM + sub * 32;  // the warp's first row
        if (have && *gave_up == 0u && m0 < walk.hi) {
          for (int g = part + half * p.split; g < BN / 16; g += 2 * p.split) {
            const int64_t n = static_cast<int64_t>(nb) * BN + 16 * g;
            if (n >= p.N) break;
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = 0.0f;
            for (int q0 = 0; q0 < p.split && m0 + lane < walk.hi; q0 += 4) {  // four parts' loads on their way at once
              float x[4][16];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                if (q0 + q >= p.split) continue;
                const uint32_t src = mapa_shared(smem0 + static_cast<uint32_t>((4 * g * BM + sub * 32 + lane) * 16),
                                                 static_cast<uint32_t>(CTAS * (q0 + q) + crank));
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                               : "=f"(x[q][i]), "=f"(x[q][i + 1]), "=f"(x[q][i + 2]), "=f"(x[q][i + 3])
                               : "r"(src + 4u * BM * i)
                               : "memory");
              }
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                if (q0 + q >= p.split) continue;
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] += x[q][i];
              }
            }
            if (p.bias != nullptr) {
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (n + i < p.N) v[i] += __bfloat162float(p.bias[n + i]);
            }
            uint4 out[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float* f = v + 8 * h;
              out[h] = make_uint4(to_out2(f[0], f[1], p.out_f16), to_out2(f[2], f[3], p.out_f16),
                                  to_out2(f[4], f[5], p.out_f16), to_out2(f[6], f[7], p.out_f16));
            }
            if (p.y_align == 16 && n + 16 <= p.N) {
              if (m0 + lane < walk.hi) {
                uint4* dst = reinterpret_cast<uint4*>(p.y + (m0 + lane) * p.ldy + n);
                dst[0] = out[0];
                dst[1] = out[1];
              }
            } else {  // two rows of 16 columns per instruction, through the warp's staging
              stg[2 * lane] = out[0];
              stg[2 * lane + 1] = out[1];
              __syncwarp();
              const int c = lane & 15;
#pragma unroll 4
              for (int r = lane >> 4; r < 32; r += 2)
                if (m0 + r < walk.hi && n + c < p.N)
                  p.y[(m0 + r) * p.ldy + n + c] = reinterpret_cast<const uint16_t*>(stg)[16 * r + c];
              __syncwarp();
            }
          }
        }
      }
    } else if constexpr (SPLIT) {  // the barriers of the end phase
      __syncthreads();
      cluster_sync();
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();  // neither CTA leaves (or frees the pair's TMEM) while the other may still signal it
  tc_fence_after();
  if (warp == 1) {
    if constexpr (PAIR)
      tmem_dealloc_pair(tmem_base, 512);
    else
      tmem_dealloc(tmem_base, 512);
  }
  if (walk.bad && lane == 0) record_data_error(p.wc, H3B_EINVAL);
}

}  // namespace wide

// ---------------------------------------------------------------------------------------------------------------
// narrow: 128 weight rows x NT tokens per CTA, K split over the cluster
// ---------------------------------------------------------------------------------------------------------------
namespace narrow {

// producer, MMA issuer, epilogue: 4 row quarters, and where a tile has more than 16 tokens 2 token halves (4 warps against 8:
// 1 x 15,360 x 5,120 16.6 us for 16.7, 32 x 5,120 x 13,824 17.8 for 17.6, 64 x 15,360 x 5,120 22.5 for 21.2)
__host__ __device__ constexpr int epi_warps(int nt) { return nt > 16 ? 8 : 4; }
__host__ __device__ constexpr int threads(int nt) { return 64 + 32 * epi_warps(nt); }
constexpr int CHUNK = 16;                  // K steps whose scales are staged together
// as in the wide form: with 0, 48 rows over 64 experts of 4,096 x 5,120 take 118 us for 105 (10 and 40: 105).  Without parts
// 1 x 5,120 x 5,120 takes 16.6 us for 8.2, 16 x 5,120 x 13,824 40 for 17
constexpr int MAX_SPLIT = 8, ROUND_COST = 20;
constexpr int PREFETCH = 3;                // K steps of the weight asked for ahead of the kernel before
constexpr int NBUF = 4;                    // TMEM buffers of NT columns: steps between the MMAs and the epilogue

__host__ __device__ constexpr int stage_bytes(int nt) { return (BLK + nt) * BLK; }
// two CTAs per SM with a ring of 4 each: more than the ~45 KB in flight that an SM's share of the memory bandwidth needs,
// and one CTA's start and end lie under the other's loads
constexpr int CTAS_PER_SM = 2, STAGES = 4;
// the epilogue follows the MMAs on the stages' barriers, whose phases it must not miss: MMAs run NBUF steps ahead at most
static_assert(STAGES >= NBUF, "a stage's barrier would turn twice before the epilogue looks");
// ring (reused for the sums that the cluster adds: NT x 128 fp32), barriers, two chunks of scales, alignment slack; at
// least a third of an SM's shared memory, so that no more than two CTAs fit and their TMEM never exceeds 512 columns (a
// CTA that waited for TMEM while its cluster waits for it could wait forever)
__host__ __device__ constexpr int smem(int nt) {
  const int need = STAGES * stage_bytes(nt) + 256 + 2 * CHUNK * nt * 4 + 1024;
  return need < 79 * 1024 ? 79 * 1024 : need;
}
__host__ __device__ constexpr bool tmem_fits(int nt) { return (233472 / (smem(nt) + 1024)) * (NBUF * nt) <= 512; }
static_assert(tmem_fits(16) && tmem_fits(32) && tmem_fits(64), "TMEM columns");
static_assert(STAGES * stage_bytes(64) >= 64 * BLK * 4 && smem(64) + 1024 <= 233472 / CTAS_PER_SM, "shared memory");

template <int NT>
__global__ void __launch_bounds__(threads(NT), CTAS_PER_SM) kernel(const __grid_constant__ CUtensorMap tmA,
                                                                   const __grid_constant__ CUtensorMap tmW,
                                                                   const __grid_constant__ Params p) {
  constexpr int STAGE_BYTES = stage_bytes(NT);
  constexpr int EPI_WARPS = epi_warps(NT), EPI_THREADS = 32 * EPI_WARPS;
  constexpr int MINE = NT / (EPI_WARPS / 4);  // tokens of an epilogue thread
  constexpr uint32_t TMEM_COLS = NBUF * NT, IDESC = idesc_make(FMT_E4M3, FMT_E4M3, 0, 128, NT);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);
  // bars: full[STAGES], used[STAGES], tempty[NBUF], done; then the TMEM address, the start and give-up flags.  used[s]: the
  // MMAs of the step in stage s are complete, for the producer and for the epilogue.
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + NBUF + 1);
  uint32_t* start_flag = tmem_slot + 1;
  volatile uint32_t* gave_up = start_flag + 1;
  float* scales = reinterpret_cast<float*>(smem + STAGES * STAGE_BYTES + 256);  // [2][CHUNK][NT]
  float* sums = reinterpret_cast<float*>(smem);                                 // [NT][128] once the ring is idle
  static_assert(8 * (2 * STAGES + NBUF + 1) + 12 <= 256, "barrier area");
  const uint32_t smem0 = smem_u32(smem), bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto used_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto tempty_bar = [&](int b) { return bar0 + 8u * (2 * STAGES + b); };
  const uint32_t done_bar = bar0 + 8u * (2 * STAGES + NBUF);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split;  // CTAs of the cluster: they share blockIdx.x / split
  const int crank = static_cast<int>(blockIdx.x) % split, nb = static_cast<int>(blockIdx.x) / split;
  if (p.offsets != nullptr) pdl_wait();  // the bounds are the first thing read
  Walk<NT> walk;
  const bool found = walk.find(p, blockIdx.y, 1);  // the same for every CTA of the cluster
  if (!found) {
    if (walk.bad && lane == 0) record_data_error(p.wc, H3B_EINVAL);
    return;
  }
  const int64_t t0 = walk.lo + static_cast<int64_t>(walk.r) * NT;  // the tile's first row of a
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.num_kb) * crank / split);
  const int kb1 = static_cast<int>(static_cast<int64_t>(p.num_kb) * (crank + 1) / split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(used_bar(s), 1);
    }
    for (int b = 0; b < NBUF; ++b) mbar_init(tempty_bar(b), EPI_WARPS);
    mbar_init(done_bar, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmW);
  }
  // The weight's first steps on their way into L2 while the kernel before ends (it may be writing them: L2 is coherent, and
  // the loads follow pdl_wait).  A chain of calls whose weights are not in L2 gains, an FFN of one row 46.3 to 44.9 us, 1 x
  // 5,120 x 13,824 16.0 to 15.5; one whose weights are in L2 loses, 1 x 5,120 x 5,120 8.15 to 8.5.  6 steps: 15.7, 20: 16.1.
  if (threadIdx.x == 64 && p.offsets == nullptr)
    for (int kb = kb0; kb < kb1 && kb < kb0 + PREFETCH; ++kb) tma_prefetch_l2_3d(&tmW, kb * BLK, nb * BLK, 0);
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  pdl_wait();
  if (threadIdx.x == 0) {
    *start_flag = status_bad(p.wc) ? 0u : 1u;
    *gave_up = 0u;
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  pdl_launch();
  const uint32_t tmem_base = *tmem_slot;
  const bool start = cluster_flag(smem_u32(start_flag));
  float acc[MINE];
#pragma unroll
  for (int i = 0; i < MINE; ++i) acc[i] = 0.0f;

  if (start) {
    if (warp == 0) {
      if (lane == 0) {
        uint32_t loaded = 0, last = 0;
        int stage = 0;
        uint32_t phase = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait_inline(used_bar(stage), phase ^ 1u, p.wc)) break;
          const uint32_t sW = smem0 + stage * STAGE_BYTES;
          mbar_arrive_expect_tx(full_bar(stage), STAGE_BYTES);
          tma_load_3d(sW, &tmW, full_bar(stage), kb * BLK, nb * BLK, walk.e);
          tma_load_2d(sW + BLK * BLK, &tmA, full_bar(stage), kb * BLK, static_cast<int32_t>(t0));
          loaded |= 1u << stage;
          last = (last & ~(1u << stage)) | (phase << stage);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        for (int s = 0; s < STAGES; ++s) {  // no TMA write in flight when the ring is given up
          if (!(loaded >> s & 1u)) continue;
          const uint64_t c0 = globaltimer();
          while (!mbar_try_wait(full_bar(s), last >> s & 1u) && globaltimer() - c0 < p.wc.timeout) {
          }
        }
      }
      __syncwarp();
      // bad bounds behind the last tile: one CTA looks at all of them
      if (blockIdx.x == 0 && blockIdx.y == 0) {
        Walk<NT> rest;
        rest.find(p, INT64_MAX, 1);
        walk.bad |= rest.bad;
      }
    } else if (warp == 1) {
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0, it = 0;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int b = it % NBUF;
          if (!mbar_wait_inline(full_bar(stage), phase, p.wc) ||
              !mbar_wait_inline(tempty_bar(b), ((it / NBUF) & 1u) ^ 1u, p.wc))
            break;
          tc_fence_after();
          const uint32_t sW = smem0 + stage * STAGE_BYTES;
          const uint64_t wdesc = sdesc_sw128(sW, 16, 1024), adesc = sdesc_sw128(sW + BLK * BLK, 16, 1024);
#pragma unroll
          for (int kk = 0; kk < BLK / 32; ++kk)
            umma_f8_ss(tmem_base + static_cast<uint32_t>(b * NT), wdesc + 2u * kk, adesc + 2u * kk, IDESC, kk != 0);
          umma_commit(used_bar(stage));
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        umma_commit(done_bar);
        const uint64_t c0 = globaltimer();
        while (!mbar_try_wait(done_bar, 0) && globaltimer() - c0 < p.wc.timeout) {
        }
      }
    } else {
      // ---------------- epilogue: thread = weight row and MINE of the tokens ----------------
      const int sub = warp & 3, half = (warp - 2) >> 2, tid = threadIdx.x - 64;
      const uint32_t tmine = tmem_base + (static_cast<uint32_t>(sub * 32) << 16) + static_cast<uint32_t>(half * MINE);
      const float* sbp = p.sb + walk.e * p.sb_exp + nb * p.sb_row;
      // sa * sb of a chunk of steps for the tile's tokens; thread tid holds values tid, tid + EPI_THREADS, ... of [CHUNK][NT]
      constexpr int PER = CHUNK * NT / EPI_THREADS;
      float next[PER];
      auto fetch = [&](int kb) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int v = tid + EPI_THREADS * i, k = kb + v / NT, tok = v % NT;
          next[i] = (k < kb1 && t0 + tok < walk.hi)
                        ? p.sa[(t0 + tok) * p.sa_row + k * p.sa_blk] * sbp[k * p.sb_blk]
                        : 0.0f;
        }
      };
      fetch(kb0);
      uint32_t it = 0, phase = 0;
      int stage = 0;
      bool ok = true;
      // every epilogue thread takes the barrier of each chunk, also after a wait that gave up
      for (int c0 = kb0; c0 < kb1; c0 += CHUNK) {
        float* sc = scales + (((c0 - kb0) / CHUNK) & 1) * CHUNK * NT;
#pragma unroll
        for (int i = 0; i < PER; ++i) sc[tid + EPI_THREADS * i] = next[i];
        asm volatile("bar.sync 1, %0;" ::"n"(EPI_THREADS) : "memory");
        if (c0 + CHUNK < kb1) fetch(c0 + CHUNK);
        const int c1 = min(c0 + CHUNK, kb1);
        const float* s = sc + half * MINE;
#pragma unroll 1
        for (int kb = c0; kb < c1; ++kb, ++it, s += NT) {
          const int b = it % NBUF;
          ok = __all_sync(0xffffffffu, ok && mbar_wait_inline(used_bar(stage), phase, p.wc));
          if (!ok) break;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
          tc_fence_after();
          const uint32_t tcur = tmine + static_cast<uint32_t>(b * NT);
          constexpr int W = 16;
          static_assert(MINE % W == 0, "16 tokens at a time");
#pragma unroll
          for (int c = 0; c < MINE; c += W) {
            uint32_t r[W];
            tmem_ld16(tcur + c, r);
            tmem_ld_wait();
            reg_fence(r);
            if (c + W == MINE) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(tempty_bar(b));
            }
#pragma unroll
            for (int i = 0; i < W; i += 4) {
              const float4 f = *reinterpret_cast<const float4*>(s + c + i);
              acc[c + i] = fmaf(__uint_as_float(r[i]), f.x, acc[c + i]);
              acc[c + i + 1] = fmaf(__uint_as_float(r[i + 1]), f.y, acc[c + i + 1]);
              acc[c + i + 2] = fmaf(__uint_as_float(r[i + 2]), f.z, acc[c + i + 2]);
              acc[c + i + 3] = fmaf(__uint_as_float(r[i + 3]), f.w, acc[c + i + 3]);
            }
          }
        }
      }
      if (!ok && lane == 0) give_up(smem_u32(start_flag + 1), split);
    }
  }
  __syncwarp();
  __syncthreads();  // the ring is idle: every load has landed and every MMA has read it
  const int col = (warp & 3) * 32 + lane;
  const int64_t n = static_cast<int64_t>(nb) * BLK + col;
  const bool epi = warp >= 2;
  const int first = epi ? (warp - 2) / 4 * MINE : 0;  // the thread's first token
  const float bias = epi && p.bias != nullptr && n < p.N ? __bfloat162float(p.bias[n]) : 0.0f;
  const int tokens = static_cast<int>(walk.hi - t0 < NT ? walk.hi - t0 : NT);
  if (split == 1) {
    if (epi && start && *gave_up == 0u && n < p.N) {
#pragma unroll
      for (int i = 0; i < MINE; ++i)
        if (first + i < tokens) p.y[(t0 + first + i) * p.ldy + n] = to_out(acc[i] + bias, p.out_f16);
    }
  } else {
    if (epi) {
#pragma unroll
      for (int i = 0; i < MINE; ++i) sums[(first + i) * BLK + col] = acc[i];
    }
    __syncwarp();
    cluster_sync();
    // CTA r of the cluster adds and stores tokens r, r + split, ..., a warp each, four weight rows per thread.  All parts'
    // loads are on their way before the first is added (64 x 5,120 x 5,120: 11.4 us, one load at a time 12.8); added in the
    // order of K
    const int64_t n4 = static_cast<int64_t>(nb) * BLK + 4 * lane;
    if (epi && start && *gave_up == 0u && n4 < p.N) {
      for (int i = crank + split * (warp - 2); i < tokens; i += EPI_WARPS * split) {
        float part[MAX_SPLIT][4];
#pragma unroll
        for (int q = 0; q < MAX_SPLIT; ++q)
          if (q < split)
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(part[q][0]), "=f"(part[q][1]), "=f"(part[q][2]), "=f"(part[q][3])
                         : "r"(mapa_shared(smem0 + static_cast<uint32_t>((i * BLK + 4 * lane) * 4), static_cast<uint32_t>(q)))
                         : "memory");
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < MAX_SPLIT; ++q)
          if (q < split)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += part[q][j];
        store4(p, (t0 + i) * p.ldy + n4, n4, v);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();  // the other CTAs have read this CTA's sums (and its start flag)
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
  if (walk.bad && lane == 0) record_data_error(p.wc, H3B_EINVAL);
}

}  // namespace narrow

// ---------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------
bool al16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; }

int load_map(CUtensorMap* map, const void* base, int64_t K, int64_t rows, int64_t ld, uint32_t box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(K), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(ld)};
  const uint32_t box[2] = {BLK, box_rows};
  return encode_tmap(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int weight_map(CUtensorMap* map, const void* base, int64_t K, int64_t N, int64_t E, int64_t ldw, int64_t stride_e) {
  const uint64_t dims[3] = {static_cast<uint64_t>(K), static_cast<uint64_t>(N), static_cast<uint64_t>(E)};
  const uint64_t strides[2] = {static_cast<uint64_t>(ldw), static_cast<uint64_t>(stride_e)};
  const uint32_t box[3] = {BLK, BLK, 1};
  return encode_tmap(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int launch(const void* kernel, dim3 grid, int threads, int smem, int cluster, void** args, cudaStream_t st, int* fit) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = fit != nullptr ? 1 : 2;
  // with `fit`: no launch, but how many such clusters run at once
  const cudaError_t e =
      fit != nullptr ? cudaOccupancyMaxActiveClusters(fit, kernel, &cfg) : cudaLaunchKernelExC(&cfg, kernel, args);
  if (e != cudaSuccess) return cuda_fail(e, fit != nullptr ? "fp8_gemm_blocks: cluster occupancy" : "fp8_gemm_blocks launch");
  return H3B_OK;
}

// How many clusters of 1 .. MAX parts (of `unit` CTAs each) run at once on a device: looked up once, -1 for none.  The
// query counts one CTA per SM for a kernel that allocates TMEM; `per_sm` do run together (measured: CTAs of 64 columns).
template <int MAX>
struct Fit {
  std::atomic<int> of[MAX_DEVICES][MAX];
  int get(const void* kernel, int threads, int smem, int unit, int per_sm, int dev, int parts, int* fit) {
    *fit = of[dev][parts - 1].load(std::memory_order_acquire);
    if (*fit != 0) return H3B_OK;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    // without this the SM's shared memory is set up for a single CTA
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return cuda_fail(e, "fp8_gemm_blocks: shared memory");
    const int cluster = unit * parts;
    const int rc = launch(kernel, dim3(static_cast<unsigned>(cluster * num_sms()), 1, 1), threads, smem, cluster, nullptr,
                          nullptr, fit);
    if (rc) return rc;
    *fit *= per_sm;
    if (*fit < 1) *fit = -1;
    of[dev][parts - 1].store(*fit, std::memory_order_release);
    return H3B_OK;
  }
};

// The number of parts of K (clusters of parts * unit CTAs, a tile each) that ends first: rounds of tiles times the steps of
// a part and `round_cost`, what a round takes besides, in steps.  A persistent grid of single parts pays that once.
// `whole` / `parts`: the kernels for one part and for more.
template <int MAX>
int pick_split(Fit<MAX>& fits, const void* whole, const void* parts, int threads, int smem, int unit, int per_sm, int dev,
               int64_t tiles, int num_kb, int round_cost, bool persistent, int* split, int* fit1, double* best_cost) {
  double& best = *best_cost;
  for (int s = 1; s <= MAX; ++s) {
    if (s > 1 && num_kb < 4 * s) break;  // four steps each at least
    int fit = 0;
    const int rc = fits.get(s == 1 ? whole : parts, threads, smem, unit, per_sm, dev, s, &fit);
    if (rc) return rc;
    if (s == 1) {
      if (fit < 1) return fail(H3B_EUNSUPPORTED, "fp8_gemm_blocks: the kernel does not fit on this device");
      *fit1 = fit;
    }
    if (fit < 1) continue;
    const double rounds = static_cast<double>((tiles + fit - 1) / fit);
    const double steps = static_cast<double>((num_kb + s - 1) / s);
    const double cost = s == 1 && persistent ? rounds * steps + round_cost : rounds * (steps + round_cost);
    if (s == 1 || cost < best) {
      best = cost;
      *split = s;
    }
  }
  return H3B_OK;
}

// a step of single CTAs against one of pairs, whose tiles they choose between: both sides measured at the choice below
constexpr double SINGLE_STEP = 1.05;
// what a call of the wide form takes longer, in steps, than ROUND_COST says of both: it joins four times the sums.  100 x 1,024
// x 5,120: 8.9 us narrow, 13.6 wide (costs 25 and 19); 65 x 5,120 x 5,120: 14.7 and 14.0 (34 and 20)
constexpr double NARROW_LEAD = 12;

struct Operands {
  const void* a;
  int64_t lda;
  const void* w;
  int64_t ldw, w_exp;
  const float* sa;
  int64_t sa_row, sa_blk;
  const float* sb;
  int64_t sb_exp, sb_row, sb_blk;
  const void* bias;
  const void* offsets;
  int off64;
  void* y;
  int64_t ldy;
  int64_t T, N, K, E;
  int out_dtype;
};

// a launch as planned: which kernels, over how many tiles, in how many parts of K
struct Plan {
  int num_nb = 0;     // column tiles
  int64_t tiles = 0;  // that there can be
  int split = 1, fit = 0;
  double cost = 0;    // in steps
};

// tiles of `rows` rows to plan for.  Where there are several groups, each ends with part of a tile: half a tile more than the
// rows make on average, sqrt(1 / 12) of one by chance, and that much is planned for, since a tile too many takes a whole
// round: 500 rows in 4 groups of 1,024 x 8,192 21 us, without it 35 (where it is not needed K has fewer parts: 700 rows in 6
// groups of 2,048 x 4,096 27 us for 22).  At least one for each group: 800 rows in 8 groups of
// 5,120 x 5,120 58 us, without it 78
int64_t expected_tiles(const Params& p, int64_t active, int64_t rows, int num_nb) {
  const int64_t most = (p.T + active * (rows - 1)) / rows;  // exact for one group
  if (p.experts == 1) return most * num_nb;
  const double mean = static_cast<double>(p.T) / static_cast<double>(rows) + 0.5 * static_cast<double>(active);
  const int64_t blocks = static_cast<int64_t>(std::ceil(mean + std::sqrt(static_cast<double>(active) / 12.0)));
  return std::max(active, std::min(blocks, most)) * num_nb;
}

template <bool PAIR>
struct WidePlan : Plan {
  static const void* whole() { return reinterpret_cast<const void*>(wide::kernel<PAIR, false>); }
  static const void* parts() { return reinterpret_cast<const void*>(wide::kernel<PAIR, true>); }
  // T rows in at most `active` groups
  int make(const Params& p, int64_t active, int dev) {
    static Fit<PAIR ? wide::MAX_SPLIT / 2 : wide::MAX_SPLIT> fits;
    constexpr int64_t ROWS = PAIR ? 2 * wide::BM : wide::BM;
    num_nb = static_cast<int>((p.N + wide::BN - 1) / wide::BN);
    tiles = (p.T + active * (ROWS - 1)) / ROWS * num_nb;
    return pick_split(fits, whole(), parts(), wide::THREADS, wide::SMEM, PAIR ? 2 : 1, 1, dev,
                      expected_tiles(p, active, ROWS, num_nb), p.num_kb, wide::ROUND_COST, true, &split, &fit, &cost);
  }
  int go(Params& p, const Operands& o, const CUtensorMap& tmW, cudaStream_t st) {
    p.num_nb = num_nb;
    p.split = split;
    CUtensorMap tmA;
    int rc = load_map(&tmA, o.a, o.K, o.T, o.lda, wide::BM);
    if (rc) return rc;
    CUtensorMap tmY = tmA;  // a valid map where no TMA store is made
    if (p.y_align == 16) {
      const uint64_t dims[2] = {static_cast<uint64_t>(p.N), static_cast<uint64_t>(p.T)};
      const uint64_t strides[1] = {static_cast<uint64_t>(p.ldy) * 2};
      const uint32_t box[2] = {64, 32};
      rc = encode_tmap(&tmY, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, p.y, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
      if (rc) return rc;
      p.tma_out = 1;
    }
    // one part: as many CTAs (pairs) as run at once walk the tiles; more: a cluster for every tile that there can be
    const int64_t clusters = split == 1 && tiles > fit ? fit : tiles;
    const int cluster = (PAIR ? 2 : 1) * split;
    void* args[] = {&tmA, const_cast<CUtensorMap*>(&tmW), &tmY, &p};
    return launch(split == 1 ? whole() : parts(), dim3(static_cast<unsigned>(cluster * clusters), 1, 1), wide::THREADS,
                  wide::SMEM, cluster, args, st, nullptr);
  }
};

template <int NT>
struct NarrowPlan : Plan {
  int64_t token_tiles = 0;
  int make(const Params& p, int64_t active, int dev) {
    static Fit<narrow::MAX_SPLIT> fits;
    num_nb = static_cast<int>((p.N + BLK - 1) / BLK);
    token_tiles = (p.T + active * (NT - 1)) / NT;
    tiles = token_tiles * num_nb;
    const void* kernel = reinterpret_cast<const void*>(narrow::kernel<NT>);
    return pick_split(fits, kernel, kernel, narrow::threads(NT), narrow::smem(NT), 1, narrow::CTAS_PER_SM, dev,
                      expected_tiles(p, active, NT, num_nb), p.num_kb, narrow::ROUND_COST, false, &split, &fit, &cost);
  }
  int go(Params& p, const Operands& o, const CUtensorMap& tmW, cudaStream_t st) {
    p.num_nb = num_nb;
    p.split = split;
    CUtensorMap tmA;
    const int rc = load_map(&tmA, o.a, o.K, o.T, o.lda, NT);
    if (rc) return rc;
    void* args[] = {&tmA, const_cast<CUtensorMap*>(&tmW), &p};
    return launch(reinterpret_cast<const void*>(narrow::kernel<NT>),
                  dim3(static_cast<unsigned>(num_nb * split), static_cast<unsigned>(token_tiles), 1), narrow::threads(NT),
                  narrow::smem(NT), split, args, st, nullptr);
  }
};

// whether the narrow form's grid, whose second axis counts row tiles, has a place for all that there can be
bool narrow_serves(const Params& p, int64_t active, int rows) { return (p.T + active * (rows - 1)) / rows <= 65535; }

template <int NT>
int launch_narrow(Params& p, const Operands& o, const CUtensorMap& tmW, int64_t active, int dev, cudaStream_t st) {
  NarrowPlan<NT> plan;
  const int rc = plan.make(p, active, dev);
  return rc ? rc : plan.go(p, o, tmW, st);
}

int gemm_blocks(const char* what, const Operands& o, cudaStream_t st) {
  const int64_t most = (1ll << 31) - 1;
  if (o.T < 0 || o.N <= 0 || o.K <= 0 || o.E <= 0)
    return fail(H3B_EINVAL, "%s: rows %lld N %lld K %lld experts %lld", what, (long long)o.T, (long long)o.N,
                (long long)o.K, (long long)o.E);
  if (o.out_dtype != H3B_OUT_BF16 && o.out_dtype != H3B_OUT_F16) return fail(H3B_EINVAL, "%s: out dtype %d", what, o.out_dtype);
  if (o.T == 0) return H3B_OK;
  if (o.a == nullptr || o.w == nullptr || o.sa == nullptr || o.sb == nullptr || o.y == nullptr)
    return fail(H3B_EINVAL, "%s: null operand", what);
  if (o.K % 16) return fail(H3B_EUNSUPPORTED, "%s: K %lld must be a multiple of 16", what, (long long)o.K);
  if (o.lda < o.K || o.ldw < o.K || o.lda % 16 || o.ldw % 16 || o.w_exp % 16 || !al16(o.a) || !al16(o.w))
    return fail(H3B_EALIGN, "%s: a and w must be 16-byte aligned with strides that are multiples of 16 and at least K", what);
  if (o.w_exp < 0 || (o.E > 1 && o.w_exp == 0) || o.sa_row < 0 || o.sa_blk < 0 || o.sb_exp < 0 || o.sb_row < 0 || o.sb_blk < 0)
    return fail(H3B_EINVAL, "%s: negative stride, or a zero one between experts", what);
  if (o.ldy < o.N) return fail(H3B_EINVAL, "%s: ldy %lld below N", what, (long long)o.ldy);
  if (o.T > most - 256 || o.N > most - 256 || o.K > most - 256 || o.E > most - 32)
    return fail(H3B_EUNSUPPORTED, "%s: sizes at or above 2^31", what);

  Params p{};
  p.T = o.T;
  p.N = o.N;
  p.num_kb = static_cast<int>((o.K + BLK - 1) / BLK);
  p.experts = static_cast<int>(o.E);
  p.offsets = o.offsets;
  p.off64 = o.off64;
  p.sa = o.sa;
  p.sa_row = o.sa_row;
  p.sa_blk = o.sa_blk;
  p.sb = o.sb;
  p.sb_exp = o.sb_exp;
  p.sb_row = o.sb_row;
  p.sb_blk = o.sb_blk;
  p.bias = static_cast<const __nv_bfloat16*>(o.bias);
  p.y = static_cast<uint16_t*>(o.y);
  p.ldy = o.ldy;
  p.out_f16 = o.out_dtype == H3B_OUT_F16;
  const uintptr_t rows_at = reinterpret_cast<uintptr_t>(o.y) | static_cast<uintptr_t>(o.ldy) * 2;
  p.y_align = rows_at % 16 == 0 ? 16 : (rows_at % 8 == 0 ? 8 : (rows_at % 4 == 0 ? 4 : 2));
  p.wc.status = device_status_word();
  p.wc.timeout = wait_timeout_ns();
  if (p.wc.status == nullptr) return fail(H3B_ECUDA, "%s: device status word", what);
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES)
    return fail(H3B_EUNSUPPORTED, "%s: device ordinal %d", what, dev);

  CUtensorMap tmW;
  int rc = weight_map(&tmW, o.w, o.K, o.N, o.E, o.ldw, o.E > 1 ? o.w_exp : o.ldw * ((o.N + 15) / 16 * 16));
  if (rc) return rc;
  const int64_t active = o.T < o.E ? o.T : o.E;  // groups that can hold a row
  const int64_t mean = (o.T + o.E - 1) / o.E;
  const int64_t narrow_nb = (o.N + BLK - 1) / BLK, wide_nb = (o.N + wide::BN - 1) / wide::BN;
  if (o.T / 16 + active > most / narrow_nb || o.T / wide::BM + active > most / (2 * wide::MAX_SPLIT) / wide_nb ||
      narrow_nb > most / narrow::MAX_SPLIT)
    return fail(H3B_EUNSUPPORTED, "%s: 2^31 tiles or more", what);
  // Few rows a group: narrow.  Dense, 64 x 15,360 x 5,120: 20.7 us narrow, 24.4 wide; grouped, uneven groups of 20 rows
  // in the mean (32 experts of 2,048 x 5,120): 75 and 102; of 38: 88 and 69, of 60: 101 and 69.  More rows: by cost, 300 rows
  // in 4 groups of 1,024 x 4,096 12 and 15.
  if (mean > (o.E > 1 ? 32 : 64) || !narrow_serves(p, active, mean <= 16 ? 16 : 32)) {
    WidePlan<true> pairs;
    WidePlan<false> singles;
    rc = pairs.make(p, active, dev);
    if (!rc) rc = singles.make(p, active, dev);
    if (rc) return rc;
    // CTA pairs read less (32 KB a step and SM instead of 48), which counts at the power cap: 8,192 x 15,360 x 5,120 713 us in
    // long runs, singles 746 (below the cap both 610); single CTAs, with tiles of half the rows, fit small and ragged work
    // better: 777 x 5,120 x 13,824 65 us against 115, 1,500 rows in 8 groups of 2,048 x 5,120 31 against 52
    const bool paired = pairs.cost <= SINGLE_STEP * singles.cost;
    if (narrow_serves(p, active, 64)) {
      NarrowPlan<64> few;
      rc = few.make(p, active, dev);
      if (rc) return rc;
      if (few.cost <= (paired ? pairs.cost : singles.cost) + NARROW_LEAD) return few.go(p, o, tmW, st);
    }
    return paired ? pairs.go(p, o, tmW, st) : singles.go(p, o, tmW, st);
  }
  // the rows of a tile that is mostly absent cost little but not nothing: 1 x 5,120 x 5,120 takes 8.1 us with tiles of 16
  // rows, 11.1 with 64; 32 x 5,120 x 13,824 18.5 us with 32 and 19.8 with 64
  if (mean <= 16) return launch_narrow<16>(p, o, tmW, active, dev, st);
  if (mean <= 32) return launch_narrow<32>(p, o, tmW, active, dev, st);
  return launch_narrow<64>(p, o, tmW, active, dev, st);
}

}  // namespace
}  // namespace h3b

using namespace h3b;

extern "C" int h3b_fp8_gemm_blocks(const void* a, int64_t lda, const void* w, int64_t ldw, const float* sa, int64_t sa_row,
                                   int64_t sa_block, const float* sb, int64_t sb_row, int64_t sb_block, const void* bias,
                                   void* y, int64_t ldy, int64_t M, int64_t N, int64_t K, int32_t out_dtype,
                                   h3b_stream_t stream) {
  const Operands o{a, lda, w, ldw, 0, sa, sa_row, sa_block, sb, 0, sb_row, sb_block, bias, nullptr, 0, y, ldy, M, N, K, 1,
                   out_dtype};
  return gemm_blocks("fp8_gemm_blocks", o, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int h3b_fp8_gemm_grouped(const void* a, int64_t lda, const void* w, int64_t w_expert, int64_t ldw,
                                    const float* sa, int64_t sa_row, int64_t sa_block, const float* sb, int64_t sb_expert,
                                    int64_t sb_row, int64_t sb_block, const void* offsets, int32_t offsets_i64, void* y,
                                    int64_t ldy, int64_t rows, int64_t experts, int64_t N, int64_t K, int32_t out_dtype,
                                    h3b_stream_t stream) {
  if (rows > 0 && offsets == nullptr) return fail(H3B_EINVAL, "fp8_gemm_grouped: offsets are required");
  const Operands o{a,  lda, w, ldw, w_expert, sa,   sa_row, sa_block, sb,        sb_expert, sb_row, sb_block, nullptr, offsets,
                   offsets_i64 != 0, y, ldy, rows, N, K, experts, out_dtype};
  return gemm_blocks("fp8_gemm_grouped", o, reinterpret_cast<cudaStream_t>(stream));
}
