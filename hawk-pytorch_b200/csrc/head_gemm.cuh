// The tcgen05 GEMM under the operators that multiply activations with the head's weight (linear_ce.cu, linear_logprobs.cu).
//
// The GEMM is one kernel: C[M,Nc] = A[M,K] . B[Nc,K]^T, bf16 operands, fp32 accumulation.
// A pair of CTAs (cta_group::2) computes a 256*MH x 256 output tile, K in blocks of 64 (128-byte swizzled rows).  What
// bounds a CTA working alone on 128x256 is operand delivery from L2: 48 KB per 512 clocks of MMA, 96 B/clk/SM; a
// pair shares B: 32 KB per CTA in the same time with MH = 1, 24 KB with MH = 2.
//   MH = 1: two TMEM accumulators, the epilogue overlaps the next tile's MMA: the logits, whose epilogue is long.
//   MH = 2: the two 256-row halves fill TMEM and share each B tile: the gradient GEMMs when K is long enough for the
//           epilogue that nothing overlaps (tensor pipe active at N8192 H2048 V8192: 79 % with MH = 1).
// Warp-specialised:
//   warp 0   : TMA producer of its CTA's halves of A and B (cp.async.bulk.tensor, ring of 5 or 4 stages);
//   warp 1   : owns TMEM (512 columns); in the leader CTA it issues tcgen05.mma for the pair;
//   warps 2-9: epilogue, two warps per TMEM lane quarter (128 columns each), overlapping the next tile's MMA.  The
//      softmax epilogue is ~10 issue slots and one MUFU operation per logit; with four warps it, not the MMA, set the
//      pace at H = 512 (N32752 V32000: 1.73 ms for 1.07e12 flop).  Tiles leave through shared memory as TMA box
//      stores: full 128-byte lines.  (fp32 rows stored 16 bytes per lane ran at 1.5 TB/s: d weight of 777 rows,
//      V31999 H1024, 92 us.)
// Persistent over tiles (grid = 2 * min(tiles, SM count / 2)).  Every mbarrier wait is bounded by a clock
// budget; on expiry the kernel records a status word, drains, frees TMEM and returns.
#pragma once

#include <algorithm>
#include <type_traits>

#include "tc05.cuh"

namespace hawk {
using namespace tc;

constexpr int BM = 256, BN = 256, BK = 64, UMMA_K = 16;  // one tcgen05.mma of the pair covers 256 x 256 x 16
constexpr int HALF_BYTES = 128 * BK * 2;                 // one CTA's half of an operand tile: 128 M or N indices x 64 K
constexpr int EPI_WARPS = 8, EPI_COLS = 128;             // columns of a tile per epilogue warp
constexpr int BOX_BYTES = 32 * 128;                      // store box: 32 rows x 64 bf16 or 32 fp32 columns
template <int MH>
struct GemmCfg {
  static constexpr int STAGES = MH == 1 ? 5 : 4;
  static constexpr int A_BYTES = MH * HALF_BYTES;               // A halves first, then the B half
  static constexpr int STAGE_BYTES = A_BYTES + HALF_BYTES;
  static constexpr int NBOX = MH == 1 ? 2 : 1;                  // store boxes per epilogue warp
  static constexpr int SMEM = STAGES * STAGE_BYTES + EPI_WARPS * NBOX * BOX_BYTES + 1024;  // + slack for 1024-byte alignment
  static constexpr int NACC = MH == 1 ? 2 : 1;
};
constexpr int GEMM_THREADS = 64 + 32 * EPI_WARPS;

enum { EPI_LOGITS = 0, EPI_OUT = 1, EPI_SCORE = 2, EPI_SCORE_KEEP = 3 };

struct EpiParams {
  int M, Nc;                 // valid rows / columns of C
  int k_per_split;           // K blocks per split (EPI_OUT); a tile index runs over tiles x splits
  // Where the rows that count are known on the device only: their number, of M or (count_is_k) of K, from which the kernel
  // plans its tiles anew.  Null = all.  Rows of A behind it may hold anything; rows of K up to the next block's end hold zeros.
  const int* count;
  int count_is_k;
  int part_rows;             // not 0, for a count of M: splits of K planned anew, too (CountedRows), in this many rows of partial sums
  // EPI_LOGITS
  float2* stats;             // [column groups of 128, M] (max, sum exp)
  float* correct;            // [M] logit at the label
  const long long* labels;   // [M]
  // EPI_SCORE, EPI_SCORE_KEEP (which also stores e^(x - max) in fp16): `correct` and `labels` as above, and
  float4* score;             // [M, column groups of 128] (max, sum exp without `ties`, sum exp (x - max) log2 e, ties)
  int groups;                // column groups
  // EPI_OUT
  int out_bf16;              // the store map's type
  const float* scale;        // device scalar multiplied in; null = 1
  const float* row_scale;    // [M] factors of the rows; null = 1
};

constexpr int MN_BOX = 64 * 128;  // bytes of one [64 columns x 64 rows] box of an MN-major operand

// tile index -> (m_tile, n_tile): groups of GROUP_M row tiles sweep all column tiles, so the tiles
// in flight share a small set of A and B tiles in L2
constexpr int GROUP_M = 8;
__device__ __forceinline__ void tile_coords(int tile, int m_tiles, int n_tiles, int& mt, int& nt) {
  const int per_group = GROUP_M * n_tiles;
  const int g = tile / per_group;
  const int first = g * GROUP_M;
  const int gm = min(GROUP_M, m_tiles - first);
  const int in = tile - g * per_group;
  mt = first + in % gm;
  nt = in / gm;
}

// one 32-column chunk of logits of one row: round to bf16, fold into the running (max, sum exp), pick the label
template <bool FULL>
__device__ __forceinline__ void softmax_chunk(const uint32_t (&v)[32], int cbase, int Nc, long long label, bool row_ok,
                                              float* correct, uint32_t (&packed)[16], float& run_m, float& run_s) {
  float2 vals[16];
  float cmax = -INFINITY;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    packed[j] = pack_bf16x2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
    vals[j] = unpack_bf16x2(packed[j]);  // the bf16-rounded logits are THE logits
    if (!FULL) {
      if (cbase + 2 * j >= Nc) vals[j].x = -INFINITY;
      if (cbase + 2 * j + 1 >= Nc) vals[j].y = -INFINITY;
    }
    cmax = fmaxf(cmax, fmaxf(vals[j].x, vals[j].y));
  }
  const float new_m = fmaxf(run_m, cmax);
  const float2 off = f2(-new_m * kLog2e);
  const float err = fmaf(new_m, kLog2e, off.x);  // off's rounding, exactly: every term below carries the factor 2^err
  float2 add = f2(0.f);
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    float2 t = fma2(vals[j], f2(kLog2e), off);
    t.x = ex2_approx(t.x);
    t.y = ex2_approx(t.y);
    add = add2(add, t);
  }
  run_s = fmaf(run_s, ex2_approx((run_m - new_m) * kLog2e), (add.x + add.y) * fmaf(err, -0.69314718f, 1.f));  // 2^-err
  run_m = new_m;
  if (row_ok && label >= cbase && label < cbase + 32) {
    const int at = (int)(label - cbase);
    float pick = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (at == 2 * j) pick = vals[j].x;
      if (at == 2 * j + 1) pick = vals[j].y;
    }
    *correct = pick;
  }
}

// One 32-column chunk of unrounded logits of one row, whose group's maximum m is known: the sums of e = e^(x - m) and of
// e (x - m) log2 e (for the entropy), the label's logit, and with KEEP e itself in fp16 (at most 1, so nothing overflows).  With APART
// `rest` is the sum of e without the elements at `apart` (m, or NaN: all of them).
template <bool FULL, bool KEEP, bool APART>
__device__ __forceinline__ void score_chunk(const uint32_t (&v)[32], float m, float apart, int cbase, int Nc, long long label, float* correct,
                                            uint32_t (&packed)[16], float2& s, float2& sx, float2& rest) {
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    float2 x = make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
    if (!FULL) {  // past the vocabulary: e = 0, and a finite factor
      if (cbase + 2 * j >= Nc) x.x = m - 256.f;
      if (cbase + 2 * j + 1 >= Nc) x.y = m - 256.f;
    }
    const float2 t = mul2(add2(x, f2(-m)), f2(kLog2e));
    const float2 e = make_float2(ex2_approx(t.x), ex2_approx(t.y));
    s = add2(s, e);
    if (APART) rest = add2(rest, make_float2(x.x == apart ? 0.f : e.x, x.y == apart ? 0.f : e.y));
    sx = fma2(e, t, sx);
    if (KEEP) packed[j] = pack_f16x2(e.x, e.y);
  }
  if (label >= cbase && label < cbase + 32 && label < Nc) {
    const int at = (int)(label - cbase);
    float pick = 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (at == j) pick = __uint_as_float(v[j]);
    *correct = pick;
  }
}

// An epilogue warp's store boxes of 32 rows x 128 bytes (lane = row; 16-byte piece index XOR row mod 8, the store's
// swizzle), NBOX of them used in turn; every store is one bulk group of lane 0, so that counting groups tells when a box
// has been read out and may be refilled.
template <int NBOX>
__device__ __forceinline__ void box_reuse(int lane) {
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(NBOX - 1) : "memory");
  __syncwarp();
}
__device__ __forceinline__ void box_put(unsigned char* box, int lane, int piece0, const uint32_t (&p)[16]) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *reinterpret_cast<uint4*>(box + lane * 128 + (((piece0 + q) ^ (lane & 7)) * 16)) =
        make_uint4(p[4 * q], p[4 * q + 1], p[4 * q + 2], p[4 * q + 3]);
}
__device__ __forceinline__ void box_store(const CUtensorMap* map, const unsigned char* box, int lane, int col, int row,
                                          int depth, const EpiParams& ep, int shift = 0) {
  fence_smem_to_tma();
  __syncwarp();
  if (lane == 0) {
    if (col < ep.Nc && row < ep.M) tma_store_3d(map, box, col, row + shift, depth);
    bulk_commit();  // an empty group where nothing is stored: the group count stays in step
  }
}

// The K blocks of a count of rows known on the device only, over at most `most` splits: at least one block (of zeros), none without
struct CountedSplits {
  int blocks, per, splits;
  __device__ __forceinline__ CountedSplits(int n, int most)
      : blocks(max(1, (n + BK - 1) / BK)), per((blocks + most - 1) / most), splits((blocks + per - 1) / per) {}
};

// The tiles of a count of M rows known on the device only: K in more splits than were planned for all rows where `pairs` of CTAs would be
// left without a tile, in whole boxes of 32 rows of partial sums to a split
struct CountedRows {
  int m_tiles, per, splits, stride;
  __device__ __forceinline__ CountedRows(int n, int tile_rows, int n_tiles, int kblocks, int planned, int part_rows, int pairs) {
    m_tiles = (n + tile_rows - 1) / tile_rows;
    stride = max(32, (n + 31) / 32 * 32);
    const int most = min(min(kblocks, 32), max(1, part_rows / stride));
    splits = min(max(planned, pairs / max(1, m_tiles * n_tiles)), most);
    per = (kblocks + splits - 1) / splits;
    splits = (kblocks + per - 1) / per;
  }
};

// ---------------------------------------------------------------------------------------------
// the GEMM
// ---------------------------------------------------------------------------------------------
// A_MN / B_MN: the operand is read as an MN-major tile, i.e. straight from a row-major [K, M] (or [K, Nc])
// tensor whose rows are the contraction index; its tensor map then has boxes of [64 columns x 64 rows],
// one box per 64 M/N indices, 8192 bytes apart in the stage.
template <int MODE, int MH, bool A_MN, bool B_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GEMM_THREADS, 1)
gemm_bf16_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const __grid_constant__ CUtensorMap map_c, int K, int m_tiles, int n_tiles, int splits, EpiParams ep,
                 int* status) {
  int split_rows = 0;  // rows of partial sums to a split where the splits were planned here
  if (ep.count) {
    const int n = *ep.count;
    if (ep.count_is_k) {
      const CountedSplits c(n, splits);
      K = c.blocks * BK;
      ep.k_per_split = c.per;
      splits = c.splits;
    } else if (MODE == EPI_OUT && ep.part_rows) {
      const CountedRows c(n, BM * MH, n_tiles, (K + BK - 1) / BK, splits, ep.part_rows, gridDim.x >> 1);
      ep.M = n;
      m_tiles = c.m_tiles;
      ep.k_per_split = c.per;
      splits = c.splits;
      split_rows = c.stride;
    } else {
      ep.M = n;
      m_tiles = (n + BM * MH - 1) / (BM * MH);
    }
  }
  using Cfg = GemmCfg<MH>;
  constexpr int KSTAGES = Cfg::STAGES, STAGE_BYTES = Cfg::STAGE_BYTES, A_BYTES = Cfg::A_BYTES, NACC = Cfg::NACC;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full_bar[KSTAGES], empty_bar[KSTAGES], tfull_bar[2], tempty_bar[2];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  constexpr uint32_t kIdescMaj = umma_idesc(BM, BN, A_MN ? 1 : 0, B_MN ? 1 : 0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int first_tile = blockIdx.x >> 1, tile_stride = gridDim.x >> 1;
  const int tiles = m_tiles * n_tiles, num_tiles = tiles * splits;
  const int kblocks = (K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < KSTAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 2 * EPI_WARPS);
    }
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc_pair(&tmem_base_slot, 512);
  fence_before();
  __syncthreads();
  cluster_sync();  // the peer's barriers are initialised before anything is signalled across
  fence_after();
  const uint32_t tmem_base = tmem_base_slot;
  volatile int* abortp = &abort_flag;

  if (warp == 0) {
    // ---------------- TMA producer (each CTA: its own halves; bytes counted on the leader's barrier) ----------------
    if (lane == 0) {
      uint32_t it = 0;
      for (int tile = first_tile; tile < num_tiles && !*abortp; tile += tile_stride) {
        int mt, nt;
        tile_coords(tile % tiles, m_tiles, n_tiles, mt, nt);
        const int kb0 = (tile / tiles) * ep.k_per_split, kb1 = min(kblocks, kb0 + ep.k_per_split);
        const int m0 = mt * BM * MH + (int)rank * 128, n0 = nt * BN + (int)rank * 128;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % KSTAGES;
          const uint32_t ph = (it / KSTAGES) & 1;
          if (!mbar_wait(&empty_bar[s], ph ^ 1, abortp)) break;
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], 2 * STAGE_BYTES);
          const uint32_t bar = map_to_rank(&full_bar[s], 0);
          unsigned char* st = smem + s * STAGE_BYTES;
#pragma unroll
          for (int hh = 0; hh < MH; ++hh) {
            if (A_MN) {
#pragma unroll
              for (int q = 0; q < 2; ++q)
                tma_load_2d_pair(st + hh * HALF_BYTES + q * MN_BOX, &map_a, bar, m0 + hh * BM + q * 64, kb * BK);
            } else {
              tma_load_2d_pair(st + hh * HALF_BYTES, &map_a, bar, kb * BK, m0 + hh * BM);
            }
          }
          if (B_MN) {
#pragma unroll
            for (int q = 0; q < 2; ++q) tma_load_2d_pair(st + A_BYTES + q * MN_BOX, &map_b, bar, n0 + q * 64, kb * BK);
          } else {
            tma_load_2d_pair(st + A_BYTES, &map_b, bar, kb * BK, n0);
          }
        }
      }
      // A wait gave up somewhere: let the copies issued last land before the pair's shared memory goes.  The leader
      // holds the barriers that count them (for both CTAs); the peer waits at the cluster barrier below.
      if (*abortp && rank == 0) drain_stages(full_bar, KSTAGES, it);
      // otherwise see every stage freed: the commits that free them are signals from the leader to this CTA
      for (uint32_t j = it > KSTAGES ? it - KSTAGES : 0; j < it && !*abortp; ++j)
        (void)mbar_wait(&empty_bar[j % KSTAGES], (j / KSTAGES) & 1, abortp);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (leader only) ----------------
    if (lane == 0 && rank == 0) {
      uint32_t it = 0, tcount = 0;
      for (int tile = first_tile; tile < num_tiles && !*abortp; tile += tile_stride, ++tcount) {
        const int acc = NACC == 2 ? (tcount & 1) : 0;
        const uint32_t aph = NACC == 2 ? ((tcount >> 1) & 1) : (tcount & 1);
        if (!mbar_wait(&tempty_bar[acc], aph ^ 1, abortp)) break;
        fence_after();
        const int kb0 = (tile / tiles) * ep.k_per_split, kb1 = min(kblocks, kb0 + ep.k_per_split);
        const uint32_t d_tmem = tmem_base + acc * BN;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % KSTAGES;
          const uint32_t ph = (it / KSTAGES) & 1;
          if (!mbar_wait(&full_bar[s], ph, abortp)) { ok = false; break; }
          fence_after();
          const uint32_t a_addr = smem_u32(smem + s * STAGE_BYTES);
          const uint32_t b_addr = a_addr + A_BYTES;
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k) {
            // K-major: 16 K-elements further along the 128-byte rows; MN-major: 16 K-rows (2048 bytes) further down
            const uint64_t bd = B_MN ? umma_desc_sw128(b_addr + k * UMMA_K * 128, MN_BOX) : umma_desc_sw128(b_addr + k * UMMA_K * 2);
#pragma unroll
            for (int hh = 0; hh < MH; ++hh) {
              const uint32_t ah = a_addr + hh * HALF_BYTES;
              const uint64_t ad = A_MN ? umma_desc_sw128(ah + k * UMMA_K * 128, MN_BOX) : umma_desc_sw128(ah + k * UMMA_K * 2);
              umma_bf16_pair(d_tmem + hh * BN, ad, bd, kIdescMaj, (kb > kb0 || k > 0) ? 1u : 0u);
            }
          }
          umma_commit_pair(&empty_bar[s]);  // frees the stage in both CTAs once these MMAs have read it
        }
        if (!ok) break;
        umma_commit_pair(&tfull_bar[acc]);  // accumulator complete (each CTA's epilogue waits on its own barrier)
      }
    }
  } else {
    // ---------------- epilogue (warps 2..9) ----------------
    const int quarter = warp & 3;  // TMEM lanes 32*quarter .. +31 are the ones this warp may read
    const int half = (warp - 2) >> 2;
    unsigned char* boxes = smem + KSTAGES * STAGE_BYTES + (warp - 2) * Cfg::NBOX * BOX_BYTES;
    const float scale = (MODE == EPI_OUT && ep.scale) ? *ep.scale : 1.f;
    uint32_t tcount = 0;
    for (int tile = first_tile; tile < num_tiles; tile += tile_stride, ++tcount) {
      if (*abortp) break;
      int mt, nt;
      tile_coords(tile % tiles, m_tiles, n_tiles, mt, nt);
      const int acc = NACC == 2 ? (tcount & 1) : 0;
      long long score_label = -1;  // requested before the wait: it is an L2 access away
      if (MODE == EPI_SCORE || MODE == EPI_SCORE_KEEP) {
        const int r = mt * BM + (int)rank * 128 + quarter * 32 + lane;
        if (r < ep.M) score_label = __ldg(ep.labels + r);
      }
      if (!mbar_wait_warp(&tfull_bar[acc], NACC == 2 ? ((tcount >> 1) & 1) : (tcount & 1), abortp)) break;  // lane 0 waits: the warp cannot diverge
      fence_after();
      const int col0 = nt * BN + half * EPI_COLS;
#pragma unroll 1
      for (int hh = 0; hh < MH; ++hh) {
      const int row0 = (mt * MH + hh) * BM + (int)rank * 128 + quarter * 32, row = row0 + lane;
      const bool row_ok = row < ep.M;
      const uint32_t taddr0 = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)((acc + hh) * BN + half * EPI_COLS);
      uint32_t v[2][32];
      tmem_ld32_async(taddr0, v[0]);

      if (MODE == EPI_SCORE || MODE == EPI_SCORE_KEEP) {
        // TMEM is read twice, for the maximum and for the sums: one maximum per row and 128 columns, against which what is
        // kept is relative, and no rescaling of running sums (which would be three more MUFU operations per row)
        constexpr bool KEEP = MODE == EPI_SCORE_KEEP;
        const int cols = ep.Nc - col0;  // valid columns from here on
        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
        for (int c = 0; c < EPI_COLS / 32; ++c) {
          tmem_ld_wait();
          tmem_ld32_async(taddr0 + ((c + 1) % (EPI_COLS / 32)) * 32, v[(c + 1) & 1]);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float a = __uint_as_float(v[c & 1][j]), b = __uint_as_float(v[c & 1][j + 1]);
            if (cols >= EPI_COLS || c * 32 + j < cols) m0 = fmaxf(m0, a);
            if (cols >= EPI_COLS || c * 32 + j + 1 < cols) m1 = fmaxf(m1, b);
          }
        }
        const float m = fmaxf(m0, m1);
        const long long label = score_label;
        // In a row whose token is all but certain the other elements are what 1 - p is made of, and lost beside its 1.  Where the
        // odd and the even columns' maxima lie so far apart that the others may be little, the elements at the maximum are kept apart
        // from the sum, and counted; where they do not, the others are 2^-9 at least, and right to 2^-13 within the sum.  Scores of 1238 rows of
        // H512 V32000 with e kept, most of their tokens likely: 50.2 us without this, 53.6 with, 54.7 with four chunks unrolled here too;
        // a check of every chunk, or of the chunk at the maximum only, 59.5; of unlikely tokens, and at H2048, 0.1 to 0.7 % more.
        const bool lone = fabsf(m0 - m1) > 6.2f;  // e^-6.2 is a little more than 2^-9
        float2 s = f2(0.f), sx = f2(0.f), rest = f2(0.f);
        const auto sums = [&](auto with) {
        constexpr bool APART = decltype(with)::value;
        const float apart = lone ? m : __int_as_float(0x7fc00000);
#pragma unroll(APART ? 2 : 4)
        for (int c = 0; c < EPI_COLS / 32; ++c) {
          tmem_ld_wait();
          if (c + 1 < EPI_COLS / 32) {
            tmem_ld32_async(taddr0 + (c + 1) * 32, v[(c + 1) & 1]);
          } else {
            // The accumulator is read: hand it back now.  The arrival is a release, which behind this tile's stores would wait for
            // their way to L2 and back.
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(map_to_rank(&tempty_bar[acc], 0));
          }
          const int cbase = col0 + c * 32;
          uint32_t packed[16];
          float* correct = ep.correct + (row_ok ? row : 0);
          if (cbase + 32 <= ep.Nc) {
            score_chunk<true, KEEP, APART>(v[c & 1], m, apart, cbase, ep.Nc, label, correct, packed, s, sx, rest);
          } else if (cbase < ep.Nc) {
            score_chunk<false, KEEP, APART>(v[c & 1], m, apart, cbase, ep.Nc, label, correct, packed, s, sx, rest);
          } else if (KEEP) {  // whole chunk past the vocabulary (same for every lane); the store clips it
#pragma unroll
            for (int j = 0; j < 16; ++j) packed[j] = 0u;
          }
          if (KEEP) {
            unsigned char* box = boxes + (c >> 1) * BOX_BYTES;
            if ((c & 1) == 0) box_reuse<2>(lane);
            box_put(box, lane, (c & 1) * 4, packed);
            if (c & 1) box_store(&map_c, box, lane, col0 + (c >> 1) * 64, row0, 0, ep);
          }
        }
        };
        const bool any = __any_sync(0xffffffffu, lone);
        if (any) sums(std::true_type{}); else sums(std::false_type{});
        const float all = s.x + s.y, others = any && lone ? rest.x + rest.y : all;
        if (row_ok && cols > 0)  // what is apart is a number of ones: the sums' difference but for their rounding
          ep.score[(long long)row * ep.groups + col0 / EPI_COLS] = make_float4(m, others, sx.x + sx.y, rintf(all - others));
      } else if (MODE == EPI_LOGITS) {
        float run_m = -INFINITY, run_s = 0.f;
        const long long label = row_ok ? ep.labels[row] : -1;
#pragma unroll
        for (int c = 0; c < EPI_COLS / 32; ++c) {
          tmem_ld_wait();
          if (c + 1 < EPI_COLS / 32) tmem_ld32_async(taddr0 + (c + 1) * 32, v[(c + 1) & 1]);
          const int cbase = col0 + c * 32;
          uint32_t packed[16];
          if (cbase + 32 <= ep.Nc) {
            softmax_chunk<true>(v[c & 1], cbase, ep.Nc, label, row_ok, ep.correct + (row_ok ? row : 0), packed, run_m, run_s);
          } else if (cbase < ep.Nc) {
            softmax_chunk<false>(v[c & 1], cbase, ep.Nc, label, row_ok, ep.correct + (row_ok ? row : 0), packed, run_m, run_s);
          } else {  // whole chunk past the vocabulary (same for every lane); the store clips it
#pragma unroll
            for (int j = 0; j < 16; ++j) packed[j] = 0u;
          }
          // box c/2 of the warp: 32 rows x 64 columns, 16-byte piece index XOR row mod 8 (the store's swizzle)
          unsigned char* box = boxes + (c >> 1) * BOX_BYTES;
          if ((c & 1) == 0) box_reuse<2>(lane);
          box_put(box, lane, (c & 1) * 4, packed);
          if (c & 1) box_store(&map_c, box, lane, col0 + (c >> 1) * 64, row0, 0, ep);
        }
        if (row_ok && col0 < ep.Nc) ep.stats[(long long)(col0 / EPI_COLS) * ep.M + row] = make_float2(run_m, run_s);
      } else {
        const int in_split = tile / tiles, split = split_rows ? 0 : in_split, shift = in_split * split_rows;
        const float f = ep.row_scale && row_ok ? scale * __ldg(ep.row_scale + row) : scale;
        auto chunk = [&](int c) -> const uint32_t(&)[32] {  // waits for chunk c, requests the next one
          tmem_ld_wait();
          if (c + 1 < EPI_COLS / 32) tmem_ld32_async(taddr0 + (c + 1) * 32, v[(c + 1) & 1]);
          return v[c & 1];
        };
        if (ep.out_bf16) {
#pragma unroll
          for (int c = 0; c < EPI_COLS / 32; ++c) {
            const uint32_t(&w)[32] = chunk(c);
            uint32_t packed[16];
#pragma unroll
            for (int j = 0; j < 16; ++j)
              packed[j] = pack_bf16x2(__uint_as_float(w[2 * j]) * f, __uint_as_float(w[2 * j + 1]) * f);
            unsigned char* box = boxes + ((c >> 1) % Cfg::NBOX) * BOX_BYTES;
            if ((c & 1) == 0) box_reuse<Cfg::NBOX>(lane);
            box_put(box, lane, (c & 1) * 4, packed);
            if (c & 1) box_store(&map_c, box, lane, col0 + (c >> 1) * 64, row0, split, ep, shift);
          }
        } else {
#pragma unroll
          for (int c = 0; c < EPI_COLS / 32; ++c) {
            const uint32_t(&w)[32] = chunk(c);
            unsigned char* box = boxes + (c % Cfg::NBOX) * BOX_BYTES;
            box_reuse<Cfg::NBOX>(lane);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint32_t scaled[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) scaled[j] = __float_as_uint(__uint_as_float(w[16 * q + j]) * f);
              box_put(box, lane, q * 4, scaled);
            }
            box_store(&map_c, box, lane, col0 + c * 32, row0, split, ep, shift);
          }
        }
      }
      }  // halves
      if (MODE != EPI_SCORE && MODE != EPI_SCORE_KEEP) {
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(map_to_rank(&tempty_bar[acc], 0));
      }
    }
    if (lane == 0) bulk_wait_all();
  }

  // ---------------- teardown ----------------
  __syncwarp();
  fence_before();
  __syncthreads();
  if (abort_flag && threadIdx.x == 0) atomicExch(status, 1);
  cluster_sync();  // neither CTA's barriers or TMEM go while the other may still signal or accumulate into them
  if (warp == 1) {
    fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ---------------------------------------------------------------------------------------------
// small kernels behind the GEMMs
// ---------------------------------------------------------------------------------------------
// A GEMM of this call abandoned a wait: make that visible in the result itself (the loss, or the first element of
// each gradient, becomes NaN), since a training loop may not read the status word for many steps.
static __global__ void ce_poison_on_abort_kernel(const int* __restrict__ status, void* a, int a_bf16, void* b, int b_bf16) {
  if (*status == 0) return;
  if (a) { if (a_bf16) *static_cast<__nv_bfloat16*>(a) = __float2bfloat16(__int_as_float(0x7fc00000)); else *static_cast<float*>(a) = __int_as_float(0x7fc00000); }
  if (b) { if (b_bf16) *static_cast<__nv_bfloat16*>(b) = __float2bfloat16(__int_as_float(0x7fc00000)); else *static_cast<float*>(b) = __int_as_float(0x7fc00000); }
}

// out = scale * sum over splits of partial [splits][n], in a fixed order; 4 elements per thread (n % 4 == 0)
template <typename TO>
__global__ void __launch_bounds__(256)
split_sum_kernel(const float* __restrict__ partial, long long n, int splits, const float* __restrict__ scale, const int* __restrict__ count,
                 TO* __restrict__ out) {
  if (count) splits = CountedSplits(*count, splits).splits;
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  float4 a = *reinterpret_cast<const float4*>(partial + i);
  for (int s = 1; s < splits; ++s) {
    const float4 b = *reinterpret_cast<const float4*>(partial + s * n + i);
    a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
  }
  const float g = scale ? *scale : 1.f;
  const float v[4] = {a.x * g, a.y * g, a.z * g, a.w * g};
  VecIO<TO, 4>::store(out + i, v);
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
// C[M, Nc] = A . B^T with bf16 operands.  A K-major operand is a row-major [M, K] (or [Nc, K]) tensor; an
// MN-major operand (A_MN / B_MN) is a row-major [K, M] (or [K, Nc]) tensor.  lda / ldb: row pitches.
template <int MODE, int MH, bool A_MN, bool B_MN>
static int launch_gemm(const __nv_bfloat16* A, long long lda, const __nv_bfloat16* B, long long ldb, void* C, bool c_f32,
                       long long ldc, int M, int Nc, int K, int splits, EpiParams ep, int* status, cudaStream_t st) {
  CUtensorMap ma, mb, mc;
  const bool oka = A_MN ? make_map_bf16(&ma, A, K, M, lda, 64) : make_map_bf16(&ma, A, M, K, lda, 128);
  const bool okb = B_MN ? make_map_bf16(&mb, B, K, Nc, ldb, 64) : make_map_bf16(&mb, B, Nc, K, ldb, 128);
  if (!oka || !okb) return HAWK_ERR_DEVICE;
  if (!C) mc = ma;  // nothing is stored through it
  else if (ep.part_rows ? !make_map_store(&mc, C, c_f32, Nc, ep.part_rows, 1, ldc, (long long)ep.part_rows * ldc)
                        : !make_map_store(&mc, C, c_f32, Nc, M, splits, ldc, (long long)M * ldc))
    return HAWK_ERR_DEVICE;
  auto kern = gemm_bf16_kernel<MODE, MH, A_MN, B_MN>;
  constexpr int GEMM_SMEM = GemmCfg<MH>::SMEM;
  // per call: the attribute belongs to the current device's copy of the kernel
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, GEMM_SMEM) != cudaSuccess) {
    (void)cudaGetLastError();
    return HAWK_ERR_LAUNCH;
  }
  const int m_tiles = (M + BM * MH - 1) / (BM * MH), n_tiles = (Nc + BN - 1) / BN, kblocks = (K + BK - 1) / BK;
  ep.M = M;
  ep.Nc = Nc;
  ep.k_per_split = (kblocks + splits - 1) / splits;
  const long long work = (long long)m_tiles * n_tiles * splits;
  const int pairs = ep.part_rows ? sm_count() / 2 : (int)std::min<long long>(work, sm_count() / 2);
  kern<<<2 * pairs, GEMM_THREADS, GEMM_SMEM, st>>>(ma, mb, mc, K, m_tiles, n_tiles, splits, ep, status);
  return launch_status();
}

// Tile height (MH) and K splits of a gradient GEMM.  With few output tiles most CTA pairs would idle (d act of 1548
// rows at H = 512: 14 tiles of 256 rows on 74 pairs, 310 us unsplit), so K is split; a K block costs 0.37 us with
// MH = 1 and 0.58 us with MH = 2 (two halves), a tile about 5 and 9 us of fill and epilogue, and splits a pass that
// sums the partials.  No split is left without K blocks.
struct GradPlan {
  int mh, splits;
};
static GradPlan plan_grad(long long M, long long Nc, long long K) {
  const long long kb = (K + BK - 1) / BK, pairs = std::max(1, sm_count() / 2);
  GradPlan best{1, 1};
  double best_us = 0;
  for (int mh = 1; mh <= 2; ++mh) {
    const long long tiles = ((M + BM * mh - 1) / (BM * mh)) * ((Nc + BN - 1) / BN);
    for (int s = 1; s <= 32 && s <= kb; ++s) {
      const long long per = (kb + s - 1) / s;
      if ((s - 1) * per >= kb) continue;
      const double waves = (double)((tiles * s + pairs - 1) / pairs);
      const double sum_us = s > 1 ? 4.0 + 4.0 * (double)M * Nc * (s + 1) / 5.0e6 : 0.0;
      const double us = waves * (mh == 1 ? per * 0.37 + 5.0 : per * 0.58 + 9.0) + sum_us;
      if (best_us == 0 || us < best_us) {
        best = GradPlan{mh, s};
        best_us = us;
      }
    }
  }
  return best;
}

static size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

// one gradient GEMM: `out` [M, Nc] in out_dtype, times *scale; `count` (null = K): how many of the K rows count, on the device
template <bool A_MN, bool B_MN>
static int grad_gemm(const __nv_bfloat16* A, long long lda, const __nv_bfloat16* B, long long ldb, void* out, int out_dtype,
                     const float* scale, int M, int Nc, int K, const int* count, float* scratch, int* status, cudaStream_t st) {
  const GradPlan plan = plan_grad(M, Nc, K);
  const int splits = plan.splits;
  EpiParams ep{};
  void* C = splits > 1 ? scratch : out;
  ep.out_bf16 = splits == 1 && out_dtype == HAWK_BF16;
  ep.scale = splits > 1 ? nullptr : scale;
  ep.count = count;
  ep.count_is_k = 1;
  int rc = plan.mh == 2
               ? launch_gemm<EPI_OUT, 2, A_MN, B_MN>(A, lda, B, ldb, C, !ep.out_bf16, Nc, M, Nc, K, splits, ep, status, st)
               : launch_gemm<EPI_OUT, 1, A_MN, B_MN>(A, lda, B, ldb, C, !ep.out_bf16, Nc, M, Nc, K, splits, ep, status, st);
  if (rc != HAWK_OK || splits == 1) return rc;
  const long long n = (long long)M * Nc;
  const unsigned blocks = (unsigned)((n / 4 + 255) / 256);
  if (out_dtype == HAWK_BF16)
    split_sum_kernel<<<blocks, 256, 0, st>>>(scratch, n, splits, scale, count, static_cast<__nv_bfloat16*>(out));
  else
    split_sum_kernel<<<blocks, 256, 0, st>>>(scratch, n, splits, scale, count, static_cast<float*>(out));
  return launch_status();
}

}  // namespace hawk
