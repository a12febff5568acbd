// mx4_gemm.cu — products of two MXFP4 operands on the 4-bit tensor cores (tcgen05.mma.kind::mxf4):
//   out[r][f] = sum over 32-blocks j of 2^(ea[r,j] - 127) 2^(eb[f,j] - 127) sum_{i in j} a[r,i] b[f,i]  (+ bias[f])
// for activation rows r and weight rows f, the weights one matrix or one for each group of consecutive
// activation rows (experts). The tensor core multiplies E2M1 codes as they are stored, applies both scales
// and adds up in f32 in tensor memory; a scale byte of 255 makes the sums that it takes part in NaN, 0 stands
// for 2^-127.
//
// The weight rows are the MMA's M side (128 per CTA), the activation rows its N side: a group's rows are cut
// into equal tiles, so a short group costs a short tile. A TMEM lane then is one feature, and a warp's stores
// of a column are 32 consecutive features of one output row.
//
// Scales come in words of four (one 128-element stretch of a row), the words of consecutive rows side by
// side, so that a group may start at any row: lane l of a warp loads the words of rows l, l + 32, l + 64 and
// l + 96 (each load coalesced) and stores them as the 16 bytes that the tensor core's scale atom (128 rows x
// 4 blocks, row r at 16 (r % 32) + 4 (r / 32)) has for it.
//
// Three kernels share this code. For many rows, pairs of CTAs (cta_group::2) work on 256 weight rows x up to 224
// activation rows, so that each SM fetches and reads half of the activation codes. For few rows, a CTA
// works on 128 weight rows x up to 64 activation rows, with more stages of weight codes in flight, and where
// there are far fewer tiles than SMs, a cluster splits a tile's K and adds the parts through distributed shared
// memory in rank order (so a result does not depend on timing).
//
// What bounds it, and measured figures (B200; device time back to back; cycles of single launches):
//   many rows: a stage of a pair (256 x 224 x 256) is 449 cycles of the tensor cores, and 34 KB come in for it on each
//   SM, at up to 54 bytes a cycle where the port from L2 gives 64. 8192^3: 189 us, 5.8 PFLOP/s, tensor work in 77 % of
//   the cycles, at 1.6 GHz under the power cap. 8192 x 5120 x 2880: 55 us, 4.4 PFLOP/s, 51 %: 100 k cycles for 120 stages
//   in line, of which about 2400 a tile (12 stages) and 17000 a launch are not the stages'. 32768 rows over 32 groups x
//   5760 x 2880: 265-320 us with the card's temperature, 3.4-4.1 PFLOP/s, 55 %.
//   few rows: HBM. 64 x 201088 x 2880: 61-63 us, 5.7-5.9 TB/s; 32 rows over 27 of 32 groups x 5760 x 2880: 44-57 us,
//   4.2-5.4 TB/s, of which about 4 us are the launch, the first stage's latency and the last epilogue.
// Tried and left out: asking L2 for the next tile's codes ahead of TMA (decode 74 us instead of 44), L2 promotion
// of 128 bytes or none (equal); taking the tensor memory only after the first loads are on their way (500 cycles
// sooner to the first stage, 5 % slower throughout); two epilogue chunks in flight (equal). Not built: tiles of 448
// activation rows in both accumulators (a quarter less L2 traffic, but nothing to compute while an epilogue of
// 2600 cycles runs, and coarser rounds of tiles).
//
// CTAs walk their tiles with the weight tile fastest: CTAs side by side share activation rows, and a group's
// weights stay in L2. Warps: 0 TMA (codes, 128-byte swizzle), 1 MMA, 2-3 and 12-17 scales (one for
// each stage of the ring, both operands' words; those of a warp's next turn are on their way while it waits for the
// stage's memory), 4-11 epilogue (two accumulators: one tile drains while the next is computed).
// Every wait is bounded; one that runs out sets the error word and the CTA winds down.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "cluster_count.h"
#include "common.cuh"
#include "mx4.h"
#include "mxf.cuh"

namespace oxg {
namespace {

using namespace sm100;
using namespace mxf;

constexpr int kTileW = 128;           // weight rows per CTA
constexpr int kStageK = 256;          // elements of K per stage: 128 bytes of codes
constexpr int kEpiWarps = 8;           // two for each quarter of the TMEM lanes, taking 32 columns in turn
constexpr int kScaleWarps = 8;         // a stage of the ring belongs to one of them
constexpr int kThreads = 32 * (2 + kEpiWarps + kScaleWarps);
constexpr int kMaxRanks = 8;           // CTAs that split a tile's K (the portable cluster size)
constexpr int kWBytes = kTileW * 128;  // a stage's weight codes

// PAIR: two CTAs per tile. NMAX: most activation rows per tile. SPLIT: a cluster per tile, K split.
template <bool PAIR_, int NMAX_, int STAGES_, bool SPLIT_>
struct Cfg {
  static constexpr bool PAIR = PAIR_, SPLIT = SPLIT_;
  static constexpr int NMAX = NMAX_, STAGES = STAGES_;
  static constexpr int CTAS = PAIR ? 2 : 1;
  static constexpr int X_GROUPS = (NMAX + 127) / 128;  // 128-row scale groups of the activation rows
  static constexpr int X_BYTES = NMAX / CTAS * 128;    // a stage's activation codes in one CTA
  static constexpr int SFW = 2 * kAtomBytes, SFX = 2 * X_GROUPS * kAtomBytes;  // two words of K each
  static constexpr int BYTES = (kWBytes + X_BYTES + SFW + SFX + 1023) / 1024 * 1024;
  static constexpr int SMEM = STAGES * BYTES + 1024;
  static constexpr int SFW_COL = 2 * NMAX, SFX_COL = SFW_COL + 8;  // TMEM columns behind the two accumulators
  static constexpr int COLS_USED = SFX_COL + 8 * X_GROUPS;
  static constexpr uint32_t TMEM_COLS = COLS_USED <= 128 ? 128 : (COLS_USED <= 256 ? 256 : 512);
  static_assert(COLS_USED <= 512 && X_BYTES % 1024 == 0, "tensor memory, swizzle atoms");
  static_assert(!(PAIR && SPLIT), "a pair does not split K");
  static_assert(STAGES <= kScaleWarps, "a scale warp for each stage of the ring");
  static_assert(!SPLIT || STAGES * BYTES >= NMAX * kTileW * 4, "the split's partial sums use the stages' memory");
};

struct Params {
  int m, n, k, groups;
  const int32_t *counts;
  const uint32_t *a_scales, *b_scales;
  const uint16_t *bias;
  void *out;
  size_t ldo;
  int n_tiles;      // weight tiles per group
  int k_steps;      // stages per tile
  int words;        // scale words per row
  int box;          // activation rows per TMA box
  int out_bf16;
  int pair_stores;  // bf16: n is even and rows start on 4-byte boundaries
  int err_word;
};
__device__ int g_err_words[kMx4ErrWords];

// Where a tile lies: its group's weight rows from f0, activation rows [row0, row0 + rows).
struct Tile {
  int g, f0, row0, rows, cols;  // cols: rows as the MMA's N
};
// The MMA's N comes in steps of 16, a pair's of 32 (each CTA holds half of its rows).
template <class C>
__host__ __device__ __forceinline__ int round_cols(int rows) {
  return (rows + 16 * C::CTAS - 1) / (16 * C::CTAS) * (16 * C::CTAS);
}

__device__ __forceinline__ void umma_mxf4_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                               uint32_t sfa_tmem, uint32_t sfb_tmem, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(sfa_tmem), "r"(sfb_tmem)
      : "memory");
}
// Arrives on the barrier at this offset in both CTAs of the pair once every MMA this thread issued before has
// completed.
__device__ __forceinline__ void umma_commit_both(uint64_t *bar) {
  umma_commit_pair(smem_addr(bar));
  umma_commit_pair(mapa_shared(smem_addr(bar), 1));
}
// An arrival on the other CTA's barrier and a wait for one, ordered between the two CTAs (without a scope both order
// a CTA's own threads only).
__device__ __forceinline__ void mbar_arrive_release_cluster(uint32_t bar_cl) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cl) : "memory");
}
__device__ __forceinline__ bool mbar_wait_acquire_cluster(uint64_t *bar, uint32_t parity, int *err, int code) {
  const long long t0 = clock64();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_addr(bar)), "r"(parity), "r"(1000000u)
        : "memory");
    if (ok) return true;
    if (clock64() - t0 > kWaitBudgetCycles) {
      atomicCAS(err, 0, code);
      return false;
    }
  }
}
// Copies 16 bytes of this CTA's shared memory to another CTA's and counts them on a barrier there. The copy comes after
// what the thread has written (and fenced for the async proxy) before it, and its count is a release between the CTAs:
// the way for rank 1 to say that its scale words are in place. An arrival with a release at cluster scope says the
// same but holds the warp for some 1400 cycles (8192 x 5120 x 2880: 61 us against 55.4, 1037 x 2880 x 4096: 12.2
// against 10.6).
__device__ __forceinline__ void copy_to_peer(uint32_t dst_cl, uint32_t src, uint32_t bar_cl) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], 16, [%2];" ::"r"(dst_cl),
               "r"(src), "r"(bar_cl)
               : "memory");
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr_cl) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr_cl)
               : "memory");
  return v;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// True in one lane of a converged warp, the same one every time. The TMA and tensor-core instructions take
// their operands from uniform registers: issued behind elect.sync by a warp that stays together they cost a few
// cycles each, behind `lane == 0` (where nothing tells the compiler that one lane is left) 40 to 130 (128
// weight rows x N x 256 of K: 513 cycles a stage at N = 256 and 400 at N = 16, against 1054 at either).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(p));
  return p != 0;
}

// A CTA's way through its tiles: item = xt * n_tiles + wt, the wt-th weight tile of activation tile xt (of group g).
struct Walk {
  int item, xt, wt, g;
};

template <class C>
__global__ void __launch_bounds__(kThreads, 1)
    mx4_gemm_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const Params p) {
  constexpr bool PAIR = C::PAIR, SPLIT = C::SPLIT;
  constexpr int STAGES = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *stages = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t full_[STAGES], empty_[STAGES];
  __shared__ uint64_t acc_full[2], acc_empty[2], mma_done;
  __shared__ __align__(16) uint8_t note_[PAIR ? STAGES : 1][16];  // where rank 1 copies to
  __shared__ uint32_t tmem_slot;
  __shared__ int cols_[STAGES];  // the MMA's N for a stage's tile, from the TMA warp
  __shared__ int tile0_[kMx4MaxGroups + 1], row0_[kMx4MaxGroups + 1], per_[kMx4MaxGroups];  // per: rows of a group's tiles

  int *const err = g_err_words + p.err_word;
  const int warp = __shfl_sync(0xFFFFFFFFu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = PAIR || SPLIT ? cluster_ctarank() : 0u;
  uint32_t n_ranks = C::CTAS;
  if (SPLIT) asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n_ranks));
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_[s], 2);  // the codes' bytes (and rank 1's note), and this CTA's scales
      mbar_init(&empty_[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kEpiWarps * C::CTAS);
    }
    mbar_init(&mma_done, 1);
    fence_mbar_init();
  }
  if (warp == 3 && elect_one()) {
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_w);
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(&tmem_slot, C::TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&tmem_slot, C::TMEM_COLS);
      tmem_relinquish();
    }
  }
  launch_dependents();
  wait_prerequisites();  // nothing above touches memory that an earlier kernel writes
  if (warp == 2 && !p.counts) {
    if (lane == 0) {
      const int t = (p.m + C::NMAX - 1) / C::NMAX;
      row0_[0] = tile0_[0] = 0;
      row0_[1] = p.m;
      tile0_[1] = t;
      per_[0] = round_cols<C>((p.m + t - 1) / t);
    }
  } else if (warp == 2) {  // running sums of the groups' rows and activation tiles
    int rows_run = 0, tiles_run = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
      const int g = g0 + lane;
      int c = (int)ld_u32_if(g < p.groups, p.counts + g);
      bool bad = c < 0;
      c = max(c, 0);
      long long r = c;  // rows up to and including this group's
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xFFFFFFFFu, r, o);
        if (lane >= o) r += t;
      }
      r += rows_run;
      bad |= r > p.m;
      if (bad && blockIdx.x == 0) atomicCAS(err, 0, kMx4ErrCounts);
      // counts beyond the rows there are: the groups end with the rows
      const int first = (int)min(r - c, (long long)p.m), last = (int)min(r, (long long)p.m);
      int t = (last - first + C::NMAX - 1) / C::NMAX;
      const int per = round_cols<C>((last - first + max(t, 1) - 1) / max(t, 1));  // equal tiles
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, t, o);
        if (lane >= o) t += u;
      }
      if (g < p.groups) {
        row0_[g + 1] = last;
        per_[g] = per;
        tile0_[g + 1] = tiles_run + t;
      }
      rows_run = __shfl_sync(0xFFFFFFFFu, last, 31);
      tiles_run += __shfl_sync(0xFFFFFFFFu, t, 31);
    }
    if (lane == 0) row0_[0] = tile0_[0] = 0;
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int total = tile0_[p.groups] * p.n_tiles;  // the launch has checked that this fits
  // tiles of this CTA (pair, cluster): item0, item0 + step, ...; stages [k_lo, k_hi) of each
  const int item0 = (int)(blockIdx.x / n_ranks);
  const int step = SPLIT ? total : (int)(gridDim.x / n_ranks);  // a split's cluster has one tile
  const int k_lo = SPLIT ? (int)((long long)p.k_steps * rank / n_ranks) : 0;
  const int k_hi = SPLIT ? (int)((long long)p.k_steps * (rank + 1) / n_ranks) : p.k_steps;

  const int step_x = step / p.n_tiles, step_w = step - step_x * p.n_tiles;

  // the last group from g on that starts at or before xt: empty ones before it start there too
  auto group_of = [&](int g, int xt) {
    if (tile0_[g + 1] > xt) return g;
    int lo = g, hi = p.groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tile0_[mid] <= xt) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  auto start = [&] {
    Walk w;
    w.item = item0;
    w.xt = item0 / p.n_tiles;
    w.wt = item0 - w.xt * p.n_tiles;
    w.g = item0 < total ? group_of(0, w.xt) : 0;
    return w;
  };
  auto advance = [&](Walk &w) {
    w.item += step;
    w.xt += step_x;
    w.wt += step_w;
    if (w.wt >= p.n_tiles) {
      w.wt -= p.n_tiles;
      ++w.xt;
    }
    if (w.item < total) w.g = group_of(w.g, w.xt);
  };
  auto tile_of = [&](const Walk &w) {
    const int first = row0_[w.g], rows = row0_[w.g + 1] - first, per = per_[w.g];
    const int i0 = (w.xt - tile0_[w.g]) * per;
    Tile t;
    t.g = w.g;
    t.f0 = w.wt * (kTileW * C::CTAS) + (PAIR ? (int)rank * kTileW : 0);
    t.row0 = first + i0;
    t.rows = min(per, rows - i0);
    t.cols = round_cols<C>(t.rows);
    return t;
  };
  auto rank0 = [&](void *at) { return PAIR ? mapa_shared(smem_addr(at), 0) : smem_addr(at); };
  // a pair's barriers may be completed from either CTA
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    return PAIR ? mbar_wait_acquire_cluster(bar, parity, err, kMx4ErrWait) : mbar_wait(bar, parity, err, kMx4ErrWait);
  };

  if (warp == 0) {
    // ------------------------------------------------------------ codes
    int s = 0, round = 0;
    bool ok = true;
    for (Walk w = start(); ok && w.item < total; advance(w)) {
      const Tile t = tile_of(w);
      const int half = t.cols / C::CTAS, boxes = (half + p.box - 1) / p.box;
      const int x0 = t.row0 + (PAIR ? (int)rank * half : 0);
      const uint32_t tx = (uint32_t)(C::CTAS * (kWBytes + boxes * p.box * 128)) + (PAIR ? 16u : 0u);  // rank 1's note
      for (int ks = k_lo; ks < k_hi; ++ks) {
        if (round > 0 && !(ok = wait(&empty_[s], (round - 1) & 1))) break;
        if (elect_one()) {
          uint8_t *st = stages + s * C::BYTES;
          cols_[s] = t.cols;
          if (rank == 0 || SPLIT) mbar_arrive_expect_tx(&full_[s], tx);
          if (PAIR) {
            const uint32_t bar = mapa_shared(smem_addr(&full_[s]), 0);
            tma_load_3d_pair(st, &tm_w, bar, ks * 128, t.f0, t.g);
            for (int b = 0; b < boxes; ++b)
              tma_load_2d_pair(st + kWBytes + b * p.box * 128, &tm_x, bar, ks * 128, x0 + b * p.box);
          } else {
            tma_load_3d(st, &tm_w, &full_[s], ks * 128, t.f0, t.g);
            for (int b = 0; b < boxes; ++b)
              tma_load_2d(st + kWBytes + b * p.box * 128, &tm_x, &full_[s], ks * 128, x0 + b * p.box);
          }
        }
        __syncwarp();
        if (++s == STAGES) {
          s = 0;
          ++round;
        }
      }
    }
    if (!ok && (rank == 0 || SPLIT)) {
      // copies in flight land before the CTA (pair) ends: stages below s have been loaded in this round. A
      // barrier whose scales never came costs one full wait, long after any copy has landed.
      for (int i = 0; i < STAGES; ++i) {
        const int last = i < s ? round : round - 1;
        if (last >= 0 && !wait(&full_[i], last & 1)) break;
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA (rank 0 of a pair)
    if (rank == 0 || SPLIT) {
      int s = 0, phase = 0, j = 0;
      bool ok = true;
      const uint32_t sfw = tmem + C::SFW_COL, sfx = tmem + C::SFX_COL;
      for (int item = item0; ok && item < total; item += step, ++j) {
        const int buf = j & 1, rr = j >> 1;
        if (rr > 0 && !(ok = wait(&acc_empty[buf], (rr - 1) & 1))) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(buf * C::NMAX);
        uint32_t id0 = 0, id2 = 0;
        for (int ks = k_lo; ks < k_hi; ++ks) {
          if (!(ok = wait(&full_[s], phase))) break;
          tc_fence_after();
          if (ks == k_lo) {
            const int cols = cols_[s];
            id0 = idesc_mxf4(kTileW * C::CTAS, cols, 0);
            id2 = idesc_mxf4(kTileW * C::CTAS, cols, 2);
          }
          if (elect_one()) {
            const uint32_t st = smem_addr(stages + s * C::BYTES), sf = st + kWBytes + C::X_BYTES;
            const int mmas = (p.k - ks * kStageK + 63) / 64;  // 4, but for the end of K
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              auto cp = [](uint32_t col, uint32_t atom) {
                if (PAIR) utccp_atom_pair(col, atom);
                else utccp_atom(col, atom);
              };
              cp(sfw + 4 * w, sf + w * kAtomBytes);
              cp(sfx + 4 * C::X_GROUPS * w, sf + C::SFW + C::X_GROUPS * w * kAtomBytes);
              if (C::X_GROUPS > 1) cp(sfx + 4 * C::X_GROUPS * w + 4, sf + C::SFW + (C::X_GROUPS * w + 1) * kAtomBytes);
            }
            const uint64_t wd = desc_sw128_kmajor(st), xd = desc_sw128_kmajor(st + kWBytes);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              if (kk < mmas) {
                const uint32_t half = (uint32_t)(kk & 1) << 31;  // scale columns 2 and 3 of the word
                const uint32_t fw = (sfw + 4 * (kk >> 1)) | half, fx = (sfx + 4 * C::X_GROUPS * (kk >> 1)) | half;
                const uint32_t add = ks > k_lo || kk > 0;
                if (PAIR) umma_mxf4_pair(d, wd + 2 * kk, xd + 2 * kk, kk & 1 ? id2 : id0, fw, fx, add);
                else umma_mxf4(d, wd + 2 * kk, xd + 2 * kk, kk & 1 ? id2 : id0, fw, fx, add);
              }
            }
            if (PAIR) umma_commit_both(&empty_[s]);
            else umma_commit(&empty_[s]);
            if (ks + 1 == k_hi) {
              if (PAIR) umma_commit_both(&acc_full[buf]);
              else umma_commit(&acc_full[buf]);
            }
          }
          __syncwarp();
          if (++s == STAGES) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      // no MMA is left when the tensor memory goes
      if (elect_one()) {
        if (PAIR) umma_commit_pair(smem_addr(&mma_done));
        else umma_commit(&mma_done);
      }
      __syncwarp();
      mbar_wait(&mma_done, 0, err, kMx4ErrWait);
    }
  } else if (warp < 4 || warp >= 4 + kEpiWarps) {
    // ------------------------------------------------------------ scales
    // a warp for each stage of the ring: both operands' words
    const int slot = warp < 4 ? warp - 2 : warp - 2 - kEpiWarps;  // 0 .. kScaleWarps - 1
    constexpr int XQ = (C::NMAX + 31) / 32;  // 32-row pieces of the activation rows
    if (slot < STAGES && item0 < total) {
      uint32_t vw[2][4], vx[2][XQ];  // the words of this warp's next stage
      Walk at = start();
      Tile t = tile_of(at);
      int ks = k_lo;
      auto skip = [&](int stages) {
        ks += stages;
        if (ks < k_hi) return;
        while (ks >= k_hi && at.item < total) {
          ks -= k_hi - k_lo;
          advance(at);
        }
        if (at.item < total) t = tile_of(at);
      };
      skip(slot);
      auto fetch = [&] {
        if (at.item >= total) return;
        const int in_w = min(p.n - t.f0, kTileW) - lane, in_x = min(p.m - t.row0, t.cols) - lane;  // this lane's rows 32 q < in
        const uint32_t *w_src = p.b_scales + (size_t)t.g * p.words * p.n + t.f0 + lane + (size_t)(2 * ks) * p.n;
        const uint32_t *x_src = p.a_scales + t.row0 + lane + (size_t)(2 * ks) * p.m;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const bool held = 2 * ks + w < p.words;
          const int lim_w = held ? in_w : 0, lim_x = held ? in_x : 0;
#pragma unroll
          for (int q = 0; q < 4; ++q) vw[w][q] = ld_u32_if(32 * q < lim_w, w_src + 32 * q);
#pragma unroll
          for (int q = 0; q < XQ; ++q) vx[w][q] = ld_u32_if(32 * q < lim_x, x_src + 32 * q);
          w_src += p.n;
          x_src += p.m;
        }
        skip(STAGES);
      };
      const int mine = ((total - 1 - item0) / step + 1) * (k_hi - k_lo) - slot;
      const int left = (mine + STAGES - 1) / STAGES;  // this warp's stages
      uint4 *sf = reinterpret_cast<uint4 *>(stages + slot * C::BYTES + kWBytes + C::X_BYTES) + lane;
      fetch();
      for (int round = 0; round < left; ++round) {
        if (round > 0 && !wait(&empty_[slot], (round - 1) & 1)) break;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          sf[w * (kAtomBytes / 16)] = make_uint4(vw[w][0], vw[w][1], vw[w][2], vw[w][3]);
#pragma unroll
          for (int q = 0; q < XQ; q += 4)
            sf[(C::SFW + (C::X_GROUPS * w + q / 4) * kAtomBytes) / 16] =
                make_uint4(vx[w][q], q + 1 < XQ ? vx[w][q + 1 < XQ ? q + 1 : q] : 0u,
                           q + 2 < XQ ? vx[w][q + 2 < XQ ? q + 2 : q] : 0u, q + 3 < XQ ? vx[w][q + 3 < XQ ? q + 3 : q] : 0u);
        }
        fence_proxy_async_smem();  // for the tensor cores
        __syncwarp();
        if (lane == 0) {
          if (PAIR && rank != 0) copy_to_peer(rank0(note_[slot]), smem_addr(sf), rank0(&full_[slot]));
          else mbar_arrive(&full_[slot]);
        }
        fetch();
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3, half = (warp - 4) >> 2;  // TMEM lane quarter; which 32-column chunks
    int j = 0;
    for (Walk w = start(); w.item < total; advance(w), ++j) {
      const Tile t = tile_of(w);
      const int buf = j & 1;
      if (!wait(&acc_full[buf], (j >> 1) & 1)) break;
      tc_fence_after();
      const int f = t.f0 + q * 32 + lane;
      const bool in = f < p.n;
      const float bias = p.bias && in && !SPLIT ? bf16_to_f32(ld_u16(p.bias + (size_t)t.g * p.n + f)) : 0.f;
      const uint32_t base = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * C::NMAX);
      const bool whole = t.f0 + kTileW <= p.n;
      for (int c0 = 32 * half; c0 < t.rows; c0 += 64) {
        uint32_t v[32];
        tmem_ld_32_async(base + (uint32_t)c0, v);
        tmem_wait_ld(v);
        if (SPLIT) {
          // this part of K: [column][feature], where the stages were (all of them have been read)
          float *part = reinterpret_cast<float *>(stages) + c0 * kTileW + q * 32 + lane;
#pragma unroll
          for (int i = 0; i < 32; ++i) part[i * kTileW] = __uint_as_float(v[i]);
        } else if (p.out_bf16 && p.pair_stores) {
          // lanes 2i and 2i + 1 trade halves: the even one stores both features of an even column, the odd
          // one of an odd column, 4 bytes each (n is even, so both exist or neither does)
          const int odd = lane & 1, lim = in ? t.rows - c0 - odd : 0;
          const size_t two = 2 * p.ldo;
          uint16_t *o = static_cast<uint16_t *>(p.out) + (size_t)(t.row0 + c0 + odd) * p.ldo + (f - odd);
          float other[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            other[i] = __shfl_xor_sync(0xFFFFFFFFu, __uint_as_float(odd ? v[2 * i] : v[2 * i + 1]) + bias, 1);
          uint32_t both[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float mine = __uint_as_float(odd ? v[2 * i + 1] : v[2 * i]) + bias;
            both[i] = odd ? pack_bf16x2(other[i], mine) : pack_bf16x2(mine, other[i]);
          }
          if (whole && c0 + 32 <= t.rows) {
#pragma unroll
            for (int i = 0; i < 16; ++i, o += two) *reinterpret_cast<uint32_t *>(o) = both[i];
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i, o += two)
              if (2 * i < lim) *reinterpret_cast<uint32_t *>(o) = both[i];
          }
        } else {
          const int lim = in ? t.rows - c0 : 0;
          const size_t o = (size_t)(t.row0 + c0) * p.ldo + f;
          if (p.out_bf16) {
            uint16_t *d = static_cast<uint16_t *>(p.out) + o;
#pragma unroll
            for (int i = 0; i < 32; ++i, d += p.ldo)
              if (i < lim) *d = (uint16_t)pack_bf16x2(__uint_as_float(v[i]) + bias, 0.f);
          } else {
            float *d = static_cast<float *>(p.out) + o;
            if (whole && c0 + 32 <= t.rows) {
#pragma unroll
              for (int i = 0; i < 32; ++i, d += p.ldo) *d = __uint_as_float(v[i]) + bias;
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i, d += p.ldo)
                if (i < lim) *d = __uint_as_float(v[i]) + bias;
            }
          }
        }
      }
      if ((total - w.item - 1) / 2 < step) continue;  // nothing waits for this accumulator any more
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR && rank != 0) mbar_arrive_release_cluster(rank0(&acc_empty[buf]));
        else mbar_arrive(&acc_empty[buf]);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (SPLIT) {
    // out = the parts of all ranks, added in rank order; rank r takes columns r, r + ranks, ..., a warp one of
    // them at a time, four features a lane, the ranks' loads all on their way before the first is added
    cluster_sync();
    if (item0 < total) {
      const Tile t = tile_of(start());
      const int f = t.f0 + 4 * lane;
      float bias[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        bias[i] = p.bias && f + i < p.n ? bf16_to_f32(ld_u16(p.bias + (size_t)t.g * p.n + f + i)) : 0.f;
      for (int c = (int)rank + warp * (int)n_ranks; c < t.rows; c += kThreads / 32 * (int)n_ranks) {
        const uint32_t part = smem_addr(stages) + (uint32_t)(c * kTileW + 4 * lane) * 4;
        float4 v[kMaxRanks];
#pragma unroll
        for (int r = 0; r < kMaxRanks; ++r)
          if (r < (int)n_ranks) v[r] = ld_cluster_f32x4(mapa_shared(part, r));
        float4 sum = v[0];
#pragma unroll
        for (int r = 1; r < kMaxRanks; ++r)
          if (r < (int)n_ranks) {
            sum.x += v[r].x;
            sum.y += v[r].y;
            sum.z += v[r].z;
            sum.w += v[r].w;
          }
        const float y[4] = {sum.x + bias[0], sum.y + bias[1], sum.z + bias[2], sum.w + bias[3]};
        const size_t o = (size_t)(t.row0 + c) * p.ldo + f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (f + i >= p.n) break;
          if (p.out_bf16) static_cast<uint16_t *>(p.out)[o + i] = (uint16_t)pack_bf16x2(y[i], 0.f);
          else static_cast<float *>(p.out)[o + i] = y[i];
        }
      }
    }
    __syncthreads();
    cluster_sync();  // no CTA leaves while another may still read its part
  }
  if (PAIR) {
    cluster_sync();
    tc_fence_after();
  }
  if (warp == 1) {
    if (PAIR) tmem_dealloc_pair(tmem, C::TMEM_COLS);
    else tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                             const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void *f = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
                   q == cudaDriverEntryPointSuccess
               ? reinterpret_cast<EncodeFn>(f)
               : (EncodeFn) nullptr;
  }();
  return fn;
}
// Rows of k / 2 code bytes in boxes of 128 bytes x box_rows, 128-byte swizzle; outside the matrix reads 0.
cudaError_t code_map(CUtensorMap *map, const void *base, int rank, int k, int rows, int groups, int box_rows) {
  EncodeFn fn = encode_fn();
  if (!fn) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {(cuuint64_t)k / 2, (cuuint64_t)rows, (cuuint64_t)groups};
  const cuuint64_t strides[2] = {(cuuint64_t)k / 2, (cuuint64_t)rows * (k / 2)};
  const cuuint32_t box[3] = {128u, (cuuint32_t)box_rows, 1u}, es[3] = {1u, 1u, 1u};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, (cuuint32_t)rank, const_cast<void *>(base), dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}


// Clusters of `ranks` CTAs that the current device holds side by side (its processing clusters are not multiples of
// it), or what its SMs would hold where it does not say.
template <class C>
int clusters_at_once(int ranks, int dev, int n_sms) {
  static ClusterCount known[kMaxRanks + 1];
  return known[ranks].get(dev, n_sms / ranks, [&] {
    auto kern = mx4_gemm_kernel<C>;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(kThreads);
    cfg.gridDim = dim3((unsigned)(n_sms / ranks * ranks));
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
      cudaGetLastError();  // not the launch's error
      n = 0;
    }
    return n;
  });
}

template <class C>
cudaError_t launch_cfg(const Mx4GemmArgs &a, Params &p, int n_sms, int dev, int ranks, cudaStream_t stream) {
  constexpr int kTile = kTileW * C::CTAS;
  p.n_tiles = (a.n + kTile - 1) / kTile;
  // no more activation tiles than this, whatever the counts are
  const long long x_tiles = a.counts ? (long long)a.m / C::NMAX + std::min(a.groups, a.m) : ((long long)a.m + C::NMAX - 1) / C::NMAX;
  // one box where all tiles are alike; else two at most (16-row steps would be seven copies a stage)
  if (a.counts) p.box = C::NMAX / C::CTAS / 2;
  else p.box = round_cols<C>((int)((a.m + x_tiles - 1) / x_tiles)) / C::CTAS;
  CUtensorMap tm_x, tm_w;
  cudaError_t st;
  if ((st = code_map(&tm_x, a.a, 2, a.k, a.m, 1, p.box))) return st;
  if ((st = code_map(&tm_w, a.b, 3, a.k, a.n, a.groups, kTileW))) return st;
  const long long tiles = x_tiles * p.n_tiles;
  if (tiles > 0x3FFFFFFF || tiles * p.k_steps > 0x7FFFFFFF) return cudaErrorInvalidValue;  // no GPU's memory holds such operands
  auto kern = mx4_gemm_kernel<C>;
  static std::atomic<uint64_t> ready{0};  // a bit for each device (of the first 64) that knows the attribute
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    if ((st = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM))) return st;
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)(C::SPLIT ? ranks : C::CTAS);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = C::SPLIT || C::PAIR ? 2 : 1;
  long long at_once = n_sms;  // tiles in work side by side; the GPU's clusters may not hold every SM
  if (C::PAIR) at_once = std::min(clusters_at_once<C>(2, dev, n_sms), n_sms / 2);
  cfg.gridDim = dim3((unsigned)(C::SPLIT ? tiles * ranks : C::CTAS * std::min(at_once, tiles)));
  return cudaLaunchKernelEx(&cfg, kern, tm_x, tm_w, p);
}

using Pair = Cfg<true, 224, 6, false>;
using Few = Cfg<false, 64, 8, false>;
using FewSplit = Cfg<false, 64, 8, true>;

}  // namespace

cudaError_t mx4_take_error(int word, int *code) {
  const size_t at = sizeof(int) * (size_t)word;
  cudaError_t st = cudaMemcpyFromSymbol(code, g_err_words, sizeof(int), at);
  const int none = 0;
  if (st == cudaSuccess && *code) st = cudaMemcpyToSymbol(g_err_words, &none, sizeof(int), at);
  return st;
}

cudaError_t launch_mx4_gemm(const Mx4GemmArgs &a, int n_sms, cudaStream_t stream) {
  if (a.m == 0 || a.n == 0 || a.groups == 0) return cudaSuccess;
  int dev = 0;
  const cudaError_t st = cudaGetDevice(&dev);
  if (st) return st;
  Params p{};
  p.m = a.m;
  p.n = a.n;
  p.k = a.k;
  p.groups = a.groups;
  p.counts = a.counts;
  p.a_scales = a.a_scales;
  p.b_scales = a.b_scales;
  p.bias = a.bias;
  p.out = a.out;
  p.ldo = a.ldo;
  p.k_steps = (a.k + kStageK - 1) / kStageK;
  p.words = (a.k + 127) / 128;
  p.out_bf16 = a.out_bf16;
  p.pair_stores = a.n % 2 == 0 && (a.ldo % 2 == 0 || a.m == 1) && (uintptr_t)a.out % 4 == 0;
  p.err_word = a.err_word;
  // Which kernel: estimates in ns from launches back to back on a B200 (k 512 .. 8192, n 640 .. 20480, m 1 .. 1024,
  // codes in L2). A launch costs 4100 with single CTAs and 5000 with pairs; a stage 265 in a CTA with up to 64
  // rows, 270 in a pair with up to 128 and 300 above; adding up a split 1300 + 17 a column. For instance 448 x 2880
  // x 2880 takes 9.0 us in pairs and 10.9 in CTAs (two rounds of tiles), 256 x 2880 x 2880 8.4 and 7.6; 64 x 2880 x
  // 8192 12.6 unsplit and 8.8 over 4 CTAs, 64 x 2880 x 2880 7.3 and 7.6. Bound by HBM they are alike (64 x 201088 x
  // 2880: 55.6 and 56.9). Groups count as if they had even shares of the rows.
  const long long held = std::min(a.groups, a.m), rows = (a.m + held - 1) / held;
  auto tiles = [&](int w, int x) { return (a.n + w - 1ll) / w * held * ((rows + x - 1) / x); };
  auto rounds = [](long long tiles, int at_once) { return (double)((tiles + at_once - 1) / at_once); };
  const long long few_tiles = tiles(kTileW, Few::NMAX), pair_tiles = tiles(2 * kTileW, Pair::NMAX);
  const double pair_ns = 5000 + rounds(pair_tiles, n_sms / 2) * p.k_steps * (rows > 128 ? 300 : 270);
  double few_ns = 4100 + rounds(few_tiles, n_sms) * p.k_steps * 265;
  int ranks = 1;
  for (int r = 2; r <= kMaxRanks && 2 * r <= p.k_steps && r * few_tiles <= n_sms; ++r) {
    const double ns = 4100 + (p.k_steps + r - 1) / r * 265. + 1300 + 17. * std::min<long long>(rows, Few::NMAX);
    if (ns < few_ns && few_tiles <= clusters_at_once<FewSplit>(r, dev, n_sms)) {
      few_ns = ns;
      ranks = r;
    }
  }
  int kernel = pair_ns < few_ns ? kMx4Pair : (ranks > 1 ? kMx4Split : kMx4Few);
  if (a.kernel != kMx4Auto) {
    kernel = a.kernel;
    ranks = a.ranks;
    // every rank has a stage to add, or the sums would be waited for in vain
    if (kernel == kMx4Split && (ranks < 2 || ranks > kMaxRanks || ranks > p.k_steps)) return cudaErrorInvalidValue;
  }
  if (a.ran) {
    a.ran[0] = kernel;
    a.ran[1] = kernel == kMx4Split ? ranks : 1;
  }
  if (kernel == kMx4Pair) return launch_cfg<Pair>(a, p, n_sms, dev, 1, stream);
  if (kernel == kMx4Split) return launch_cfg<FewSplit>(a, p, n_sms, dev, ranks, stream);
  return launch_cfg<Few>(a, p, n_sms, dev, 1, stream);
}

}  // namespace oxg
