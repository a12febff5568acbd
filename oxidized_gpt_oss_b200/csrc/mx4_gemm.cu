// mx4_gemm.cu — products of two MXFP4 operands on the 4-bit tensor cores (tcgen05.mma.kind::mxf4):
//   out[r][f] = sum over 32-blocks j of 2^(ea[r,j] - 127) 2^(eb[f,j] - 127) sum_{i in j} a[r,i] b[f,i]  (+ bias[f])
// for activation rows r and weight rows f, the weights one matrix or one for each group of consecutive
// activation rows (experts). The tensor core multiplies E2M1 codes as they are stored, applies both scales
// and adds up in f32 in tensor memory; a scale byte of 255 makes the sums that it takes part in NaN, 0 stands
// for 2^-127.
//
// The weight rows are the MMA's M side (128 a tile), the activation rows its N side (up to kTileN a tile,
// in steps of 16: a group's rows are cut into equal tiles, so a short group costs a short tile and one row
// costs 16). A TMEM lane then is one feature, and a warp's stores of a column are 32 consecutive features of
// one output row.
//
// Scales come in words of four (one 128-element stretch of a row), the words of consecutive rows side by
// side, so that a group may start at any row: a warp's 32 lanes fetch 32 rows' words with one coalesced
// 4-byte cp.async each and drop them where the tensor core's 512-byte atom (128 rows x 4 blocks, row r at
// 16 (r % 32) + 4 (r / 32)) wants them.
//
// One CTA per SM walks its tiles (weight tile fastest, so CTAs side by side share activation rows and a
// group's weights stay in L2). Warps: 0 TMA (codes, 128-byte swizzle), 1 MMA, 2 scales, 3 idle, 4-7
// epilogue (two accumulators, so it drains one tile while the next is computed).
// Every wait is bounded; one that runs out sets the error word and the CTA winds down.
#include <cuda.h>

#include <algorithm>

#include "common.cuh"
#include "mx4.h"
#include "mxf.cuh"

namespace oxg {
namespace {

using namespace sm100;
using namespace mxf;

constexpr int kTileW = 128;                      // weight rows per tile
constexpr int kTileN = 224;                      // most activation rows per tile
constexpr int kStageK = 256;                     // elements of K per stage: 128 bytes of codes
constexpr int kBoxN = 32;                        // activation rows per TMA box
constexpr int kWBytes = kTileW * 128;            // a stage's weight codes
constexpr int kXBytes = kTileN * 128;            // a stage's activation codes
constexpr int kSfw = 2 * kAtomBytes;             // two words of K for 128 weight rows
constexpr int kSfx = 4 * kAtomBytes;             // two words for each 128 activation rows
constexpr int kStageBytes = kWBytes + kXBytes + kSfw + kSfx;
constexpr int kStages = 4;
constexpr int kThreads = 256;
constexpr int kEpiWarps = 4;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kSfwCol = 2 * kTileN, kSfxCol = kSfwCol + 8;  // behind the two accumulators
static_assert(kStageBytes % 1024 == 0 && kSfxCol + 16 <= kTmemCols, "stage and tensor-memory layout");

struct Params {
  int m, n, k, groups;
  const int32_t *counts;
  const uint32_t *a_scales, *b_scales;
  const uint16_t *bias;
  void *out;
  size_t ldo;
  int n_tiles;     // weight tiles per group
  int k_steps;     // stages per tile
  int words;       // scale words per row
  int out_bf16;
  int pair_stores;  // bf16 rows start on 4-byte boundaries
  int *err;
};

// Where a tile lies: its group's weight rows from f0, activation rows [row0, row0 + rows).
struct Tile {
  int g, f0, row0, rows, cols;  // cols: rows rounded up to the MMA's 16
};

// Copies 4 bytes (or writes 0) asynchronously.
__device__ __forceinline__ void cp_async_4_zfill(uint32_t dst, const void *src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4u : 0u) : "memory");
}

__global__ void __launch_bounds__(kThreads, 1)
    mx4_gemm_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *stages = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t full_[kStages], scaled_[kStages], empty_[kStages];
  __shared__ uint64_t acc_full[2], acc_empty[2], mma_done;
  __shared__ uint32_t tmem_slot;
  __shared__ int tile0_[kMx4MaxGroups + 1], row0_[kMx4MaxGroups + 1];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_[s], 1);
      mbar_init(&scaled_[s], 1);
      mbar_init(&empty_[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kEpiWarps);
    }
    mbar_init(&mma_done, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  if (warp == 2) {  // running sums of the groups' rows and activation tiles
    int rows_run = 0, tiles_run = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
      const int g = g0 + lane;
      int c = g < p.groups ? (p.counts ? __ldg(p.counts + g) : p.m) : 0;
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
      if (bad && blockIdx.x == 0) atomicCAS(p.err, 0, kMx4ErrCounts);
      // counts beyond the rows there are: the groups end with the rows
      const int first = (int)min(r - c, (long long)p.m), last = (int)min(r, (long long)p.m);
      int t = (last - first + kTileN - 1) / kTileN;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, t, o);
        if (lane >= o) t += u;
      }
      if (g < p.groups) {
        row0_[g + 1] = last;
        tile0_[g + 1] = tiles_run + t;
      }
      rows_run = __shfl_sync(0xFFFFFFFFu, last, 31);
      tiles_run += __shfl_sync(0xFFFFFFFFu, t, 31);
    }
    if (lane == 0) row0_[0] = tile0_[0] = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const long long total = (long long)tile0_[p.groups] * p.n_tiles;

  auto tile_at = [&](long long item) {
    const int xt = (int)(item / p.n_tiles);
    int lo = 0, hi = p.groups;  // the last group that starts at or before xt: empty ones before it start there too
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tile0_[mid] <= xt) lo = mid;
      else hi = mid;
    }
    const int first = row0_[lo], rows = row0_[lo + 1] - first, nt = tile0_[lo + 1] - tile0_[lo];
    const int step = ((rows + nt - 1) / nt + 15) & ~15;  // equal tiles, a multiple of 16 rows
    Tile t;
    t.g = lo;
    t.f0 = (int)(item - (long long)xt * p.n_tiles) * kTileW;
    const int i0 = (xt - tile0_[lo]) * step;
    t.row0 = first + i0;
    t.rows = max(0, min(step, rows - i0));
    t.cols = max(16, (t.rows + 15) & ~15);
    return t;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ codes
    if (lane == 0) {
      prefetch_tmap(&tm_x);
      prefetch_tmap(&tm_w);
      int s = 0, round = 0;
      int last_round[kStages];
#pragma unroll
      for (int i = 0; i < kStages; ++i) last_round[i] = -1;
      bool ok = true;
      for (long long item = blockIdx.x; ok && item < total; item += gridDim.x) {
        const Tile t = tile_at(item);
        const int boxes = (t.cols + kBoxN - 1) / kBoxN;
        for (int ks = 0; ks < p.k_steps; ++ks) {
          if (round > 0 && !(ok = mbar_wait(&empty_[s], (round - 1) & 1, p.err, kMx4ErrWait))) break;
          uint8_t *st = stages + s * kStageBytes;
          mbar_arrive_expect_tx(&full_[s], (uint32_t)(kWBytes + boxes * kBoxN * 128));
          tma_load_3d(st, &tm_w, &full_[s], ks * 128, t.f0, t.g);
          for (int b = 0; b < boxes; ++b)
            tma_load_2d(st + kWBytes + b * kBoxN * 128, &tm_x, &full_[s], ks * 128, t.row0 + b * kBoxN);
          last_round[s] = round;
          if (++s == kStages) {
            s = 0;
            ++round;
          }
        }
      }
      if (!ok)  // copies in flight land before the CTA ends
        for (int i = 0; i < kStages; ++i)
          if (last_round[i] >= 0) mbar_wait(&full_[i], last_round[i] & 1, p.err, kMx4ErrWait);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA
    if (lane == 0) {
      int s = 0, phase = 0, j = 0;
      bool ok = true;
      const uint32_t sfw = tmem + kSfwCol, sfx = tmem + kSfxCol;
      for (long long item = blockIdx.x; ok && item < total; item += gridDim.x, ++j) {
        const Tile t = tile_at(item);
        const int buf = j & 1, rr = j >> 1;
        if (rr > 0 && !(ok = mbar_wait(&acc_empty[buf], (rr - 1) & 1, p.err, kMx4ErrWait))) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(buf * kTileN);
        const uint32_t id0 = idesc_mxf4(kTileW, t.cols, 0), id2 = idesc_mxf4(kTileW, t.cols, 2);
        for (int ks = 0; ks < p.k_steps; ++ks) {
          if (!(ok = mbar_wait(&full_[s], phase, p.err, kMx4ErrWait) && mbar_wait(&scaled_[s], phase, p.err, kMx4ErrWait))) break;
          tc_fence_after();
          const uint32_t st = smem_addr(stages + s * kStageBytes), sf = st + kWBytes + kXBytes;
          const int mmas = min(4, (p.k - ks * kStageK + 63) / 64);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            utccp_atom(sfw + 4 * w, sf + w * kAtomBytes);
            utccp_atom(sfx + 8 * w, sf + kSfw + 2 * w * kAtomBytes);
            if (t.cols > 128) utccp_atom(sfx + 8 * w + 4, sf + kSfw + (2 * w + 1) * kAtomBytes);
          }
          const uint64_t wd = desc_sw128_kmajor(st), xd = desc_sw128_kmajor(st + kWBytes);
          for (int kk = 0; kk < mmas; ++kk) {
            const uint32_t half = (uint32_t)(kk & 1) << 31;  // scale columns 2 and 3 of the word
            umma_mxf4(d, wd + 2 * kk, xd + 2 * kk, kk & 1 ? id2 : id0, (sfw + 4 * (kk >> 1)) | half,
                      (sfx + 8 * (kk >> 1)) | half, (ks | kk) != 0);
          }
          umma_commit(&empty_[s]);
          if (++s == kStages) {
            s = 0;
            phase ^= 1;
          }
        }
        if (ok) umma_commit(&acc_full[buf]);
      }
      umma_commit(&mma_done);  // no MMA is left when the tensor memory goes
      mbar_wait(&mma_done, 0, p.err, kMx4ErrWait);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ scales
    // kAhead stages' copies are in flight; a stage is handed over when its own have landed
    constexpr int kAhead = kStages - 2;  // so one stage is handed over while the oldest is still being read
    long long issued = 0;
    int s = 0, round = 0, done_s = 0;
    bool ok = true;
    auto hand_over = [&] {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&scaled_[done_s]);
      if (++done_s == kStages) done_s = 0;
    };
    for (long long item = blockIdx.x; ok && item < total; item += gridDim.x) {
      const Tile t = tile_at(item);
      const uint32_t *wsf = p.b_scales + (size_t)t.g * p.words * p.n;
      for (int ks = 0; ks < p.k_steps; ++ks) {
        if (round > 0 && !(ok = mbar_wait(&empty_[s], (round - 1) & 1, p.err, kMx4ErrWait))) break;
        const uint32_t sf = smem_addr(stages + s * kStageBytes + kWBytes + kXBytes) + 16 * lane;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int kw = 2 * ks + w;
          const bool in_k = kw < p.words;
          const uint32_t *ws = wsf + (size_t)(in_k ? kw : 0) * p.n, *xs = p.a_scales + (size_t)(in_k ? kw : 0) * p.m;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int f = t.f0 + 32 * q + lane;
            const bool in = in_k && f < p.n;
            cp_async_4_zfill(sf + w * kAtomBytes + 4 * q, ws + (in ? f : 0), in);
          }
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            if (32 * q >= t.cols) break;
            const int r = t.row0 + 32 * q + lane;
            const bool in = in_k && r < p.m;
            cp_async_4_zfill(sf + kSfw + (2 * w + (q >> 2)) * kAtomBytes + 4 * (q & 3), xs + (in ? r : 0), in);
          }
        }
        cp_async_commit();
        if (++s == kStages) {
          s = 0;
          ++round;
        }
        if (++issued > kAhead) {
          cp_async_wait<kAhead>();
          hand_over();
        }
      }
    }
    cp_async_wait<0>();
    for (long long i = issued > kAhead ? issued - kAhead : 0; i < issued; ++i) hand_over();
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;  // TMEM lane quarter
    int j = 0;
    for (long long item = blockIdx.x; item < total; item += gridDim.x, ++j) {
      const Tile t = tile_at(item);
      const int buf = j & 1;
      if (!mbar_wait(&acc_full[buf], (j >> 1) & 1, p.err, kMx4ErrWait)) break;
      tc_fence_after();
      const int f = t.f0 + q * 32 + lane;
      const bool in = f < p.n;
      const float bias = p.bias && in ? bf16_to_f32(__ldg(p.bias + (size_t)t.g * p.n + f)) : 0.f;
      const uint32_t base = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * kTileN);
      for (int c0 = 0; c0 < t.rows; c0 += 32) {
        uint32_t v[32];
        tmem_ld_32_async(base + (uint32_t)c0, v);
        tmem_wait_ld(v);
        if (!p.out_bf16) {
          float *o = static_cast<float *>(p.out) + (size_t)(t.row0 + c0) * p.ldo + f;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (in && c0 + i < t.rows) o[(size_t)i * p.ldo] = __uint_as_float(v[i]) + bias;
        } else {
          // lanes 2i and 2i + 1 trade halves: the even one stores both features of an even column, the odd
          // one of an odd column, 4 bytes each
          const int odd = lane & 1, fe = f - odd;
          uint16_t *o = static_cast<uint16_t *>(p.out) + (size_t)(t.row0 + c0 + odd) * p.ldo + fe;
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float v0 = __uint_as_float(v[i]) + bias, v1 = __uint_as_float(v[i + 1]) + bias;
            const float other = __shfl_xor_sync(0xFFFFFFFFu, odd ? v0 : v1, 1);
            const float lo = odd ? other : v0, hi = odd ? v1 : other;
            uint32_t both;
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(both) : "f"(hi), "f"(lo));
            if (c0 + i + odd >= t.rows) continue;
            uint16_t *dst = o + (size_t)i * p.ldo;
            if (fe + 1 < p.n && p.pair_stores) {
              *reinterpret_cast<uint32_t *>(dst) = both;
            } else {
              if (fe < p.n) dst[0] = (uint16_t)both;
              if (fe + 1 < p.n) dst[1] = (uint16_t)(both >> 16);
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[buf]);
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, kTmemCols);
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

}  // namespace

cudaError_t launch_mx4_gemm(const Mx4GemmArgs &a, int n_sms, cudaStream_t stream) {
  if (a.m == 0 || a.n == 0) return cudaSuccess;
  CUtensorMap tm_x, tm_w;
  cudaError_t st;
  if ((st = code_map(&tm_x, a.a, 2, a.k, a.m, 1, kBoxN))) return st;
  if ((st = code_map(&tm_w, a.b, 3, a.k, a.n, a.groups, kTileW))) return st;
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
  p.n_tiles = (a.n + kTileW - 1) / kTileW;
  p.k_steps = (a.k + kStageK - 1) / kStageK;
  p.words = (a.k + 127) / 128;
  p.out_bf16 = a.out_bf16;
  p.pair_stores = a.ldo % 2 == 0 && (uintptr_t)a.out % 4 == 0;
  p.err = a.err;
  // no more activation tiles than this, whatever the counts are
  const long long x_tiles = a.counts ? (long long)a.m / kTileN + std::min(a.groups, a.m) : ((long long)a.m + kTileN - 1) / kTileN;
  const unsigned grid = (unsigned)std::min<long long>(n_sms, x_tiles * p.n_tiles);
  constexpr int smem = kStages * kStageBytes + 1024;
  if ((st = cudaFuncSetAttribute(mx4_gemm_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem))) return st;
  mx4_gemm_kernel<<<grid, kThreads, smem, stream>>>(tm_x, tm_w, p);
  return cudaGetLastError();
}

}  // namespace oxg
