// Softmax cross entropy over the tied vocabulary matrix, and its gradient, without ever keeping the logits.
//
//   z = h W^T   (n x vocab, fp32 accumulators in tensor memory)
//   lse_i = log sum_v exp z_iv        loss_i = lse_i - z_i,t(i)        (0 where the target is ignored)
//   dz_iv = g_i (exp(z_iv - lse_i) - [v = t(i)])        dh = dz W        dW = dz^T h
//
// All products but those of at most 64 rows (loss_few_kernel) run in one persistent tcgen05 kernel on CTA pairs
// (cta_group::2, 256 x 256 tiles: each CTA stages 128 rows of A and 128 rows of B per 64-deep k block, so a tile needs a
// third less L2 traffic than two 128 x 256 tiles), fed by TMA through a ring of 5 or 6 stages, with the accumulators of
// two tiles in tensor memory so that the epilogue of one runs under the MMAs of the next.
// Measured (vocabulary 51866, hidden 1280, bf16), as the clocks allow: forward of 16381 rows 1340 to 1625 us, 1.3 to 1.6
// PFLOP/s, the tensor pipe 95% active; gradient of 8189 rows 2575 to 2740 us, 1.2 PFLOP/s by the formulas, which do not count
// the logits that are formed again; of 211 rows (fp16) 125 to 139 us, of which dW's 133 MB of stores and dh's 133 MB of loads
// take 40 at the memory's rate and overlap little.
//   * forward: the epilogue reduces each 128-column half tile to (max, sum of exponentials) per row, the target
//     left out; loss_combine_kernel joins the halves of all vocabulary tiles and the target's logit. Reads h and W, writes 8 bytes per
//     row and half tile.
//   * gradient: the vocabulary is taken in pieces whose dz (16 bits) fits the scratch and mostly L2. Per piece one
//     launch recomputes z and writes dz, a second one has both products of it: dh (contraction over the piece; fp32
//     partial sums per k split, carried from piece to piece) and dW (contraction over the rows, final).
// The target's logit is not taken from the tensor core, whose truncating sums are short by 1e-6 of it and more: where the target
// has nearly all of the probability, that is more than the loss, and than exp(z - lse) - 1. It is a dot product of its own
// (exact_logit), its column left out of the statistics: then the loss is log1p(others / target) and dz_t = expm1(z_t - lse), and
// what the others' sums lack is a small part of either. (Five rows over 226 tokens, all of them sure: the gradient was off by a tenth.) Two warps have it beside the products in the forward pass, CTAs beside h's copy in the gradient.
// 16-bit dz: exp(z - lse) - [v = t] lies in [-1, 1] whatever g is, so it is stored without g (times 2^12 in fp16,
// which keeps probabilities down to 2^-36 above the smallest subnormal); g multiplies dh's rows in fp32 at the end, and
// is folded into the 16-bit copy of h that dW's product reads, relative to the largest |g|, so that with equal
// weights nothing is rounded a second time. fp16: the copy is taken up to 2^15 by a power of two, so that rows of small
// weight keep their bits as far as 2^-29 of the largest |h g|.
#include "fw_host.h"
#include "fw_tc.cuh"

namespace fw {

FW_DEFINE_ERROR_WORD();

__device__ __forceinline__ void loss_flag(unsigned bits) { atomicOr(&g_fw_dev_error, bits); }

constexpr int kBM = 256, kBN = 256, kBK = 64;  // tile of a CTA pair
constexpr uint32_t kHalfBytes = 128 * kBK * 2;  // a CTA's share of A (or B) per stage: 16 KB
constexpr uint32_t kStageBytes = 2 * kHalfBytes;
constexpr uint32_t kOutBytes = 32 * 128;  // an epilogue warp's 32 rows of 128 bytes on their way to global memory
constexpr int kMGroup = 32;  // row tiles that run against a vocabulary tile before the next one: h stays in L2
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

enum Kind { kStats, kDz, kGrads };  // what a launch computes
constexpr int stages_of(int kind) { return kind == kGrads ? 5 : 6; }
// Epilogue warps: twice as many where the products are short (dW of few rows) and the epilogue has little to compute.
constexpr int epi_warps(int kind) { return kind == kGrads ? 16 : 8; }
constexpr int target_warps(int kind) { return kind == kStats ? 2 : 0; }
constexpr int threads_of(int kind) { return 32 * (2 + epi_warps(kind) + target_warps(kind)); }
constexpr int smem_of(int kind) {
  return stages_of(kind) * kStageBytes + (kind == kStats ? 0 : epi_warps(kind) * kOutBytes) + 1024;
}
// The tensor core's fp32 additions truncate: the 80 of a contraction of 1280 leave logits 1.3e-6 (bf16) or 2.4e-6 (fp16)
// of their size short. The gradient, whose logits (but the targets') are rounded to 16 bits as probabilities next, leaves it at that. For
// the loss, an fp32 result, it adds up at most 10 or 7 k blocks at a time, and the epilogue adds
// those segments rounding to nearest: below 8e-7 for any contraction. The tensor core is at the next segment meanwhile;
// shorter ones leave it idle during a tile's exponentials (16381 rows: none 1265 us, 10 1355, 7 1466, 4 1850).
template <typename T>
__host__ __device__ constexpr int segment_of(int kbs) {
  constexpr int most = Type16<T>::kBf16 ? 10 : 7;
  return (kbs + (kbs + most - 1) / most - 1) / ((kbs + most - 1) / most);
}

struct LossArgs {
  int n, hidden, width;      // rows, hidden size, columns of this launch's vocabulary piece
  int v0, vocab;             // first vocabulary row of the piece; all rows
  int m_tiles, n_tiles;      // kStats, kDz: over (rows, piece); kGrads: dW over (piece, hidden)
  int dh_m_tiles, splits;    // kGrads: dh over (rows, hidden), each tile's contraction in `splits` parts
  int64_t ignore;
  const int64_t* targets;
  const float* lse;
  float2* stats;             // [2 * all n tiles][n]
  float *target_logit, *target_rest;  // [n], kStats
  const void *h, *w;         // kStats
  const float* target_dz;    // [n], kDz: what dz is at the target
  void* dz;                  // [n][ld_dz]
  int64_t ld_dz;
  float dz_scale;            // the factor stored with dz
  float* part;               // [splits][n][hidden]
  void* dw;                  // [vocab][hidden]
  const float* unscale;      // what loss_scale_kernel's copy of h has to be multiplied with
  int first_piece, accumulate;
  bool chunks;               // MN-major maps over [hidden / 64][rows][64]; hidden is a multiple of 64
};

// A row that counts: its target is a vocabulary row and not the one to be ignored.
__device__ __forceinline__ bool counts(int64_t target, int64_t ignore, int vocab) {
  return target >= 0 && target < vocab && target != ignore;
}

// x + y as a number and what its rounding lost (Knuth's two-sum), the latter added to what was lost before.
__device__ __forceinline__ float2 add_exact(float2 x, float2 y) {
  const float t = x.x + y.x, back = t - x.x;
  return make_float2(t, ((x.x - (t - back)) + (y.x - back)) + (x.y + y.y));
}

// h . w by one warp, as a number and a rest: 256 sums of a few terms each in fp32, which round to nearest (1280 terms: five
// each, off by 5 x 2^-24 of their size at most, and by a sixteenth of 2^-23 of the whole together as a rule), added up with
// the rests. (Beside the products of 16381 rows: 1560 us, without it 1548; the 256 added up in 64 bits 1575, all sums in 64
// bits 1590.)
template <typename T>
__device__ __forceinline__ float2 exact_logit(const T* h, const T* w, int hidden, int lane) {
  float acc[8] = {};
#pragma unroll 4
  for (int i = lane; i < hidden / 8; i += 32) {
    const uint4 x = reinterpret_cast<const uint4*>(h)[i], y = reinterpret_cast<const uint4*>(w)[i];
    const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = Type16<T>::unpack(xw[j]), b = Type16<T>::unpack(yw[j]);
      acc[2 * j] = fmaf(a.x, b.x, acc[2 * j]);
      acc[2 * j + 1] = fmaf(a.y, b.y, acc[2 * j + 1]);
    }
  }
  float2 sum = make_float2(acc[0], 0.f);
#pragma unroll
  for (int j = 1; j < 8; ++j) sum = add_exact(sum, make_float2(acc[j], 0.f));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    sum = add_exact(sum, make_float2(__shfl_xor_sync(0xffffffffu, sum.x, o), __shfl_xor_sync(0xffffffffu, sum.y, o)));
  if (!(fabsf(sum.x) < INFINITY)) sum.y = 0.f;  // infinities leave a NaN there
  return sum;
}
// Rows first, first + step, ...: the logits of their targets.
template <typename T>
__device__ __forceinline__ void target_logits(const LossArgs& a, int first, int step, int lane) {
  for (int row = first; row < a.n; row += step) {
    const int64_t t = a.targets[row];
    if (!counts(t, a.ignore, a.vocab)) continue;
    const float2 z = exact_logit(static_cast<const T*>(a.h) + static_cast<int64_t>(row) * a.hidden,
                                 static_cast<const T*>(a.w) + t * a.hidden, a.hidden, lane);
    if (lane == 0) {
      a.target_logit[row] = z.x;
      a.target_rest[row] = z.y;
    }
  }
}

struct Tile {
  int m0, n0, kb0, kbs;
  int split;
  bool dh;  // kGrads
};

template <int kKind>
__device__ __forceinline__ int tile_count(const LossArgs& a) {
  return kKind == kGrads ? a.dh_m_tiles * a.splits * a.n_tiles + a.m_tiles * a.n_tiles : a.m_tiles * a.n_tiles;
}

template <int kKind>
__device__ __forceinline__ Tile tile_at(const LossArgs& a, int t) {
  Tile x;
  if (kKind != kGrads) {
    // groups of kMGroup row tiles; within a group the row tiles run against one vocabulary tile after the other
    const int per = kMGroup * a.n_tiles, grp = t / per, in = t - grp * per;
    const int rows = min(kMGroup, a.m_tiles - grp * kMGroup);
    x.m0 = (grp * kMGroup + in % rows) * kBM;
    x.n0 = in / rows * kBN;
    x.kb0 = 0;
    x.kbs = (a.hidden + kBK - 1) / kBK;
    x.split = 0;
    x.dh = false;
    return x;
  }
  const int dh_tiles = a.dh_m_tiles * a.splits * a.n_tiles;
  x.dh = t < dh_tiles;
  if (x.dh) {
    const int kb = (a.width + kBK - 1) / kBK;
    x.n0 = t % a.n_tiles * kBN;
    const int u = t / a.n_tiles;
    x.split = u % a.splits;
    x.m0 = u / a.splits * kBM;
    x.kb0 = static_cast<int>(static_cast<int64_t>(kb) * x.split / a.splits);
    x.kbs = static_cast<int>(static_cast<int64_t>(kb) * (x.split + 1) / a.splits) - x.kb0;
  } else {
    t -= dh_tiles;
    x.n0 = t % a.n_tiles * kBN;
    x.m0 = t / a.n_tiles * kBM;
    x.kb0 = 0;
    x.kbs = (a.n + kBK - 1) / kBK;
    x.split = 0;
  }
  return x;
}

// A CTA's 128 rows of an operand for one k block. K-major: one box of 64 k x 128 rows. MN-major: boxes of 64 rows
// (contiguous) x 64 k, both as one copy where the map has chunks of 64 for its third dimension (gradient of 8189 rows,
// a copy a box: 2780 us, 2684).
template <bool kMn>
__device__ __forceinline__ void load_half(uint8_t* dst, const CUtensorMap* map, uint32_t rbar, int row, int k,
                                          bool chunks) {
  if (kMn && chunks) {
    tma_load_3d_pair(dst, map, rbar, 0, k, row >> 6);
  } else if (kMn) {
    tma_load_2d_pair(dst, map, rbar, row, k);
    tma_load_2d_pair(dst + kHalfBytes / 2, map, rbar, row + 64, k);
  } else {
    tma_load_2d_pair(dst, map, rbar, k, row);
  }
}

template <bool kMn>
__device__ __forceinline__ uint64_t half_desc(uint32_t addr) {
  return kMn ? sw128_mn_desc(addr, kHalfBytes / 2) : sw128_desc(addr);
}

template <typename T, bool kAMn, bool kBMn>
__device__ __forceinline__ void mma_block(uint32_t d, uint32_t a_addr, bool fresh) {
  constexpr uint32_t idesc = make_idesc(kBM, kBN, Type16<T>::kBf16, kAMn, kBMn);
  const uint64_t ad = half_desc<kAMn>(a_addr), bd = half_desc<kBMn>(a_addr + kHalfBytes);
#pragma unroll
  for (int kk = 0; kk < kBK / 16; ++kk)
    tc_mma_pair(d, ad + kk * (kAMn ? 128 : 2), bd + kk * (kBMn ? 128 : 2), idesc, fresh && kk == 0 ? 0u : 1u);
}

// tmA, tmB: the operands of kStats, kDz and of kGrads' dh; tmA2, tmB2: of kGrads' dW. tmOut: dz or dW, tmPart: dh's sums.
template <int kKind, typename T>
__global__ void __launch_bounds__(threads_of(kKind), 1) __cluster_dims__(2, 1, 1)
    loss_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmA2, const __grid_constant__ CUtensorMap tmB2,
                     const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ CUtensorMap tmPart, LossArgs a) {
  constexpr int kStages = stages_of(kKind);
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_base_sh;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pairs = gridDim.x >> 1, first = blockIdx.x >> 1;
  const int tiles = tile_count<kKind>(a);

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);   // leader's: both CTAs' bytes, one arrival
      mbar_init(&empty_bar[s], 1);  // each CTA's: the pair's MMAs have read the stage
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * epi_warps(kKind));  // leader's: both CTAs' epilogue warps have drained the buffer
    }
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    if (kKind == kGrads) {
      tma_prefetch_desc(&tmA2);
      tma_prefetch_desc(&tmB2);
    }
  }
  if (warp == 1) tmem_alloc_pair(&tmem_base_sh, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += pairs) {
        const Tile x = tile_at<kKind>(a, t);
        for (int kb = 0; kb < x.kbs; ++kb, ++it) {
          const int s = it % kStages;
          if (it >= kStages && !mbar_wait(&empty_bar[s], ((it / kStages) & 1u) ^ 1u)) {
            loss_flag(FW_DEVERR_TIMEOUT);
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], 2 * kStageBytes);
          const uint32_t rbar = cluster_map(&full_bar[s], 0);
          uint8_t* dst = smem + s * kStageBytes;
          const int row_a = x.m0 + 128 * static_cast<int>(rank), row_b = x.n0 + 128 * static_cast<int>(rank);
          const int k = (x.kb0 + kb) * kBK;
          if (kKind != kGrads) {
            load_half<false>(dst, &tmA, rbar, row_a, k, false);
            load_half<false>(dst + kHalfBytes, &tmB, rbar, row_b, k, false);
          } else if (x.dh) {
            load_half<false>(dst, &tmA, rbar, row_a, k, false);
            load_half<true>(dst + kHalfBytes, &tmB, rbar, row_b, k, a.chunks);
          } else {
            load_half<true>(dst, &tmA2, rbar, row_a, k, true);
            load_half<true>(dst + kHalfBytes, &tmB2, rbar, row_b, k, a.chunks);
          }
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {  // the whole warp runs the loop, one lane issues
      int it = 0, local = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += pairs) {
        const Tile x = tile_at<kKind>(a, t);
        const int segment = kKind == kStats ? segment_of<T>(x.kbs) : x.kbs;
        for (int kb0 = 0; kb0 < x.kbs && ok; kb0 += segment, ++local) {
          const int buf = local & 1;
          if (local >= 2) ok = mbar_wait_warp(&acc_empty[buf], ((local >> 1) & 1u) ^ 1u);
          tc_fence_after();
          const uint32_t d = tmem + buf * kBN;
          const int kb1 = min(x.kbs, kb0 + segment);
          for (int kb = kb0; kb < kb1 && ok; ++kb, ++it) {
            const int s = it % kStages;
            ok = mbar_wait_warp(&full_bar[s], (it / kStages) & 1u);
            if (!ok) break;
            tc_fence_after();
            const uint32_t at = base + s * kStageBytes;
            if (elect_one()) {
              if (kKind != kGrads)
                mma_block<T, false, false>(d, at, kb == kb0);
              else if (x.dh)
                mma_block<T, false, true>(d, at, kb == kb0);
              else
                mma_block<T, true, true>(d, at, kb == kb0);
              tc_commit_pair(&empty_bar[s]);
            }
            __syncwarp();
          }
          if (elect_one()) tc_commit_pair(&acc_full[buf]);
          __syncwarp();
        }
      }
      if (!ok && lane == 0) loss_flag(FW_DEVERR_TIMEOUT);
    }
  } else if (warp >= 2 + epi_warps(kKind)) {  // kStats, beside the products
    target_logits<T>(a, blockIdx.x * target_warps(kKind) + warp - 2 - epi_warps(kKind), gridDim.x * target_warps(kKind), lane);
  } else {
    // Warp w reads tensor-memory lanes 32 (w % 4) .. + 31 (one row of the tile per thread) and columns
    // kCols ((w - 2) / 4) .. + kCols - 1. dz, dW and dh's sums go through 4 KB of shared memory a warp (rows of 128
    // bytes, 128-byte swizzle) to tensor stores: 16 bytes a thread straight to rows 2560 bytes apart took three times
    // as long.
    const int q = warp & 3, part = (warp - 2) >> 2;
    const uint32_t drained = cluster_map(&acc_empty[0], 0);
    constexpr int kCols = 2 * 4 * 128 / epi_warps(kKind);  // columns of a warp
    uint8_t* out = smem + kStages * kStageBytes + (warp - 2) * kOutBytes;
    bool failed = false;
    int local = 0;
    for (int t = first; t < tiles && !failed; t += pairs) {
      const Tile x = tile_at<kKind>(a, t);
      const int row0 = x.m0 + 128 * static_cast<int>(rank) + q * 32;  // the warp's first row
      const int row = row0 + lane;
      const int c0 = x.n0 + kCols * part;
      int64_t target = -1;  // relative to this launch's vocabulary piece
      float neg_lse = 0.f, target_dz = 0.f;
      bool kept = false;
      if (kKind != kGrads && row < a.n) {
        const int64_t tg = a.targets[row];
        kept = counts(tg, a.ignore, a.vocab);
        if (kept) target = tg - a.v0;
        if (kKind == kDz) neg_lse = -a.lse[row] * kLog2e;
        if (kKind == kDz && kept) target_dz = a.target_dz[row];
      }
      if (kKind == kStats) {
        float z[128];
        const int segment = segment_of<T>(x.kbs);
        for (int kb0 = 0; kb0 < x.kbs; kb0 += segment, ++local) {
          const int buf = local & 1;
          if (!mbar_wait_warp(&acc_full[buf], (local >> 1) & 1u)) {
            failed = true;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem + (static_cast<uint32_t>(q * 32) << 16) + buf * kBN + 128 * part;
          if (row0 < a.n) {  // else none of this warp's rows is one
#pragma unroll
            for (int c = 0; c < 128; c += 16) {
              uint32_t r[16];
              tc_ld16(d + c, r);
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) z[c + j] = kb0 == 0 ? __uint_as_float(r[j]) : z[c + j] + __uint_as_float(r[j]);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(drained + 8 * buf);
        }
        if (failed) break;
        if (row0 >= a.n) continue;
        if (c0 + 128 > a.width) {  // columns behind the vocabulary count as -inf
#pragma unroll
          for (int j = 0; j < 128; ++j)
            if (c0 + j >= a.width) z[j] = -INFINITY;
        }
        if (target >= c0 && target < c0 + 128) {  // joined by loss_combine_kernel
          const int at = static_cast<int>(target) - c0;
#pragma unroll
          for (int j = 0; j < 128; ++j)
            if (j == at) z[j] = -INFINITY;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 128; j += 2) mx[(j >> 1) & 3] = fmaxf(fmaxf(mx[(j >> 1) & 3], z[j]), z[j + 1]);
        // the maximum in powers of two, rounded once: the sum is relative to exactly this number
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * kLog2e;
        const float off = top == -INFINITY ? 0.f : -top;
        float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int j = 0; j < 128; j += 2) {
          const float2 e = fma2(make_float2(z[j], z[j + 1]), make_float2(kLog2e, kLog2e), make_float2(off, off));
          acc[(j >> 1) & 1] = add2(acc[(j >> 1) & 1], make_float2(ex2(e.x), ex2(e.y)));
        }
        acc[0] = add2(acc[0], acc[1]);
        if (row < a.n)
          a.stats[static_cast<int64_t>(2 * (x.n0 / kBN) + part) * a.n + row] = make_float2(top, acc[0].x + acc[0].y);
        __syncwarp();
        continue;
      }
      const int buf = local & 1;
      if (!mbar_wait_warp(&acc_full[buf], (local >> 1) & 1u)) {
        failed = true;
        break;
      }
      ++local;
      tc_fence_after();
      const uint32_t d = tmem + (static_cast<uint32_t>(q * 32) << 16) + buf * kBN + kCols * part;
      const bool wide = kKind == kGrads && x.dh;  // fp32 rows of 32 columns, else 16-bit rows of 64
      const bool direct = kKind == kGrads && !x.dh && a.accumulate;
      const float f = kKind == kGrads && !x.dh ? *a.unscale / a.dz_scale : 1.f;
      const int rows = kKind == kDz || wide ? a.n : a.width;
#pragma unroll 1
      for (int c = 0; c < (row0 < rows ? kCols : 0); c += 32) {
        uint32_t r[32];
        tc_load32(d + c, r);
        tc_wait_ld();
        const int col = c0 + c;
        if (kKind == kDz) {
          const int at = target >= col && target < col + 32 ? static_cast<int>(target) - col : -1;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float p = j == at ? target_dz : ex2(fmaf(__uint_as_float(r[j]), kLog2e, neg_lse));
            r[j] = __float_as_uint(kept ? p * a.dz_scale : 0.f);
          }
        } else if (!wide) {
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * f);
        }
        // dW added to what is there, 16 bytes a thread: 211 rows (fp16) 262 us against 125 that write, 8189 rows 2710 to 2820
        // against 2620 to 2760.
        if (direct) {
          if (row < a.width) {
            uint4* dst =
                reinterpret_cast<uint4*>(static_cast<T*>(a.dw) + (static_cast<int64_t>(a.v0) + row) * a.hidden + col);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (col + 8 * j >= a.hidden) break;
              const uint4 o = dst[j];
              const uint32_t ow[4] = {o.x, o.y, o.z, o.w};
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 u = Type16<T>::unpack(ow[i]);
                w[i] = Type16<T>::pack(__uint_as_float(r[8 * j + 2 * i]) + u.x, __uint_as_float(r[8 * j + 2 * i + 1]) + u.y);
              }
              dst[j] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          __syncwarp();
          continue;
        }
        const bool first_half = wide || c % 64 == 0;
        if (first_half) {  // the last store has read the buffer
          if (lane == 0) tma_store_wait_read();
          __syncwarp();
        }
        uint8_t* mine = out + lane * 128;
        if (wide) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(mine + ((j ^ (lane & 7)) << 4)) =
                make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int chunk = (c % 64) / 8 + j;
            *reinterpret_cast<uint4*>(mine + ((chunk ^ (lane & 7)) << 4)) =
                make_uint4(Type16<T>::pack(__uint_as_float(r[8 * j]), __uint_as_float(r[8 * j + 1])),
                           Type16<T>::pack(__uint_as_float(r[8 * j + 2]), __uint_as_float(r[8 * j + 3])),
                           Type16<T>::pack(__uint_as_float(r[8 * j + 4]), __uint_as_float(r[8 * j + 5])),
                           Type16<T>::pack(__uint_as_float(r[8 * j + 6]), __uint_as_float(r[8 * j + 7])));
          }
        }
        if (wide || c % 64 == 32) {
          fence_proxy_async_shared();
          __syncwarp();
          // rows and columns behind the end of a partly covered box are not written
          const int at = wide ? col : col - 32;
          if (lane == 0 && at < (kKind == kDz ? a.width : a.hidden)) {
            if (!wide)
              tma_store_2d(&tmOut, out, at, row0);
            else if (a.first_piece)
              tma_store_3d(&tmPart, out, at, row0, x.split);
            else
              tma_add_3d(&tmPart, out, at, row0, x.split);
            tma_store_commit();
          }
        }
        __syncwarp();  // the next load is a warp-wide instruction
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(drained + 8 * buf);
    }
    if (kKind != kStats && lane == 0) tma_store_wait();
    if (failed && lane == 0) loss_flag(FW_DEVERR_TIMEOUT);
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no CTA leaves while its peer's barriers or tensor memory are in use
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// Forward of at most 64 rows (one transcript, the drafts of a few tokens): bound by reading W once, where a tile of 256 rows
// would keep the tensor core busy for as long with rows that do not exist. The operands change places: 128 rows of W are
// the M of a product, the kN >= n rows of h its N. One CTA an SM takes an equal, contiguous share of the vocabulary in
// equal tiles of `box` <= 128 rows, each k block of which is one copy. 27 rows of 1280, vocabulary of 51866: 31 us with the
// join, W at 4.9 TB/s (copies of 32 rows 37; in tiles of 256 rows 42; 64 rows 35, and 35 to 37 there). A thread owns a
// vocabulary row of each tile: it keeps maximum and sum of every row of h over its tiles by itself, and the CTA joins its
// 128 threads once, at the end.
constexpr int kFewRows = 64, kFewStages = 6, kFewThreads = 32 * 7;
constexpr uint32_t few_stage(int rows) { return kHalfBytes + rows * 128; }
constexpr int few_smem(int rows) { return kFewStages * few_stage(rows) + 1024; }

template <typename T, int kN>
__global__ void __launch_bounds__(kFewThreads, 1)
    loss_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmH, LossArgs a, int share,
                    int box) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kFewStages], empty_bar[kFewStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int s_target[kN];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  constexpr uint32_t kColumns = 2 * kN;
  if (warp == 0 && lane == 0) {
    for (int s = 0; s < kFewStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4);
    }
    mbar_fence_init();
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmH);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_base_sh, kColumns);
    tmem_relinquish();
  }
  for (int i = threadIdx.x; i < kN; i += kFewThreads) {
    const int64_t t = i < a.n ? a.targets[i] : -1;
    s_target[i] = counts(t, a.ignore, a.vocab) ? static_cast<int>(t) : -1;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem = tmem_base_sh;
  const int v0 = blockIdx.x * share, v1 = min(a.vocab, v0 + share);
  const int kbs = (a.hidden + kBK - 1) / kBK, segment = segment_of<T>(kbs);

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int v = v0; v < v1 && ok; v += box) {
        for (int kb = 0; kb < kbs; ++kb, ++it) {
          const int s = it % kFewStages;
          if (it >= kFewStages && !mbar_wait(&empty_bar[s], ((it / kFewStages) & 1u) ^ 1u)) {
            loss_flag(FW_DEVERR_TIMEOUT);
            ok = false;
            break;
          }
          uint8_t* dst = smem + s * few_stage(kN);
          mbar_arrive_expect_tx(&full_bar[s], (box + kN) * 128);  // of the tile's 128 rows the others are not used
          tma_load_2d(dst, &tmW, &full_bar[s], kb * kBK, v);
          tma_load_2d(dst + kHalfBytes, &tmH, &full_bar[s], kb * kBK, 0);
        }
      }
    }
  } else if (warp == 1) {  // the whole warp runs the loop, one lane issues
    constexpr uint32_t idesc = make_idesc(128, kN, Type16<T>::kBf16, false, false);
    int it = 0, local = 0;
    bool ok = true;
    for (int v = v0; v < v1 && ok; v += box) {
      for (int kb0 = 0; kb0 < kbs && ok; kb0 += segment, ++local) {
        const int buf = local & 1;
        if (local >= 2) ok = mbar_wait_warp(&acc_empty[buf], ((local >> 1) & 1u) ^ 1u);
        tc_fence_after();
        for (int kb = kb0; kb < min(kbs, kb0 + segment) && ok; ++kb, ++it) {
          const int s = it % kFewStages;
          ok = mbar_wait_warp(&full_bar[s], (it / kFewStages) & 1u);
          if (!ok) break;
          tc_fence_after();
          const uint64_t ad = sw128_desc(base + s * few_stage(kN)), bd = sw128_desc(base + s * few_stage(kN) + kHalfBytes);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kBK / 16; ++kk)
              tc_mma_f16(tmem + buf * kN, ad + 2 * kk, bd + 2 * kk, idesc, kb != kb0 || kk != 0 ? 1u : 0u);
            tc_commit(&empty_bar[s]);
          }
          __syncwarp();
        }
        if (elect_one()) tc_commit(&acc_full[buf]);
        __syncwarp();
      }
    }
    if (!ok && lane == 0) loss_flag(FW_DEVERR_TIMEOUT);
  } else if (warp == 6) {
    target_logits<T>(a, blockIdx.x, gridDim.x, lane);
  } else {
    const int q = warp & 3, mine = q * 32 + lane;  // this thread's vocabulary row of a tile
    float top[kN], sum[kN];
#pragma unroll
    for (int c = 0; c < kN; ++c) top[c] = -INFINITY, sum[c] = 0.f;
    int local = 0;
    bool ok = true;
    for (int v = v0; v < v1 && ok; v += box) {
      float z[kN];
      for (int kb0 = 0; kb0 < kbs; kb0 += segment, ++local) {
        const int buf = local & 1;
        ok = mbar_wait_warp(&acc_full[buf], (local >> 1) & 1u);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < kN; c += 16) {
          uint32_t r[16];
          tc_ld16(tmem + (static_cast<uint32_t>(q * 32) << 16) + buf * kN + c, r);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) z[c + j] = kb0 == 0 ? __uint_as_float(r[j]) : z[c + j] + __uint_as_float(r[j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[buf]);
      }
      if (!ok) break;
      if (mine < box && v + mine < v1) {
#pragma unroll
        for (int c = 0; c < kN; ++c) {
          if (s_target[c] == v + mine) z[c] = -INFINITY;  // joined by loss_combine_kernel
          // maxima in powers of two, rounded once: the sum is relative to exactly this number
          const float m = fmaxf(top[c], z[c] * kLog2e), off = m == -INFINITY ? 0.f : -m;
          sum[c] = sum[c] * ex2(top[c] + off) + ex2(fmaf(z[c], kLog2e, off));
          top[c] = m;
        }
      }
      __syncwarp();
    }
    if (!ok && lane == 0) loss_flag(FW_DEVERR_TIMEOUT);
    // All products are done, so the stages are free: [kN][128] maxima, then sums.
    float* s_top = reinterpret_cast<float*>(smem);
    float* s_sum = s_top + kN * 128;
    if (ok) {
#pragma unroll
      for (int c = 0; c < kN; ++c) {
        s_top[c * 128 + mine] = top[c];
        s_sum[c * 128 + mine] = sum[c];
      }
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    for (int c = q; c < a.n && ok; c += 4) {
      float t[4], m = -INFINITY, l = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        t[i] = s_top[c * 128 + 32 * i + lane];
        m = fmaxf(m, t[i]);
      }
      m = warp_max(m);
      const float off = m == -INFINITY ? 0.f : -m;
#pragma unroll
      for (int i = 0; i < 4; ++i) l = fmaf(s_sum[c * 128 + 32 * i + lane], ex2(t[i] + off), l);
      l = warp_sum(l);
      if (lane == 0) a.stats[static_cast<int64_t>(blockIdx.x) * a.n + c] = make_float2(m, l);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, kColumns);
}

// Joins the (max, sum) of all half tiles (shares) of a row, both in powers of two, so that the differences of maxima are exact:
// 32 rows per CTA (lanes), the half tiles over its warps.
constexpr int kCombineThreads = 1024;
__global__ void __launch_bounds__(kCombineThreads) loss_combine_kernel(const float2* __restrict__ stats, int halves,
                                                                       int n, const int64_t* __restrict__ targets,
                                                                       int64_t ignore, int vocab, float* loss, float* lse) {
  constexpr int kWarps = kCombineThreads / 32;
  __shared__ float2 s_part[kWarps][32];
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x * 32 + lane;
  float top = -INFINITY, sum = 0.f;
  if (row < n) {
#pragma unroll 8
    for (int i = warp; i < halves; i += kWarps) {
      const float2 v = stats[static_cast<int64_t>(i) * n + row];
      const float m = fmaxf(top, v.x), off = m == -INFINITY ? 0.f : -m;
      sum = sum * ex2(top + off) + v.y * ex2(v.x + off);
      top = m;
    }
  }
  s_part[warp][lane] = make_float2(top, sum);
  __syncthreads();
  if (warp != 0 || row >= n) return;
  float m = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_part[w][lane].x);
  const float off = m == -INFINITY ? 0.f : -m;
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) s += s_part[w][lane].y * ex2(s_part[w][lane].x + off);
  const int64_t t = targets[row];
  if (t != ignore && (t < 0 || t >= vocab)) loss_flag(FW_DEVERR_BAD_INDEX);
  float l, nll = 0.f;
  if (!counts(t, ignore, vocab)) {
    l = m == -INFINITY ? logf(s) : fmaf(m, kLn2, logf(s));
  } else {
    const float z = loss[row], rest = lse[row];  // held the target's logit, which is not among the others
    const float gap = fmaf(-rest, kLog2e, fmaf(-z, kLog2e, m));  // how far the others' maximum is above it, in powers of two
    if (gap > 0.f) {
      l = fmaf(m, kLn2, logf(s + ex2(-gap)));
      nll = (l - z) - rest;
    } else {
      nll = log1pf(s * ex2(gap));
      l = z + (rest + nll);
    }
  }
  lse[row] = l;
  loss[row] = nll;
}

constexpr int kScaleThreads = 256, kRangeBlocks = 592;
__device__ __forceinline__ float block_max(float m, float* shared) {
  m = warp_max(m);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kScaleThreads / 32; ++w) m = fmaxf(m, shared[w]);
  return m;
}

// Gradient in fp16, before all else: each CTA's largest finite |g| and |h g| of the rows that count.
__global__ void __launch_bounds__(kScaleThreads) loss_range_kernel(const half* __restrict__ h, const float* __restrict__ g,
                                                                   const int64_t* __restrict__ targets, int64_t ignore,
                                                                   int vocab, int n, int hidden, float2* __restrict__ range) {
  __shared__ float s_max[2][kScaleThreads / 32];
  pdl_trigger();
  const int packs = hidden / 8;
  float big = 0.f, product = 0.f;
#pragma unroll 4
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kScaleThreads + threadIdx.x; i < static_cast<int64_t>(n) * packs;
       i += static_cast<int64_t>(gridDim.x) * kScaleThreads) {
    const int row = static_cast<int>(i / packs);
    const int64_t t = targets[row];
    const float w = fabsf(g[row]);
    const uint4 v = reinterpret_cast<const uint4*>(h)[i];
    if (!counts(t, ignore, vocab) || !(w < INFINITY)) continue;
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
    big = fmaxf(big, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 x = Type16<half>::unpack(u[j]);
      if (fabsf(x.x) < INFINITY) product = fmaxf(product, fabsf(x.x) * w);
      if (fabsf(x.y) < INFINITY) product = fmaxf(product, fabsf(x.y) * w);
    }
  }
  big = block_max(big, s_max[0]);
  product = block_max(product, s_max[1]);
  if (threadIdx.x == 0) range[blockIdx.x] = make_float2(big, product);
}

// Gradient, before the products: h scaled by g relative to the largest finite |g| of the rows that count, zero in rows that
// do not; further CTAs (from `blocks` on) have what dz is at the rows' targets. bf16: each CTA finds that |g| by itself from L2. fp16: loss_range_kernel has, and the power of two that takes the
// largest |h g| to [2^14, 2^15) besides (1 at least, 2^24 at most). *unscale takes both back.
template <typename T>
__global__ void __launch_bounds__(kScaleThreads) loss_scale_kernel(const T* __restrict__ h, const float* __restrict__ g,
                                                         const int64_t* __restrict__ targets, int64_t ignore,
                                                         int vocab, int n, int hidden, T* __restrict__ scaled,
                                                         float* __restrict__ unscale, const float2* __restrict__ range,
                                                         int ranges, int blocks, const T* __restrict__ w,
                                                         const float* __restrict__ lse, float* __restrict__ target_dz) {
  __shared__ float s_max[2][kScaleThreads / 32];
  pdl_trigger();
  if (static_cast<int>(blockIdx.x) >= blocks) {
    const int lane = threadIdx.x & 31;
    for (int row = (blockIdx.x - blocks) * (kScaleThreads / 32) + (threadIdx.x >> 5); row < n;
         row += (gridDim.x - blocks) * (kScaleThreads / 32)) {
      const int64_t t = targets[row];
      if (!counts(t, ignore, vocab)) continue;
      const float2 z = exact_logit(h + static_cast<int64_t>(row) * hidden, w + t * hidden, hidden, lane);
      if (lane == 0) target_dz[row] = expm1f((z.x - lse[row]) + z.y);
    }
    if (!Type16<T>::kBf16) pdl_wait();
    return;
  }
  float m = 0.f, up = 1.f;
  if (Type16<T>::kBf16 || blockIdx.x == 0) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const int64_t t = targets[i];
      const float v = fabsf(g[i]);
      const bool bad = t != ignore && (t < 0 || t >= vocab);
      if (bad && blockIdx.x == 0) loss_flag(FW_DEVERR_BAD_INDEX);
      if (t != ignore && !bad && v < INFINITY) m = fmaxf(m, v);  // NaN fails the comparison
    }
  }
  if (!Type16<T>::kBf16) {
    float product = 0.f;
    pdl_wait();
    for (int i = threadIdx.x; i < ranges; i += kScaleThreads) {
      m = fmaxf(m, range[i].x);
      product = fmaxf(product, range[i].y);
    }
    m = block_max(m, s_max[0]);
    product = block_max(product, s_max[1]) / m;
    // below 2^16, as |g| / m is at most 1; neither 0, nor infinite for want of fp32's range
    if (product > 0.f && product < 131072.f) {
      const int exponent = static_cast<int>(__float_as_uint(product) >> 23) - 127;
      up = __uint_as_float(static_cast<uint32_t>(min(max(14 - exponent, 0), 24) + 127) << 23);
    }
  } else {
    m = block_max(m, s_max[0]);
  }
  if (m == 0.f) m = 1.f;
  if (blockIdx.x == 0 && threadIdx.x == 0) *unscale = m / up;
  const int packs = hidden / 8;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < static_cast<int64_t>(n) * packs;
       i += static_cast<int64_t>(blocks) * blockDim.x) {
    const int row = static_cast<int>(i / packs);
    const bool kept = counts(targets[row], ignore, vocab);
    const float f = kept ? g[row] / m * up : 0.f;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (kept) {
      v = reinterpret_cast<const uint4*>(h)[i];
      uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 u = Type16<T>::unpack(w[j]);
        w[j] = Type16<T>::pack(u.x * f, u.y * f);
      }
    }
    reinterpret_cast<uint4*>(scaled)[i] = v;
  }
}

// Gradient, after the products: dh = T(g / dz_scale * sum over the k splits), zero in rows that do not count.
template <typename T>
__global__ void __launch_bounds__(256) loss_dh_kernel(const float* __restrict__ part, int splits,
                                                      const float* __restrict__ g, const int64_t* __restrict__ targets,
                                                      int64_t ignore, int vocab, int n, int hidden, float dz_scale,
                                                      T* __restrict__ dh) {
  pdl_wait();
  const int packs = hidden / 8;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= static_cast<int64_t>(n) * packs) return;
  const int row = static_cast<int>(i / packs);
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (counts(targets[row], ignore, vocab)) {
    float acc[8] = {};
    const float4* src = reinterpret_cast<const float4*>(part) + 2 * i;
    const int64_t step = static_cast<int64_t>(n) * packs * 2;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const float4 x = src[s * step], y = src[s * step + 1];
      acc[0] += x.x, acc[1] += x.y, acc[2] += x.z, acc[3] += x.w;
      acc[4] += y.x, acc[5] += y.y, acc[6] += y.z, acc[7] += y.w;
    }
    const float f = g[row] / dz_scale;
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = Type16<T>::pack(acc[2 * j] * f, acc[2 * j + 1] * f);
  }
  reinterpret_cast<uint4*>(dh)[i] = v;
}

// ------------------------------------------------------------------------------------------------
// Host side
static int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

constexpr int kPairs = 74;                        // CTA pairs of a B200
constexpr int64_t kDzBytes = int64_t(112) << 20;  // a piece's dz at most: it and what it meets stay mostly in L2

struct LossLayout {
  int n_tiles;
  int box, share;  // loss_few_kernel: vocabulary rows of a tile, of a CTA; 0 where it is not used
  int parts;  // (max, sum) of a row
  int64_t total;
};
static LossLayout loss_layout(int n, int vocab) {
  LossLayout l;
  l.n_tiles = (vocab + kBN - 1) / kBN;
  const int rows = up(vocab, 2 * kPairs) / (2 * kPairs), tiles = (rows + 127) / 128;  // of a CTA an SM
  l.box = n > kFewRows ? 0 : rows < 32 ? 32 : (rows + tiles - 1) / tiles;
  l.share = l.box * tiles;
  l.parts = l.share > 0 ? (vocab + l.share - 1) / l.share : 2 * l.n_tiles;
  l.total = static_cast<int64_t>(l.parts) * n * static_cast<int64_t>(sizeof(float2));
  return l;
}

struct GradLayout {
  int pieces, width, splits;  // width: columns of a piece, a multiple of the tile
  // offsets (range: loss_scale_kernel's factor, then loss_range_kernel's results; target: dz at the targets); all bytes
  int64_t range, target, dz, part, total;
};

// Time of a piece of `c` vocabulary tiles, in k blocks of the CTA pair that has the most to do (tiles are dealt out in turn,
// dh's before dW's). A tile costs one k block more than its contraction, and 12 at least (its epilogue), a launch 15.
// dh's fp32 sums, read and written for each piece and split, cost as much as a k block (0.27 us) for every 100000.
static int64_t piece_time(int64_t m, int64_t nh, int64_t kb_n, int64_t kb_h, int64_t c, int64_t splits) {
  const int64_t dh = m * nh * splits, all = dh + c * nh;
  const int64_t t_dh = (c * (kBN / kBK) + splits - 1) / splits + 1, t_dw = kb_n + 1 > 12 ? kb_n + 1 : 12;
  int64_t most = 0;
  const int64_t turns[3] = {0, dh % kPairs, all % kPairs};  // where the number of dh's, or of all tiles, changes
  for (int64_t p : turns) {
    const int64_t here_dh = (dh - p + kPairs - 1) / kPairs, here = (all - p + kPairs - 1) / kPairs;
    const int64_t t = here_dh * t_dh + (here - here_dh) * t_dw;
    if (t > most) most = t;
  }
  return most + (m * c + kPairs - 1) / kPairs * (kb_h + 1) + 30;
}

static GradLayout grad_layout(int n, int vocab, int hidden) {
  GradLayout l{};
  const int64_t tiles = (vocab + kBN - 1) / kBN, m = up(n > 0 ? n : 1, kBM) / kBM, nh = up(hidden, kBN) / kBN;
  const int64_t kb_n = up(n, kBK) / kBK, kb_h = up(hidden, kBK) / kBK;
  int64_t most = kDzBytes / (2 * static_cast<int64_t>(n > 0 ? n : 1)) / kBN;
  if (most < 1) most = 1;
  // Pieces from as few as dz allows, and parts of dh's contraction (few rows: dh has few tiles, whose contraction is as long
  // as the piece), so that the pairs end together. With as few pieces as possible, and parts until every pair has a tile of
  // dh: 1024 rows of 1280 339 us, 2048 rows 824, 8189 rows 2756; so 325, 729, 2713.
  const int64_t least = (tiles + most - 1) / most;
  int64_t best = -1;
  for (int64_t pieces = least; pieces <= least + 4 && pieces <= tiles; ++pieces) {
    const int64_t per = (tiles + pieces - 1) / pieces, whole = (tiles - 1) / per, last = tiles - whole * per;
    // at least 4 k blocks a part, and one in the last piece, whose last tile may be cut
    const int64_t kb = (vocab < per * kBN ? up(vocab, kBK) : per * kBN) / kBK / 4;
    const int64_t kb_last = (vocab - whole * per * kBN + kBK - 1) / kBK;
    for (int64_t splits = 1; splits <= 16; ++splits) {
      if (splits > 1 && (splits > kb || splits > kb_last)) break;
      const int64_t t = whole * piece_time(m, nh, kb_n, kb_h, per, splits) +
                        piece_time(m, nh, kb_n, kb_h, last, splits) + (whole + 1) * splits * n * hidden / 100000;
      if (best >= 0 && t >= best) continue;
      best = t;
      l.pieces = static_cast<int>(whole + 1);
      l.width = static_cast<int>(per * kBN);
      l.splits = static_cast<int>(splits);
    }
  }
  l.range = up(static_cast<int64_t>(n) * hidden * 2, 256);
  l.target = l.range + up((1 + kRangeBlocks) * static_cast<int64_t>(sizeof(float2)), 256);
  l.dz = l.target + up(static_cast<int64_t>(n) * 4, 256);
  l.part = l.dz + up(static_cast<int64_t>(n) * l.width * 2, 256);
  l.total = l.part + static_cast<int64_t>(l.splits) * n * hidden * 4;
  return l;
}

// 2-D map with 128-byte swizzle over rows of `inner` contiguous 16-bit elements; boxes of 64 x box_outer.
static int make_map(CUtensorMap* m, CUtensorMapDataType type, const void* ptr, int64_t inner, int64_t outer, int64_t ld,
                    int box_outer) {
  EncodeTiledFn enc = tensor_map_encode_fn();
  if (!enc) return set_error(FW_ERR_LAUNCH, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
  cuuint32_t box[2] = {64, static_cast<cuuint32_t>(box_outer)};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(m, type, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(FW_ERR_ARG, "lm_head_loss: tensor map encode failed (%d)", static_cast<int>(r));
  return FW_OK;
}

// The same rows as {64, outer, chunks of 64}: boxes of 64 x 64 x 2 chunks.
static int make_chunk_map(CUtensorMap* m, CUtensorMapDataType type, const void* ptr, int64_t chunks, int64_t outer,
                          int64_t ld) {
  EncodeTiledFn enc = tensor_map_encode_fn();
  if (!enc) return set_error(FW_ERR_LAUNCH, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {64, static_cast<cuuint64_t>(outer), static_cast<cuuint64_t>(chunks)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld) * 2, 128};
  cuuint32_t box[3] = {64, 64, 2};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(m, type, 3, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(FW_ERR_ARG, "lm_head_loss: tensor map encode failed (%d)", static_cast<int>(r));
  return FW_OK;
}

// 3-D map over fp32 sums [splits][n][hidden]; boxes of 32 x 32.
static int make_part_map(CUtensorMap* m, const void* ptr, int hidden, int n, int splits) {
  EncodeTiledFn enc = tensor_map_encode_fn();
  if (!enc) return set_error(FW_ERR_LAUNCH, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(hidden), static_cast<cuuint64_t>(n), static_cast<cuuint64_t>(splits)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(hidden) * 4, static_cast<cuuint64_t>(hidden) * 4 * n};
  cuuint32_t box[3] = {32, 32, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(ptr), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(FW_ERR_ARG, "lm_head_loss: tensor map encode failed (%d)", static_cast<int>(r));
  return FW_OK;
}

template <int kKind, typename T>
static int launch_gemm(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& ta2, const CUtensorMap& tb2,
                       const CUtensorMap& tout, const CUtensorMap& tpart, const LossArgs& a, int tiles, cudaStream_t s,
                       bool pdl) {
  constexpr int kLossSmem = smem_of(kKind);
  auto kern = loss_gemm_kernel<kKind, T>;
  cudaError_t e = ensure_smem(kern, kLossSmem);
  if (e == cudaSuccess) {
    const int pairs = num_sms() / 2;
    e = launch(kern, dim3(2 * (tiles < pairs ? tiles : pairs)), dim3(threads_of(kKind)), kLossSmem, s, pdl, ta, tb, ta2,
               tb2, tout, tpart, a);
  }
  return launch_status(e, "lm_head_loss");
}

template <typename T, int kN>
static int launch_few(const CUtensorMap& tw, const void* h, const LossArgs& a, int share, int box,
                      cudaStream_t s) {
  CUtensorMap th;
  int rc = make_map(&th, Type16<T>::kMap, h, a.hidden, a.n, a.hidden, kN);
  if (rc) return rc;
  auto kern = loss_few_kernel<T, kN>;
  cudaError_t e = ensure_smem(kern, few_smem(kN));
  if (e == cudaSuccess)
    e = launch(kern, dim3((a.vocab + share - 1) / share), dim3(kFewThreads), few_smem(kN), s, false, tw, th, a, share, box);
  return launch_status(e, "lm_head_loss");
}

template <typename T>
static int run_loss(const void* h, const void* w, const int64_t* targets, float* loss, float* lse, int n, int vocab,
                    int hidden, int64_t ignore, void* ws, cudaStream_t s) {
  const LossLayout l = loss_layout(n, vocab);
  CUtensorMap ta, tb;
  LossArgs a{};
  a.n = n;
  a.hidden = hidden;
  a.width = a.vocab = vocab;
  a.m_tiles = (n + kBM - 1) / kBM;
  a.n_tiles = l.n_tiles;
  a.ignore = ignore;
  a.targets = targets;
  a.stats = static_cast<float2*>(ws);
  a.target_logit = loss;  // replaced by the results when the halves are joined
  a.target_rest = lse;
  a.h = h;
  a.w = w;
  int rc = make_map(&tb, Type16<T>::kMap, w, hidden, vocab, hidden, l.share > 0 ? l.box : 128);
  if (rc) return rc;
  if (l.share > 0) {
    rc = n <= 32 ? launch_few<T, 32>(tb, h, a, l.share, l.box, s) : launch_few<T, kFewRows>(tb, h, a, l.share, l.box, s);
  } else {
    rc = make_map(&ta, Type16<T>::kMap, h, hidden, n, hidden, 128);
    if (!rc) rc = launch_gemm<kStats, T>(ta, tb, ta, tb, ta, ta, a, a.m_tiles * a.n_tiles, s, false);
  }
  if (rc) return rc;
  cudaError_t e = launch(loss_combine_kernel, dim3((n + 31) / 32), dim3(kCombineThreads), 0, s, true,
                         static_cast<const float2*>(a.stats), l.parts, n, targets, ignore, vocab, loss, lse);
  return launch_status(e, "lm_head_loss combine");
}

template <typename T>
static int run_loss_grad(const void* h, const void* w, const int64_t* targets, const float* lse, const float* g,
                         void* dh, void* dw, int n, int vocab, int hidden, int64_t ignore, int accumulate, void* ws,
                         cudaStream_t s) {
  const GradLayout l = grad_layout(n, vocab, hidden);
  uint8_t* b = static_cast<uint8_t*>(ws);
  T* scaled = reinterpret_cast<T*>(b);
  float* unscale = reinterpret_cast<float*>(b + l.range);
  float2* range = reinterpret_cast<float2*>(b + l.range) + 1;
  float* target_dz = reinterpret_cast<float*>(b + l.target);
  void* dz = b + l.dz;
  float* part = reinterpret_cast<float*>(b + l.part);
  const float dz_scale = Type16<T>::kBf16 ? 1.f : 4096.f;
  const int64_t packs = static_cast<int64_t>(n) * (hidden / 8);
  const int64_t blocks = (packs + 255) / 256;
  const int ranges = static_cast<int>(blocks < kRangeBlocks ? blocks : kRangeBlocks);
  cudaError_t e = cudaSuccess;
  int rc = FW_OK;
  if (!Type16<T>::kBf16) {
    e = launch(loss_range_kernel, dim3(ranges), dim3(kScaleThreads), 0, s, false, static_cast<const half*>(h), g, targets,
               ignore, vocab, n, hidden, range);
    rc = launch_status(e, "lm_head_loss_grad range");
    if (rc) return rc;
  }
  const int most = 4 * num_sms(), rows = (n + kScaleThreads / 32 - 1) / (kScaleThreads / 32);
  const int scaling = static_cast<int>(blocks < most ? blocks : most);
  e = launch(loss_scale_kernel<T>, dim3(scaling + (rows < most ? rows : most)), dim3(kScaleThreads), 0, s, !Type16<T>::kBf16,
             static_cast<const T*>(h), g, targets, ignore, vocab, n, hidden, scaled, unscale,
             static_cast<const float2*>(range), ranges, scaling, static_cast<const T*>(w), lse, target_dz);
  rc = launch_status(e, "lm_head_loss_grad scale");
  CUtensorMap ta, tb, ga, gb, ga2, gb2, tz, tw, tp;
  if (!rc) rc = make_map(&ta, Type16<T>::kMap, h, hidden, n, hidden, 128);
  const bool chunks = hidden % 64 == 0;
  if (!rc)
    rc = chunks ? make_chunk_map(&gb2, Type16<T>::kMap, scaled, hidden / 64, n, hidden)
                : make_map(&gb2, Type16<T>::kMap, scaled, hidden, n, hidden, 64);
  if (!rc) rc = make_part_map(&tp, part, hidden, n, l.splits);
  for (int p = 0; p < l.pieces && !rc; ++p) {
    const int v0 = p * l.width, width = vocab - v0 < l.width ? vocab - v0 : l.width;
    const T* wp = static_cast<const T*>(w) + static_cast<int64_t>(v0) * hidden;
    rc = make_map(&tb, Type16<T>::kMap, wp, hidden, width, hidden, 128);
    if (!rc) rc = make_map(&ga, Type16<T>::kMap, dz, width, n, l.width, 128);
    if (!rc)
      rc = chunks ? make_chunk_map(&gb, Type16<T>::kMap, wp, hidden / 64, width, hidden)
                  : make_map(&gb, Type16<T>::kMap, wp, hidden, width, hidden, 64);
    // whole chunks: what dz holds behind `width` gives rows of dW that are not stored
    if (!rc) rc = make_chunk_map(&ga2, Type16<T>::kMap, dz, (width + 63) / 64, n, l.width);
    if (!rc) rc = make_map(&tz, Type16<T>::kMap, dz, width, n, l.width, 32);
    if (!rc && dw != nullptr)
      rc = make_map(&tw, Type16<T>::kMap, static_cast<T*>(dw) + static_cast<int64_t>(v0) * hidden, hidden, width, hidden, 32);
    if (!rc && dw == nullptr) tw = tz;  // not used
    if (rc) return rc;
    LossArgs a{};
    a.n = n;
    a.hidden = hidden;
    a.width = width;
    a.v0 = v0;
    a.vocab = vocab;
    a.m_tiles = (n + kBM - 1) / kBM;
    a.n_tiles = (width + kBN - 1) / kBN;
    a.ignore = ignore;
    a.targets = targets;
    a.lse = lse;
    a.dz = dz;
    a.ld_dz = l.width;
    a.dz_scale = dz_scale;
    a.target_dz = target_dz;
    rc = launch_gemm<kDz, T>(ta, tb, ta, tb, tz, tz, a, a.m_tiles * a.n_tiles, s, true);
    if (rc) return rc;
    a.m_tiles = dw != nullptr ? (width + kBM - 1) / kBM : 0;
    a.n_tiles = (hidden + kBN - 1) / kBN;
    a.dh_m_tiles = dh != nullptr ? (n + kBM - 1) / kBM : 0;
    a.splits = l.splits;
    a.part = part;
    a.dw = dw;
    a.unscale = unscale;
    a.first_piece = p == 0;
    a.accumulate = accumulate;
    a.chunks = chunks;
    rc = launch_gemm<kGrads, T>(ga, gb, ga2, gb2, tw, tp, a, (a.dh_m_tiles * a.splits + a.m_tiles) * a.n_tiles, s, true);
  }
  if (rc || dh == nullptr) return rc;
  e = launch(loss_dh_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, true,
             static_cast<const float*>(part), l.splits, g, targets, ignore, vocab, n, hidden, dz_scale,
             static_cast<T*>(dh));
  return launch_status(e, "lm_head_loss_grad dh");
}

// Checks that both entry points share.
static int check_loss(const char* what, const void* h, const void* w, const int64_t* targets, int n, int vocab,
                      int hidden, int dtype, const void* ws, int64_t ws_bytes, int64_t need) {
  FW_REQUIRE(n >= 0 && n <= (1 << 22) && vocab > 0 && vocab <= (1 << 22), FW_ERR_SHAPE,
             "%s: n and vocab must be at most %d", what, 1 << 22);
  FW_REQUIRE(hidden > 0 && hidden % 8 == 0 && hidden <= 65536, FW_ERR_SHAPE,
             "%s: hidden must be a multiple of 8, at most 65536", what);
  FW_REQUIRE(dtype == FW_F16 || dtype == FW_BF16, FW_ERR_ARG, "%s: dtype must be fp16 or bf16", what);
  FW_REQUIRE(n == 0 || (h && w && targets && ws), FW_ERR_NULL, "%s: h, w, targets and workspace are required", what);
  FW_REQUIRE(aligned16(h) && aligned16(w) && aligned16(ws), FW_ERR_ALIGN,
             "%s: h, w and workspace must be 16-byte aligned", what);
  FW_REQUIRE(n == 0 || ws_bytes >= need, FW_ERR_SHAPE, "%s: workspace too small (%lld of %lld bytes)", what,
             static_cast<long long>(ws_bytes), static_cast<long long>(need));
  return FW_OK;
}

unsigned int read_loss_errors(bool clear) {
  unsigned int v = 0, zero = 0;
  cudaMemcpyFromSymbol(&v, g_fw_dev_error, sizeof(v));
  if (clear && v) cudaMemcpyToSymbol(g_fw_dev_error, &zero, sizeof(zero));
  return v;
}

}  // namespace fw

using namespace fw;

extern "C" {

int fw_lm_head_loss_workspace(int n, int vocab, int64_t* bytes) {
  FW_REQUIRE(bytes != nullptr, FW_ERR_NULL, "lm_head_loss_workspace: bytes is NULL");
  FW_REQUIRE(n >= 0 && n <= (1 << 22) && vocab > 0 && vocab <= (1 << 22), FW_ERR_SHAPE,
             "lm_head_loss: n and vocab must be at most %d", 1 << 22);
  *bytes = loss_layout(n, vocab).total;
  return FW_OK;
}

int fw_lm_head_loss(const void* h, const void* w, const int64_t* targets, float* loss, float* lse, int n, int vocab,
                    int hidden, int64_t ignore_index, int dtype, void* workspace, int64_t workspace_bytes,
                    fw_stream_t stream) {
  int64_t need = 0;
  int rc = fw_lm_head_loss_workspace(n, vocab, &need);
  if (!rc) rc = check_loss("lm_head_loss", h, w, targets, n, vocab, hidden, dtype, workspace, workspace_bytes, need);
  if (rc || n == 0) return rc;
  FW_REQUIRE(loss && lse, FW_ERR_NULL, "lm_head_loss: loss and lse are required");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == FW_F16
             ? run_loss<half>(h, w, targets, loss, lse, n, vocab, hidden, ignore_index, workspace, s)
             : run_loss<__nv_bfloat16>(h, w, targets, loss, lse, n, vocab, hidden, ignore_index, workspace, s);
}

int fw_lm_head_loss_grad_workspace(int n, int vocab, int hidden, int64_t* bytes) {
  FW_REQUIRE(bytes != nullptr, FW_ERR_NULL, "lm_head_loss_grad_workspace: bytes is NULL");
  FW_REQUIRE(n >= 0 && n <= (1 << 22) && vocab > 0 && vocab <= (1 << 22) && hidden > 0 && hidden <= 65536,
             FW_ERR_SHAPE, "lm_head_loss_grad: n and vocab must be at most %d, hidden at most 65536", 1 << 22);
  *bytes = grad_layout(n, vocab, hidden).total;
  return FW_OK;
}

int fw_lm_head_loss_grad(const void* h, const void* w, const int64_t* targets, const float* lse, const float* g,
                         void* dh, void* dw, int n, int vocab, int hidden, int64_t ignore_index, int accumulate,
                         int dtype, void* workspace, int64_t workspace_bytes, fw_stream_t stream) {
  int64_t need = 0;
  int rc = fw_lm_head_loss_grad_workspace(n, vocab, hidden, &need);
  if (!rc)
    rc = check_loss("lm_head_loss_grad", h, w, targets, n, vocab, hidden, dtype, workspace, workspace_bytes, need);
  if (rc) return rc;
  FW_REQUIRE(aligned16(dh) && aligned16(dw), FW_ERR_ALIGN, "lm_head_loss_grad: dh and dw must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n == 0) {
    if (dw == nullptr || accumulate) return FW_OK;
    return launch_status(cudaMemsetAsync(dw, 0, static_cast<size_t>(vocab) * hidden * 2, s), "lm_head_loss_grad");
  }
  FW_REQUIRE(lse && g, FW_ERR_NULL, "lm_head_loss_grad: lse and g are required");
  FW_REQUIRE(dh != nullptr || dw != nullptr, FW_ERR_NULL, "lm_head_loss_grad: at least one of dh and dw is required");
  return dtype == FW_F16 ? run_loss_grad<half>(h, w, targets, lse, g, dh, dw, n, vocab, hidden, ignore_index,
                                               accumulate, workspace, s)
                         : run_loss_grad<__nv_bfloat16>(h, w, targets, lse, g, dh, dw, n, vocab, hidden, ignore_index,
                                                        accumulate, workspace, s);
}

}  // extern "C"
