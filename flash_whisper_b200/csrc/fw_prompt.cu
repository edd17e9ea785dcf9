// Attention over whole prompts: packed sequences of different lengths, causal or not, grouped heads, any number of
// queries per sequence (a whole prompt, a chunk behind a kept prefix, a single token), and its gradient.
//
//   s_ij = scale q_i . k_j for the keys j that query i sees: j < lk, and with `causal` j <= i + lk - lq (the last query
//   sees the last key)        lse_i = log sum_j exp s_ij        o_i = sum_j exp(s_ij - lse_i) v_j
// A query that sees no key has o = 0 and lse = -inf.
//
// Forward (prompt_attn_kernel): a CTA takes two tiles of 128 query rows of one sequence and one key head. The rows of
// a tile are (token, head of the group) pairs, tokens major, so that one read of K and V serves the whole group and a
// single token of a grouped model still fills several rows. S = Q K^T and O += P V run on tcgen05 with S, P and O in
// tensor memory (P, 16 bits, is the A operand from there: it never passes through shared memory); one thread owns a
// row, so maximum and sum need no exchange. S has a buffer of its own besides P: the next block's Q K^T runs while the
// current block's exponentials are computed, and the two tiles alternate on the tensor core. The running maximum moves
// only when a row exceeds it by 2^8, so O is seldom rescaled. What bounds it: 128 x 128 exponentials take twice as
// long as the tile's two products of depth 64.
// Few rows (serving): the keys are split over several CTAs, whose partial results prompt_join_kernel joins.
#include "fw_host.h"
#include "fw_tc.cuh"

namespace fw {

FW_DEFINE_ERROR_WORD();

__device__ __forceinline__ void prompt_flag(unsigned bits) { atomicOr(&g_fw_dev_error, bits); }

constexpr float kLog2 = 1.4426950408889634f;
constexpr int kRows = 128;  // query rows of a tile, keys of a block
constexpr uint32_t kTileBytes = kRows * 64 * 2;  // 16 KB
constexpr int kKvStages = 3;
constexpr int kFwdSmem = 2 * kTileBytes + 2 * kKvStages * kTileBytes + 1024;
constexpr int kFwdThreads = 32 * 10;  // 4 + 4 softmax warps (one tile each), MMA, TMA

struct PromptArgs {
  const int64_t *cu_q, *cu_k;  // [seqs + 1]
  int seqs, heads, kv_heads, group;
  int tokens;        // query tokens of a tile: 128 / group
  int64_t rows_q, rows_k;
  float scale_log2;  // scale * log2 e
  int causal, splits;
  void* out;
  int64_t out_token, out_head;  // strides, elements
  float* lse;                   // [heads][rows_q], may be null
  float *part_o, *part_lse;     // splits > 1: [splits][rows_q][heads][64], [splits][heads][rows_q]
};

// Where a work item lies: a pair of query tiles of one sequence.
struct Item {
  int64_t q0, k0;  // first rows of the sequence
  int lq, lk;
  int tile;        // index of the item within its sequence; -1: no such item
};

// Finds item `index` (counting ceil(lq / per) items per sequence), by one warp. Sequences whose offsets are out of
// order or out of range have none and set the error bit.
__device__ __forceinline__ Item find_item(const int64_t* cu_a, const int64_t* cu_b, int64_t rows_a, int64_t rows_b,
                                          int seqs, int per, int64_t index, int lane) {
  Item it;
  it.tile = -1;
  int64_t before = 0;
  for (int b0 = 0; b0 < seqs; b0 += 32) {
    const int b = b0 + lane;
    int64_t a0 = 0, a1 = 0, c0 = 0, c1 = 0;
    if (b < seqs) {
      a0 = cu_a[b], a1 = cu_a[b + 1], c0 = cu_b[b], c1 = cu_b[b + 1];
      if (a0 < 0 || a1 < a0 || a1 > rows_a || c0 < 0 || c1 < c0 || c1 > rows_b) {
        prompt_flag(FW_DEVERR_BAD_INDEX);
        a1 = a0;
      }
    }
    const int64_t n = (a1 - a0 + per - 1) / per;
    int64_t incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const int64_t start = before + incl - n;
    const unsigned hit = __ballot_sync(0xffffffffu, index >= start && index < start + n);
    if (hit != 0) {
      const int src = __ffs(hit) - 1;
      it.tile = static_cast<int>(index - __shfl_sync(0xffffffffu, start, src));
      it.q0 = __shfl_sync(0xffffffffu, a0, src);
      it.lq = static_cast<int>(__shfl_sync(0xffffffffu, a1, src) - it.q0);
      it.k0 = __shfl_sync(0xffffffffu, c0, src);
      it.lk = static_cast<int>(__shfl_sync(0xffffffffu, c1, src) - it.k0);
      return it;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return it;
}

template <typename T>
__global__ void __launch_bounds__(kFwdThreads, 1) prompt_attn_kernel(const __grid_constant__ CUtensorMap tmQ,
                                                                     const __grid_constant__ CUtensorMap tmK,
                                                                     const __grid_constant__ CUtensorMap tmV,
                                                                     PromptArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_q, full_k[kKvStages], empty_k[kKvStages], full_v[kKvStages],
      empty_v[kKvStages], landed_v, s_full[2], s_free[2], p_full[2], o_done[2];
  __shared__ uint32_t tmem_base_sh;
  __shared__ Item s_item;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  uint8_t* ks = smem + 2 * kTileBytes;
  uint8_t* vs = ks + kKvStages * kTileBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // blockIdx.x = (item * kv_heads + key head) * splits + split
  const int split = blockIdx.x % a.splits;
  const int kvh = blockIdx.x / a.splits % a.kv_heads;
  if (warp == 8) tmem_alloc(&tmem_base_sh, 512);
  if (warp == 9) {
    const Item it = find_item(a.cu_q, a.cu_k, a.rows_q, a.rows_k, a.seqs, 2 * a.tokens,
                              blockIdx.x / a.splits / a.kv_heads, lane);
    if (lane == 0) {
      s_item = it;
      mbar_init(&bar_q, 1);
      mbar_init(&landed_v, 1);
      for (int i = 0; i < kKvStages; ++i) {
        mbar_init(&full_k[i], 1);
        mbar_init(&empty_k[i], 1);
        mbar_init(&full_v[i], 1);
        mbar_init(&empty_v[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[i], 1);  // scores of the tile's next block are in tensor memory
        mbar_init(&s_free[i], 4);  // its softmax warps have read them
        mbar_init(&p_full[i], 4);  // P is in tensor memory
        mbar_init(&o_done[i], 1);  // P V has been added to O
      }
      mbar_fence_init();
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;
  Item it = s_item;
  if (it.tile >= 0) {
    // Causal: the items of a sequence from its end, so that the longest start first.
    const int items = (it.lq + 2 * a.tokens - 1) / (2 * a.tokens);
    const int tile = a.causal ? items - 1 - it.tile : it.tile;
    const int shift = it.lk - it.lq;
    int tok[2], blocks[2];  // first token of each tile; key blocks that it sees
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      tok[t] = (2 * tile + t) * a.tokens;
      const int last = min(it.lq, tok[t] + a.tokens) - 1;  // its last token
      const int seen = tok[t] >= it.lq ? 0 : a.causal ? max(0, min(it.lk, last + shift + 1)) : it.lk;
      blocks[t] = (seen + kRows - 1) / kRows;
    }
    const int all = max(blocks[0], blocks[1]);
    const int j0 = static_cast<int>(static_cast<int64_t>(all) * split / a.splits);
    const int cnt = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / a.splits) - j0;
    const int nt[2] = {max(0, min(cnt, blocks[0] - j0)), max(0, min(cnt, blocks[1] - j0))};

    if (warp == 9) {
      // ---- loads
      if (lane == 0 && cnt > 0) {
        const uint32_t bytes = static_cast<uint32_t>(a.tokens * a.group) * 128;
        mbar_arrive_expect_tx(&bar_q, nt[1] > 0 ? 2 * bytes : bytes);
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (t == 0 || nt[1] > 0)
            tma_load_3d(smem + t * kTileBytes, &tmQ, &bar_q, 0, kvh * a.group, static_cast<int>(it.q0 + tok[t]));
      }
      bool ok = true;
      for (int jj = 0; jj < cnt && ok; ++jj) {
        const int s = jj % kKvStages;
        const uint32_t ph = ((jj / kKvStages) & 1u) ^ 1u;
        const int key = (j0 + jj) * kRows, row = static_cast<int>(it.k0) + key, valid = it.lk - key;
        uint8_t* vdst = vs + s * kTileBytes;
        if (lane == 0) {
          if (jj >= kKvStages) ok = mbar_wait(&empty_k[s], ph);
          if (ok) {
            mbar_arrive_expect_tx(&full_k[s], kTileBytes);
            tma_load_3d(ks + s * kTileBytes, &tmK, &full_k[s], 0, kvh, row);
            if (jj >= kKvStages) ok = mbar_wait(&empty_v[s], ph);
          }
          if (ok) {
            uint64_t* bar = valid >= kRows ? &full_v[s] : &landed_v;
            mbar_arrive_expect_tx(bar, kTileBytes);
            tma_load_3d(vdst, &tmV, bar, 0, kvh, row);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (ok && valid < kRows) {
          // The rows behind the sequence's last key belong to somebody else and may hold anything; P is 0 there, and
          // 0 x NaN must not reach O.
          ok = mbar_wait_warp(&landed_v, 0);  // once per CTA: only the last block is cut short
          for (int i = valid * 8 + lane; i < kRows * 8; i += 32)
            reinterpret_cast<uint4*>(vdst)[i] = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full_v[s]);
        }
        if (!ok && lane == 0) prompt_flag(FW_DEVERR_TIMEOUT);
      }
    } else if (warp == 8) {
      // ---- products
      if (lane == 0 && cnt > 0) {
        constexpr uint32_t idesc_s = make_idesc(kRows, kRows, Type16<T>::kBf16, false, false);
        constexpr uint32_t idesc_o = make_idesc(kRows, 64, Type16<T>::kBf16, false, true);
        bool ok = mbar_wait(&bar_q, 0);
        for (int jj = -1; jj < cnt && ok; ++jj) {
          if (jj + 1 < cnt) {  // S of the next block
            const int s = (jj + 1) % kKvStages;
            ok = mbar_wait(&full_k[s], ((jj + 1) / kKvStages) & 1u);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (!ok || jj + 1 >= nt[t]) continue;
              if (jj >= 0) ok = mbar_wait(&s_free[t], jj & 1u);
              tc_fence_after();
              const uint64_t qd = sw128_desc(base + t * kTileBytes);
              const uint64_t kd = sw128_desc(base + (2 + s) * kTileBytes);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                tc_mma_f16(tmem + t * 128, qd + 2 * kk, kd + 2 * kk, idesc_s, kk != 0 ? 1u : 0u);
              tc_commit(&s_full[t]);
            }
            tc_commit(&empty_k[s]);
          }
          if (jj < 0 || !ok) continue;
          const int s = jj % kKvStages;
          ok = mbar_wait(&full_v[s], (jj / kKvStages) & 1u);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || jj >= nt[t]) continue;
            ok = mbar_wait(&p_full[t], jj & 1u);
            tc_fence_after();
            const uint64_t vd = sw128_mn_desc(base + (2 + kKvStages + s) * kTileBytes, kTileBytes);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              tc_mma_ta(tmem + 256 + t * 64, tmem + 384 + t * 64 + 8 * kk, vd + 128 * kk, idesc_o,
                        jj != 0 || kk != 0 ? 1u : 0u);
            tc_commit(&o_done[t]);
          }
          tc_commit(&empty_v[s]);
        }
        if (!ok) prompt_flag(FW_DEVERR_TIMEOUT);
      }
    } else {
      // ---- softmax: thread = row
      const int t = warp >> 2;
      const int r = (warp & 3) * 32 + lane;
      const int n = nt[t];
      const int token = tok[t] + r / a.group, head = kvh * a.group + r % a.group;
      const bool live = r < a.tokens * a.group && token < it.lq;
      const bool warp_live = __any_sync(0xffffffffu, live);
      const int limit = a.causal ? min(it.lk - 1, token + shift) : it.lk - 1;  // the last key that it sees
      const int safe = a.causal ? min(it.lk - 1, tok[t] + shift) : it.lk - 1;  // that every row of the tile sees
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t ts = tmem + lanes + t * 128, to = tmem + lanes + 256 + t * 64, tp = tmem + lanes + 384 + t * 64;
      const float c = a.scale_log2;
      float top = -INFINITY, sum = 0.f;
      bool ok = true;
      for (int jj = 0; jj < n; ++jj) {
        ok = mbar_wait_warp(&s_full[t], jj & 1u);
        if (!ok) break;
        if (!warp_live) {  // no row of this warp counts: whatever P holds in its lanes stays in them
          // not before the other warps' arrivals of the block before have been used up
          ok = jj == 0 || mbar_wait_warp(&o_done[t], (jj - 1) & 1u);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive(&s_free[t]);
            mbar_arrive(&p_full[t]);
          }
          continue;
        }
        tc_fence_after();
        uint32_t x[4][32];
#pragma unroll
        for (int i = 0; i < 4; ++i) tc_load32(ts + 32 * i, x[i]);
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[t]);
        const int key = (j0 + jj) * kRows;
        if (key + kRows - 1 > safe) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (key + i > limit) x[i >> 5][i & 31] = 0xff800000u;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(x[i >> 5][i & 31]));
        const float cand = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
        const bool move = cand > top + 8.f || (top == -INFINITY && cand > top);
        bool waited = jj == 0;
        if (__any_sync(0xffffffffu, move)) {
          const float next = move ? cand : top;
          const float f = top == -INFINITY ? 0.f : ex2(top - next);
          sum *= move ? f : 1.f;
          top = next;
          if (jj > 0) {
            ok = mbar_wait_warp(&o_done[t], (jj - 1) & 1u);
            if (!ok) break;
            waited = true;
            tc_fence_after();
            uint32_t o[32];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              tc_load32(to + 32 * i, o);
              tc_wait_ld();
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (move) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tc_store32(to + 32 * i, o);
            }
          }
        }
        const float off = top == -INFINITY ? 0.f : -top;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t p[2][32];
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          const float e0 = ex2(fmaf(__uint_as_float(x[i >> 4][(2 * i) & 31]), c, off));
          const float e1 = ex2(fmaf(__uint_as_float(x[i >> 4][(2 * i + 1) & 31]), c, off));
          acc[i & 1] += e0;
          acc[2 + (i & 1)] += e1;
          p[i >> 5][i & 31] = Type16<T>::pack(e0, e1);
        }
        sum += (acc[0] + acc[1]) + (acc[2] + acc[3]);
        if (!waited) {  // P of the previous block has been read
          ok = mbar_wait_warp(&o_done[t], (jj - 1) & 1u);
          if (!ok) break;
          tc_fence_after();
        }
        tc_store32(tp, p[0]);
        tc_store32(tp + 32, p[1]);
        tc_wait_store();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (ok && n > 0 && warp_live) ok = mbar_wait_warp(&o_done[t], (n - 1) & 1u);
      if (!ok && lane == 0) prompt_flag(FW_DEVERR_TIMEOUT);
      if (ok && warp_live) {
        tc_fence_after();
        uint32_t o[2][32];
        if (n > 0) {
          tc_load32(to, o[0]);
          tc_load32(to + 32, o[1]);
          tc_wait_ld();
        }
        const bool none = sum == 0.f;  // no key seen (here)
        const float inv = none ? 0.f : 1.f / sum;
        const float lse = none ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
        if (live) {
          const int64_t row = it.q0 + token;
#pragma unroll
          for (int i = 0; i < 64; ++i)
            o[i >> 5][i & 31] = none ? 0u : __float_as_uint(__uint_as_float(o[i >> 5][i & 31]) * inv);
          if (a.splits > 1) {
            uint4* dst = reinterpret_cast<uint4*>(a.part_o + ((split * a.rows_q + row) * a.heads + head) * 64);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint32_t* u = &o[i >> 3][4 * (i & 7)];
              dst[i] = make_uint4(u[0], u[1], u[2], u[3]);
            }
            a.part_lse[(static_cast<int64_t>(split) * a.heads + head) * a.rows_q + row] = lse;
          } else {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * a.out_token + head * a.out_head);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint32_t* u = &o[i >> 2][8 * (i & 3)];
              dst[i] = make_uint4(Type16<T>::pack(__uint_as_float(u[0]), __uint_as_float(u[1])),
                                  Type16<T>::pack(__uint_as_float(u[2]), __uint_as_float(u[3])),
                                  Type16<T>::pack(__uint_as_float(u[4]), __uint_as_float(u[5])),
                                  Type16<T>::pack(__uint_as_float(u[6]), __uint_as_float(u[7])));
            }
            if (a.lse != nullptr) a.lse[head * a.rows_q + row] = lse;
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) {
    tmem_relinquish();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the key splits of a (row, head), one warp each: o = sum_s exp(lse_s - lse) o_s.
template <typename T>
__global__ void __launch_bounds__(128) prompt_join_kernel(PromptArgs a) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (i >= a.rows_q * a.heads) return;
  const int64_t row = i / a.heads;
  const int head = static_cast<int>(i % a.heads);
  // rows that belong to no sequence keep what they hold; sequences with bad offsets were left out above
  int64_t lo = 0, hi = a.seqs;  // the sequence with cu_q[lo] <= row < cu_q[lo + 1]
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (a.cu_q[mid] <= row)
      lo = mid;
    else
      hi = mid;
  }
  const int64_t k0 = a.cu_k[lo], k1 = a.cu_k[lo + 1];
  if (row < a.cu_q[lo] || row >= a.cu_q[lo + 1] || a.cu_q[lo] < 0 || a.cu_q[lo + 1] > a.rows_q || k0 < 0 || k1 < k0 ||
      k1 > a.rows_k)
    return;
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_lse[(static_cast<int64_t>(s) * a.heads + head) * a.rows_q + row]);
  const float off = top == -INFINITY ? 0.f : -top * kLog2;
  float sum = 0.f;
  float2 o = make_float2(0.f, 0.f);
  for (int s = 0; s < a.splits; ++s) {
    const float f = ex2(fmaf(a.part_lse[(static_cast<int64_t>(s) * a.heads + head) * a.rows_q + row], kLog2, off));
    const float2 v =
        reinterpret_cast<const float2*>(a.part_o + ((static_cast<int64_t>(s) * a.rows_q + row) * a.heads + head) * 64)[lane];
    sum += f;
    o.x = fmaf(f, v.x, o.x);
    o.y = fmaf(f, v.y, o.y);
  }
  const bool none = sum == 0.f;
  const float inv = none ? 0.f : 1.f / sum;
  reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + row * a.out_token + head * a.out_head)[lane] =
      none ? 0u : Type16<T>::pack(o.x * inv, o.y * inv);
  if (lane == 0 && a.lse != nullptr) a.lse[head * a.rows_q + row] = none ? -INFINITY : top + logf(sum);
}

// ------------------------------------------------------------------------------------------------
// Host side
// Splits of the keys: none when the query tiles fill the SMs; else as many as make two CTAs an SM, up to one per key
// block of an average sequence. From sizes only (the offsets are on the device).
static int prompt_splits(int64_t rows_q, int64_t rows_k, int seqs, int kv_heads, int group) {
  const int64_t items = (rows_q / (2 * (kRows / group)) + seqs) * kv_heads;  // at most
  const int64_t blocks = seqs > 0 ? (rows_k / seqs + kRows - 1) / kRows : 1;
  int64_t s = items > 0 ? 2 * 148 / items : 1;
  if (s > blocks) s = blocks;
  return static_cast<int>(s < 1 ? 1 : s > 64 ? 64 : s);
}

// 3-D map {64, heads, rows} with 128-byte swizzle; boxes of 64 x box_heads x box_rows.
static int make_rows_map(CUtensorMap* m, CUtensorMapDataType type, const void* ptr, int64_t rows, int heads,
                         int64_t token, int64_t head, int box_heads, int box_rows) {
  EncodeTiledFn enc = tensor_map_encode_fn();
  if (!enc) return set_error(FW_ERR_LAUNCH, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {64, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(head) * 2, static_cast<cuuint64_t>(token) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(m, type, 3, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(FW_ERR_ARG, "prompt_attention: tensor map encode failed (%d)", static_cast<int>(r));
  return FW_OK;
}

template <typename T>
static int run_prompt(const fw_rows_t& q, const fw_rows_t& k, const fw_rows_t& v, PromptArgs a, cudaStream_t s) {
  CUtensorMap tq, tk, tv;
  const int64_t items = (a.rows_q / (2 * a.tokens) + a.seqs) * a.kv_heads * a.splits;
  FW_REQUIRE(items < (int64_t(1) << 31), FW_ERR_SHAPE, "prompt_attention: too many query tiles");
  // no keys at all: any valid address serves, nothing is read through it
  const bool keys = a.rows_k > 0;
  int rc = make_rows_map(&tq, Type16<T>::kMap, q.ptr, a.rows_q, a.heads, q.token, q.head, a.group, a.tokens);
  if (!rc) rc = keys ? make_rows_map(&tk, Type16<T>::kMap, k.ptr, a.rows_k, a.kv_heads, k.token, k.head, 1, kRows) : FW_OK;
  if (!rc) rc = keys ? make_rows_map(&tv, Type16<T>::kMap, v.ptr, a.rows_k, a.kv_heads, v.token, v.head, 1, kRows) : FW_OK;
  if (rc) return rc;
  auto kern = prompt_attn_kernel<T>;
  cudaError_t e = ensure_smem(kern, kFwdSmem);
  if (e == cudaSuccess)
    e = launch(kern, dim3(static_cast<unsigned>(items)), dim3(kFwdThreads), kFwdSmem, s, false, tq, keys ? tk : tq,
               keys ? tv : tq, a);
  rc = launch_status(e, "prompt_attention");
  if (rc || a.splits == 1) return rc;
  e = launch(prompt_join_kernel<T>, dim3(static_cast<unsigned>((a.rows_q * a.heads + 3) / 4)), dim3(128), 0, s, true, a);
  return launch_status(e, "prompt_attention join");
}

static int check_rows(const char* what, const char* name, const fw_rows_t& x, int heads, int64_t rows) {
  FW_REQUIRE(rows == 0 || x.ptr, FW_ERR_NULL, "%s: %s is required", what, name);
  FW_REQUIRE(aligned16(x.ptr) && x.token % 8 == 0 && x.head % 8 == 0, FW_ERR_ALIGN,
             "%s: %s must start on 16 bytes and have strides of a multiple of 8 elements", what, name);
  FW_REQUIRE(x.head >= 64 && x.token >= 64 && x.token < (int64_t(1) << 36) && x.head < (int64_t(1) << 36) &&
                 (heads == 1 || rows <= 1 || x.token >= x.head * (heads - 1) + 64 || x.head >= x.token * (rows - 1) + 64),
             FW_ERR_SHAPE, "%s: %s has overlapping or negative strides", what, name);
  return FW_OK;
}

static int check_prompt(const char* what, const int64_t* cu_q, const int64_t* cu_k, int seqs, int64_t rows_q,
                        int64_t rows_k, int heads, int kv_heads, float scale, int dtype) {
  FW_REQUIRE(seqs >= 0 && rows_q >= 0 && rows_k >= 0 && rows_q < (int64_t(1) << 30) && rows_k < (int64_t(1) << 30),
             FW_ERR_SHAPE, "%s: bad sizes", what);
  FW_REQUIRE(kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads / kv_heads <= kRows && heads <= 65536,
             FW_ERR_SHAPE, "%s: heads must be a multiple of kv_heads, at most 128 times as many", what);
  FW_REQUIRE(scale > 0.f && scale < INFINITY, FW_ERR_ARG, "%s: scale must be positive and finite", what);
  FW_REQUIRE(dtype == FW_F16 || dtype == FW_BF16, FW_ERR_ARG, "%s: dtype must be fp16 or bf16", what);
  FW_REQUIRE(seqs == 0 || (cu_q && cu_k), FW_ERR_NULL, "%s: cu_q and cu_k are required", what);
  return FW_OK;
}

unsigned int read_prompt_errors(bool clear) {
  unsigned int v = 0, zero = 0;
  cudaMemcpyFromSymbol(&v, g_fw_dev_error, sizeof(v));
  if (clear && v) cudaMemcpyToSymbol(g_fw_dev_error, &zero, sizeof(zero));
  return v;
}

}  // namespace fw

using namespace fw;

extern "C" {

int fw_prompt_attention_workspace(int64_t rows_q, int64_t rows_k, int seqs, int heads, int kv_heads, int64_t* bytes) {
  FW_REQUIRE(bytes != nullptr, FW_ERR_NULL, "prompt_attention_workspace: bytes is NULL");
  int rc = check_prompt("prompt_attention", bytes, bytes, seqs, rows_q, rows_k, heads, kv_heads, 1.f, FW_F16);
  if (rc) return rc;
  const int splits = prompt_splits(rows_q, rows_k, seqs, kv_heads, heads / kv_heads);
  *bytes = splits > 1 ? splits * rows_q * heads * (64 + 1) * 4 : 0;
  return FW_OK;
}

int fw_prompt_attention(const fw_rows_t* q, const fw_rows_t* k, const fw_rows_t* v, const fw_rows_t* out, float* lse,
                        const int64_t* cu_q, const int64_t* cu_k, int seqs, int64_t rows_q, int64_t rows_k, int heads,
                        int kv_heads, float scale, int causal, int dtype, void* workspace, int64_t workspace_bytes,
                        fw_stream_t stream) {
  FW_REQUIRE(q && k && v && out, FW_ERR_NULL, "prompt_attention: q, k, v and out are required");
  int rc = check_prompt("prompt_attention", cu_q, cu_k, seqs, rows_q, rows_k, heads, kv_heads, scale, dtype);
  if (!rc) rc = check_rows("prompt_attention", "q", *q, heads, rows_q);
  if (!rc) rc = check_rows("prompt_attention", "k", *k, kv_heads, rows_k);
  if (!rc) rc = check_rows("prompt_attention", "v", *v, kv_heads, rows_k);
  if (!rc) rc = check_rows("prompt_attention", "out", *out, heads, rows_q);
  if (rc) return rc;
  int64_t need = 0;
  rc = fw_prompt_attention_workspace(rows_q, rows_k, seqs, heads, kv_heads, &need);
  if (rc) return rc;
  FW_REQUIRE(need == 0 || (workspace && aligned16(workspace)), FW_ERR_ALIGN,
             "prompt_attention: a 16-byte aligned workspace is required");
  FW_REQUIRE(workspace_bytes >= need, FW_ERR_SHAPE, "prompt_attention: workspace too small (%lld of %lld bytes)",
             static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  if (seqs == 0 || rows_q == 0) return FW_OK;
  PromptArgs a{};
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.seqs = seqs;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.group = heads / kv_heads;
  a.tokens = kRows / a.group;
  a.rows_q = rows_q;
  a.rows_k = rows_k;
  a.scale_log2 = scale * kLog2;
  a.causal = causal != 0;
  a.splits = prompt_splits(rows_q, rows_k, seqs, kv_heads, a.group);
  a.out = out->ptr;
  a.out_token = out->token;
  a.out_head = out->head;
  a.lse = lse;
  a.part_o = static_cast<float*>(workspace);
  a.part_lse = a.part_o + static_cast<int64_t>(a.splits) * rows_q * heads * 64;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == FW_F16 ? run_prompt<half>(*q, *k, *v, a, s) : run_prompt<__nv_bfloat16>(*q, *k, *v, a, s);
}

}  // extern "C"
