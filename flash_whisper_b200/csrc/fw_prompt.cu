// Attention over whole prompts: packed sequences of different lengths, causal or not, grouped heads, any number of
// queries per sequence (a whole prompt, a chunk behind a kept prefix, a single token), and its gradient.
//
//   s_ij = scale q_i . k_j for the keys j that query i sees: j < lk, and with `causal` j <= i + lk - lq (the last query
//   sees the last key)        lse_i = log sum_j exp s_ij        o_i = sum_j exp(s_ij - lse_i) v_j
// A query that sees no key has o = 0 and lse = -inf.
//
// Forward (prompt_attn_kernel): a CTA takes 128 query rows of one sequence and one key head. The rows of a tile are (token, head of the group) pairs, tokens major, so that one read of K and V serves the whole group and a
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
constexpr int kKStages = 3, kVStages = 2;  // 97 KB with Q: two CTAs an SM
constexpr int kFwdSmem = (1 + kKStages + kVStages) * kTileBytes + 1024;
constexpr int kFwdThreads = 32 * 6;  // 4 softmax warps, products, loads

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

// Where a work item lies: a tile of one sequence.
struct Item {
  int64_t q0, k0;  // first rows of the sequence
  int lq, lk;
  int tile;        // index of the item within its sequence; -1: no such item
  int seq;
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
      it.seq = b0 + src;
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
__global__ void __launch_bounds__(kFwdThreads, 2) prompt_attn_kernel(const __grid_constant__ CUtensorMap tmQ,
                                                                     const __grid_constant__ CUtensorMap tmK,
                                                                     const __grid_constant__ CUtensorMap tmV,
                                                                     PromptArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_q, full_k[kKStages], empty_k[kKStages], full_v[kVStages],
      empty_v[kVStages], landed_v, s_full, s_free, p_full, o_done;
  __shared__ uint32_t tmem_base_sh;
  __shared__ Item s_item;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  uint8_t* ks = smem + kTileBytes;
  uint8_t* vs = ks + kKStages * kTileBytes;
  const int warp = warp_index(), lane = threadIdx.x & 31;

  // blockIdx.x = (item * kv_heads + key head) * splits + split
  const int split = blockIdx.x % a.splits;
  const int kvh = blockIdx.x / a.splits % a.kv_heads;
  if (warp == 4) {
    tmem_alloc(&tmem_base_sh, 256);
    tmem_relinquish();
  }
  if (warp == 5) {
    const Item it = find_item(a.cu_q, a.cu_k, a.rows_q, a.rows_k, a.seqs, a.tokens,
                              blockIdx.x / a.splits / a.kv_heads, lane);
    if (lane == 0) {
      s_item = it;
      mbar_init(&bar_q, 1);
      mbar_init(&landed_v, 1);
      for (int i = 0; i < kKStages; ++i) {
        mbar_init(&full_k[i], 1);
        mbar_init(&empty_k[i], 1);
      }
      for (int i = 0; i < kVStages; ++i) {
        mbar_init(&full_v[i], 1);
        mbar_init(&empty_v[i], 1);
      }
      mbar_init(&s_full, 1);  // scores of the next block are in tensor memory
      mbar_init(&s_free, 4);  // the softmax warps have read them
      mbar_init(&p_full, 4);  // P is in tensor memory
      mbar_init(&o_done, 1);  // P V has been added to O
      mbar_fence_init();
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;  // columns: S 0, P 128, O 192
  const Item it = s_item;
  if (it.tile >= 0) {
    // Causal: the tiles of a sequence from its end, so that the longest start first.
    const int items = (it.lq + a.tokens - 1) / a.tokens;
    const int tok = (a.causal ? items - 1 - it.tile : it.tile) * a.tokens;  // the tile's first token
    const int shift = it.lk - it.lq;
    const int last = min(it.lq, tok + a.tokens) - 1;
    const int all = ((a.causal ? max(0, last + shift + 1) : it.lk) + kRows - 1) / kRows;  // key blocks that it sees
    const int j0 = static_cast<int>(static_cast<int64_t>(all) * split / a.splits);
    const int cnt = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / a.splits) - j0;

    if (warp == 5) {
      // ---- loads
      if (lane == 0 && cnt > 0) {
        mbar_arrive_expect_tx(&bar_q, static_cast<uint32_t>(a.tokens * a.group) * 128);
        tma_load_3d(smem, &tmQ, &bar_q, 0, kvh * a.group, static_cast<int>(it.q0 + tok));
      }
      bool ok = true;
      for (int jj = 0; jj < cnt && ok; ++jj) {
        const int s = jj % kKStages, sv = jj % kVStages;
        const int key = (j0 + jj) * kRows, row = static_cast<int>(it.k0) + key, valid = it.lk - key;
        uint8_t* vdst = vs + sv * kTileBytes;
        if (lane == 0) {
          if (jj >= kKStages) ok = mbar_wait(&empty_k[s], ((jj / kKStages) & 1u) ^ 1u);
          if (ok) {
            mbar_arrive_expect_tx(&full_k[s], kTileBytes);
            tma_load_3d(ks + s * kTileBytes, &tmK, &full_k[s], 0, kvh, row);
            if (jj >= kVStages) ok = mbar_wait(&empty_v[sv], ((jj / kVStages) & 1u) ^ 1u);
          }
          if (ok) {
            uint64_t* bar = valid >= kRows ? &full_v[sv] : &landed_v;
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
          if (lane == 0) mbar_arrive(&full_v[sv]);
        }
        if (!ok && lane == 0) prompt_flag(FW_DEVERR_TIMEOUT);
      }
    } else if (warp == 4) {
      // ---- products (the whole warp runs the loop, one lane issues)
      if (cnt > 0) {
        constexpr uint32_t idesc_s = make_idesc(kRows, kRows, Type16<T>::kBf16, false, false);
        constexpr uint32_t idesc_o = make_idesc(kRows, 64, Type16<T>::kBf16, false, true);
        const uint64_t qd = sw128_desc(base);
        bool ok = mbar_wait_warp(&bar_q, 0);
        for (int jj = -1; jj < cnt && ok; ++jj) {
          if (jj + 1 < cnt) {  // S of the next block
            const int s = (jj + 1) % kKStages;
            ok = mbar_wait_warp(&full_k[s], ((jj + 1) / kKStages) & 1u);
            if (ok && jj >= 0) ok = mbar_wait_warp(&s_free, jj & 1u);
            if (!ok) break;
            tc_fence_after();
            const uint64_t kd = sw128_desc(base + (1 + s) * kTileBytes);
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) tc_mma_f16(tmem, qd + 2 * kk, kd + 2 * kk, idesc_s, kk != 0 ? 1u : 0u);
              tc_commit(&s_full);
              tc_commit(&empty_k[s]);
            }
            __syncwarp();
          }
          if (jj < 0) continue;
          const int s = jj % kVStages;
          ok = mbar_wait_warp(&full_v[s], (jj / kVStages) & 1u) && mbar_wait_warp(&p_full, jj & 1u);
          if (!ok) break;
          tc_fence_after();
          const uint64_t vd = sw128_mn_desc(base + (1 + kKStages + s) * kTileBytes, kTileBytes);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              tc_mma_ta(tmem + 192, tmem + 128 + 8 * kk, vd + 128 * kk, idesc_o, jj != 0 || kk != 0 ? 1u : 0u);
            tc_commit(&o_done);
            tc_commit(&empty_v[s]);
          }
          __syncwarp();
        }
        if (!ok && lane == 0) prompt_flag(FW_DEVERR_TIMEOUT);
      }
    } else {
      // ---- softmax: thread = row
      const int r = warp * 32 + lane;
      const int token = tok + r / a.group, head = kvh * a.group + r % a.group;
      const bool live = r < a.tokens * a.group && token < it.lq;
      const bool warp_live = __any_sync(0xffffffffu, live);
      const int limit = a.causal ? min(it.lk - 1, token + shift) : it.lk - 1;  // the last key that it sees
      const int safe = a.causal ? min(it.lk - 1, tok + shift) : it.lk - 1;     // that every row of the tile sees
      const uint32_t ts = tmem + (static_cast<uint32_t>(warp * 32) << 16), tp = ts + 128, to = ts + 192;
      const float c = a.scale_log2;
      float top = -INFINITY, sum = 0.f;
      bool ok = true;
      for (int jj = 0; jj < cnt; ++jj) {
        ok = mbar_wait_warp(&s_full, jj & 1u);
        if (!ok) break;
        if (!warp_live) {  // no row of this warp counts: whatever P holds in its lanes stays in them
          // not before the other warps' arrivals of the block before have been used up
          ok = jj == 0 || mbar_wait_warp(&o_done, (jj - 1) & 1u);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive(&s_free);
            mbar_arrive(&p_full);
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
        if (lane == 0) mbar_arrive(&s_free);
        const int key = (j0 + jj) * kRows;
        if (key + kRows - 1 > safe) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (key + i > limit) x[i >> 5][i & 31] = 0xff800000u;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; i += 2)
          mx[(i >> 1) & 3] = fmaxf(fmaxf(mx[(i >> 1) & 3], __uint_as_float(x[i >> 5][i & 31])),
                                   __uint_as_float(x[i >> 5][(i + 1) & 31]));
        const float cand = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
        const bool move = cand > top + 8.f || (top == -INFINITY && cand > top);
        if (jj > 0) {  // P of the block before has been read, O is complete
          ok = mbar_wait_warp(&o_done, (jj - 1) & 1u);
          if (!ok) break;
          tc_fence_after();
        }
        if (__any_sync(0xffffffffu, move)) {
          const float next = move ? cand : top;
          const float f = !move ? 1.f : top == -INFINITY ? 0.f : ex2(top - next);
          sum *= f;
          top = next;
          if (jj > 0) {
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
              uint32_t o[16];
              tc_ld16(to + 16 * i, o);
              tc_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k)
                if (move) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tc_store16(to + 16 * i, o);
            }
          }
        }
        const float off = top == -INFINITY ? 0.f : -top;
        float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint32_t p[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 e = fma2(make_float2(__uint_as_float(x[h][2 * i]), __uint_as_float(x[h][2 * i + 1])),
                            make_float2(c, c), make_float2(off, off));
            e = make_float2(ex2(e.x), ex2(e.y));
            acc[i & 1] = add2(acc[i & 1], e);
            p[i] = Type16<T>::pack(e.x, e.y);
          }
          tc_store16(tp + 16 * h, p);
        }
        acc[0] = add2(acc[0], acc[1]);
        sum += acc[0].x + acc[0].y;
        tc_wait_store();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full);
      }
      if (ok && cnt > 0 && warp_live) ok = mbar_wait_warp(&o_done, (cnt - 1) & 1u);
      if (!ok && lane == 0) prompt_flag(FW_DEVERR_TIMEOUT);
      if (ok && warp_live) {
        tc_fence_after();
        uint32_t o[2][32];
        if (cnt > 0) {
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
  if (warp == 4) tmem_dealloc(tmem, 256);
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
// Gradient
//
//   delta_i = do_i . o_i      p_ij = exp(s_ij - lse_i)      ds_ij = p_ij (do_i . v_j - delta_i)
//   dv_j = sum_i p_ij do_i    dk_j = scale sum_i ds_ij q_i  dq_i = scale sum_j ds_ij k_j
// (dv and dk summed over the heads of the group). prompt_delta_kernel writes what both need of lse and delta per row;
// prompt_grad_kernel has CTAs of two roles, which share one pipeline, so that nothing is summed by atomics and
// results do not vary: a key role owns 128 keys of a key head and walks the queries (128 tokens of one head a step), a
// query role owns 128 (token, head) rows and walks the keys (128 a step). The probabilities are computed in both.
//   first products:   X = A1 B1^T, Y = A2 B2^T       key role: A = K, V   B = Q, dO;    query role: A = Q, dO  B = K, V
//   second products:  key role: dV += P^T dO, dK += dS^T Q;      query role: dQ += dS K
// Each step's B tile pair serves both products (K-major in the first, MN-major in the second). X, twice, and Y are in
// tensor memory; P and dS, the A operands of the second products, are written over X. 16 softmax warps (32 rows x 32
// columns each) compute a step's exponentials from X while the tensor core is still at the step before's second
// products and this step's Y, and need Y only then: a step's hand-overs hide behind the exponentials. A1 and A2 stay for
// the CTA's whole life, in shared memory in the key role (tensor memory is full) and in tensor memory in the query role.
// fp16 range: P is kept times 2^8, and dS times 2^4 over the power of two of the largest |do| (of the row in the query
// role, of the call in the key role), so that gradients of any size keep their bits; bf16 needs neither.
constexpr int kStep = 128;  // B rows of a step
constexpr int kGradStages = 4;
constexpr uint32_t kGradStage = 2 * kTileBytes;
constexpr int kGradSmem = 2 * kTileBytes + kGradStages * kGradStage + 1024;
constexpr int kGradThreads = 32 * 18;  // 16 softmax warps, products, loads
constexpr int kDeltaBlocks = 592;

struct GradArgs {
  PromptArgs p;
  const void *q, *k, *v, *o, *dout;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head, d_token, d_head;
  void *dq, *dk, *dv;
  int64_t dq_token, dq_head, dk_token, dk_head, dv_token, dv_head;
  // [heads][stat_rows]: log2 of P's factor - lse log2 e, and -delta, four rows of the first and then of the second at a
  // time; a sequence's rows start at stat_start()
  float* stat;
  int64_t stat_rows;
  float* largest;     // [kDeltaBlocks]: largest finite |do| each block met
  int64_t key_items;  // CTAs of the key role
  float scale;
};

// First row of sequence `seq` in stat: a multiple of 4 (16 bytes at least), behind the previous sequence's rows.
__device__ __forceinline__ int64_t stat_start(int64_t q0, int seq) { return ((q0 + 3) / 4 + seq) * 4; }

__device__ __forceinline__ float* stat_at(const GradArgs& g, int head, int64_t row) {
  return g.stat + (head * g.stat_rows + row / 4 * 4) * 2 + row % 4;
}

template <typename T>
__global__ void __launch_bounds__(256) prompt_delta_kernel(GradArgs g) {
  __shared__ float s_max[8];
  pdl_trigger();
  const PromptArgs& a = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t units = a.rows_q * a.heads;
  constexpr float kP = Type16<T>::kBf16 ? 0.f : 8.f;  // log2 of the factor that P carries
  float big = 0.f;
  for (int64_t u0 = (static_cast<int64_t>(blockIdx.x) * 8 + warp) * 4; u0 < units; u0 += static_cast<int64_t>(gridDim.x) * 32) {
    const int64_t u = u0 + (lane >> 3);
    float dot = 0.f;
    bool mine = u < units;
    int64_t row = 0, q0 = 0;
    int head = 0, seq = 0;
    if (mine) {
      row = u / a.heads;
      head = static_cast<int>(u % a.heads);
      int lo = 0, hi = a.seqs;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.cu_q[mid] <= row)
          lo = mid;
        else
          hi = mid;
      }
      seq = lo;
      q0 = a.cu_q[lo];
      mine = q0 >= 0 && q0 <= row && row < a.cu_q[lo + 1];  // rows of no sequence may hold anything
    }
    if (mine) {
      const uint4 d = reinterpret_cast<const uint4*>(static_cast<const T*>(g.dout) + row * g.d_token + head * g.d_head)[lane & 7];
      const uint4 o = reinterpret_cast<const uint4*>(static_cast<const T*>(g.o) + row * g.o_token + head * g.o_head)[lane & 7];
      const uint32_t dw[4] = {d.x, d.y, d.z, d.w}, ow[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = Type16<T>::unpack(dw[i]), y = Type16<T>::unpack(ow[i]);
        dot = fmaf(x.x, y.x, fmaf(x.y, y.y, dot));
        if (fabsf(x.x) < INFINITY) big = fmaxf(big, fabsf(x.x));
        if (fabsf(x.y) < INFINITY) big = fmaxf(big, fabsf(x.y));
      }
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (mine && (lane & 7) == 0) {
      float* st = stat_at(g, head, stat_start(q0, seq) + row - q0);
      st[0] = kP - a.lse[head * a.rows_q + row] * kLog2;
      st[4] = -dot;
    }
  }
  big = warp_max(big);
  if (lane == 0) s_max[warp] = big;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < 8; ++w) big = fmaxf(big, s_max[w]);
    g.largest[blockIdx.x] = big;
  }
}

// The power of two that takes x into [1, 2); 1 for 0, and within what fp32 holds.
__device__ __forceinline__ float normalizer(float x) {
  const int e = static_cast<int>(__float_as_uint(x) >> 23);  // x >= 0 and finite
  return e == 0 ? 1.f : __uint_as_float(static_cast<uint32_t>(min(254 - e, 227)) << 23);
}

// One softmax warp's share of a CTA's steps: 32 of the 128 columns. kKeys: the statistics are per column, from the
// step's stage, else the row's own.
struct GradRow {
  int steps, per_head, begin;
  int lo0, hi0;     // columns [lo0, hi0) of the whole walk count for this row
  float off, del;   // of this row (query role): stat's two
  float c, norm;
  uint32_t tx, ty;  // tensor memory: X (the second one 128 columns on) and Y, this warp's columns and lanes
  uint64_t *x_full, *y_full, *p_full, *full;
};
template <typename T, bool kKeys>
__device__ __forceinline__ bool grad_steps(const GradRow& g, int h, const float (*stat)[2 * kStep], int lane) {
  const float2 c2 = make_float2(g.c, g.c), n2 = make_float2(g.norm, g.norm);
  int block = 0;  // j % per_head in the key role
  for (int j = 0; j < g.steps; ++j) {
    const int s = j % kGradStages;
    const uint32_t tx = g.tx + 128 * (j & 1);
    // the statistics have landed for the first products; this thread's own view of them
    const uint32_t there = kKeys ? mbar_test(g.full + s, (j / kGradStages) & 1u) : 1u;
    if (!mbar_wait_warp(g.x_full + (j & 1), (j >> 1) & 1u)) return false;
    if (kKeys && !mbar_wait_tested(there, g.full + s, (j / kGradStages) & 1u)) return false;
    tc_fence_after();
    uint32_t x[32], y[32], p[16];
    tc_load32(tx, x);
    tc_wait_ld();
    const int at = (g.begin + block) * kStep + 32 * h;
    if (++block == g.per_head && kKeys) block = 0;
    const int lo = g.lo0 - at, hi = g.hi0 - at;
    const bool cut = __any_sync(0xffffffffu, lo > 0 || hi < 32);
    const float4* st = reinterpret_cast<const float4*>(&stat[s][64 * h]);
#pragma unroll
    for (int q = 0; q < 8; ++q) {  // four columns at a time
      float4 off = make_float4(g.off, g.off, g.off, g.off);
      if (kKeys) off = st[2 * q];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int k = 4 * q + 2 * i;
        const float2 e = fma2(make_float2(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), c2,
                              i == 0 ? make_float2(off.x, off.y) : make_float2(off.z, off.w));
        x[k] = __float_as_uint(ex2(e.x)), x[k + 1] = __float_as_uint(ex2(e.y));
      }
    }
    if (cut) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < lo || i >= hi) x[i] = 0u;
    }
    if (kKeys) {  // P over the X that this warp has read
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = Type16<T>::pack(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
      tc_store16(tx, p);
    }
    if (!mbar_wait_warp(g.y_full, j & 1u)) return false;
    tc_fence_after();
    tc_load32(g.ty, y);
    tc_wait_ld();
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      float4 del = make_float4(g.del, g.del, g.del, g.del);
      if (kKeys) del = st[2 * q + 1];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int k = 4 * q + 2 * i;
        float2 d = add2(make_float2(__uint_as_float(y[k]), __uint_as_float(y[k + 1])),
                        i == 0 ? make_float2(del.x, del.y) : make_float2(del.z, del.w));
        if (!Type16<T>::kBf16) d = mul2(d, n2);
        d = mul2(d, make_float2(__uint_as_float(x[k]), __uint_as_float(x[k + 1])));
        y[k] = __float_as_uint(d.x), y[k + 1] = __float_as_uint(d.y);
      }
    }
    if (cut) {  // 0 x what a foreign row gave may be NaN
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < lo || i >= hi) y[i] = 0u;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = Type16<T>::pack(__uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1]));
    tc_store16(tx + 16, p);
    tc_wait_store();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(g.p_full);
  }
  return true;
}

template <typename T>
__global__ void __launch_bounds__(kGradThreads, 1)
    prompt_grad_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmD,
                       const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, GradArgs g) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(16) float s_stat[kGradStages][2 * kStep];
  __shared__ __align__(8) uint64_t full[kGradStages], empty[kGradStages], landed, x_full[2], y_full, p_full, a_ready,
      done;
  __shared__ uint32_t tmem_base_sh;
  __shared__ Item s_item;
  __shared__ float s_norm, s_big[2][kRows];
  const PromptArgs& a = g.p;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* stages = smem_raw + (base - raw) + 2 * kTileBytes;  // behind A1 and A2 of the key role
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const bool keys = blockIdx.x < g.key_items;  // the role
  const int64_t index = keys ? blockIdx.x : blockIdx.x - g.key_items;
  const int kvh = static_cast<int>(index % a.kv_heads);

  if (warp == 16) tmem_alloc(&tmem_base_sh, 512);
  if (warp == 17) {
    const Item it = keys ? find_item(a.cu_k, a.cu_q, a.rows_k, a.rows_q, a.seqs, kRows, index / a.kv_heads, lane)
                         : find_item(a.cu_q, a.cu_k, a.rows_q, a.rows_k, a.seqs, a.tokens, index / a.kv_heads, lane);
    if (lane == 0) {
      s_item = it;
      for (int i = 0; i < kGradStages; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], 1);
      }
      mbar_init(&landed, 1);
      mbar_init(&x_full[0], 1);  // X of an even or odd step is in tensor memory
      mbar_init(&x_full[1], 1);
      mbar_init(&y_full, 1);     // Y is
      mbar_init(&p_full, 16);    // P and dS are, and Y has been read
      mbar_init(&a_ready, keys ? 1 : 16);
      mbar_init(&done, 1);
      mbar_fence_init();
      tma_prefetch_desc(keys ? &tmQ : &tmK);
      tma_prefetch_desc(keys ? &tmD : &tmV);
    }
  }
  pdl_wait();
  if (warp == 16 && !Type16<T>::kBf16) {
    float m = 0.f;
    for (int i = lane; i < kDeltaBlocks; i += 32) m = fmaxf(m, g.largest[i]);
    m = warp_max(m);
    if (lane == 0) s_norm = normalizer(m);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;
  Item it = s_item;
  if (it.tile >= 0) {
    if (keys) {  // find_item was asked with the roles of q and k swapped
      const int64_t r = it.q0;
      const int n = it.lq;
      it.q0 = it.k0, it.lq = it.lk;
      it.k0 = r, it.lk = n;
    }
    const int shift = it.lk - it.lq;
    // Key role: keys first .. first + 127, token blocks from `begin` on for each head of the group. Query role: tokens
    // from `first` on, all key blocks that the last of them sees.
    int first, begin, per_head, steps;
    if (keys) {
      first = it.tile * kRows;
      begin = a.causal ? max(0, first - shift) / kStep : 0;
      per_head = max(0, (it.lq + kStep - 1) / kStep - begin);
      steps = per_head * a.group;
    } else {
      const int items = (it.lq + a.tokens - 1) / a.tokens;
      first = (a.causal ? items - 1 - it.tile : it.tile) * a.tokens;  // causal: the longest first
      const int last = min(it.lq, first + a.tokens) - 1;
      begin = 0;
      per_head = steps = ((a.causal ? max(0, min(it.lk, last + shift + 1)) : it.lk) + kStep - 1) / kStep;
    }

    if (warp == 17) {
      // ---- loads
      if (keys && lane == 0 && steps > 0) {  // A1 = K, A2 = V; rows behind the sequence are rows of no result
        mbar_arrive_expect_tx(&a_ready, 2 * kTileBytes);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          tma_load_3d(stages - (2 - i) * kTileBytes, i == 0 ? &tmK : &tmV, &a_ready, 0, kvh,
                      static_cast<int>(it.k0) + first);
      }
      bool ok = true;
      uint32_t cut = 0;  // tiles that end inside a step so far
      for (int j = 0; j < steps && ok; ++j) {
        const int s = j % kGradStages;
        const int head = keys ? kvh * a.group + j / per_head : kvh;
        const int at = (begin + (keys ? j % per_head : j)) * kStep;
        const int valid = (keys ? it.lq : it.lk) - at;
        const int row = static_cast<int>(keys ? it.q0 : it.k0) + at;
        uint8_t* dst = stages + s * kGradStage;
        if (lane == 0) {
          if (j >= kGradStages) ok = mbar_wait(&empty[s], ((j / kGradStages) & 1u) ^ 1u);
          if (ok) {
            uint64_t* bar = valid >= kStep ? &full[s] : &landed;
            mbar_arrive_expect_tx(bar, kGradStage + (keys ? kStep * 8 : 0));
            tma_load_3d(dst, keys ? &tmQ : &tmK, bar, 0, head, row);
            tma_load_3d(dst + kTileBytes, keys ? &tmD : &tmV, bar, 0, head, row);
            if (keys)
              bulk_g2s(s_stat[s], stat_at(g, head, stat_start(it.q0, it.seq) + at), kStep * 8, bar);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (ok && valid < kStep) {
          // Rows behind the sequence's end may hold anything, and 0 x NaN must not reach a sum over them.
          ok = mbar_wait_warp(&landed, cut & 1u);
          ++cut;
          for (int i = valid * 8 + lane; i < kStep * 8; i += 32) {
            reinterpret_cast<uint4*>(dst)[i] = make_uint4(0u, 0u, 0u, 0u);
            reinterpret_cast<uint4*>(dst + kTileBytes)[i] = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[s]);
        }
        if (!ok && lane == 0) prompt_flag(FW_DEVERR_TIMEOUT);
      }
    } else if (warp == 16) {
      // ---- products (the whole warp runs the loop, one lane issues)
      if (steps > 0) {
        constexpr uint32_t idesc1 = make_idesc(kRows, kStep, Type16<T>::kBf16, false, false);
        constexpr uint32_t idesc2 = make_idesc(kRows, 64, Type16<T>::kBf16, false, true);
        const uint64_t a1 = sw128_desc(base), a2 = a1 + (kTileBytes >> 4);
        bool ok = mbar_wait_warp(&a_ready, 0);
        for (int j = -2; j < steps && ok; ++j) {
          if (j >= 0) ok = mbar_wait_warp(&p_full, j & 1u);
          if (ok && j + 2 < steps) ok = mbar_wait_warp(&full[(j + 2) % kGradStages], ((j + 2) / kGradStages) & 1u);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            if (j + 1 >= 0 && j + 1 < steps) {  // Y of the next step: the last one has been read
              const uint64_t b2 = sw128_desc(base + 2 * kTileBytes + (j + 1) % kGradStages * kGradStage + kTileBytes);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) {
                if (keys)
                  tc_mma_f16(tmem + 256, a2 + 2 * kk, b2 + 2 * kk, idesc1, kk != 0 ? 1u : 0u);
                else
                  tc_mma_ta(tmem + 256, tmem + 416 + 8 * kk, b2 + 2 * kk, idesc1, kk != 0 ? 1u : 0u);
              }
              tc_commit(&y_full);
            }
            const uint32_t x = tmem + 128 * (j & 1);
            if (j >= 0) {
              const uint64_t b1 = sw128_mn_desc(base + 2 * kTileBytes + j % kGradStages * kGradStage, kTileBytes),
                             b2 = b1 + (kTileBytes >> 4);
#pragma unroll
              for (int kk = 0; kk < 8; ++kk) {  // warp group g left its 32 columns of P and dS from 32 g and 32 g + 16 on
                const uint32_t p = x + 32 * (kk >> 1) + 8 * (kk & 1);
                if (keys) tc_mma_ta(tmem + 384, p, b2 + 128 * kk, idesc2, j != 0 || kk != 0 ? 1u : 0u);
                tc_mma_ta(tmem + 448, p + 16, b1 + 128 * kk, idesc2, j != 0 || kk != 0 ? 1u : 0u);
              }
              tc_commit(&empty[j % kGradStages]);
            }
            if (j + 2 < steps) {  // X of the step after the next, over P and dS of this one
              const uint64_t b1 = sw128_desc(base + 2 * kTileBytes + (j + 2) % kGradStages * kGradStage);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) {
                if (keys)
                  tc_mma_f16(x, a1 + 2 * kk, b1 + 2 * kk, idesc1, kk != 0 ? 1u : 0u);
                else
                  tc_mma_ta(x, tmem + 384 + 8 * kk, b1 + 2 * kk, idesc1, kk != 0 ? 1u : 0u);
              }
              tc_commit(&x_full[j & 1]);
            }
          }
          __syncwarp();
        }
        if (elect_one()) tc_commit(&done);
        if (!ok && lane == 0) prompt_flag(FW_DEVERR_TIMEOUT);
      }
    } else {
      // ---- softmax: thread = row of the A operands; warps 4 g .. 4 g + 3 work on columns 32 g .. + 31 of a step
      const int grp = warp >> 2;
      const int r = (warp & 3) * 32 + lane;
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const int token = keys ? 0 : first + r / a.group;
      const int head = keys ? kvh : kvh * a.group + r % a.group;
      const bool live = keys ? first + r < it.lk : r < a.tokens * a.group && token < it.lq;
      const int64_t row = keys ? it.k0 + first + r : it.q0 + token;
      GradRow gr;
      gr.off = gr.del = 0.f;
      if (!keys) {
        // the A operands into tensor memory: each warp group takes half the columns of A1 = Q (0, 1) or A2 = dO (2, 3)
        const bool second = grp >= 2;
        const T* src = static_cast<const T*>(second ? g.dout : g.q) + row * (second ? g.d_token : g.q_token) +
                       head * (second ? g.d_head : g.q_head);
        uint32_t x[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (live) v = reinterpret_cast<const uint4*>(src)[4 * (grp & 1) + i];
          x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
        }
        if (!Type16<T>::kBf16 && second) {
          float big = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 v = Type16<T>::unpack(x[i]);
            if (fabsf(v.x) < INFINITY) big = fmaxf(big, fabsf(v.x));
            if (fabsf(v.y) < INFINITY) big = fmaxf(big, fabsf(v.y));
          }
          s_big[grp & 1][r] = big;
        }
        tc_store16(tmem + lanes + 384 + 16 * grp, x);
        tc_wait_store();
        if (live) {
          const float* st = stat_at(g, head, stat_start(it.q0, it.seq) + token);
          gr.off = st[0];
          gr.del = st[4];
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&a_ready);
      }
      asm volatile("bar.sync 1, 512;" ::: "memory");  // s_big
      gr.steps = steps, gr.per_head = per_head, gr.begin = begin;
      gr.c = a.scale_log2;
      // the factor of dS besides P's
      gr.norm = Type16<T>::kBf16 ? 1.f : 0.0625f * (keys ? s_norm : normalizer(fmaxf(s_big[0][r], s_big[1][r])));
      gr.tx = tmem + lanes + 32 * grp;
      gr.ty = tmem + lanes + 256 + 32 * grp;
      gr.x_full = x_full, gr.y_full = &y_full, gr.p_full = &p_full;
      gr.full = full;
      bool ok;
      if (keys) {
        gr.hi0 = it.lq;
        gr.lo0 = a.causal ? first + r - shift : 0;
        ok = grad_steps<T, true>(gr, grp, s_stat, lane);
      } else {
        gr.lo0 = 0;
        gr.hi0 = (a.causal ? min(it.lk - 1, token + shift) : it.lk - 1) + 1;
        ok = grad_steps<T, false>(gr, grp, s_stat, lane);
      }
      if (ok && steps > 0) ok = mbar_wait_warp(&done, 0);
      if (!ok && lane == 0) prompt_flag(FW_DEVERR_TIMEOUT);
      // ---- results: 32 columns each of dK (groups 0, 1) and dV (2, 3), or of dQ (0, 1)
      if (ok && (keys || grp < 2)) {
        tc_fence_after();
        const bool dv = grp >= 2;
        uint32_t x[32];
        if (steps > 0) {
          tc_load32(tmem + lanes + (dv ? 384 : 448) + 32 * (grp & 1), x);
          tc_wait_ld();
        }
        if (live) {
          constexpr float kUnP = Type16<T>::kBf16 ? 1.f : 1.f / 256.f;
          const float f = dv ? kUnP : g.scale * kUnP / gr.norm;
          T* dst = static_cast<T*>(keys ? (dv ? g.dv : g.dk) : g.dq) +
                   row * (keys ? (dv ? g.dv_token : g.dk_token) : g.dq_token) +
                   head * (keys ? (dv ? g.dv_head : g.dk_head) : g.dq_head) + 32 * (grp & 1);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int e = 8 * i + 2 * k;
              w[k] = steps > 0 ? Type16<T>::pack(__uint_as_float(x[e]) * f, __uint_as_float(x[e + 1]) * f) : 0u;
            }
            reinterpret_cast<uint4*>(dst)[i] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 16) {
    tmem_relinquish();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------------------
// Host side
// Splits of the keys: none when the query tiles fill the SMs; else as many as make two CTAs an SM, up to one per key
// block of an average sequence. From sizes only (the offsets are on the device).
static int prompt_splits(int64_t rows_q, int64_t rows_k, int seqs, int kv_heads, int group) {
  const int64_t items = (rows_q / (kRows / group) + seqs) * kv_heads;  // at most
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
  const int64_t items = (a.rows_q / a.tokens + a.seqs) * a.kv_heads * a.splits;
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

template <typename T>
static int run_prompt_grad(const fw_rows_t& q, const fw_rows_t& k, const fw_rows_t& v, const fw_rows_t& d, GradArgs g,
                           cudaStream_t s) {
  const PromptArgs& a = g.p;
  const int64_t query_items = a.rows_q > 0 ? (a.rows_q / a.tokens + a.seqs) * a.kv_heads : 0;
  g.key_items = a.rows_k > 0 ? (a.rows_k / kRows + a.seqs) * a.kv_heads : 0;
  FW_REQUIRE(query_items + g.key_items < (int64_t(1) << 31), FW_ERR_SHAPE, "prompt_attention_grad: too many tiles");
  if (query_items + g.key_items == 0) return FW_OK;
  if (a.rows_q > 0) {
    cudaError_t e = launch(prompt_delta_kernel<T>, dim3(kDeltaBlocks), dim3(256), 0, s, false, g);
    const int rc = launch_status(e, "prompt_attention_grad delta");
    if (rc) return rc;
  }
  CUtensorMap tq{}, td{}, tk{}, tv{};
  int rc = FW_OK;
  if (a.rows_q > 0) {
    rc = make_rows_map(&tq, Type16<T>::kMap, q.ptr, a.rows_q, a.heads, q.token, q.head, 1, kStep);
    if (!rc) rc = make_rows_map(&td, Type16<T>::kMap, d.ptr, a.rows_q, a.heads, d.token, d.head, 1, kStep);
  }
  if (!rc && a.rows_k > 0) {
    rc = make_rows_map(&tk, Type16<T>::kMap, k.ptr, a.rows_k, a.kv_heads, k.token, k.head, 1, kStep);
    if (!rc) rc = make_rows_map(&tv, Type16<T>::kMap, v.ptr, a.rows_k, a.kv_heads, v.token, v.head, 1, kStep);
  }
  if (rc) return rc;
  if (a.rows_q == 0) tq = tk, td = tv;  // nothing is read through them
  if (a.rows_k == 0) tk = tq, tv = td;
  auto kern = prompt_grad_kernel<T>;
  cudaError_t e = ensure_smem(kern, kGradSmem);
  if (e == cudaSuccess)
    e = launch(kern, dim3(static_cast<unsigned>(g.key_items + query_items)), dim3(kGradThreads), kGradSmem, s,
               a.rows_q > 0, tq, td, tk, tv, g);
  return launch_status(e, "prompt_attention_grad");
}

static int64_t grad_stat_rows(int64_t rows_q, int seqs) {  // room for a step's copy behind the last row
  return (rows_q + 3) / 4 * 4 + 4 * static_cast<int64_t>(seqs) + 4 + kStep;
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

int fw_prompt_attention_grad_workspace(int64_t rows_q, int64_t rows_k, int seqs, int heads, int kv_heads,
                                       int64_t* bytes) {
  FW_REQUIRE(bytes != nullptr, FW_ERR_NULL, "prompt_attention_grad_workspace: bytes is NULL");
  int rc = check_prompt("prompt_attention_grad", bytes, bytes, seqs, rows_q, rows_k, heads, kv_heads, 1.f, FW_F16);
  if (rc) return rc;
  *bytes = kDeltaBlocks * 4 + heads * grad_stat_rows(rows_q, seqs) * 8;
  return FW_OK;
}

int fw_prompt_attention_grad(const fw_rows_t* q, const fw_rows_t* k, const fw_rows_t* v, const fw_rows_t* out,
                             const fw_rows_t* dout, const float* lse, const int64_t* cu_q, const int64_t* cu_k,
                             int seqs, int64_t rows_q, int64_t rows_k, int heads, int kv_heads, float scale, int causal,
                             int dtype, const fw_rows_t* dq, const fw_rows_t* dk, const fw_rows_t* dv, void* workspace,
                             int64_t workspace_bytes, fw_stream_t stream) {
  const char* what = "prompt_attention_grad";
  FW_REQUIRE(q && k && v && out && dout && dq && dk && dv, FW_ERR_NULL,
             "%s: q, k, v, out, dout, dq, dk and dv are required", what);
  int rc = check_prompt(what, cu_q, cu_k, seqs, rows_q, rows_k, heads, kv_heads, scale, dtype);
  if (!rc) rc = check_rows(what, "q", *q, heads, rows_q);
  if (!rc) rc = check_rows(what, "k", *k, kv_heads, rows_k);
  if (!rc) rc = check_rows(what, "v", *v, kv_heads, rows_k);
  if (!rc) rc = check_rows(what, "out", *out, heads, rows_q);
  if (!rc) rc = check_rows(what, "dout", *dout, heads, rows_q);
  if (!rc) rc = check_rows(what, "dq", *dq, heads, rows_q);
  if (!rc) rc = check_rows(what, "dk", *dk, kv_heads, rows_k);
  if (!rc) rc = check_rows(what, "dv", *dv, kv_heads, rows_k);
  if (rc) return rc;
  int64_t need = 0;
  rc = fw_prompt_attention_grad_workspace(rows_q, rows_k, seqs, heads, kv_heads, &need);
  if (rc) return rc;
  if (seqs == 0) return FW_OK;
  FW_REQUIRE(lse || rows_q == 0, FW_ERR_NULL, "%s: lse is required", what);
  FW_REQUIRE(workspace && aligned16(workspace), FW_ERR_ALIGN, "%s: a 16-byte aligned workspace is required", what);
  FW_REQUIRE(workspace_bytes >= need, FW_ERR_SHAPE, "%s: workspace too small (%lld of %lld bytes)", what,
             static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  GradArgs g{};
  PromptArgs& a = g.p;
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
  a.splits = 1;
  a.lse = const_cast<float*>(lse);
  g.q = q->ptr, g.q_token = q->token, g.q_head = q->head;
  g.k = k->ptr, g.k_token = k->token, g.k_head = k->head;
  g.v = v->ptr, g.v_token = v->token, g.v_head = v->head;
  g.o = out->ptr, g.o_token = out->token, g.o_head = out->head;
  g.dout = dout->ptr, g.d_token = dout->token, g.d_head = dout->head;
  g.dq = dq->ptr, g.dq_token = dq->token, g.dq_head = dq->head;
  g.dk = dk->ptr, g.dk_token = dk->token, g.dk_head = dk->head;
  g.dv = dv->ptr, g.dv_token = dv->token, g.dv_head = dv->head;
  g.largest = static_cast<float*>(workspace);
  g.stat = g.largest + kDeltaBlocks;
  g.stat_rows = grad_stat_rows(rows_q, seqs);
  g.scale = scale;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == FW_F16 ? run_prompt_grad<half>(*q, *k, *v, *dout, g, s)
                         : run_prompt_grad<__nv_bfloat16>(*q, *k, *v, *dout, g, s);
}

}  // extern "C"
