// Attention over whole prompts: packed sequences of different lengths, causal or not, grouped heads, any number of
// queries per sequence (a whole prompt, a chunk behind a kept prefix, a single token).
//
//   s_ij = scale q_i . k_j for the keys j that query i sees: j < lk, and with `causal` j <= i + lk - lq (the last query
//   sees the last key)        lse_i = log sum_j exp s_ij        o_i = sum_j exp(s_ij - lse_i) v_j
// A query that sees no key has o = 0 and lse = -inf.
//
// prompt_attn_kernel: a CTA takes 128 query rows of one sequence and one key head. The rows of a tile are (token, head of
// the group) pairs, tokens major, so that one read of K and V serves the whole group and a single token of a grouped model
// still fills several rows. S = Q K^T and O += P V run on tcgen05 with S, P and O in tensor memory (P, 16 bits, is the A
// operand from there: it never passes through shared memory); one thread owns a row, so maximum and sum need no exchange.
// S has a buffer of its own besides P: the next block's Q K^T runs while the current block's exponentials are computed,
// and two CTAs share an SM, so that the softmax of one fills the waits of the other. The running maximum moves only when
// a row exceeds it by 2^8, so O is seldom rescaled. What bounds it: 128 x 128 exponentials take twice as long as the
// tile's two products of depth 64; an eighth of them run on the FMA pipe instead. Six sequences up to 4096, 32 heads on 8 (bf16):
// 235 to 248 us as the clocks allow, 0.62 to 0.66 PFLOP/s, the special-function unit 45% and the tensor pipe 25% active, 39%
// of issue slots: the latency of the softmax warps' own chain. (Moving the maximum only past a threshold and exponentials on
// the FMA pipe are published techniques.)
// Few rows (serving): the keys are split over several CTAs, whose partial results prompt_join_kernel joins; where there
// are so few that tiles would be empty, prompt_few_kernel takes the place of the tensor core.
#include "fw_prompt.cuh"

namespace fw {

constexpr int kKStages = 3, kVStages = 2;  // 97 KB with Q: two CTAs an SM
constexpr int kFwdSmem = (1 + kKStages + kVStages) * kTileBytes + 1024;
constexpr int kFwdThreads = 32 * 6;  // 4 softmax warps, products, loads

// What a CTA has of its item: first token of the tile, first key block and number of them (this split's).
struct Span {
  int tok, j0, cnt;
};
__device__ __forceinline__ Span span_of(const PromptArgs& a, const Item& it, int split) {
  // Causal: the tiles of a sequence from its end, so that the longest start first.
  const int items = (it.lq + a.tokens - 1) / a.tokens;
  Span x;
  x.tok = (a.causal ? items - 1 - it.tile : it.tile) * a.tokens;
  const int last = min(it.lq, x.tok + a.tokens) - 1;
  const int all = ((a.causal ? max(0, last + it.lk - it.lq + 1) : it.lk) + kRows - 1) / kRows;  // key blocks that it sees
  x.j0 = static_cast<int>(static_cast<int64_t>(all) * split / a.splits);
  x.cnt = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / a.splits) - x.j0;
  return x;
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
  __shared__ Span s_span;
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
    const Item it = find_item(a.cu_q, a.cu_k, a.rows_q, a.rows_k, a.seqs, a.tokens, a.few,
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
      const Span x = span_of(a, it, split);
      s_span = x;
      if (it.tile >= 0 && x.cnt > 0) {  // the first loads need nobody else
        mbar_arrive_expect_tx(&bar_q, static_cast<uint32_t>(a.tokens * a.group) * 128);
        tma_load_3d(smem, &tmQ, &bar_q, 0, kvh * a.group, static_cast<int>(it.q0) + x.tok);
        mbar_arrive_expect_tx(&full_k[0], kTileBytes);
        tma_load_3d(ks, &tmK, &full_k[0], 0, kvh, static_cast<int>(it.k0) + x.j0 * kRows);
        tma_prefetch_desc(&tmV);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;  // columns: S 0, P 128, O 192
  const Item it = s_item;
  if (it.tile >= 0) {
    const int tok = s_span.tok, j0 = s_span.j0, cnt = s_span.cnt, shift = it.lk - it.lq;

    if (warp == 5) {
      // ---- loads
      bool ok = true;
      for (int jj = 0; jj < cnt && ok; ++jj) {
        const int s = jj % kKStages, sv = jj % kVStages;
        const int key = (j0 + jj) * kRows, row = static_cast<int>(it.k0) + key, valid = it.lk - key;
        uint8_t* vdst = vs + sv * kTileBytes;
        if (lane == 0) {
          if (jj >= kKStages) ok = mbar_wait(&empty_k[s], ((jj / kKStages) & 1u) ^ 1u);
          if (ok) {
            if (jj > 0) {  // the first one is on its way
              mbar_arrive_expect_tx(&full_k[s], kTileBytes);
              tma_load_3d(ks + s * kTileBytes, &tmK, &full_k[s], 0, kvh, row);
            }
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
            // every eighth pair on the FMA pipe (267 us with every fourth, 263 with none, 248)
            e = i % 8 == 7 ? ex2_fma(e) : make_float2(ex2(e.x), ex2(e.y));
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
        const bool none = top == -INFINITY && sum == sum;  // no key seen (here), and no NaN
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
  pdl_wait();  // what follows this kernel follows prompt_few_kernel, beside which it may run
}

// Few query rows per sequence and key head (single tokens while decoding): a tile of 128 rows would be nearly empty, and
// the work is to read K and V once. One CTA per (sequence, key head, split of the keys), every warp on its own, 32 keys at
// a time: eight lanes read a key's 128 bytes, four keys a load, so a lane has 8 of the 64 dimensions of every fourth key.
// 128 tokens over caches up to 1500, 20 heads, 498 MB: 87 us, 5.7 TB/s (with a key a lane each load touched 32 lines and
// the L1 bound it: 122 us; with 5 CTAs an SM 93). Scores are fp32 dot
// products, reduced over the eight lanes so that each lane ends with one key's; in P V the four groups of lanes sum their
// own keys until the end. V's loads are issued before the scores are computed. The warps' results are joined in shared
// memory. kR is 2 if the sequence has more than one row; those of more than two take several turns, those of more than
// a.few queries are left to the tiles.
constexpr int kFewWarps = 4;
struct FewRows {
  const void *q, *k, *v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
};
template <int kR>
struct FewShared {
  alignas(16) float q[kR][64];
  float top[kFewWarps][kR], sum[kFewWarps][kR];
  float2 o[kFewWarps][kR][32];
};
template <typename T, int kR>
__device__ __forceinline__ void few_rows(const FewRows& x, const PromptArgs& a, FewShared<kR>& sh, int64_t q0, int lq, int64_t k0,
                                         int lk, int kvh, int split) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, shift = lk - lq;
  const int rows = lq * a.group;  // (token, head of the group), tokens major
  // this warp's keys
  const int parts = a.splits * kFewWarps, part = split * kFewWarps + warp;
  const int tiles = (lk + 31) / 32;
  const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * part / parts);
  const int t1 = static_cast<int>(static_cast<int64_t>(tiles) * (part + 1) / parts);
  const int group = lane >> 3, at = lane & 7;  // of lanes, place in it
  const T* kb = static_cast<const T*>(x.k) + k0 * x.k_token + kvh * x.k_head + 8 * at;
  const T* vb = static_cast<const T*>(x.v) + k0 * x.v_token + kvh * x.v_head + 8 * at;

  for (int r0 = 0; r0 < rows; r0 += kR) {
    __syncthreads();
    for (int i = threadIdx.x; i < kR * 32; i += 32 * kFewWarps) {
      const int r = r0 + i / 32, d = i % 32 * 2;
      float2 f = make_float2(0.f, 0.f);
      if (r < rows)
        f = Type16<T>::unpack(*reinterpret_cast<const uint32_t*>(static_cast<const T*>(x.q) + (q0 + r / a.group) * x.q_token +
                                                                 (kvh * a.group + r % a.group) * x.q_head + d));
      sh.q[i / 32][d] = f.x;
      sh.q[i / 32][d + 1] = f.y;
    }
    __syncthreads();
    float top[kR], sum[kR], o[kR][8];
    int limit[kR];
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      top[r] = -INFINITY;
      sum[r] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[r][i] = 0.f;
      const int token = (r0 + r) / a.group;
      limit[r] = r0 + r >= rows ? -1 : a.causal ? min(lk - 1, token + shift) : lk - 1;
    }
    for (int t = t0; t < t1; ++t) {
      uint4 kw[8], vw[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = 32 * t + 4 * i + group;
        kw[i] = key < lk ? *reinterpret_cast<const uint4*>(kb + key * x.k_token) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = 32 * t + 4 * i + group;
        vw[i] = key < lk ? *reinterpret_cast<const uint4*>(vb + key * x.v_token) : make_uint4(0u, 0u, 0u, 0u);
      }
      const int key = 32 * t + 4 * at + group;  // whose score this lane ends with
      float p[kR];
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        const float4 qa = *reinterpret_cast<const float4*>(&sh.q[r][8 * at]);
        const float4 qb = *reinterpret_cast<const float4*>(&sh.q[r][8 * at + 4]);
        float s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 e = Type16<T>::unpack(kw[i].x), f = Type16<T>::unpack(kw[i].y);
          const float2 g = Type16<T>::unpack(kw[i].z), h = Type16<T>::unpack(kw[i].w);
          s[i] = fmaf(e.x, qa.x, fmaf(e.y, qa.y, fmaf(f.x, qa.z, f.y * qa.w))) +
                 fmaf(g.x, qb.x, fmaf(g.y, qb.y, fmaf(h.x, qb.z, h.y * qb.w)));
        }
        // sums over the eight lanes; each step halves the keys that a lane keeps
#pragma unroll
        for (int d = 4; d > 0; d >>= 1) {
          const bool upper = (at & d) != 0;
#pragma unroll
          for (int i = 0; i < d; ++i) {
            const float give = upper ? s[i] : s[i + d], keep = upper ? s[i + d] : s[i];
            s[i] = keep + __shfl_xor_sync(0xffffffffu, give, d);
          }
        }
        const float z = key <= limit[r] ? s[0] * a.scale_log2 : -INFINITY;
        const float m = fmaxf(top[r], warp_max(z));
        const float off = m == -INFINITY ? 0.f : -m;
        const float f = ex2(top[r] + off);
        p[r] = ex2(z + off);
        sum[r] = fmaf(sum[r], f, p[r]);  // this lane's keys
#pragma unroll
        for (int i = 0; i < 8; ++i) o[r][i] *= f;
        top[r] = m;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 e = Type16<T>::unpack(vw[i].x), f = Type16<T>::unpack(vw[i].y);
        const float2 g = Type16<T>::unpack(vw[i].z), h = Type16<T>::unpack(vw[i].w);
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          const float w = __shfl_sync(0xffffffffu, p[r], 8 * group + i);
          o[r][0] = fmaf(w, e.x, o[r][0]), o[r][1] = fmaf(w, e.y, o[r][1]);
          o[r][2] = fmaf(w, f.x, o[r][2]), o[r][3] = fmaf(w, f.y, o[r][3]);
          o[r][4] = fmaf(w, g.x, o[r][4]), o[r][5] = fmaf(w, g.y, o[r][5]);
          o[r][6] = fmaf(w, h.x, o[r][6]), o[r][7] = fmaf(w, h.y, o[r][7]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const float l = warp_sum(sum[r]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // over the four groups
        o[r][i] += __shfl_xor_sync(0xffffffffu, o[r][i], 8);
        o[r][i] += __shfl_xor_sync(0xffffffffu, o[r][i], 16);
      }
      if (group == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sh.o[warp][r][4 * at + i] = make_float2(o[r][2 * i], o[r][2 * i + 1]);
      }
      if (lane == 0) {
        sh.top[warp][r] = top[r];
        sh.sum[warp][r] = l;
      }
    }
    __syncthreads();
    for (int r = warp; r < kR && r0 + r < rows; r += kFewWarps) {
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) m = fmaxf(m, sh.top[w][r]);
      const float off = m == -INFINITY ? 0.f : -m;
      float l = 0.f;
      float2 e = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        const float f = ex2(sh.top[w][r] + off);
        const float2 y = sh.o[w][r][lane];
        l = fmaf(sh.sum[w][r], f, l);
        e = make_float2(fmaf(y.x, f, e.x), fmaf(y.y, f, e.y));
      }
      const bool none = l == 0.f;
      const float inv = none ? 0.f : 1.f / l;
      e = none ? make_float2(0.f, 0.f) : make_float2(e.x * inv, e.y * inv);
      const float lse = none ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      const int64_t row = q0 + (r0 + r) / a.group;
      const int head = kvh * a.group + (r0 + r) % a.group;
      if (a.splits > 1) {
        reinterpret_cast<float2*>(a.part_o + ((split * a.rows_q + row) * a.heads + head) * 64)[lane] = e;
        if (lane == 0) a.part_lse[(static_cast<int64_t>(split) * a.heads + head) * a.rows_q + row] = lse;
      } else {
        reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + row * a.out_token + head * a.out_head)[lane] =
            Type16<T>::pack(e.x, e.y);
        if (lane == 0 && a.lse != nullptr) a.lse[head * a.rows_q + row] = lse;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(32 * kFewWarps, 4) prompt_few_kernel(const FewRows x, const PromptArgs a) {
  __shared__ FewShared<2> sh;
  const int split = blockIdx.x % a.splits;
  const int kvh = blockIdx.x / a.splits % a.kv_heads;
  const int seq = blockIdx.x / a.splits / a.kv_heads;
  pdl_trigger();
  const int64_t q0 = a.cu_q[seq], q1 = a.cu_q[seq + 1], k0 = a.cu_k[seq], k1 = a.cu_k[seq + 1];
  if (q0 < 0 || q1 < q0 || q1 > a.rows_q || k0 < 0 || k1 < k0 || k1 > a.rows_k) {
    if (threadIdx.x == 0) prompt_flag(FW_DEVERR_BAD_INDEX);
    return;
  }
  if (q1 - q0 > a.few) return;
  const int lq = static_cast<int>(q1 - q0), lk = static_cast<int>(k1 - k0), rows = lq * a.group;
  if (rows <= 1)
    few_rows<T>(x, a, reinterpret_cast<FewShared<1>&>(sh), q0, lq, k0, lk, kvh, split);
  else
    few_rows<T>(x, a, sh, q0, lq, k0, lk, kvh, split);
}

// Whether `row` lies in a sequence that has been computed, by one warp. Every sequence is looked at, each by its own offsets: a
// search by bisection would stop at a sequence with bad offsets and miss the good one behind it. (Where keys are split there
// are at most 592 sequences.) Of those that tiles compute, one that begins before the end of a good one in front does not count.
// Many sequences of few rows are tried by bisection first (512 single tokens: 23.7 us a call in a graph without, 21.2), few are not
// (8: 10.9 us with, 10.2).
__device__ __forceinline__ bool row_is_computed(const PromptArgs& a, int64_t row, int lane) {
  if (a.seqs > 128) {
    int lo = 0, hi = a.seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (a.cu_q[mid] <= row)
        lo = mid;
      else
        hi = mid;
    }
    const int64_t q0 = a.cu_q[lo], q1 = a.cu_q[lo + 1];
    if (good_sequence(a, lo) && q0 <= row && row < q1 && q1 - q0 <= a.few) return true;
  }
  int reach = 0;  // furthest end of a good sequence so far
  constexpr int U = 4;  // turns of 32 whose loads are in flight together
  for (int b0 = 0; b0 < a.seqs; b0 += 32 * U) {
    int first[U], end[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = b0 + 32 * u + lane;
      first[u] = end[u] = 0;
      if (b < a.seqs && good_sequence(a, b)) first[u] = static_cast<int>(a.cu_q[b]), end[u] = static_cast<int>(a.cu_q[b + 1]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned holds = __ballot_sync(0xffffffffu, first[u] <= row && row < end[u]);
      if (first[u] == end[u]) end[u] = 0;
      if (holds != 0) {
        const int at = __ffs(holds) - 1;
        const int q0 = __shfl_sync(0xffffffffu, first[u], at), q1 = __shfl_sync(0xffffffffu, end[u], at);
        return q1 - q0 <= a.few || max(reach, __reduce_max_sync(0xffffffffu, lane < at ? end[u] : 0)) <= q0;
      }
      reach = max(reach, __reduce_max_sync(0xffffffffu, end[u]));
    }
  }
  return false;
}

// Joins the key splits of a (row, head), one warp each: o = sum_s exp(lse_s - lse) o_s.
template <typename T>
__global__ void __launch_bounds__(128) prompt_join_kernel(PromptArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int64_t row = i / a.heads;
  const int head = static_cast<int>(i % a.heads);
  // rows that belong to no sequence keep what they hold, and so do those of sequences that were left out above; the offsets are
  // the caller's, so the search need not wait
  const bool computed = i < a.rows_q * a.heads && row_is_computed(a, row, lane);
  pdl_wait();
  if (!computed) return;
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
// From sizes only (the offsets are on the device): rows of an average sequence and key head, and whether they are few
// enough for prompt_few_kernel. 64 sequences over caches up to 1500, 20 heads: one row 53 us, two 63, four 95; tiles of
// 128 rows 62 for any of them.
// The average says nothing of the longest: a sequence of more than kFewMost rows, a prompt that came in among single
// tokens, goes to the tiles all the same, in a launch beside the other (none where rows_q leaves no room for one). 600
// single tokens and a prompt of 600, keys up to 1500, 20 heads, 2.3 GB: 365 us, with all of it in tiles 541.
constexpr int kFewRows = 2, kFewMost = 32;
static int64_t average_rows(int64_t rows_q, int seqs, int group) {
  return seqs > 0 ? (rows_q + seqs - 1) / seqs * group : 0;
}
static bool few_rows(int64_t rows_q, int seqs, int group) { return average_rows(rows_q, seqs, group) <= kFewRows; }

// Splits of the keys: none when the query tiles fill the SMs; else as many as make four CTAs an SM, each with two key
// blocks (of 128 keys) of an average sequence at least.
static int prompt_splits(int64_t rows_q, int64_t rows_k, int seqs, int kv_heads, int group) {
  const int64_t items =
      (few_rows(rows_q, seqs, group) ? seqs : rows_q / (kRows / group) + seqs) * static_cast<int64_t>(kv_heads);
  const int64_t blocks = seqs > 0 ? (rows_k / seqs + kRows - 1) / kRows : 1;
  int64_t s = items > 0 ? 4 * 148 / items : 1;
  if (few_rows(rows_q, seqs, group))
    s = s * 2 > blocks ? blocks : s * 2;  // small CTAs
  else if (s > (blocks + 1) / 2)
    s = (blocks + 1) / 2;
  return static_cast<int>(s < 1 ? 1 : s > 64 ? 64 : s);
}

template <typename T>
static int run_tiles(const fw_rows_t& q, const fw_rows_t& k, const fw_rows_t& v, const PromptArgs& a, int64_t items,
                     cudaStream_t s) {
  FW_REQUIRE(items < (int64_t(1) << 31), FW_ERR_SHAPE, "prompt_attention: too many query tiles");
  CUtensorMap tq, tk, tv;
  // no keys at all: any valid address serves, nothing is read through it
  const bool keys = a.rows_k > 0;
  int rc = make_rows_map(&tq, Type16<T>::kMap, q.ptr, a.rows_q, a.heads, q.token, q.head, a.group, a.tokens);
  if (!rc) rc = keys ? make_rows_map(&tk, Type16<T>::kMap, k.ptr, a.rows_k, a.kv_heads, k.token, k.head, 1, kRows) : FW_OK;
  if (!rc) rc = keys ? make_rows_map(&tv, Type16<T>::kMap, v.ptr, a.rows_k, a.kv_heads, v.token, v.head, 1, kRows) : FW_OK;
  if (rc) return rc;
  auto kern = prompt_attn_kernel<T>;
  cudaError_t e = ensure_smem(kern, kFwdSmem);
  if (e == cudaSuccess)
    e = launch(kern, dim3(static_cast<unsigned>(items)), dim3(kFwdThreads), kFwdSmem, s, a.few > 0, tq, keys ? tk : tq,
               keys ? tv : tq, a);
  return launch_status(e, "prompt_attention");
}

template <typename T>
static int run_prompt(const fw_rows_t& q, const fw_rows_t& k, const fw_rows_t& v, PromptArgs a, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  int rc = FW_OK;
  const int64_t rows = average_rows(a.rows_q, a.seqs, a.group);
  const int64_t few = static_cast<int64_t>(a.seqs) * a.kv_heads * a.splits;
  if (rows <= kFewRows && few < (int64_t(1) << 31)) {
    a.few = kFewMost / a.group;
    const FewRows x{q.ptr, k.ptr, v.ptr, q.token, q.head, k.token, k.head, v.token, v.head};
    e = launch(prompt_few_kernel<T>, dim3(static_cast<unsigned>(few)), dim3(32 * kFewWarps), 0, s, false, x, a);
    rc = launch_status(e, "prompt_attention few rows");
    if (rc) return rc;
  }
  // sequences of more than a.few queries: rows_q / (few + 1) at most
  const int64_t longer = a.rows_q / (a.few + 1) < a.seqs ? a.rows_q / (a.few + 1) : a.seqs;
  const int64_t items = longer == 0 ? 0 : (a.rows_q / a.tokens + longer) * a.kv_heads * a.splits;
  if (items > 0) rc = run_tiles<T>(q, k, v, a, items, s);
  if (rc || a.splits == 1) return rc;
  e = launch(prompt_join_kernel<T>, dim3(static_cast<unsigned>((a.rows_q * a.heads + 3) / 4)), dim3(128), 0, s, true, a);
  return launch_status(e, "prompt_attention join");
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
