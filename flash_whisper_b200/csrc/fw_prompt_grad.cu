// Gradient of the attention over packed sequences (fw_prompt.cu).
//
//   delta_i = do_i . o_i      p_ij = exp(s_ij - lse_i)      ds_ij = p_ij (do_i . v_j - delta_i)
//   dv_j = sum_i p_ij do_i    dk_j = scale sum_i ds_ij q_i  dq_i = scale sum_j ds_ij k_j
// (dv and dk summed over the heads of the group). prompt_delta_kernel writes what the products need of lse, delta and
// |do| per row.
//
// prompt_grad_kernel is persistent, one CTA an SM; its CTAs draw work items of two kinds, so that nothing is summed by
// atomics and results do not vary: a key item has 128 keys of a key head and walks the queries (128 tokens of one head a
// step), a query item has 128 (token, head) rows and walks the keys (128 a step). The probabilities are computed in both.
//   first products:   X = A1 B1^T, Y = A2 B2^T       key item: A = K, V   B = Q, dO;    query item: A = Q, dO  B = K, V
//   second products:  key item: dV += P^T dO, dK += dS^T Q;      query item: dQ += dS K
// A1 and A2 stay in shared memory for the item, each step's B tile pair serves both products (K-major in the first,
// MN-major in the second). X, twice, and Y are in tensor memory; P and dS, the A operands of the second products, are
// written over X. 16 softmax warps (32 rows x 32 columns each) compute a step's exponentials from X and need Y only after
// them; Y of the next step is issued, by a warp of its own, as soon as Y has been read, and the second products and X of
// the step after the next once P and dS are there: a step's hand-overs hide behind the exponentials. Steps run on across
// items: the loads and the first products of the next item start while the results of the last one are read out (with one
// CTA per item 24 CTAs an SM spent 8 us each outside of their steps).
// Six sequences up to 4096, 32 heads on 8 (bf16): 611 to 704 us as the clocks allow, 0.55 to 0.63 PFLOP/s of what the
// formulas need, the special-function unit 46% and the tensor pipe 40% active. Tried and slower (611 on that box): steps of 64
// with two sets of X and Y and 8 warps on each (693), all products from one warp (674: its waits add to the products' time), A
// in tensor memory with P and dS over Y (715), the two halves of the warps taking turns at the exponentials (667), a quarter of
// the exponentials as polynomials on the FMA pipe (no change).
// fp16 range: P is kept times 2^8, and dS times 2^12 over the powers of two of the largest norm ||v|| (of the call) and of
// ||do|| (of the row in a query item, the largest of the call in a key item), so that gradients of any size keep their bits and
// none overflows: |do . v - delta| is at most twice the product of the norms, so what is kept stays below 2^15. (The largest
// elements bound it too, but 64 times as far off where one element is large.) bf16 needs neither.
#include "fw_prompt.cuh"

namespace fw {

constexpr int kStep = 128;  // B rows of a step
constexpr int kGradStages = 4;
constexpr uint32_t kGradStage = 2 * kTileBytes;
constexpr int kGradSmem = 4 * kTileBytes + kGradStages * kGradStage + 1024;  // two pairs of A, the stages
constexpr int kGradThreads = 32 * 19;  // 16 softmax warps, X and second products, loads, Y
constexpr int kDeltaBlocks = 592;
constexpr int kRing = 4;  // items known ahead; the first products look two steps, so at most two items, ahead

struct GradArgs {
  PromptArgs p;
  const void *o, *dout, *v;
  int64_t o_token, o_head, d_token, d_head, v_token, v_head;
  void *dq, *dk, *dv;
  int64_t dq_token, dq_head, dk_token, dk_head, dv_token, dv_head;
  // [heads][stat_rows]: log2 of P's factor - lse log2 e, and -delta, four rows of the first and then of the second at a
  // time; a sequence's rows start at stat_start()
  float* stat;
  int64_t stat_rows;
  float* norm;                   // fp16: [heads][stat_rows], the power of two that takes a row's ||do|| to [1, 2)
  float* largest;                // fp16: [2][kDeltaBlocks], largest ||do||^2 and ||v||^2 each block met
  unsigned* next;                // the next work item to be drawn
  int64_t key_items, all_items;  // key items come first: they are the longer ones
  float scale;
};

// First row of sequence `seq` in stat: a multiple of 4 (16 bytes at least), behind the previous sequence's rows.
__device__ __forceinline__ int64_t stat_start(int64_t q0, int seq) { return ((q0 + 3) / 4 + seq) * 4; }

__device__ __forceinline__ float* stat_at(const GradArgs& g, int head, int64_t row) {
  return g.stat + (head * g.stat_rows + row / 4 * 4) * 2 + row % 4;
}

// The power of two that takes the root of x, a sum of squares of fp16 numbers, into [1, 2); 1 for 0.
__device__ __forceinline__ float normalizer(float x) {
  const int e = static_cast<int>(__float_as_uint(x) >> 23) - 127;
  return x == 0.f ? 1.f : __uint_as_float(static_cast<uint32_t>(127 - (e >> 1)) << 23);
}

// The good sequence that holds `row` of those that `cu` (cu_q or cu_k) divides, -1 for none. A warp's lanes may ask for
// different rows, negative ones for nothing. Bisection; offsets out of order mislead it, and a good sequence behind them is
// found by looking at each. `ordered`: whether they are in order, -1 until it is needed.
__device__ __forceinline__ int sequence_at(const PromptArgs& a, const int64_t* cu, int64_t row, int* ordered, int lane) {
  const auto holds = [&](int b) { return good_sequence(a, b) && cu[b] <= row && row < cu[b + 1]; };
  int found = -1;
  if (row >= 0) {
    int lo = 0, hi = a.seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (cu[mid] <= row)
        lo = mid;
      else
        hi = mid;
    }
    if (holds(lo)) found = lo;
  }
  const bool lost = row >= 0 && found < 0;
  if (__any_sync(0xffffffffu, lost)) {
    if (*ordered < 0) {
      bool back = false;
#pragma unroll 8
      for (int b = lane; b < a.seqs; b += 32) back |= cu[b] > cu[b + 1];
      *ordered = !__any_sync(0xffffffffu, back);
    }
    if (lost && !*ordered) {
      for (int b = 0; b < a.seqs && found < 0; ++b)
        if (holds(b)) found = b;
    }
    __syncwarp();
  }
  return found;
}

// Sum of squares, of finite elements.
template <typename T>
__device__ __forceinline__ float square(uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = Type16<T>::unpack(w[i]);
    if (fabsf(x.x) < INFINITY) sum = fmaf(x.x, x.x, sum);
    if (fabsf(x.y) < INFINITY) sum = fmaf(x.y, x.y, sum);
  }
  return sum;
}

// fp16: a second half of the grid looks for the largest ||v|| (as a second loop of the same CTAs: 51 us for eight transcripts
// up to 448, 20 heads; so 49, and 46 without ||v||).
template <typename T>
__global__ void __launch_bounds__(256, 8) prompt_delta_kernel(GradArgs g) {
  __shared__ float s_max[8];
  pdl_trigger();
  if (blockIdx.x == 0 && threadIdx.x == 0) *g.next = 0u;
  const PromptArgs& a = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool values = !Type16<T>::kBf16 && blockIdx.x >= kDeltaBlocks;
  const int64_t first = ((blockIdx.x - (values ? kDeltaBlocks : 0)) * 8 + warp) * 4;
  constexpr int kUnits = kDeltaBlocks * 32;  // (row, head) pairs of a turn
  constexpr float kP = Type16<T>::kBf16 ? 0.f : 8.f;  // log2 of the factor that P carries
  float big = 0.f;
  int ordered = -1;
  if (values) {
    const int64_t units = a.rows_k * a.kv_heads;
    for (int64_t u0 = first; u0 < units; u0 += kUnits) {
      const int64_t u = u0 + (lane >> 3);
      const int64_t row = u < units ? u / a.kv_heads : -1;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (row >= 0)
        v = reinterpret_cast<const uint4*>(static_cast<const T*>(g.v) + row * g.v_token + u % a.kv_heads * g.v_head)[lane & 7];
      float sum = sequence_at(a, a.cu_k, row, &ordered, lane) >= 0 ? square<T>(v) : 0.f;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      big = fmaxf(big, sum);
    }
  } else {
    const int64_t units = a.rows_q * a.heads;
    for (int64_t u0 = first; u0 < units; u0 += kUnits) {
      const int64_t u = u0 + (lane >> 3);
      const int64_t row = u < units ? u / a.heads : -1;
      const int head = static_cast<int>(u % a.heads);
      const int seq = sequence_at(a, a.cu_q, row, &ordered, lane);  // rows of no sequence may hold anything
      float dot = 0.f, sum = 0.f;
      if (seq >= 0) {
        const uint4 d =
            reinterpret_cast<const uint4*>(static_cast<const T*>(g.dout) + row * g.d_token + head * g.d_head)[lane & 7];
        const uint4 o = reinterpret_cast<const uint4*>(static_cast<const T*>(g.o) + row * g.o_token + head * g.o_head)[lane & 7];
        const uint32_t dw[4] = {d.x, d.y, d.z, d.w}, ow[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = Type16<T>::unpack(dw[i]), y = Type16<T>::unpack(ow[i]);
          dot = fmaf(x.x, y.x, fmaf(x.y, y.y, dot));
        }
        if (!Type16<T>::kBf16) sum = square<T>(d);
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) {
        dot += __shfl_xor_sync(0xffffffffu, dot, o);
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
      }
      big = fmaxf(big, sum);
      if (seq >= 0 && (lane & 7) == 0) {
        const int64_t q0 = a.cu_q[seq], at = stat_start(q0, seq) + row - q0;
        float* st = stat_at(g, head, at);
        st[0] = kP - a.lse[head * a.rows_q + row] * kLog2;
        st[4] = -dot;
        if (!Type16<T>::kBf16) g.norm[head * g.stat_rows + at] = normalizer(sum);
      }
    }
  }
  if (Type16<T>::kBf16) return;
  big = warp_max(big);
  if (lane == 0) s_max[warp] = big;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < 8; ++w) big = fmaxf(big, s_max[w]);
    g.largest[blockIdx.x] = big;
  }
}

// One softmax warp's share of an item's steps: 32 of the 128 columns. kKeys: the statistics are per column, from the
// step's stage, else the row's own.
struct GradRow {
  int steps, per_head, begin;  // steps are numbered on from item to item: this one's are first .. first + steps - 1
  int lo0, hi0;     // columns [lo0, hi0) of the whole walk count for this row
  float off, del;   // of this row (query role): stat's two
  float c, norm;
  uint32_t tx, ty;  // tensor memory: X (the second one 128 columns on) and Y, this warp's columns and lanes
  uint64_t *x_full, *y_full, *y_free, *p_full, *full;
};
template <typename T, bool kKeys>
__device__ __forceinline__ bool grad_steps(const GradRow& g, int first, int h, const float (*stat)[2 * kStep], int lane) {
  const float2 c2 = make_float2(g.c, g.c), n2 = make_float2(g.norm, g.norm);
  int block = 0;  // j % per_head in the key role
  for (int j = first; j < first + g.steps; ++j) {
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
    uint32_t keep = 0;  // bit i: column i counts
    if (cut && hi > 0 && lo < 32) keep = (0xffffffffu >> (32 - min(hi, 32))) & (0xffffffffu << max(lo, 0));
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
        if (!(keep & (1u << i))) x[i] = 0u;
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
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(g.y_free);
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
        if (!(keep & (1u << i))) y[i] = 0u;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = Type16<T>::pack(__uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1]));
    tc_store16(tx + 16, p);
    tc_wait_store();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(g.p_full + (j & 1));
  }
  return true;
}

// A work item as every role reads it.
struct GradItem {
  int64_t q0, k0;
  int lq, lk;
  int first;                   // first key, or first token, of A
  int begin, per_head, steps;  // key item: token blocks from `begin` on for each head of the group
  int kvh, seq;
  int keys;  // the kind
  int end;   // no more items
};

// Where the warp that issues the products is in the sequence of steps.
struct GradCursor {
  int item = -1, left = 0, step = -1;  // item number; its steps behind this one; step number
  bool keys = false, fresh = false, last = false, end = false;

  // To the next step, once its item is known.
  __device__ __forceinline__ bool next(const GradItem* items, uint64_t* item_full) {
    if (left == 0) {
      ++item;
      if (!mbar_wait_warp(item_full + item % kRing, (item / kRing) & 1u)) return false;
      const GradItem& x = items[item % kRing];
      end = x.end != 0;
      if (end) return true;
      keys = x.keys != 0;
      left = x.steps;
      fresh = true;
    } else {
      fresh = false;
    }
    --left;
    last = left == 0;
    ++step;
    return true;
  }
};

template <typename T>
__global__ void __launch_bounds__(kGradThreads, 1)
    prompt_grad_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmD,
                       const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                       const __grid_constant__ CUtensorMap tmQa, const __grid_constant__ CUtensorMap tmDa, GradArgs g) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(16) float s_stat[kGradStages][2 * kStep];
  __shared__ __align__(8) uint64_t full[kGradStages], empty[kGradStages], landed, x_full[2], y_full, y_free, p_full[2],
      a_full[2], a_free[2], done, item_full[kRing], item_free[kRing];
  __shared__ uint32_t tmem_base_sh;
  __shared__ GradItem s_item[kRing];
  __shared__ float s_norm, s_norm_v;  // powers of two for the call's largest ||do|| and ||v||, the second for the latter alone
  const PromptArgs& a = g.p;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);  // A1 | A2 of even and of odd items, then the stages
  const int warp = warp_index(), lane = threadIdx.x & 31;

  if (warp == 16) {
    tmem_alloc(&tmem_base_sh, 512);
    tmem_relinquish();
  }
  if (warp == 17 && lane == 0) {
    for (int i = 0; i < kGradStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&landed, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&x_full[i], 1);  // X of an even or odd step is in tensor memory
      // P and dS of an even or odd step are there. One barrier for both would not do: a warp has given Y back before it
      // stores dS, so another could run ahead to the next step and arrive in its place. Its next arrival on the barrier of
      // the same parity follows x_full of two steps on, which is issued only after this step's sixteen have been waited for.
      mbar_init(&p_full[i], 16);
      mbar_init(&a_full[i], 1);  // A1 and A2 of an even or odd item have landed
      mbar_init(&a_free[i], 2);  // its X and its Y are done
    }
    mbar_init(&y_full, 1);   // Y is in tensor memory
    mbar_init(&y_free, 16);  // it has been read
    mbar_init(&done, 1);     // an item's results are
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_free[i], 18);  // every role but the loads has read the entry for the last time
    }
    mbar_fence_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // prompt_delta_kernel runs beside all this and the first loads, up to here for those who read what it writes
  if (warp < 17) {
    pdl_wait();
    if (!Type16<T>::kBf16) {
      if (warp == 16) {
        float m = 0.f, v = 0.f;
        for (int i = lane; i < kDeltaBlocks; i += 32) {
          m = fmaxf(m, g.largest[i]);
          v = fmaxf(v, g.largest[kDeltaBlocks + i]);
        }
        m = warp_max(m);
        v = warp_max(v);
        if (lane == 0) s_norm_v = normalizer(v), s_norm = normalizer(m) * s_norm_v;
        __syncwarp();
      }
      asm volatile("bar.sync 1, 544;" ::: "memory");
    }
  }
  const uint32_t tmem = tmem_base_sh;  // columns: X 0 and 128, Y 256, dV 384, dK or dQ 448

  if (warp == 17) {
    // ---- items and loads
    bool ok = true, end = false;
    uint32_t cut = 0;  // tiles that end inside a step so far
    int step = 0;
    // The first item is this CTA's by its number; the next ones are drawn while the one before is being loaded.
    unsigned ahead = blockIdx.x;
    bool waited = false;
    auto draw = [&] {
      if (!waited) pdl_wait();  // the counter, and the statistics, are prompt_delta_kernel's
      waited = true;
      if (lane == 0) ahead = gridDim.x + atomicAdd(g.next, 1u);
    };
    for (int n = 0; ok && !end; ++n) {
      // The next item with something to do. Rows without a step (keys that no query sees, queries that see no key) have
      // zero gradients, written here.
      GradItem x;
      while (true) {
        const int64_t index = __shfl_sync(0xffffffffu, ahead, 0);
        x.end = index >= g.all_items;
        if (x.end) break;
        x.keys = index < g.key_items;
        const int in = static_cast<int>(x.keys ? index : index - g.key_items);
        x.kvh = in % a.kv_heads;
        const Item it = x.keys ? find_item(a.cu_k, a.cu_q, a.rows_k, a.rows_q, a.seqs, kRows, 0, in / a.kv_heads, lane)
                               : find_item(a.cu_q, a.cu_k, a.rows_q, a.rows_k, a.seqs, a.tokens, 0, in / a.kv_heads, lane);
        if (it.tile < 0) {
          draw();
          continue;
        }
        x.seq = it.seq;
        x.q0 = x.keys ? it.k0 : it.q0, x.lq = x.keys ? it.lk : it.lq;  // find_item was asked with q and k swapped
        x.k0 = x.keys ? it.q0 : it.k0, x.lk = x.keys ? it.lq : it.lk;
        const int shift = x.lk - x.lq;
        if (x.keys) {
          x.first = it.tile * kRows;
          x.begin = a.causal ? max(0, x.first - shift) / kStep : 0;
          x.per_head = max(0, (x.lq + kStep - 1) / kStep - x.begin);
          x.steps = x.per_head * a.group;
        } else {
          const int tiles = (x.lq + a.tokens - 1) / a.tokens;
          x.first = (a.causal ? tiles - 1 - it.tile : it.tile) * a.tokens;  // causal: the longest first
          const int last = min(x.lq, x.first + a.tokens) - 1;
          x.begin = 0;
          x.per_head = x.steps = ((a.causal ? max(0, min(x.lk, last + shift + 1)) : x.lk) + kStep - 1) / kStep;
        }
        if (x.steps > 0) break;
        const int rows = x.keys ? min(kRows, x.lk - x.first) : min(a.tokens, x.lq - x.first) * a.group;
        for (int i = lane; i < rows * 8; i += 32) {
          const int r = i >> 3, c = (i & 7) * 8;
          if (x.keys) {
            const int64_t row = x.k0 + x.first + r;
            *reinterpret_cast<uint4*>(static_cast<T*>(g.dk) + row * g.dk_token + x.kvh * g.dk_head + c) =
                make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(static_cast<T*>(g.dv) + row * g.dv_token + x.kvh * g.dv_head + c) =
                make_uint4(0u, 0u, 0u, 0u);
          } else {
            const int64_t row = x.q0 + x.first + r / a.group;
            *reinterpret_cast<uint4*>(static_cast<T*>(g.dq) + row * g.dq_token +
                                      (x.kvh * a.group + r % a.group) * g.dq_head + c) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        draw();
      }
      end = x.end != 0;
      if (n >= kRing) ok = mbar_wait_warp(&item_free[n % kRing], ((n / kRing) & 1u) ^ 1u);
      if (!ok) break;
      if (lane == 0) {
        s_item[n % kRing] = x;
        mbar_arrive(&item_full[n % kRing]);
      }
      __syncwarp();
      if (end) break;

      // A1 and A2; rows behind the sequence (or behind the tile) give rows that are not stored
      if (n >= 2) ok = mbar_wait_warp(&a_free[n & 1], ((n >> 1) & 1u) ^ 1u);
      if (!ok) break;
      if (lane == 0) {
        uint8_t* dst = smem + (n & 1) * 2 * kTileBytes;
        uint64_t* bar = &a_full[n & 1];
        mbar_arrive_expect_tx(bar, x.keys ? 2 * kTileBytes : static_cast<uint32_t>(2 * a.tokens * a.group) * 128);
        const int row = static_cast<int>(x.keys ? x.k0 : x.q0) + x.first;
        tma_load_3d(dst, x.keys ? &tmK : &tmQa, bar, 0, x.keys ? x.kvh : x.kvh * a.group, row);
        tma_load_3d(dst + kTileBytes, x.keys ? &tmV : &tmDa, bar, 0, x.keys ? x.kvh : x.kvh * a.group, row);
      }
      int block = x.begin, head = x.keys ? x.kvh * a.group : x.kvh;
      for (int j = 0; j < x.steps && ok; ++j, ++step) {
        const int s = step % kGradStages;
        const int at = block * kStep;
        const int valid = (x.keys ? x.lq : x.lk) - at;
        const int row = static_cast<int>(x.keys ? x.q0 : x.k0) + at;
        uint8_t* dst = smem + 4 * kTileBytes + s * kGradStage;
        if (step >= kGradStages) ok = mbar_wait_warp(&empty[s], ((step / kGradStages) & 1u) ^ 1u);
        if (!ok) break;
        uint64_t* bar = valid >= kStep ? &full[s] : &landed;
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, kGradStage + (x.keys ? kStep * 8 : 0));
          tma_load_3d(dst, x.keys ? &tmQ : &tmK, bar, 0, head, row);
          tma_load_3d(dst + kTileBytes, x.keys ? &tmD : &tmV, bar, 0, head, row);
        }
        __syncwarp();
        if (j == 0) draw();
        if (x.keys && lane == 0) bulk_g2s(s_stat[s], stat_at(g, head, stat_start(x.q0, x.seq) + at), kStep * 8, bar);
        __syncwarp();
        if (valid < kStep) {
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
        if (++block == x.begin + x.per_head) block = x.begin, ++head;
      }
    }
    if (!ok && lane == 0) prompt_flag(FW_DEVERR_TIMEOUT);
  } else if (warp == 16) {
    // ---- second products, and X of the step after the next over their P and dS (the whole warp runs the loop, one lane
    // issues)
    constexpr uint32_t idesc_x = make_idesc(kRows, kStep, Type16<T>::kBf16, false, false);
    constexpr uint32_t idesc_o = make_idesc(kRows, 64, Type16<T>::kBf16, false, true);
    const uint32_t b_base = base + 4 * kTileBytes;
    GradCursor cx, cs;
    bool ok = true;
    for (int j = -2; ok; ++j) {
      const uint32_t x = tmem + 128 * (j & 1);
      if (j >= 0) {
        ok = cs.next(s_item, item_full);
        if (!ok || cs.end) break;
        ok = mbar_wait_warp(&p_full[j & 1], (j >> 1) & 1u);
        if (!ok) break;
        tc_fence_after();
        const uint64_t b1 = sw128_mn_desc(b_base + j % kGradStages * kGradStage, kTileBytes),
                       b2 = b1 + (kTileBytes >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {  // warp group g left its 32 columns of P and dS from 32 g and 32 g + 16 on
            const uint32_t p = x + 32 * (kk >> 1) + 8 * (kk & 1);
            if (cs.keys) tc_mma_ta(tmem + 384, p, b2 + 128 * kk, idesc_o, !cs.fresh || kk != 0 ? 1u : 0u);
            tc_mma_ta(tmem + 448, p + 16, b1 + 128 * kk, idesc_o, !cs.fresh || kk != 0 ? 1u : 0u);
          }
          tc_commit(&empty[j % kGradStages]);
          if (cs.last) tc_commit(&done);
        }
        __syncwarp();
        if (cs.last && lane == 0) mbar_arrive(&item_free[cs.item % kRing]);
      }
      if (cx.end) continue;
      ok = cx.next(s_item, item_full);
      if (!ok || cx.end) continue;
      if (cx.fresh) ok = mbar_wait_warp(&a_full[cx.item & 1], (cx.item >> 1) & 1u);
      if (ok) ok = mbar_wait_warp(&full[(j + 2) % kGradStages], ((j + 2) / kGradStages) & 1u);
      if (!ok) break;
      tc_fence_after();
      const uint64_t a1 = sw128_desc(base + (cx.item & 1) * 2 * kTileBytes);
      const uint64_t b1 = sw128_desc(b_base + (j + 2) % kGradStages * kGradStage);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) tc_mma_f16(x, a1 + 2 * kk, b1 + 2 * kk, idesc_x, kk != 0 ? 1u : 0u);
        tc_commit(&x_full[j & 1]);
        if (cx.last) tc_commit(&a_free[cx.item & 1]);
      }
      __syncwarp();
    }
    if (!ok && lane == 0) prompt_flag(FW_DEVERR_TIMEOUT);
  } else if (warp == 18) {
    // ---- Y
    constexpr uint32_t idesc = make_idesc(kRows, kStep, Type16<T>::kBf16, false, false);
    GradCursor c;
    bool ok = true;
    while (true) {
      ok = c.next(s_item, item_full);
      if (!ok || c.end) break;
      const int j = c.step, s = j % kGradStages;
      if (c.fresh) ok = mbar_wait_warp(&a_full[c.item & 1], (c.item >> 1) & 1u);
      if (ok) ok = mbar_wait_warp(&full[s], (j / kGradStages) & 1u);
      if (ok && j > 0) ok = mbar_wait_warp(&y_free, (j - 1) & 1u);
      if (!ok) break;
      tc_fence_after();
      const uint64_t a2 = sw128_desc(base + (c.item & 1) * 2 * kTileBytes + kTileBytes);
      const uint64_t b2 = sw128_desc(base + 4 * kTileBytes + s * kGradStage + kTileBytes);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) tc_mma_f16(tmem + 256, a2 + 2 * kk, b2 + 2 * kk, idesc, kk != 0 ? 1u : 0u);
        tc_commit(&y_full);
        if (c.last) tc_commit(&a_free[c.item & 1]);
      }
      __syncwarp();
      if (c.last && lane == 0) mbar_arrive(&item_free[c.item % kRing]);
    }
    if (!ok && lane == 0) prompt_flag(FW_DEVERR_TIMEOUT);
  } else {
    // ---- softmax: thread = row of A; warps 4 g .. 4 g + 3 work on columns 32 g .. + 31 of a step
    const int grp = warp >> 2;
    const int r = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    int step = 0;
    bool ok = true;
    for (int n = 0; ok; ++n) {
      ok = mbar_wait_warp(&item_full[n % kRing], (n / kRing) & 1u);
      if (!ok) break;
      const GradItem it = s_item[n % kRing];
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_free[n % kRing]);
      if (it.end) break;
      const bool keys = it.keys != 0;
      const int shift = it.lk - it.lq;
      const int token = keys ? 0 : it.first + r / a.group;
      const int head = keys ? it.kvh : it.kvh * a.group + r % a.group;
      const bool live = keys ? it.first + r < it.lk : r < a.tokens * a.group && token < it.lq;
      const int64_t row = keys ? it.k0 + it.first + r : it.q0 + token;
      GradRow gr;
      gr.steps = it.steps, gr.per_head = it.per_head, gr.begin = it.begin;
      gr.c = a.scale_log2;
      gr.off = gr.del = 0.f;
      gr.norm = 1.f;  // the factor of dS besides P's
      if (!Type16<T>::kBf16 && keys) gr.norm = 16.f * s_norm;
      if (!keys && live) {
        const int64_t at = stat_start(it.q0, it.seq) + token;
        const float* st = stat_at(g, head, at);
        gr.off = st[0];
        gr.del = st[4];
        if (!Type16<T>::kBf16) gr.norm = 16.f * s_norm_v * g.norm[head * g.stat_rows + at];
      }
      gr.tx = tmem + lanes + 32 * grp;
      gr.ty = tmem + lanes + 256 + 32 * grp;
      gr.x_full = x_full, gr.y_full = &y_full, gr.y_free = &y_free, gr.p_full = p_full;
      gr.full = full;
      if (keys) {
        gr.hi0 = it.lq;
        gr.lo0 = a.causal ? it.first + r - shift : 0;
        ok = grad_steps<T, true>(gr, step, grp, s_stat, lane);
      } else {
        gr.lo0 = 0;
        gr.hi0 = (a.causal ? min(it.lk - 1, token + shift) : it.lk - 1) + 1;
        ok = grad_steps<T, false>(gr, step, grp, s_stat, lane);
      }
      step += it.steps;
      if (ok) ok = mbar_wait_warp(&done, n & 1u);
      // ---- results: 32 columns each of dK (groups 0, 1) and dV (2, 3), or of dQ (0, 1)
      if (ok && (keys || grp < 2)) {
        tc_fence_after();
        const bool dv = grp >= 2;
        uint32_t x[32];
        tc_load32(tmem + lanes + (dv ? 384 : 448) + 32 * (grp & 1), x);
        tc_wait_ld();
        tc_fence_before();
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
              w[k] = Type16<T>::pack(__uint_as_float(x[e]) * f, __uint_as_float(x[e + 1]) * f);
            }
            reinterpret_cast<uint4*>(dst)[i] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) prompt_flag(FW_DEVERR_TIMEOUT);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 16) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------------------------------------
// Host side
template <typename T>
static int run_prompt_grad(const fw_rows_t& q, const fw_rows_t& k, const fw_rows_t& v, const fw_rows_t& d, GradArgs g,
                           cudaStream_t s) {
  const PromptArgs& a = g.p;
  const int64_t query_items = a.rows_q > 0 ? (a.rows_q / a.tokens + a.seqs) * a.kv_heads : 0;
  g.key_items = a.rows_k > 0 ? (a.rows_k / kRows + a.seqs) * a.kv_heads : 0;
  g.all_items = g.key_items + query_items;
  FW_REQUIRE(g.all_items < (int64_t(1) << 31), FW_ERR_SHAPE, "prompt_attention_grad: too many tiles");
  if (g.all_items == 0) return FW_OK;
  cudaError_t e = launch(prompt_delta_kernel<T>, dim3(Type16<T>::kBf16 ? kDeltaBlocks : 2 * kDeltaBlocks), dim3(256), 0, s,
                         false, g);
  int rc = launch_status(e, "prompt_attention_grad delta");
  if (rc) return rc;
  CUtensorMap tq{}, td{}, tk{}, tv{}, tqa{}, tda{};
  if (a.rows_q > 0) {
    rc = make_rows_map(&tq, Type16<T>::kMap, q.ptr, a.rows_q, a.heads, q.token, q.head, 1, kStep);
    if (!rc) rc = make_rows_map(&td, Type16<T>::kMap, d.ptr, a.rows_q, a.heads, d.token, d.head, 1, kStep);
    if (!rc) rc = make_rows_map(&tqa, Type16<T>::kMap, q.ptr, a.rows_q, a.heads, q.token, q.head, a.group, a.tokens);
    if (!rc) rc = make_rows_map(&tda, Type16<T>::kMap, d.ptr, a.rows_q, a.heads, d.token, d.head, a.group, a.tokens);
  }
  if (!rc && a.rows_k > 0) {
    rc = make_rows_map(&tk, Type16<T>::kMap, k.ptr, a.rows_k, a.kv_heads, k.token, k.head, 1, kStep);
    if (!rc) rc = make_rows_map(&tv, Type16<T>::kMap, v.ptr, a.rows_k, a.kv_heads, v.token, v.head, 1, kStep);
  }
  if (rc) return rc;
  if (a.rows_q == 0) tq = tk, td = tv, tqa = tk, tda = tv;  // nothing is read through them
  if (a.rows_k == 0) tk = tq, tv = td;
  auto kern = prompt_grad_kernel<T>;
  e = ensure_smem(kern, kGradSmem);
  if (e == cudaSuccess) {
    const int64_t grid = g.all_items < num_sms() ? g.all_items : num_sms();
    e = launch(kern, dim3(static_cast<unsigned>(grid)), dim3(kGradThreads), kGradSmem, s, true, tq, td, tk, tv, tqa, tda,
               g);
  }
  return launch_status(e, "prompt_attention_grad");
}

static int64_t grad_stat_rows(int64_t rows_q, int seqs) {  // room for a step's copy behind the last row
  return (rows_q + 3) / 4 * 4 + 4 * static_cast<int64_t>(seqs) + 4 + kStep;
}

unsigned int read_prompt_grad_errors(bool clear) {
  unsigned int v = 0, zero = 0;
  cudaMemcpyFromSymbol(&v, g_fw_dev_error, sizeof(v));
  if (clear && v) cudaMemcpyToSymbol(g_fw_dev_error, &zero, sizeof(zero));
  return v;
}

}  // namespace fw

using namespace fw;

extern "C" {

int fw_prompt_attention_grad_workspace(int64_t rows_q, int64_t rows_k, int seqs, int heads, int kv_heads,
                                       int64_t* bytes) {
  FW_REQUIRE(bytes != nullptr, FW_ERR_NULL, "prompt_attention_grad_workspace: bytes is NULL");
  int rc = check_prompt("prompt_attention_grad", bytes, bytes, seqs, rows_q, rows_k, heads, kv_heads, 1.f, FW_F16);
  if (rc) return rc;
  *bytes = (2 * kDeltaBlocks + 4) * 4 + heads * grad_stat_rows(rows_q, seqs) * 12;
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
  g.o = out->ptr, g.o_token = out->token, g.o_head = out->head;
  g.dout = dout->ptr, g.d_token = dout->token, g.d_head = dout->head;
  g.v = v->ptr, g.v_token = v->token, g.v_head = v->head;
  g.dq = dq->ptr, g.dq_token = dq->token, g.dq_head = dq->head;
  g.dk = dk->ptr, g.dk_token = dk->token, g.dk_head = dk->head;
  g.dv = dv->ptr, g.dv_token = dv->token, g.dv_head = dv->head;
  g.largest = static_cast<float*>(workspace);
  g.next = reinterpret_cast<unsigned*>(g.largest + 2 * kDeltaBlocks);
  g.stat = g.largest + 2 * kDeltaBlocks + 4;
  g.stat_rows = grad_stat_rows(rows_q, seqs);
  g.norm = g.stat + 2 * heads * g.stat_rows;
  g.scale = scale;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == FW_F16 ? run_prompt_grad<half>(*q, *k, *v, *dout, g, s)
                         : run_prompt_grad<__nv_bfloat16>(*q, *k, *v, *dout, g, s);
}

}  // extern "C"
