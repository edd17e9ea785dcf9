// Token embedding of whole (packed) transcripts and its gradient.
//
// Forward: out_i = T(scale E[id_i] + P[pos_i]), fp32 arithmetic, one rounding. One warp per row with 16-byte
// accesses; bound by HBM (32749 rows of 1280 bf16, 168 MB: 33 us a call, 5.1 TB/s).
//
// Gradient: dE[v] = scale sum_{i: id_i = v} dout_i, the sum in fp32 in a fixed order. Tokens repeat a lot (text
// is close to a Zipf law), so the rows of one token are brought together by a stable sort instead of adding them
// with atomics, whose order would change the result from run to run:
//   1. embed_sort_kernel: one cluster sorts (id, row) by id, an LSD radix sort of 8 bits a pass whose digit counts are
//      exchanged over distributed shared memory. It needs 8 SMs and is latency, so
//   2. embed_fill_kernel, which writes the zero rows of the dense gradient, runs beside it (it waits for the sort only
//      at its end, which keeps the order for what follows). Each CTA finds the ids that occur in its range of the
//      vocabulary by reading the id list itself (L2).
//   3. embed_sum_kernel: equal chunks of the sorted list, so a frequent token costs no CTA more than a rare one; a
//      run of equal ids inside a chunk is written at once, a run that crosses a chunk's end leaves fp32 partials.
//   4. embed_merge_kernel: adds the partials of each crossing run in chunk order.
// Bound by HBM (the gradient is written once, dout read once) and, for few tokens, by the sort's latency: 32749 tokens over
// 51866 rows of 1280 (bf16, 217 MB) 67 us, 3.2 TB/s (sort 22 and zero rows 23 side by side, sums 29, crossing runs 12);
// 3584 tokens (fp16, 142 MB) 37 us.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "fw_common.cuh"
#include "fw_host.h"

namespace fw {

namespace cg = cooperative_groups;

FW_DEFINE_ERROR_WORD();

__device__ __forceinline__ void embed_flag(unsigned bits) { atomicOr(&g_fw_dev_error, bits); }

__device__ __forceinline__ float to_f(half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ half from_f<half>(float v) {
  return __float2half(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16(v);
}
template <>
__device__ __forceinline__ float from_f<float>(float v) {
  return v;
}

// VEC consecutive elements as one access: 16 bytes where rows allow it, one element otherwise.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// ------------------------------------------------------------------------------------------------
// Forward
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_scaled_kernel(const T* __restrict__ embed, const T* __restrict__ pos,
                                                           const int64_t* __restrict__ ids,
                                                           const int64_t* __restrict__ positions, T* __restrict__ out,
                                                           int n, int vocab, int max_pos, int hidden, float scale) {
  using P = Pack<T, VEC>;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);  // may pass 2^31 at the end
  const int lane = threadIdx.x & 31;
  if (row >= n) return;
  int64_t id = ids[row], at = pos != nullptr ? positions[row] : 0;
  if (id < 0 || id >= vocab || (pos != nullptr && (at < 0 || at >= max_pos))) {
    if (lane == 0) embed_flag(FW_DEVERR_BAD_INDEX);
    id = id < 0 ? 0 : (id >= vocab ? vocab - 1 : id);
    at = at < 0 ? 0 : (at >= max_pos ? max_pos - 1 : at);
  }
  const P* e = reinterpret_cast<const P*>(embed + static_cast<size_t>(id) * hidden);
  const P* q = reinterpret_cast<const P*>(pos + (pos != nullptr ? static_cast<size_t>(at) * hidden : 0));
  P* o = reinterpret_cast<P*>(out + static_cast<size_t>(row) * hidden);
  const int packs = hidden / VEC;
  constexpr int U = 5;  // 5 x 32 lanes x 16 bytes = one row of 1280 16-bit elements in flight
  for (int i0 = lane; i0 < packs; i0 += 32 * U) {
    P a[U], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + 32 * u < packs) a[u] = e[i0 + 32 * u];
    if (pos != nullptr) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + 32 * u < packs) b[u] = q[i0 + 32 * u];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + 32 * u >= packs) continue;
      P r;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float x = to_f(a[u].v[j]);
        r.v[j] = from_f<T>(pos != nullptr ? fmaf(x, scale, to_f(b[u].v[j])) : x * scale);
      }
      o[i0 + 32 * u] = r;
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Gradient, steps 1 and 2: sort, zero rows
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortCtas = 8;  // the sorting cluster (portable size)
constexpr int kFillThreads = 1024;
constexpr int kFillRows = 32 * kFillThreads;  // vocabulary rows one CTA can mark in its shared bitmap

struct SortParams {
  const int64_t* ids;
  uint32_t *keys[2], *rows[2];  // ping-pong buffers [n]; the result lands in keys[passes & 1]
  int n, vocab, passes;
  int64_t padding;
  unsigned* crossing;  // [0]: how many chunks are listed behind it
};

__device__ __forceinline__ void cluster_sync_all() {  // release / acquire at cluster scope
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A token's key: its id, or `vocab` (sorted behind every row) for padding and ids out of range.
__device__ __forceinline__ uint32_t sort_key(const SortParams& p, int64_t id, bool flag) {
  if (id < 0 || id >= p.vocab) {
    if (flag && (id != p.padding || id == -1)) embed_flag(FW_DEVERR_BAD_INDEX);
    return static_cast<uint32_t>(p.vocab);
  }
  return id == p.padding ? static_cast<uint32_t>(p.vocab) : static_cast<uint32_t>(id);
}

// Zero rows of the gradient where no token names them, each CTA a range of the vocabulary.
__global__ void __launch_bounds__(kFillThreads) embed_fill_kernel(SortParams p, uint8_t* dembed, int64_t row_bytes,
                                                                  bool wide) {
  __shared__ uint32_t bits[kFillThreads];
  pdl_trigger();
  const int per = (p.vocab + gridDim.x - 1) / gridDim.x;
  const int end = min(p.vocab, (static_cast<int>(blockIdx.x) + 1) * per);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int v0 = blockIdx.x * per; v0 < end; v0 += kFillRows) {
    const int v1 = min(end, v0 + kFillRows);
    bits[threadIdx.x] = 0u;
    __syncthreads();
    constexpr int U = 8;
    for (int i0 = threadIdx.x; i0 < p.n; i0 += U * kFillThreads) {
      int64_t id[U];
#pragma unroll
      for (int u = 0; u < U; ++u) id[u] = i0 + u * kFillThreads < p.n ? p.ids[i0 + u * kFillThreads] : -1;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (id[u] >= v0 && id[u] < v1 && id[u] != p.padding)
          atomicOr(&bits[(id[u] - v0) >> 5], 1u << ((id[u] - v0) & 31));
    }
    __syncthreads();
    for (int v = v0 + warp; v < v1; v += kFillThreads / 32) {
      if ((bits[(v - v0) >> 5] >> ((v - v0) & 31)) & 1u) continue;
      uint8_t* row = dembed + static_cast<int64_t>(v) * row_bytes;
      if (wide) {
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
        for (int64_t i = lane; i < row_bytes / 16; i += 32) reinterpret_cast<uint4*>(row)[i] = zero;
      } else {
        for (int64_t i = lane; i < row_bytes / 2; i += 32) reinterpret_cast<uint16_t*>(row)[i] = 0;
      }
    }
    __syncthreads();
  }
  pdl_wait();  // what follows this kernel follows the sort
}

__global__ void __launch_bounds__(kSortThreads, 1) embed_sort_kernel(SortParams p) {
  __shared__ uint32_t s_hist[kSortWarps][256];  // per warp: counts, then next positions within this CTA
  __shared__ uint32_t s_total[256], s_base[256], s_scan[8];
  pdl_trigger();
  if (blockIdx.x == 0 && threadIdx.x == 0) p.crossing[0] = 0u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = cluster.num_blocks();
  const int rank = cluster.block_rank();
  // this warp's contiguous share [begin, end) of the list, a whole number of 32-element steps
  const int steps = (p.n + 32 * kSortWarps * ctas - 1) / (32 * kSortWarps * ctas);
  const int64_t begin64 = (static_cast<int64_t>(rank) * kSortWarps + warp) * steps * 32;
  const int begin = static_cast<int>(begin64 < p.n ? begin64 : p.n);
  const int end = static_cast<int>(begin64 + steps * 32 < p.n ? begin64 + steps * 32 : p.n);
  constexpr int U = 4;  // steps whose loads are in flight together

  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = 8 * pass;
    const uint32_t* kin = p.keys[pass & 1];
    const uint32_t* rin = p.rows[pass & 1];
    uint32_t* kout = p.keys[(pass + 1) & 1];
    uint32_t* rout = p.rows[(pass + 1) & 1];
    for (int d = lane; d < 256; d += 32) s_hist[warp][d] = 0u;
    __syncwarp();
    for (int i0 = begin + lane; i0 < end; i0 += 32 * U) {
      uint32_t k[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + 32 * u < end) k[u] = pass == 0 ? sort_key(p, p.ids[i0 + 32 * u], true) : __ldcg(kin + i0 + 32 * u);
#pragma unroll
      for (int u = 0; u < U; ++u)  // counts only: their order is of no account
        if (i0 + 32 * u < end) atomicAdd(&s_hist[warp][(k[u] >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid < 256) {  // digit tid: exclusive prefix over this CTA's warps
      uint32_t sum = 0;
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = s_hist[w][tid];
        s_hist[w][tid] = sum;
        sum += c;
      }
      s_total[tid] = sum;
    }
    cluster_sync_all();  // every CTA's totals are there
    uint32_t before = 0, all = 0, incl = 0;
    if (tid < 256) {
#pragma unroll
      for (int r = 0; r < kSortCtas; ++r) {
        const uint32_t c = r < ctas ? *cluster.map_shared_rank(&s_total[tid], r) : 0u;
        all += c;
        before += r < rank ? c : 0u;
      }
      incl = all;  // inclusive scan over the digits: within warps, then across the 8 warps
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
      }
      if (lane == 31) s_scan[warp] = incl;
    }
    __syncthreads();
    if (tid < 256) {
      uint32_t pre = 0;
      for (int w = 0; w < warp; ++w) pre += s_scan[w];
      s_base[tid] = pre + incl - all + before;
    }
    __syncthreads();
    for (int i0 = begin; i0 < end; i0 += 32 * U) {
      uint32_t k[U], r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + 32 * u + lane;
        k[u] = r[u] = 0;
        if (i < end) {
          k[u] = pass == 0 ? sort_key(p, p.ids[i], false) : __ldcg(kin + i);
          r[u] = pass == 0 ? static_cast<uint32_t>(i) : __ldcg(rin + i);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i0 + 32 * u >= end) break;
        const bool live = i0 + 32 * u + lane < end;
        const uint32_t d = live ? (k[u] >> shift) & 255u : 256u;  // lanes behind the end form a group of their own
        const unsigned peers = __match_any_sync(0xffffffffu, d);
        const int below = __popc(peers & ((1u << lane) - 1u));
        if (live) {
          const uint32_t at = s_base[d] + s_hist[warp][d] + below;
          __stcg(kout + at, k[u]);
          __stcg(rout + at, r[u]);
        }
        __syncwarp();
        if (live && below == 0) s_hist[warp][d] += __popc(peers);
        __syncwarp();
      }
    }
    cluster_sync_all();  // the pass's output is visible, and no CTA still reads another's totals
  }
}

// ------------------------------------------------------------------------------------------------
// Gradient, steps 3 and 4: sums
struct SumParams {
  const uint32_t *keys, *rows;  // sorted
  float* part;                  // [2][chunks][hidden]: a chunk's run that began before it, its run that goes on
  unsigned* crossing;           // [1 + chunks]: count and list of the chunks in which a crossing run begins (any order)
  int n, vocab, hidden, chunk, chunks;
  float scale;
  bool accumulate;
};

template <typename T, int VEC>
__device__ __forceinline__ void write_row(const SumParams& p, T* dembed, uint32_t key, int col, const float (&acc)[VEC]) {
  using P = Pack<T, VEC>;
  P* at = reinterpret_cast<P*>(dembed + static_cast<size_t>(key) * p.hidden + col);
  P r;
  if (p.accumulate) r = *at;
#pragma unroll
  for (int j = 0; j < VEC; ++j) r.v[j] = from_f<T>(p.accumulate ? fmaf(acc[j], p.scale, to_f(r.v[j])) : acc[j] * p.scale);
  *at = r;
}

constexpr int kMaxChunk = 32;       // at most a warp: a CTA looks at its keys with one thread each
constexpr int kSliceBytes = 1280;   // of a row that a CTA has in shared memory: 40 KB for a chunk, 5 CTAs an SM
constexpr int kBulkRows = 8;        // rows that share an mbarrier
constexpr int kSumThreads = 128;

// One CTA: a chunk of the sorted list, a slice of the columns. Whole 16-byte rows (VEC > 1) come by bulk copies, all of
// the chunk's at once, which needs no registers for what is in flight (loads into registers, 4 a thread: 74 us for the
// call of 32749 rows of 1280, 67 so).
template <typename T, int VEC>
__global__ void __launch_bounds__(kSumThreads) embed_sum_kernel(const T* __restrict__ dout, T* __restrict__ dembed,
                                                                SumParams p, int slice) {
  using P = Pack<T, VEC>;
  extern __shared__ __align__(16) uint8_t s_rows[];  // VEC > 1: [chunk][slice]
  __shared__ uint32_t s_key[kMaxChunk + 2], s_row[kMaxChunk];  // keys with one neighbour on each side
  __shared__ __align__(8) uint64_t s_bar[kMaxChunk / kBulkRows];
  const int tid = threadIdx.x;
  if (VEC > 1 && tid < kMaxChunk / kBulkRows) {
    mbar_init(&s_bar[tid], 1);
    mbar_fence_init();
  }
  pdl_wait();
  pdl_trigger();
  const int c0 = blockIdx.x * p.chunk, len = min(p.chunk, p.n - c0);
  const uint32_t none = 0xffffffffu, vocab = static_cast<uint32_t>(p.vocab);
  if (tid < len + 2) {
    const int at = c0 - 1 + tid;
    s_key[tid] = at >= 0 && at < p.n ? p.keys[at] : none;
    if (tid >= 1 && tid <= len) s_row[tid - 1] = p.rows[at];
  }
  __syncthreads();
  const int count = __syncthreads_count(tid < len && s_key[tid + 1] < vocab);  // padding and bad ids are sorted last
  const int first = blockIdx.y * slice, width = min(slice, p.hidden - first);  // this CTA's columns
  if (VEC > 1 && tid < kMaxChunk / kBulkRows) {
    const int rows = min(kBulkRows, count - tid * kBulkRows);
    const unsigned bytes = static_cast<unsigned>(width) * sizeof(T);
    if (rows > 0) mbar_arrive_expect_tx(&s_bar[tid], rows * bytes);
    for (int i = tid * kBulkRows; i < tid * kBulkRows + rows; ++i)
      bulk_g2s(s_rows + i * bytes, dout + static_cast<size_t>(s_row[i]) * p.hidden + first, bytes, &s_bar[tid]);
  }
  if (tid == 0 && blockIdx.y == 0 && count == len && s_key[len + 1] == s_key[len] && s_key[len] < vocab &&
      (s_key[1] != s_key[len] || s_key[0] != s_key[1]))
    p.crossing[1 + atomicAdd(p.crossing, 1u)] = blockIdx.x;  // a run begins here and goes on
  bool ok = true;
  for (int col = tid * VEC; col < width; col += kSumThreads * VEC) {
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    bool from_before = s_key[1] == s_key[0];
#pragma unroll 4
    for (int i = 0; i < count; ++i) {
      P x;
      if (VEC > 1) {
        if (i % kBulkRows == 0) ok = ok && mbar_wait(&s_bar[i / kBulkRows], 0);
        x = *reinterpret_cast<const P*>(s_rows + (i * width + col) * sizeof(T));
      } else {
        x = *reinterpret_cast<const P*>(dout + static_cast<size_t>(s_row[i]) * p.hidden + first + col);
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += to_f(x.v[j]);
      const bool goes_on = s_key[i + 2] == s_key[i + 1];
      if (goes_on && i + 1 < len) continue;
      if (from_before || goes_on) {  // crosses the chunk's start or end
        float* dst = p.part + (static_cast<size_t>(from_before ? 0 : p.chunks) + blockIdx.x) * p.hidden + first + col;
#pragma unroll
        for (int j = 0; j < VEC; ++j) dst[j] = acc[j];
      } else {
        write_row<T, VEC>(p, dembed, s_key[i + 1], first + col, acc);
      }
      from_before = false;
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    }
  }
  if (VEC > 1 && tid == 0) {  // no CTA leaves with copies in flight, whatever columns its threads had
    for (int k = 0; k * kBulkRows < count; ++k) ok = mbar_wait(&s_bar[k], 0) && ok;
  }
  if (!ok) embed_flag(FW_DEVERR_TIMEOUT);
}

// For each chunk in which a run begins that goes on behind it: adds the run's partials. Eight warps take an eighth of the
// run's chunks each for the same 32 x VEC columns, and the eighths are added in order.
constexpr int kMergeWarps = 16, kMergeParts = 8;
template <typename T, int VEC>
__global__ void __launch_bounds__(32 * kMergeWarps) embed_merge_kernel(T* __restrict__ dembed, SumParams p) {
  __shared__ float s_sum[kMergeWarps / kMergeParts][kMergeParts][32 * VEC];
  pdl_wait();
  const unsigned listed = p.crossing[0];
  // an item: a listed run and a slice of the columns
  constexpr int kCols = 32 * VEC * (kMergeWarps / kMergeParts);
  const unsigned slices = (p.hidden + kCols - 1) / kCols;
  for (unsigned item = blockIdx.x; item < listed * slices; item += gridDim.x) {
    const int c = p.crossing[1 + item / slices];
    const int col0 = item % slices * kCols;
    const uint32_t key = p.keys[(c + 1) * p.chunk - 1];
    int more = 0;  // chunks behind this one that begin inside the run
    while (true) {
      const int64_t at = static_cast<int64_t>(c + 1 + more + threadIdx.x) * p.chunk;
      const int hit = __syncthreads_count(at < p.n && p.keys[at] == key);
      more += hit;
      if (hit < static_cast<int>(blockDim.x)) break;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slice = warp / kMergeParts, part = warp % kMergeParts;
    const int m0 = static_cast<int>(static_cast<int64_t>(more) * part / kMergeParts);
    const int m1 = static_cast<int>(static_cast<int64_t>(more) * (part + 1) / kMergeParts);
    const int col = col0 + (slice * 32 + lane) * VEC;
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    if (col < p.hidden) {
      const float* tail = p.part + (static_cast<size_t>(p.chunks) + c) * p.hidden + col;
      const float* head = p.part + static_cast<size_t>(c + 1) * p.hidden + col;
      if (part == 0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = tail[j];
      }
#pragma unroll 8
      for (int m = m0; m < m1; ++m) {
        using F = Pack<float, VEC < 4 ? VEC : 4>;  // at most 16 bytes an access: all that the workspace is aligned to
        constexpr int W = VEC < 4 ? VEC : 4;
#pragma unroll
        for (int k = 0; k < VEC; k += W) {
          const F x = *reinterpret_cast<const F*>(head + static_cast<size_t>(m) * p.hidden + k);
#pragma unroll
          for (int j = 0; j < W; ++j) acc[k + j] += x.v[j];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) s_sum[slice][part][j * 32 + lane] = acc[j];
    __syncthreads();
    if (part == 0 && col < p.hidden) {
#pragma unroll
      for (int q = 1; q < kMergeParts; ++q) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += s_sum[slice][q][j * 32 + lane];
      }
      write_row<T, VEC>(p, dembed, key, col, acc);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------
// Host side
// Sorted positions per CTA of embed_sum_kernel: 32 keeps the partials small; below 8192 tokens 8, so that the
// gather still covers the SMs.
static int sum_chunk(int n) { return n >= 8192 ? 32 : 8; }

struct EmbedGradLayout {
  int64_t list, crossing, part, total;  // bytes of one of the four lists, offsets, all
  int chunk, chunks;
};

static EmbedGradLayout embed_grad_layout(int n, int hidden) {
  EmbedGradLayout l;
  l.list = (static_cast<int64_t>(n) * 4 + 255) / 256 * 256;
  l.chunk = sum_chunk(n);
  l.chunks = (n + l.chunk - 1) / l.chunk;
  l.crossing = 4 * l.list;
  l.part = l.crossing + (static_cast<int64_t>(l.chunks) * 4 + 4 + 255) / 256 * 256;
  l.total = l.part + 2 * static_cast<int64_t>(l.chunks) * hidden * 4;
  return l;
}

template <typename T, int VEC>
static int run_embed_grad(const void* dout, void* dembed, const EmbedGradLayout& l, SortParams sp, SumParams q,
                          cudaStream_t s) {
  // equal slices of whole packs
  const int packs = q.hidden / VEC, most = kSliceBytes / static_cast<int>(sizeof(T)) / VEC;
  const int slices = (packs - 1) / most + 1;
  FW_REQUIRE(slices <= 65535, FW_ERR_SHAPE, "embed_grad: hidden is too large");
  const int slice = (packs + slices - 1) / slices * VEC;
  // Sorting CTAs: one up to 2048 tokens, where cluster barriers would cost more than they save.
  const int ctas = sp.n <= 2048 ? 1 : kSortCtas;
  cudaError_t e = cudaSuccess;
  int rc = FW_OK;
  if (q.n > 0) {
    e = launch_cluster(embed_sort_kernel, dim3(ctas), dim3(kSortThreads), 0, s, false, ctas, sp);
    rc = launch_status(e, "embed_grad sort");
    if (rc) return rc;
  }
  if (!q.accumulate) {
    const int64_t row_bytes = static_cast<int64_t>(q.hidden) * sizeof(T);
    const int sms = num_sms() - ctas;  // the sort has the others
    const int grid = sp.vocab < sms ? sp.vocab : sms;
    e = launch(embed_fill_kernel, dim3(grid), dim3(kFillThreads), 0, s, q.n > 0, sp, static_cast<uint8_t*>(dembed),
               row_bytes, row_bytes % 16 == 0 && aligned16(dembed));
    rc = launch_status(e, "embed_grad fill");
  }
  if (rc || q.n == 0) return rc;
  const int smem = VEC > 1 ? l.chunk * slice * static_cast<int>(sizeof(T)) : 0;
  e = launch(embed_sum_kernel<T, VEC>, dim3(l.chunks, slices), dim3(kSumThreads), smem, s, true,
             static_cast<const T*>(dout), static_cast<T*>(dembed), q, slice);
  rc = launch_status(e, "embed_grad sum");
  if (rc || l.chunks < 2) return rc;
  e = launch(embed_merge_kernel<T, VEC>, dim3(l.chunks - 1 < 4 * num_sms() ? l.chunks - 1 : 4 * num_sms()),
             dim3(32 * kMergeWarps), 0, s, true, static_cast<T*>(dembed), q);
  return launch_status(e, "embed_grad merge");
}

template <typename T, int VEC>
static int run_embed_scaled(const void* embed, const void* pos, const int64_t* ids, const int64_t* positions,
                            void* out, int n, int vocab, int max_pos, int hidden, float scale, cudaStream_t s) {
  const int warps = n >= 8 * num_sms() ? 8 : 1;  // few rows: spread over the SMs
  cudaError_t e = launch(embed_scaled_kernel<T, VEC>, dim3((static_cast<int64_t>(n) + warps - 1) / warps), dim3(32 * warps), 0, s, false,
                         static_cast<const T*>(embed), static_cast<const T*>(pos), ids, positions,
                         static_cast<T*>(out), n, vocab, max_pos, hidden, scale);
  return launch_status(e, "embed_scaled");
}

unsigned int read_embed_errors(bool clear) {
  unsigned int v = 0, zero = 0;
  cudaMemcpyFromSymbol(&v, g_fw_dev_error, sizeof(v));
  if (clear && v) cudaMemcpyToSymbol(g_fw_dev_error, &zero, sizeof(zero));
  return v;
}

}  // namespace fw

using namespace fw;

extern "C" {

int fw_embed_scaled(const void* embed, const void* pos_embed, const int64_t* ids, const int64_t* positions, void* out,
                    int n, int vocab, int max_pos, int hidden, float scale, int dtype, fw_stream_t stream) {
  FW_REQUIRE(embed && (n == 0 || (ids && out)), FW_ERR_NULL, "embed_scaled: embed, ids and out are required");
  FW_REQUIRE(n == 0 || (pos_embed == nullptr) == (positions == nullptr), FW_ERR_ARG,
             "embed_scaled: pos_embed and positions must be given together");
  FW_REQUIRE(n >= 0 && vocab > 0 && hidden > 0 && hidden <= (1 << 30) && (pos_embed == nullptr || max_pos > 0), FW_ERR_SHAPE,
             "embed_scaled: bad sizes");
  FW_REQUIRE(dtype >= FW_F16 && dtype <= FW_F32, FW_ERR_ARG, "embed_scaled: dtype must be fp16, bf16 or fp32");
  const int size = dtype == FW_F32 ? 4 : 2;
  FW_REQUIRE((reinterpret_cast<uintptr_t>(embed) | reinterpret_cast<uintptr_t>(pos_embed) |
              reinterpret_cast<uintptr_t>(out)) % size == 0,
             FW_ERR_ALIGN, "embed_scaled: pointers must be aligned to their type");
  if (n == 0) return FW_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = hidden * static_cast<int64_t>(size) % 16 == 0 && aligned16(embed) && aligned16(out) && aligned16(pos_embed);
#define FW_EMBED(T, V) \
  return run_embed_scaled<T, V>(embed, pos_embed, ids, positions, out, n, vocab, max_pos, hidden, scale, s)
  if (dtype == FW_F16) {
    if (wide) FW_EMBED(half, 8);
    FW_EMBED(half, 1);
  }
  if (dtype == FW_BF16) {
    if (wide) FW_EMBED(__nv_bfloat16, 8);
    FW_EMBED(__nv_bfloat16, 1);
  }
  if (wide) FW_EMBED(float, 4);
  FW_EMBED(float, 1);
#undef FW_EMBED
}

int fw_embed_grad_workspace(int n, int hidden, int64_t* bytes) {
  FW_REQUIRE(bytes != nullptr, FW_ERR_NULL, "embed_grad_workspace: bytes is NULL");
  FW_REQUIRE(n >= 0 && n <= (1 << 30) && hidden > 0, FW_ERR_SHAPE, "embed_grad: bad sizes");
  *bytes = embed_grad_layout(n, hidden).total;
  return FW_OK;
}

int fw_embed_grad(const void* dout, const int64_t* ids, void* dembed, int n, int vocab, int hidden, float scale,
                  int64_t padding_idx, int accumulate, int dtype, void* workspace, int64_t workspace_bytes,
                  fw_stream_t stream) {
  FW_REQUIRE(dembed && (n == 0 || (dout && ids && workspace)), FW_ERR_NULL,
             "embed_grad: dout, ids, dembed and workspace are required");
  FW_REQUIRE(n >= 0 && n <= (1 << 30) && vocab > 0 && vocab <= (1 << 30) && hidden > 0, FW_ERR_SHAPE,
             "embed_grad: bad sizes");
  FW_REQUIRE(dtype >= FW_F16 && dtype <= FW_F32, FW_ERR_ARG, "embed_grad: dtype must be fp16, bf16 or fp32");
  const int size = dtype == FW_F32 ? 4 : 2;
  FW_REQUIRE((reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dembed)) % size == 0, FW_ERR_ALIGN,
             "embed_grad: pointers must be aligned to their type");
  FW_REQUIRE(aligned16(workspace), FW_ERR_ALIGN, "embed_grad: workspace must be 16-byte aligned");
  const EmbedGradLayout l = embed_grad_layout(n, hidden);
  FW_REQUIRE(n == 0 || workspace_bytes >= l.total, FW_ERR_SHAPE, "embed_grad: workspace too small (%lld of %lld bytes)",
             static_cast<long long>(workspace_bytes), static_cast<long long>(l.total));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n == 0 && accumulate) return FW_OK;
  SortParams sp{};
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  sp.ids = ids;
  for (int i = 0; i < 2; ++i) {
    sp.keys[i] = reinterpret_cast<uint32_t*>(ws + i * l.list);
    sp.rows[i] = reinterpret_cast<uint32_t*>(ws + (2 + i) * l.list);
  }
  sp.n = n;
  sp.vocab = vocab;
  sp.padding = padding_idx;
  while ((static_cast<int64_t>(vocab) >> (8 * sp.passes)) != 0) ++sp.passes;  // the largest key is `vocab`
  SumParams q{};
  q.keys = sp.keys[sp.passes & 1];
  q.rows = sp.rows[sp.passes & 1];
  q.part = reinterpret_cast<float*>(ws + l.part);
  q.crossing = sp.crossing = reinterpret_cast<unsigned*>(ws + l.crossing);
  q.n = n;
  q.vocab = vocab;
  q.hidden = hidden;
  q.chunk = l.chunk;
  q.chunks = l.chunks;
  q.scale = scale;
  q.accumulate = accumulate != 0;
  const bool wide = hidden * static_cast<int64_t>(size) % 16 == 0 && aligned16(dout) && aligned16(dembed);
  if (dtype == FW_F16)
    return wide ? run_embed_grad<half, 8>(dout, dembed, l, sp, q, s) : run_embed_grad<half, 1>(dout, dembed, l, sp, q, s);
  if (dtype == FW_BF16)
    return wide ? run_embed_grad<__nv_bfloat16, 8>(dout, dembed, l, sp, q, s)
                : run_embed_grad<__nv_bfloat16, 1>(dout, dembed, l, sp, q, s);
  return wide ? run_embed_grad<float, 4>(dout, dembed, l, sp, q, s) : run_embed_grad<float, 1>(dout, dembed, l, sp, q, s);
}

}  // extern "C"
