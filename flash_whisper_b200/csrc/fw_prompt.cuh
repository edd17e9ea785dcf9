// What the packed attention (fw_prompt.cu) and its gradient (fw_prompt_grad.cu) share: the arguments, the search for a
// work item among the sequences, tensor maps and checks.
#pragma once

#include "fw_host.h"
#include "fw_tc.cuh"

namespace fw {

FW_DEFINE_ERROR_WORD();

__device__ __forceinline__ void prompt_flag(unsigned bits) { atomicOr(&g_fw_dev_error, bits); }

constexpr float kLog2 = 1.4426950408889634f;
constexpr int kRows = 128;  // query rows of a tile, keys of a block
constexpr uint32_t kTileBytes = kRows * 64 * 2;  // 16 KB

struct PromptArgs {
  const int64_t *cu_q, *cu_k;  // [seqs + 1]
  int seqs, heads, kv_heads, group;
  int tokens;        // query tokens of a tile: 128 / group
  int64_t rows_q, rows_k;
  float scale_log2;  // scale * log2 e
  int causal, splits;
  int few;           // forward: sequences of at most so many queries are prompt_few_kernel's
  void* out;
  int64_t out_token, out_head;  // strides, elements
  float* lse;                   // [heads][rows_q], may be null
  float *part_o, *part_lse;     // splits > 1: [splits][rows_q][heads][64], [splits][heads][rows_q]
};

// Offsets in order and in range: what does not hold of them leaves a sequence out.
__device__ __forceinline__ bool good_sequence(const PromptArgs& a, int b) {
  const int64_t q0 = a.cu_q[b], q1 = a.cu_q[b + 1], k0 = a.cu_k[b], k1 = a.cu_k[b + 1];
  return q0 >= 0 && q1 >= q0 && q1 <= a.rows_q && k0 >= 0 && k1 >= k0 && k1 <= a.rows_k;
}

// Where a work item lies: a tile of one sequence.
struct Item {
  int64_t q0, k0;  // first rows of the sequence
  int lq, lk;
  int tile;        // index of the item within its sequence; -1: no such item
  int seq;
};

// Finds item `index` (counting ceil(lq / per) items per sequence of more than `skip` rows), by one warp, 32 U sequences at
// a time. Sequences whose offsets are out of order or out of range have none and set the error bit. Launches have room for
// sequences that share no rows. Only behind bad offsets can one begin before the end of a good one in front of it; it has no
// items either, lest those behind it find no room.
template <int U>
__device__ __forceinline__ Item find_among(const int64_t* cu_a, const int64_t* cu_b, int64_t rows_a, int64_t rows_b,
                                           int seqs, int per, int skip, int index, int lane) {
  Item it{};
  it.tile = -1;
  bool disorder = false;  // bad offsets so far
  int reach = 0;          // if so, the furthest end of a good sequence so far
  for (int b0 = 0; b0 < seqs; b0 += 32 * U) {
    const int b = b0 + U * lane;
    int64_t a[U + 1], c[U + 1];
#pragma unroll
    for (int u = 0; u <= U; ++u) {
      a[u] = b + u <= seqs ? cu_a[b + u] : 0;
      c[u] = b + u <= seqs ? cu_b[b + u] : 0;
    }
    int n[U], sum = 0;
    unsigned bad = 0;  // bit u
#pragma unroll
    for (int u = 0; u < U; ++u) {
      n[u] = 0;
      if (b + u >= seqs) continue;
      if (a[u] < 0 || a[u + 1] < a[u] || a[u + 1] > rows_a || c[u] < 0 || c[u + 1] < c[u] || c[u + 1] > rows_b) {
        prompt_flag(FW_DEVERR_BAD_INDEX);
        bad |= 1u << u;
        continue;
      }
      const unsigned rows = static_cast<unsigned>(a[u + 1] - a[u]);
      if (rows > static_cast<unsigned>(skip)) n[u] = (rows + per - 1) / static_cast<unsigned>(per);
      sum += n[u];
    }
    if (disorder || __any_sync(0xffffffffu, bad != 0)) {
      if (!disorder) reach = max(0, static_cast<int>(__shfl_sync(0xffffffffu, b0 > 0 ? a[0] : 0, 0)));  // in order up to here
      disorder = true;
      int end[U], front = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        end[u] = b + u < seqs && !(bad & (1u << u)) && a[u + 1] > a[u] ? static_cast<int>(a[u + 1]) : 0;
        front = max(front, end[u]);
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, front, o);
        if (lane >= o) front = max(front, x);
      }
      const int all = __shfl_sync(0xffffffffu, front, 31);
      front = __shfl_up_sync(0xffffffffu, front, 1);
      front = lane == 0 ? reach : max(reach, front);
      reach = max(reach, all);
      sum = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (a[u] < front) n[u] = 0;
        front = max(front, end[u]);
        sum += n[u];
      }
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    int at = index - (incl - sum);  // within this lane's items
    const unsigned hit = __ballot_sync(0xffffffffu, at >= 0 && at < sum);
    if (hit != 0) {
      int seq = -1, tile = 0, q0 = 0, lq = 0, k0 = 0, lk = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (seq < 0 && at < n[u]) {
          seq = b + u, tile = at;
          q0 = static_cast<int>(a[u]), lq = static_cast<int>(a[u + 1] - a[u]);
          k0 = static_cast<int>(c[u]), lk = static_cast<int>(c[u + 1] - c[u]);
        }
        at -= n[u];
      }
      const int src = __ffs(hit) - 1;
      it.seq = __shfl_sync(0xffffffffu, seq, src);
      it.tile = __shfl_sync(0xffffffffu, tile, src);
      it.q0 = __shfl_sync(0xffffffffu, q0, src);
      it.lq = __shfl_sync(0xffffffffu, lq, src);
      it.k0 = __shfl_sync(0xffffffffu, k0, src);
      it.lk = __shfl_sync(0xffffffffu, lk, src);
      return it;
    }
    index -= __shfl_sync(0xffffffffu, incl, 31);
  }
  return it;
}
// Four sequences a lane where there are many (forward, 1000 of 100 rows, 20 heads: 1564 us with one, 1114), one up to two
// turns (37 of 448 rows: 99 us with four, 94).
__device__ __forceinline__ Item find_item(const int64_t* cu_a, const int64_t* cu_b, int64_t rows_a, int64_t rows_b,
                                          int seqs, int per, int skip, int index, int lane) {
  return seqs <= 64 ? find_among<1>(cu_a, cu_b, rows_a, rows_b, seqs, per, skip, index, lane)
                    : find_among<4>(cu_a, cu_b, rows_a, rows_b, seqs, per, skip, index, lane);
}

// ------------------------------------------------------------------------------------------------
// Host side
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

static int check_rows(const char* what, const char* name, const fw_rows_t& x, int heads, int64_t rows) {
  FW_REQUIRE(rows == 0 || x.ptr, FW_ERR_NULL, "%s: %s is required", what, name);
  FW_REQUIRE(aligned16(x.ptr) && x.token % 8 == 0 && x.head % 8 == 0, FW_ERR_ALIGN,
             "%s: %s must start on 16 bytes and have strides of a multiple of 8 elements", what, name);
  FW_REQUIRE(x.head >= 64 && x.token >= 64 && x.token < (int64_t(1) << 36) && x.head < (int64_t(1) << 36) &&
                 (heads == 1 || rows <= 1 || x.token >= x.head * (heads - 1) + 64 || (x.head - 64) / x.token >= rows - 1),
             FW_ERR_SHAPE, "%s: %s has overlapping or negative strides", what, name);
  return FW_OK;
}

static int check_prompt(const char* what, const int64_t* cu_q, const int64_t* cu_k, int seqs, int64_t rows_q,
                        int64_t rows_k, int heads, int kv_heads, float scale, int dtype) {
  FW_REQUIRE(seqs >= 0 && rows_q >= 0 && rows_k >= 0 && rows_q < (int64_t(1) << 30) && rows_k < (int64_t(1) << 30),
             FW_ERR_SHAPE, "%s: bad sizes", what);
  FW_REQUIRE(kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads / kv_heads <= kRows && heads <= 65536,
             FW_ERR_SHAPE, "%s: heads must be a multiple of kv_heads, at most 128 times as many", what);
  FW_REQUIRE(scale > 0.f && scale * kLog2 < INFINITY, FW_ERR_ARG, "%s: scale must be positive and finite", what);
  FW_REQUIRE(dtype == FW_F16 || dtype == FW_BF16, FW_ERR_ARG, "%s: dtype must be fp16 or bf16", what);
  FW_REQUIRE(seqs == 0 || (cu_q && cu_k), FW_ERR_NULL, "%s: cu_q and cu_k are required", what);
  return FW_OK;
}

}  // namespace fw
