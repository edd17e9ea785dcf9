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

}  // namespace fw
