// Attention of several new tokens per sequence over a paged KV cache (paged_chunk.hip):
// parameters and host entries.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "akt_common.hpp"

namespace akt {

constexpr int kCkThreads = 256;  // four waves
constexpr int kCkRows = 128;     // rows (token, query head of the group) of a unit
constexpr int kCkBlock = 128;    // keys of a block, the grain in which units are cut
constexpr int kCkUnitCost = 128;  // cost of a unit's start and end, in keys
// Rows of a sequence and kv head up to which the waves of a workgroup share out the keys.
constexpr int kCkSplitRows = 64;
constexpr int kCkSplit = 1, kCkTiles = 2;  // the kernels of a launch

struct ChunkParams {
  const half_t* q;     // [total_q, Hq, D] rows (strides q_st, q_sh)
  const half_t* pool;  // [P, 2, Hkv, page, D]
  half_t* o;           // [total_q, Hq, D] contiguous
  float* lse;          // [total_q, Hq] or null
  const int32_t* q_indptr;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last_len;
  int* arrive;     // [4 * workgroups] arrival counters (zero between launches)
  char* partials;  // two slots of slot_bytes to a workgroup
  int64_t q_st, q_sh;
  int64_t sp, skv, sh;  // page, K/V and head strides of the pool (elements)
  int ss;               // slot stride (elements, < 2^22)
  int total_q, total_pages, num_pool_pages;
  int B, Hq, Hkv, G;
  int TR;              // tokens of a unit: kCkRows / G
  uint32_t g_magic;    // ceil(2^16 / G): n / G = n * g_magic >> 16 for n < kCkRows
  int page_size;
  uint32_t page_magic;  // min(2^32 - 1, floor(2^32 / page_size))
  int causal;
  int neg_q;       // 1: softmax_scale < 0, computed as (-Q) K^T at |softmax_scale|
  float qk_scale;  // |softmax_scale| * log2(e), at least FLT_MIN
  int wgs;         // workgroups of the launch
  int split_tokens;  // sequences of up to so many new tokens are the split kernel's
  int paths;         // kCkSplit | kCkTiles
  int min_keys;    // fewest keys (with unit costs) of a workgroup's range, at least kCkBlock
};

// Bytes of a partial slot: per wave the fp32 O of 32 rows as it sits in registers
// and a 16-byte (m, l, exact l, -) row for each.
__host__ __device__ constexpr int64_t chunk_wave_bytes(int D) { return 32 * D * 4 + 32 * 16; }
__host__ __device__ constexpr int64_t chunk_slot_bytes(int D) { return 4 * chunk_wave_bytes(D); }

// Workgroups to a CU.
__host__ __device__ constexpr int chunk_wgs_per_cu(int D) { return D <= 128 ? 2 : 1; }

int chunk_launch_64(const ChunkParams& p, bool bf16, hipStream_t st);
int chunk_launch_128(const ChunkParams& p, bool bf16, hipStream_t st);
int chunk_launch_256(const ChunkParams& p, bool bf16, hipStream_t st);

}  // namespace akt
