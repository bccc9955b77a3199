// Attention of several new tokens per sequence over a paged KV cache (paged_chunk.hip):
// parameters and host entries.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "akt_common.hpp"

namespace akt {

constexpr int kCkRows = 128;  // query heads that a kv head may have: a token's rows are in one unit
constexpr int kCkBlock = 128;    // keys of a block, the grain in which units are cut
constexpr int kCkUnitCost = 128;  // cost of a unit's start and end, in keys
// Rows of a sequence and kv head up to which waves share out the keys.  Past 32, two waves of a
// team would load each key, and tiles of mostly idle rows are faster up to D = 128 (us, shared
// out / tiles: 40 rows, 16 sequences over 500 to 4000 keys 59.4 / 54.1, 64 sequences of 64 rows
// 164 / 143, two of 64 rows over 30000 90 / 64); at D = 256, where a tile has half the waves, one
// of 64 rows over 30000 takes 88 / 117, 16 over 500 to 4000 67 / 65.
__host__ __device__ constexpr int chunk_split_rows(int D) { return D <= 128 ? 32 : 64; }
constexpr int kCkFew = 1, kCkMany = 2;
// A key of a unit of many rows costs a workgroup as much as so many of a unit of few (us at 1.4,
// 2 and 3, 777 new tokens beside 15 single ones: D = 128 73.9 / 69.4 / 72.4, D = 256 77.6 / 83.6
// / 97.8, D = 64 75.2 / 69.8 / 67.9; 2000 beside 7 after 3000 to 9000, D = 128 327 / 334 / 592).
__host__ __device__ constexpr double chunk_tile_cost(int D) { return D <= 128 ? 2.0 : 1.4; }

struct ChunkParams {
  const half_t* q;     // [total_q, Hq, D] rows (strides q_st, q_sh)
  const half_t* pool;  // [P, 2, Hkv, page, D]
  half_t* o;           // [total_q, Hq, D] contiguous
  float* lse;          // [total_q, Hq] or null
  const int32_t* q_indptr;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last_len;
  int* arrive;     // arrival counters, one to a wave and range (zero between launches)
  char* partials;  // two slots to a range
  int64_t q_st, q_sh;
  int64_t sp, skv, sh;  // page, K/V and head strides of the pool (elements)
  int ss;               // slot stride (elements, < 2^22)
  int total_q, total_pages, num_pool_pages;
  int B, Hq, Hkv, G;
  int TR;              // tokens of a unit: 32 waves / G
  uint32_t g_magic;    // ceil(2^16 / G): n / G = n * g_magic >> 16 for n < 256
  int page_size;
  uint32_t page_magic;  // min(2^32 - 1, floor(2^32 / page_size))
  int causal;
  int neg_q;       // 1: softmax_scale < 0, computed as (-Q) K^T at |softmax_scale|
  float qk_scale;  // |softmax_scale| * log2(e), at least FLT_MIN
  int split_tokens;  // sequences of up to so many new tokens share out their keys
  int kinds;         // sequences that there can be: kCkFew | kCkMany
  int wgs;
  int many_counter;      // where the second kind's arrival counters
  int64_t many_partial;  // and partials begin
  int min_keys;    // fewest keys (with unit costs) of a range, at least kCkBlock
};

// Waves of a workgroup.  Up to D = 128 eight share a tile of 64 keys (one workgroup to a CU):
// half the loads, LDS stores and barriers a wave, and faster for most sizes (us, four waves /
// eight): D = 128, 32 heads over 8: 32 tokens after 200 26.6 / 24.6, 777 after 0 41.0 / 36.2,
// 777 after 8000 153 / 142, 2048 after 30000 1239 / 1101; D = 64, 64 heads over 16: 8 x 1024
// after 0 150 / 144, 1024 after 10000 250 / 226, 100 after 1000 22.7 / 24.3.
__host__ __device__ constexpr int chunk_waves(int D) { return D <= 128 ? 8 : 4; }

// Bytes of a wave's part of a partial slot: fp32 O of 32 rows as it sits in registers and a
// 16-byte (m, l, exact l, -) row for each.  Where four waves share out the keys, a wave
// holds its share of the pieces of O: a quarter, or (rows for two waves) half.
__host__ __device__ constexpr int64_t chunk_wave_bytes(int D) { return 32 * D * 4 + 32 * 16; }
__host__ __device__ constexpr int64_t chunk_split_wave_bytes(int D) {
  return 32 * D * 4 / (chunk_split_rows(D) > 32 ? 2 : 4) + 32 * 16;
}

// Waves to a SIMD.
__host__ __device__ constexpr int chunk_waves_per_simd(int D) { return D <= 128 ? 2 : 1; }

int chunk_launch_64(const ChunkParams& p, bool bf16, hipStream_t st);
int chunk_launch_128(const ChunkParams& p, bool bf16, hipStream_t st);
int chunk_launch_256(const ChunkParams& p, bool bf16, hipStream_t st);

}  // namespace akt
