// Page copies within a paged KV cache (gfx950): the first t slots of page src[i] become those
// of page dst[i], K and V of every head (a fork's last page, copy on write, compaction).
//
// HBM-bound: 2 x 2 Hkv t D elements.  A workgroup moves a fixed number of 16-byte chunks of
// one page, every lane's loads before its stores.  Pages outside the pool are skipped.
// 1000 pages of 64 tokens, 8 heads, D = 128: 107 us (524 MB, 4.9 TB/s, where a large copy
// reaches 5.1).
#include "akt_common.hpp"
#include "akt_host.hpp"

namespace akt {
namespace {

constexpr int kPThreads = 256;
constexpr int kPPerLane = 4;  // chunks of a lane

struct CopyParams {
  half_t* pool;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* tokens;  // null: whole pages
  int64_t sp, skv, sh, ss;
  int page_size, cpr, Hkv, num_pool_pages;
  int per_head;  // chunks of a head's K (or V) in a page
  int per_page;  // 2 Hkv per_head
  int blocks;    // workgroups to a page
};

__global__ __launch_bounds__(kPThreads) void paged_copy_kernel(CopyParams p) {
  const int i = (int)(blockIdx.x / (uint32_t)p.blocks);
  const int part = (int)(blockIdx.x - (uint32_t)i * p.blocks);
  const int s = p.src[i], d = p.dst[i];
  if ((uint32_t)s >= (uint32_t)p.num_pool_pages || (uint32_t)d >= (uint32_t)p.num_pool_pages ||
      s == d)
    return;
  const int n = p.tokens ? min(p.tokens[i], p.page_size) : p.page_size;
  const half_t* from = p.pool + s * p.sp;
  half_t* to = p.pool + d * p.sp;
  uint4_t x[kPPerLane];
  int64_t at[kPPerLane];
#pragma unroll
  for (int k = 0; k < kPPerLane; ++k) {
    const int c = (part * kPPerLane + k) * kPThreads + (int)threadIdx.x;
    at[k] = -1;
    if (c < p.per_page) {
      const int head = (int)((uint32_t)c / (uint32_t)p.per_head);  // K heads, then V heads
      const int rem = c - head * p.per_head;
      const int slot = (int)((uint32_t)rem / (uint32_t)p.cpr);
      if (slot < n) {
        const int v = head >= p.Hkv;
        at[k] = v * p.skv + (head - v * p.Hkv) * p.sh + slot * p.ss + 8 * (rem - slot * p.cpr);
        x[k] = ld16(from + at[k]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kPPerLane; ++k)
    if (at[k] >= 0) st16(to + at[k], x[k]);
}

}  // namespace
}  // namespace akt

using namespace akt;

extern "C" int akt_paged_copy(void* kv_cache, const int32_t* src, const int32_t* dst,
                              const int32_t* num_tokens, int64_t n, int64_t num_kv_heads,
                              int64_t head_dim, int64_t page_size, int64_t num_pool_pages,
                              const int64_t kv_stride[5], void* stream) {
  clear_error();
  AKT_CHECK(n >= 0 && num_kv_heads > 0 && num_pool_pages >= 0, "sizes must be non-negative");
  AKT_CHECK(head_dim > 0 && head_dim % 8 == 0 && head_dim <= 1024,
            "head_dim must be a positive multiple of 8 up to 1024");
  AKT_CHECK(page_size > 0 && page_size < (1 << 20), "page_size out of range");
  if (n == 0) return AKT_OK;
  AKT_CHECK(kv_cache && src && dst && kv_stride, "all pointers are required");
  AKT_CHECK(kv_stride[4] == 1, "head_dim stride must be 1");
  for (int j = 0; j < 4; ++j) AKT_CHECK(kv_stride[j] >= 0, "kv strides must be non-negative");
  AKT_CHECK(rows_aligned16(kv_cache, kv_stride, 4), "tensors must have 16-byte aligned rows");
  const int64_t per_head = page_size * (head_dim / 8);
  AKT_CHECK(num_kv_heads < (1 << 20) && 2 * num_kv_heads * per_head < (1ll << 30),
            "a page is too large");
  CopyParams p = {};
  p.pool = (half_t*)kv_cache;
  p.src = src;
  p.dst = dst;
  p.tokens = num_tokens;
  p.sp = kv_stride[0];
  p.skv = kv_stride[1];
  p.sh = kv_stride[2];
  p.ss = kv_stride[3];
  p.page_size = (int)page_size;
  p.cpr = (int)(head_dim / 8);
  p.Hkv = (int)num_kv_heads;
  p.num_pool_pages = (int)(num_pool_pages < (1ll << 31) ? num_pool_pages : (1ll << 31) - 1);
  p.per_head = (int)per_head;
  p.per_page = (int)(2 * num_kv_heads * per_head);
  p.blocks = (int)ceil_div(p.per_page, kPThreads * kPPerLane);
  AKT_CHECK(n < (1ll << 31) && grid_fits(n * p.blocks, kPThreads), "too many pages");
  KernelTimer timer;
  timer.launch(paged_copy_kernel, dim3((unsigned)(n * p.blocks)), dim3(kPThreads), 0,
               (hipStream_t)stream, p);
  return check_launch("paged_copy_kernel");
}
