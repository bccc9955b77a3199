// Kept tokens close up within a paged KV cache (gfx950): of each (sequence, kv head), slot j takes K
// and V of token ind[j], for the listed tokens j = 0 .. nnz - 1, and row j of the sums takes that
// token's; sums behind the last kept token become 0.
//
// In place.  A listed token never moves towards the end (ind[j] >= j; an entry that asks for that
// is skipped), so slot j is not the source of a later entry, and a batch of entries whose rows are all
// read before any is written never destroys one that a later batch needs; the next batch's rows are
// on their way meanwhile.  A workgroup owns a 128-byte column of K (or V) of one (sequence, kv head)
// and takes the entries in order; columns do not touch each other.  A page that a sequence shares can
// be replaced: the slots of dst_indices, where they differ from the table's, take the rows instead.
//
// Bound by memory: 4 D bytes read and 4 D written a kept token and kv head.  What it measured at 8
// kv heads and D = 128, after steps (16 sequences of 1,025 to 1,088 tokens, 1,024 kept: 136 MB) and
// after prompts (8 of 4,000 to 9,000 tokens, 2,500 kept, bf16: 167 MB): 25.6 and 44.4 us, or 5.3 and
// 3.8 TB/s; without the look-ahead 26.1 and 56.2.  The prompts' case is 256 columns, one to a compute
// unit, so what bounds it is how many rows of its column a workgroup has in flight.
//   Columns of 64 bytes would be twice as many, and every line of 128 bytes would be touched by two
// workgroups: 35.6 and 47.9 us (one sequence of 8,000 tokens to 4,000: 15.3 instead of 24.6).
//   Batches of 128, 256 and 512 rows: 24.9, 25.6 and 29.0 us (step), 47.8, 44.4 and 44.3 (prompt);
// more rows than that spill.
#include "akt_common.hpp"
#include "akt_host.hpp"

namespace akt {
namespace {

constexpr int kEThreads = 1024;
constexpr int kELanes = 8;                   // 16-byte chunks of a column
constexpr int kERows = kEThreads / kELanes;  // rows at a time
constexpr int kEPer = 2;                     // and times to a batch
constexpr int kEBatch = kERows * kEPer;

struct KeepParams {
  half_t* pool;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last_len;
  const int32_t* dst;  // page table entries of the slots written; null: the table's
  const int32_t* ind;  // [B, Hkv, keep]
  const int32_t* nnz;  // [B, Hkv]
  float* w;            // [N, Hkv, L]; may be null
  const int32_t* rows;
  int64_t sp, skv, sh, ss;
  int64_t w_sn, w_sh, N, L;
  int B, Hkv, cpr, columns, keep, page_size, total_pages, num_pool_pages;
  uint32_t page_magic;
};

__device__ __forceinline__ int keep_page(const KeepParams& p, int n) {
  const int q = (int)__umulhi((uint32_t)n, p.page_magic);
  return n - q * p.page_size >= p.page_size ? q + 1 : q;
}

// Waits for a value that was loaded: what reads a register waits for it, a barrier alone does not.
template <typename T>
__device__ __forceinline__ void arrived(const T& x) {
  asm volatile("" ::"v"(x));
}

__global__ __launch_bounds__(kEThreads) void paged_keep_kernel(KeepParams p) {
  const int tid = threadIdx.x;
  // Consecutive workgroups: the columns of one (sequence, kv head).
  const int parts = 2 * p.columns + (p.w ? 1 : 0);
  const int unit = blockIdx.x / parts, part = blockIdx.x - unit * parts;
  const int b = unit / p.Hkv, h = unit - b * p.Hkv;
  const int ip0 = min(max(p.indptr[b], 0), p.total_pages);
  const int np = min(max(p.indptr[b + 1], ip0), p.total_pages) - ip0;
  const int len = np > 0 ? (np - 1) * p.page_size + min(max(p.last_len[b], 0), p.page_size) : 0;
  const int nnz = min(min(max(p.nnz[unit], 0), p.keep), len);
  const int32_t* const ind = p.ind + (int64_t)unit * p.keep;
  if (part == 2 * p.columns) {
    // ---- the sums.
    const int64_t row = p.rows ? (int64_t)p.rows[b] : b;
    if (row < 0 || row >= p.N) return;
    float* const w = p.w + row * p.w_sn + h * p.w_sh;
    for (int j0 = 0; j0 < nnz; j0 += kEThreads * kEPer) {
      float x[kEPer];
      bool ok[kEPer];
#pragma unroll
      for (int k = 0; k < kEPer; ++k) {
        const int j = j0 + k * kEThreads + tid;
        const int t = j < nnz ? ind[j] : -1;
        ok[k] = j < nnz && t >= j && t < len && j < p.L;
        x[k] = ok[k] && t < p.L ? w[t] : 0.f;
      }
      // Every wave's sums are here (not merely asked for) before any is overwritten.
#pragma unroll
      for (int k = 0; k < kEPer; ++k) arrived(x[k]);
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kEPer; ++k)
        if (ok[k]) w[j0 + k * kEThreads + tid] = x[k];
    }
    __syncthreads();
    const int end = (int)min((int64_t)len, p.L);
    for (int j = nnz + tid; j < end; j += kEThreads) w[j] = 0.f;
    return;
  }
  // ---- a column of K or V.
  const int v = part >= p.columns;
  const int chunk = (part - v * p.columns) * kELanes + tid % kELanes;
  half_t* const base = p.pool + v * p.skv + h * p.sh + 8 * chunk;
  const bool mine = chunk < p.cpr;
  // A batch's entries, the pages of their rows, and the rows are looked up one batch after another:
  // while a batch is written, the rows of the next one, the pages of the one after it and the entries of
  // the third are on their way.  Loads come back in the order in which they are asked for, so the
  // rows go last: the next batch's looking up does not wait for them.
  struct Pages {
    int t[kEPer], sid[kEPer], did[kEPer];  // t: token, -1: none
  };
  struct Rows {
    uint4_t x[kEPer];
    half_t* to[kEPer];  // null: not moved
  };
  const int32_t* const dst = p.dst ? p.dst : p.indices;
  auto slot = [&](int i, int k) -> int { return i * kEBatch + k * kERows + tid / kELanes; };
  int e[kEPer];
  Pages g;
  auto load_entries = [&](int i) {
#pragma unroll
    for (int k = 0; k < kEPer; ++k) e[k] = ind[min(slot(i, k), nnz - 1)];
  };
  auto load_pages = [&](int i) {
#pragma unroll
    for (int k = 0; k < kEPer; ++k) {
      const int j = slot(i, k);
      g.t[k] = j < nnz && e[k] >= j && e[k] < len ? e[k] : -1;
      g.sid[k] = p.indices[ip0 + keep_page(p, max(g.t[k], 0))];
      g.did[k] = dst[ip0 + keep_page(p, min(j, nnz - 1))];
    }
  };
  const half_t* src[kEPer];
  auto find_rows = [&](int i, Rows& r) {
#pragma unroll
    for (int k = 0; k < kEPer; ++k) {
      const int j = slot(i, k), t = g.t[k];
      const bool move = mine && t >= 0 && (uint32_t)g.sid[k] < (uint32_t)p.num_pool_pages &&
                        (uint32_t)g.did[k] < (uint32_t)p.num_pool_pages &&
                        (t != j || g.sid[k] != g.did[k]);
      src[k] = base + g.sid[k] * p.sp + (t - keep_page(p, max(t, 0)) * p.page_size) * p.ss;
      r.to[k] = move ? base + g.did[k] * p.sp + (j - keep_page(p, j) * p.page_size) * p.ss : nullptr;
    }
  };
  auto load_rows = [&](Rows& r) {
#pragma unroll
    for (int k = 0; k < kEPer; ++k)
      if (r.to[k]) r.x[k] = ld16(src[k]);
  };
  if (nnz == 0) return;
  Rows ra, rb;
  load_entries(0);
  load_pages(0);
  load_entries(1);
  find_rows(0, ra);
  load_pages(1);
  load_entries(2);
  load_rows(ra);
  auto batch = [&](int i, Rows& r, Rows& next) {
    find_rows(i + 1, next);
    load_pages(i + 2);
    load_entries(i + 3);
    load_rows(next);
    // Every wave's rows are here (not merely asked for) before any is overwritten.
#pragma unroll
    for (int k = 0; k < kEPer; ++k) arrived(r.x[k]);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kEPer; ++k)
      if (r.to[k]) st16(r.to[k], r.x[k]);
  };
  for (int i = 0; i * kEBatch < nnz; i += 2) {
    batch(i, ra, rb);
    if ((i + 1) * kEBatch >= nnz) break;
    batch(i + 1, rb, ra);
  }
}

}  // namespace
}  // namespace akt

using namespace akt;

extern "C" int akt_paged_keep(void* kv_cache, const int32_t* kv_page_indptr,
                              const int32_t* kv_page_indices, const int32_t* kv_last_page_len,
                              const int32_t* dst_page_indices, const int32_t* sparse_ind,
                              const int32_t* sparse_nnz, float* weights, const int32_t* rows,
                              int64_t batch, int64_t num_kv_heads, int64_t head_dim,
                              int64_t page_size, int64_t total_pages, int64_t num_pool_pages,
                              int64_t keep, int64_t num_rows, int64_t row_len,
                              const int64_t kv_stride[5], const int64_t weight_stride[2],
                              void* stream) {
  clear_error();
  AKT_CHECK(batch >= 0 && total_pages >= 0 && num_pool_pages >= 0 && keep >= 0 && num_rows >= 0 &&
                row_len >= 0 && num_kv_heads > 0,
            "sizes must be non-negative");
  AKT_CHECK(head_dim > 0 && head_dim % 8 == 0 && head_dim <= 1024,
            "head_dim must be a positive multiple of 8 up to 1024");
  AKT_CHECK(page_size > 0 && page_size < (1 << 20), "page_size out of range");
  AKT_CHECK(total_pages < (1ll << 31) && total_pages * page_size < (1ll << 30),
            "the page table spans too many tokens");
  AKT_CHECK(batch < (1ll << 30) && num_kv_heads < (1 << 20) && keep < (1ll << 30),
            "problem too large");
  if (batch == 0 || total_pages == 0) return AKT_OK;
  AKT_CHECK(kv_cache && kv_page_indptr && kv_page_indices && kv_last_page_len &&
                (sparse_ind || keep == 0) && sparse_nnz && kv_stride,
            "all pointers are required");
  AKT_CHECK(kv_stride[4] == 1, "head_dim stride must be 1");
  AKT_CHECK(rows_aligned16(kv_cache, kv_stride, 4), "tensors must have 16-byte aligned rows");
  AKT_CHECK(!weights || (weight_stride && aligned4(weights) && (rows || num_rows >= batch)),
            "weights need strides and a row for every sequence");
  KeepParams p = {};
  p.pool = (half_t*)kv_cache;
  p.indptr = kv_page_indptr;
  p.indices = kv_page_indices;
  p.last_len = kv_last_page_len;
  p.dst = dst_page_indices;
  p.ind = sparse_ind;
  p.nnz = sparse_nnz;
  p.w = weights;
  p.rows = rows;
  p.sp = kv_stride[0];
  p.skv = kv_stride[1];
  p.sh = kv_stride[2];
  p.ss = kv_stride[3];
  if (weights) {
    p.w_sn = weight_stride[0];
    p.w_sh = weight_stride[1];
  }
  p.N = num_rows;
  p.L = row_len;
  p.B = (int)batch;
  p.Hkv = (int)num_kv_heads;
  p.cpr = (int)(head_dim / 8);
  p.columns = (int)ceil_div(p.cpr, kELanes);
  p.keep = (int)keep;
  p.page_size = (int)page_size;
  p.total_pages = (int)total_pages;
  p.num_pool_pages = (int)(num_pool_pages < (1ll << 31) ? num_pool_pages : (1ll << 31) - 1);
  const uint64_t magic = (1ull << 32) / (uint64_t)page_size;
  p.page_magic = (uint32_t)(magic < 0xffffffffull ? magic : 0xffffffffull);
  const int64_t blocks = batch * num_kv_heads * (2 * p.columns + (weights ? 1 : 0));
  AKT_CHECK(blocks < (1ll << 31) && grid_fits(blocks, kEThreads), "problem too large");
  KernelTimer timer;
  timer.launch(paged_keep_kernel, dim3((unsigned)blocks), dim3(kEThreads), 0, (hipStream_t)stream, p);
  return check_launch("paged_keep_kernel");
}
