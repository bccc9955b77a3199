// Selection of the heaviest tokens (gfx950): of the first len entries of a row of sums, the first
// `first`, the last `recent`, and of those between the heaviest, `keep` in all, as an ascending
// index list (-1 padded) and a count, the form of the sparse decodes.  Equal sums go to the lower
// index; a NaN counts as heavier than any number; -0 equals 0.
//
// One 1024-thread workgroup to a row.  The sums become 32-bit keys of the same order, and the key
// of the lightest token that is still kept is found digit by digit (11, 11 and 10 bits): a
// histogram in LDS of the keys that share the digits found so far, then a sum from the top that stops
// at the bin where the count is reached.  The last pass walks the row in order and ranks what is
// kept: heavier keys, and equal ones while any are wanted.  Lanes count in eight copies of a histogram
// (lane mod 8), since sums of probabilities crowd into few binades.
//
// What bounds it: the passes of one workgroup over its row (L2 after the first), their LDS counts
// and barriers; HBM reads a row once.
#include "akt_common.hpp"
#include "akt_host.hpp"

namespace akt {
namespace {

constexpr int kHThreads = 1024;
constexpr int kHWaves = kHThreads / kWave;
constexpr int kHRun = 4;                       // consecutive entries to a lane
constexpr int kHStep = kHThreads * kHRun;  // entries to a step
constexpr int kHBins = 2048;
constexpr int kHCopies = 8;

struct HeavyParams {
  const float* w;  // [N, H, L]
  const int32_t* lengths;
  const int32_t* rows;
  int32_t* ind;  // [B, H, keep]
  int32_t* nnz;  // [B, H]
  int64_t w_sn, w_sh, N;
  int L, H, keep, first, recent;
};

// Keys in the order of the numbers.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 becomes 0
  const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return x != x ? 0xffffffffu : k;
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ uint32_t wave_sum_scan(uint32_t v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t u = (uint32_t)__shfl_up((int)v, d, 64);
    if (lane >= d) v += u;
  }
  return v;
}

__global__ __launch_bounds__(kHThreads) void kept_heaviest_kernel(HeavyParams p) {
  __shared__ __attribute__((aligned(16))) uint32_t hist[kHBins * kHCopies];
  __shared__ uint32_t wave_tot[2][kHWaves];
  __shared__ uint32_t found[2];  // digit, and how many are wanted of its keys
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int b = blockIdx.x / p.H, h = blockIdx.x - b * p.H;
  int32_t* const out = p.ind + (int64_t)blockIdx.x * p.keep;
  const int64_t row = p.rows ? (int64_t)p.rows[b] : b;
  const int len = row < 0 || row >= p.N ? 0 : min(max(p.lengths[b], 0), p.L);
  if (len <= p.keep) {
    for (int i = tid; i < p.keep; i += kHThreads) out[i] = i < len ? i : -1;
    if (tid == 0) p.nnz[blockIdx.x] = len;
    return;
  }
  const float* const w = p.w + row * p.w_sn + h * p.w_sh;
  const int lo = p.first, hi = len - p.recent;
  // The entries from e on that this lane looks at (entries past the row's end read as 0).
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)w, 0, len * 4, kBufferWord3);
  auto load = [&](int e) {
    return as_float4u(
        __builtin_bit_cast(uint4_t, __builtin_amdgcn_raw_buffer_load_b128(rsrc, e * 4, 0, 0)));
  };

  // ---- the key of the lightest kept entry: digits found so far, their mask, entries wanted.
  uint32_t key = 0, mask = 0;
  uint32_t want = (uint32_t)(p.keep - p.first - p.recent);
  if (want > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t digits = pass == 2 ? 1023u : 2047u;
      for (int i = tid; i < kHBins * kHCopies; i += kHThreads) hist[i] = 0;
      __syncthreads();
      for (int e = lo / kHRun * kHRun + tid * kHRun; e < hi; e += kHStep) {
        const float4_t x = load(e);
#pragma unroll
        for (int i = 0; i < kHRun; ++i) {
          const uint32_t k = order_key(x[i]);
          if (e + i >= lo && e + i < hi && (k & mask) == key)
            atomicAdd(&hist[((k >> shift) & digits) * kHCopies + (lane & (kHCopies - 1))], 1u);
        }
      }
      __syncthreads();
      // Thread t sums bins from the top: 2047 - 2 t and the one below it.
      uint32_t c[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4_t* v = reinterpret_cast<const uint4_t*>(hist + (kHBins - 1 - 2 * tid - i) * kHCopies);
#pragma unroll
        for (int j = 0; j < kHCopies / 4; ++j) c[i] += v[j][0] + v[j][1] + v[j][2] + v[j][3];
      }
      const uint32_t incl = wave_sum_scan(c[0] + c[1], lane);
      if (lane == 63) wave_tot[0][wave] = incl;
      __syncthreads();
      uint32_t before = incl - c[0] - c[1];
      for (int i = 0; i < wave; ++i) before += wave_tot[0][i];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (before < want && before + c[i] >= want) {
          found[0] = (uint32_t)(kHBins - 1 - 2 * tid - i);
          found[1] = want - before;
        }
        before += c[i];
      }
      __syncthreads();
      key |= found[0] << shift;
      mask |= digits << shift;
      want = found[1];
    }
  }

  // ---- the kept entries in order: heavier than the key, or equal while any are wanted.
  const bool none = p.keep == p.first + p.recent;
  int kept = 0, equal = 0;  // before this step
  const int wanted = (int)want;
  int buf = 0;
  float4_t nxt = load(tid * kHRun);
  for (int e0 = 0; e0 < len; e0 += kHStep, buf ^= 1) {
    const float4_t x = nxt;
    if (e0 + kHStep < len) nxt = load(e0 + kHStep + tid * kHRun);
    const int e = e0 + tid * kHRun;
    uint32_t cnt = 0;  // kept for sure in the low half, equal ones in the high half
    uint32_t sure = 0, same = 0;
#pragma unroll
    for (int i = 0; i < kHRun; ++i) {
      const uint32_t k = order_key(x[i]);
      const bool in = e + i >= lo && e + i < hi;
      const bool s = e + i < len && (!in || (!none && k > key));
      const bool q = in && !none && k == key;
      sure |= (s ? 1u : 0u) << i;
      same |= (q ? 1u : 0u) << i;
    }
    cnt = (uint32_t)__builtin_popcount(sure) | (uint32_t)__builtin_popcount(same) << 16;
    const uint32_t incl = wave_sum_scan(cnt, lane);
    if (lane == 63) wave_tot[buf][wave] = incl;
    __syncthreads();
    uint32_t before = incl - cnt, total = 0;
#pragma unroll
    for (int i = 0; i < kHWaves; ++i) {
      const uint32_t t = wave_tot[buf][i];
      if (i < wave) before += t;
      total += t;
    }
    int sb = kept + (int)(before & 0xffffu), qb = equal + (int)(before >> 16);
#pragma unroll
    for (int i = 0; i < kHRun; ++i) {
      const bool s = (sure >> i) & 1, q = (same >> i) & 1;
      if (s || (q && qb < wanted)) {
        const int slot = sb + min(qb, wanted);
        if (slot < p.keep) out[slot] = e + i;
      }
      sb += s;
      qb += q;
    }
    kept += (int)(total & 0xffffu);
    equal += (int)(total >> 16);
  }
  if (tid == 0) p.nnz[blockIdx.x] = p.keep;
}

}  // namespace
}  // namespace akt

using namespace akt;

extern "C" int akt_kept_index_heaviest(const float* weights, const int32_t* lengths,
                                       const int32_t* rows, int32_t* sparse_ind,
                                       int32_t* sparse_nnz, int64_t batch, int64_t num_heads,
                                       int64_t num_rows, int64_t row_len,
                                       const int64_t weight_stride[2], int64_t keep, int64_t first,
                                       int64_t recent, void* stream) {
  clear_error();
  AKT_CHECK(batch >= 0 && num_heads >= 0 && num_rows >= 0 && row_len >= 0,
            "sizes must be non-negative");
  AKT_CHECK(keep >= 0 && first >= 0 && recent >= 0 && first <= keep && recent <= keep - first,
            "keep must be at least first + recent");
  AKT_CHECK(row_len < (1ll << 28) && keep < (1ll << 31), "rows are too long");
  AKT_CHECK(batch < (1ll << 31) && num_heads < (1 << 20) &&
                grid_fits(batch * num_heads, kHThreads),
            "too many rows");
  if (batch == 0 || num_heads == 0) return AKT_OK;
  AKT_CHECK(lengths && (sparse_ind || keep == 0) && sparse_nnz &&
                (weights || num_rows == 0 || row_len == 0) && weight_stride,
            "all pointers are required");
  AKT_CHECK(aligned4(weights), "weights must be 4-byte aligned");
  AKT_CHECK(rows || num_rows >= batch, "weights need a row for every sequence");
  HeavyParams p = {};
  p.w = weights;
  p.lengths = lengths;
  p.rows = rows;
  p.ind = sparse_ind;
  p.nnz = sparse_nnz;
  p.w_sn = weight_stride[0];
  p.w_sh = weight_stride[1];
  p.N = num_rows;
  p.L = (int)row_len;
  p.H = (int)num_heads;
  p.keep = (int)keep;
  p.first = (int)first;
  p.recent = (int)recent;
  KernelTimer timer;
  timer.launch(kept_heaviest_kernel, dim3((unsigned)(batch * num_heads)), dim3(kHThreads), 0,
               (hipStream_t)stream, p);
  return check_launch("kept_heaviest_kernel");
}
