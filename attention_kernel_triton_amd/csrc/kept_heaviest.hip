// Selection of the heaviest tokens (gfx950): of the first len entries of a row of sums, the first
// `first`, the last `recent`, and of those between the heaviest, `keep` in all, as an ascending
// index list (-1 padded) and a count, the form of the sparse decodes.  Equal sums go to the lower
// index; a NaN counts as heavier than any number; -0 equals 0.
//
// One workgroup to a row.  The sums become 32-bit keys of the same order, and the key of the lightest
// entry that is still kept is found digit by digit (11, 11 and 10 bits): a histogram in LDS of the
// candidates that share the digits found so far, then a sum from the top that stops at the bin where
// the count is reached, or at all digits that matter: where the bin's candidates are just those still
// wanted, lower digits decide nothing (with hardly any equal sums the third is never looked at).  Then
// what is kept is ranked in the row's order: heavier candidates, and equal ones while any are wanted.
// Lanes count in four or eight copies of a histogram (lane mod that), since sums of probabilities crowd into few
// binades.
//
// Rows of up to 64 k entries are read once and stay in registers (a wave's entries are consecutive,
// so that ranks need the other waves once); longer ones are read again for each pass.
//
// What bounds it: with few rows, the round trips, LDS counts and barriers of one workgroup.  128 rows
// of about 1,060, 1,024 kept: 7.4 to 7.8 us, of which a launch is 4; 64 rows of 20,000 to 40,000,
// 4,000 kept: 25.7 us, of which the loads take 2, a digit's counts 1.7 and its search 1, what is
// written 3 to 6 (the entries as they are ranked, scattered over 64 lanes' slots).
#include <type_traits>

#include "akt_common.hpp"
#include "akt_host.hpp"

namespace akt {
namespace {

constexpr int kHThreads = 1024;  // of the kernel for long rows
constexpr int kHWaves = kHThreads / kWave;
constexpr int kHRun = 4;                       // consecutive entries to a lane
constexpr int kHStep = kHThreads * kHRun;  // entries to a step
constexpr int kHBins = 2048;

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

// What a workgroup's row asks for; false: all of it is kept, and written.
struct HeavyRow {
  const float* w;
  int len, lo, hi;  // entries, and the candidates among them: lo .. hi - 1
};
template <int NT>
__device__ __forceinline__ bool heavy_row(const HeavyParams& p, HeavyRow& r) {
  const int b = blockIdx.x / p.H, h = blockIdx.x - b * p.H;
  const int64_t row = p.rows ? (int64_t)p.rows[b] : b;
  r.len = row < 0 || row >= p.N ? 0 : min(max(p.lengths[b], 0), p.L);
  if (r.len <= p.keep) {
    int32_t* const out = p.ind + (int64_t)blockIdx.x * p.keep;
    for (int i = threadIdx.x; i < p.keep; i += NT) out[i] = i < r.len ? i : -1;
    if (threadIdx.x == 0) p.nnz[blockIdx.x] = r.len;
    return false;
  }
  r.w = p.w + row * p.w_sn + h * p.w_sh;
  r.lo = p.first;
  r.hi = r.len - p.recent;
  return true;
}

// The digits found so far of the lightest kept candidate's key: those in `mask` are `key`, and of the
// candidates that share them `want` are kept.
struct HeavyKey {
  uint32_t key, mask, want;
};
// LDS of the search: NC copies of a histogram, wave sums, and what a digit's search found.
template <int NT, int NC>
struct HeavyLds {
  uint4_t hist[kHBins * NC / 4];
  uint32_t tot[2][NT / kWave];
  uint32_t digit, want, count;
};
// Finds the digits.  count(f): calls f(k) for the key k of each of the thread's candidates, and may
// call it for 0, which is no number's key and the last in order.
template <int NT, int NC, typename F>
__device__ __forceinline__ HeavyKey find_key(HeavyLds<NT, NC>& lds, uint32_t want, F count) {
  constexpr int BPT = kHBins / NT;  // bins to a thread
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  uint32_t* const hist = reinterpret_cast<uint32_t*>(lds.hist) + (lane & (NC - 1));
  HeavyKey r = {0, 0, want};
  // One digit; whether the next ones matter.
  auto digit = [&](auto pass_c) -> bool {
    constexpr int kPass = decltype(pass_c)::value;
    constexpr int kShift = kPass == 0 ? 21 : kPass == 1 ? 10 : 0;
    constexpr uint32_t kDigits = kPass == 2 ? 1023u : 2047u;
#pragma unroll
    for (int i = 0; i < kHBins * NC / 4 / NT; ++i) lds.hist[i * NT + tid] = uint4_t{0, 0, 0, 0};
    __syncthreads();
    count([&](uint32_t k) {
      if (kPass == 0 || (k & r.mask) == r.key)
        atomicAdd(&hist[((k >> kShift) & kDigits) * NC], 1u);
    });
    __syncthreads();
    // Thread t sums bins from the top: those from kHBins - 1 - BPT t down.
    uint32_t c[BPT], mine = 0;
#pragma unroll
    for (int i = 0; i < BPT; ++i) {
      const uint4_t* v = lds.hist + (kHBins - 1 - BPT * tid - i) * NC / 4;
      c[i] = 0;
#pragma unroll
      for (int j = 0; j < NC / 4; ++j) c[i] += v[j][0] + v[j][1] + v[j][2] + v[j][3];
      mine += c[i];
    }
    const uint32_t incl = wave_inclusive_scan(mine);
    if (lane == 63) lds.tot[0][wave] = incl;
    __syncthreads();
    uint32_t before = incl - mine;
#pragma unroll
    for (int i = 0; i < NT / kWave; ++i) {
      const uint32_t t = lds.tot[0][i];
      before += i < wave ? t : 0;
    }
#pragma unroll
    for (int i = 0; i < BPT; ++i) {
      if (before < r.want && before + c[i] >= r.want) {
        lds.digit = (uint32_t)(kHBins - 1 - BPT * tid - i);
        lds.want = r.want - before;
        lds.count = c[i];
      }
      before += c[i];
    }
    __syncthreads();
    r.key |= (uint32_t)uniform((int)lds.digit) << kShift;
    r.mask |= kDigits << kShift;
    r.want = (uint32_t)uniform((int)lds.want);
    return r.want != (uint32_t)uniform((int)lds.count);
  };
  if (want > 0 && digit(std::integral_constant<int, 0>{}) &&
      digit(std::integral_constant<int, 1>{}))
    digit(std::integral_constant<int, 2>{});
  return r;
}

// Rows in registers.  Wave w has as many consecutive entries as the others, a multiple of 256; lane l
// of its 64-entry chunk c has entry 64 c + l, so that a ballot has a chunk's bits in order.
template <int NT, int PER>
__global__ __launch_bounds__(NT) void kept_heaviest_kernel(HeavyParams p) {
  constexpr int NC = NT == 1024 ? 8 : 4, NW = NT / kWave;
  __shared__ HeavyLds<NT, NC> lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  HeavyRow r;
  if (!heavy_row<NT>(p, r)) return;
  const int len = uniform(r.len), lo = r.lo, hi = uniform(r.hi);
  const int groups = (len + 256 * NW - 1) / (256 * NW);  // of four chunks, to a wave
  const int e0 = wave * groups * 256;
  // (Loads past the row's end read 0.)
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)r.w, 0, len * 4, kBufferWord3);
  uint32_t key[PER];  // 0: not a candidate (no number's key)
#pragma unroll
  for (int c = 0; c < PER; c += 4)
    if (c / 4 < groups)
#pragma unroll
      for (int i = c; i < c + 4; ++i)
        key[i] = __builtin_amdgcn_raw_buffer_load_b32(rsrc, (e0 + 64 * i + lane) * 4, 0, 0);
#pragma unroll
  for (int c = 0; c < PER; c += 4)
    if (c / 4 < groups) {
#pragma unroll
      for (int i = c; i < c + 4; ++i) key[i] = order_key(__uint_as_float(key[i]));
      const int e = e0 + 64 * c;
      if (e < lo || e + 256 > hi)  // wave-uniform
#pragma unroll
        for (int i = c; i < c + 4; ++i) {
          const int at = e0 + 64 * i + lane;
          key[i] = at >= lo && at < hi ? key[i] : 0;
        }
    }
  const HeavyKey f = find_key<NT, NC>(lds, (uint32_t)(p.keep - p.first - p.recent), [&](auto add) {
#pragma unroll
    for (int c = 0; c < PER; c += 4)
      if (c / 4 < groups)
#pragma unroll
        for (int i = c; i < c + 4; ++i) add(key[i]);
  });
  // Bits of the entries kept for sure (heavier candidates, and those that are no candidates), and of
  // the equal ones, of which the first f.want are kept; where no candidate is, nothing is heavier or
  // equal.  Chunk i's go to LDS by lane i, and then thread t takes chunk t of the row.
  const uint32_t mask = f.mask, least = f.mask ? f.key : 1u;
  uint32_t sl = 0, sh = 0, ql = 0, qh = 0;
#pragma unroll
  for (int c = 0; c < PER; c += 4)
    if (c / 4 < groups)
#pragma unroll
      for (int i = c; i < c + 4; ++i) {
        const uint32_t k = key[i] & mask;
        uint64_t s = __ballot(k > least);
        const uint64_t q = __ballot(k == least);
        const int e = e0 + 64 * i;
        if (e < lo || e + 64 > hi) s |= __ballot(e + lane < lo || (e + lane >= hi && e + lane < len));
        sl = lane == i ? (uint32_t)s : sl;
        sh = lane == i ? (uint32_t)(s >> 32) : sh;
        ql = lane == i ? (uint32_t)q : ql;
        qh = lane == i ? (uint32_t)(q >> 32) : qh;
      }
  uint4_t* const bits = lds.hist;  // (its last reads are behind find_key's last barrier)
  if (lane < 4 * groups) bits[wave * 4 * groups + lane] = uint4_t{sl, sh, ql, qh};
  __syncthreads();
  const int chunks = 4 * groups * NW;  // of the row: at most one to a thread
  const uint4_t m = tid < chunks ? bits[tid] : uint4_t{0, 0, 0, 0};
  uint64_t keep = (uint64_t)m[1] << 32 | m[0], equal = (uint64_t)m[3] << 32 | m[2];
  const uint32_t s0 = (uint32_t)__builtin_popcountll(keep), q0 = (uint32_t)__builtin_popcountll(equal);
  const uint32_t si = wave_inclusive_scan(s0), qi = wave_inclusive_scan(q0);
  if (lane == 63) {
    lds.tot[0][wave] = si;
    lds.tot[1][wave] = qi;
  }
  __syncthreads();
  int slot = (int)(si - s0), before = (int)(qi - q0);  // kept for sure, and equal, before the chunk
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const int s = (int)lds.tot[0][i], q = (int)lds.tot[1][i];
    slot += i < wave ? s : 0;
    before += i < wave ? q : 0;
  }
  const int wanted = (int)f.want;
  slot += min(before, wanted);
  for (int n = wanted - before; equal && n > 0; --n) {
    keep |= equal & -equal;
    equal &= equal - 1;
  }
  // Every wave writes its chunks: lane l the entry of bit l, behind those of the bits below.
  if (tid < chunks) bits[tid] = uint4_t{(uint32_t)keep, (uint32_t)(keep >> 32), (uint32_t)slot, 0};
  __syncthreads();
  int32_t* const out = p.ind + (int64_t)blockIdx.x * p.keep;
#pragma unroll
  for (int c = 0; c < PER; c += 4)
    if (c / 4 < groups) {
      uint4_t b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = bits[wave * 4 * groups + c + i];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = (int)(b[i][2] + __builtin_amdgcn_mbcnt_hi(
                                           b[i][1], __builtin_amdgcn_mbcnt_lo(b[i][0], 0)));
        const bool is = ((lane < 32 ? b[i][0] : b[i][1]) >> (lane & 31)) & 1;
        if (is && at < p.keep) out[at] = e0 + 64 * (c + i) + lane;
      }
    }
  if (tid == 0) p.nnz[blockIdx.x] = p.keep;
}

// Rows of any length, read again for each pass.
__global__ __launch_bounds__(kHThreads) void kept_heaviest_long_kernel(HeavyParams p) {
  constexpr int NC = 8;
  __shared__ HeavyLds<kHThreads, NC> lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  HeavyRow r;
  if (!heavy_row<kHThreads>(p, r)) return;
  const int len = r.len, lo = r.lo, hi = r.hi;
  int32_t* const out = p.ind + (int64_t)blockIdx.x * p.keep;
  // The entries from e on that this lane looks at (entries past the row's end read as 0).
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)r.w, 0, len * 4, kBufferWord3);
  auto load = [&](int e) {
    return as_float4u(
        __builtin_bit_cast(uint4_t, __builtin_amdgcn_raw_buffer_load_b128(rsrc, e * 4, 0, 0)));
  };
  const HeavyKey f =
      find_key<kHThreads, NC>(lds, (uint32_t)(p.keep - p.first - p.recent), [&](auto add) {
        constexpr int kAhead = 4;  // steps in flight
        for (int e = lo / kHRun * kHRun + tid * kHRun; e < hi; e += kAhead * kHStep) {
          float4_t x[kAhead];
#pragma unroll
          for (int s = 0; s < kAhead; ++s) x[s] = load(e + s * kHStep);
#pragma unroll
          for (int s = 0; s < kAhead; ++s)
#pragma unroll
            for (int i = 0; i < kHRun; ++i) {
              const int at = e + s * kHStep + i;
              if (at >= lo && at < hi) add(order_key(x[s][i]));
            }
        }
      });
  const uint32_t key = f.key, mask = f.mask;

  // ---- the kept entries in order: heavier than the key, or equal while any are wanted.
  const bool none = mask == 0;  // no candidate is kept
  int kept = 0, equal = 0;  // before this step
  const int wanted = (int)f.want;
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
      const uint32_t k = order_key(x[i]) & mask;
      const bool in = e + i >= lo && e + i < hi;
      const bool s = e + i < len && (!in || (!none && k > key));
      const bool q = in && !none && k == key;
      sure |= (s ? 1u : 0u) << i;
      same |= (q ? 1u : 0u) << i;
    }
    cnt = (uint32_t)__builtin_popcount(sure) | (uint32_t)__builtin_popcount(same) << 16;
    const uint32_t incl = wave_inclusive_scan(cnt);
    if (lane == 63) lds.tot[buf][wave] = incl;
    __syncthreads();
    uint32_t before = incl - cnt, total = 0;
#pragma unroll
    for (int i = 0; i < kHWaves; ++i) {
      const uint32_t t = lds.tot[buf][i];
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
  // Few threads to a short row have few bins and waves to meet; the registers hold what a row
  // needs (us, half of 32 rows of so many kept, 256 threads / 1024: 1,000 6.4 / 8.2, 2,000 7.3 /
  // 8.1, 4,000 9.7 / 8.6, 8,000 13.7 / 10.7; 32,000 with 32 / 64 entries to a thread 21.1 / 21.9; read
  // again for each pass 35.4, and of 65,000 65 against 36).
  KernelTimer timer;
  const dim3 grid((unsigned)(batch * num_heads));
  hipStream_t st = (hipStream_t)stream;
  auto large = [&](auto kernel) { timer.launch(kernel, grid, dim3(1024), 0, st, p); };
  if (row_len <= 2048) timer.launch(kept_heaviest_kernel<256, 8>, grid, dim3(256), 0, st, p);
  else if (row_len <= 16384) large(kept_heaviest_kernel<1024, 16>);
  else if (row_len <= 32768) large(kept_heaviest_kernel<1024, 32>);
  else if (row_len <= 65536) large(kept_heaviest_kernel<1024, 64>);
  else timer.launch(kept_heaviest_long_kernel, grid, dim3(kHThreads), 0, st, p);
  return check_launch("kept_heaviest_kernel");
}
