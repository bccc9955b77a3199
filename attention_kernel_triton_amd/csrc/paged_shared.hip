// Attention with shared prefixes over a paged KV cache (gfx950): the join of a row's two states.
//
// A row (token, query head) of a sequence in a group sees the group's prefix and its sequence's
// own keys.  paged_chunk_kernel serves both in one launch: a group's tokens together are one more
// sequence, whose keys are the prefix, so a prefix's K and V are read once for all rows of the
// group (matrix pipe: 4 D FLOPs a row and key) and its ranges are cut and balanced with those of the own
// keys.  Every part leaves, for each row, the maximum m of its scores (log2 units), the sums l and
// x of its rounded and unrounded 2^(s - m), and the sum a of P.V, all in 32 bits: in the row's place
// among the own keys' or the prefixes' states where a unit is one part, else in its range's slot,
// and the row's place says which ranges (state_row).  Here, over a row's parts i, with M = max m_i and
// f_i = 2^(m_i - M):
//   O = sum f_i a_i / sum f_i l_i,   LSE = (M + log2(sum f_i x_i)) ln 2.
// The parts are taken in their order, so the result does not depend on the run.
//
// Bound by memory (the caches, mostly): 4 D + 16 bytes read a part and row, 2 D written a row; with few
// rows by the round trips to the places, the slots, and the slots' later batches.  Joining in
// the kernel before by the last part to arrive cost more: the parts of a cut unit ended one by one,
// and the wave that came last joined all rows alone (a decode step of 32 sequences behind 4,096
// tokens: 50.6 us so, 28.3 now, 5 of them here; of 64 k rows in two or three parts 26 us of 325).
#include <type_traits>

#include "akt_common.hpp"
#include "akt_host.hpp"
#include "attn_tile.hpp"
#include "paged_chunk.hpp"

namespace akt {
namespace {

constexpr int kJoinThreads = 256;
// Up to so many threads' work, two share it: half the round trips where threads are few (us, one /
// two to a row's dims, the whole call: 256 threads 13.3 / 12.6, 32 k 33.6 / 32.2, 87 k 36.2 / 35.5,
// 131 k 81.8 / 82.4; four are no better than two).
constexpr int64_t kJoinPairLanes = 3 << 15;

// PG threads share the parts of a row's 4 dims: those of one thread are PG parts apart.
template <int D, bool BF16, int PG>
__global__ __launch_bounds__(kJoinThreads) void shared_join_kernel(ChunkParams p) {
  constexpr int LPR = D / 4;  // lanes to a row, 4 dims each
  constexpr int RPB = kJoinThreads / LPR / PG;  // rows to a workgroup
  static_assert(RPB >= 1, "a row's threads are in one workgroup");
  const int rows = p.total_q * p.Hq;
  const int pg = PG == 1 ? 0 : (int)threadIdx.x / (LPR * RPB);
  const int in = (int)threadIdx.x % (LPR * RPB);
  const int row_at = (int)blockIdx.x * RPB + in / LPR, c = in % LPR;
  const int row = PG == 1 ? row_at : min(row_at, rows - 1);
  if (row >= rows) return;
  const float4_t* const ml = reinterpret_cast<const float4_t*>(p.states);
  const float4_t* const so = reinterpret_cast<const float4_t*>(p.states + (int64_t)rows * 32);
  float m = -__builtin_inff(), l = 0.f, x = 0.f;
  float4_t o = {0.f, 0.f, 0.f, 0.f};
  // Takes a part in; one whose keys the row did not see (l = 0) has no sums.
  auto take = [&](float4_t s, float4_t a) {
    if (s[1] == 0.f) return;
    const float top = __builtin_elementwise_maximum(m, s[0]);
    const float f = l == 0.f ? 0.f : fast_exp2(m - top), h = fast_exp2(s[0] - top);
    m = top;
    l = f * l + h * s[1];
    x = f * x + h * s[2];
    o = f * o + h * a;
  };
  const float4_t own = ml[row], pre = ml[rows + row];
  const float4_t own_o = so[(int64_t)row * LPR + c], pre_o = so[((int64_t)rows + row) * LPR + c];
  // Tokens of no sequence have no state.
  const int tok = (int)((uint32_t)row / (uint32_t)p.Hq);
  const bool none = tok < p.q_indptr[0] || tok >= p.q_indptr[p.B];
  if (PG == 1 && none) return;
  const bool more = __float_as_int(own[3]) & kStateMore;
#pragma unroll
  for (int src = 0; src < 2; ++src) {
    const float4_t s = src ? pre : own;
    const int tag = __float_as_int(s[3]);
    if (none || (src && !more)) break;
    if (!(tag & kStateCut)) {
      if (pg == src % PG) take(s, src ? pre_o : own_o);
      continue;
    }
    // A row that no part wrote (q_indptr not in order) holds anything: what it names is kept within
    // the slots.
    const bool many = (tag & kStateMany) && (p.kinds & kCkMany);
    const int slot_rows = many ? 32 * chunk_waves(D) : 32;
    const int ranges = many ? p.wgs : p.wgs * chunk_waves(D);
    const int wf = min(max(__float_as_int(s[0]), 0), ranges), wl = min(__float_as_int(s[1]), ranges - 1);
    const int at = min(max(__float_as_int(s[2]), 0), slot_rows - 1);
    const char* const slots = p.partials + (many ? p.many_partial : 0);
    // So many parts in flight; repeats of the last one are not taken.
    auto batch = [&](int w, auto n_c) {
      constexpr int N = decltype(n_c)::value;
      float4_t ps[N], po[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int v = min(w + k * PG, wl);
        const char* slot = slots + (2 * (int64_t)v + (v == wf ? 1 : 0)) * slot_rows * state_bytes(D);
        ps[k] = reinterpret_cast<const float4_t*>(slot)[at];
        po[k] = reinterpret_cast<const float4_t*>(slot + slot_rows * 16)[(int64_t)at * LPR + c];
      }
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (w + k * PG <= wl) take(ps[k], po[k]);
    };
    int w = wf + pg;
    for (; wl - w >= 4 * PG; w += 8 * PG) batch(w, std::integral_constant<int, 8>{});
    if (wl - w >= 2 * PG) batch(w, std::integral_constant<int, 4>{});
    else if (w <= wl) batch(w, std::integral_constant<int, 2>{});
  }
  if constexpr (PG > 1) {
    __shared__ float4_t sm_ml[kJoinThreads], sm_o[kJoinThreads];
    sm_ml[threadIdx.x] = float4_t{m, l, x, 0.f};
    sm_o[threadIdx.x] = o;
    __syncthreads();
    if (pg || row_at >= rows || none) return;
#pragma unroll
    for (int k = 1; k < PG; ++k) take(sm_ml[k * LPR * RPB + in], sm_o[k * LPR * RPB + in]);
  }
  const float inv = l == 0.f ? 0.f : __builtin_amdgcn_rcpf(l);
  typedef Elt<BF16> E;
  *reinterpret_cast<uint2*>(p.o + (int64_t)row * D + 4 * c) =
      uint2{E::pack2(o[0] * inv, o[1] * inv), E::pack2(o[2] * inv, o[3] * inv)};
  if (p.lse && c == 0)
    p.lse[row] = l == 0.f ? -__builtin_inff() : (m + __log2f(x)) * kLn2;
}

template <int D, bool BF16>
int launch_join(const ChunkParams& p, hipStream_t st) {
  const int64_t lanes = (int64_t)p.total_q * p.Hq * (D / 4);
  const dim3 block(kJoinThreads);
  KernelTimer timer;
  if (lanes <= kJoinPairLanes) {
    const dim3 grid((unsigned)ceil_div(lanes * 2, kJoinThreads));
    timer.launch(shared_join_kernel<D, BF16, 2>, grid, block, 0, st, p);
  } else {
    const dim3 grid((unsigned)ceil_div(lanes, kJoinThreads));
    timer.launch(shared_join_kernel<D, BF16, 1>, grid, block, 0, st, p);
  }
  return check_launch("shared_join_kernel");
}
template <int D>
int launch_join(const ChunkParams& p, bool bf16, hipStream_t st) {
  return bf16 ? launch_join<D, true>(p, st) : launch_join<D, false>(p, st);
}

}  // namespace

int shared_merge_launch(const ChunkParams& p, int head_dim, bool bf16, hipStream_t st) {
  if (head_dim == 64) return launch_join<64>(p, bf16, st);
  if (head_dim == 256) return launch_join<256>(p, bf16, st);
  return launch_join<128>(p, bf16, st);
}

}  // namespace akt
