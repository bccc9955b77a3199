// Attention with shared prefixes over a paged KV cache (gfx950): the join of a row's two states.
//
// A row (token, query head) of a sequence in a group sees the group's prefix and its sequence's
// own keys.  paged_chunk_kernel serves both in one launch: a group's tokens together are one more
// sequence, whose keys are the prefix, so a prefix's K and V are read once for all rows of the
// group (matrix pipe: 4 D FLOPs a row and key) and its ranges are cut and balanced with those of the own
// keys.  Either part leaves, for each row, the maximum m of its scores (log2 units), the sums l and
// x of its rounded and unrounded 2^(s - m), and the sum a of P.V, all in 32 bits.  Here, with
// M = max(m_own, m_prefix) and f = 2^(m - M) for each:
//   O = (f_own a_own + f_prefix a_prefix) / (f_own l_own + f_prefix l_prefix),
//   LSE = (M + log2(f_own x_own + f_prefix x_prefix)) ln 2.
// HBM (or the caches)-bound: 8 D bytes read and 2 D written a row.
#include <type_traits>

#include "akt_common.hpp"
#include "akt_host.hpp"
#include "attn_tile.hpp"
#include "paged_chunk.hpp"

namespace akt {
namespace {

constexpr int kJoinThreads = 256;

template <int D, bool BF16>
__global__ __launch_bounds__(kJoinThreads) void shared_join_kernel(ChunkParams p) {
  constexpr int LPR = D / 4;  // lanes to a row, 4 dims each
  const int rows = p.total_q * p.Hq;
  const int i = (int)(blockIdx.x * kJoinThreads + threadIdx.x);
  const int row = i / LPR, c = i % LPR;
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
  if (tok < p.q_indptr[0] || tok >= p.q_indptr[p.B]) return;
  const bool more = __float_as_int(own[3]) & kStateMore;
#pragma unroll
  for (int src = 0; src < 2; ++src) {
    const float4_t s = src ? pre : own;
    const int tag = __float_as_int(s[3]);
    if (src && !more) break;
    if (!(tag & kStateCut)) {
      take(s, src ? pre_o : own_o);
      continue;
    }
    const int wf = __float_as_int(s[0]), wl = __float_as_int(s[1]), at = __float_as_int(s[2]);
    const bool many = tag & kStateMany;
    const int slot_rows = many ? 32 * chunk_waves(D) : 32;
    const char* const slots = p.partials + (many ? p.many_partial : 0);
    // So many parts in flight; repeats of the last one are not taken.
    auto batch = [&](int w, auto n_c) {
      constexpr int N = decltype(n_c)::value;
      float4_t ps[N], po[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int v = min(w + k, wl);
        const char* slot = slots + (2 * (int64_t)v + (v == wf ? 1 : 0)) * slot_rows * state_bytes(D);
        ps[k] = reinterpret_cast<const float4_t*>(slot)[at];
        po[k] = reinterpret_cast<const float4_t*>(slot + slot_rows * 16)[(int64_t)at * LPR + c];
      }
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (w + k <= wl) take(ps[k], po[k]);
    };
    int w = wf;
    for (; wl - w >= 4; w += 8) batch(w, std::integral_constant<int, 8>{});
    if (wl - w >= 2) batch(w, std::integral_constant<int, 4>{});
    else if (w <= wl) batch(w, std::integral_constant<int, 2>{});
  }
  const float inv = l == 0.f ? 0.f : __builtin_amdgcn_rcpf(l);
  typedef Elt<BF16> E;
  *reinterpret_cast<uint2*>(p.o + (int64_t)row * D + 4 * c) =
      uint2{E::pack2(o[0] * inv, o[1] * inv), E::pack2(o[2] * inv, o[3] * inv)};
  if (p.lse && c == 0)
    p.lse[row] = l == 0.f ? -__builtin_inff() : (m + __log2f(x)) * kLn2;
}

template <int D>
int launch_join(const ChunkParams& p, bool bf16, hipStream_t st) {
  const int64_t lanes = (int64_t)p.total_q * p.Hq * (D / 4);
  const dim3 grid((unsigned)ceil_div(lanes, kJoinThreads)), block(kJoinThreads);
  if (bf16) hipLaunchKernelGGL((shared_join_kernel<D, true>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((shared_join_kernel<D, false>), grid, block, 0, st, p);
  return check_launch("shared_join_kernel");
}

}  // namespace

int shared_merge_launch(const ChunkParams& p, int head_dim, bool bf16, hipStream_t st) {
  if (head_dim == 64) return launch_join<64>(p, bf16, st);
  if (head_dim == 256) return launch_join<256>(p, bf16, st);
  return launch_join<128>(p, bf16, st);
}

}  // namespace akt
