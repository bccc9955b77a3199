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
#include "akt_common.hpp"
#include "akt_host.hpp"
#include "attn_tile.hpp"
#include "paged_chunk.hpp"

namespace akt {
namespace {

constexpr int kJoinThreads = 256;

template <int D, bool BF16>
__global__ __launch_bounds__(kJoinThreads) void shared_join_kernel(ChunkParams p) {
  constexpr int CPR = D / 8;  // lanes to a row, 8 dims each
  const int rows = p.total_q * p.Hq;
  const int i = (int)(blockIdx.x * kJoinThreads + threadIdx.x);
  const int row = i / CPR, c = i % CPR;
  if (row >= rows) return;
  // Tokens of no sequence have no state.
  const int tok = (int)((uint32_t)row / (uint32_t)p.Hq);
  if (tok < p.q_indptr[0] || tok >= p.q_indptr[p.B]) return;
  const float4_t* ml = reinterpret_cast<const float4_t*>(p.states);
  const float* so = reinterpret_cast<const float*>(p.states + (int64_t)rows * 32);
  const float4_t own = ml[row];
  const float4_t* a = reinterpret_cast<const float4_t*>(so + (int64_t)row * D + 8 * c);
  const float4_t* b = reinterpret_cast<const float4_t*>(so + ((int64_t)rows + row) * D + 8 * c);
  float4_t o[2] = {a[0], a[1]};
  float m = own[0], l = own[1], x = own[2];
  if (l == 0.f) o[0] = o[1] = float4_t{0.f, 0.f, 0.f, 0.f};  // no key seen: not written
  if (own[3] != 0.f) {
    const float4_t pre = ml[rows + row];
    if (pre[1] != 0.f) {
      const float top = __builtin_elementwise_maximum(m, pre[0]);
      const float f = l == 0.f ? 0.f : fast_exp2(m - top), h = fast_exp2(pre[0] - top);
      m = top;
      l = f * l + h * pre[1];
      x = f * x + h * pre[2];
      o[0] = f * o[0] + h * b[0];
      o[1] = f * o[1] + h * b[1];
    }
  }
  const float inv = l == 0.f ? 0.f : __builtin_amdgcn_rcpf(l);
  typedef Elt<BF16> E;
  st16(p.o + (int64_t)row * D + 8 * c,
       uint4_t{E::pack2(o[0][0] * inv, o[0][1] * inv), E::pack2(o[0][2] * inv, o[0][3] * inv),
               E::pack2(o[1][0] * inv, o[1][1] * inv), E::pack2(o[1][2] * inv, o[1][3] * inv)});
  if (p.lse && c == 0)
    p.lse[row] = l == 0.f ? -__builtin_inff() : (m + __log2f(x)) * kLn2;
}

template <int D>
int launch_join(const ChunkParams& p, bool bf16, hipStream_t st) {
  const int64_t lanes = (int64_t)p.total_q * p.Hq * (D / 8);
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
