// Attention of a chunk of new tokens over a paged KV cache (gfx950).
//
// Sequence b has n_b query tokens (rows q_indptr[b] .. q_indptr[b + 1] of q) and len_b
// cached tokens (the page table's count, its new ones among them).  Query i sits at
// position len_b - n_b + i and sees the keys up to its own position (causal) or all
// len_b (not causal):
//   O = softmax(scale q K^T) V,  LSE = ln sum_j exp(scale q.k_j).
// It serves chunked prefill, the verification of drafted tokens, mixed batches and
// single-token decode in one launch.  What bounds it is HBM (K and V once) while a kv head has
// few rows, the matrix pipe when it has many.
//
// Units.  The rows of one (sequence, kv head) are its (token, query head of the group)
// pairs, token major; a unit is a run of up to 32 chunk_waves rows (256; 128 at D = 256) of
// whole tokens, which share every K and V row.  Sequences of up to chunk_split_rows rows to a kv head
// (few tokens) and those of more (many) are served differently:
// - many: wave w of a workgroup owns rows 32 w .. 32 w + 31, and all waves walk the same keys,
//   staged in LDS once for all of them;
// - few: there are rows for one wave only (two at D = 256), so four waves (a team) share out the
//   keys, each loading its own, and merge at the part's end.
//
// Ranges.  The units of a kind stand one behind another on an axis of keys (sequence by sequence,
// kv head by kv head, row block by row block), each as long as the keys it sees plus
// kCkUnitCost for its start and end.  The axis is cut into equal ranges, one to a workgroup
// (many) or team (few), so a launch is balanced whatever the mix of chunk and context lengths,
// and nothing of it has to be known on the host: every wave computes the axis's length and its
// own place on it from the tables (a scan over the sequences, 64 at a time).  Where both kinds
// can occur the workgroups are shared between them by the lengths of the two axes, which every
// workgroup computes alike (split_share).  A unit is
// cut only at multiples of kCkBlock keys from its start: block kb of a unit that
// starts at U belongs to the range that holds U + kb + kCkBlock - 1.  With
// ranges of at least kCkBlock that gives every range of a cut unit at least one
// block, and no two cut units start in the same range, so the first one's
// number names the unit's arrival counters.  Range x's partial of a unit that started
// before it is slot 2 x, of one that starts in it slot 2 x + 1.
//
// Merge.  Waves store their partial O, m and l with device-scope stores, wait for them,
// and count themselves on the counter of (unit, wave); the last one merges all partials
// in the order of the ranges (not of arrival, so results do not depend on it) and
// leaves the counter at zero.  Nothing waits for another workgroup.
//
// Shared prefixes (SHARED).  A group's tokens together are one more sequence behind the others, whose
// keys are the prefix, seen whole by every row.  Every part leaves a state (state_row), a second
// kernel joins them (paged_shared.hip), and units of few rows are served by paged_shared_few.hpp.
// At D = 128 these instances spill 5 to 27 vector registers, outside the walks over keys but for
// three reloads a block in the one with pages that are not whole 16-token groups and with the LSE.
//
// Tiles (many).  As in the dense prefill kernel: K and V tiles go global -> registers -> one
// of four LDS buffers, three tiles ahead; both products run transposed so that a lane owns
// a row; the running max is raised only when a step's sum says so.  The page ids of a tile
// are loaded by every wave a tile before its rows, one id to a lane; pages of whole
// 16-token groups put each wave's loads on one page, whose base is then scalar.
// Keys past the unit's last one and keys of pages outside the pool read as zeros
// and score -inf.
//
// P in 16 bits.  P.V takes P in V's type (an MFMA's operands share one; what the rounding leaves would
// take a second product).  The normaliser sums the rounded P, so that numerator and normaliser
// round alike; sums are fp32, and the LSE sums the unrounded P.  Errors against 64 bits
// are up to 1.4 times those of 32-bit P (fp16 2.9e-4 / 2.1e-4, bf16 2.4e-3 / 1.7e-3, most of it
// the output's own rounding).
//
// Masked values.  Scores are masked with a select.  V rows that some of the unit's rows see
// and some do not are multiplied by zeros too, which an infinity or NaN in V would turn into
// NaN: in tiles (steps, where waves share out the keys) that hold such rows, infinities and NaNs
// are staged as zeros, and in the rare unit that has any they are added at its end to the rows that
// see them (add_not_finite), from the first key of the first such tile on.  Elsewhere they go
// through the product (where an infinity whose probability rounds to 0 in the type becomes NaN).
//
// Measured (us a call among others; D = 128, 8 kv heads unless said): 32 single tokens over 255
// to 8191 keys 89 (389 MB, 4.36 TB/s); 3 to 7 drafted tokens of 16 sequences, 64 query heads, 58
// (2.8 TB/s: starts and merges beside a few steps a wave); 777 new tokens beside 15 single ones
// 65; 2048 tokens after 30000, 32 query heads, bf16 993 to 1045 (1.0 PFLOP/s, matrix pipe 48% busy);
// D = 256, 4 kv heads, 100 to 300 tokens, not causal, 61 (293 TFLOP/s: one wave a SIMD, 17% busy,
// 312 partials of 76 units); 777 tokens after 2000, 32 query heads, 63 (479 TFLOP/s: 344 partials of
// 104 units); D = 64, 16 kv heads, 8 x 1024 tokens 140 (491 TFLOP/s).
#include <float.h>
#include <math.h>

#include <cmath>
#include <type_traits>

#include "akt_host.hpp"
#include "attn_tile.hpp"
#include "paged_chunk.hpp"

namespace akt {
namespace {

constexpr int kCkNBuf = 4;  // LDS tile buffers
constexpr float kCkSlack = 8.0f;  // log2 units a row's max may rise before it is rescaled
constexpr float kCkStepLimit = 32.0f * 256.0f;  // row sum of a step that stays unchecked
// Running max of a row that has seen no key: finite, so that exp2(-inf - m) is 0.
constexpr float kCkFloor = -1e30f;
#define AKT_C_NEG_INF (-__builtin_inff())

__host__ __device__ constexpr int ck_tile_keys(int D) { return D <= 128 ? 64 : 32; }
__host__ __device__ constexpr int ck_mix_mfma(int D) { return D == 64 ? 8 : (D == 128 ? 10 : 16); }
__host__ __device__ constexpr int ck_mix_valu(int D) { return D == 128 ? 1 : 2; }

__device__ __forceinline__ int64_t uniform64(int64_t v) {
  const uint32_t lo = (uint32_t)uniform((int)(uint32_t)v);
  const uint32_t hi = (uint32_t)uniform((int)(uint32_t)(v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ int64_t shfl64(int64_t v, int src) {
  return (int64_t)(((uint64_t)shfl_u((uint32_t)(v >> 32), src) << 32) | shfl_u((uint32_t)v, src));
}
// floor(a / b) for 0 <= a < 2^50, b >= 1: doubles hold both, and the quotient's distance
// to the next integer (at least 1 / b) is more than its rounding.
__device__ __forceinline__ int64_t div_range64(int64_t a, int64_t b) {
  return uniform64((int64_t)((double)a / (double)b));
}
__device__ __forceinline__ int div_range(int64_t a, int64_t b) {
  return uniform((int)((double)a / (double)b));
}

template <bool SHARED>
struct Seq {
  int q0, n;    // first query row, query tokens
  int ip0, len;  // first page table entry, cached tokens
};
// In a launch with shared prefixes a group's tokens together are a sequence too, whose keys are
// the prefix: it has a table of its own, and every token sees all of it.
template <>
struct Seq<true> {
  int q0, n, ip0, len;
  int prefix;  // a group and its prefix
  int more;    // a sequence of a group: its rows have a prefix's state too
};
template <typename S>
__device__ __forceinline__ int is_prefix(const S& s) {
  return s.prefix;
}
__device__ __forceinline__ int is_prefix(const Seq<false>&) { return 0; }
template <bool SHARED>
__device__ __forceinline__ int num_seqs(const ChunkParams& p) {
  return SHARED ? p.B + p.groups : p.B;
}
// With shared prefixes a workgroup keeps the sequences' places in LDS, unless there are too many.
constexpr int kCkTable = 1024;
__device__ __forceinline__ bool in_table(const ChunkParams& p) {
  return p.B + p.groups <= kCkTable;
}
// Table entries outside their ranges are taken clamped, so nothing outside the arrays is
// touched.
struct Prefix {
  int b0, b1, ip0, len;  // sequences b0 .. b1 - 1, first page table entry, tokens
};
__device__ __forceinline__ Prefix load_prefix(const ChunkParams& p, int i) {
  Prefix x;
  x.b0 = min(max(p.group_indptr[i], 0), p.B);
  x.b1 = min(max(p.group_indptr[i + 1], x.b0), p.B);
  x.ip0 = min(max(p.prefix_indptr[i], 0), p.prefix_pages);
  const int np = min(max(p.prefix_indptr[i + 1], x.ip0), p.prefix_pages) - x.ip0;
  x.len = np > 0 ? (np - 1) * p.page_size + min(max(p.prefix_last[i], 0), p.page_size) : 0;
  return x;
}
template <bool SHARED>
__device__ __forceinline__ Seq<SHARED> load_seq(const ChunkParams& p, int b,
                                                const int4* table = nullptr) {
  Seq<SHARED> s;
  if constexpr (SHARED) {
    s.prefix = b >= p.B;
    if (table) {
      const int4 t = table[b];
      return Seq<SHARED>{t.x, t.y & 0x3fffffff, t.z, t.w, s.prefix, t.y >> 30};
    }
    s.more = !s.prefix && p.groups > 0 && b >= p.group_indptr[0] && b < p.group_indptr[p.groups];
    if (s.prefix) {
      const Prefix x = load_prefix(p, b - p.B);
      s.q0 = min(max(p.q_indptr[x.b0], 0), p.total_q);
      s.n = x.b1 > x.b0 ? min(max(p.q_indptr[x.b1], s.q0), p.total_q) - s.q0 : 0;
      s.ip0 = x.ip0;
      s.len = x.len;
      return s;
    }
  }
  s.q0 = min(max(p.q_indptr[b], 0), p.total_q);
  s.n = min(max(p.q_indptr[b + 1], s.q0), p.total_q) - s.q0;
  s.ip0 = min(max(p.indptr[b], 0), p.total_pages);
  const int np = min(max(p.indptr[b + 1], s.ip0), p.total_pages) - s.ip0;
  s.len = np > 0 ? (np - 1) * p.page_size + min(max(p.last_len[b], 0), p.page_size) : 0;
  return s;
}
// The same for a wave-uniform b, in scalar registers.
template <bool SHARED>
__device__ __forceinline__ Seq<SHARED> load_seq_uniform(const ChunkParams& p, int b,
                                                        const int4* table) {
  const Seq<SHARED> s = load_seq<SHARED>(p, b, table);
  if constexpr (SHARED)
    return Seq<SHARED>{uniform(s.q0), uniform(s.n), uniform(s.ip0), uniform(s.len), uniform(s.prefix),
                       uniform(s.more)};
  else
    return Seq<SHARED>{uniform(s.q0), uniform(s.n), uniform(s.ip0), uniform(s.len)};
}
__device__ __forceinline__ int row_blocks(const ChunkParams& p, int n) {
  return (int)(((uint32_t)n + p.TR - 1) / (uint32_t)p.TR);
}
// Whether a row of the sequence (unit) sees the keys up to its own position only.
template <typename S>
__device__ __forceinline__ bool is_causal(const ChunkParams& p, const S& s) {
  return p.causal && !is_prefix(s);
}
template <bool SHARED>
__device__ __forceinline__ constexpr int unit_cost() {
  return SHARED ? kSharedUnitCost : kCkUnitCost;
}
// Lengths on the axis.  Causal row block r sees min(n, (r + 1) TR) keys past the context;
// the axis takes the context as at least 0 (a table with n > len breaks the contract).
template <bool SHARED>
__device__ __forceinline__ int64_t unit_start(const ChunkParams& p, const Seq<SHARED>& s, int64_t r) {
  if (!is_causal(p, s)) return r * (s.len + unit_cost<SHARED>());
  return r * (max(s.len - s.n, 0) + unit_cost<SHARED>()) + p.TR * (r * (r + 1) / 2);
}
template <bool SHARED>
__device__ __forceinline__ int64_t head_length(const ChunkParams& p, const Seq<SHARED>& s) {
  const int64_t R = row_blocks(p, s.n);
  if (R == 0) return 0;
  if (!is_causal(p, s)) return R * (s.len + unit_cost<SHARED>());
  return unit_start(p, s, R - 1) + max(s.len - s.n, 0) + s.n + unit_cost<SHARED>();
}
// n / page_size for 0 <= n < 2^31.
__device__ __forceinline__ int page_of(const ChunkParams& p, int n) {
  const int q = (int)__umulhi((uint32_t)n, p.page_magic);
  return n - q * p.page_size >= p.page_size ? q + 1 : q;
}

// A unit and the part of its keys that a workgroup serves.
template <bool SHARED>
struct Unit {
  int q0;     // first query row (token) in q
  int ntok;   // its tokens
  int kvh;    // kv head
  int first;  // position of its first token (non-causal: unused)
  int len;    // cached tokens of the sequence
  int kend;   // keys that it sees
  int ip0;    // first page table entry of the sequence
};
template <>
struct Unit<true> {
  int q0, ntok, kvh, first, len, kend, ip0;
  int prefix;  // a group's rows and its prefix's keys
  int more;    // the rows have a prefix's state too (own keys)
};
__device__ __forceinline__ int is_prefix(const Unit<false>&) { return 0; }
__device__ __forceinline__ const int32_t* page_ids(const ChunkParams& p, const Unit<false>&) {
  return p.indices;
}
__device__ __forceinline__ const int32_t* page_ids(const ChunkParams& p, const Unit<true>& u) {
  return u.prefix ? p.prefix_indices : p.indices;
}

// Where a part of a unit leaves a row's state (m, l, exact l, tag) and its sums of P.V: a unit
// that is one part in the row's place (at: token, query head) among the own keys' or the prefixes'
// rows, a part of a cut one in its range's slot; the first part then leaves the ranges of the
// unit's first and last part and the row's place in their slots instead.
struct StateRow {
  float4_t* ml;
  float* o;
  float tag;
};
__device__ __forceinline__ float4_t* state_ml(const ChunkParams& p, const Unit<true>& u) {
  return reinterpret_cast<float4_t*>(p.states) + (u.prefix ? (int64_t)p.total_q * p.Hq : 0);
}
template <int D>
__device__ __forceinline__ StateRow state_row(const ChunkParams& p, const Unit<true>& u, int64_t at,
                                              bool whole, bool first, int range, int64_t start,
                                              int64_t Lw, int block, bool many, int slot_rows,
                                              int row) {
  const int tag = u.more ? kStateMore : 0;
  if (whole) {
    const int64_t rows = (int64_t)p.total_q * p.Hq;
    return StateRow{state_ml(p, u) + at,
                    reinterpret_cast<float*>(p.states + rows * 32) + ((u.prefix ? rows : 0) + at) * D,
                    __int_as_float(tag)};
  }
  const int last = (u.kend - 1) / block * block;
  const int wf = div_range(start + block - 1, Lw), wl = div_range(start + last + block - 1, Lw);
  if (first)
    state_ml(p, u)[at] = float4_t{__int_as_float(wf), __int_as_float(wl), __int_as_float(row),
                                  __int_as_float(tag | kStateCut | (many ? kStateMany : 0))};
  char* const slot =
      p.partials + (many ? p.many_partial : 0) + (2 * (int64_t)range + (range == wf ? 1 : 0)) * slot_rows * state_bytes(D);
  return StateRow{reinterpret_cast<float4_t*>(slot) + row,
                  reinterpret_cast<float*>(slot + slot_rows * 16) + (int64_t)row * D, 0.f};
}

// Scores of the keys that a row does not see become -inf: of the step's 32 those past its
// first room + 1, and those whose bit of `valid` is 0.
__device__ __forceinline__ void mask_scores(float16_t& s, uint32_t valid, int room, int g) {
  const uint32_t see = room < 0 ? 0u : valid & (0xffffffffu >> (31 - min(room, 31)));
  const uint32_t mine = see >> (4 * g);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int keep = __builtin_amdgcn_sbfe((int)mine, 8 * (i >> 2) + (i & 3), 1);  // 0 or -1
    s[i] = __int_as_float((__float_as_int(s[i]) & keep) | (0xff800000 & ~keep));
  }
}

// Takes a partial's (m, l, x) into a row's running ones, rescaling what is summed so far where
// m is a new maximum; returns the factor of the partial's O.
template <typename F>
__device__ __forceinline__ float merge_in(float4_t ml, float& m, float& l, float& x, F rescale) {
  if (ml[0] > m) {
    const float sc = fast_exp2(m - ml[0]);  // 0 for the first
    rescale(sc);
    l *= sc;
    x *= sc;
    m = ml[0];
  }
  const float f = fast_exp2(ml[0] - m);
  l += f * ml[1];
  x += f * ml[2];
  return f;
}

// Replaces infinities and NaNs by zeros; returns whether any lane of the wave had one.
template <bool BF16, int N>
__device__ __forceinline__ bool zero_not_finite(uint4_t (&v)[N]) {
  typedef unsigned short ushort2_v __attribute__((ext_vector_type(2)));
  constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
  ushort2_v top = {0, 0};
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int w = 0; w < 4; ++w)
      top = __builtin_elementwise_max(top, __builtin_bit_cast(ushort2_v, v[i][w] & 0x7fff7fffu));
  const bool any = __any(top.x >= kExp || top.y >= kExp);
  if (any) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t lo = (v[i][w] & kExp) == kExp ? 0xffff0000u : ~0u;
        const uint32_t hi = (v[i][w] & (kExp << 16)) == (kExp << 16) ? 0x0000ffffu : ~0u;
        v[i][w] &= lo & hi;
      }
  }
  return any;
}

// Adds the infinities and NaNs of keys j0 .. j1 - 1 of V, which were staged as zeros, to the O
// of the rows that see them (a key's probability is positive).  Lane (l32, g) holds dims
// 32 n + 8 k + 4 g .. + 3 of row l32, whose last key is lim.
template <int D, bool BF16, bool SHARED>
__device__ __forceinline__ void add_not_finite(const ChunkParams& p, const Unit<SHARED>& u, int j0, int j1,
                                               int g, int lim, float16_t (&oacc)[D / 32]) {
  constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
#pragma clang loop unroll(disable)
  for (int j = j0; j < j1; ++j) {
    const int lp = page_of(p, j), id = page_ids(p, u)[u.ip0 + lp];
    if ((uint32_t)id >= (uint32_t)p.num_pool_pages || j > lim) continue;
    const half_t* row = p.pool + id * p.sp + p.skv + u.kvh * p.sh +
                        (int64_t)(j - lp * p.page_size) * p.ss + 4 * g;
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint2 v = *reinterpret_cast<const uint2*>(row + 32 * n + 8 * k);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t x = ((i < 2 ? v.x : v.y) >> (16 * (i & 1))) & 0xffffu;
          float f;
          if constexpr (BF16) f = __uint_as_float(x << 16);
          else f = (float)__builtin_bit_cast(half_t, (uint16_t)x);
          oacc[n][4 * k + i] += (x & kExp) == kExp ? f : 0.f;
        }
      }
  }
}

// The units of the ranges of workgroup `block` of W, on the axis of the sequences of few tokens
// (SPLIT) or of many.  lds: the workgroup's tile buffers.  total: the axis's length, where prefixes
// are shared.
template <int D, bool BF16, bool GRP, bool LSE, bool SHARED, bool SPLIT>
__device__ __forceinline__ void chunk_range(const ChunkParams& p, char* lds, const int4* table,
                                            int block, int W, int64_t total = 0) {
  constexpr int WAVES = chunk_waves(D);
  typedef Elt<BF16> E;
  typedef typename E::v8 v8;
  constexpr int kThreads = 64 * WAVES;
  constexpr int kBN = ck_tile_keys(D);  // keys per staged tile
  constexpr int KS = D / 16;            // MFMA k-steps over the head dim
  constexpr int HALF = D / 2;
  constexpr int NT = D / 32;       // 32-dim output tiles
  constexpr int CPR = D / 8;       // 16-byte chunks per row
  constexpr int ROWB = D * 2;      // bytes per row
  constexpr int TILEB = kBN * ROWB;
  constexpr int BUFB = 2 * TILEB;  // K then V
  constexpr int PER_T = kBN * CPR / kThreads;  // chunks per thread per matrix
  constexpr int RPC = 64 / CPR;                  // rows of a wave's 64 chunks
  static_assert(16 % RPC == 0, "a wave's chunks lie in one 16-key group");
  // Waves that serve a range: all of a workgroup's, or, where they share out the keys, four, so
  // that one range's start and merge overlap with another's loads on the same CU.
  constexpr int TW = SPLIT ? 4 : WAVES;
  __shared__ float4_t sm_ml[WAVES][32];
  __shared__ int sm_bad[WAVES];
  __shared__ int sm_team[WAVES / TW];  // arrivals of each team at its barriers

  const int tid0 = threadIdx.x;
  const int wave = uniform(tid0 >> 6);

  // ---- this workgroup's (team's) range of the axis.  Workgroup i runs on XCD i % 8, so
  // consecutive ranges go to one XCD's L2; the second teams have the axis's second half, which
  // leaves them idle where it is cut into one range to a workgroup.
  const int team = SPLIT ? wave / TW : 0, twave = wave - team * TW;
  const int wg = team * W + (block % 8) * (W / 8) + block / 8;
  const int lane0 = tid0 & 63;
  // The sequences that this kernel serves.
  auto mine = [&](const Seq<SHARED>& s) { return s.n > 0 && (s.n <= p.split_tokens) == SPLIT; };
  auto seq_length = [&](int b) -> int64_t {
    if (b >= num_seqs<SHARED>(p)) return 0;
    const Seq<SHARED> s = load_seq<SHARED>(p, b, table);
    return mine(s) ? head_length(p, s) * p.Hkv : 0;
  };
  auto scan64 = [&](int64_t v) -> int64_t {  // inclusive sum over the lanes
    if constexpr (SHARED) return wave_inclusive_scan64(v);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int64_t u = shfl64(v, lane0 - d < 0 ? 0 : lane0 - d);
      if (lane0 >= d) v += u;
    }
    return v;
  };
  int64_t Lw = 0, x0 = 0, x1 = 0;
  const int ranges = W * (WAVES / TW);
  if (SPLIT && WAVES > TW) {
    if (tid0 < WAVES / TW) sm_team[tid0] = 0;
    __syncthreads();
  }
  // Barrier of a team's waves: each counts itself in, and waits until all have (they are of
  // one workgroup, and none waits for anything but its team).
  int team_target = 0;
  auto team_sync = [&]() {
    if constexpr (WAVES == TW) {
      __syncthreads();
    } else {
      team_target += TW;
      if (lane0 == 0)
        __hip_atomic_fetch_add(&sm_team[team], 1, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_WORKGROUP);
      while (uniform(__hip_atomic_load(&sm_team[team], __ATOMIC_ACQUIRE,
                                       __HIP_MEMORY_SCOPE_WORKGROUP)) < team_target)
        __builtin_amdgcn_s_sleep(1);
    }
  };
  const float c = p.qk_scale;
  // ---- the keys [k0, k1) of a unit of many rows, by all waves.
  auto serve = [&](const Unit<SHARED>& u, int k0, int k1, int64_t Ustart) {
    // The lane number is opaque here, so that what is derived from it lives no longer than
    // this part (held across the units' loop it would not fit the registers).
    int lane = tid0 & 63;
    asm volatile("" : "+v"(lane));
    const int l32 = lane & 31, g = lane >> 5, tid = 64 * wave + lane;
    // K rows for S^T: key l32 of the step, chunks g * HALF / 8 + s.
    int koff[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) koff[k] = l32 * ROWB + (((g * HALF / 8) + k) ^ tswz<D>(l32)) * 16;
    // V^T through the transposing read: see prefill_kernel.
    const int s16 = lane & 15;
    const int vrow = 4 * g + (s16 >> 2);
    const int vcl = 2 * ((lane >> 4) & 1) + ((s16 & 3) >> 1);
    int voff[NT], voffh[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      voff[n] = TILEB + vrow * ROWB + (((4 * n + vcl) ^ tswz<D>(vrow)) * 16) + (s16 & 1) * 8;
      voffh[n] =
          TILEB + (vrow + 8) * ROWB + (((4 * n + vcl) ^ tswz<D>(vrow + 8)) * 16) + (s16 & 1) * 8;
    }
    const int lrow = 32 * wave + l32;                          // this lane's row of the unit
    const int ltok = (int)((uint32_t)lrow * p.g_magic >> 16);  // and its token
    const int rows = u.ntok * p.G;
    const bool active = 32 * wave < rows;
    const bool whole = k0 == 0 && k1 == u.kend;
    const int nb = (k1 - k0 + 63) / 64;  // blocks of 64 keys: two steps
    const int n_tiles = 64 / kBN * nb;
    const half_t* const Kh = p.pool + u.kvh * p.sh;

    // Places of the keys, a block of 64 at a time: lane l holds key l's.
    struct Keys {
      int lo, hi;   // byte offset of its K row from Kh
      uint64_t ok;  // keys that can be read: before the unit's end, on pages of the pool
    };
    int id_next, slot_next;  // of the block whose ids are on their way
    auto load_ids = [&](int m) {
      const int key = min(k0 + 64 * m + lane, u.kend - 1);
      const int lp = page_of(p, key);
      slot_next = key - lp * p.page_size;
      id_next = page_ids(p, u)[u.ip0 + lp];
    };
    auto place = [&](int m) -> Keys {
      const bool ok =
          k0 + 64 * m + lane < u.kend && (uint32_t)id_next < (uint32_t)p.num_pool_pages;
      const int64_t off = ok ? 2 * (id_next * p.sp + (int64_t)slot_next * p.ss) : 0;
      return Keys{(int)(uint32_t)off, (int)(uint32_t)((uint64_t)off >> 32), __ballot(ok)};
    };
    uint4_t kst[PER_T], vst[PER_T];
    // Rows of a tile whose first key is key `first` (0 or 32) of its block.
    auto load_tile = [&](const Keys& keys, int first, uint4_t (&kd)[PER_T], uint4_t (&vd)[PER_T]) {
      if constexpr (GRP) {
        // Each of this wave's loads takes RPC rows, which lie in one page.
        const uint32_t off = (uint32_t)((lane / CPR) * p.ss * 2 + (lane % CPR) * 16);
        const char* base[PER_T];
#pragma unroll
        for (int i = 0; i < PER_T; ++i) {
          const int row = first + (wave * 64 + i * kThreads) / CPR;
          base[i] = (const char*)Kh +
                    (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane(keys.hi, row) << 32) |
                              (uint32_t)__builtin_amdgcn_readlane(keys.lo, row));
        }
        const bool full = kBN == 64 ? keys.ok == ~0ull : (uint32_t)(keys.ok >> first) == ~0u;
        if (full) {
#pragma unroll
          for (int i = 0; i < PER_T; ++i) {
            kd[i] = ld16(base[i] + off);
            vd[i] = ld16(base[i] + 2 * p.skv + off);
          }
        } else {
#pragma unroll
          for (int i = 0; i < PER_T; ++i) {
            const int row = first + (wave * 64 + i * kThreads) / CPR;
            const int n = __builtin_popcount((uint32_t)(keys.ok >> row) & ((1u << RPC) - 1));
            const int bytes = n > 0 ? (n - 1) * p.ss * 2 + ROWB : 0;
            const auto kr =
                __builtin_amdgcn_make_buffer_rsrc((void*)base[i], 0, bytes, kBufferWord3);
            const auto vr = __builtin_amdgcn_make_buffer_rsrc((void*)(base[i] + 2 * p.skv), 0,
                                                              bytes, kBufferWord3);
            kd[i] =
                __builtin_bit_cast(uint4_t, __builtin_amdgcn_raw_buffer_load_b128(kr, off, 0, 0));
            vd[i] =
                __builtin_bit_cast(uint4_t, __builtin_amdgcn_raw_buffer_load_b128(vr, off, 0, 0));
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < PER_T; ++i) {
          const int row = first + (tid + i * kThreads) / CPR;
          const uint32_t lo = shfl_u((uint32_t)keys.lo, row), hi = shfl_u((uint32_t)keys.hi, row);
          kd[i] = vd[i] = uint4_t{0, 0, 0, 0};
          if ((keys.ok >> row) & 1) {
            const char* src = (const char*)Kh + (int64_t)(((uint64_t)hi << 32) | lo) +
                              (tid + i * kThreads) % CPR * 16;
            kd[i] = ld16(src);
            vd[i] = ld16(src + 2 * p.skv);
          }
        }
      }
    };
    // Tile j, whose first key is k0 + kBN j, into the buffer at LDS offset buf.
    bool bad = false;
    auto store_tile = [&](int j, int buf, const uint4_t (&kd)[PER_T], uint4_t (&vd)[PER_T]) {
      if (is_causal(p, u) && k0 + (j + 1) * kBN > u.first + 1)  // keys that not every row sees
        bad |= zero_not_finite<BF16>(vd);
#pragma unroll
      for (int i = 0; i < PER_T; ++i) {
        const int ch = tid + i * kThreads;
        const int row = ch / CPR, cc = ch % CPR;
        const int off = buf + row * ROWB + ((cc ^ tswz<D>(row)) * 16);
        *reinterpret_cast<uint4_t*>(lds + off) = kd[i];
        *reinterpret_cast<uint4_t*>(lds + TILEB + off) = vd[i];
      }
    };

    // Last key of this lane's row (rows past the unit's: of its last token), and the
    // first of the wave's rows' last keys, up to which nothing is masked.
    const int lim = is_causal(p, u) ? u.first + min(ltok, u.ntok - 1) : u.len - 1;
    const int lim_min =
        is_causal(p, u) ? u.first + min((int)((uint32_t)(32 * wave) * p.g_magic >> 16), u.ntok - 1)
                 : u.len - 1;

    // ---- Q^T fragments: lane -> row, dims g*HALF + 8s + e.
    v8 qf[KS];
    {
      const int hl = lrow - ltok * p.G;
      const half_t* src = p.q + (int64_t)(u.q0 + ltok) * p.q_st +
                          (int64_t)(u.kvh * p.G + hl) * p.q_sh + g * HALF;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint4_t v = {0, 0, 0, 0};
        if (lrow < rows) v = ld16(src + 8 * k);
        if (p.neg_q) v ^= uint4_t{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
        qf[k] = E::as8(v);
      }
    }
    float16_t oacc[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) oacc[n][i] = 0.f;
    float m_run = kCkFloor, l_part = 0.f, x_part = 0.f;  // x: the sum of the unrounded P

    float16_t sA, sB;
    uint32_t pA[8], pB[8];
    v8 vf[2][NT];
    // P.V(-1) of step 0 multiplies zeros by zeros.
#pragma unroll
    for (int i = 0; i < 8; ++i) pB[i] = 0u;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n) vf[h][n] = E::as8(uint4_t{0, 0, 0, 0});

    // Fragments from LDS offset `at` of a step's rows.
    auto load_kf = [&](int at, v8 (&kf)[KS]) {
#pragma unroll
      for (int k = 0; k < KS; ++k)
        kf[k] = E::as8(*reinterpret_cast<const uint4_t*>(lds + at + koff[k]));
    };
    auto load_vf = [&](int at) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint2 lo = ds_read_tr16(lds + at + voff[n] + h * 16 * ROWB);
          const uint2 hi = ds_read_tr16(lds + at + voffh[n] + h * 16 * ROWB);
          vf[h][n] = E::as8(uint4_t{lo.x, lo.y, hi.x, hi.y});
        }
    };
    auto qk_mfma = [&](const v8 (&kf)[KS], float16_t& dst) {
#pragma unroll
      for (int i = 0; i < 16; ++i) dst[i] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) dst = E::mfma(kf[k], qf[k], dst);
    };
    auto pv_mfma = [&](const uint32_t (&pk)[8]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const v8 bop = E::as8(uint4_t{pk[4 * h], pk[4 * h + 1], pk[4 * h + 2], pk[4 * h + 3]});
#pragma unroll
        for (int n = 0; n < NT; ++n) oacc[n] = E::mfma(vf[h][n], bop, oacc[n]);
      }
    };
    auto softmax = [&](const float16_t& ss, uint32_t (&pk)[8], float& l_step, float& x_step) {
      float ls = 0.f, xs = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float p0 = fast_exp2(__builtin_fmaf(ss[i], c, -m_run));
        const float p1 = fast_exp2(__builtin_fmaf(ss[i + 1], c, -m_run));
        pk[i >> 1] = E::pack2(p0, p1);
        if constexpr (LSE) xs += p0 + p1;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ls = E::dot2(pk[i], E::kOnes, ls);
      l_step = ls;
      x_step = xs;
    };
    // Masks step t: keys past a row, and keys (bit of `valid`) of pages outside the pool.
    auto mask_step = [&](int kh0, uint32_t valid, float16_t& ss) {
      if (kh0 + 31 > lim_min || valid != 0xffffffffu) {  // wave-uniform
        mask_scores(ss, valid, lim - kh0, g);
      }
    };
    auto row_max = [&](const float16_t& sv) {
      float mx = sv[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = __builtin_elementwise_maximum(mx, sv[i]);
      float ma, mb;
      swap32(mx, ma, mb);
      return __builtin_elementwise_maximum(ma, mb) * c;
    };
    // One step, as in prefill_kernel: with no dependence between them, P.V of the
    // previous step, S of the next (K at LDS offset knext) and the softmax of this one (V at
    // vcur).
    auto step = [&](int kh0, uint32_t valid, int knext, int vcur, float16_t& scur,
                    float16_t& snext, const uint32_t (&pprev)[8], uint32_t (&pcur)[8]) {
      mask_step(kh0, valid, scur);
      v8 kf[KS];
      load_kf(knext, kf);
      pv_mfma(pprev);
      qk_mfma(kf, snext);
      load_vf(vcur);
      float l_step, x_step;
      softmax(scur, pcur, l_step, x_step);
#pragma unroll
      for (int i = 0; i < ck_mix_mfma(D); ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, ck_mix_valu(D), 0);
      }
      if (__any(!(l_step <= kCkStepLimit))) {  // rare
        const float mx = row_max(scur);
        const bool raise = mx > m_run + kCkSlack;
        const float alpha = raise ? fast_exp2(m_run - mx) : 1.f;
        l_part *= alpha;
        x_part *= alpha;
        if (raise) {
          m_run = mx;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) oacc[n][i] *= alpha;
        }
        softmax(scur, pcur, l_step, x_step);
      }
      l_part += l_step;
      x_part += x_step;
    };

    // ---- the walk.  While tile j is computed, tile j + 1 is published, j + 2 is written and
    // j + 3 is on its way; the ids of the block after it too.
    Keys keys;                 // of the last block placed
    uint64_t ok0, ok1, ok2;    // readable keys of the block of the next body and those after it
    load_ids(0);
    __syncthreads();  // the last unit's LDS reads are done
    {
      uint4_t ka[PER_T], va[PER_T], kb[PER_T], vb[PER_T];
      keys = place(0);
      load_ids(1);
      ok0 = keys.ok;
      load_tile(keys, 0, ka, va);
      if constexpr (kBN == 32) {
        load_tile(keys, 32, kb, vb);
        keys = place(1);
        ok1 = keys.ok;
        ok2 = 0;
        load_ids(2);
        if (n_tiles > 2) load_tile(keys, 0, kst, vst);
        store_tile(0, 0, ka, va);
        store_tile(1, BUFB, kb, vb);
      } else {
        keys = place(1);
        ok1 = keys.ok;
        load_ids(2);
        if (n_tiles > 1) load_tile(keys, 0, kb, vb);
        keys = place(2);
        ok2 = keys.ok;
        load_ids(3);
        if (n_tiles > 2) load_tile(keys, 0, kst, vst);
        store_tile(0, 0, ka, va);
        if (n_tiles > 1) store_tile(1, BUFB, kb, vb);
      }
    }
    __syncthreads();
    {
      v8 kf[KS];
      load_kf(0, kf);
      qk_mfma(kf, sA);
    }
    mask_step(k0, (uint32_t)ok0, sA);
    {
      const float mx = row_max(sA);
      m_run = mx < kCkFloor ? kCkFloor : mx;  // a NaN stays
    }
#pragma clang loop unroll(disable)
    for (int m = 0; m < nb; ++m) {  // keys 64 m .. 64 m + 63 of the part
      const uint64_t ok = ok0;
      ok0 = ok1;
      if constexpr (kBN == 32) {
        const int b0 = 2 * (m & 1) * BUFB, b1 = b0 + BUFB, b2 = 2 * BUFB - b0;
        __syncthreads();
        if (m + 1 < nb) {
          store_tile(2 * m + 2, b2, kst, vst);
          load_tile(keys, 32, kst, vst);
        }
        if (m + 2 < nb) {
          keys = place(m + 2);
          ok1 = keys.ok;
          load_ids(m + 3);
        }
        if (active) step(k0 + 64 * m, (uint32_t)ok, b1, b0, sA, sB, pB, pA);
        __syncthreads();
        if (m + 1 < nb) store_tile(2 * m + 3, b2 + BUFB, kst, vst);
        if (m + 2 < nb) load_tile(keys, 0, kst, vst);
        if (active) step(k0 + 64 * m + 32, (uint32_t)(ok >> 32), b2, b1, sB, sA, pA, pB);
      } else {
        const int b0 = (m & 3) * BUFB, b1 = ((m + 1) & 3) * BUFB, b2 = ((m + 2) & 3) * BUFB;
        constexpr int kHalf = 32 * ROWB;
        ok1 = ok2;
        __syncthreads();
        if (m + 2 < nb) store_tile(m + 2, b2, kst, vst);
        if (m + 3 < nb) {
          keys = place(m + 3);
          ok2 = keys.ok;
          load_tile(keys, 0, kst, vst);
          load_ids(m + 4);
        }
        if (active) {
          step(k0 + 64 * m, (uint32_t)ok, b0 + kHalf, b0, sA, sB, pB, pA);
          step(k0 + 64 * m + 32, (uint32_t)(ok >> 32), b1, b0 + kHalf, sB, sA, pA, pB);
        }
      }
    }
    if (active) pv_mfma(pB);  // P.V of the last step

    // ---- end of the part: partial or output, each wave for its own rows.
    if (lane == 0) sm_bad[wave] = bad;
    __syncthreads();  // every tile read is done
    if (!active) return;
    int any_bad = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) any_bad |= sm_bad[w];
    if (uniform(any_bad))  // from the first tile that store_tile took the values out of
      add_not_finite<D, BF16, SHARED>(p, u, k0 + max(u.first + 1 - k0, 0) / kBN * kBN, k1, g, lim, oacc);
    float l_row = xor32_sum(l_part);
    float x_row = LSE ? xor32_sum(x_part) : 0.f;
    if constexpr (SHARED) {
      if (lrow >= rows) return;
      const int64_t at = (int64_t)(u.q0 + ltok) * p.Hq + u.kvh * p.G + (lrow - ltok * p.G);
      const StateRow to = state_row<D>(p, u, at, whole, k0 == 0, wg, Ustart, Lw, kCkBlock,
                                       true, 32 * WAVES, lrow);
      if (g == 0) *to.ml = float4_t{m_run, l_row, x_row, to.tag};
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          st16(to.o + 32 * n + 8 * k + 4 * g,
               as_uint4f(float4_t{oacc[n][4 * k], oacc[n][4 * k + 1], oacc[n][4 * k + 2],
                                  oacc[n][4 * k + 3]}));
      return;
    }
    if (!whole) {
      constexpr int64_t kWaveB = chunk_wave_bytes(D), kSlotB = WAVES * kWaveB;
      const int kb_last = (u.kend - 1) / kCkBlock * kCkBlock;
      const int wf = div_range(Ustart + kCkBlock - 1, Lw);
      const int wl = div_range(Ustart + kb_last + kCkBlock - 1, Lw);
      auto slot_of = [&](int w) -> char* {
        return p.partials + p.many_partial + (2 * (int64_t)w + (w == wf ? 1 : 0)) * kSlotB +
               wave * kWaveB;
      };
      char* mine = slot_of(wg);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          st16_device(mine, (uint32_t)(((4 * n + k) * 64 + lane) * 16),
                      as_uint4f(float4_t{oacc[n][4 * k], oacc[n][4 * k + 1], oacc[n][4 * k + 2],
                                         oacc[n][4 * k + 3]}));
      if (g == 0)
        st16_device(mine, (uint32_t)(NT * 4096 + l32 * 16),
                    as_uint4f(float4_t{m_run, l_row, x_row, 0.f}));
      // The stores (device scope) are complete before the count.
      __builtin_amdgcn_s_waitcnt(0);
      int prev = 0;
      if (lane == 0) prev = atomicAdd(&p.arrive[p.many_counter + WAVES * wf + wave], 1);
      if (uniform(prev) != wl - wf) return;
      if (lane == 0) atomicExch(&p.arrive[p.many_counter + WAVES * wf + wave], 0);
      constexpr int UB = D == 64 ? 4 : 2;  // partials in flight
      m_run = AKT_C_NEG_INF;
      l_row = x_row = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[n][i] = 0.f;
#pragma clang loop unroll(disable)
      for (int w = wf; w <= wl; w += UB) {
        float4_t ml[UB], ov[UB][4 * NT];
#pragma unroll
        for (int k = 0; k < UB; ++k) {
          const char* src = slot_of(min(w + k, wl));
          ml[k] = as_float4u(ld16_device(src, (uint32_t)(NT * 4096 + l32 * 16)));
#pragma unroll
          for (int i = 0; i < 4 * NT; ++i)
            ov[k][i] = as_float4u(ld16_device(src, (uint32_t)((i * 64 + lane) * 16)));
        }
#pragma unroll
        for (int k = 0; k < UB; ++k) {
          if (w + k > wl) break;
          const float f = merge_in(ml[k], m_run, l_row, x_row, [&](float sc) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 16; ++i) oacc[n][i] *= sc;
          });
#pragma unroll
          for (int i = 0; i < 4 * NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) oacc[i / 4][4 * (i % 4) + j] += f * ov[k][i][j];
        }
      }
    }
    // Output rows through LDS, so that every lane stores 16 contiguous bytes.
    const float inv = l_row == 0.f ? 0.f : __builtin_amdgcn_rcpf(l_row);
    if (LSE && g == 0 && lrow < rows)
      p.lse[(int64_t)(u.q0 + ltok) * p.Hq + u.kvh * p.G + (lrow - ltok * p.G)] =
          l_row == 0.f ? AKT_C_NEG_INF : (m_run + __log2f(x_row)) * kLn2;
    char* ost = lds + wave * (32 * ROWB);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float16_t& a = oacc[n];
        const uint2 hv = {E::pack2(a[4 * k] * inv, a[4 * k + 1] * inv),
                          E::pack2(a[4 * k + 2] * inv, a[4 * k + 3] * inv)};
        const int chunk = (4 * n + k) ^ eswz(l32);
        *reinterpret_cast<uint2*>(ost + l32 * ROWB + chunk * 16 + 8 * g) = hv;
      }
#pragma unroll 2
    for (int idx = lane; idx < 32 * CPR; idx += 64) {
      const int lr = idx / CPR, cc = idx % CPR;
      const uint4_t v = *reinterpret_cast<const uint4_t*>(ost + lr * ROWB + ((cc ^ eswz(lr)) * 16));
      const int row = 32 * wave + lr;
      const int tok = (int)((uint32_t)row * p.g_magic >> 16);
      if (row < rows)
        st16(p.o + ((int64_t)(u.q0 + tok) * p.Hq + u.kvh * p.G + (row - tok * p.G)) * D + 8 * cc,
             v);
    }
  };

  // ---- the keys [k0, k1) of a unit of up to 32 RG rows: few rows, so the keys are what is
  // shared out.  Wave w has rows 32 (w % RG) .. and takes the 32-key steps w / RG, + KG, ...
  // of the part, each on its own: K goes from global memory straight into the fragments'
  // registers, V through the wave's own LDS for the transposing reads, both loaded again as
  // soon as the step has used them, with no barrier before the waves' results are merged.
  auto serve_split = [&](const Unit<SHARED>& u, int k0, int k1, int64_t Ustart, auto rg_c) {
    // The lane number is opaque here, so that what is derived from it lives no longer than
    // this part (held across the units' loop it would not fit the registers).
    int lane = tid0 & 63;
    asm volatile("" : "+v"(lane));
    const int l32 = lane & 31, g = lane >> 5;
    // V^T through the transposing read: see prefill_kernel.
    const int s16 = lane & 15;
    const int vrow = 4 * g + (s16 >> 2);
    const int vcl = 2 * ((lane >> 4) & 1) + ((s16 & 3) >> 1);
    int voff[NT], voffh[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      voff[n] = vrow * ROWB + (((4 * n + vcl) ^ tswz<D>(vrow)) * 16) + (s16 & 1) * 8;
      voffh[n] =
          (vrow + 8) * ROWB + (((4 * n + vcl) ^ tswz<D>(vrow + 8)) * 16) + (s16 & 1) * 8;
    }
    constexpr int RG = decltype(rg_c)::value, KG = TW / RG;
    constexpr int OB = 32 * D * 4;   // bytes of a wave's O
    constexpr int NQ = 4 * NT / KG;  // 4-element pieces of O that a wave merges
    static_assert(WAVES * OB <= kCkNBuf * BUFB, "the waves' O fit the tile buffers");
    static_assert(NQ % 2 == 0, "whole 16-byte chunks");
    const int rg = twave % RG, kg = twave / RG;
    const int rows = u.ntok * p.G;
    const bool active = 32 * rg < rows;
    const int n_steps = active ? (k1 - k0 + 31) / 32 : 0;
    const half_t* const Kh = p.pool + u.kvh * p.sh;
    const int row = 32 * rg + l32;
    const int tok = (int)((uint32_t)row * p.g_magic >> 16);
    const int lim = is_causal(p, u) ? u.first + min(tok, u.ntok - 1) : u.len - 1;
    const int lim_min =
        is_causal(p, u) ? u.first + min((int)((uint32_t)(32 * rg) * p.g_magic >> 16), u.ntok - 1)
                 : u.len - 1;
    char* const vst = lds + wave * OB;

    // Lane (l32, g) loads chunks 2 k + g of the K and V rows of key l32 of a step.  Ids are loaded
    // a step before the rows.
    int id_next = 0, slot_next = 0;
    auto load_ids = [&](int t) {
      const int key = min(k0 + 32 * t + l32, u.kend - 1);
      const int lp = page_of(p, key);
      slot_next = key - lp * p.page_size;
      id_next = page_ids(p, u)[u.ip0 + lp];
    };
    uint32_t valid = 0, valid_next = 0;  // keys that can be read: in the pool, before the unit's end
    const half_t* src = p.q;
    // The place of a step's row.  A key that cannot be read takes a row of q (any readable row
    // does: its score is masked, its V zeroed).
    auto place = [&](int t) {
      const bool ok =
          k0 + 32 * t + l32 < u.kend && (uint32_t)id_next < (uint32_t)p.num_pool_pages;
      valid_next = (uint32_t)__ballot(ok);
      src = (ok ? Kh + id_next * p.sp + (int64_t)slot_next * p.ss : p.q) + 8 * g;
    };
    uint4_t kf[KS], vr[KS];
    auto load_k = [&]() {
#pragma unroll
      for (int k = 0; k < KS; ++k) kf[k] = ld16(src + 16 * k);
    };
    auto load_v = [&]() {
      if (valid_next == 0xffffffffu) {
#pragma unroll
        for (int k = 0; k < KS; ++k) vr[k] = ld16(src + p.skv + 16 * k);
      } else {
        const bool ok = (valid_next >> l32) & 1;
#pragma unroll
        for (int k = 0; k < KS; ++k) vr[k] = ok ? ld16(src + p.skv + 16 * k) : uint4_t{0, 0, 0, 0};
      }
    };

    v8 qf[KS];
    {
      const half_t* src = p.q + (int64_t)(u.q0 + tok) * p.q_st +
                          (int64_t)(u.kvh * p.G + row - tok * p.G) * p.q_sh + 8 * g;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint4_t v = {0, 0, 0, 0};
        if (row < rows) v = ld16(src + 16 * k);
        if (p.neg_q) v ^= uint4_t{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
        qf[k] = E::as8(v);
      }
    }
    float16_t oacc[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) oacc[n][i] = 0.f;
    float m_run = kCkFloor, l_part = 0.f, x_part = 0.f;
    auto frag = [&](int h, int n) -> v8 {  // V^T of the staged rows
      const uint2 lo = ds_read_tr16(vst + voff[n] + h * 16 * ROWB);
      const uint2 hi = ds_read_tr16(vst + voffh[n] + h * 16 * ROWB);
      return E::as8(uint4_t{lo.x, lo.y, hi.x, hi.y});
    };

    team_sync();  // the last unit's LDS reads are done
    bool bad = false;
    if (kg < n_steps) {
      load_ids(kg);
      place(kg);
      load_k();
      load_v();
      load_ids(kg + KG);
    }
#pragma clang loop unroll(disable)
    for (int t = kg; t < n_steps; t += KG) {
      const int kh0 = k0 + 32 * t;
      const bool more = t + KG < n_steps;
      valid = valid_next;
      float16_t sv;
#pragma unroll
      for (int i = 0; i < 16; ++i) sv[i] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) sv = E::mfma(E::as8(kf[k]), qf[k], sv);
      if (more) {
        place(t + KG);
        load_k();
      }
      if (is_causal(p, u) && kh0 + 31 > u.first)  // keys that not every row sees
        bad |= zero_not_finite<BF16>(vr);
#pragma unroll
      for (int k = 0; k < KS; ++k)
        *reinterpret_cast<uint4_t*>(vst + l32 * ROWB + (((2 * k + g) ^ tswz<D>(l32)) * 16)) = vr[k];
      if (more) {
        load_v();
        load_ids(t + 2 * KG);
      }
      if (kh0 + 31 > lim_min || valid != 0xffffffffu) {  // wave-uniform
        mask_scores(sv, valid, lim - kh0, g);
      }
      float mx = sv[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = __builtin_elementwise_maximum(mx, sv[i]);
      float ma, mb;
      swap32(mx, ma, mb);
      const float m_new =
          __builtin_elementwise_maximum(m_run, __builtin_elementwise_maximum(ma, mb) * c);
      if (__any(!(m_new <= m_run + kCkSlack))) {
        // The slack leaves P below 2^kCkSlack.  The first keys' rise from the floor scales zeros.
        const float alpha = fast_exp2(m_run - m_new);
        l_part *= alpha;
        x_part *= alpha;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) oacc[n][i] *= alpha;
        m_run = m_new;
      }
      uint32_t pk[8];
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float p0 = fast_exp2(__builtin_fmaf(sv[i], c, -m_run));
        const float p1 = fast_exp2(__builtin_fmaf(sv[i + 1], c, -m_run));
        pk[i >> 1] = E::pack2(p0, p1);
        if constexpr (LSE) x_part += p0 + p1;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) l_part = E::dot2(pk[i], E::kOnes, l_part);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const v8 bop = E::as8(uint4_t{pk[4 * h], pk[4 * h + 1], pk[4 * h + 2], pk[4 * h + 3]});
#pragma unroll
        for (int n = 0; n < NT; ++n) oacc[n] = E::mfma(frag(h, n), bop, oacc[n]);
      }
    }
    if (bad)
      for (int t = kg; t < n_steps; t += KG)
        if (k0 + 32 * t + 31 > u.first)  // a step that the values were taken out of
          add_not_finite<D, BF16, SHARED>(p, u, k0 + 32 * t, min(k0 + 32 * t + 32, u.kend), g, lim, oacc);

    // ---- merge of the KG waves that share rows: piece 4 n + k of O (dims 32 n + 8 k + 4 g ..
    // + 3 of row l32) of every lane lies at [wave][piece][lane]; the wave with key group kg
    // then sums pieces NQ kg .. of all.
    float l_row = xor32_sum(l_part);
    float x_row = LSE ? xor32_sum(x_part) : 0.f;
    if (g == 0) sm_ml[wave][l32] = float4_t{m_run, l_row, x_row, 0.f};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *reinterpret_cast<uint4_t*>(vst + ((4 * n + k) * 64 + lane) * 16) =
            as_uint4f(float4_t{oacc[n][4 * k], oacc[n][4 * k + 1], oacc[n][4 * k + 2],
                               oacc[n][4 * k + 3]});
    team_sync();
    if (!active) return;
    float4_t acc[NQ];
    {
      float f[KG];
      m_run = AKT_C_NEG_INF;
#pragma unroll
      for (int w = 0; w < KG; ++w)
        m_run = __builtin_elementwise_maximum(m_run, sm_ml[team * TW + w * RG + rg][l32][0]);
      l_row = x_row = 0.f;
#pragma unroll
      for (int w = 0; w < KG; ++w) {
        const float4_t ml = sm_ml[team * TW + w * RG + rg][l32];
        f[w] = fast_exp2(ml[0] - m_run);
        l_row += f[w] * ml[1];
        x_row += f[w] * ml[2];
      }
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        acc[i] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < KG; ++w)
          acc[i] += f[w] * as_float4u(*reinterpret_cast<const uint4_t*>(
                               lds + (team * TW + w * RG + rg) * OB + ((NQ * kg + i) * 64 + lane) * 16));
      }
    }
    if (!(k0 == 0 && k1 == u.kend)) {
      // Partial: this wave's pieces and the row's (m, l); the last of the unit's workgroups
      // merges them, wave by wave.
      constexpr int64_t kWaveB = chunk_split_wave_bytes(D), kSlotB = TW * kWaveB;
      constexpr uint32_t kMl = (uint32_t)kWaveB - 512;  // the rows' (m, l)
      const int kb_last = (u.kend - 1) / kCkBlock * kCkBlock;
      const int wf = div_range(Ustart + kCkBlock - 1, Lw);
      const int wl = div_range(Ustart + kb_last + kCkBlock - 1, Lw);
      auto slot_of = [&](int w) -> char* {
        return p.partials + (2 * (int64_t)w + (w == wf ? 1 : 0)) * kSlotB + twave * kWaveB;
      };
      char* mine = slot_of(wg);
      if (row < rows) {
#pragma unroll
        for (int i = 0; i < NQ; ++i)
          st16_device(mine, (uint32_t)((i * 64 + lane) * 16), as_uint4f(acc[i]));
        if (g == 0)
          st16_device(mine, kMl + l32 * 16,
                      as_uint4f(float4_t{m_run, l_row, x_row, 0.f}));
      }
      __builtin_amdgcn_s_waitcnt(0);
      int prev = 0;
      if (lane == 0) prev = atomicAdd(&p.arrive[TW * wf + twave], 1);
      if (uniform(prev) != wl - wf) return;
      if (lane == 0) atomicExch(&p.arrive[TW * wf + twave], 0);
      if (row < rows) {
        constexpr int UB = 32 / NQ < 8 ? 32 / NQ : 8;  // partials in flight
        m_run = AKT_C_NEG_INF;
        l_row = x_row = 0.f;
#pragma unroll
        for (int i = 0; i < NQ; ++i) acc[i] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma clang loop unroll(disable)
        for (int w = wf; w <= wl; w += UB) {
          float4_t ml[UB], ov[UB][NQ];
#pragma unroll
          for (int k = 0; k < UB; ++k) {
            const char* src = slot_of(min(w + k, wl));
            ml[k] = as_float4u(ld16_device(src, kMl + l32 * 16));
#pragma unroll
            for (int i = 0; i < NQ; ++i)
              ov[k][i] = as_float4u(ld16_device(src, (uint32_t)((i * 64 + lane) * 16)));
          }
#pragma unroll
          for (int k = 0; k < UB; ++k) {
            if (w + k > wl) break;
            const float f = merge_in(ml[k], m_run, l_row, x_row, [&](float sc) {
#pragma unroll
              for (int i = 0; i < NQ; ++i) acc[i] *= sc;
            });
#pragma unroll
            for (int i = 0; i < NQ; ++i) acc[i] += f * ov[k][i];
          }
        }
      }
    }
    const float inv = l_row == 0.f ? 0.f : __builtin_amdgcn_rcpf(l_row);
    const int64_t at = (int64_t)(u.q0 + tok) * p.Hq + u.kvh * p.G + (row - tok * p.G);
    if (LSE && kg == 0 && g == 0 && row < rows)
      p.lse[at] = l_row == 0.f ? AKT_C_NEG_INF : (m_run + __log2f(x_row)) * kLn2;
    // The lane halves hold 8-byte halves of a row's 16-byte chunks: half 0 takes chunk i
    // whole, half 1 chunk i + 1.
#pragma unroll
    for (int i = 0; i < NQ; i += 2) {
      uint2 hv[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        hv[k] = uint2{E::pack2(acc[i + k][0] * inv, acc[i + k][1] * inv),
                      E::pack2(acc[i + k][2] * inv, acc[i + k][3] * inv)};
      const uint2 send = g == 0 ? hv[1] : hv[0];
      const uint2 recv = {(uint32_t)__shfl_xor((int)send.x, 32, 64),
                          (uint32_t)__shfl_xor((int)send.y, 32, 64)};
      const uint4_t v = g == 0 ? uint4_t{hv[0].x, hv[0].y, recv.x, recv.y}
                               : uint4_t{recv.x, recv.y, hv[1].x, hv[1].y};
      if (row < rows) st16(p.o + at * D + 8 * (NQ * kg + i + g), v);
    }
  };

  // ---- the units of the range: first the one that reaches out of its end, then the others
  // from its start on.  A range that is about as long as a unit then goes through a unit's
  // head and the tail of the unit before it in the order of their keys, so the
  // workgroups of one kv head, which share an L2, read the same keys at the same time.
  int last_b = -1, last_kvh = 0, last_r = 0;
#pragma clang loop unroll(disable)
  for (int pass = 0; pass < 2; ++pass) {
    int64_t len = 0, inc = 0;
    if constexpr (!SHARED) {
      len = seq_length(lane0);
      inc = scan64(len);
    }
    if (pass == 0) {
      int seqs = 0;
      if constexpr (!SHARED) {
        total = uniform64(shfl64(inc, 63));
        seqs = __builtin_popcountll(__ballot(len > 0));
        for (int jb = 64; jb < p.B; jb += 64) {
          const int64_t more = seq_length(jb + lane0);
          total += uniform64(shfl64(scan64(more), 63));
          seqs += __builtin_popcountll(__ballot(more > 0));
        }
      }
      // Where few units share the axis, one range to a workgroup, not one to a team: half the
      // partials to a unit (us, D = 128 over 8 kv heads, a team / a workgroup: one token after
      // 30000 54.5 / 42.8, two of those 71.5 / 62.0, four after 10000 49.8 / 45.9; eight after
      // 10000, past the limit, 76 either way).
      const int used = SPLIT && seqs * p.Hkv <= W / 8 ? W : ranges;
      Lw = SHARED ? div_range64(total + used - 1, used) : (total + used - 1) / used;
      if (Lw < p.min_keys) Lw = p.min_keys;
      Lw = uniform64(Lw);
      x0 = wg * Lw;
      if (x0 >= total) return;
      x1 = x0 + Lw < total ? x0 + Lw : total;
    }
    // The unit that holds x: sequence, kv head, row block.
    const int64_t x = pass == 0 ? x1 - 1 : x0;
    int b = 0;
    int64_t U = 0;  // the sequence's start
    for (int jb = 0;;) {
      if constexpr (SHARED) {  // (here and nowhere else: every copy is fetched cold)
        len = seq_length(jb + lane0);
        inc = scan64(len);
      }
      const uint64_t m = __ballot(U + inc > x);
      if (m) {
        const int l = __builtin_ctzll(m);
        b = uniform(jb + l);
        U += SHARED ? read_lane64(inc - len, l) : uniform64(shfl64(inc - len, l));
        break;
      }
      U += SHARED ? read_lane64(inc, 63) : uniform64(shfl64(inc, 63));
      jb += 64;
      if constexpr (!SHARED) {
        len = seq_length(jb + lane0);
        inc = scan64(len);
      }
    }
    Seq<SHARED> s = load_seq_uniform<SHARED>(p, b, table);
    int64_t hlen = uniform64(head_length(p, s));
    int kvh = div_range(x - U, hlen);
    int64_t hs = uniform64(U + kvh * hlen);  // the head's start
    int R = uniform(row_blocks(p, s.n)), r = 0;
    for (int lo = 1, hi = R; lo < hi;) {  // last r with unit_start(r) <= x - hs
      const int mid = (lo + hi) / 2;
      if (unit_start(p, s, mid) <= x - hs) {
        r = mid;
        lo = mid + 1;
      } else {
        hi = mid;
      }
    }
    for (;;) {
      if (b == last_b && kvh == last_kvh && r == last_r) return;
      Unit<SHARED> u;
      const int t0 = r * p.TR;
      u.q0 = uniform(s.q0 + t0);
      u.ntok = uniform(min(p.TR, s.n - t0));
      u.kvh = kvh;
      u.first = uniform(s.len - s.n + t0);
      u.len = uniform(s.len);
      u.kend = uniform(is_causal(p, s) ? max(u.first + u.ntok, 0) : s.len);
      u.ip0 = uniform(s.ip0);
      if constexpr (SHARED) {
        u.prefix = uniform(s.prefix);
        u.more = uniform(s.more);
      }
      const int64_t us = uniform64(hs + unit_start(p, s, r));
      // Blocks from the first at or past x - us - (kCkBlock - 1) on are those of the ranges
      // from x on.
      auto cut = [&](int64_t x) -> int {
        const int64_t d = x - us;
        return uniform(d >= u.kend + kCkBlock ? u.kend
                       : d < kCkBlock         ? 0
                                              : min((int)d / kCkBlock * kCkBlock, u.kend));
      };
      const int k0 = cut(x0), k1 = cut(x1);
      if (u.kend == 0) {
        // Nothing to see: zeros, by the workgroup of what would be the first block.
        const int rows = u.ntok * p.G;
        if (x0 - us < kCkBlock && x1 - us >= kCkBlock)
          for (int idx = 64 * twave + lane0; idx < rows * CPR; idx += 64 * TW) {
            const int row = idx / CPR;
            const int tok = (int)((uint32_t)row * p.g_magic >> 16);
            const int64_t at = (int64_t)(u.q0 + tok) * p.Hq + u.kvh * p.G + (row - tok * p.G);
            if constexpr (SHARED) {
              if (idx % CPR == 0)
                state_ml(p, u)[at] = float4_t{AKT_C_NEG_INF, 0.f, 0.f,
                                              __int_as_float(u.more ? kStateMore : 0)};
              continue;
            }
            st16(p.o + at * D + idx % CPR * 8, uint4_t{0, 0, 0, 0});
            if (LSE && idx % CPR == 0) p.lse[at] = AKT_C_NEG_INF;
          }
      } else if (k0 < k1) {
        if constexpr (!SPLIT) serve(u, k0, k1, us);
        else if (chunk_split_rows(D) <= 32 || u.ntok * p.G <= 32)
          serve_split(u, k0, k1, us, std::integral_constant<int, 1>{});
        else if constexpr (chunk_split_rows(D) > 32)
          serve_split(u, k0, k1, us, std::integral_constant<int, 2>{});
      }
      if (pass == 0) {
        if (us <= x0) return;  // the range lies in this unit
        last_b = b;
        last_kvh = kvh;
        last_r = r;
        break;
      }
      if (++r < R) continue;
      r = 0;
      hs += hlen;
      if (++kvh < p.Hkv) continue;
      kvh = 0;
      do {
        if (++b == num_seqs<SHARED>(p)) return;
        s = load_seq_uniform<SHARED>(p, b, table);
      } while (!mine(s));
      R = uniform(row_blocks(p, s.n));
      hlen = uniform64(head_length(p, s));
    }
  }
}

#ifdef AKT_CHUNK_SHARED
#include "paged_shared_few.hpp"
#else
template <int D, bool BF16, bool LSE>
__device__ __forceinline__ void shared_few(const ChunkParams&, char*, const int4*, int, int, int64_t) {}
#endif

// Workgroups (of all W, a multiple of 8) for the sequences of few tokens, where a launch may hold
// both kinds: in proportion to the lengths of the two axes, a key of the other weighing 1 for a
// unit of hardly any rows up to chunk_tile_cost for one of all rows.
template <int D>
__device__ __forceinline__ int split_share(const ChunkParams& p, int W) {
  constexpr int kRows = 32 * chunk_waves(D);
  const int lane = threadIdx.x & 63;
  double few = 0, many = 0;
  for (int b = lane; b < p.B; b += 64) {
    const Seq<false> s = load_seq<false>(p, b);
    const double len = (double)head_length(p, s);
    if (s.n <= p.split_tokens) few += len;
    else
      many += len * (1 + (chunk_tile_cost(D) - 1) / kRows * min((double)s.n * p.G, (double)kRows));
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    few += __shfl_xor(few, d, 64);
    many += __shfl_xor(many, d, 64);
  }
  if (many == 0) return W;
  if (few == 0) return 0;
  const int s = 8 * (int)(W / 8 * (few / (few + many)) + 0.5);
  return uniform(min(max(s, 8), W - 8));
}
// The same where prefixes are shared (a key weighs kSharedTileCostLow to kSharedTileCost), and the
// lengths of the two axes.
struct Shares {
  int64_t few, many;
  int wgs;
};
template <int D>
__device__ __forceinline__ Shares shared_shares(const ChunkParams& p, const int4* table, int W) {
  constexpr float kRows = 32 * chunk_waves(D);
  constexpr float kLow = kSharedTileCostLow, kSlope = (kSharedTileCost - kSharedTileCostLow) / kRows;
  const int lane = threadIdx.x & 63;
  int64_t few = 0, many = 0;
  float cost = 0;
  for (int b = lane; b < num_seqs<true>(p); b += 64) {
    const Seq<true> s = load_seq<true>(p, b, table);
    if (s.n <= p.split_tokens) {
      if (s.n > 0) few += s.len + kWaveUnitCost;
    } else {
      const int64_t len = head_length(p, s);
      many += len;
      cost += (float)len * (kLow + kSlope * min((float)s.n * p.G, kRows));
    }
  }
  few = read_lane64(wave_inclusive_scan64(few), 63);
  many = read_lane64(wave_inclusive_scan64(many), 63);
  cost = wave_sum(cost);
  const int s = 8 * (int)((float)(W / 8) * ((float)few / ((float)few + cost)) + 0.5f);
  const int wgs = many == 0 ? W : few == 0 ? 0 : min(max(s, 8), W - 8);
  return Shares{few * p.Hkv, many * p.Hkv, wgs};
}

template <int D, bool BF16, bool GRP, bool LSE, bool SHARED>
__global__ __launch_bounds__(64 * chunk_waves(D))
__attribute__((amdgpu_waves_per_eu(chunk_waves_per_simd(D), chunk_waves_per_simd(D))))
void paged_chunk_kernel(ChunkParams p) {
  __shared__ __attribute__((aligned(16)))
  char lds[kCkNBuf * 2 * ck_tile_keys(D) * D * 2];
  const int block = blockIdx.x, W = gridDim.x;
  const int4* table = nullptr;
  if constexpr (SHARED) {
    __shared__ int4 sm_table[kCkTable];
    __shared__ int sm_end;  // end of the last sequence's tokens
    if (in_table(p)) {
      for (int b = threadIdx.x; b < num_seqs<true>(p); b += 64 * chunk_waves(D)) {
        if (b < p.B) {
          const Seq<true> s = load_seq<true>(p, b);
          sm_table[b] = int4{s.q0, s.n | s.more << 30, s.ip0, s.len};  // (n < 2^30)
          if (b == p.B - 1) sm_end = min(max(p.q_indptr[p.B], 0), p.total_q);
        } else {  // its tokens from the sequences' places, below
          const Prefix x = load_prefix(p, b - p.B);
          sm_table[b] = int4{x.b0, x.b1, x.ip0, x.len};
        }
      }
      __syncthreads();
      table = sm_table;
      if (threadIdx.x < 64)
        for (int b = p.B + threadIdx.x; b < num_seqs<true>(p); b += 64) {
          const int4 t = sm_table[b];
          const int q0 = t.x < p.B ? sm_table[t.x].x : sm_end;
          const int q1 = t.y < p.B ? sm_table[t.y].x : sm_end;
          int n = t.y > t.x ? max(q1 - q0, 0) : 0;
          // A sequence of many rows alone behind a prefix without keys has none (us, 16 prompts of 300
          // tokens, all such: 119 with empty units, 92 so; of few rows 64 single tokens over 100 keys
          // 20.9 / 23.7, 32 over 500 23.5 / 26.0: there the empty units spread the keys over more waves).
          if (t.w == 0 && t.y == t.x + 1 && n > p.split_tokens) {
            sm_table[t.x].y &= 0x3fffffff;  // no state of a prefix to join
            n = 0;
          }
          sm_table[b] = int4{q0, n, t.z, t.w};
        }
      // Read by other lanes of the wave in shared_shares, by the other waves behind the barrier after it.
      wave_lds_sync();
    }
  }
  // The share goes through LDS: passed on in a register, it made the compiler spill 96 more
  // of them in what follows.
  __shared__ int sm_share;
  if constexpr (SHARED) {
    __shared__ int64_t sm_total[2];
    if (threadIdx.x < 64) {
      const Shares c = shared_shares<D>(p, table, W);
      if (threadIdx.x == 0) {
        sm_share = c.wgs;
        sm_total[0] = c.few;
        sm_total[1] = c.many;
      }
    }
    __syncthreads();
    const int S = uniform(sm_share);
    if (block < S) shared_few<D, BF16, LSE>(p, lds, table, block, S, uniform64(sm_total[0]));
    else
      chunk_range<D, BF16, GRP, LSE, true, false>(p, lds, table, block - S, W - S,
                                                  uniform64(sm_total[1]));
  } else {
    const int share = p.kinds == (kCkFew | kCkMany) ? split_share<D>(p, W) : p.kinds == kCkFew ? W : 0;
    if (threadIdx.x == 0) sm_share = share;
    __syncthreads();
    const int S = uniform(sm_share);
    if (block < S) chunk_range<D, BF16, GRP, LSE, false, true>(p, lds, table, block, S);
    else
      chunk_range<D, BF16, GRP, LSE, false, false>(p, lds, table, block - S, W - S);
  }
}

#ifdef AKT_CHUNK_SHARED
constexpr bool kShared = true;
#else
constexpr bool kShared = false;
#endif

template <int D, bool BF16, bool GRP>
int launch_lse(const ChunkParams& p, hipStream_t st) {
  KernelTimer timer;
  const dim3 grid(p.wgs), block(64 * chunk_waves(D));
  if (p.lse) timer.launch(paged_chunk_kernel<D, BF16, GRP, true, kShared>, grid, block, 0, st, p);
  else timer.launch(paged_chunk_kernel<D, BF16, GRP, false, kShared>, grid, block, 0, st, p);
  return check_launch("paged_chunk_kernel");
}

template <int D>
int launch_chunk(const ChunkParams& p, bool bf16, hipStream_t st) {
  if (p.page_size % 16 == 0)
    return bf16 ? launch_lse<D, true, true>(p, st) : launch_lse<D, false, true>(p, st);
  return bf16 ? launch_lse<D, true, false>(p, st) : launch_lse<D, false, false>(p, st);
}

}  // namespace

// Each head dim is instantiated in a translation unit of its own (they compile side by
// side), with shared prefixes and without: this one holds D = 128 and the entry points, the
// others include it.
#ifndef AKT_CHUNK_TU
#define AKT_CHUNK_TU 128
#endif
#define AKT_CAT_(a, b) a##b
#define AKT_CAT(a, b) AKT_CAT_(a, b)
#ifdef AKT_CHUNK_SHARED
int AKT_CAT(shared_launch_, AKT_CHUNK_TU)(const ChunkParams& p, bool bf16, hipStream_t st) {
  return launch_chunk<AKT_CHUNK_TU>(p, bf16, st);
}
#else
int AKT_CAT(chunk_launch_, AKT_CHUNK_TU)(const ChunkParams& p, bool bf16, hipStream_t st) {
  return launch_chunk<AKT_CHUNK_TU>(p, bf16, st);
}
#endif
#if AKT_CHUNK_TU == 128 && !defined(AKT_CHUNK_SHARED)

namespace {

constexpr int kCkMinKeys = 256;

// How a call is served.
struct ChunkPlan {
  int split_tokens, kinds;
  int64_t wgs, many_counter, many_partial;  // where the counters and partials of the second kind begin
  int64_t counters, partial_bytes;
};

// Workgroups of an axis: as many as are resident, fewer where it is too short for them (bounded
// from above by what the host knows: every sequence as long as all pages).
int64_t axis_wgs(double units, int64_t tokens, int64_t resident) {
  const double wgs = ceil(units * (double)(tokens + kCkUnitCost) / kCkMinKeys);
  return wgs < (double)resident ? round_up((int64_t)wgs, 8) : resident;
}

// groups < 0: no shared prefixes.
ChunkPlan chunk_plan(int64_t batch, int64_t total_q, int64_t Hkv, int64_t G, int64_t D,
                     int64_t page_size, int64_t total_pages, int64_t groups,
                     int64_t prefix_pages) {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
      cus <= 0 || cus > 1024)
    cus = 256;  // no device: what an MI355X has
  const bool shared = groups >= 0;
  const int64_t tokens = page_size * (total_pages + (shared ? prefix_pages : 0));
  // Sequences with new tokens, and their new tokens; a group's once more.
  int64_t seqs = batch < total_q ? batch : total_q, rows = total_q;
  if (shared) {
    seqs += groups < total_q ? groups : total_q;
    rows += total_q;
  }
  const int waves = chunk_waves((int)D);
  const int64_t resident = round_up((int64_t)cus * chunk_waves_per_simd((int)D) * 4 / waves, 8);
  ChunkPlan c = {};
  // Sequences of up to chunk_split_rows rows to a kv head share out their keys.  How many tokens a
  // sequence has is known on the device alone, unless there is one, or all are few.
  c.split_tokens = (int)((shared ? 32 : chunk_split_rows((int)D)) / G);
  const bool few = total_q <= c.split_tokens;
  if (!few && batch == 1) c.split_tokens = 0;
  if (c.split_tokens > 0) c.kinds |= kCkFew;
  if (!few) c.kinds |= kCkMany;
  double units = 0;
  if (c.kinds & kCkFew) units += (double)Hkv * seqs;
  if (c.kinds & kCkMany) units += (double)Hkv * (rows / (32 * waves / G) + seqs);
  c.wgs = axis_wgs(units, tokens, resident);
  if (c.kinds == (kCkFew | kCkMany) && c.wgs < 16) c.wgs = 16;  // eight of each kind
  // Two partial slots to a range, whichever kind a workgroup serves.
  if (c.kinds & kCkFew) {
    c.many_counter = c.wgs * waves;
    c.many_partial = 2 * c.wgs * waves *
                     (shared ? 32 * state_bytes((int)D) : chunk_split_wave_bytes((int)D));
  }
  c.counters = c.many_counter + (c.kinds & kCkMany ? c.wgs * waves : 0);
  c.partial_bytes =
      c.many_partial + (c.kinds & kCkMany ? 2 * c.wgs * waves * chunk_wave_bytes((int)D) : 0);
  return c;
}

bool sizes_served(int64_t Hq, int64_t Hkv, int64_t D) {
  return Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= kCkRows &&
         (D == 64 || D == 128 || D == 256);
}

size_t workspace_bytes_of(const ChunkPlan& c, int64_t states) {
  return (size_t)(round_up(AKT_WORKSPACE_ZERO_BYTES, 256) + round_up(c.partial_bytes, 256) + states);
}

// What a call with shared prefixes has besides.
struct SharedArgs {
  const int32_t *group_indptr, *prefix_indptr, *prefix_indices, *prefix_last;
  int64_t groups, prefix_pages;
};

int chunk_call(const void* q, const int32_t* q_indptr, const void* kv_cache,
               const int32_t* kv_page_indptr, const int32_t* kv_page_indices,
               const int32_t* kv_last_page_len, const SharedArgs* shared, void* o, float* lse,
               int64_t batch, int64_t total_q, int64_t num_q_heads, int64_t num_kv_heads,
               int64_t head_dim, int64_t page_size, int64_t total_pages, int64_t num_pool_pages,
               const int64_t q_stride[3], const int64_t kv_stride[5], float softmax_scale,
               int causal, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  AKT_CHECK(dtype == AKT_DTYPE_F16 || dtype == AKT_DTYPE_BF16,
            "dtype must be AKT_DTYPE_F16 or AKT_DTYPE_BF16, got %d", dtype);
  AKT_CHECK(batch >= 0 && total_q >= 0 && total_pages >= 0 && num_pool_pages >= 0,
            "sizes must be non-negative");
  AKT_CHECK(!shared || (shared->groups >= 0 && shared->prefix_pages >= 0),
            "sizes must be non-negative");
  AKT_CHECK(num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0,
            "num_q_heads (%lld) must be a positive multiple of num_kv_heads (%lld)",
            (long long)num_q_heads, (long long)num_kv_heads);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return set_error(AKT_ERR_UNSUPPORTED, "chunk attention head_dim %lld not supported (64, 128, 256)",
                     (long long)head_dim);
  if (num_q_heads / num_kv_heads > kCkRows)
    return set_error(AKT_ERR_UNSUPPORTED, "chunk attention serves up to %d query heads per kv head",
                     kCkRows);
  AKT_CHECK(page_size > 0 && page_size < (1 << 20), "page_size out of range");
  AKT_CHECK(batch < (1ll << 30) && total_q < (1ll << 30) && num_q_heads < (1 << 20),
            "problem too large");
  AKT_CHECK(total_pages < (1ll << 31) && total_pages * page_size < (1ll << 30),
            "the page table spans too many tokens");
  AKT_CHECK(!shared || (shared->groups < (1ll << 30) && shared->prefix_pages < (1ll << 31) &&
                        shared->prefix_pages * page_size < (1ll << 30)),
            "the prefixes' page table spans too many tokens");
  AKT_CHECK(!shared || total_q * num_q_heads < (1ll << 31) / 64, "too many query rows");
  AKT_CHECK(std::isfinite(softmax_scale), "softmax_scale must be finite");
  if (batch == 0 || total_q == 0) return AKT_OK;
  AKT_CHECK(q && q_indptr && kv_cache && kv_page_indptr && kv_last_page_len && o && q_stride &&
                kv_stride && (kv_page_indices || total_pages == 0),
            "all pointers are required");
  AKT_CHECK(!shared || (shared->group_indptr && shared->prefix_indptr &&
                        (shared->prefix_last || shared->groups == 0) &&
                        (shared->prefix_indices || shared->prefix_pages == 0)),
            "all pointers are required");
  AKT_CHECK(q_stride[2] == 1 && kv_stride[4] == 1, "head_dim stride must be 1");
  AKT_CHECK(rows_aligned16(q, q_stride, 2) && rows_aligned16(kv_cache, kv_stride, 4) &&
                aligned16(o) && (!lse || aligned4(lse)),
            "tensors must have 16-byte aligned rows");
  AKT_CHECK(kv_stride[3] >= 0 && kv_stride[3] < (1 << 22), "slot stride out of range [0, 2^22)");
  const int64_t G = num_q_heads / num_kv_heads;
  const ChunkPlan plan =
      chunk_plan(batch, total_q, num_kv_heads, G, head_dim, page_size, total_pages,
                 shared ? shared->groups : -1, shared ? shared->prefix_pages : 0);
  const size_t need =
      workspace_bytes_of(plan, shared ? 2 * total_q * num_q_heads * state_bytes((int)head_dim) : 0);
  if (!workspace || workspace_bytes < need)
    return set_error(AKT_ERR_WORKSPACE, "chunk attention needs a workspace of %zu bytes, got %zu",
                     need, workspace ? workspace_bytes : (size_t)0);
  AKT_CHECK(aligned16(workspace), "the workspace must be 16-byte aligned");
  AKT_CHECK(plan.counters <= (int64_t)(AKT_WORKSPACE_ZERO_BYTES - 256) / 4,
            "too many workgroups");

  ChunkParams p = {};
  p.q = (const half_t*)q;
  p.pool = (const half_t*)kv_cache;
  p.o = (half_t*)o;
  p.lse = lse;
  p.q_indptr = q_indptr;
  p.indptr = kv_page_indptr;
  p.indices = kv_page_indices;
  p.last_len = kv_last_page_len;
  p.arrive = (int*)((char*)workspace + 256);
  p.partials = (char*)workspace + round_up(AKT_WORKSPACE_ZERO_BYTES, 256);
  p.q_st = q_stride[0];
  p.q_sh = q_stride[1];
  p.sp = kv_stride[0];
  p.skv = kv_stride[1];
  p.sh = kv_stride[2];
  p.ss = (int)kv_stride[3];
  p.total_q = (int)total_q;
  p.total_pages = (int)total_pages;
  p.num_pool_pages = (int)(num_pool_pages < (1ll << 31) ? num_pool_pages : (1ll << 31) - 1);
  p.B = (int)batch;
  p.Hq = (int)num_q_heads;
  p.Hkv = (int)num_kv_heads;
  p.G = (int)G;
  p.TR = (int)(32 * chunk_waves((int)head_dim) / G);
  p.g_magic = (uint32_t)((65536 + G - 1) / G);
  p.page_size = (int)page_size;
  const uint64_t magic = (1ull << 32) / (uint64_t)page_size;
  p.page_magic = (uint32_t)(magic < 0xffffffffull ? magic : 0xffffffffull);
  p.causal = causal ? 1 : 0;
  // As in prefill: a negative scale flips Q's sign, a zero one becomes FLT_MIN.
  p.neg_q = softmax_scale < 0.f ? 1 : 0;
  p.qk_scale = fmaxf(fabsf(softmax_scale) * kLog2e, FLT_MIN);
  p.min_keys = kCkMinKeys;
  p.split_tokens = plan.split_tokens;
  p.kinds = plan.kinds;
  p.wgs = (int)plan.wgs;
  p.many_counter = (int)plan.many_counter;
  p.many_partial = plan.many_partial;
  hipStream_t st = (hipStream_t)stream;
  const bool bf16 = dtype == AKT_DTYPE_BF16;
  if (!shared) {
    if (head_dim == 64) return chunk_launch_64(p, bf16, st);
    if (head_dim == 256) return chunk_launch_256(p, bf16, st);
    return chunk_launch_128(p, bf16, st);
  }
  p.group_indptr = shared->group_indptr;
  p.prefix_indptr = shared->prefix_indptr;
  p.prefix_indices = shared->prefix_indices;
  p.prefix_last = shared->prefix_last;
  p.groups = (int)shared->groups;
  p.prefix_pages = (int)shared->prefix_pages;
  p.states = p.partials + round_up(plan.partial_bytes, 256);
  const int rc = head_dim == 64    ? shared_launch_64(p, bf16, st)
                 : head_dim == 256 ? shared_launch_256(p, bf16, st)
                                   : shared_launch_128(p, bf16, st);
  return rc != AKT_OK ? rc : shared_merge_launch(p, (int)head_dim, bf16, st);
}

}  // namespace
}  // namespace akt

using namespace akt;

extern "C" size_t akt_chunk_paged_workspace_size(int64_t batch, int64_t total_q,
                                                 int64_t num_q_heads, int64_t num_kv_heads,
                                                 int64_t head_dim, int64_t page_size,
                                                 int64_t total_pages) {
  if (batch <= 0 || total_q <= 0 || page_size <= 0 || total_pages < 0 ||
      !sizes_served(num_q_heads, num_kv_heads, head_dim))
    return 0;
  return workspace_bytes_of(chunk_plan(batch, total_q, num_kv_heads, num_q_heads / num_kv_heads,
                                       head_dim, page_size, total_pages, -1, 0), 0);
}

extern "C" int akt_chunk_paged_fwd(const void* q, const int32_t* q_indptr, const void* kv_cache,
                                   const int32_t* kv_page_indptr, const int32_t* kv_page_indices,
                                   const int32_t* kv_last_page_len, void* o, float* lse,
                                   int64_t batch, int64_t total_q, int64_t num_q_heads,
                                   int64_t num_kv_heads, int64_t head_dim, int64_t page_size,
                                   int64_t total_pages, int64_t num_pool_pages,
                                   const int64_t q_stride[3], const int64_t kv_stride[5],
                                   float softmax_scale, int causal, int dtype, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  return chunk_call(q, q_indptr, kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len,
                    nullptr, o, lse, batch, total_q, num_q_heads, num_kv_heads, head_dim, page_size,
                    total_pages, num_pool_pages, q_stride, kv_stride, softmax_scale, causal, dtype,
                    workspace, workspace_bytes, stream);
}

extern "C" size_t akt_shared_prefix_paged_workspace_size(int64_t batch, int64_t total_q,
                                                         int64_t num_q_heads, int64_t num_kv_heads,
                                                         int64_t head_dim, int64_t page_size,
                                                         int64_t total_pages, int64_t groups,
                                                         int64_t prefix_pages) {
  if (batch <= 0 || total_q <= 0 || page_size <= 0 || total_pages < 0 || groups < 0 ||
      prefix_pages < 0 || !sizes_served(num_q_heads, num_kv_heads, head_dim))
    return 0;
  return workspace_bytes_of(chunk_plan(batch, total_q, num_kv_heads, num_q_heads / num_kv_heads,
                                       head_dim, page_size, total_pages, groups, prefix_pages),
                            2 * total_q * num_q_heads * state_bytes((int)head_dim));
}

extern "C" int akt_shared_prefix_paged_fwd(
    const void* q, const int32_t* q_indptr, const void* kv_cache, const int32_t* kv_page_indptr,
    const int32_t* kv_page_indices, const int32_t* kv_last_page_len, const int32_t* group_indptr,
    const int32_t* prefix_page_indptr, const int32_t* prefix_page_indices,
    const int32_t* prefix_last_page_len, void* o, float* lse, int64_t batch, int64_t total_q,
    int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t page_size,
    int64_t total_pages, int64_t groups, int64_t prefix_pages, int64_t num_pool_pages,
    const int64_t q_stride[3], const int64_t kv_stride[5], float softmax_scale, int causal,
    int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const SharedArgs shared = {group_indptr, prefix_page_indptr, prefix_page_indices,
                             prefix_last_page_len, groups, prefix_pages};
  return chunk_call(q, q_indptr, kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len,
                    &shared, o, lse, batch, total_q, num_q_heads, num_kv_heads, head_dim, page_size,
                    total_pages, num_pool_pages, q_stride, kv_stride, softmax_scale, causal, dtype,
                    workspace, workspace_bytes, stream);
}

namespace akt {
#endif  // AKT_CHUNK_TU
}  // namespace akt
