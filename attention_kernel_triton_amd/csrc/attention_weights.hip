// Attention that cached tokens draw, summed over calls (gfx950):
//   w[row_b, h, j] += sum over the tokens i of sequence b that see key j, and the query heads of kv
//                     head h, of exp(scale q_i . k_j - lse_i).
// q, lse and the page table are those of an attention call (paged decode, chunk or shared
// prefix); sequence b's token i sits at position len_b - n_b + i, as there.
//
// S = Q K^T is computed with rows (token, query head of the group; token major) along the registers
// and keys along the lanes (v_mfma_f32_32x32x16), so a lane sums its key's weights in registers, and
// every sum has one owner and one order: no atomics on the sums, and results do not depend on the run.
// The two kinds of sequences are served by workgroups of their own, in one launch (share_of):
//
// Few rows (at most 32 to a kv head).  HBM-bound: K is read once.  The keys of a (sequence, kv head)
// are cut into steps of 32 (64 at D = 64), which stand on an axis; a wave serves a range of it as one
// stream, with the keys of the next step and the page ids of the one after it on their way while a step
// is computed.  Waves do not meet.
//
// Many rows.  Bound by the three VALU instructions to a score (fma, exp2, add) and the MFMAs, which
// mostly add up.  A tile is 256 keys of one (sequence, kv head), wave w's the keys 64 w .. 64 w + 63 of
// them, which it reads into registers once; the rows that see the tile go by in blocks of 32, staged
// in LDS two blocks at a time for the four waves, the scores of one block computed beside the weights of the
// one before.  A block's 16 terms are summed before they join the total.  The tiles stand on an axis,
// each as long as its blocks plus kWTileCost, which is cut into equal ranges, one to a workgroup.  A tile
// of many blocks may be cut: its parts leave their sums in slots (two to a range, as in
// paged_chunk.hip) and count themselves; the last one adds them up in the order of the ranges.
//
// The workgroups stay for the whole launch and find their ranges from the page table (no plan on the
// host).
//
// The weights are 2^(scale log2(e) s - lse log2(e)) in 32 bits: q and k are taken as they are, s, the
// exponent and all sums are 32-bit, so the sums are as near to 64 bits as a plain 32-bit form (3e-8).
// Keys that a row does not see are left out by a select, rows that saw none (lse -inf) count nothing.
//
// What it measured (us; bf16 or fp16, 32 query heads over 8, D = 128): one token each of 32 sequences over
// 256 to 8,192 keys 43.6 (201 MB, 4.6 TB/s; 63.7 with a tile of 256 keys to a workgroup and no
// look-ahead), 2,048 tokens after 6,000 139 (118 GFLOP, 850 TFLOP/s; 312 with one block of rows staged
// at a time and whole tiles: 256 keys of each of 8 heads are 256 tiles of unlike lengths).  There a
// block of 32 rows by 256 keys takes a wave about 142 VALU instructions beside its 16 MFMAs; the matrix
// pipe is busy 38% of the time, and two workgroups to a processor take 1.07 us a block each where one
// alone takes 0.85: the two kinds of instructions hardly overlap.  (At D = 128 the kernel spills eight
// vector registers, at the tiles' starts and ends, not in the walk over the blocks.)  Five tokens after twelve: 5.3,
// of which a launch is 4; the rest is the sequences' table, the page ids, K and q, one after another.
#include <math.h>

#include <cmath>

#include "akt_host.hpp"
#include "attn_tile.hpp"

namespace akt {
namespace {

constexpr int kWWaves = 4;
constexpr int kWThreads = 64 * kWWaves;
constexpr int kWKeys = 64;                   // keys of a wave
constexpr int kWTile = kWKeys * kWWaves;  // and of a workgroup
// Cost of a tile's start and end, in blocks of rows, and of a tile with keys that not every row sees,
// in G blocks: its masked blocks take longer (us, 2,048 tokens after 6,000: 143.2; with 3 and 12 for the
// first 144.2 and 144.4, with 1 and 4 for the second 143.6 and 145.3).
constexpr int kWTileCost = 6;
constexpr int kWDiagCost = 2;
constexpr int kWTable = 1024;                // sequences whose places a workgroup keeps in LDS
constexpr int kWFew = 32;                    // rows of a sequence and kv head that are few

struct WeightParams {
  const half_t* q;
  const half_t* pool;
  const float* lse;  // [total_q, Hq]
  float* w;          // [N, Hkv, L]
  const int32_t* q_indptr;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last_len;
  const int32_t* rows;  // row of w of each sequence; null: its own number
  int64_t q_st, q_sh;
  int64_t sp, sh, ss;  // page, head and slot strides of the pool
  int64_t w_sn, w_sh;
  int N;
  int64_t L;
  int total_q, total_pages, num_pool_pages;
  int B, Hq, Hkv, G;
  int page_size;
  uint32_t page_magic;  // min(2^32 - 1, floor(2^32 / page_size))
  uint32_t g_magic;     // the same for G
  int causal;
  int window;  // only the last so many of a sequence's tokens count
  float scale;  // softmax_scale * log2(e)
  int* arrive;      // a counter to a range (zero between launches)
  float* partials;  // two slots of kWTile sums to a range
};

// n / d for 0 <= n < 2^31, given magic = min(2^32 - 1, floor(2^32 / d)).
__device__ __forceinline__ int div_magic(int n, int d, uint32_t magic) {
  const int q = (int)__umulhi((uint32_t)n, magic);
  return n - q * d >= d ? q + 1 : q;
}

struct WSeq {
  int q0, n;  // first token of q that counts, tokens that count
  int ip0, len;
  int row;    // of the sums; -1: none
};
// Table entries outside their ranges are taken clamped, so nothing outside the arrays is touched.
__device__ __forceinline__ WSeq load_wseq(const WeightParams& p, int b) {
  WSeq s;
  const int q0 = min(max(p.q_indptr[b], 0), p.total_q);
  const int n = min(max(p.q_indptr[b + 1], q0), p.total_q) - q0;
  s.ip0 = min(max(p.indptr[b], 0), p.total_pages);
  const int np = min(max(p.indptr[b + 1], s.ip0), p.total_pages) - s.ip0;
  s.len = np > 0 ? (np - 1) * p.page_size + min(max(p.last_len[b], 0), p.page_size) : 0;
  s.n = min(n, p.window);
  s.q0 = q0 + n - s.n;
  s.row = p.rows ? p.rows[b] : b;
  if ((uint32_t)s.row >= (uint32_t)p.N) s.row = -1;
  return s;
}

// The tiles of one (sequence, kv head) on the axis.  A tile's blocks of rows are those from `skip`
// on: the first t0 tiles hold keys that every row sees (all blocks), tile t0 + i skips f0 + 8 G i.
struct WHead {
  int64_t full;  // blocks and cost of a tile that skips none
  int tiles, t0, f0, step, diag;
};
__device__ __forceinline__ WHead head_of(const WeightParams& p, const WSeq& s) {
  WHead h;
  h.full = (int64_t)(((int64_t)s.n * p.G + 31) / 32) + kWTileCost;
  h.tiles = s.n > 0 ? (s.len + kWTile - 1) / kWTile : 0;
  const int first = s.len - s.n;  // position of the first row
  h.t0 = !p.causal ? h.tiles : first < 0 ? 0 : min(first / kWTile + 1, h.tiles);
  h.f0 = (int)((int64_t)max(h.t0 * kWTile - first, 0) * p.G / 32);
  h.step = kWTile / 32 * p.G;
  h.diag = kWDiagCost * p.G;
  return h;
}
__device__ __forceinline__ int64_t skipped(const WHead& h, int t) {
  return t < h.t0 ? 0 : h.f0 + (int64_t)(t - h.t0) * h.step;
}
// Start of tile t (t = tiles: the length of all).
__device__ __forceinline__ int64_t tile_start(const WHead& h, int t) {
  const int64_t i = max(t - h.t0, 0);
  return t * h.full - i * h.f0 - i * (i - 1) / 2 * h.step + i * h.diag;
}
__device__ __forceinline__ int64_t w_uniform64(int64_t v) {
  const uint32_t lo = (uint32_t)uniform((int)(uint32_t)v);
  const uint32_t hi = (uint32_t)uniform((int)(uint32_t)(v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
// floor(a / b) for 0 <= a < 2^50, b >= 1 (see div_range in paged_chunk.hip).
__device__ __forceinline__ int64_t w_div(int64_t a, int64_t b) {
  return w_uniform64((int64_t)((double)a / (double)b));
}

template <int D>
__host__ __device__ constexpr int weight_waves() {
  return D <= 128 ? 2 : 1;  // waves to a SIMD
}

// Sequences' places: in LDS, unless there are too many.
struct WTable {
  const int4* seq;  // null: load_wseq
  const int* row;
};
__device__ __forceinline__ WSeq seq_of(const WeightParams& p, const WTable& t, int b) {
  if (!t.seq) return load_wseq(p, b);
  const int4 s = t.seq[b];
  return WSeq{s.x, s.y, s.z, s.w, t.row[b]};
}
// The kinds; a sequence that has no row of sums is of neither.
__device__ __forceinline__ bool is_few(const WeightParams& p, const WSeq& s) {
  return s.n > 0 && s.row >= 0 && s.n * p.G <= kWFew;
}
__device__ __forceinline__ bool is_many(const WeightParams& p, const WSeq& s) {
  return s.row >= 0 && s.n * p.G > kWFew;
}

// Keys of a step of few rows, and what a unit's start costs a wave, in steps.
__host__ __device__ constexpr int few_keys(int D) { return D <= 64 ? 64 : 32; }
constexpr int kFewCost = 1;
__device__ __forceinline__ int few_length(const WSeq& s, int keys) {
  return s.len > 0 ? (s.len + keys - 1) / keys + kFewCost : 0;
}

// A step of few rows.
struct FewWStep {
  int b, kvh;      // b = -1: the range is done
  int64_t start;   // of the unit on the axis
  int q0, n, ip0, len, row;
  int j, j1;       // the step, and the first that is not the wave's
};

template <int D, bool BF16>
__device__ __forceinline__ void few_weights(const WeightParams& p, const WTable& tab, int block,
                                            int W) {
  typedef Elt<BF16> E;
  constexpr int KS = D / 16;
  constexpr int KEYS = few_keys(D), NC = KEYS / 32;  // columns of 32 keys
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int l32 = lane & 31, g = lane >> 5;
  // ---- this wave's range: consecutive ones go to one XCD (workgroup i runs on XCD i % 8).
  const int range = ((block % 8) * (W / 8) + block / 8) * kWWaves + wave;
  auto seq_length = [&](int b) -> int64_t {
    if (b >= p.B) return 0;
    const WSeq s = seq_of(p, tab, b);
    return is_few(p, s) ? (int64_t)few_length(s, KEYS) * p.Hkv : 0;
  };
  int64_t length = seq_length(lane), inc = wave_inclusive_scan64(length);
  int64_t total = read_lane64(inc, 63);
  for (int jb = 64; jb < p.B; jb += 64)
    total += read_lane64(wave_inclusive_scan64(seq_length(jb + lane)), 63);
  const int64_t Lw = w_div(total + W * kWWaves - 1, W * kWWaves);
  const int64_t x0 = range * Lw;
  if (x0 >= total) return;
  const int64_t x1 = x0 + Lw < total ? x0 + Lw : total;

  auto take_seq = [&](FewWStep& s) -> bool {
    const WSeq q = seq_of(p, tab, s.b);
    s.q0 = uniform(q.q0);
    s.n = uniform(q.n);
    s.ip0 = uniform(q.ip0);
    s.len = uniform(q.len);
    s.row = uniform(q.row);
    return uniform(is_few(p, q) && q.len > 0);
  };
  // The first step of the unit that s names, or of the next one with steps in the range.
  auto enter = [&](FewWStep& s) {
    for (;;) {
      if (s.start >= x1) {
        s.b = -1;
        return;
      }
      const int steps = (s.len + KEYS - 1) / KEYS;
      s.j = uniform((int)min(max(x0 - s.start, (int64_t)0), (int64_t)steps));
      s.j1 = uniform((int)min(x1 - s.start, (int64_t)steps));
      if (s.j < s.j1) return;
      s.start = w_uniform64(s.start + steps + kFewCost);
      if (++s.kvh < p.Hkv) continue;
      s.kvh = 0;
      do {
        if (++s.b >= p.B) {
          s.b = -1;
          return;
        }
      } while (!take_seq(s));
    }
  };
  auto advance = [&](FewWStep& s) {
    if (++s.j < s.j1) return;
    s.start = w_uniform64(s.start + (s.len + KEYS - 1) / KEYS + kFewCost);
    if (++s.kvh == p.Hkv) {
      s.kvh = 0;
      do {
        if (++s.b >= p.B) {
          s.b = -1;
          return;
        }
      } while (!take_seq(s));
    }
    enter(s);
  };
  FewWStep cur;
  {
    int64_t at = 0;
    for (int jb = 0;;) {
      const uint64_t m = __ballot(at + inc > x0);
      if (m) {
        const int l = __builtin_ctzll(m);
        cur.b = uniform(jb + l);
        at += read_lane64(inc - length, l);
        break;
      }
      at += read_lane64(inc, 63);
      jb += 64;
      if (jb >= p.B) return;
      length = seq_length(jb + lane);
      inc = wave_inclusive_scan64(length);
    }
    take_seq(cur);
    const int unit = (cur.len + KEYS - 1) / KEYS + kFewCost;
    cur.kvh = uniform((int)w_div(x0 - at, unit));
    cur.start = w_uniform64(at + (int64_t)cur.kvh * unit);
    enter(cur);
  }
  if (cur.b < 0) return;

  // ---- loads.  Lane (l32, g) takes chunks 2 k + g of keys l32 (and 32 + l32) of a step.
  int id[NC], slot[NC];
  auto load_ids = [&](const FewWStep& s) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int key = min(s.j * KEYS + 32 * i + l32, s.len - 1);
      const int lp = div_magic(key, p.page_size, p.page_magic);
      slot[i] = key - lp * p.page_size;
      id[i] = p.indices[s.ip0 + lp];
    }
  };
  // Loads come back in the order in which they are asked for: a step's page ids are asked for before
  // the keys of the step before it, so that waiting for them does not wait for those.
  auto load_k = [&](const FewWStep& s, const FewWStep& after, uint4_t (&kf)[NC][KS], bool (&ok)[NC]) {
    const half_t* src[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      ok[i] = s.j * KEYS + 32 * i + l32 < s.len && (uint32_t)id[i] < (uint32_t)p.num_pool_pages;
      // A key that cannot be read takes a row of q: its sum is not written.
      src[i] = (ok[i] ? p.pool + id[i] * p.sp + s.kvh * p.sh + (int64_t)slot[i] * p.ss : p.q) + 8 * g;
    }
    if (after.b >= 0) load_ids(after);
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int k = 0; k < KS; ++k) kf[i][k] = ld16(src[i] + 16 * k);
  };
  // Rows: fragments of row l32 (the last one's again behind it) and its lse, which is looked at when the
  // unit's first step is served (its keys, asked for before, then need not be waited for here).
  uint4_t qf[KS];
  float lse_row;
  bool fresh = true;
  auto load_rows = [&](const FewWStep& s) {
    const int row = min(l32, s.n * p.G - 1), tok = div_magic(row, p.G, p.g_magic);
    const int head = s.kvh * p.G + row - tok * p.G;
    const half_t* src = p.q + (int64_t)(s.q0 + tok) * p.q_st + (int64_t)head * p.q_sh + 8 * g;
    lse_row = p.lse[(int64_t)(s.q0 + tok) * p.Hq + head];
#pragma unroll
    for (int k = 0; k < KS; ++k) qf[k] = ld16(src + 16 * k);
    fresh = true;
  };
  // -lse log2(e) of the rows of the lane's registers: register 4 j + i of half g is row 8 j + 4 g + i.
  float nl[16];
  uint32_t gone = 0;  // bit i: row i is not there, or drew on none (lse -inf)
  auto take_rows = [&](const FewWStep& s) {
    const int rows = s.n * p.G;
    const bool none = l32 >= rows || lse_row == -__builtin_inff();
    const float n = none ? -__builtin_inff() : -lse_row * kLog2e;
    gone = (uint32_t)__ballot(none);
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (8 * (r / 4) < rows)  // wave-uniform
        nl[r] = __shfl(n, 8 * (r / 4) + 4 * g + r % 4, 64);
    fresh = false;
  };
  const float c = p.scale;
  // Weights of a step's keys, added to their sums by half g for keys 32 g + l32 (one column: half 0).
  auto serve = [&](const FewWStep& s, const uint4_t (&kf)[NC][KS], const bool (&ok)[NC], float old) {
    const int rows = s.n * p.G, first = s.len - s.n, key = s.j * KEYS + l32;
    float16_t sc[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[i][r] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) sc[i] = E::mfma(E::as8(qf[k]), E::as8(kf[i][k]), sc[i]);
    }
    float sum[NC] = {};
    bool odd = p.causal && s.j * KEYS + KEYS - 1 > first;  // keys that not every row sees
    if (!odd) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (8 * j < rows)  // wave-uniform
#pragma unroll
          for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              sum[i] += fast_exp2(__builtin_fmaf(sc[i][4 * j + r], c, nl[4 * j + r]));
      // A score that is not finite makes NaN of a row that is not there or drew on none.
      bool nan = false;
#pragma unroll
      for (int i = 0; i < NC; ++i) nan |= sum[i] != sum[i];
      odd = __any(nan);
    }
    if (odd) {
#pragma unroll
      for (int i = 0; i < NC; ++i) sum[i] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (8 * j < rows)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = 8 * j + 4 * g + r;
            const int last = (gone >> row) & 1 ? -1
                             : p.causal               ? first + div_magic(row, p.G, p.g_magic)
                                                      : s.len - 1;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
              const float e = fast_exp2(__builtin_fmaf(sc[i][4 * j + r], c, nl[4 * j + r]));
              sum[i] += last >= key + 32 * i ? e : 0.f;
            }
          }
    }
    float out = xor32_sum(sum[0]);
    bool mine = ok[0] && g == 0;
    if constexpr (NC == 2) {
      const float out1 = xor32_sum(sum[1]);
      if (g) {
        out = out1;
        mine = ok[1];
      }
    }
    const int at = s.j * KEYS + (NC == 2 ? lane : l32);
    if (mine && at < p.L) p.w[s.row * p.w_sn + s.kvh * p.w_sh + at] = old + out;
  };
  auto load_old = [&](const FewWStep& s) -> float {
    const int at = min(s.j * KEYS + (NC == 2 ? lane : l32), s.len - 1);
    return at < p.L ? p.w[s.row * p.w_sn + s.kvh * p.w_sh + at] : 0.f;
  };

  // ---- the stream.
  uint4_t kA[NC][KS], kB[NC][KS];
  bool okA[NC], okB[NC];
  load_ids(cur);
  load_rows(cur);
  FewWStep next = cur;
  advance(next);
  load_k(cur, next, kA, okA);
  auto step = [&](uint4_t (&k0)[NC][KS], bool (&ok0)[NC], uint4_t (&k1)[NC][KS], bool (&ok1)[NC]) -> bool {
    FewWStep after = next;
    if (next.b >= 0) advance(after);
    const float old = load_old(cur);
    if (next.b >= 0) load_k(next, after, k1, ok1);
    if (fresh) take_rows(cur);
    serve(cur, k0, ok0, old);
    if (next.b < 0) return false;
    if (next.b != cur.b || next.kvh != cur.kvh) load_rows(next);
    cur = next;
    next = after;
    return true;
  };
#pragma clang loop unroll(disable)
  for (;;) {
    if (!step(kA, okA, kB, okB)) return;
    if (!step(kB, okB, kA, okA)) return;
  }
}

// A tile and the part of its blocks that a workgroup serves.
struct WTile {
  int b, kvh, t;
  int64_t start;   // on the axis
  int q0, n, ip0, len;
  int row;             // of the sums; -1: none
  int blocks, j0, j1;  // its blocks of rows, and those of the part
  int r0;              // row of block j0
};

// LDS of a workgroup of many rows.
template <int D>
struct ManyLds {
  static constexpr int kStage = 64;  // rows to a stage: two blocks
  char q[2][kStage * D * 2];
  // A wave may still add the weights of a stage's second block while another stores the stage after
  // the next, so rows' numbers are kept for longer than the rows.
  float4_t nl[4][kStage / 4];  // -lse log2(e) of each row
  int4 lim[4][kStage / 4];     // last key that each row sees, -1: none
  int last;
};

template <int D, bool BF16>
__device__ __forceinline__ void many_weights(const WeightParams& p, const WTable& tab,
                                             ManyLds<D>& lds, int block, int W) {
  typedef Elt<BF16> E;
  constexpr int KS = D / 16;
  constexpr int CPR = D / 8;
  constexpr int ROWB = D * 2;
  constexpr int kStage = ManyLds<D>::kStage;
  constexpr int PER_T = kStage * CPR / kWThreads;  // chunks of a stage to a thread
  constexpr int kPass = kWThreads / CPR;           // rows between a thread's chunks
  constexpr int kFirst = 32;  // VALU instructions of a step before its first MFMA, while rows arrive
  auto& lds_q = lds.q;
  auto& lds_nl = lds.nl;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int l32 = lane & 31, g = lane >> 5;

  // ---- this workgroup's range.  Workgroup i runs on XCD i % 8: consecutive ranges go to one XCD.
  const int wg = (block % 8) * (W / 8) + block / 8;
  auto seq_length = [&](int b) -> int64_t {
    if (b >= p.B) return 0;
    const WSeq s = seq_of(p, tab, b);
    if (!is_many(p, s)) return 0;
    const WHead h = head_of(p, s);
    return tile_start(h, h.tiles) * p.Hkv;
  };
  int64_t length = seq_length(lane), inc = wave_inclusive_scan64(length);
  int64_t total = read_lane64(inc, 63);
  for (int jb = 64; jb < p.B; jb += 64)
    total += read_lane64(wave_inclusive_scan64(seq_length(jb + lane)), 63);
  const int64_t Lw = max(w_div(total + W - 1, W), (int64_t)(kWTileCost + 1));
  const int64_t x0 = wg * Lw;
  if (x0 >= total) return;
  const int64_t x1 = x0 + Lw < total ? x0 + Lw : total;

  // ---- the tiles of the range, from the one that holds x0 on.  `head` is of the tile entered last.
  WHead head;
  auto take_seq = [&](WTile& a) {
    const WSeq s = seq_of(p, tab, a.b);
    a.q0 = uniform(s.q0);
    a.n = uniform(s.n);
    a.ip0 = uniform(s.ip0);
    a.len = uniform(s.len);
    a.row = uniform(s.row);
    head = head_of(p, WSeq{a.q0, a.n, a.ip0, a.len, a.row});
    if (!is_many(p, WSeq{a.q0, a.n, a.ip0, a.len, a.row})) head.tiles = 0;
  };
  // The part of the tile that a names; one without blocks is passed over.
  auto enter = [&](WTile& a) {
    for (;;) {
      if (a.start >= x1) {
        a.b = -1;
        return;
      }
      const int64_t skip = skipped(head, a.t);
      a.blocks = uniform((int)(head.full - kWTileCost - skip));
      a.j0 = uniform((int)min(max(x0 - a.start, (int64_t)0), (int64_t)a.blocks));
      a.j1 = uniform((int)min(x1 - a.start, (int64_t)a.blocks));
      a.r0 = uniform((int)(32 * (skip + a.j0)));
      if (a.j0 < a.j1) return;
      a.start = w_uniform64(a.start + a.blocks + kWTileCost + (a.t >= head.t0 ? head.diag : 0));
      if (++a.t < head.tiles) continue;
      a.t = 0;
      if (++a.kvh < p.Hkv) continue;
      a.kvh = 0;
      do {
        if (++a.b >= p.B) {
          a.b = -1;
          return;
        }
        take_seq(a);
      } while (head.tiles == 0);
    }
  };
  auto advance = [&](WTile& a) {
    a.start = w_uniform64(a.start + a.blocks + kWTileCost + (a.t >= head.t0 ? head.diag : 0));
    if (++a.t == head.tiles) {
      a.t = 0;
      if (++a.kvh == p.Hkv) {
        a.kvh = 0;
        do {
          if (++a.b >= p.B) {
            a.b = -1;
            return;
          }
          take_seq(a);
        } while (head.tiles == 0);
      }
    }
    enter(a);
  };
  WTile cur;
  {
    int64_t at = 0;
    for (int jb = 0;;) {
      const uint64_t m = __ballot(at + inc > x0);
      if (m) {
        const int l = __builtin_ctzll(m);
        cur.b = uniform(jb + l);
        at += read_lane64(inc - length, l);
        break;
      }
      at += read_lane64(inc, 63);
      jb += 64;
      if (jb >= p.B) return;
      length = seq_length(jb + lane);
      inc = wave_inclusive_scan64(length);
    }
    take_seq(cur);
    const int64_t per = tile_start(head, head.tiles);
    cur.kvh = (int)w_div(x0 - at, per);
    at += cur.kvh * per;
    cur.t = 0;
    for (int lo = 1, hi = head.tiles; lo < hi;) {  // last t whose start is at or before x0
      const int mid = (lo + hi) / 2;
      if (at + tile_start(head, mid) <= x0) {
        cur.t = mid;
        lo = mid + 1;
      } else {
        hi = mid;
      }
    }
    cur.t = uniform(cur.t);
    cur.start = w_uniform64(at + tile_start(head, cur.t));
    enter(cur);
  }
  if (cur.b < 0) return;

  // ---- K: lane (l32, g) holds chunks 2 k + g of keys l32 and 32 + l32 of the wave's.
  uint4_t kf[2][KS];
  bool ok[2];
  auto load_k = [&](const WTile& a) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = a.t * kWTile + kWKeys * wave + 32 * i + l32;
      const int kk = min(key, a.len - 1), lp = div_magic(kk, p.page_size, p.page_magic);
      const int id = p.indices[a.ip0 + lp];
      ok[i] = key < a.len && (uint32_t)id < (uint32_t)p.num_pool_pages;
      // A key that cannot be read takes a row of q: its sum is not written.
      const half_t* src = (ok[i] ? p.pool + id * p.sp + a.kvh * p.sh +
                                       (int64_t)(kk - lp * p.page_size) * p.ss
                                 : p.q) + 8 * g;
#pragma unroll
      for (int k = 0; k < KS; ++k) kf[i][k] = ld16(src + 16 * k);
    }
  };

  // ---- rows, a stage at a time: global memory -> registers -> LDS.  A thread's chunks are those of
  // column tid % CPR of rows tid / CPR + kPass i.
  uint4_t st[PER_T];
  float nl_st = 0.f;
  int lim_st = -1;
  // Of the next stage to load: the thread's chunks (address and head of each row), and the row whose
  // numbers it looks up (threads 0 .. kStage - 1).
  const half_t* qsrc[PER_T];
  int hd[PER_T], row0;
  const float* lsrc;
  int tokr, hdr;
  // From a row to the one kStage behind it: heads and tokens on, and back by G heads for one more
  // token where that is past the last.
  const int adv_t = kStage / p.G, adv_h = kStage - adv_t * p.G;
  const int64_t q_adv = adv_t * p.q_st + adv_h * p.q_sh, q_wrap = p.q_st - p.G * p.q_sh;
  auto start_rows = [&](const WTile& a) {
    row0 = a.r0 + tid / CPR;
#pragma unroll
    for (int i = 0; i < PER_T; ++i) {
      const int row = row0 + kPass * i, tok = div_magic(row, p.G, p.g_magic);
      hd[i] = row - tok * p.G;
      qsrc[i] = p.q + (int64_t)(a.q0 + tok) * p.q_st + (int64_t)(a.kvh * p.G + hd[i]) * p.q_sh +
                tid % CPR * 8;
    }
    tokr = div_magic(a.r0 + tid, p.G, p.g_magic);
    hdr = a.r0 + tid - tokr * p.G;
    lsrc = p.lse + (int64_t)(a.q0 + tokr) * p.Hq + a.kvh * p.G + hdr;
  };
  auto load_stage = [&](const WTile& a) {
    const int rows = a.n * p.G;
#pragma unroll
    for (int i = 0; i < PER_T; ++i) {
      // (A row past the last takes any: no key is seen by it.)
      st[i] = ld16(row0 + kPass * i < rows ? qsrc[i] : p.q);
      qsrc[i] += q_adv;
    }
    row0 += kStage;
    if (adv_h) {
#pragma unroll
      for (int i = 0; i < PER_T; ++i) {
        hd[i] += adv_h;
        if (hd[i] >= p.G) {
          hd[i] -= p.G;
          qsrc[i] += q_wrap;
        }
      }
    }
    if (wave * 64 < kStage) {
      const bool in = tokr < a.n;
      const float l = *(in ? lsrc : p.lse);
      // A row that saw no key (lse -inf) drew on none.
      const bool none = l == -__builtin_inff();
      nl_st = none ? l : -l * kLog2e;
      lim_st = in && !none ? (p.causal ? a.len - a.n + tokr : a.len - 1) : -1;
      lsrc += adv_t * p.Hq + adv_h;
      tokr += adv_t;
      hdr += adv_h;
      if (hdr >= p.G) {
        hdr -= p.G;
        lsrc += p.Hq - p.G;
        ++tokr;
      }
    }
  };
  auto store_stage = [&](int stage) {
    const int buf = stage & 1;
#pragma unroll
    for (int i = 0; i < PER_T; ++i) {
      const int row = tid / CPR + kPass * i, cc = tid % CPR;
      *reinterpret_cast<uint4_t*>(lds_q[buf] + row * ROWB + ((cc ^ tswz<D>(row)) * 16)) = st[i];
    }
    if (wave * 64 < kStage) {
      reinterpret_cast<float*>(lds_nl[stage & 3])[tid] = nl_st;
      reinterpret_cast<int*>(lds.lim[stage & 3])[tid] = lim_st;
    }
  };

  const float c = p.scale;
  float w[2];
  // A block's rows, as fragments: chunk 2 k + g of row l32 lies at ((2 k) ^ g ^ tswz) = k's bits over
  // the rest of the address.
  const int frag0 = l32 * ROWB + ((g ^ tswz<D>(l32)) * 16);
  auto load_frags = [&](int stage, int half, uint4_t (&a)[KS]) {
    const char* const base = lds_q[stage & 1] + 32 * half * ROWB;
#pragma unroll
    for (int k = 0; k < KS; ++k) a[k] = *reinterpret_cast<const uint4_t*>(base + (frag0 ^ (32 * k)));
  };
  // Scores of a block.
  auto scores = [&](const uint4_t (&a)[KS], float16_t (&sc)[2]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[0][i] = sc[1][i] = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      sc[0] = E::mfma(E::as8(a[k]), E::as8(kf[0][k]), sc[0]);
      sc[1] = E::mfma(E::as8(a[k]), E::as8(kf[1][k]), sc[1]);
    }
  };
  // A block's weights: register 4 j + i of half g is row 8 j + 4 g + i.
  auto add_seen = [&](int stage, int half, const float16_t (&sc)[2], int key) {
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4_t nl = lds_nl[stage & 3][8 * half + 2 * j + g];
      const int4 lim = lds.lim[stage & 3][8 * half + 2 * j + g];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int l = i == 0 ? lim.x : i == 1 ? lim.y : i == 2 ? lim.z : lim.w;
        const float e0 = fast_exp2(__builtin_fmaf(sc[0][4 * j + i], c, nl[i]));
        const float e1 = fast_exp2(__builtin_fmaf(sc[1][4 * j + i], c, nl[i]));
        sum[0] += l >= key ? e0 : 0.f;
        sum[1] += l >= key + 32 ? e1 : 0.f;
      }
    }
    w[0] += sum[0];
    w[1] += sum[1];
  };

  for (;;) {
    load_k(cur);
    const int wkey = cur.t * kWTile + kWKeys * wave;  // the wave's first key
    const bool live = wkey < cur.len;
    const int nb = cur.j1 - cur.j0;
    start_rows(cur);
    load_stage(cur);
    // Half g adds to the sums of keys 32 g + l32.
    const int key = wkey + lane;
    const bool mine = (g ? ok[1] : ok[0]) && key < p.L;
    float* const dst = p.w + cur.row * p.w_sn + cur.kvh * p.w_sh + key;
    const bool whole = nb == cur.blocks;
    float old = 0.f;
    if (whole && mine) old = *dst;
    __syncthreads();  // the last tile's LDS reads are done
    store_stage(0);
    if (nb > 2) load_stage(cur);
    __syncthreads();

    w[0] = w[1] = 0.f;
    float16_t sA[2], sB[2];
    uint4_t fr[KS];
    if (live) {
      load_frags(0, 0, fr);
      scores(fr, sA);
    }
    // Scores of block i + 1 beside the weights of block i; a stage is published while its
    // predecessor's second block goes by.
    // The blocks whose rows are all there and see all of the wave's keys begin from row rfull on; in
    // them nothing is masked.  (A row that drew on none has a weight of 0 there, or NaN where a
    // score is not finite: then the block is summed again with its rows' limits.)
    const int rows = cur.n * p.G;
    const int rfull = p.causal ? max(wkey + kWKeys - 1 - (cur.len - cur.n), 0) * p.G
                               : (wkey + kWKeys <= cur.len ? 0 : rows);
    auto step = [&](int stage, int half, float16_t (&sc)[2], float16_t (&sn)[2]) {
      const int r = cur.r0 + kStage * stage + 32 * half;
      if (r >= rfull && r + 32 <= rows) {
        float4_t nl[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) nl[j] = lds_nl[stage & 3][8 * half + 2 * j + g];
        load_frags(stage + half, half ^ 1, fr);
        __builtin_amdgcn_sched_barrier(0);  // all of the block's reads are asked for first
        scores(fr, sn);
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sum[0] += fast_exp2(__builtin_fmaf(sc[0][4 * j + i], c, nl[j][i]));
            sum[1] += fast_exp2(__builtin_fmaf(sc[1][4 * j + i], c, nl[j][i]));
          }
        }
        __builtin_amdgcn_sched_group_barrier(0x402, kFirst, 0);
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x402, (96 - kFirst) / (2 * KS), 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (__any(sum[0] != sum[0] || sum[1] != sum[1])) {
          add_seen(stage, half, sc, wkey + l32);
        } else {
          w[0] += sum[0];
          w[1] += sum[1];
        }
      } else {
        load_frags(stage + half, half ^ 1, fr);
        add_seen(stage, half, sc, wkey + l32);
        scores(fr, sn);
      }
    };
    int i = 0, stage = 0;
#pragma clang loop unroll(disable)
    for (;;) {
      if (i + 1 == nb) break;
      if (live) step(stage, 0, sA, sB);
      if (++i + 1 == nb) {
        sA[0] = sB[0];
        sA[1] = sB[1];
        break;
      }
      store_stage(stage + 1);
      if (i + 3 < nb) load_stage(cur);
      __syncthreads();
      if (live) step(stage, 1, sB, sA);
      ++i;
      ++stage;
    }
    if (live) add_seen(stage, i & 1, sA, wkey + l32);
    const float w0 = xor32_sum(w[0]), w1 = xor32_sum(w[1]);
    const float sum = g ? w1 : w0;
    if (whole) {
      if (mine) *dst = old + sum;
    } else {
      // ---- a part: its sums to the slot, and the last one of the tile adds them all.
      const int wf = (int)w_div(cur.start, Lw), wl = (int)w_div(cur.start + cur.blocks - 1, Lw);
      auto slot_of = [&](int x) -> float* {
        return p.partials + (2 * (int64_t)x + (x == wf ? 1 : 0)) * kWTile + tid;
      };
      __hip_atomic_store(slot_of(wg), sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      // Every wave's store (device scope) is complete before the count.
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      if (tid == 0) {
        const int prev = atomicAdd(&p.arrive[wf], 1);
        if (prev == wl - wf) atomicExch(&p.arrive[wf], 0);
        lds.last = prev == wl - wf;
      }
      __syncthreads();
      if (lds.last) {
        float all = 0.f;
        for (int x = wf; x <= wl; ++x)
          all += __hip_atomic_load(slot_of(x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (mine) *dst += all;
      }
    }
    advance(cur);
    if (cur.b < 0) return;
  }
}

// Workgroups (of all W, a multiple of 8) for the sequences of few rows, by the lengths of the two
// axes: a step of few rows takes a workgroup's wave about as long as a block of many the workgroup.
template <int D>
__device__ __forceinline__ int share_of(const WeightParams& p, const WTable& tab, int W) {
  const int lane = threadIdx.x & 63;
  float few = 0, many = 0;
  for (int b = lane; b < p.B; b += 64) {
    const WSeq s = seq_of(p, tab, b);
    if (is_few(p, s)) few += (float)few_length(s, few_keys(D));
    if (is_many(p, s)) {
      const WHead h = head_of(p, s);
      many += (float)tile_start(h, h.tiles);
    }
  }
  few = wave_sum(few);
  many = wave_sum(many);
  if (many == 0) return W;
  if (few == 0) return 0;
  const int s = 8 * (int)((float)(W / 8) * (few / (few + many)) + 0.5f);
  return uniform(min(max(s, 8), W - 8));
}

template <int D, bool BF16>
__global__ __launch_bounds__(kWThreads) __attribute__((amdgpu_waves_per_eu(weight_waves<D>(), weight_waves<D>())))
void attention_weights_kernel(WeightParams p) {
  __shared__ __attribute__((aligned(16))) ManyLds<D> lds;
  __shared__ int4 lds_seq[kWTable];
  __shared__ int lds_row[kWTable];
  WTable tab = {nullptr, nullptr};
  if (p.B <= kWTable) {
    for (int b = threadIdx.x; b < p.B; b += kWThreads) {
      const WSeq s = load_wseq(p, b);
      lds_seq[b] = int4{s.q0, s.n, s.ip0, s.len};
      lds_row[b] = s.row;
    }
    __syncthreads();
    tab = WTable{lds_seq, lds_row};
  }
  const int W = gridDim.x, S = share_of<D>(p, tab, W);
  if ((int)blockIdx.x < S) few_weights<D, BF16>(p, tab, blockIdx.x, S);
  else many_weights<D, BF16>(p, tab, lds, blockIdx.x - S, W - S);
}

// Workgroups: as many as are resident, fewer where there are fewer tiles and blocks than that
// (bounded from above by what the host knows).
template <int D>
int64_t weight_wgs(int64_t batch, int64_t total_q, int64_t Hkv, int64_t G, int64_t tokens) {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
      cus <= 0 || cus > 1024)
    cus = 256;  // no device: what an MI355X has
  const int64_t resident = round_up((int64_t)cus * weight_waves<D>(), 8);
  const double tiles = (double)(tokens / kWTile + batch) * Hkv;
  const double blocks = tiles * (double)(total_q * G / 32 + 1 + kWTileCost + kWDiagCost * G);
  const double wgs = ceil(blocks / (kWTileCost + 1)) + 16;  // eight of each kind at least
  return wgs < (double)resident ? round_up((int64_t)wgs, 8) : resident;
}
int64_t weight_wgs(int64_t batch, int64_t total_q, int64_t Hkv, int64_t G, int64_t D,
                   int64_t tokens) {
  return D == 64    ? weight_wgs<64>(batch, total_q, Hkv, G, tokens)
         : D == 256 ? weight_wgs<256>(batch, total_q, Hkv, G, tokens)
                    : weight_wgs<128>(batch, total_q, Hkv, G, tokens);
}

template <int D>
int launch_weights(const WeightParams& p, bool bf16, int64_t wgs, hipStream_t st) {
  KernelTimer timer;
  const dim3 grid((unsigned)wgs), block(kWThreads);
  if (bf16) timer.launch(attention_weights_kernel<D, true>, grid, block, 0, st, p);
  else timer.launch(attention_weights_kernel<D, false>, grid, block, 0, st, p);
  return check_launch("attention_weights_kernel");
}

}  // namespace
}  // namespace akt

using namespace akt;

extern "C" size_t akt_attention_weights_paged_workspace_size(
    int64_t batch, int64_t total_q, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
    int64_t page_size, int64_t total_pages) {
  if (batch <= 0 || total_q <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || page_size <= 0 ||
      total_pages < 0 || num_q_heads % num_kv_heads ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return 0;
  const int64_t wgs = weight_wgs(batch, total_q, num_kv_heads, num_q_heads / num_kv_heads, head_dim,
                                 page_size * total_pages);
  return (size_t)(round_up(AKT_WORKSPACE_ZERO_BYTES, 256) + 2 * wgs * kWTile * 4);
}

extern "C" int akt_attention_weights_paged(
    const void* q, const int32_t* q_indptr, const float* lse, const void* kv_cache,
    const int32_t* kv_page_indptr, const int32_t* kv_page_indices, const int32_t* kv_last_page_len,
    float* weights, const int32_t* rows, int64_t batch, int64_t total_q, int64_t num_q_heads,
    int64_t num_kv_heads, int64_t head_dim, int64_t page_size, int64_t total_pages,
    int64_t num_pool_pages, int64_t num_rows, int64_t row_len, const int64_t q_stride[3],
    const int64_t kv_stride[5], const int64_t weight_stride[2], float softmax_scale, int causal,
    int64_t window, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  AKT_CHECK(dtype == AKT_DTYPE_F16 || dtype == AKT_DTYPE_BF16,
            "dtype must be AKT_DTYPE_F16 or AKT_DTYPE_BF16, got %d", dtype);
  AKT_CHECK(batch >= 0 && total_q >= 0 && total_pages >= 0 && num_pool_pages >= 0 && num_rows >= 0 &&
                row_len >= 0 && window >= 0,
            "sizes must be non-negative");
  AKT_CHECK(num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0,
            "num_q_heads (%lld) must be a positive multiple of num_kv_heads (%lld)",
            (long long)num_q_heads, (long long)num_kv_heads);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return set_error(AKT_ERR_UNSUPPORTED, "attention weights head_dim %lld not supported (64, 128, 256)",
                     (long long)head_dim);
  AKT_CHECK(page_size > 0 && page_size < (1 << 20), "page_size out of range");
  const int64_t G = num_q_heads / num_kv_heads;
  AKT_CHECK(batch < (1ll << 30) && total_q < (1ll << 30) && num_q_heads < (1 << 20) &&
                total_q * G < (1ll << 30),
            "problem too large");
  AKT_CHECK(total_pages < (1ll << 31) && total_pages * page_size < (1ll << 30),
            "the page table spans too many tokens");
  AKT_CHECK(std::isfinite(softmax_scale), "softmax_scale must be finite");
  if (batch == 0 || total_q == 0 || total_pages == 0 || num_rows == 0 || row_len == 0 || window == 0)
    return AKT_OK;
  AKT_CHECK(q && q_indptr && lse && kv_cache && kv_page_indptr && kv_page_indices &&
                kv_last_page_len && weights && q_stride && kv_stride && weight_stride,
            "all pointers are required");
  AKT_CHECK(rows || num_rows >= batch, "weights need a row for every sequence");
  AKT_CHECK(q_stride[2] == 1 && kv_stride[4] == 1, "head_dim stride must be 1");
  AKT_CHECK(rows_aligned16(q, q_stride, 2) && rows_aligned16(kv_cache, kv_stride, 4) &&
                aligned4(lse) && aligned4(weights),
            "tensors must have 16-byte aligned rows");
  // The axis stays below 2^50 (w_div).
  AKT_CHECK((double)(total_pages * page_size / kWTile + batch) * num_kv_heads *
                    (double)(total_q * G / 32 + 1 + kWTileCost + kWDiagCost * G) < 1e15,
            "problem too large");
  const int64_t wgs =
      weight_wgs(batch, total_q, num_kv_heads, G, head_dim, page_size * total_pages);
  const size_t need = akt_attention_weights_paged_workspace_size(
      batch, total_q, num_q_heads, num_kv_heads, head_dim, page_size, total_pages);
  if (!workspace || workspace_bytes < need)
    return set_error(AKT_ERR_WORKSPACE, "attention weights need a workspace of %zu bytes, got %zu",
                     need, workspace ? workspace_bytes : (size_t)0);
  AKT_CHECK(aligned16(workspace), "the workspace must be 16-byte aligned");
  AKT_CHECK(wgs <= (int64_t)(AKT_WORKSPACE_ZERO_BYTES - 256) / 4, "too many workgroups");
  WeightParams p = {};
  p.q = (const half_t*)q;
  p.pool = (const half_t*)kv_cache;
  p.lse = lse;
  p.w = weights;
  p.q_indptr = q_indptr;
  p.indptr = kv_page_indptr;
  p.indices = kv_page_indices;
  p.last_len = kv_last_page_len;
  p.rows = rows;
  p.q_st = q_stride[0];
  p.q_sh = q_stride[1];
  p.sp = kv_stride[0];
  p.sh = kv_stride[2];
  p.ss = kv_stride[3];
  p.w_sn = weight_stride[0];
  p.w_sh = weight_stride[1];
  p.N = (int)(num_rows < (1ll << 31) ? num_rows : (1ll << 31) - 1);
  p.L = row_len;
  p.total_q = (int)total_q;
  p.total_pages = (int)total_pages;
  p.num_pool_pages = (int)(num_pool_pages < (1ll << 31) ? num_pool_pages : (1ll << 31) - 1);
  p.B = (int)batch;
  p.Hq = (int)num_q_heads;
  p.Hkv = (int)num_kv_heads;
  p.G = (int)G;
  p.page_size = (int)page_size;
  auto magic = [](int64_t d) {
    const uint64_t m = (1ull << 32) / (uint64_t)d;
    return (uint32_t)(m < 0xffffffffull ? m : 0xffffffffull);
  };
  p.page_magic = magic(page_size);
  p.g_magic = magic(G);
  p.causal = causal ? 1 : 0;
  p.window = (int)(window < (1ll << 30) ? window : (1ll << 30));
  p.scale = softmax_scale * kLog2e;
  p.arrive = (int*)((char*)workspace + 256);
  p.partials = (float*)((char*)workspace + round_up(AKT_WORKSPACE_ZERO_BYTES, 256));
  hipStream_t st = (hipStream_t)stream;
  const bool bf16 = dtype == AKT_DTYPE_BF16;
  if (head_dim == 64) return launch_weights<64>(p, bf16, wgs, st);
  if (head_dim == 256) return launch_weights<256>(p, bf16, wgs, st);
  return launch_weights<128>(p, bf16, wgs, st);
}
