// Rotary positions (gfx950): of the new tokens of a paged KV cache, written into it, and of
// dense Q and K.
//
// Frequency f of a head's first `rot` dims turns the pair (a, b) of dims (f, f + rot / 2)
// (half layout) or (2 f, 2 f + 1) (interleaved) at position t by the angle t inv_freq[f]:
//   a' = factor (a cos - b sin),  b' = factor (a sin + b cos);
// the dims from rot on are copied.  The transposed map (the gradient of the outputs taken
// to that of the inputs; at factor 1 the inverse) turns by the negative angle.
//
// Angles.  t inv_freq reaches 10^6 radians and more, where 32 bits hold it to no better than
// 0.06; it is formed in 64 bits, in turns, and only its fraction is rounded to 32
// for v_sin_f32 / v_cos_f32, which take turns.  cos and sin are computed once per
// token and frequency a lane holds and used for all its heads.
//
// HBM-bound: every element is read once and written once.  A lane handles units of 16
// elements (eight pairs: two 16-byte chunks, loads and stores whole); with 64 a
// multiple of the D / 16 units of a row, a lane keeps its eight frequencies from row to row.
// Rows whose rotated part does not fill units (rot % 16 != 0, or other head dims) take
// the generic kernels: a lane handles 8 elements of a row and loads each one's partner.
//
// Measured: dense Q and K of 8 x 1024 tokens, 64 + 16 heads, D = 64: 36 to 37 us (168 MB, 4.6 TB/s,
// where a large copy reaches 5.1); 4 appended prompts of 1000 to 3001 tokens, 32 + 8 heads,
// D = 128: 51.6 us (219 MB, 4.2 TB/s); 64 single tokens: 6.5 us, launch and look-ups.  Generic:
// dense 8 x 1024 tokens, 32 + 8 heads, D = 192: 92 us (252 MB, 2.7 TB/s; D = 128, whole units,
// 168 MB in 30 us); 4 x 2000 appended tokens, D = 80: 67 us (123 MB, 1.8 TB/s).
#include <math.h>

#include <cmath>

#include "akt_common.hpp"
#include "akt_host.hpp"

namespace akt {
namespace {

constexpr int kRThreads = 256;
constexpr int kRWaves = kRThreads / 64;
constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)

template <bool BF16>
__device__ __forceinline__ float r_lo(uint32_t u) {
  if constexpr (BF16) return __uint_as_float(u << 16);
  return (float)as_half2(u)[0];
}
template <bool BF16>
__device__ __forceinline__ float r_hi(uint32_t u) {
  if constexpr (BF16) return __uint_as_float(u & 0xffff0000u);
  return (float)as_half2(u)[1];
}
template <bool BF16>
__device__ __forceinline__ uint32_t r_pack(float lo, float hi) {
  if constexpr (BF16) return pack_bf16x2(lo, hi);
  return pack_half2(lo, hi);
}

// cos and sin, times factor, of position t at a frequency in turns per position.
__device__ __forceinline__ void turn_of(double turns, double t, float factor, float& cs, float& sn) {
  const double a = t * turns;
  const float f = (float)(a - __builtin_rint(a));  // [-1/2, 1/2]
  cs = __builtin_amdgcn_cosf(f) * factor;
  sn = __builtin_amdgcn_sinf(f) * factor;
}

// Eight pairs.  Half layout: x holds the eight a, y the eight b; interleaved: x holds pairs
// 0..3 and y pairs 4..7.
template <bool BF16, bool INTER>
__device__ __forceinline__ void rotate8(uint4_t& x, uint4_t& y, const float (&cs)[8],
                                        const float (&sn)[8]) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (INTER) {
      const float a0 = r_lo<BF16>(x[w]), b0 = r_hi<BF16>(x[w]);
      const float a1 = r_lo<BF16>(y[w]), b1 = r_hi<BF16>(y[w]);
      x[w] = r_pack<BF16>(a0 * cs[w] - b0 * sn[w], a0 * sn[w] + b0 * cs[w]);
      y[w] = r_pack<BF16>(a1 * cs[4 + w] - b1 * sn[4 + w], a1 * sn[4 + w] + b1 * cs[4 + w]);
    } else {
      const float a0 = r_lo<BF16>(x[w]), a1 = r_hi<BF16>(x[w]);
      const float b0 = r_lo<BF16>(y[w]), b1 = r_hi<BF16>(y[w]);
      const int f = 2 * w;
      x[w] = r_pack<BF16>(a0 * cs[f] - b0 * sn[f], a1 * cs[f + 1] - b1 * sn[f + 1]);
      y[w] = r_pack<BF16>(a0 * sn[f] + b0 * cs[f], a1 * sn[f + 1] + b1 * cs[f + 1]);
    }
  }
}

// The generic form: 8 elements from dim 8 col of a row.  Element e is dim d = 8 col + e with
// partner pd[e] and pair (cos, sign sin); dims from rot on have pd = -1.
struct Gen8 {
  int pd[8];
  float cs[8], sn[8];
};
__device__ __forceinline__ void gen_plan(Gen8& p, int col, int rot, bool inter,
                                         const double* inv_freq, double t, float factor) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int d = 8 * col + e, half = rot / 2;
    p.pd[e] = -1;
    p.cs[e] = p.sn[e] = 0.f;
    if (d < rot) {
      const bool second = inter ? (d & 1) : d >= half;
      const int f = inter ? d / 2 : (second ? d - half : d);
      p.pd[e] = inter ? (d ^ 1) : (second ? d - half : d + half);
      turn_of(inv_freq[f] * kTurn, t, factor, p.cs[e], p.sn[e]);
      if (!second) p.sn[e] = -p.sn[e];
    }
  }
}
template <bool BF16>
__device__ __forceinline__ uint4_t gen_apply(const Gen8& p, const half_t* row, int col) {
  const uint16_t* r16 = reinterpret_cast<const uint16_t*>(row);
  uint4_t x = ld16(row + 8 * col);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    float v[2];
    bool keep[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int e = 2 * w + k;
      keep[k] = p.pd[e] < 0;
      const uint32_t o = keep[k] ? 0u : (uint32_t)r16[p.pd[e]];
      const float own = k ? r_hi<BF16>(x[w]) : r_lo<BF16>(x[w]);
      v[k] = own * p.cs[e] + r_lo<BF16>(o) * p.sn[e];
    }
    const uint32_t r = r_pack<BF16>(v[0], v[1]);
    x[w] = (keep[0] ? x[w] & 0xffffu : r & 0xffffu) |
           (keep[1] ? x[w] & 0xffff0000u : r & 0xffff0000u);
  }
  return x;
}

// ---------------------------------------------------------------------------
// Dense Q [B, Hq, S, D] and K [B, Hkv, S, D].
// ---------------------------------------------------------------------------
struct DenseParams {
  const half_t* x[2];  // Q, K
  half_t* o[2];        // contiguous
  int64_t sb[2], sh[2], ss[2];
  int H[2];
  const double* inv_freq;
  const void* pos;  // null: 0 .. S - 1
  int64_t pos_sb, pos_ss;
  int pos_bits;
  int B, S, D, rot;
  int inter, transpose;
  float factor;
  int hc;  // heads of a block
  int tpb;  // tokens of a wave
};

__device__ __forceinline__ double position_of(const DenseParams& p, int b, int s) {
  double t = (double)s;
  if (p.pos) {
    const int64_t i = b * p.pos_sb + s * p.pos_ss;
    t = p.pos_bits == 64 ? (double)((const int64_t*)p.pos)[i] : (double)((const int32_t*)p.pos)[i];
  }
  return p.transpose ? -t : t;
}

// A wave takes 64 / (D / 16) tokens and hc heads: one load serves consecutive rows.
template <bool BF16, bool INTER>
__global__ __launch_bounds__(kRThreads) void rotary_dense_kernel(DenseParams p) {
  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  const int upr = p.D / 16;
  const int64_t tok = ((int64_t)blockIdx.x * kRWaves + wave) * p.tpb + lane / upr;
  if (tok >= (int64_t)p.B * p.S) return;
  const int col = lane % upr;
  const int b = (int)(tok / p.S), s = (int)(tok - (int64_t)b * p.S);
  const bool turned = 16 * col < p.rot;
  float cs[8], sn[8];
  // Chunks of the unit, in elements; past the rotated part they follow one another.
  const int d0 = !INTER && turned ? 8 * col : 16 * col;
  const int d1 = !INTER && turned ? p.rot / 2 + 8 * col : 16 * col + 8;
  if (turned) {
    const double t = position_of(p, b, s);
#pragma unroll
    for (int f = 0; f < 8; ++f)
      turn_of(p.inv_freq[8 * col + f] * kTurn, t, p.factor, cs[f], sn[f]);
  }
  const int heads = p.H[0] + p.H[1];
  const int h1 = min(heads, (int)(blockIdx.y + 1) * p.hc);
#pragma unroll 4
  for (int h = blockIdx.y * p.hc; h < h1; ++h) {
    const int w = h >= p.H[0];
    const int hh = w ? h - p.H[0] : h;
    const half_t* src = p.x[w] + b * p.sb[w] + hh * p.sh[w] + s * p.ss[w];
    half_t* dst = p.o[w] + (((int64_t)b * p.H[w] + hh) * p.S + s) * p.D;
    uint4_t x = ld16(src + d0), y = ld16(src + d1);
    if (turned) rotate8<BF16, INTER>(x, y, cs, sn);
    st16(dst + d0, x);
    st16(dst + d1, y);
  }
}

// One (token, 8 elements) to a thread, over hc heads.
template <bool BF16>
__global__ __launch_bounds__(kRThreads) void rotary_dense_gen_kernel(DenseParams p) {
  const int cpr = p.D / 8;
  const int64_t i = (int64_t)blockIdx.x * kRThreads + threadIdx.x;
  if (i >= (int64_t)p.B * p.S * cpr) return;
  const int64_t tok = i / cpr;
  const int col = (int)(i - tok * cpr);
  const int b = (int)(tok / p.S), s = (int)(tok - (int64_t)b * p.S);
  Gen8 g;
  gen_plan(g, col, p.rot, p.inter, p.inv_freq, position_of(p, b, s), p.factor);
  const int heads = p.H[0] + p.H[1];
  const int h1 = min(heads, (int)(blockIdx.y + 1) * p.hc);
  for (int h = blockIdx.y * p.hc; h < h1; ++h) {
    const int w = h >= p.H[0];
    const int hh = w ? h - p.H[0] : h;
    st16(p.o[w] + (((int64_t)b * p.H[w] + hh) * p.S + s) * p.D + 8 * col,
         gen_apply<BF16>(g, p.x[w] + b * p.sb[w] + hh * p.sh[w] + s * p.ss[w], col));
  }
}

// ---------------------------------------------------------------------------
// New tokens of a paged cache: q rotated into a new tensor, k rotated and v copied into the
// pool.  Positions, pages and slots as in paged_append_kernel.
// ---------------------------------------------------------------------------
struct AppendRotaryParams {
  const half_t* q;
  const half_t* k;
  const half_t* v;
  half_t* qo;  // contiguous [total, Hq, D]
  half_t* pool;
  const int32_t* append_indptr;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last_len;
  const double* inv_freq;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  int64_t sp, skv, sh, ss;
  int total;
  int B, Hq, Hkv, D, rot, inter;
  float factor;
  int page_size, num_pool_pages, total_pages;
};

struct Place {
  int pos;         // -1: the token belongs to no sequence
  int page, slot;  // page -1: not stored
};
// Sequence, position, page and slot of token tok, wave-uniform.  Page table entries outside
// their range are taken clamped.
__device__ __forceinline__ Place place_of(const AppendRotaryParams& p, int tok, int lane) {
  int cnt = 0;  // sequences that start at or before tok
  for (int jb = 0; jb < p.B; jb += 64) {
    const int j = jb + lane;
    const int aj = j < p.B ? p.append_indptr[j] : INT32_MAX;
    cnt += __popcll(__ballot(aj <= tok));
  }
  Place r = {-1, -1, 0};
  const int b = uniform(cnt) - 1;
  if (b < 0) return r;
  const int a0 = p.append_indptr[b], a1 = p.append_indptr[b + 1];
  const int ip0 = min(max(p.indptr[b], 0), p.total_pages);
  const int np = min(max(p.indptr[b + 1], ip0), p.total_pages) - ip0;
  const int last = min(max(p.last_len[b], 0), p.page_size);
  const int len = (np - 1) * p.page_size + last;  // total_pages * page_size < 2^30
  const int64_t pos = (int64_t)len - ((int64_t)a1 - tok);
  if (tok < a0 || tok >= a1 || np <= 0 || pos < 0) return r;
  r.pos = (int)pos;
  const int lp = (int)((uint32_t)r.pos / (uint32_t)p.page_size);
  r.slot = r.pos - lp * p.page_size;
  const int pg = p.indices[ip0 + lp];
  if ((uint32_t)pg < (uint32_t)p.num_pool_pages) r.page = pg;
  return r;
}

// Rows of a token: q heads, then k, then v.
__device__ __forceinline__ const half_t* row_src(const AppendRotaryParams& p, int tok, int h) {
  const int hk = h - p.Hq, hv = hk - p.Hkv;
  if (hk < 0) return p.q + tok * p.q_st + h * p.q_sh;
  return hv < 0 ? p.k + tok * p.k_st + hk * p.k_sh : p.v + tok * p.v_st + hv * p.v_sh;
}
// Destination of row h; none for a k or v row of a token without a page.
__device__ __forceinline__ half_t* row_dst(const AppendRotaryParams& p, int tok, const Place& pl,
                                           int h) {
  const int hk = h - p.Hq, hv = hk - p.Hkv;
  if (hk < 0) return p.qo + ((int64_t)tok * p.Hq + h) * p.D;
  if (pl.page < 0) return nullptr;
  half_t* slot = p.pool + pl.page * p.sp + pl.slot * p.ss;
  return hv < 0 ? slot + hk * p.sh : slot + p.skv + hv * p.sh;
}

// One wave to a token.  The rows are loaded before the token's place is known: its look-up,
// three dependent loads, runs meanwhile.
constexpr int kRBatch = 3;  // steps in flight

template <bool BF16, bool INTER>
__global__ __launch_bounds__(kRThreads) void append_rotary_kernel(AppendRotaryParams p) {
  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  const int tok = (int)blockIdx.x * kRWaves + wave;
  if (tok >= p.total) return;
  const int upr = p.D / 16;
  const int col = lane % upr, h_lane = lane / upr;
  const bool turned = 16 * col < p.rot;
  const int heads = p.Hq + 2 * p.Hkv, rotated = p.Hq + p.Hkv;
  const int hpw = 64 / upr;  // rows to a step
  // Chunks of a unit, in elements (rotated rows of the half layout, others).
  const int d0 = !INTER && turned ? 8 * col : 16 * col;
  const int d1 = !INTER && turned ? p.rot / 2 + 8 * col : 16 * col + 8;
  uint4_t x[kRBatch], y[kRBatch];
  auto load = [&](int h0) {
#pragma unroll
    for (int k = 0; k < kRBatch; ++k) {
      const int h = h0 + k * hpw + h_lane;
      if (h < heads) {
        const half_t* src = row_src(p, tok, h);
        const bool r = h < rotated;
        x[k] = ld16(src + (r ? d0 : 16 * col));
        y[k] = ld16(src + (r ? d1 : 16 * col + 8));
      }
    }
  };
  load(0);
  const Place pl = place_of(p, tok, lane);
  if (pl.pos < 0) return;
  float cs[8], sn[8];
  if (turned) {
#pragma unroll
    for (int f = 0; f < 8; ++f)
      turn_of(p.inv_freq[8 * col + f] * kTurn, (double)pl.pos, p.factor, cs[f], sn[f]);
  }
  for (int h0 = 0;;) {
#pragma unroll
    for (int k = 0; k < kRBatch; ++k) {
      const int h = h0 + k * hpw + h_lane;
      if (h < heads) {
        const bool r = h < rotated;
        if (turned && r) rotate8<BF16, INTER>(x[k], y[k], cs, sn);
        if (half_t* dst = row_dst(p, tok, pl, h)) {
          st16(dst + (r ? d0 : 16 * col), x[k]);
          st16(dst + (r ? d1 : 16 * col + 8), y[k]);
        }
      }
    }
    h0 += kRBatch * hpw;
    if (h0 >= heads) break;  // wave-uniform
    load(h0);
  }
}

template <bool BF16>
__global__ __launch_bounds__(kRThreads) void append_rotary_gen_kernel(AppendRotaryParams p) {
  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  const int tok = (int)blockIdx.x * kRWaves + wave;
  if (tok >= p.total) return;
  const Place pl = place_of(p, tok, lane);
  if (pl.pos < 0) return;
  const int cpr = p.D / 8;
  const int heads = p.Hq + 2 * p.Hkv, rotated = p.Hq + p.Hkv;
  // Column by column (64 at a time where a row has more): a lane keeps its plan.
  const int cw = min(cpr, 64), hpw = 64 / cw;
  if (lane >= cw * hpw) return;
  for (int col = lane % cw; col < cpr; col += cw) {
    Gen8 g;
    gen_plan(g, col, p.rot, p.inter, p.inv_freq, (double)pl.pos, p.factor);
    for (int h = lane / cw; h < heads; h += hpw) {
      const half_t* src = row_src(p, tok, h);
      const uint4_t x = h < rotated ? gen_apply<BF16>(g, src, col) : ld16(src + 8 * col);
      if (half_t* dst = row_dst(p, tok, pl, h)) st16(dst + 8 * col, x);
    }
  }
}

// Whether rows split into units whose columns a lane keeps.
bool whole_units(int64_t D, int64_t rot) {
  return rot % 16 == 0 && D % 16 == 0 && D <= 1024 && 64 % (D / 16) == 0;
}

int check_rotation(int64_t head_dim, int64_t rotary_dim, float factor, int dtype) {
  AKT_CHECK(dtype == AKT_DTYPE_F16 || dtype == AKT_DTYPE_BF16,
            "dtype must be AKT_DTYPE_F16 or AKT_DTYPE_BF16, got %d", dtype);
  AKT_CHECK(head_dim > 0 && head_dim % 8 == 0 && head_dim <= 1024,
            "head_dim must be a positive multiple of 8 up to 1024");
  AKT_CHECK(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim,
            "rotary_dim (%lld) must be even and in (0, head_dim]", (long long)rotary_dim);
  AKT_CHECK(std::isfinite(factor), "factor must be finite");
  return AKT_OK;
}

}  // namespace
}  // namespace akt

using namespace akt;

extern "C" int akt_rotary_fwd(const void* q, const void* k, void* q_out, void* k_out,
                              const double* inv_freq, const void* positions, int position_bits,
                              int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
                              int64_t seq_len, int64_t head_dim, int64_t rotary_dim,
                              const int64_t q_stride[4], const int64_t k_stride[4],
                              const int64_t position_stride[2], int interleaved, int transpose,
                              float factor, int dtype, void* stream) {
  clear_error();
  if (int rc = check_rotation(head_dim, rotary_dim, factor, dtype)) return rc;
  AKT_CHECK(batch >= 0 && seq_len >= 0 && num_q_heads > 0 && num_kv_heads >= 0,
            "sizes must be non-negative");
  AKT_CHECK(batch < (1ll << 31) && seq_len < (1ll << 31) && num_q_heads < (1 << 20) &&
                num_kv_heads < (1 << 20),
            "problem too large");
  AKT_CHECK(!positions || position_bits == 32 || position_bits == 64,
            "position_bits must be 32 or 64");
  if (batch == 0 || seq_len == 0) return AKT_OK;
  AKT_CHECK(q && q_out && inv_freq && q_stride && (num_kv_heads == 0 || (k && k_out && k_stride)) &&
                (!positions || position_stride),
            "all pointers are required");
  AKT_CHECK(q_stride[3] == 1 && (num_kv_heads == 0 || k_stride[3] == 1),
            "head_dim stride must be 1");
  AKT_CHECK(rows_aligned16(q, q_stride, 3) && aligned16(q_out) &&
                (num_kv_heads == 0 || (rows_aligned16(k, k_stride, 3) && aligned16(k_out))),
            "tensors must have 16-byte aligned rows");
  DenseParams p = {};
  p.x[0] = (const half_t*)q;
  p.o[0] = (half_t*)q_out;
  p.sb[0] = q_stride[0]; p.sh[0] = q_stride[1]; p.ss[0] = q_stride[2];
  p.H[0] = (int)num_q_heads;
  if (num_kv_heads) {
    p.x[1] = (const half_t*)k;
    p.o[1] = (half_t*)k_out;
    p.sb[1] = k_stride[0]; p.sh[1] = k_stride[1]; p.ss[1] = k_stride[2];
    p.H[1] = (int)num_kv_heads;
  }
  p.inv_freq = inv_freq;
  p.pos = positions;
  p.pos_bits = position_bits;
  if (positions) {
    p.pos_sb = position_stride[0];
    p.pos_ss = position_stride[1];
  }
  p.B = (int)batch;
  p.S = (int)seq_len;
  p.D = (int)head_dim;
  p.rot = (int)rotary_dim;
  p.inter = interleaved ? 1 : 0;
  p.transpose = transpose ? 1 : 0;
  p.factor = factor;
  const bool units = whole_units(head_dim, rotary_dim);
  const int64_t tokens = batch * seq_len;
  p.tpb = units ? (int)(64 / (head_dim / 16)) : 0;
  const int64_t blocks = units ? ceil_div(tokens, (int64_t)p.tpb * kRWaves)
                               : ceil_div(tokens * (head_dim / 8), kRThreads);
  AKT_CHECK(grid_fits(blocks, kRThreads), "problem too large");
  // Heads of a block: as many as leave about four workgroups to a CU, so that cos and sin
  // serve many heads in a large launch and a small one fills the chip.
  const int64_t heads = num_q_heads + num_kv_heads;
  int64_t hc = ceil_div(heads * blocks, 1024);
  hc = hc < 1 ? 1 : (hc > heads ? heads : hc);
  if (ceil_div(heads, hc) > 65535) hc = ceil_div(heads, 65535);
  p.hc = (int)hc;
  const dim3 grid((unsigned)blocks, (unsigned)ceil_div(heads, hc));
  hipStream_t st = (hipStream_t)stream;
  KernelTimer timer;
  const bool bf16 = dtype == AKT_DTYPE_BF16;
  if (!units) {
    if (bf16) timer.launch(rotary_dense_gen_kernel<true>, grid, dim3(kRThreads), 0, st, p);
    else timer.launch(rotary_dense_gen_kernel<false>, grid, dim3(kRThreads), 0, st, p);
  } else if (bf16) {
    if (p.inter) timer.launch(rotary_dense_kernel<true, true>, grid, dim3(kRThreads), 0, st, p);
    else timer.launch(rotary_dense_kernel<true, false>, grid, dim3(kRThreads), 0, st, p);
  } else {
    if (p.inter) timer.launch(rotary_dense_kernel<false, true>, grid, dim3(kRThreads), 0, st, p);
    else timer.launch(rotary_dense_kernel<false, false>, grid, dim3(kRThreads), 0, st, p);
  }
  return check_launch("rotary_dense_kernel");
}

extern "C" int akt_paged_kv_append_rotary(
    const void* q, const void* k_new, const void* v_new, void* q_out, const int32_t* append_indptr,
    void* kv_cache, const int32_t* kv_page_indptr, const int32_t* kv_page_indices,
    const int32_t* kv_last_page_len, const double* inv_freq, int64_t batch, int64_t total_new,
    int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t rotary_dim,
    int64_t page_size, int64_t total_pages, int64_t num_pool_pages, const int64_t q_stride[3],
    const int64_t k_new_stride[3], const int64_t v_new_stride[3], const int64_t kv_stride[5],
    int interleaved, float factor, int dtype, void* stream) {
  clear_error();
  if (int rc = check_rotation(head_dim, rotary_dim, factor, dtype)) return rc;
  AKT_CHECK(batch >= 0 && total_new >= 0 && total_pages >= 0 && num_pool_pages >= 0 &&
                num_q_heads > 0 && num_kv_heads > 0,
            "sizes must be non-negative");
  AKT_CHECK(batch < (1ll << 30) && total_new < (1ll << 30) && total_pages < (1ll << 31) &&
                num_q_heads < (1 << 20) && num_kv_heads < (1 << 20),
            "problem too large");
  AKT_CHECK(page_size > 0 && page_size < (1 << 20), "page_size out of range");
  AKT_CHECK(total_pages * page_size < (1ll << 30), "the page table spans too many tokens");
  if (batch == 0 || total_new == 0) return AKT_OK;
  AKT_CHECK(q && k_new && v_new && q_out && append_indptr && kv_cache && kv_page_indptr &&
                (kv_page_indices || total_pages == 0) && kv_last_page_len && inv_freq && q_stride &&
                k_new_stride && v_new_stride && kv_stride,
            "all pointers are required");
  AKT_CHECK(q_stride[2] == 1 && k_new_stride[2] == 1 && v_new_stride[2] == 1 && kv_stride[4] == 1,
            "head_dim stride must be 1");
  AKT_CHECK(rows_aligned16(q, q_stride, 2) && rows_aligned16(k_new, k_new_stride, 2) &&
                rows_aligned16(v_new, v_new_stride, 2) && rows_aligned16(kv_cache, kv_stride, 4) &&
                aligned16(q_out),
            "tensors must have 16-byte aligned rows");
  AKT_CHECK(grid_fits(ceil_div(total_new, kRWaves), kRThreads), "too many tokens");
  AppendRotaryParams p = {};
  p.q = (const half_t*)q;
  p.k = (const half_t*)k_new;
  p.v = (const half_t*)v_new;
  p.qo = (half_t*)q_out;
  p.pool = (half_t*)kv_cache;
  p.append_indptr = append_indptr;
  p.indptr = kv_page_indptr;
  p.indices = kv_page_indices;
  p.last_len = kv_last_page_len;
  p.inv_freq = inv_freq;
  p.q_st = q_stride[0]; p.q_sh = q_stride[1];
  p.k_st = k_new_stride[0]; p.k_sh = k_new_stride[1];
  p.v_st = v_new_stride[0]; p.v_sh = v_new_stride[1];
  p.sp = kv_stride[0];
  p.skv = kv_stride[1];
  p.sh = kv_stride[2];
  p.ss = kv_stride[3];
  p.total = (int)total_new;
  p.B = (int)batch;
  p.Hq = (int)num_q_heads;
  p.Hkv = (int)num_kv_heads;
  p.D = (int)head_dim;
  p.rot = (int)rotary_dim;
  p.inter = interleaved ? 1 : 0;
  p.factor = factor;
  p.page_size = (int)page_size;
  p.num_pool_pages = (int)(num_pool_pages < (1ll << 31) ? num_pool_pages : (1ll << 31) - 1);
  p.total_pages = (int)total_pages;
  const dim3 grid((unsigned)ceil_div(total_new, kRWaves)), blk(kRThreads);
  hipStream_t st = (hipStream_t)stream;
  KernelTimer timer;
  const bool bf16 = dtype == AKT_DTYPE_BF16;
  if (!whole_units(head_dim, rotary_dim)) {
    if (bf16) timer.launch(append_rotary_gen_kernel<true>, grid, blk, 0, st, p);
    else timer.launch(append_rotary_gen_kernel<false>, grid, blk, 0, st, p);
  } else if (bf16) {
    if (p.inter) timer.launch(append_rotary_kernel<true, true>, grid, blk, 0, st, p);
    else timer.launch(append_rotary_kernel<true, false>, grid, blk, 0, st, p);
  } else {
    if (p.inter) timer.launch(append_rotary_kernel<false, true>, grid, blk, 0, st, p);
    else timer.launch(append_rotary_kernel<false, false>, grid, blk, 0, st, p);
  }
  return check_launch("append_rotary_kernel");
}
