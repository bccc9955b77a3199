// Attention that cached tokens draw, summed over calls (gfx950):
//   w[row_b, h, j] += sum over the tokens i of sequence b that see key j, and the query heads of kv
//                     head h, of exp(scale q_i . k_j - lse_i).
// q, lse and the page table are those of an attention call (paged decode, chunk or shared
// prefix); sequence b's token i sits at position len_b - n_b + i, as there.
//
// A workgroup owns 256 keys of one (sequence, kv head), wave w keys 64 w .. 64 w + 63 of them, and
// reads them into registers once; the rows (token, query head of the group; token major) go by in
// blocks of 32, staged in LDS once for the four waves.  S = Q K^T is computed with rows along the
// registers and keys along the lanes (two v_mfma_f32_32x32x16 columns), so a lane sums its
// key's weights in registers and every sum has one owner and one order: no atomics, and results do
// not depend on the run.  A block's 16 terms are summed before they join the total.
//
// What bounds it: HBM (K once) for few rows; for many the three VALU instructions to a score (fma,
// exp2, add) beside 1/1024 of an MFMA k-step each.
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
  int64_t N, L;
  int total_q, total_pages, num_pool_pages;
  int B, Hq, Hkv, G;
  int page_size;
  uint32_t page_magic;  // min(2^32 - 1, floor(2^32 / page_size))
  uint32_t g_magic;     // the same for G
  int causal;
  int window;  // only the last so many of a sequence's tokens count
  float scale;  // softmax_scale * log2(e)
};

// n / d for 0 <= n < 2^31, given magic = min(2^32 - 1, floor(2^32 / d)).
__device__ __forceinline__ int div_magic(int n, int d, uint32_t magic) {
  const int q = (int)__umulhi((uint32_t)n, magic);
  return n - q * d >= d ? q + 1 : q;
}

struct WSeq {
  int q0, n, first;  // first row of q that counts, rows that count, position of the first
  int ip0, len;
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
  s.first = s.len - s.n;
  return s;
}

template <int D, bool BF16>
__global__ __launch_bounds__(kWThreads) __attribute__((amdgpu_waves_per_eu(2)))
void attention_weights_kernel(WeightParams p) {
  typedef Elt<BF16> E;
  typedef typename E::v8 v8;
  constexpr int KS = D / 16;
  constexpr int CPR = D / 8;
  constexpr int ROWB = D * 2;
  constexpr int PER_T = 32 * CPR / kWThreads;  // chunks of a block of rows to a thread
  __shared__ __attribute__((aligned(16))) char lds_q[2][32 * ROWB];
  __shared__ float4_t lds_nl[2][8];  // -lse log2(e) of each row
  __shared__ int lds_lim[2][32];     // last key that the row sees, -1: none
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int l32 = lane & 31, g = lane >> 5;

  // ---- this workgroup's tile: sequence by sequence, kv head by kv head.
  int b = 0, item = 0;
  {
    const int x = blockIdx.x;
    int before = 0;
    for (int jb = 0;; jb += 64) {
      if (jb >= p.B) return;
      int tiles = 0;
      if (jb + lane < p.B) {
        const WSeq s = load_wseq(p, jb + lane);
        if (s.n > 0) tiles = (s.len + kWTile - 1) / kWTile * p.Hkv;
      }
      int inc = tiles;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int u = __shfl_up(inc, d, 64);
        if (lane >= d) inc += u;
      }
      const uint64_t m = __ballot(before + inc > x);
      if (m) {
        const int l = __builtin_ctzll(m);
        b = uniform(jb + l);
        item = uniform(x - before - __shfl(inc - tiles, l, 64));
        break;
      }
      before += uniform(__shfl(inc, 63, 64));
    }
  }
  const WSeq sq = load_wseq(p, b);
  const int q0 = uniform(sq.q0), n = uniform(sq.n), first = uniform(sq.first);
  const int ip0 = uniform(sq.ip0), len = uniform(sq.len);
  const int64_t wrow = p.rows ? (int64_t)p.rows[b] : b;
  if (wrow < 0 || wrow >= p.N) return;
  const int tiles = (len + kWTile - 1) / kWTile;
  // (A malformed table may count more tiles than the scan's sums hold.)
  if (tiles <= 0 || item < 0 || item >= tiles * p.Hkv) return;
  const int kvh = item / tiles, key0 = (item - kvh * tiles) * kWTile;
  const int rows = n * p.G;

  // ---- K: lane (l32, g) holds chunks 2 k + g of keys l32 and 32 + l32 of the wave's.
  const int wkey = key0 + kWKeys * wave;
  v8 kf[2][KS];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int key = wkey + 32 * c + l32;
    const int kk = min(key, len - 1);
    const int lp = div_magic(kk, p.page_size, p.page_magic);
    const int id = p.indices[ip0 + lp];
    const bool ok = key < len && (uint32_t)id < (uint32_t)p.num_pool_pages;
    const half_t* src = p.pool + id * p.sp + kvh * p.sh + (int64_t)(kk - lp * p.page_size) * p.ss + 8 * g;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      uint4_t v = {0, 0, 0, 0};
      if (ok) v = ld16(src + 16 * k);
      kf[c][k] = E::as8(v);
    }
  }

  // ---- blocks of rows, from the first that holds a row which sees the tile's first key.
  uint4_t st[PER_T];
  float nl_st = 0.f;
  int lim_st = -1;
  auto load_block = [&](int r0) {
#pragma unroll
    for (int i = 0; i < PER_T; ++i) {
      const int ch = tid + i * kWThreads;
      const int row = r0 + ch / CPR;
      st[i] = uint4_t{0, 0, 0, 0};
      if (row < rows) {
        const int tok = div_magic(row, p.G, p.g_magic);
        st[i] = ld16(p.q + (int64_t)(q0 + tok) * p.q_st +
                     (int64_t)(kvh * p.G + row - tok * p.G) * p.q_sh + ch % CPR * 8);
      }
    }
    if (tid < 32) {
      const int row = r0 + tid;
      lim_st = -1;
      nl_st = 0.f;
      if (row < rows) {
        const int tok = div_magic(row, p.G, p.g_magic);
        const float l = p.lse[(int64_t)(q0 + tok) * p.Hq + kvh * p.G + row - tok * p.G];
        nl_st = -l * kLog2e;
        // A row that saw no key (lse -inf) drew on none.
        if (l != -__builtin_inff()) lim_st = p.causal ? first + tok : len - 1;
      }
    }
  };
  auto store_block = [&](int buf) {
#pragma unroll
    for (int i = 0; i < PER_T; ++i) {
      const int ch = tid + i * kWThreads;
      const int row = ch / CPR, cc = ch % CPR;
      *reinterpret_cast<uint4_t*>(lds_q[buf] + row * ROWB + ((cc ^ tswz<D>(row)) * 16)) = st[i];
    }
    if (tid < 32) {
      reinterpret_cast<float*>(lds_nl[buf])[tid] = nl_st;
      lds_lim[buf][tid] = lim_st;
    }
  };
  float w[2] = {0.f, 0.f};
  int r0 = 0;
  if (p.causal && key0 > first) r0 = (int)((int64_t)(key0 - first) * p.G / 32 * 32);
  load_block(r0);
  store_block(0);
  __syncthreads();
  const float c = p.scale;
#pragma clang loop unroll(disable)
  for (int buf = 0; r0 < rows; r0 += 32, buf ^= 1) {
    const bool more = r0 + 32 < rows;
    if (more) load_block(r0 + 32);
    if (wkey < len) {
      float16_t s[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) s[0][i] = s[1][i] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const v8 a = E::as8(*reinterpret_cast<const uint4_t*>(
            lds_q[buf] + l32 * ROWB + (((2 * k + g) ^ tswz<D>(l32)) * 16)));
        s[0] = E::mfma(a, kf[0][k], s[0]);
        s[1] = E::mfma(a, kf[1][k], s[1]);
      }
      // Register 4 j + i of half g is row 8 j + 4 g + i.
      if (__ballot(lds_lim[buf][l32] >= wkey + kWKeys - 1) == ~0ull) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4_t nl = lds_nl[buf][2 * j + g];
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += fast_exp2(__builtin_fmaf(s[t][4 * j + i], c, nl[i]));
          }
          w[t] += sum;
        }
      } else {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int key = wkey + 32 * t + l32;
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4_t nl = lds_nl[buf][2 * j + g];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float e = fast_exp2(__builtin_fmaf(s[t][4 * j + i], c, nl[i]));
              sum += lds_lim[buf][8 * j + 4 * g + i] >= key ? e : 0.f;
            }
          }
          w[t] += sum;
        }
      }
    }
    if (more) store_block(buf ^ 1);
    __syncthreads();
  }

  // ---- half g writes keys 32 g + l32.
  const float w0 = xor32_sum(w[0]), w1 = xor32_sum(w[1]);
  const int key = wkey + lane;
  const int id = p.indices[ip0 + div_magic(min(key, len - 1), p.page_size, p.page_magic)];
  if (key < len && key < p.L && (uint32_t)id < (uint32_t)p.num_pool_pages) {
    float* dst = p.w + wrow * p.w_sn + kvh * p.w_sh + key;
    *dst += g ? w1 : w0;
  }
}

template <int D>
int launch_weights(const WeightParams& p, bool bf16, int64_t blocks, hipStream_t st) {
  KernelTimer timer;
  const dim3 grid((unsigned)blocks), block(kWThreads);
  if (bf16) timer.launch(attention_weights_kernel<D, true>, grid, block, 0, st, p);
  else timer.launch(attention_weights_kernel<D, false>, grid, block, 0, st, p);
  return check_launch("attention_weights_kernel");
}

}  // namespace
}  // namespace akt

using namespace akt;

extern "C" int akt_attention_weights_paged(
    const void* q, const int32_t* q_indptr, const float* lse, const void* kv_cache,
    const int32_t* kv_page_indptr, const int32_t* kv_page_indices, const int32_t* kv_last_page_len,
    float* weights, const int32_t* rows, int64_t batch, int64_t total_q, int64_t num_q_heads,
    int64_t num_kv_heads, int64_t head_dim, int64_t page_size, int64_t total_pages,
    int64_t num_pool_pages, int64_t num_rows, int64_t row_len, const int64_t q_stride[3],
    const int64_t kv_stride[5], const int64_t weight_stride[2], float softmax_scale, int causal,
    int64_t window, int dtype, void* stream) {
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
  // Tiles that there can be at most.
  const int64_t tiles = (total_pages * page_size / kWTile + batch) * num_kv_heads;
  AKT_CHECK(tiles < (1ll << 31) && grid_fits(tiles, kWThreads), "problem too large");
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
  p.N = num_rows;
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
  hipStream_t st = (hipStream_t)stream;
  const bool bf16 = dtype == AKT_DTYPE_BF16;
  if (head_dim == 64) return launch_weights<64>(p, bf16, tiles, st);
  if (head_dim == 256) return launch_weights<256>(p, bf16, tiles, st);
  return launch_weights<128>(p, bf16, tiles, st);
}
