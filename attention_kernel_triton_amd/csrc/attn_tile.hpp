// Pieces shared by the kernels that multiply 32-row MFMA blocks of queries with staged K / V
// tiles: the operand element type, the LDS swizzles of tile and output rows, and a
// division by small integers.
#pragma once

#include "akt_common.hpp"

namespace akt {

// Operand element type of a kernel instance: fp16 (v_mfma_f32_32x32x16_f16,
// P rounded to fp16 as the reference does) or bf16 (the bf16 MFMA, P rounded
// to bf16, since both MFMA operands share one type).  Global loads and the
// LDS staging move raw 16-byte chunks and do not depend on it.
template <bool BF16>
struct Elt {
  typedef half8_t v8;
  static constexpr uint32_t kOnes = 0x3c003c00u;  // (1, 1)
  static __device__ __forceinline__ v8 as8(uint4_t u) { return __builtin_bit_cast(v8, u); }
  static __device__ __forceinline__ float16_t mfma(v8 a, v8 b, float16_t c) {
    return mfma32x32x16(a, b, c);
  }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack_half2(lo, hi); }
  static __device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
    return ::akt::dot2(a, b, c);
  }
};
template <>
struct Elt<true> {
  typedef bf16x8_t v8;
  static constexpr uint32_t kOnes = 0x3f803f80u;  // (1, 1)
  static __device__ __forceinline__ v8 as8(uint4_t u) { return __builtin_bit_cast(v8, u); }
  static __device__ __forceinline__ float16_t mfma(v8 a, v8 b, float16_t c) {
    return mfma32x32x16_bf16(a, b, c);
  }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
    return dot2_bf16(a, b, c);
  }
};

// Chunk-position swizzle of a K / V tile row: chunk c (16 bytes) of row r lies at position
// c ^ tswz(r) of the row, so that the K reads (16 consecutive rows, one chunk each) and the
// transposing V reads (four rows, four chunks) use all LDS banks.  A function of r mod 16, with
// tswz(r + 8) = tswz(r) ^ 2.
// - 64- and 192-dim rows (128 / 384 bytes) start on bank 0 or 32 by row
//   parity: over 16 consecutive rows the even rows' values are a permutation
//   of 0..7, and so are the odd rows' (K reads), and rows 4i + j and 4i + j + 2
//   differ in bit 2 (V reads: their 4-chunk blocks land in different halves).
// - 128- and 256-dim rows (256 / 512 bytes) all start on bank 0: 16
//   consecutive rows get a permutation of 0..15, and rows 4i..4i+3 differ in
//   bits 2..3.
template <int D>
__device__ __forceinline__ int tswz(int r) {
  if constexpr (D == 64 || D == 192) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  else return ((r & 3) << 2) | ((r >> 2) & 3);
}
// Chunk-position swizzle of the epilogue's O staging rows.
__device__ __forceinline__ int eswz(int r) { return ((r & 3) << 1) | ((r >> 2) & 1); }

// n / d for 0 <= n < 2^22 and d >= 1, given inv = 1 / d rounded to float:
// the float estimate is within one of the quotient, and one correction step
// makes it exact.  (n / d through the integer divide sequence costs several
// dependent VALU-to-SALU round trips at the start of every workgroup.)
__device__ __forceinline__ int div_small(int n, int d, float inv) {
  int q = (int)((float)n * inv);
  const int r = n - q * d;
  q += (r >= d ? 1 : 0) - (r < 0 ? 1 : 0);
  return q;
}

}  // namespace akt
