// 4-bit microscaled matrices (e2m1 codes, one 8-bit scale per block of
// columns): device layouts and the small helpers that the quantiser and the
// product share.
#pragma once

#include "blut_common.cuh"
#include "blut_internal.h"

namespace blut {

// A matrix [rows][cols] is held over Kp = cols rounded up to 128 columns;
// the codes past `cols` are zero.
//
// FP4 layout (what the quantisers write and the product reads as its token
// operand):
//   codes   [Kp / 32][rows][16 B]  32 columns of a row, column 2j in the low
//           half of byte j;
//   scales  [Kp / 64 (nvfp4) | Kp / 128 (mxfp4)][rows][4 B]  the scales of
//           four consecutive blocks of a row.
// Any run of rows is contiguous inside a chunk of 32 columns, so a token tile
// that starts at any row is fetched by bulk copies, and 8 rows of a chunk are
// one 128-byte core matrix of tcgen05.mma's K-major operand without swizzle.
//
// Tiled layout (the weight operand): per (128-row tile, 128-column block)
// one unit, block after block:
//   codes   4 chunks x 128 rows x 16 B
//   scales  512 B per 4 scales of a row, row r at (r % 32) * 16 + (r / 32) * 4:
//           the order in which tcgen05.cp 32x128b brings them to tensor memory.
// Rows past the matrix are zero.
constexpr int kFp4BlockCols = 128;
constexpr int kFp4UnitCodes = 128 * 64;

__host__ __device__ inline bool fp4_valid(const blut_fp4_desc& d) {
  return (d.kind == BLUT_FP4_NV || d.kind == BLUT_FP4_MX) && d.rows > 0 && d.cols > 0 && d.rows < (1ll << 31) &&
         d.cols <= (1ll << 24);
}
__host__ __device__ inline int fp4_kblocks(int64_t cols) { return (int)((cols + kFp4BlockCols - 1) / kFp4BlockCols); }
// Scale words (4 bytes of a row) per 128 columns.
__host__ __device__ inline int fp4_words(int kind) { return kind == BLUT_FP4_NV ? 2 : 1; }
__host__ __device__ inline int fp4_block(int kind) { return kind == BLUT_FP4_NV ? 16 : 32; }
__host__ __device__ inline int fp4_unit_bytes(int kind) { return kFp4UnitCodes + 512 * fp4_words(kind); }

// blut_fp4_quantize whose kernel lets a following early launch (blut_fp4_linear's product) begin.
int fp4_quantize_for_product(const blut_fp4_desc& d, const void* x, int32_t dtype, int64_t ld, const float* g,
                             void* codes, void* scales, cudaStream_t stream);

// e4m3 byte (0 .. 0x7E) -> float.
__device__ __forceinline__ float e4m3_f32(uint32_t b) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)b));
  return __half2float(__ushort_as_half((uint16_t)(h2 & 0xFFFFu)));
}
// The scale a byte stands for: e4m3 (0x7F: NaN), or 2^(byte - 127) (0xFF: NaN).
template <bool kMX>
__device__ __forceinline__ float fp4_scale_f32(uint32_t b) {
  if constexpr (kMX) {
    return __uint_as_float(b == 255 ? 0x7FC00000u : b == 0 ? 0x00400000u : b << 23);
  } else {
    return e4m3_f32(b);
  }
}
// Eight e2m1 codes (low half first) -> four float16 pairs.
__device__ __forceinline__ void e2m1x8_f16(uint32_t w, uint32_t* h) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
// Eight floats -> eight e2m1 codes, round to nearest even, at most 6.
__device__ __forceinline__ uint32_t e2m1x8(const float* v) {
  uint32_t d;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(d)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return d;
}

}  // namespace blut
