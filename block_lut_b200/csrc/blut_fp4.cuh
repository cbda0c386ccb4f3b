// 4-bit microscaled matrices (e2m1 codes, one 8-bit scale per block of
// columns): device layouts and the small helpers that the quantiser and the
// product share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

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

constexpr uint32_t kSiluEnd = 0x7F7FFF00u;  // bits of the largest float32 less 2^-16 of it
// More than the error of a float32 estimate of silu(gate) * up / (s g): 2^-17.8
// of the product (silu_mul_f32), four roundings of the quotient.
constexpr float kSiluWin = 0x1p-17f;

template <int DT>
struct Elem;
template <>
struct Elem<BLUT_F16> {
  using T = uint16_t;
  static __device__ __forceinline__ float f(uint16_t v) { return __half2float(__ushort_as_half(v)); }
  static __device__ __forceinline__ uint16_t from(float v) { return __half_as_ushort(__float2half_rn(v)); }
};
template <>
struct Elem<BLUT_BF16> {
  using T = uint16_t;
  static __device__ __forceinline__ float f(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
  static __device__ __forceinline__ uint16_t from(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
};
template <>
struct Elem<BLUT_F32> {
  using T = float;
  static __device__ __forceinline__ float f(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};

// 16 consecutive values of a row, zeros past the n valid ones.
template <int DT>
__device__ __forceinline__ void load16(const typename Elem<DT>::T* p, int n, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = i < n ? Elem<DT>::f(p[i]) : 0.0f;
}

// 16 values of a row as they are in memory.  kVec: the boundary in bytes that
// every such run starts on (32 or 16), or 0 for any other.
template <int DT>
struct Raw {
  static constexpr int kN = DT == BLUT_F32 ? 4 : 2;
  uint4 w[kN];
};
template <int DT, int kVec>
__device__ __forceinline__ void raw_load(const typename Elem<DT>::T* p, Raw<DT>& r) {
  if constexpr (kVec == 16) {
#pragma unroll
    for (int i = 0; i < Raw<DT>::kN; ++i) r.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  } else {
#pragma unroll
    for (int i = 0; i < Raw<DT>::kN; i += 2)
      asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
          : "=r"(r.w[i].x), "=r"(r.w[i].y), "=r"(r.w[i].z), "=r"(r.w[i].w), "=r"(r.w[i + 1].x), "=r"(r.w[i + 1].y),
            "=r"(r.w[i + 1].z), "=r"(r.w[i + 1].w)
          : "l"(reinterpret_cast<const uint4*>(p) + i));
  }
}
template <int DT>
__device__ __forceinline__ void raw_unpack(const Raw<DT>& r, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < Raw<DT>::kN; ++i) {
    const uint32_t w[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == BLUT_F32) {
        v[4 * i + j] = __uint_as_float(w[j]);
      } else if constexpr (DT == BLUT_BF16) {
        v[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
        v[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        v[8 * i + 2 * j] = f.x;
        v[8 * i + 2 * j + 1] = f.y;
      }
    }
  }
}

// max(a, |b|, |c|); NaN if one of them is.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(fabsf(b)), "f"(fabsf(c)));
  return d;
}

// Border between e2m1 codes c and c + 1 (c = 0 .. 6).
__device__ __forceinline__ float e2m1_border(uint32_t c) {
  return c < 4 ? 0.25f + 0.5f * (float)c : c == 4 ? 2.5f : c == 5 ? 3.5f : 5.0f;
}
// Code of |x| between the neighbours lo and lo + 1, by the exact quotient.
__device__ __forceinline__ uint32_t e2m1_decide(double ax, double unit, uint32_t lo) {
  const double border = (double)e2m1_border(lo) * unit;
  return ax > border || (ax == border && (lo & 1)) ? lo + 1 : lo;
}
__device__ __forceinline__ uint32_t e4m3x2_sat(float hi, float lo) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
// Neighbouring codes lo and hi (lo = hi: decided) for a quotient at border /
// unit of them: hi where x is past the border, the even one on it.  A border
// times its small factor (at most 7 bits) is exact, so the sign of the fused
// difference is that of x - border * factor * g.
__device__ __forceinline__ bool past_border(float x, float border, float g, uint32_t lo) {
  const float d = fmaf(-border, g, x);
  return d > 0.0f || (d == 0.0f && (lo & 1));
}
// e4m3(a / (6 g)) by the exact quotient; t is that quotient up to 2^-21.
__device__ __forceinline__ uint32_t e4m3_scale(float a, float g, float t) {
  const uint32_t both = e4m3x2_sat(t * (1.0f + 0x1p-20f), t * (1.0f - 0x1p-20f));
  uint32_t lo = both & 0xFFu;
  const uint32_t hi = both >> 8;
  if (lo != hi && past_border(a, 3.0f * (e4m3_f32(lo) + e4m3_f32(hi)), g, lo)) lo = hi;
  return lo;
}
// The same of a float64 value.
__device__ __forceinline__ uint32_t e4m3_scale_f64(double a, float g) {
  const float t = (float)(a / (6.0 * (double)g));
  const uint32_t both = e4m3x2_sat(t * (1.0f + 0x1p-20f), t * (1.0f - 0x1p-20f));
  uint32_t lo = both & 0xFFu;
  const uint32_t hi = both >> 8;
  if (lo != hi) {
    const double border = 3.0 * ((double)e4m3_f32(lo) + (double)e4m3_f32(hi)) * (double)g;
    if (a > border || (a == border && (lo & 1))) lo = hi;
  }
  return lo;
}

// The scale byte and the 16 codes of this lane's columns.  A block is one
// lane (nvfp4) or two neighbouring lanes (mxfp4).  v: the values; kSilu:
// float32 approximations, and `unsure` is raised for a block that a more
// exact form could change.
template <int DT, bool kMX, bool kSilu>
__device__ __forceinline__ uint2 encode16(const float (&v)[16], float g, bool& unsure, uint32_t& sbyte) {
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; i += 2) most = max3_abs(most, v[i], v[i + 1]);
  uint32_t top = __float_as_uint(most) & 0x7FFFFFFFu;  // bits of non-negative floats order as integers, NaN last
  if (kMX) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
  // an infinity or a NaN: the block has no scale (whether a product passes
  // float32's end is not for an estimate to say)
  const bool bad = kSilu ? top > 0x7F800000u : top >= 0x7F800000u;
  if (kSilu) unsure |= top >= kSiluEnd;
  const float a = __uint_as_float(top);
  float r, unit = 0.0f;
  if constexpr (kMX) {
    const int e = (int)(top >> 23);
    sbyte = e > 2 ? (uint32_t)(e - 2) : 0u;
    r = __uint_as_float((254u - sbyte) << 23);
    if (kSilu) {  // near a power of two, or where float32 has lost digits
      unsure |= (__float_as_uint(a * (1.0f + kSiluWin)) >> 23) != (__float_as_uint(a * (1.0f - kSiluWin)) >> 23);
      unsure |= top - 1u < 0x0D800000u - 1u;  // 0 < a < 2^-100
    }
  } else {
    const float t = a * __frcp_rn(6.0f * g);
    if (kSilu) {
      const uint32_t both = e4m3x2_sat(t * (1.0f + kSiluWin), t * (1.0f - kSiluWin));
      sbyte = both & 0xFFu;
      unsure |= sbyte != both >> 8;
    } else {
      sbyte = e4m3_scale(a, g, t);
    }
    unit = e4m3_f32(sbyte);
    r = unit > 0.0f ? __frcp_rn(unit * g) : 0.0f;
  }
  uint2 c;
  if constexpr (kMX && !kSilu) {
    float w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = v[i] * r;
    c = make_uint2(e2m1x8(w), e2m1x8(w + 8));
  } else {
    constexpr float kWin = kSilu ? kSiluWin : 0x1p-21f;
    const float ru = r * (1.0f + kWin), rd = r * (1.0f - kWin);
    float w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = v[i] * rd;
    c = make_uint2(e2m1x8(w), e2m1x8(w + 8));
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = v[i] * ru;
    uint32_t d0 = c.x ^ e2m1x8(w), d1 = c.y ^ e2m1x8(w + 8);
    if constexpr (!kSilu && DT == BLUT_F32) {
      if (d0 | d1) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          uint32_t& cw = i < 8 ? c.x : c.y;
          const int sh = 4 * (i & 7);
          if (((i < 8 ? d0 : d1) >> sh) & 15u) {
            const uint32_t lo = (cw >> sh) & 7u;
            if (past_border(fabsf(v[i]), e2m1_border(lo) * unit, g, lo)) cw += 1u << sh;
          }
        }
      }
    } else if constexpr (!kSilu) {
      // a 16-bit x this near to a border is the border rounded to x's type:
      // the code alone tells which x it was
      while (d0 | d1) {
        const bool second = d0 == 0;
        const uint32_t d = second ? d1 : d0;
        const int sh = (__ffs(d) - 1) & 28;
        const uint32_t lo = ((second ? c.y : c.x) >> sh) & 7u;
        const float border = e2m1_border(lo) * unit;
        const uint32_t up = past_border(Elem<DT>::f(Elem<DT>::from(border * g)), border, g, lo) ? 1u << sh : 0u;
        const uint32_t left = d & ~(15u << sh);
        if (second)
          c.y += up, d1 = left;
        else
          c.x += up, d0 = left;
      }
    } else {
      unsure |= (d0 | d1) != 0;
    }
  }
  if (kSilu) {
    unsure = unsure && !bad;
    if (kMX) unsure |= __shfl_xor_sync(0xFFFFFFFFu, unsure ? 1 : 0, 1) != 0;
  }
  if (bad) {
    sbyte = kMX ? 0xFFu : 0x7Fu;
    c = make_uint2(0, 0);
  }
  return c;
}

}  // namespace blut
