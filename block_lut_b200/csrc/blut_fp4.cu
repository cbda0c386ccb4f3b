// Quantisation of rows to 4-bit microscaled form, its way back, and the
// layout conversions (include/blut.h, "4-bit microscaled").
//
//   nvfp4  s = e4m3(max|x| / (6 g)) per 16 columns, one float32 g per matrix
//   mxfp4  s = 2^(floor(log2 max|x|) - 2) per 32 columns
//   q = e2m1(x / (s g)), round to nearest even, saturating at 6
//
// Each rounding goes by the exact quotient, so that the result is a function
// of the inputs alone and not of how a division is carried out.  The mxfp4
// quotient is a power of two and exact in float32.  For nvfp4 a code is
// computed from x * (1 / (s g)) twice, with the reciprocal moved up and down
// by 2^-21, more than its error; where both give the same code, no border
// lies between them and the code is right.  Where they differ, the border is
// compared with x in float64, in which border * s * g (2 + 4 + 24 bits) is
// exact.  Borders are met often when g is a power of two (0.8 % of bf16
// values are ties) and cost a few instructions each.  silu(gate) * up is
// rounded once, to its code: it is computed in float32 (relative error below
// 2^-20, window 2^-18); a block with a value near a border is done again in
// float64 (about 1 block in 2000).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "blut_fp4.cuh"

namespace blut {
namespace {

constexpr int kQRows = 8;      // rows per CTA, a warp each
constexpr int kQCols = 512;    // columns per CTA, 16 per lane
constexpr int kQChunks = kQCols / 32;
constexpr int kQPitch = kQRows * 16 + 16;  // bytes of a staged chunk: 16 more than its rows, against bank conflicts
constexpr float kMinGlobal = 7.888609052210118e-31f;  // 2^-100

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

// 16 consecutive values of a row, zeros past the n valid ones.  kVec: the
// address of every such run is a multiple of 16 bytes.
template <int DT, bool kVec>
__device__ __forceinline__ void load16(const typename Elem<DT>::T* p, int n, float (&v)[16]) {
  if (kVec && n >= 16) {
    if constexpr (DT == BLUT_F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p) + i);
        v[4 * i] = a.x, v[4 * i + 1] = a.y, v[4 * i + 2] = a.z, v[4 * i + 3] = a.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(p) + i);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[8 * i + 2 * j] = Elem<DT>::f((uint16_t)(w[j] & 0xFFFFu));
          v[8 * i + 2 * j + 1] = Elem<DT>::f((uint16_t)(w[j] >> 16));
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = i < n ? Elem<DT>::f(p[i]) : 0.0f;
  }
}

// silu(g) * u in float32, relative error below 2^-20 for g >= -80.
__device__ __forceinline__ float silu_mul_f32(float g, float u) { return __fdividef(g, 1.0f + expf(-g)) * u; }
__device__ __forceinline__ double silu_mul_f64(double g, double u) { return g / (1.0 + exp(-g)) * u; }

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
// e4m3(a / (6 g)) by the exact quotient; t is that quotient up to 2^-21.
__device__ __forceinline__ uint32_t e4m3_scale(double a, float g, float t) {
  const uint32_t both = e4m3x2_sat(t * (1.0f + 0x1p-20f), t * (1.0f - 0x1p-20f));
  uint32_t lo = both & 0xFFu;
  const uint32_t hi = both >> 8;
  if (lo != hi) {
    const double border = 0.5 * ((double)e4m3_f32(lo) + (double)e4m3_f32(hi)) * (6.0 * (double)g);
    if (a > border || (a == border && (lo & 1))) lo = hi;
  }
  return lo;
}

// The scale byte and the 16 codes of this lane's columns.  A block is one
// lane (nvfp4) or two neighbouring lanes (mxfp4).  v: the values; kSilu:
// float32 approximations whose exact forms exact(j) gives.
template <bool kMX, bool kSilu, class Exact>
__device__ __forceinline__ uint2 encode16(const float (&v)[16], float g, bool unsure, uint32_t& sbyte, Exact exact) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  if (kMX) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
  const bool bad = top >= 0x7F800000u;  // an infinity or a NaN: the block has no scale
  const float a = __uint_as_float(top);
  float r, unit = 0.0f;
  if constexpr (kMX) {
    const int e = (int)(top >> 23);
    sbyte = e > 2 ? (uint32_t)(e - 2) : 0u;
    r = __uint_as_float((254u - sbyte) << 23);
    if (kSilu) {  // near a power of two, or where float32 has lost digits
      unsure |= (__float_as_uint(a * (1.0f + 0x1p-18f)) >> 23) != (__float_as_uint(a * (1.0f - 0x1p-18f)) >> 23);
      unsure |= a < 0x1p-100f && top != 0;
      unsure |= __shfl_xor_sync(0xFFFFFFFFu, unsure ? 1 : 0, 1) != 0;
    }
  } else {
    const float t = a * __frcp_rn(6.0f * g);
    if (kSilu) {
      const uint32_t both = e4m3x2_sat(t * (1.0f + 0x1p-18f), t * (1.0f - 0x1p-18f));
      sbyte = both & 0xFFu;
      unsure |= sbyte != both >> 8;
    } else {
      sbyte = e4m3_scale((double)a, g, t);
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
    constexpr float kWin = kSilu ? 0x1p-18f : 0x1p-21f;
    const float ru = r * (1.0f + kWin), rd = r * (1.0f - kWin);
    float w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = v[i] * rd;
    c = make_uint2(e2m1x8(w), e2m1x8(w + 8));
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = v[i] * ru;
    uint32_t d0 = c.x ^ e2m1x8(w), d1 = c.y ^ e2m1x8(w + 8);
    if constexpr (!kSilu) {
      if (d0 | d1) {
        const double un = (double)unit * (double)g;  // 4 + 24 bits: exact
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          uint32_t& cw = i < 8 ? c.x : c.y;
          const int sh = 4 * (i & 7);
          if (((i < 8 ? d0 : d1) >> sh) & 15u) {
            const uint32_t lo = (cw >> sh) & 7u;
            cw += (e2m1_decide((double)fabsf(v[i]), un, lo) - lo) << sh;
          }
        }
      }
    } else {
      unsure |= (d0 | d1) != 0;
      if (kMX) unsure |= __shfl_xor_sync(0xFFFFFFFFu, unsure ? 1 : 0, 1) != 0;
      if (unsure && !bad) {  // mxfp4: both lanes of the block or neither
        double m = 0.0;
#pragma unroll 1
        for (int i = 0; i < 16; ++i) m = fmax(m, fabs(exact(i)));
        double un;
        if constexpr (kMX) {
          m = fmax(m, __shfl_xor_sync(3u << (threadIdx.x & 30u), m, 1));
          const int e = m > 0.0 ? ilogb(m) - 2 : -127;
          sbyte = (uint32_t)(min(max(e, -127), 127) + 127);
          un = ldexp(1.0, (int)sbyte - 127);
        } else {
          sbyte = e4m3_scale(m, g, (float)(m / (6.0 * (double)g)));
          un = (double)e4m3_f32(sbyte) * (double)g;
        }
        c = make_uint2(0, 0);
#pragma unroll 1
        for (int i = 0; i < 16; ++i) {
          const double x = exact(i);
          uint32_t q = 0;
#pragma unroll 1
          for (uint32_t k = 0; k < 7 && q == k && un > 0.0; ++k) q = e2m1_decide(fabs(x), un, k);
          q |= signbit(x) ? 8u : 0u;
          if (i < 8)
            c.x |= q << (4 * i);
          else
            c.y |= q << (4 * (i - 8));
        }
      }
    }
  }
  if (bad) {
    sbyte = kMX ? 0xFFu : 0x7Fu;
    c = make_uint2(0, 0);
  }
  return c;
}

// x [rows][ld] -> FP4 layout.  A warp takes one row and 512 columns; codes
// and scales go through shared memory, so that each store to a chunk covers
// 8 rows.  Bound by memory: rows * cols * (2 B in, 0.5 + 1/16 or 1/32 B out).
template <int DT, bool kMX, bool kSilu, bool kVec>
__global__ void __launch_bounds__(32 * kQRows)
    fp4_quantize_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t ld, const int32_t* __restrict__ row_index,
                        int64_t src_rows, const float* __restrict__ gptr, int64_t rows, int cols, int kp,
                        uint8_t* __restrict__ codes, uint32_t* __restrict__ scales) {
  __shared__ alignas(16) uint8_t sc[kQChunks * kQPitch];
  __shared__ uint32_t ss[kQCols / 64][kQRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row0 = (int64_t)blockIdx.x * kQRows, row = row0 + warp;
  const int col0 = blockIdx.y * kQCols, col = col0 + 16 * lane;
  const int n = min(16, max(0, cols - col));
  const float g = kMX ? 1.0f : __ldg(gptr);
  int64_t src = row < rows ? row : -1;
  if (row_index && src >= 0) {
    src = row_index[row];
    if (src >= src_rows) src = -1;
  }
  float v[16];
  bool unsure = false;
  const typename Elem<DT>::T* p = x + (src < 0 ? 0 : src) * ld + col;
  if (src < 0 || n == 0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.0f;
  } else if constexpr (kSilu) {
    float u[16];
    load16<DT, kVec>(p, n, v);
    load16<DT, kVec>(p + cols, n, u);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      unsure |= v[i] < -80.0f;  // exp(-gate) nears the end of float32
      v[i] = silu_mul_f32(v[i], u[i]);
    }
  } else {
    load16<DT, kVec>(p, n, v);
  }
  uint32_t sbyte;
  const uint2 c = encode16<kMX, kSilu>(v, g, unsure, sbyte, [&](int i) {
    if (src < 0 || i >= n) return 0.0;
    return silu_mul_f64((double)Elem<DT>::f(p[i]), (double)Elem<DT>::f(p[cols + i]));
  });
  *reinterpret_cast<uint2*>(sc + (lane >> 1) * kQPitch + warp * 16 + (lane & 1) * 8) = c;
  {
    uint8_t* s8 = reinterpret_cast<uint8_t*>(ss);
    if (kMX) {
      if ((lane & 1) == 0) s8[((lane >> 3) * kQRows + warp) * 4 + ((lane >> 1) & 3)] = (uint8_t)sbyte;
    } else {
      s8[((lane >> 2) * kQRows + warp) * 4 + (lane & 3)] = (uint8_t)sbyte;
    }
  }
  __syncthreads();
  const int t = threadIdx.x, r = t & (kQRows - 1);
  if (row0 + r >= rows) return;
  const int ch = t >> 3;  // 32 threads' worth of chunks: 16 chunks x 8 rows use half the threads
  if (t < kQChunks * kQRows) {
    if (col0 + 32 * ch < kp)
      *reinterpret_cast<uint4*>(codes + (((int64_t)(col0 / 32) + ch) * rows + row0 + r) * 16) =
          *reinterpret_cast<const uint4*>(sc + ch * kQPitch + r * 16);
  } else {
    constexpr int kWordCols = kMX ? 128 : 64;
    const int w = ch - kQChunks;
    if (w < kQCols / kWordCols && col0 + kWordCols * w < kp)
      scales[((int64_t)(col0 / kWordCols) + w) * rows + row0 + r] = ss[w][r];
  }
}

// g = max(max|x| / 2688, 2^-100) over the finite values: with it the largest
// block's scale is 448.  out[0]: g, out[1] and out[2]: the running maximum's
// bits and the CTAs that are done (zeroed before the launch).  The maximum
// does not depend on the order of the atomics.
template <int DT, bool kSilu, bool kVec>
__global__ void __launch_bounds__(256)
    fp4_global_scale_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t ld, int64_t rows, int cols,
                            float* out) {
  const int per_row = (cols + 15) / 16;
  const int64_t total = rows * per_row;
  uint32_t top = 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per_row;
    const int col = (int)(i - row * per_row) * 16, n = min(16, cols - col);
    const typename Elem<DT>::T* p = x + row * ld + col;
    float v[16];
    load16<DT, kVec>(p, n, v);
    if constexpr (kSilu) {
      float u[16];
      load16<DT, kVec>(p + cols, n, u);
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = silu_mul_f32(v[j], u[j]);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const uint32_t b = __float_as_uint(v[j]) & 0x7FFFFFFFu;
      top = max(top, b < 0x7F800000u ? b : 0u);
    }
  }
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  __shared__ uint32_t part[8];
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) top = max(top, part[i]);
    uint32_t* u = reinterpret_cast<uint32_t*>(out);
    atomicMax(u + 1, top);
    __threadfence();
    if (atomicAdd(u + 2, 1u) == gridDim.x - 1) {
      __threadfence();
      out[0] = fmaxf(__fdiv_rn(__uint_as_float(atomicMax(u + 1, 0u)), 2688.0f), kMinGlobal);
    }
  }
}

// FP4 layout -> q * s * g, [rows][ld]; the product q * s is exact.
template <int DT, bool kMX, bool kVec>
__global__ void __launch_bounds__(32 * kQRows)
    fp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint32_t* __restrict__ scales,
                          const float* __restrict__ gptr, typename Elem<DT>::T* __restrict__ out, int64_t ld,
                          int64_t rows, int cols, int kp) {
  __shared__ alignas(16) uint8_t sc[kQChunks * kQPitch];
  __shared__ uint32_t ss[kQCols / 64][kQRows];
  constexpr int kWordCols = kMX ? 128 : 64;
  const int64_t row0 = (int64_t)blockIdx.x * kQRows;
  const int col0 = blockIdx.y * kQCols;
  const float g = kMX || !gptr ? 1.0f : __ldg(gptr);
  {
    const int t = threadIdx.x, r = t & (kQRows - 1), ch = t >> 3;
    if (row0 + r < rows) {
      if (t < kQChunks * kQRows) {
        if (col0 + 32 * ch < kp)
          *reinterpret_cast<uint4*>(sc + ch * kQPitch + r * 16) =
              __ldg(reinterpret_cast<const uint4*>(codes + (((int64_t)(col0 / 32) + ch) * rows + row0 + r) * 16));
      } else {
        const int w = ch - kQChunks;
        if (w < kQCols / kWordCols && col0 + kWordCols * w < kp)
          ss[w][r] = __ldg(scales + ((int64_t)(col0 / kWordCols) + w) * rows + row0 + r);
      }
    }
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = row0 + warp;
  const int col = col0 + 16 * lane, n = min(16, cols - col);
  if (row >= rows || n <= 0) return;
  const uint2 c = *reinterpret_cast<const uint2*>(sc + (lane >> 1) * kQPitch + warp * 16 + (lane & 1) * 8);
  const uint32_t sb = kMX ? (ss[lane >> 3][warp] >> (8 * ((lane >> 1) & 3))) & 0xFFu
                          : (ss[lane >> 2][warp] >> (8 * (lane & 3))) & 0xFFu;
  const float s = fp4_scale_f32<kMX>(sb);
  typename Elem<DT>::T o[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 q = e2m1x2_f32(((i < 4 ? c.x : c.y) >> (8 * (i & 3))) & 0xFFu);
    o[2 * i] = Elem<DT>::from(q.x * s * g);
    o[2 * i + 1] = Elem<DT>::from(q.y * s * g);
  }
  typename Elem<DT>::T* p = out + row * ld + col;
  if (kVec && n == 16) {
    constexpr int kV = 16 / sizeof(o[0]);
#pragma unroll
    for (int i = 0; i < 16 / kV; ++i) reinterpret_cast<uint4*>(p)[i] = *reinterpret_cast<const uint4*>(o + kV * i);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < n) p[i] = o[i];
  }
}

// Row-major bytes (a checkpoint's) <-> FP4 layout, one (row, 128-column
// block) per thread; load time only.
template <bool kMX, bool kExport>
__global__ void fp4_rows_kernel(uint8_t* rc, uint8_t* rs, int64_t rows, int cols, uint8_t* codes, uint8_t* scales) {
  const int64_t row = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (row >= rows) return;
  constexpr int kB = kMX ? 32 : 16;
  const int kb = blockIdx.y, nb = (cols + kB - 1) / kB, nbytes = nb * kB / 2;
  for (int i = 0; i < 64; ++i) {  // 64 bytes of codes
    const int b = kb * 64 + i;
    uint8_t* f = codes + (((int64_t)kb * 4 + (i >> 4)) * rows + row) * 16 + (i & 15);
    if (kExport) {
      if (b < nbytes) rc[row * nbytes + b] = *f;
    } else {
      uint8_t v = b < nbytes ? rc[row * nbytes + b] : 0;
      if (2 * b >= cols)
        v = 0;  // columns past the matrix hold zeros
      else if (2 * b + 1 >= cols)
        v &= 0x0F;
      *f = v;
    }
  }
  constexpr int kPer = 128 / kB;
  for (int i = 0; i < kPer; ++i) {
    const int b = kb * kPer + i;
    uint8_t* f = scales + (((int64_t)kb * (kPer / 4) + (i >> 2)) * rows + row) * 4 + (i & 3);
    if (kExport) {
      if (b < nb) rs[row * nb + b] = *f;
    } else {
      *f = b < nb ? rs[row * nb + b] : 0;
    }
  }
}

// FP4 layout -> tiled layout: one (row of a tile, 128-column block) per thread.
__global__ void fp4_pack_kernel(const uint4* __restrict__ codes, const uint32_t* __restrict__ scales, int64_t rows,
                                int kblocks, int words, uint8_t* __restrict__ tiled) {
  const int r = threadIdx.x, b = blockIdx.y;
  const int64_t t = blockIdx.x, row = t * 128 + r;
  const bool in = row < rows;
  uint8_t* u = tiled + (t * kblocks + b) * (int64_t)(kFp4UnitCodes + 512 * words);
  for (int c = 0; c < 4; ++c)
    reinterpret_cast<uint4*>(u)[c * 128 + r] = in ? codes[((int64_t)b * 4 + c) * rows + row] : make_uint4(0, 0, 0, 0);
  for (int w = 0; w < words; ++w)
    *reinterpret_cast<uint32_t*>(u + kFp4UnitCodes + 512 * w + (r & 31) * 16 + (r >> 5) * 4) =
        in ? scales[((int64_t)b * words + w) * rows + row] : 0u;
}

inline bool aligned16(const void* p, int64_t ld_bytes) { return (((uintptr_t)p) | (uintptr_t)ld_bytes) % 16 == 0; }
inline int64_t elem_size(int dtype) { return dtype == BLUT_F32 ? 4 : 2; }
inline int launched() { return cudaGetLastError() == cudaSuccess ? BLUT_OK : BLUT_ERR_LAUNCH; }

template <int DT, bool kSilu>
int launch_quantize(const blut_fp4_desc& d, const void* x, int64_t ld, const int32_t* row_index, int64_t src_rows,
                    const float* g, void* codes, void* scales, cudaStream_t stream) {
  using T = typename Elem<DT>::T;
  const int64_t es = sizeof(T);
  const bool vec = aligned16(x, ld * es) && (!kSilu || (d.cols * es) % 16 == 0);
  const int kp = fp4_kblocks(d.cols) * kFp4BlockCols;
  const dim3 grid((unsigned)((d.rows + kQRows - 1) / kQRows), (unsigned)((kp + kQCols - 1) / kQCols));
#define BLUT_Q(MX, VEC)                                                                                            \
  fp4_quantize_kernel<DT, MX, kSilu, VEC><<<grid, 32 * kQRows, 0, stream>>>(                                       \
      static_cast<const T*>(x), ld, row_index, src_rows, g, d.rows, (int)d.cols, kp, static_cast<uint8_t*>(codes), \
      static_cast<uint32_t*>(scales))
  if (d.kind == BLUT_FP4_MX) {
    if (vec) BLUT_Q(true, true); else BLUT_Q(true, false);
  } else {
    if (vec) BLUT_Q(false, true); else BLUT_Q(false, false);
  }
#undef BLUT_Q
  return launched();
}

int quantize(const blut_fp4_desc* d, const void* x, int32_t dtype, int64_t ld, const int32_t* row_index,
             int64_t src_rows, const float* g, void* codes, void* scales, bool silu, cudaStream_t stream) {
  if (!d || !fp4_valid(*d) || !x || !codes || !scales || ld < (silu ? 2 : 1) * d->cols || src_rows <= 0)
    return BLUT_ERR_INVALID;
  if (!row_index && src_rows != d->rows) return BLUT_ERR_INVALID;
  if (d->kind == BLUT_FP4_NV && !g) return BLUT_ERR_INVALID;
  if (((uintptr_t)codes | (uintptr_t)scales) % 16 != 0 || (uintptr_t)x % elem_size(dtype) != 0) return BLUT_ERR_INVALID;
#define BLUT_Q(DT)                                                                                            \
  return silu ? launch_quantize<DT, true>(*d, x, ld, row_index, src_rows, g, codes, scales, stream)           \
              : launch_quantize<DT, false>(*d, x, ld, row_index, src_rows, g, codes, scales, stream)
  switch (dtype) {
    case BLUT_F16: BLUT_Q(BLUT_F16);
    case BLUT_BF16: BLUT_Q(BLUT_BF16);
    case BLUT_F32: BLUT_Q(BLUT_F32);
    default: return BLUT_ERR_UNSUPPORTED;
  }
#undef BLUT_Q
}

template <int DT>
int launch_global(const void* x, int64_t rows, int64_t cols, int64_t ld, bool silu, float* out, cudaStream_t stream) {
  using T = typename Elem<DT>::T;
  const int64_t es = sizeof(T);
  const bool vec = aligned16(x, ld * es) && (!silu || (cols * es) % 16 == 0);
  const int64_t ctas = (rows * ((cols + 15) / 16) + 255) / 256;
  const unsigned grid = (unsigned)(ctas < 148 * 8 ? ctas : 148 * 8);
  const T* p = static_cast<const T*>(x);
  if (silu) {
    if (vec) fp4_global_scale_kernel<DT, true, true><<<grid, 256, 0, stream>>>(p, ld, rows, (int)cols, out);
    else fp4_global_scale_kernel<DT, true, false><<<grid, 256, 0, stream>>>(p, ld, rows, (int)cols, out);
  } else {
    if (vec) fp4_global_scale_kernel<DT, false, true><<<grid, 256, 0, stream>>>(p, ld, rows, (int)cols, out);
    else fp4_global_scale_kernel<DT, false, false><<<grid, 256, 0, stream>>>(p, ld, rows, (int)cols, out);
  }
  return launched();
}

template <int DT>
int launch_dequantize(const blut_fp4_desc& d, const void* codes, const void* scales, const float* g, void* out,
                      int64_t ld, cudaStream_t stream) {
  using T = typename Elem<DT>::T;
  const bool vec = aligned16(out, ld * (int64_t)sizeof(T));
  const int kp = fp4_kblocks(d.cols) * kFp4BlockCols;
  const dim3 grid((unsigned)((d.rows + kQRows - 1) / kQRows), (unsigned)((d.cols + kQCols - 1) / kQCols));
#define BLUT_D(MX, VEC)                                                                                    \
  fp4_dequantize_kernel<DT, MX, VEC><<<grid, 32 * kQRows, 0, stream>>>(                                    \
      static_cast<const uint8_t*>(codes), static_cast<const uint32_t*>(scales), g, static_cast<T*>(out), ld, d.rows, \
      (int)d.cols, kp)
  if (d.kind == BLUT_FP4_MX) {
    if (vec) BLUT_D(true, true); else BLUT_D(true, false);
  } else {
    if (vec) BLUT_D(false, true); else BLUT_D(false, false);
  }
#undef BLUT_D
  return launched();
}

int rows_convert(const blut_fp4_desc* d, void* rc, void* rs, void* codes, void* scales, bool exp, cudaStream_t st) {
  if (!d || !fp4_valid(*d) || !rc || !rs || !codes || !scales) return BLUT_ERR_INVALID;
  if (((uintptr_t)codes | (uintptr_t)scales) % 16 != 0) return BLUT_ERR_INVALID;
  const dim3 grid((unsigned)((d->rows + 127) / 128), (unsigned)fp4_kblocks(d->cols));
  if (grid.y > 65535) return BLUT_ERR_UNSUPPORTED;
  uint8_t *a = (uint8_t*)rc, *b = (uint8_t*)rs, *c = (uint8_t*)codes, *s = (uint8_t*)scales;
  if (d->kind == BLUT_FP4_MX) {
    if (exp) fp4_rows_kernel<true, true><<<grid, 128, 0, st>>>(a, b, d->rows, (int)d->cols, c, s);
    else fp4_rows_kernel<true, false><<<grid, 128, 0, st>>>(a, b, d->rows, (int)d->cols, c, s);
  } else {
    if (exp) fp4_rows_kernel<false, true><<<grid, 128, 0, st>>>(a, b, d->rows, (int)d->cols, c, s);
    else fp4_rows_kernel<false, false><<<grid, 128, 0, st>>>(a, b, d->rows, (int)d->cols, c, s);
  }
  return launched();
}

inline cudaStream_t S(void* s) { return reinterpret_cast<cudaStream_t>(s); }

}  // namespace
}  // namespace blut

using namespace blut;

extern "C" {

int64_t blut_fp4_codes_bytes(const blut_fp4_desc* d) {
  if (!d || !fp4_valid(*d)) return BLUT_ERR_INVALID;
  return d->rows * fp4_kblocks(d->cols) * 64;
}

int64_t blut_fp4_scales_bytes(const blut_fp4_desc* d) {
  if (!d || !fp4_valid(*d)) return BLUT_ERR_INVALID;
  return d->rows * fp4_kblocks(d->cols) * 4 * fp4_words(d->kind);
}

int64_t blut_fp4_tiled_bytes(const blut_fp4_desc* d) {
  if (!d || !fp4_valid(*d)) return BLUT_ERR_INVALID;
  return (d->rows + 127) / 128 * fp4_kblocks(d->cols) * fp4_unit_bytes(d->kind);
}

int blut_fp4_global_scale(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t ld, int32_t silu_mul,
                          float* out, void* stream) {
  if (!x || !out || rows <= 0 || cols <= 0 || cols > (1ll << 24) || ld < (silu_mul ? 2 : 1) * cols ||
      (uintptr_t)out % 16 != 0 || (uintptr_t)x % elem_size(dtype) != 0)
    return BLUT_ERR_INVALID;
  if (dtype != BLUT_F16 && dtype != BLUT_BF16 && dtype != BLUT_F32) return BLUT_ERR_UNSUPPORTED;
  if (cudaMemsetAsync(out, 0, 16, S(stream)) != cudaSuccess) return BLUT_ERR_CUDA;
  switch (dtype) {
    case BLUT_F16: return launch_global<BLUT_F16>(x, rows, cols, ld, silu_mul != 0, out, S(stream));
    case BLUT_BF16: return launch_global<BLUT_BF16>(x, rows, cols, ld, silu_mul != 0, out, S(stream));
    default: return launch_global<BLUT_F32>(x, rows, cols, ld, silu_mul != 0, out, S(stream));
  }
}

int blut_fp4_quantize(const blut_fp4_desc* d, const void* x, int32_t dtype, int64_t ld, const int32_t* row_index,
                      int64_t src_rows, const float* global_scale, void* codes, void* scales, void* stream) {
  return quantize(d, x, dtype, ld, row_index, src_rows, global_scale, codes, scales, false, S(stream));
}

int blut_fp4_silu_mul_quantize(const blut_fp4_desc* d, const void* gate_up, int32_t dtype, int64_t ld,
                               const float* global_scale, void* codes, void* scales, void* stream) {
  return quantize(d, gate_up, dtype, ld, nullptr, d ? d->rows : 0, global_scale, codes, scales, true, S(stream));
}

int blut_fp4_dequantize(const blut_fp4_desc* d, const void* codes, const void* scales, const float* global_scale,
                        void* out, int32_t dtype, int64_t ld, void* stream) {
  if (!d || !fp4_valid(*d) || !codes || !scales || !out || ld < d->cols) return BLUT_ERR_INVALID;
  if (((uintptr_t)codes | (uintptr_t)scales) % 16 != 0 || (uintptr_t)out % elem_size(dtype) != 0)
    return BLUT_ERR_INVALID;
  switch (dtype) {
    case BLUT_F16: return launch_dequantize<BLUT_F16>(*d, codes, scales, global_scale, out, ld, S(stream));
    case BLUT_BF16: return launch_dequantize<BLUT_BF16>(*d, codes, scales, global_scale, out, ld, S(stream));
    case BLUT_F32: return launch_dequantize<BLUT_F32>(*d, codes, scales, global_scale, out, ld, S(stream));
    default: return BLUT_ERR_UNSUPPORTED;
  }
}

int blut_fp4_import(const blut_fp4_desc* d, const void* row_codes, const void* row_scales, void* codes, void* scales,
                    void* stream) {
  return rows_convert(d, const_cast<void*>(row_codes), const_cast<void*>(row_scales), codes, scales, false, S(stream));
}

int blut_fp4_export(const blut_fp4_desc* d, const void* codes, const void* scales, void* row_codes, void* row_scales,
                    void* stream) {
  return rows_convert(d, row_codes, row_scales, const_cast<void*>(codes), const_cast<void*>(scales), true, S(stream));
}

int blut_fp4_pack_tiled(const blut_fp4_desc* d, const void* codes, const void* scales, void* tiled, void* stream) {
  if (!d || !fp4_valid(*d) || !codes || !scales || !tiled) return BLUT_ERR_INVALID;
  if (((uintptr_t)codes | (uintptr_t)scales | (uintptr_t)tiled) % 16 != 0) return BLUT_ERR_INVALID;
  const dim3 grid((unsigned)((d->rows + 127) / 128), (unsigned)fp4_kblocks(d->cols));
  if (grid.y > 65535) return BLUT_ERR_UNSUPPORTED;
  fp4_pack_kernel<<<grid, 128, 0, S(stream)>>>(static_cast<const uint4*>(codes), static_cast<const uint32_t*>(scales),
                                               d->rows, (int)grid.y, fp4_words(d->kind),
                                               static_cast<uint8_t*>(tiled));
  return launched();
}

}  // extern "C"
