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
// compared with x by one fused multiply-add, whose sign is exact (border * s
// has 7 bits).  Borders are met often when g is a power of two or comes from
// x's own maximum (0.8 % of bf16 values are ties) and cost a few instructions
// each.  silu(gate) * up is
// rounded once, to its code: it is computed in float32 from the hardware's
// approximate exponential and reciprocal (relative error below 2^-17.8, window
// 2^-17); a block with a value near a border is done again in float64, a
// column a lane (about 1 block in 3000).
//
// All kernels here are bound by instructions before they are bound by memory,
// so a warp takes several rows of one 512-column stretch: their loads are in
// flight together and the address arithmetic is shared.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "blut_fp4.cuh"

namespace blut {
namespace {

constexpr int kQWarps = 8;
constexpr int kQCols = 512;    // columns per CTA, 16 per lane
constexpr int kQChunks = kQCols / 32;
constexpr float kMinGlobal = 7.888609052210118e-31f;  // 2^-100

// silu(g) * u in float32 for g >= -80, relative error below 2^-17.8: at g =
// -80 the exponent g * log2(e) is rounded by up to 2^-18, and its constant,
// off by 2^-25.6, moves it by 2^-19.3, which together cost ln 2 * 5.36e-6 =
// 3.72e-6; ex2 costs 2^-22, rcp 2^-23, the sum and two products 2^-24 each:
// 4.25e-6 in all.
__device__ __forceinline__ float silu_mul_f32(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return g * (r * u);  // g * r would lose digits where g is below float32's normal range
}
__device__ __forceinline__ double silu_mul_f64(double g, double u) { return g / (1.0 + exp(-g)) * u; }

// Block `block` (16 or 32 columns from column c0 of a row of gate and up) of
// silu(gate) * up in float64: one column a lane, the whole warp.  The lanes
// that hold the block's codes get them and the scale.
template <int DT, bool kMX>
__device__ __noinline__ void encode_block_f64(const typename Elem<DT>::T* row, int cols, int c0, float g, int owner,
                                              uint2& c, uint32_t& sbyte) {
  const int lane = threadIdx.x & 31;
  double x = 0.0;
  if (lane < (kMX ? 32 : 16) && c0 + lane < cols)
    x = silu_mul_f64((double)Elem<DT>::f(row[c0 + lane]), (double)Elem<DT>::f(row[cols + c0 + lane]));
  double m = fabs(x);
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmax(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
  const bool bad = __any_sync(0xFFFFFFFFu, isnan(x)) || isinf((float)m);  // not finite as a float32
  uint32_t s;
  double unit;
  if constexpr (kMX) {
    s = m > 0.0 ? (uint32_t)(min(max(ilogb(m) - 2, -127), 127) + 127) : 0u;
    unit = ldexp(1.0, (int)s - 127);
  } else {
    s = e4m3_scale_f64(m, g);
    unit = (double)e4m3_f32(s) * (double)g;
  }
  uint32_t q = 0;
#pragma unroll
  for (uint32_t k = 0; k < 7; ++k)
    if (unit > 0.0 && q == k) q = e2m1_decide(fabs(x), unit, k);
  q |= signbit(x) ? 8u : 0u;
  if (bad) s = kMX ? 0xFFu : 0x7Fu, q = 0;
  q <<= 4 * (lane & 7);  // eight lanes make a word
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) q |= __shfl_xor_sync(0xFFFFFFFFu, q, d);
  const int from = kMX ? 16 * (lane & 1) : 0;  // mxfp4: the odd lane holds columns 16 .. 31
  const uint2 w = make_uint2(__shfl_sync(0xFFFFFFFFu, q, from), __shfl_sync(0xFFFFFFFFu, q, from + 8));
  if (kMX ? (lane | 1) == (owner | 1) : lane == owner) c = w, sbyte = s;
}

// 16 columns a lane of a row (null: zeros) with n columns left, any boundary.
template <int DT>
__device__ __forceinline__ void load_row(const typename Elem<DT>::T* p, int n, typename Elem<DT>::T* buf, float (&v)[16]) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int c = 32 * j + lane;
    buf[c + (c >> 4)] = p && c < n ? p[c] : typename Elem<DT>::T(0);
  }
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = Elem<DT>::f(buf[17 * lane + j]);
}

// Bytes of a staged chunk: 16 more than its rows, against bank conflicts.
__host__ __device__ constexpr int q_pitch(int rows) { return rows * 16 + 16; }

// x [rows][ld] -> FP4 layout.  A warp takes kPer rows of one 512-column
// stretch, 16 columns a lane; codes and scales go through shared memory, so
// that each store to a chunk covers all the CTA's rows.  The rows are taken
// from the last to the first: what was written last (x by the layer before,
// or what blut_fp4_global_scale read last) is what the L2 still holds.
template <int DT, bool kMX, bool kSilu, int kVec, int kPer>
__global__ void __launch_bounds__(32 * kQWarps, kPer > 1 ? 4 : 1)
    fp4_quantize_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t ld, const int32_t* __restrict__ row_index,
                        int64_t src_rows, const float* __restrict__ gptr, int64_t rows, int cols, int kp,
                        uint8_t* __restrict__ codes, uint32_t* __restrict__ scales, int signal) {
  // the product that follows in the same call may start its weight copies
  if (signal) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int kRows = kQWarps * kPer, kPitch = q_pitch(kRows);
  constexpr int kWordCols = kMX ? 128 : 64, kWords = kQCols / kWordCols;
  __shared__ alignas(16) uint8_t sc[kQChunks * kPitch];
  __shared__ uint32_t ss[kWords * kRows];
  __shared__ typename Elem<DT>::T sx[kVec ? 1 : kQWarps][kVec ? 1 : kQCols + kQCols / 16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row0 = (int64_t)(gridDim.x - 1 - blockIdx.x) * kRows;
  const int col0 = blockIdx.y * kQCols, col = col0 + 16 * lane;
  const int n = min(16, max(0, cols - col));
  const float g = kMX ? 1.0f : __ldg(gptr);
  const typename Elem<DT>::T* p[kPer];  // null: no row, or no columns
  Raw<DT> raw[kPer], raw_up[kSilu ? kPer : 1];
  const auto src_of = [&](int64_t row) -> int64_t {  // row of x, below 0 for none
    if (row >= rows) return -1;
    if (!row_index) return row;
    const int64_t src = row_index[row];
    return src < src_rows ? src : -1;
  };
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int64_t src = src_of(row0 + warp + kQWarps * i);
    p[i] = src < 0 || n == 0 ? nullptr : x + src * ld + col;
    if (kVec && n == 16 && p[i]) {
      raw_load<DT, kVec>(p[i], raw[i]);
      if constexpr (kSilu) raw_load<DT, kVec>(p[i] + cols, raw_up[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    float v[16];
    bool unsure = false;
    if constexpr (kVec == 0) {
      // rows on any boundary: the warp reads them side by side and passes
      // them on in shared memory (16 columns a lane, a gap after each)
      const int64_t srow = src_of(row0 + warp + kQWarps * i);
      load_row<DT>(srow < 0 ? nullptr : x + srow * ld + col0, cols - col0, sx[warp], v);
      if constexpr (kSilu) {
        float u[16], least = 0.0f;
        load_row<DT>(srow < 0 ? nullptr : x + srow * ld + cols + col0, cols - col0, sx[warp], u);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          least = fminf(least, v[j]);
          v[j] = silu_mul_f32(v[j], u[j]);
        }
        unsure = least < -80.0f;
      }
    } else if (!p[i]) {
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = 0.0f;
    } else {
      if (kVec && n == 16)
        raw_unpack<DT>(raw[i], v);
      else
        load16<DT>(p[i], n, v);
      if constexpr (kSilu) {
        float u[16], least = 0.0f;
        if (kVec && n == 16)
          raw_unpack<DT>(raw_up[i], u);
        else
          load16<DT>(p[i] + cols, n, u);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          least = fminf(least, v[j]);
          v[j] = silu_mul_f32(v[j], u[j]);
        }
        unsure = least < -80.0f;  // exp(-gate) nears the end of float32
      }
    }
    uint32_t sbyte;
    uint2 c = encode16<DT, kMX, kSilu>(v, g, unsure, sbyte);
    const int r = warp + kQWarps * i;
    if constexpr (kSilu) {
      for (uint32_t todo = __ballot_sync(0xFFFFFFFFu, unsure); todo;) {
        const int owner = __ffs(todo) - 1;
        todo &= ~((kMX ? 3u : 1u) << owner);  // mxfp4: both lanes of a block are marked, the even one comes first
        encode_block_f64<DT, kMX>(x + (row0 + r) * ld, cols, col0 + 16 * owner, g, owner, c, sbyte);
      }
    }
    *reinterpret_cast<uint2*>(sc + (lane >> 1) * kPitch + r * 16 + (lane & 1) * 8) = c;
    uint8_t* s8 = reinterpret_cast<uint8_t*>(ss);
    if (kMX) {
      if ((lane & 1) == 0) s8[((lane >> 3) * kRows + r) * 4 + ((lane >> 1) & 3)] = (uint8_t)sbyte;
    } else {
      s8[((lane >> 2) * kRows + r) * 4 + (lane & 3)] = (uint8_t)sbyte;
    }
  }
  __syncthreads();
  const int left = (int)min((int64_t)kRows, rows - row0);
  uint8_t* dst = codes + ((int64_t)(col0 / 32) * rows + row0) * 16;
  const int nch = min(kQChunks, (kp - col0) / 32);
#pragma unroll
  for (int t = threadIdx.x; t < kQChunks * kRows; t += 32 * kQWarps) {
    const int ch = t / kRows, r = t % kRows;
    if (ch < nch && r < left)
      *reinterpret_cast<uint4*>(dst + ((int64_t)ch * rows + r) * 16) =
          *reinterpret_cast<const uint4*>(sc + ch * kPitch + r * 16);
  }
  uint32_t* sdst = scales + (int64_t)(col0 / kWordCols) * rows + row0;
#pragma unroll
  for (int t = threadIdx.x; t < kWords * kRows; t += 32 * kQWarps) {
    const int w = t / kRows, r = t % kRows;
    if (w * kWordCols < kp - col0 && r < left) sdst[(int64_t)w * rows + r] = ss[t];
  }
}

// Largest finite |silu(g) * u| of a warp's values, each rounded once to
// float32 (top: its bits).  Only values within 2^-16 of the largest seen so
// far are computed in float64: both this value and `run`, that largest in the
// float32 form, are off by less than 2^-17.  For gates below -80 the float32 form ends;
// |u| * 1.5e-33 is more than |silu(g) * u| there.
template <int N>
__device__ __forceinline__ void silu_top(const float (&g)[N], const float (&u)[N], uint32_t& run, uint32_t& top) {
  float h[N], most = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const bool far = g[j] < -80.0f;
    h[j] = far ? fabsf(u[j]) * 1.5e-33f : fabsf(silu_mul_f32(g[j], u[j]));
    if (!far && h[j] < 3.4e38f) most = fmaxf(most, h[j]);
  }
  run = max(run, __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(most)));
  const float floor = __uint_as_float(run) * (1.0f - 2.0f * kSiluWin);
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (h[j] >= floor && h[j] > 0.0f) {
      const uint32_t b = __float_as_uint(fabsf((float)silu_mul_f64((double)g[j], (double)u[j])));
      if (b < 0x7F800000u) top = max(top, b);
    }
}

// g = max(max|x| / 2688, 2^-100) over the finite values: with it the largest
// block's scale is 448.  out[0]: g, out[1] and out[2]: the running maximum's
// bits and the CTAs that are done (zeroed before the launch).  The maximum
// does not depend on the order of the atomics.
template <int DT, bool kSilu, int kVec>
__global__ void __launch_bounds__(256)
    fp4_global_scale_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t ld, int64_t rows, int cols,
                            const typename Elem<DT>::T* __restrict__ tail, int ntail, float* out) {
  uint32_t top = 0, run = 0;
  if (blockIdx.x == 0)  // what a matrix read as one long row leaves over
    for (int c = threadIdx.x; c < ntail; c += 256) {
      const uint32_t b = __float_as_uint(Elem<DT>::f(tail[c])) & 0x7FFFFFFFu;
      top = max(top, b < 0x7F800000u ? b : 0u);
    }
  if constexpr (kVec == 0) {  // rows on any boundary: columns side by side
    const int stretches = (cols + 2047) / 2048;
    const int64_t drow = gridDim.x / stretches;
    const int dst = gridDim.x % stretches;
    int64_t row = blockIdx.x / stretches;
    for (int st = blockIdx.x % stretches; row < rows;) {
      const int c0 = st * 2048 + threadIdx.x;
      const typename Elem<DT>::T* p = x + row * ld;
      float v[8], u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = c0 + 256 * j;
        v[j] = c < cols ? Elem<DT>::f(p[c]) : 0.0f;
        if constexpr (kSilu) u[j] = c < cols ? Elem<DT>::f(p[cols + c]) : 0.0f;
      }
      if constexpr (kSilu) {
        silu_top<8>(v, u, run, top);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t b = __float_as_uint(v[j]) & 0x7FFFFFFFu;
          top = max(top, b < 0x7F800000u ? b : 0u);
        }
      }
      row += drow, st += dst;
      if (st >= stretches) st -= stretches, ++row;
    }
  } else {
    constexpr int kDepth = 2;  // stretches of 16 columns in flight
    const int per_row = (cols + 15) / 16;
    const int64_t stride = (int64_t)gridDim.x * 256, first = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t srow = stride / per_row;
    const int scol = (int)(stride - srow * per_row);
    int64_t row = first / per_row;
    int c = (int)(first - row * per_row);
    while (__any_sync(0xFFFFFFFFu, row < rows)) {  // the warp stays together
      Raw<DT> raw[kDepth], raw_up[kSilu ? kDepth : 1];
      const typename Elem<DT>::T* p[kDepth];
      int n[kDepth];
#pragma unroll
      for (int i = 0; i < kDepth; ++i) {
        n[i] = row < rows ? min(16, cols - 16 * c) : 0;
        p[i] = x + row * ld + 16 * c;
        if (n[i] == 16) {
          raw_load<DT, kVec>(p[i], raw[i]);
          if constexpr (kSilu) raw_load<DT, kVec>(p[i] + cols, raw_up[i]);
        }
        row += srow, c += scol;
        if (c >= per_row) c -= per_row, ++row;
      }
#pragma unroll
      for (int i = 0; i < kDepth; ++i) {
        float v[16];
        if (n[i] == 16)
          raw_unpack<DT>(raw[i], v);
        else
          load16<DT>(p[i], n[i], v);
        if constexpr (kSilu) {
          float u[16];
          if (n[i] == 16)
            raw_unpack<DT>(raw_up[i], u);
          else
            load16<DT>(p[i] + cols, n[i], u);
          silu_top<16>(v, u, run, top);
          continue;
        }
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; j += 2) most = max3_abs(most, v[j], v[j + 1]);
        if (__float_as_uint(most) < 0x7F800000u) {
          top = max(top, __float_as_uint(most));
        } else {  // something is not finite: value by value
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const uint32_t b = __float_as_uint(v[j]) & 0x7FFFFFFFu;
            top = max(top, b < 0x7F800000u ? b : 0u);
          }
        }
      }
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

// FP4 layout -> q * s * g, [rows][ld]; the product q * s is exact (for nvfp4
// in float16 too: 6 bits, 2^-10 .. 2688).
template <int DT, bool kMX, bool kVec, int kPer>
__global__ void __launch_bounds__(32 * kQWarps)
    fp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint32_t* __restrict__ scales,
                          const float* __restrict__ gptr, typename Elem<DT>::T* __restrict__ out, int64_t ld,
                          int64_t rows, int cols, int kp) {
  constexpr int kRows = kQWarps * kPer, kPitch = q_pitch(kRows);
  constexpr int kWordCols = kMX ? 128 : 64, kWords = kQCols / kWordCols;
  __shared__ alignas(16) uint8_t sc[kQChunks * kPitch];
  __shared__ uint32_t ss[kWords * kRows];
  __shared__ alignas(16) typename Elem<DT>::T sx[kVec ? 1 : kQWarps][kVec ? 8 : 256];
  const int64_t row0 = (int64_t)blockIdx.x * kRows;
  const int col0 = blockIdx.y * kQCols;
  const float g = kMX || !gptr ? 1.0f : __ldg(gptr);
  const int left = (int)min((int64_t)kRows, rows - row0);
  {
    const uint8_t* src = codes + ((int64_t)(col0 / 32) * rows + row0) * 16;
    const int nch = min(kQChunks, (kp - col0) / 32);
#pragma unroll
    for (int t = threadIdx.x; t < kQChunks * kRows; t += 32 * kQWarps) {
      const int ch = t / kRows, r = t % kRows;
      if (ch < nch && r < left)
        *reinterpret_cast<uint4*>(sc + ch * kPitch + r * 16) =
            __ldg(reinterpret_cast<const uint4*>(src + ((int64_t)ch * rows + r) * 16));
    }
    const uint32_t* ssrc = scales + (int64_t)(col0 / kWordCols) * rows + row0;
#pragma unroll
    for (int t = threadIdx.x; t < kWords * kRows; t += 32 * kQWarps) {
      const int w = t / kRows, r = t % kRows;
      if (w * kWordCols < kp - col0 && r < left) ss[t] = __ldg(ssrc + (int64_t)w * rows + r);
    }
  }
  __syncthreads();
  // A lane writes 16 bytes at a time, the warp 512 contiguous ones: kCols
  // columns of a stretch of 32 * kCols, stretch after stretch.
  constexpr int kCols = DT == BLUT_F32 ? 4 : 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint8_t* s8 = reinterpret_cast<const uint8_t*>(ss);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = warp + kQWarps * i;
    if (r >= left) break;
    typename Elem<DT>::T* p = out + (row0 + r) * ld + col0;
#pragma unroll
    for (int k = 0; k < kQCols / (32 * kCols); ++k) {
      const int c = k * 32 * kCols + lane * kCols, n = cols - col0 - c;  // column inside the 512
      if (kVec ? n <= 0 : cols - col0 - k * 32 * kCols <= 0) break;
      const int blk = c / (kMX ? 32 : 16);
      const float s = fp4_scale_f32<kMX>(s8[((blk >> 2) * kRows + r) * 4 + (blk & 3)]);
      uint32_t cw = *reinterpret_cast<const uint32_t*>(sc + (c >> 5) * kPitch + r * 16 + ((c & 31) >> 3) * 4);
      if (kCols == 4) cw >>= 4 * (c & 4);
      uint32_t q[4], o[4];
      e2m1x8_f16(cw, q);
      const __half2 sh = __float2half2_rn(kMX ? 0.0f : s);
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) {
        __half2 h = *reinterpret_cast<const __half2*>(&q[j]);
        if constexpr (!kMX) h = __hmul2(h, sh);
        float2 f = __half22float2(h);
        if constexpr (kMX) {
          f.x *= s, f.y *= s;
        } else {
          f.x *= g, f.y *= g;
        }
        if constexpr (DT == BLUT_F32) {
          o[2 * j] = __float_as_uint(f.x);
          o[2 * j + 1] = __float_as_uint(f.y);
        } else if constexpr (DT == BLUT_BF16) {
          const __nv_bfloat162 b = __float22bfloat162_rn(f);
          o[j] = *reinterpret_cast<const uint32_t*>(&b);
        } else {
          const __half2 b = __float22half2_rn(f);
          o[j] = *reinterpret_cast<const uint32_t*>(&b);
        }
      }
      if constexpr (kVec) {
        if (n >= kCols) {
          *reinterpret_cast<uint4*>(p + c) = make_uint4(o[0], o[1], o[2], o[3]);
        } else {
#pragma unroll
          for (int j = 0; j < kCols; ++j) {
            if (j >= n) break;
            if constexpr (DT == BLUT_F32)
              p[c + j] = __uint_as_float(o[j]);
            else
              p[c + j] = (uint16_t)(o[j / 2] >> (16 * (j & 1)));
          }
        }
      } else {  // rows on any boundary: a lane's values side by side first
        typename Elem<DT>::T* buf = sx[warp];
        __syncwarp();
        *reinterpret_cast<uint4*>(buf + lane * kCols) = make_uint4(o[0], o[1], o[2], o[3]);
        __syncwarp();
        const int c1 = k * 32 * kCols, left1 = cols - col0 - c1;
#pragma unroll
        for (int j = 0; j < kCols; ++j)
          if (32 * j + lane < left1) p[c1 + 32 * j + lane] = buf[32 * j + lane];
      }
    }
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

// Boundary that p, and p plus multiples of the two byte distances, start on: 32, 16 or 0.
inline int alignment(const void* p, int64_t a, int64_t b) {
  const uint64_t all = (uint64_t)(uintptr_t)p | (uint64_t)a | (uint64_t)b;
  return all % 32 == 0 ? 32 : all % 16 == 0 ? 16 : 0;
}
inline int64_t elem_size(int dtype) { return dtype == BLUT_F32 ? 4 : 2; }
inline int launched() { return cudaGetLastError() == cudaSuccess ? BLUT_OK : BLUT_ERR_LAUNCH; }

// Rows a warp takes: several once that still leaves every SM a few CTAs, one
// below.  nvfp4 of bf16 rows x 2048, one against several: 32 rows 1.7 against
// 3.1 us, 4096 (below the border) 7.8 against 8.2, 8192 (above) 13.4 against
// 12.4, 32768 45.0 against 36.1; the way back 1.9 against 2.5, 7.2 against 5.8,
// 13.1 against 8.2, 45.0 against 30.5.
inline bool many_rows(int64_t rows, int kp) {
  return rows * ((kp + kQCols - 1) / kQCols) >= 148ll * 4 * 4 * kQWarps;
}

template <int DT, bool kMX, bool kSilu, int kVec, int kPer>
void launch_quantize_as(const blut_fp4_desc& d, const void* x, int64_t ld, const int32_t* row_index, int64_t src_rows,
                        const float* g, void* codes, void* scales, int signal, int kp, cudaStream_t stream) {
  const dim3 grid((unsigned)((d.rows + kPer * kQWarps - 1) / (kPer * kQWarps)), (unsigned)((kp + kQCols - 1) / kQCols));
  fp4_quantize_kernel<DT, kMX, kSilu, kVec, kPer><<<grid, 32 * kQWarps, 0, stream>>>(
      static_cast<const typename Elem<DT>::T*>(x), ld, row_index, src_rows, g, d.rows, (int)d.cols, kp,
      static_cast<uint8_t*>(codes), static_cast<uint32_t*>(scales), signal);
}

template <int DT, bool kSilu>
int launch_quantize(const blut_fp4_desc& d, const void* x, int64_t ld, const int32_t* row_index, int64_t src_rows,
                    const float* g, void* codes, void* scales, int signal, cudaStream_t stream) {
  const int64_t es = sizeof(typename Elem<DT>::T);
  const int vec = alignment(x, ld * es, kSilu ? d.cols * es : 0);
  const int kp = fp4_kblocks(d.cols) * kFp4BlockCols;
  // Four CTAs per SM, and the rows that their 64 registers hold: nvfp4 of
  // 32768 x 2048 bf16 takes 36.1 us with 4 rows (3 CTAs: 37.9, 2 rows: 39.9,
  // one: 44.9), mxfp4 31.2 (33.4, 33.7, 36.5); float32 52.6 with 2 (3 CTAs:
  // 55.9, one row: 54.5, 4 rows: 84.5); the SiLU form of 196608 x 1408, mxfp4
  // fp16, 238 with 2 (3 CTAs: 265, one row: 280, 4 rows: 293).  Rows on other
  // than 16-byte boundaries take one row a warp whatever their number: 20000 x
  // 2319 bf16 42.5 us (nvfp4) and 38.8 (mxfp4) against 41.3 and 37.9 with 4,
  // too little for another set of kernels.
  constexpr int kMany = kSilu || DT == BLUT_F32 ? 2 : 4;
  const bool many = many_rows(d.rows, kp);
#define BLUT_Q(MX, VEC, PER) \
  launch_quantize_as<DT, MX, kSilu, VEC, PER>(d, x, ld, row_index, src_rows, g, codes, scales, signal, kp, stream)
#define BLUT_V(MX)                                                                                      \
  if (vec == 32) { if (many) BLUT_Q(MX, 32, kMany); else BLUT_Q(MX, 32, 1); }                             \
  else if (vec == 16) { if (many) BLUT_Q(MX, 16, kMany); else BLUT_Q(MX, 16, 1); }                        \
  else BLUT_Q(MX, 0, 1)
  if (d.kind == BLUT_FP4_MX) {
    BLUT_V(true);
  } else {
    BLUT_V(false);
  }
#undef BLUT_V
#undef BLUT_Q
  return launched();
}

int quantize(const blut_fp4_desc* d, const void* x, int32_t dtype, int64_t ld, const int32_t* row_index,
             int64_t src_rows, const float* g, void* codes, void* scales, bool silu, bool signal,
             cudaStream_t stream) {
  if (!d || !fp4_valid(*d) || !x || !codes || !scales || ld < (silu ? 2 : 1) * d->cols || src_rows <= 0)
    return BLUT_ERR_INVALID;
  if (!row_index && src_rows != d->rows) return BLUT_ERR_INVALID;
  if (d->kind == BLUT_FP4_NV && !g) return BLUT_ERR_INVALID;
  if (((uintptr_t)codes | (uintptr_t)scales) % 16 != 0 || (uintptr_t)x % elem_size(dtype) != 0) return BLUT_ERR_INVALID;
#define BLUT_Q(DT)                                                                                            \
  return silu ? launch_quantize<DT, true>(*d, x, ld, row_index, src_rows, g, codes, scales, signal, stream)   \
              : launch_quantize<DT, false>(*d, x, ld, row_index, src_rows, g, codes, scales, signal, stream)
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
  int vec = alignment(x, ld * es, silu ? cols * es : 0);
  const T *p = static_cast<const T*>(x), *tail = p;
  int ntail = 0;
  if (!silu && vec == 0 && (rows == 1 || ld == cols) && (uintptr_t)x % 16 == 0 && rows * cols >= 4096) {
    // rows without gaps: their boundaries do not matter to a maximum
    const int64_t total = rows * cols;
    rows = total / 4096;
    cols = ld = 4096;
    ntail = (int)(total - rows * 4096);
    tail = p + rows * 4096;
    vec = alignment(x, ld * es, 0);
  }
  const int64_t ctas = (rows * ((cols + 15) / 16) + 255) / 256;
  const unsigned grid = (unsigned)std::min<int64_t>(ctas, 148 * 5);  // one round of CTAs
#define BLUT_G(SILU, VEC) \
  fp4_global_scale_kernel<DT, SILU, VEC><<<grid, 256, 0, stream>>>(p, ld, rows, (int)cols, tail, ntail, out)
  if (silu) {
    if (vec == 32) BLUT_G(true, 32); else if (vec == 16) BLUT_G(true, 16); else BLUT_G(true, 0);
  } else {
    if (vec == 32) BLUT_G(false, 32); else if (vec == 16) BLUT_G(false, 16); else BLUT_G(false, 0);
  }
#undef BLUT_G
  return launched();
}

template <int DT, bool kMX, bool kVec, int kPer>
void launch_dequantize_as(const blut_fp4_desc& d, const void* codes, const void* scales, const float* g, void* out,
                          int64_t ld, int kp, cudaStream_t stream) {
  const dim3 grid((unsigned)((d.rows + kPer * kQWarps - 1) / (kPer * kQWarps)),
                  (unsigned)((d.cols + kQCols - 1) / kQCols));
  fp4_dequantize_kernel<DT, kMX, kVec, kPer><<<grid, 32 * kQWarps, 0, stream>>>(
      static_cast<const uint8_t*>(codes), static_cast<const uint32_t*>(scales), g,
      static_cast<typename Elem<DT>::T*>(out), ld, d.rows, (int)d.cols, kp);
}

template <int DT>
int launch_dequantize(const blut_fp4_desc& d, const void* codes, const void* scales, const float* g, void* out,
                      int64_t ld, cudaStream_t stream) {
  const bool vec = alignment(out, ld * (int64_t)sizeof(typename Elem<DT>::T), 0) != 0;
  const int kp = fp4_kblocks(d.cols) * kFp4BlockCols;
  const bool many = many_rows(d.rows, kp);
#define BLUT_D(MX, VEC, PER) launch_dequantize_as<DT, MX, VEC, PER>(d, codes, scales, g, out, ld, kp, stream)
  if (d.kind == BLUT_FP4_MX) {
    if (!vec) BLUT_D(true, false, 1); else if (many) BLUT_D(true, true, 4); else BLUT_D(true, true, 1);
  } else {
    if (!vec) BLUT_D(false, false, 1); else if (many) BLUT_D(false, true, 4); else BLUT_D(false, true, 1);
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

int fp4_quantize_for_product(const blut_fp4_desc& d, const void* x, int32_t dtype, int64_t ld, const float* g,
                             void* codes, void* scales, cudaStream_t stream) {
  return quantize(&d, x, dtype, ld, nullptr, d.rows, g, codes, scales, false, true, stream);
}

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
  return quantize(d, x, dtype, ld, row_index, src_rows, global_scale, codes, scales, false, false, S(stream));
}

int blut_fp4_silu_mul_quantize(const blut_fp4_desc* d, const void* gate_up, int32_t dtype, int64_t ld,
                               const float* global_scale, void* codes, void* scales, void* stream) {
  return quantize(d, gate_up, dtype, ld, nullptr, d ? d->rows : 0, global_scale, codes, scales, true, false,
                  S(stream));
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
