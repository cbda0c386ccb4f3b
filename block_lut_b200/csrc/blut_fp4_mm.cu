// Products of 4-bit microscaled matrices on the block-scaled tensor cores
// (blut_fp4_matmul): y[t] = W x_t for all rows of x, or for runs of rows with
// one W per run.
//
//   y[t][n] = g_x g_w sum_k (q s)_w[n][k] (q s)_x[t][k],  float32 sums
//
// A work item is a tile of 128 weight rows x NT tokens (D^T: weight rows are
// tensor-memory lanes, tokens are columns, so that a few tokens cost a narrow
// MMA and not a padded one).  A CTA takes items in turn, or shares one with
// the CTAs of its cluster (split K).  Per 128 columns of K:
//
//  * warp 0 fetches the tile's unit - 8 KB of codes and the scales of 128
//    rows, contiguous - with one bulk copy, and the tokens' codes with four
//    (a run of rows is contiguous per 32 columns);
//  * warps 2, 3 copy the tokens' scales, word by word, into the order that
//    tcgen05.cp reads: they are the one operand whose position in a tile
//    depends on where the run of rows starts;
//  * warp 1 copies both scales to tensor memory (tcgen05.cp, 32x128b,
//    replicated to the four lane quarters) and issues two tcgen05.mma of
//    K = 64, kind::mxf4nvf4 (a scale per 16) or kind::mxf4 (a scale per 32),
//    M = 128, N = the tile's tokens rounded to 16;
//  * the warps from 4 on turn a finished accumulator into rows of y, a lane
//    quarter each, while the others run ahead into the next item.
//
// Where there are few tiles, a cluster of 2, 4 or 8 CTAs splits K: each leaves
// its partial tile in its shared memory and sums a share of the tokens over
// the cluster in rank order, so the result is the same in every run and no
// workspace is needed.
//
// Every wait is bounded; one that runs out raises the CTA's abort flag and
// the device status, and every role then leaves its loop, lets what it has in
// flight land, and frees the tensor memory.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "blut_fp4.cuh"
#include "blut_mm.cuh"
#include "blut_tc.cuh"

namespace blut {
namespace {

__device__ int g_fp4_status;

constexpr int kEpiWarp0 = 4;   // first epilogue warp
constexpr int kEpiStage = 2048;  // bytes an epilogue warp transposes in: 32 tokens x 32 rows of 16 bits
constexpr int kHeader = 1024;  // barriers and flags
constexpr int kFuseRows = 8;   // most rows that the product quantises itself

template <bool kMX, int NT>
struct Fp4Cfg {
  static constexpr int kWords = kMX ? 1 : 2;           // scale words per 128 columns
  static constexpr int kGroups = (NT + 127) / 128;     // 128-token groups of the scales
  static constexpr int kA = kFp4UnitCodes + 512 * kWords;
  static constexpr int kB = NT * 64;
  static constexpr int kSB = 512 * kWords * kGroups;
  static constexpr int kStage = kA + kB + kSB;
  // Two CTAs per SM (three for few tokens) keep copies in flight while one of
  // them starts or stores.
  static constexpr int kCtas = NT <= 64 ? 3 : 2;
  // Epilogue warps per lane quarter: two where an item has many tokens, since
  // the accumulator is not free for the next item before it is read.
  static constexpr int kEpi = NT > 128 ? 2 : 1;
  static constexpr int kThreads = 32 * (kEpiWarp0 + 4 * kEpi);
  static constexpr int kFixed = kHeader + 4 * kEpi * kEpiStage;
  static constexpr int kStages = ((kCtas == 3 ? 73 * 1024 : 112 * 1024) - kFixed) / kStage;
  static constexpr int kSmem = kFixed + kStages * kStage;  // and the table of runs, launch()
  // Tensor memory: NT accumulator columns, then slots of scales; a slot holds
  // one block, 4 columns per word for the weights and for each token group.
  static constexpr int kCols = NT <= 64 ? 128 : 256;
  static constexpr int kWordCols = 4 + 4 * kGroups;
  static constexpr int kSlotCols = kWords * kWordCols;
  static constexpr int kSlots = (kCols - NT) / kSlotCols < kStages ? (kCols - NT) / kSlotCols : kStages;
  static_assert(kStages >= 2 && kStages <= 8 && kSlots >= 2, "ring");
};

struct Fp4Params {
  const uint8_t* w;
  int64_t wstride;
  const float* wg;
  const int32_t* offsets;
  int experts;
  const uint8_t* xc;
  const uint32_t* xs;
  const float* xg;
  int64_t x_rows;
  const void* x;    // kFuse: x before quantisation, its row pitch in elements,
  int64_t x_ld;     // columns, and whether its rows start on 16-byte boundaries
  int cols, x_vec;
  int n;        // weight rows
  int kblocks;  // 128-column blocks
  int row_tiles;
  int token_tiles;  // one matrix: their number
  int tn;           // tokens of an item, at most NT
  int split_log;    // log2 of the CTAs of a cluster along K
  void* y;
  int64_t ldy;
  int out_dtype;
  int vec;      // rows of y start on 16-byte boundaries
  int tma;      // y is described by the kernel's tensor map
  uint64_t wait_ns;
};

struct Fp4Header {
  uint64_t wfull[8], sfull[8], empty[8], acc_full, acc_empty, fin;
  uint32_t tmem;
  int abort_flag;
  int items;
};
static_assert(sizeof(Fp4Header) <= kHeader, "header");

// One work item: tokens row0 .. row0 + cnt - 1 of x, weight rows 128 tile ..
struct Fp4Item {
  int expert, row0, cnt, tile;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_peer4(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\t"
      "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
}
// Waits until the kernels before this one on the stream are complete (a
// launch that may begin before that, see launch()); otherwise does nothing.
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// One lane of a converged warp; the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// Low word of the no-swizzle K-major descriptor (tc_desc) of a shared
// address, whose bits from 18 up may name the CTA in its cluster, in two
// parts: the stage's, and what an operand inside it adds; the high word is
// constant.
__device__ __forceinline__ uint32_t desc_base(uint32_t saddr) { return (saddr >> 4) & 0x3FFFu; }
__device__ __forceinline__ constexpr uint32_t desc_add(uint32_t offset, uint32_t lbo) {
  return (offset >> 4) + ((lbo >> 4) << 16);
}
constexpr uint32_t kDescHi = (128u >> 4) | (1u << 14);  // 128 bytes between 8-row groups, version 1

// 32 rows x 16 bytes of shared memory to 4 columns of all four lane quarters.
__device__ __forceinline__ void cp_scales(uint32_t taddr, uint32_t lo) {
  asm volatile(
      "{\n\t.reg .b64 s;\n\tmov.b64 s, {%1, %2};\n\ttcgen05.cp.cta_group::1.32x128b.warpx4 [%0], s;\n\t}" ::"r"(taddr),
      "r"(lo), "n"(kDescHi)
      : "memory");
}

template <bool kMX>
__device__ __forceinline__ void mma_fp4(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                        uint32_t acc) {
  if constexpr (kMX) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "mov.b64 a, {%1, %7};\n\tmov.b64 b, {%2, %7};\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc), "n"(kDescHi)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "mov.b64 a, {%1, %7};\n\tmov.b64 b, {%2, %7};\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], a, b, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc), "n"(kDescHi)
        : "memory");
  }
}

// Instruction descriptor: A and B e2m1 K-major, M = 128, N = n, scales e4m3
// or e8m0; mxfp4's scale word holds the scales of two MMAs, bytes 0-1 and 2-3.
template <bool kMX>
__device__ __forceinline__ uint32_t idesc_fp4(int n, int step) {
  const uint32_t id = kMX ? 2u * step : 0u;
  return (id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((kMX ? 1u : 0u) << 23) | (1u << 27) |
         (id << 29);
}

// The runs' first rows and the number of token tiles before each run, tab[e]
// and tab[E + 1 + e], e = 0 .. E, by one warp; returns the number of tiles.  A
// run is cut into ceil(rows / tn) tiles.  Offsets are clamped to [0, x_rows],
// so none leads out of the buffers.
__device__ int table_of_runs(const Fp4Params& p, int lane, int* tab) {
  int before = 0;
  for (int e0 = 0; e0 < p.experts; e0 += 128) {  // four runs per lane
    int o[5], tiles = 0;
#pragma unroll
    for (int j = 0; j < 5; ++j) {
      const int e = min(e0 + 4 * lane + j, p.experts);
      o[j] = (int)min((int64_t)max(p.offsets[e], 0), p.x_rows);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) tiles += (max(o[j + 1] - o[j], 0) + p.tn - 1) / p.tn;
    int incl = tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, incl, d);
      if (lane >= d) incl += v;
    }
    int t = before + incl - tiles;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = e0 + 4 * lane + j;
      if (e < p.experts) {
        tab[e] = o[j];
        tab[p.experts + 1 + e] = t;
        t += (max(o[j + 1] - o[j], 0) + p.tn - 1) / p.tn;
        if (e == p.experts - 1) tab[p.experts] = o[j + 1], tab[2 * p.experts + 1] = t;
      }
    }
    before += __shfl_sync(0xFFFFFFFFu, incl, 31);
  }
  return before;
}

// Item `i`, by a converged warp: row tiles of one token tile follow each other.
__device__ __forceinline__ Fp4Item item_of(const Fp4Params& p, int i, int lane, const int* tab) {
  Fp4Item t;
  const int y = i / p.row_tiles;
  t.tile = i - y * p.row_tiles;
  if (p.experts) {
    const int* first = tab + p.experts + 1;
    int e = -1;  // the last run that starts at or before tile y has it: runs without tiles start where the next does
    for (int e0 = 0; e0 < p.experts; e0 += 32)
      e += __popc(__ballot_sync(0xFFFFFFFFu, e0 + lane < p.experts && first[min(e0 + lane, p.experts)] <= y));
    t.expert = e;
    const int in = (y - first[e]) * p.tn, cnt = tab[e + 1] - tab[e];
    t.row0 = tab[e] + in;
    t.cnt = min(p.tn, cnt - in);
  } else {
    t.expert = 0;
    t.row0 = y * p.tn;
    t.cnt = (int)min((int64_t)p.tn, p.x_rows - t.row0);
  }
  return t;
}

// Two values in a 16-bit type, the first in the low half.
template <int kOut>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (kOut == BLUT_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
__device__ __forceinline__ void store1(const Fp4Params& p, int64_t token, int64_t row, float v) {
  if (row >= p.n) return;
  const int64_t i = token * p.ldy + row;
  if (p.out_dtype == BLUT_F32)
    static_cast<float*>(p.y)[i] = v;
  else
    static_cast<uint16_t*>(p.y)[i] = p.out_dtype == BLUT_BF16 ? f32_to_act<true>(v) : f32_to_act<false>(v);
}
// Rows row .. row + 3 (row % 4 == 0) of one token.
__device__ __forceinline__ void store4(const Fp4Params& p, int64_t token, int64_t row, float4 v) {
  if (p.vec && row + 4 <= p.n) {
    const int64_t i = token * p.ldy + row;
    if (p.out_dtype == BLUT_F32)
      *reinterpret_cast<float4*>(static_cast<float*>(p.y) + i) = v;
    else
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.y) + i) =
          p.out_dtype == BLUT_BF16 ? make_uint2(pack2<BLUT_BF16>(v.x, v.y), pack2<BLUT_BF16>(v.z, v.w))
                                   : make_uint2(pack2<BLUT_F16>(v.x, v.y), pack2<BLUT_F16>(v.z, v.w));
  } else {
    store1(p, token, row, v.x);
    store1(p, token, row + 1, v.y);
    store1(p, token, row + 2, v.z);
    store1(p, token, row + 3, v.w);
  }
}

// 16 lanes (from the address's lane) x 32 columns of 32 bits, in the layout
// of an mma accumulator: register 4c + 2h + j of a thread is lane
// l / 4 + 8 h, column 8 c + 2 (l % 4) + j.
__device__ __forceinline__ void tc_ld_16x32(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}

// Bulk tensor store of a warp's stage, 32 tokens x 32 rows of the matrix, to
// y at (row, token); tokens past y are not written.
__device__ __forceinline__ void store_box(const CUtensorMap* map, uint32_t saddr, int row, int token) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];\n\t"
               "cp.async.bulk.commit_group;" ::"l"(map),
               "r"(row), "r"(token), "r"(saddr)
               : "memory");
}

// An epilogue warp's 32 weight rows x cnt tokens as 16-bit rows of y: pairs
// of tokens are packed as an mma accumulator holds them and stmatrix
// transposes 8 x 8 of them at a time into rows of 64 bytes per token, whose
// 16-byte pieces are swapped about against bank conflicts (and as a tensor
// map with 64-byte swizzle expects them).  From there a full stretch of 32
// tokens leaves as one bulk tensor store (map not null); a stretch that ends
// inside, or a y without a map, as stores of 32 rows of 8 tokens, 16 bytes a
// lane; rows on other boundaries, or a partial tile, 2 bytes a lane, a
// token's rows side by side.  Plain stores alone kept the accumulator for
// 4500 cycles of an item of 16 000 (128 x 192, K = 2048).  y: token 0, the warp's first row `row`,
// of which `left` are rows of the matrix; vec: rows of y start on 16-byte
// boundaries; c0, cstep: the warp's stretches; pending: a bulk store of this
// or an earlier item (whose row tile may have been a full one where this one
// is cut) may still be reading the stage; read: called once the accumulator
// has been read.
template <int kOut, class Read>
__device__ __forceinline__ void store_tile16(uint32_t tcol, int cnt, float alpha, uint8_t* stage, uint16_t* y,
                                             int64_t ldy, int left, bool vec, int lane, int c0, int cstep,
                                             const CUtensorMap* map, bool pending, int row, int token0, int rows_in_y,
                                             Read read) {
  const uint32_t saddr = smem_u32(stage);
  if (c0 >= cnt) read();
#pragma unroll 1
  for (int c = c0; c < cnt; c += cstep) {
    uint32_t v[2][16], w[4][4];
    tc_ld_16x32(tcol + c, v[0]);
    tc_ld_16x32(tcol + c + (16u << 16), v[1]);
    tc_wait_ld16(v[0]);
    tc_wait_ld16(v[1]);
    if (c + cstep >= cnt) read();
#pragma unroll
    for (int tg = 0; tg < 4; ++tg)  // 8 tokens x 32 rows: four 8 x 8 matrices
#pragma unroll
      for (int rg = 0; rg < 4; ++rg)
        w[tg][rg] = pack2<kOut>(__uint_as_float(v[rg >> 1][4 * tg + 2 * (rg & 1)]) * alpha,
                                __uint_as_float(v[rg >> 1][4 * tg + 2 * (rg & 1) + 1]) * alpha);
    if (pending) {  // not before the stage's last store has read it
      if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      __syncwarp();
    }
#pragma unroll
    for (int tg = 0; tg < 4; ++tg) {
      // lane 8 rg + i gives the address of token i, rows 8 rg .. 8 rg + 7
      const int t = 8 * tg + (lane & 7), piece = (lane >> 3) ^ ((t >> 1) & 3);
      asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(saddr + t * 64 +
                                                                                                 piece * 16),
                   "r"(w[tg][0]), "r"(w[tg][1]), "r"(w[tg][2]), "r"(w[tg][3])
                   : "memory");
    }
    // a box may reach past the item's tokens where y ends there too
    if (map && (c + 32 <= cnt || token0 + cnt == rows_in_y)) {
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) store_box(map, saddr, row, token0 + c);
      continue;
    }
    __syncwarp();
    if (vec && left == 32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = 8 * j + (lane >> 2);
        if (c + t < cnt)
          *reinterpret_cast<uint4*>(y + (int64_t)(c + t) * ldy + (lane & 3) * 8) =
              *reinterpret_cast<const uint4*>(stage + t * 64 + ((lane & 3) ^ ((t >> 1) & 3)) * 16);
      }
    } else if (lane < left) {  // a token's rows side by side, 2 bytes a lane
#pragma unroll 8
      for (int t = 0; t < min(32, cnt - c); ++t)
        y[(int64_t)(c + t) * ldy + lane] =
            *reinterpret_cast<const uint16_t*>(stage + t * 64 + ((lane >> 3) ^ ((t >> 1) & 3)) * 16 + (lane & 7) * 2);
    }
    __syncwarp();
  }
}

// This CTA's share of the tokens, summed over the cluster's partial tiles in
// rank order.  A thread takes 4 rows of a token; its loads are in flight
// together.
template <int S, int kThreads>
__device__ __forceinline__ void reduce_cluster(const Fp4Params& p, const float* part, int rank, int cnt, int64_t row0,
                                               int64_t col0, float alpha) {
  const int quad = 4 * (threadIdx.x & 31);
  for (int c = rank + S * (threadIdx.x >> 5); c < cnt; c += S * (kThreads / 32)) {
    const uint32_t a = smem_u32(part + c * 128 + quad);
    float4 v[S];
#pragma unroll
    for (int q = 0; q < S; ++q) v[q] = ld_peer4(a, q);
    float4 t = v[0];
#pragma unroll
    for (int q = 1; q < S; ++q) t.x += v[q].x, t.y += v[q].y, t.z += v[q].z, t.w += v[q].w;
    store4(p, row0 + c, col0 + quad, make_float4(t.x * alpha, t.y * alpha, t.z * alpha, t.w * alpha));
  }
}

// kFuse: 0, x comes in 4-bit form; 1 + dtype, warps 2, 3 quantise its (at
// most 8) rows themselves, 16 columns a lane and block: a launch and a pass
// through memory less, where a call is little else.
template <bool kMX, int NT, int kFuse>
__global__ void __launch_bounds__(Fp4Cfg<kMX, NT>::kThreads, Fp4Cfg<kMX, NT>::kCtas)
    fp4_mm_kernel(const __grid_constant__ Fp4Params p, const __grid_constant__ CUtensorMap ymap) {
  using C = Fp4Cfg<kMX, NT>;
  extern __shared__ __align__(1024) uint8_t fp4_smem[];
  Fp4Header* h = reinterpret_cast<Fp4Header*>(fp4_smem);
  uint8_t* ring = fp4_smem + kHeader;
  uint8_t* epi = ring + C::kStages * C::kStage;
  int* tab = reinterpret_cast<int*>(epi + 4 * C::kEpi * kEpiStage);
  volatile int* abort_flag = &h->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = 1 << p.split_log;
  const int rank = split > 1 ? (int)cluster_rank() : 0;
  const int first = blockIdx.x >> p.split_log, step = gridDim.x >> p.split_log;
  const int b0 = p.kblocks * rank >> p.split_log;  // this CTA's K range
  const int nb = (p.kblocks * (rank + 1) >> p.split_log) - b0;

  // Warp 0 sets the barriers up, lists the runs, and starts the first weight
  // copies at once, beside the tensor-memory allocation of warp 1.
  const auto bring_w = [&](const Fp4Item& t, int b, int it) {
    const int s = it % C::kStages;
    const uint32_t bar = smem_u32(h->wfull + s);
    mbar_expect_tx(bar, C::kA + (kFuse ? 0u : 4 * (uint32_t)t.cnt * 16));
    bulk_g2s(smem_u32(ring + s * C::kStage), p.w + t.expert * p.wstride + ((int64_t)t.tile * p.kblocks + b0 + b) * C::kA,
             C::kA, bar);
  };
  Fp4Item t0 = {0, 0, 0, 0};
  int started = 0;
  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < C::kStages; ++s) {
        mbar_init(smem_u32(h->wfull + s), 1);
        mbar_init(smem_u32(h->sfull + s), 2);
        mbar_init(smem_u32(h->empty + s), 1);
      }
      mbar_init(smem_u32(&h->acc_full), 1);
      mbar_init(smem_u32(&h->acc_empty), 4 * C::kEpi);
      mbar_init(smem_u32(&h->fin), 1);
      h->abort_flag = 0;
      fence_mbar_init();
    }
    const int tiles = p.experts ? table_of_runs(p, lane, tab) : p.token_tiles;
    if (lane == 0) h->items = tiles * p.row_tiles;
    __syncwarp();
    if (first < tiles * p.row_tiles) {
      t0 = item_of(p, first, lane, tab);
      started = min(nb, C::kStages);
      if (lane == 0)
        for (int b = 0; b < started; ++b) bring_w(t0, b, b);
    }
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&h->tmem)),
                 "r"(C::kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = h->tmem;
  const int items = h->items;

  if (warp == 0) {
    // ------------------------------------------------------------ producer --
    // Converged, like the MMA warp below, with one lane issuing: a copy issued
    // by a lone lane costs as much as the data it brings takes.
    if (first < items) {
      if (!kFuse) grid_dependency_wait();  // x may still be in the making; the weights are not
      const uint32_t ring_addr = smem_u32(ring), full_addr = smem_u32(h->wfull);
      const int64_t xstep = p.x_rows * 16;
      const bool leader = elect_one();
      int it = 0;  // blocks over all items: the ring goes on from one to the next
      bool ok = true;
      for (int i = first; i < items && ok; i += step) {
        const Fp4Item t = i == first ? t0 : item_of(p, i, lane, tab);
        const uint8_t* wsrc = p.w + t.expert * p.wstride + ((int64_t)t.tile * p.kblocks + b0) * C::kA;
        const uint8_t* xsrc = p.xc + ((int64_t)b0 * 4 * p.x_rows + t.row0) * 16;
        const uint32_t xbytes = (uint32_t)t.cnt * 16;
        for (int b = 0; b < nb; ++b, ++it, wsrc += C::kA) {
          const int s = it % C::kStages;
          if (it >= C::kStages) {
            ok = __all_sync(0xFFFFFFFFu, wait_or_abort(smem_u32(h->empty + s), (uint32_t)(it / C::kStages - 1) & 1u,
                                                       abort_flag, &g_fp4_status, p.wait_ns));
            if (!ok) break;
          }
          const uint32_t bar = full_addr + 8 * s, dst = ring_addr + s * C::kStage;
          if (leader) {
            if (it >= started) {
              mbar_expect_tx(bar, C::kA + (kFuse ? 0u : 4 * xbytes));
              bulk_g2s(dst, wsrc, C::kA, bar);
            }
            if (!kFuse) {
              bulk_g2s(dst + C::kA, xsrc, xbytes, bar);
              bulk_g2s(dst + C::kA + NT * 16, xsrc + xstep, xbytes, bar);
              bulk_g2s(dst + C::kA + 2 * NT * 16, xsrc + 2 * xstep, xbytes, bar);
              bulk_g2s(dst + C::kA + 3 * NT * 16, xsrc + 3 * xstep, xbytes, bar);
            }
          }
          __syncwarp();
          xsrc += 4 * xstep;
        }
      }
      // whatever the other roles do, no copy is in flight when the CTA ends
      if (lane == 0)
        for (int j = max(0, it - C::kStages); j < it; ++j)
          wait_drain(smem_u32(h->wfull + j % C::kStages), (uint32_t)(j / C::kStages) & 1u);
      __syncwarp();
    }
  } else if (warp == 1) {
    // ----------------------------------------------------------------- MMA --
    // The whole warp runs the loop, so that addresses and descriptors are
    // uniform values, and one lane issues; run by a single lane, the same
    // instructions took 75 cycles each to issue.  The barriers of a block
    // are polled by a lane each.
    const uint32_t tm = __shfl_sync(0xFFFFFFFFu, tmem, 0);
    const uint32_t ring_desc = desc_base(smem_u32(ring));
    const bool leader = elect_one();
    bool ok = true;
    int it = 0, acc = 0;
    for (int i = first; i < items && ok; i += step, ++acc) {
      const uint32_t n = (uint32_t)__shfl_sync(0xFFFFFFFFu, (item_of(p, i, lane, tab).cnt + 15) & ~15, 0);
      const uint32_t idesc0 = idesc_fp4<kMX>(n, 0), idesc1 = idesc_fp4<kMX>(n, 1);
      for (int b = 0; b < nb; ++b, ++it) {
        const int s = it % C::kStages;
        {
          const uint64_t* bar = lane == 1 ? h->sfull + s : h->wfull + s;
          uint32_t ph = (uint32_t)(it / C::kStages) & 1u;
          if (C::kSlots < C::kStages && lane == 2 && it >= C::kSlots) {
            // the MMAs that read this slot of scales are done
            const int j = it - C::kSlots;
            bar = h->empty + j % C::kStages;
            ph = (uint32_t)(j / C::kStages) & 1u;
          }
          if (lane == 3 && b == 0 && acc > 0) {  // the accumulator has been read
            bar = &h->acc_empty;
            ph = (uint32_t)(acc - 1) & 1u;
          }
          ok = __all_sync(0xFFFFFFFFu, wait_or_abort(smem_u32(bar), ph, abort_flag, &g_fp4_status, p.wait_ns));
        }
        if (!ok) break;
        __syncwarp();
        tc_fence_after();
        const uint32_t st = ring_desc + s * (C::kStage >> 4);
        const uint32_t slot = tm + NT + (it % C::kSlots) * C::kSlotCols;
        if (leader) {
#pragma unroll
          for (int w = 0; w < C::kWords; ++w) {
            cp_scales(slot + w * C::kWordCols, st + desc_add(kFp4UnitCodes + 512 * w, 512));
#pragma unroll
            for (int g = 0; g < C::kGroups; ++g)
              cp_scales(slot + w * C::kWordCols + 4 + 4 * g,
                        st + desc_add(C::kA + C::kB + 512 * (w * C::kGroups + g), 512));
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t sc = slot + (kMX ? 0 : k * C::kWordCols);
            mma_fp4<kMX>(tm, st + desc_add(k * 4096, 2048), st + desc_add(C::kA + k * 2 * NT * 16, NT * 16),
                         k ? idesc1 : idesc0, sc, sc + 4, (uint32_t)(b | k));
          }
          tc_commit(smem_u32(h->empty + s));
          if (b == nb - 1) tc_commit(smem_u32(&h->acc_full));
        }
        __syncwarp();
      }
    }
    if (!ok && it > 0 && leader) {  // gave up: let the MMAs issued so far finish
      tc_commit(smem_u32(&h->fin));
      wait_drain(smem_u32(&h->fin), 0);
    }
    __syncwarp();
  } else if (kFuse && warp < kEpiWarp0) {
    // ------------------------------------------------------ x to 4-bit form --
    if constexpr (kFuse != 0) {
      constexpr int DT = kFuse - 1;
      constexpr int kAhead = DT == BLUT_F32 ? 2 : 4;  // blocks of x in registers
      using T = typename Elem<DT>::T;
      const int t64 = threadIdx.x - 64, r = t64 >> 3, u = t64 & 7;  // row, and 16 columns of the block's 128
      grid_dependency_wait();
      const float g = kMX ? 1.0f : __ldg(p.xg);
      const uint32_t cdst = C::kA + (u >> 1) * NT * 16 + r * 16 + (u & 1) * 8;
      const uint32_t sdst = C::kA + C::kB + r * 16 + (kMX ? u >> 1 : (u >> 2) * 512 + (u & 3));
      bool ok = true;
      int it = 0;
      for (int i = first; i < items && ok; i += step) {
        const Fp4Item t = item_of(p, i, lane, tab);
        const bool in = r < t.cnt;
        const T* src = static_cast<const T*>(p.x) + (int64_t)(t.row0 + (in ? r : 0)) * p.x_ld;
        Raw<DT> raw[kAhead];
        const auto fetch = [&](int b, Raw<DT>& w) {
          const int col = (b0 + b) * 128 + 16 * u;
          if (p.x_vec && in && b < nb && col + 16 <= p.cols) raw_load<DT, 16>(src + col, w);
        };
#pragma unroll
        for (int j = 0; j < kAhead; ++j) fetch(j, raw[j]);
        for (int c = 0; c < nb && ok; c += kAhead) {
#pragma unroll
          for (int j = 0; j < kAhead; ++j) {
            const int b = c + j, s = it % C::kStages;
            if (b < nb && ok) {
              const int col = (b0 + b) * 128 + 16 * u, n = in ? min(16, max(0, p.cols - col)) : 0;
              float v[16];
              if (p.x_vec && n == 16)
                raw_unpack<DT>(raw[j], v);
              else
                load16<DT>(src + col, n, v);
              fetch(b + kAhead, raw[j]);
              uint32_t sbyte;
              bool unsure = false;
              const uint2 code = encode16<DT, kMX, false>(v, g, unsure, sbyte);
              if (it >= C::kStages) {
                ok = wait_or_abort(smem_u32(h->empty + s), (uint32_t)(it / C::kStages - 1) & 1u, abort_flag,
                                   &g_fp4_status, p.wait_ns);
                ok = __all_sync(0xFFFFFFFFu, ok);
              }
              if (ok) {
                uint8_t* st = ring + s * C::kStage;
                *reinterpret_cast<uint2*>(st + cdst) = code;
                if (!kMX || (u & 1) == 0) st[sdst] = (uint8_t)sbyte;
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(h->sfull + s));
              }
              ++it;
            }
          }
        }
      }
    }
  } else if (warp < kEpiWarp0) {
    // -------------------------------------------------------- token scales --
    // Copied a word at a time, without registers in between.  Copies of up to
    // kAhead blocks are in flight; before it waits for a free stage a warp
    // hands over all it has, so nobody waits for what is already here.
    constexpr int kWordsAll = C::kWords * NT;
    constexpr int kIt = (kWordsAll + 63) / 64;
    constexpr int kAhead = 3;
    const int t64 = threadIdx.x - 64;
    const int64_t words = (int64_t)C::kWords * p.x_rows;
    const uint32_t ring_addr = smem_u32(ring);
    bool ok = true;
    int it = 0, given = 0;  // blocks copied, and handed over
    const auto give = [&] {
      fence_proxy_async();  // tcgen05.cp reads what was written here
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(h->sfull + given % C::kStages));
      ++given;
    };
    grid_dependency_wait();
    for (int i = first; i < items && ok; i += step) {
      const Fp4Item t = item_of(p, i, lane, tab);
      const uint32_t* src[kIt];
      uint32_t dst[kIt];
      bool on[kIt];
#pragma unroll
      for (int q = 0; q < kIt; ++q) {
        const int idx = t64 + 64 * q, r = idx % NT, w = idx / NT;
        on[q] = idx < kWordsAll && r < t.cnt;
        src[q] = p.xs + ((int64_t)b0 * C::kWords + w) * p.x_rows + t.row0 + r;
        dst[q] = C::kA + C::kB + (w * C::kGroups + r / 128) * 512 + (r % 32) * 16 + ((r % 128) / 32) * 4;
      }
      for (int b = 0; b < nb; ++b) {
        const int s = it % C::kStages;
        if (it >= C::kStages) {
          const uint32_t bar = smem_u32(h->empty + s), ph = (uint32_t)(it / C::kStages - 1) & 1u;
          if (!__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, ph))) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            while (given < it) give();
            ok = __all_sync(0xFFFFFFFFu, wait_or_abort(bar, ph, abort_flag, &g_fp4_status, p.wait_ns));
            if (!ok) break;
          }
        }
#pragma unroll
        for (int q = 0; q < kIt; ++q) {
          if (on[q])
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(ring_addr + s * C::kStage + dst[q]), "l"(src[q])
                         : "memory");
          src[q] += words;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (++it - given == kAhead) {
          asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
          give();
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    while (ok && given < it) give();
  } else if (split == 1) {
    // ------------------------------------------------------------ epilogue --
    const int q = warp & 3, part = (warp - kEpiWarp0) >> 2;  // lane quarter (a warp may read its own only), share
    uint8_t* stage = epi + (warp - kEpiWarp0) * kEpiStage;
    const uint32_t tcol = tmem + ((uint32_t)(32 * q) << 16);
    grid_dependency_wait();
    const float gx = p.xg ? __ldg(p.xg) : 1.0f;
    int acc = 0;
    for (int i = first; i < items; i += step, ++acc) {
      const Fp4Item t = item_of(p, i, lane, tab);
      const float alpha = gx * (p.wg ? __ldg(p.wg + t.expert) : 1.0f);
      const int64_t row = (int64_t)t.tile * 128 + 32 * q;
      if (!__all_sync(0xFFFFFFFFu, wait_or_abort(smem_u32(&h->acc_full), (uint32_t)acc & 1u, abort_flag, &g_fp4_status,
                                                 p.wait_ns)))
        break;
      tc_fence_after();
      const int left = (int)min((int64_t)32, p.n - row);  // rows of the matrix among this warp's
      const auto read = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&h->acc_empty));
      };
      if (left <= 0) {
        read();
      } else if (p.out_dtype != BLUT_F32) {
        uint16_t* y = static_cast<uint16_t*>(p.y) + (int64_t)t.row0 * p.ldy + row;
        // (a box that y's last rows cut is written in 16-byte pieces, past them)
        const CUtensorMap* map = p.tma && left == 32 ? &ymap : nullptr;
        if (p.out_dtype == BLUT_BF16)
          store_tile16<BLUT_BF16>(tcol, t.cnt, alpha, stage, y, p.ldy, left, p.vec, lane, 32 * part, 32 * C::kEpi, map,
                                  p.tma, (int)row, t.row0, (int)p.x_rows, read);
        else
          store_tile16<BLUT_F16>(tcol, t.cnt, alpha, stage, y, p.ldy, left, p.vec, lane, 32 * part, 32 * C::kEpi, map,
                                 p.tma, (int)row, t.row0, (int)p.x_rows, read);
      } else {
#pragma unroll 1
        for (int c = 16 * part; c < t.cnt; c += 16 * C::kEpi) {
          uint32_t v[16];
          tc_ld16(tcol + c, v);
          tc_wait_ld16(v);
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c + j < t.cnt) store1(p, t.row0 + c + j, row + lane, __uint_as_float(v[j]) * alpha);
        }
        read();
      }
    }
    if (p.tma && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }

  if (split > 1 && first < items) {
    // ----------------------------------- one item, K split over the cluster --
    const Fp4Item t = item_of(p, first, lane, tab);
    float* part = reinterpret_cast<float*>(ring);  // free: the last MMA has read it
    bool ok = __all_sync(0xFFFFFFFFu, wait_or_abort(smem_u32(&h->acc_full), 0, abort_flag, &g_fp4_status, p.wait_ns));
    tc_fence_after();
    if (warp >= kEpiWarp0 && ok) {  // (K is split for NT <= 128 only: four warps)
      const int q = warp & 3;
#pragma unroll 1
      for (int c = 0; c < t.cnt; c += 16) {
        uint32_t v[16];
        tc_ld16(tmem + ((uint32_t)(32 * q) << 16) + c, v);
        tc_wait_ld16(v);
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c + j) * 128 + 32 * q + lane] = __uint_as_float(v[j]);
      }
    }
    cluster_sync();
    grid_dependency_wait();
    const float alpha = (p.xg ? __ldg(p.xg) : 1.0f) * (p.wg ? __ldg(p.wg + t.expert) : 1.0f);
    if (ok) {
      if (split == 2)
        reduce_cluster<2, C::kThreads>(p, part, rank, t.cnt, t.row0, (int64_t)t.tile * 128, alpha);
      else if (split == 4)
        reduce_cluster<4, C::kThreads>(p, part, rank, t.cnt, t.row0, (int64_t)t.tile * 128, alpha);
      else
        reduce_cluster<8, C::kThreads>(p, part, rank, t.cnt, t.row0, (int64_t)t.tile * 128, alpha);
    }
    cluster_sync();  // no CTA leaves while another still reads its partial tile
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kCols));
}

// The map of a 16-bit y [x_rows][n] for boxes of 32 tokens x 32 rows.
bool y_map(const Fp4Params& p, CUtensorMap* map) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<Encode> encode{nullptr};
  Encode fn = encode.load(std::memory_order_acquire);
  if (!fn) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      return false;
    fn = reinterpret_cast<Encode>(f);
    encode.store(fn, std::memory_order_release);
  }
  const cuuint64_t dims[2] = {(cuuint64_t)p.n, (cuuint64_t)p.x_rows}, pitch[1] = {(cuuint64_t)p.ldy * 2};
  const cuuint32_t box[2] = {32, 32}, one[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, p.y, dims, pitch, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// early: the launch may begin while the kernel before it, which writes x, is
// still running (it waits in grid_dependency_wait before it reads x).
template <bool kMX, int NT, int kFuse = 0>
int launch(Fp4Params& p, int64_t items, bool early, cudaStream_t stream) {
  using C = Fp4Cfg<kMX, NT>;
  auto kern = fp4_mm_kernel<kMX, NT, kFuse>;
  constexpr int kMaxSmem = C::kSmem + (2 * kMaxExperts + 2) * 4;
  static std::atomic<int> sms_of[kMaxDevices];  // 0: not set up yet
  const int dev = cache_device();
  int sms = dev < 0 ? 0 : sms_of[dev].load(std::memory_order_acquire);
  if (sms == 0) {
    int d = 0;
    if (cudaGetDevice(&d) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, d) != cudaSuccess ||
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem) != cudaSuccess ||
        cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, 100) != cudaSuccess)
      return BLUT_ERR_CUDA;
    if (dev >= 0) sms_of[dev].store(sms, std::memory_order_release);
  }
  const int split = 1 << p.split_log;
  // large items leave by bulk tensor stores (the map costs the host under a
  // microsecond, which the smallest calls would notice)
  CUtensorMap map = {};
  p.tma = NT >= 128 && split == 1 && p.vec && p.out_dtype != BLUT_F32 && y_map(p, &map);
  cudaLaunchConfig_t cfg = {};
  // one CTA (cluster) per item where K is split, else as many as run at once
  cfg.gridDim = dim3((unsigned)(split > 1 ? items * split : std::min<int64_t>(items, (int64_t)sms * C::kCtas)));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem + (p.experts ? (2 * p.experts + 2) * 4 : 0);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (split > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = (unsigned)split;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (early) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  return cudaLaunchKernelEx(&cfg, kern, (const Fp4Params)p, (const CUtensorMap)map) == cudaSuccess ? BLUT_OK
                                                                                                   : BLUT_ERR_LAUNCH;
}

// Tokens of an item for one matrix and more than 128 tokens: as few tiles as
// 192 allow, cut evenly.  Against tiles of 192: 256 x 11264 x 2048 11.5 ->
// 11.2 us, 300 x 2816 x 2048 10.5 either way.  More and smaller tiles that
// fill the last round of CTAs better gain next to nothing (1999 x 5000 x 1400:
// 16.6 us with 192, 16.4 with 176, 160 and 144, 18.7 with 128).
int tokens_per_item(int64_t m) {
  const int64_t tiles = (m + 191) / 192;
  return (int)(((m + tiles - 1) / tiles + 15) / 16 * 16);
}

template <bool kMX>
int dispatch(Fp4Params& p, int64_t m, int fuse, bool early, cudaStream_t stream) {
  p.row_tiles = (p.n + 127) / 128;
  // Tokens per matrix: their number for one matrix, the mean for runs (their
  // lengths are on the device).  In us with items of 32, 64, 128, 192 tokens:
  //   one matrix 11264 x 2048,  32 tokens   9.6   9.5
  //                             64          9.7  11.0   9.7  10.3
  //                            128         10.3  11.0  11.4  11.1
  //                            256         14.7  11.2  10.7  11.2
  //   64 of 2816 x 2048, mean   12         39.1  39.7  37.9  41.4
  //                             48         47.5  45.5  42.8  45.2
  //                             96         69.5  55.1  48.4  54.5
  //                            192          121  80.6  69.5  64.5
  // The mean cannot see a few runs with most of the rows, nor rows behind the
  // last run: 22 runs of 512 tokens' six rows each, the longest 509, take 31.6
  // (64) against 25.9 (128), one run of 2048 25.6 (32) against 13.7 (192), and 128 rows of
  // 45 runs in a buffer of 7808 33.3 (192) against 30.6 (32).
  const int64_t mean = p.experts ? (m + p.experts - 1) / p.experts : m;
  const int nt = mean <= 32 ? 32 : mean <= 64 ? 64 : mean <= 128 ? 128 : 192;
  p.tn = nt == 192 && !p.experts ? tokens_per_item(m) : nt;
  // bound on the token tiles: every run may end in a partial one
  const int64_t tiles = p.experts ? m / nt + std::min<int64_t>(p.experts, m) : (m + p.tn - 1) / p.tn;
  const int64_t items = tiles * p.row_tiles;
  if (items * 8 > INT32_MAX) return BLUT_ERR_UNSUPPORTED;
  p.token_tiles = (int)tiles;
  p.split_log = 0;
  if (nt <= 128)
    while (p.split_log < 3 && (items << p.split_log) * 2 <= (nt <= 64 ? 444 : 296) && p.kblocks >= 4 << p.split_log)
      ++p.split_log;
  switch (fuse) {
    case 1 + BLUT_F16: return launch<kMX, 32, 1 + BLUT_F16>(p, items, early, stream);
    case 1 + BLUT_BF16: return launch<kMX, 32, 1 + BLUT_BF16>(p, items, early, stream);
    case 1 + BLUT_F32: return launch<kMX, 32, 1 + BLUT_F32>(p, items, early, stream);
  }
  switch (nt) {
    case 32: return launch<kMX, 32>(p, items, early, stream);
    case 64: return launch<kMX, 64>(p, items, early, stream);
    case 128: return launch<kMX, 128>(p, items, early, stream);
    default: return launch<kMX, 192>(p, items, early, stream);
  }
}

int fp4_check(const blut_fp4_mm_args* a) {
  if (!a || !fp4_valid(a->w) || !a->w_tiled || !a->x_codes || !a->x_scales || !a->y) return BLUT_ERR_INVALID;
  if (a->x_rows <= 0 || a->x_rows > kMaxSlots || a->y_ld < a->w.rows) return BLUT_ERR_INVALID;
  if (a->num_experts < 0 || a->num_experts > kMaxExperts || (a->num_experts && !a->offsets)) return BLUT_ERR_INVALID;
  if (a->num_experts > 1 && (a->w_stride < blut_fp4_tiled_bytes(&a->w) || a->w_stride % 16)) return BLUT_ERR_INVALID;
  if (((uintptr_t)a->w_tiled | (uintptr_t)a->x_codes | (uintptr_t)a->x_scales) % 16 != 0) return BLUT_ERR_INVALID;
  if (a->out_dtype != BLUT_F16 && a->out_dtype != BLUT_BF16 && a->out_dtype != BLUT_F32) return BLUT_ERR_UNSUPPORTED;
  if ((uintptr_t)a->y % (a->out_dtype == BLUT_F32 ? 4 : 2) != 0) return BLUT_ERR_INVALID;
  return BLUT_OK;
}

// x not null: x's rows are quantised by the product (at most kFuseRows of them).
int fp4_product(const blut_fp4_mm_args* a, bool early, const void* x, int x_dtype, int64_t x_ld, cudaStream_t s) {
  const int rc = fp4_check(a);
  if (rc != BLUT_OK) return rc;
  Fp4Params p = {};
  p.w = static_cast<const uint8_t*>(a->w_tiled);
  p.wstride = a->w_stride;
  p.wg = a->w_scale;
  p.offsets = a->offsets;
  p.experts = a->num_experts;
  p.xc = static_cast<const uint8_t*>(a->x_codes);
  p.xs = static_cast<const uint32_t*>(a->x_scales);
  p.xg = a->x_scale;
  p.x_rows = a->x_rows;
  p.n = (int)a->w.rows;
  p.kblocks = fp4_kblocks(a->w.cols);
  p.y = a->y;
  p.ldy = a->y_ld;
  p.out_dtype = a->out_dtype;
  p.vec = ((uintptr_t)a->y | (uintptr_t)(a->y_ld * (a->out_dtype == BLUT_F32 ? 4 : 2))) % 16 == 0;
  p.wait_ns = wait_limit_ns();
  const int fuse = x ? 1 + x_dtype : 0;
  if (x) {
    p.x = x;
    p.x_ld = x_ld;
    p.cols = (int)a->w.cols;
    p.x_vec = ((uintptr_t)x | (uintptr_t)(x_ld * (x_dtype == BLUT_F32 ? 4 : 2))) % 16 == 0;
  }
  return a->w.kind == BLUT_FP4_MX ? dispatch<true>(p, a->x_rows, fuse, early, s)
                                  : dispatch<false>(p, a->x_rows, fuse, early, s);
}

// Workspace of blut_fp4_linear: x in 4-bit form (unless the product quantises
// it), then its g (unless it is given or there is none).
struct LinearWs {
  int64_t scales, g, total;
};
LinearWs linear_ws(const blut_fp4_desc& w, int64_t m, bool given) {
  blut_fp4_desc d = w;
  d.rows = m;
  LinearWs l = {};
  if (m > kFuseRows) {
    l.scales = align256(blut_fp4_codes_bytes(&d));
    l.g = l.scales + align256(blut_fp4_scales_bytes(&d));
  }
  l.total = l.g + (w.kind == BLUT_FP4_NV && !given ? 256 : 0);
  return l;
}

}  // namespace
}  // namespace blut

using namespace blut;

extern "C" {

int blut_fp4_matmul(const blut_fp4_mm_args* a, void* stream) {
  return fp4_product(a, false, nullptr, 0, 0, reinterpret_cast<cudaStream_t>(stream));
}

int64_t blut_fp4_linear_workspace_size(const blut_fp4_desc* w, int64_t x_rows, int32_t scale_given) {
  if (!w || !fp4_valid(*w) || x_rows <= 0 || x_rows > kMaxSlots) return BLUT_ERR_INVALID;
  return linear_ws(*w, x_rows, scale_given != 0).total;
}

int blut_fp4_linear(const blut_fp4_mm_args* args, const void* x, int32_t x_dtype, int64_t x_ld, void* workspace,
                    size_t workspace_bytes, void* stream) {
  if (!args || !fp4_valid(args->w) || !x || (uintptr_t)workspace % 16) return BLUT_ERR_INVALID;
  if (args->x_rows <= 0 || args->x_rows > kMaxSlots || args->num_experts || x_ld < args->w.cols) return BLUT_ERR_INVALID;
  if (x_dtype != BLUT_F16 && x_dtype != BLUT_BF16 && x_dtype != BLUT_F32) return BLUT_ERR_UNSUPPORTED;
  if ((uintptr_t)x % (x_dtype == BLUT_F32 ? 4 : 2)) return BLUT_ERR_INVALID;
  blut_fp4_mm_args a = *args;
  if (a.w.kind == BLUT_FP4_MX) a.x_scale = nullptr;
  const LinearWs ws = linear_ws(a.w, a.x_rows, a.x_scale != nullptr);
  if (ws.total && (!workspace || workspace_bytes < (size_t)ws.total)) return BLUT_ERR_WORKSPACE;
  uint8_t* base = static_cast<uint8_t*>(workspace);
  const bool fuse = a.x_rows <= kFuseRows;
  a.x_codes = fuse ? a.w_tiled : base;  // not read where the product quantises x
  a.x_scales = fuse ? a.w_tiled : base + ws.scales;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int rc = fp4_check(&a);
  if (rc != BLUT_OK) return rc;
  if (a.w.kind == BLUT_FP4_NV && !a.x_scale) {
    float* g = reinterpret_cast<float*>(base + ws.g);
    rc = blut_fp4_global_scale(x, x_dtype, a.x_rows, a.w.cols, x_ld, 0, g, stream);
    if (rc != BLUT_OK) return rc;
    a.x_scale = g;
  }
  if (fuse) return fp4_product(&a, false, x, x_dtype, x_ld, s);
  blut_fp4_desc d = a.w;
  d.rows = a.x_rows;
  rc = fp4_quantize_for_product(d, x, x_dtype, x_ld, a.x_scale, base, base + ws.scales, s);
  return rc == BLUT_OK ? fp4_product(&a, true, nullptr, 0, 0, s) : rc;
}

int blut_fp4_check_status(void* stream) {
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int st = 0, zero = 0;
  if (cudaMemcpyFromSymbolAsync(&st, g_fp4_status, sizeof(int), 0, cudaMemcpyDeviceToHost, s) != cudaSuccess ||
      cudaStreamSynchronize(s) != cudaSuccess)
    return BLUT_ERR_CUDA;
  if (!st) return BLUT_OK;
  if (cudaMemcpyToSymbolAsync(g_fp4_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s) != cudaSuccess ||
      cudaStreamSynchronize(s) != cudaSuccess)
    return BLUT_ERR_CUDA;
  return BLUT_ERR_TIMEOUT;
}

}  // extern "C"
