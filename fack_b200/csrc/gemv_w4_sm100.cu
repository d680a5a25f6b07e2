// gemv_w4_sm100.cu -- products of a few tokens with 4-bit weights (sm_100a).
//
//   y[m, n] = sum_k x[m, k] * (c[n, k] - z[k/G, n]) * s[k/G, n]
//
// with codes c in 0..15 packed two a byte along K (even k in the low nibble),
// one scale and optionally one zero point (else 8) per output row and group of
// G consecutive k, x and y bf16 or fp16.  With a plan of tokens sorted by
// expert the same for every expert's rows and weights.
//
// The call is the weight stream, N*K/2 bytes that are read once: 13 T codes a
// second at the memory's rate, which leaves a scheduler about 22 cycles for each
// warp-wide word of 8 codes a lane.  So instructions count as much as bytes:
//   * The products go to the warp MMA (m16n8k16, fp32 accumulators): 16 weight
//     rows x 8 tokens.  A word of 8 codes becomes four operand registers of the
//     exact 16-bit floats c - z with one shift, four masks and four fma (see
//     Codes): every product is exact, and the only roundings are fp32 additions,
//     the fp32 scale per group and the last one to the output type.
//   * The pairs (i, i + 4) that a mask picks out of a word are met by the tokens in
//     the same order (the MMA does not care which k goes where, if both operands
//     agree).
//   * One warp of a CTA brings the data (TMA boxes of weights, scales and zero
//     points, one bulk copy a token) into a ring of stages; eight multiply, each
//     its own rows of one of `split` slices of K.  CTAs are persistent over a list
//     of (expert, row tile, token tile) items, and the ring runs on from one item
//     into the next.  Rows per warp, slices and rows per item follow a cost model
//     (see plan): few rows are split along K, many are dealt out evenly.
// Measured on B200, one call after another: 65536 x 7168 (235 MB), groups of 128, bf16, with
// one token 51 us = 4.6 TB/s, with eight 53, with thirteen 78; groups of 64 with zero
// points, fp16, thirteen 85.  With parts left out (one / thirteen tokens, groups of 128):
// copies alone 44 / 51, without the products 44 / 54, without the unpacking 47 / 68.  So
// neither part alone adds much to the copies: a warp's products wait for its unpacking and
// its sums for the products, two warps a scheduler (four with eight tokens) do not hide it
// all, and 46 % (61 %) of the issue slots are taken, 20 (17) instructions a word.
// The warp MMA, not tcgen05: a form that unpacks into tensor memory (the codes as A,
// 128 rows x 64 k a step, sixteen warps) was built and gave 88-94 us for one token and
// 94-106 for thirteen.  Its products cost next to nothing (9 cycles for 128 x 16 x 16),
// but a lane then unpacks as much, adds 16 sums a group instead of 8, and pays stores,
// loads and waits of tensor memory: 32 instructions a word.  Tokens in three 8-bit
// digits and codes as they are (exact, a third of the unpacking) were measured with
// the int8 MMA (56 / 71 / 126 us for 1 / 8 / 13 tokens: three times the MMAs and
// accumulators) and the fp8 MMA (92 us: mma.sync converts its operands here).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <mutex>
#include <type_traits>

#include "../../include/fack_gemm.h"
#include "fack_internal.h"
#include "sm100_ptx.cuh"

namespace fack_w4 {

using namespace fack;

constexpr int kWarps = 8;                      // that multiply; one more brings the data
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kBlkK = 128;                     // k per warp and stage
constexpr int kMaxStages = 8;
constexpr int kMaxExperts = 1024;
constexpr int kMaxTopk = 64;
constexpr unsigned kStW4 = 256u;               // status flag: a wait in these kernels gave up

struct Args {
  const void* x;                               // [rows or tokens, K]
  int64_t ldx;
  const uint8_t* w;                            // [E, N, K/2]
  const void* scales;                          // [E, K/G, N]
  const uint8_t* zeros;                        // [E, K/G, N] or NULL
  void* y;                                     // [rows, N]
  int64_t ldy;
  const int* src;                              // pair of each sorted row, NULL: row r of x is row r of y
  const int* offsets;                          // [E + 1], NULL: one weight, all rows
  int rows, topk, N, K, G, E;
  int tile;                                    // tokens per tile (<= 8 NT)
  int split;                                   // slices of K among a CTA's warps: 1, 2, 4 or 8
  int groups;                                  // 16-row groups of an item: more than (R - 1) share, at most R share
  int stages;
  int scale_f32;
  unsigned int* status;
  uint64_t timeout_ns;
};

// A word's codes 0..7 as four registers of two 16-bit floats each, exactly
// (c - z) / kScale, codes i and i + 4 together.  A masked code is a subnormal, c or
// 16c units of the type's smallest (in bf16 the top bit of 16c is the exponent's
// lowest, where the normal numbers go on at the same spacing), and one fused
// multiply-add scales it and takes the zero point away: 1 shift, 4 masks, 4 fma
// for 8 codes.  Or-ing the code into 128 or 1024 and subtracting takes 3 shifts;
// shifts and masks run at half the rate of the fma (95 -> 74 us for 16 rows of
// 4096 x 7168 in an earlier form of the kernel).
template <typename T> struct Codes;
template <> struct Codes<__nv_bfloat16> {
  using T2 = __nv_bfloat162;
  static constexpr uint32_t kLow = 0x7f007f00u, kHigh = 0x7d007d00u;   // 2^127, 2^123: c * 2^-133 -> c * 2^-6
  static constexpr uint32_t kMinusEight = 0xbe00be00u;                 // -8 * 2^-6
  static constexpr uint32_t kNegate = 0xff00ff00u;                     // z * 2^-133 -> -z * 2^-6
  static constexpr float kScale = 64.0f;
  static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Codes<__half> {
  using T2 = __half2;
  static constexpr uint32_t kLow = 0x78007800u, kHigh = 0x68006800u;   // 2^15, 2^11: c * 2^-24 -> c * 2^-9
  static constexpr uint32_t kMinusEight = 0xa400a400u;                 // -8 * 2^-9
  static constexpr uint32_t kNegate = 0xf800f800u;                     // z * 2^-24 -> -z * 2^-9
  static constexpr float kScale = 512.0f;
  static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <typename T>
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
  using T2 = typename Codes<T>::T2;
  const T2 r = __hfma2(*reinterpret_cast<const T2*>(&a), *reinterpret_cast<const T2*>(&b), *reinterpret_cast<const T2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename T>
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  using T2 = typename Codes<T>::T2;
  const T2 r = __hmul2(*reinterpret_cast<const T2*>(&a), *reinterpret_cast<const T2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename T>
__device__ __forceinline__ void unpack_codes(uint32_t w, uint32_t minus_z, uint32_t (&h)[4]) {
  const uint32_t v = w >> 8;
  h[0] = fma2<T>(w & 0x000f000fu, Codes<T>::kLow, minus_z);
  h[1] = fma2<T>(w & 0x00f000f0u, Codes<T>::kHigh, minus_z);
  h[2] = fma2<T>(v & 0x000f000fu, Codes<T>::kLow, minus_z);
  h[3] = fma2<T>(v & 0x00f000f0u, Codes<T>::kHigh, minus_z);
}

// d = a * b + c on the warp's 16 x 8 tile
#define FACK_W4_MMA(TYPE)                                                                                              \
  asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE                                                           \
      ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"                                       \
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                                                 \
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]))
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1, const float (&c)[4], __nv_bfloat16*) {
  FACK_W4_MMA("bf16");
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1, const float (&c)[4], __half*) {
  FACK_W4_MMA("f16");
}
#undef FACK_W4_MMA
// d (+)= a * b: the first product of a group starts from zero
template <typename T>
__device__ __forceinline__ void mma_step(float (&d)[4], bool first, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (first)
    mma16816(d, a0, a1, a2, a3, b0, b1, zero, static_cast<T*>(nullptr));
  else
    mma16816(d, a0, a1, a2, a3, b0, b1, d, static_cast<T*>(nullptr));
}

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&v)[1]) { v[0] = lds32(a); }
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&v)[2]) {
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(a));
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ float scale_of(uint32_t bits, __nv_bfloat16*) { return __uint_as_float(bits << 16); }
__device__ __forceinline__ float scale_of(uint32_t bits, __half*) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}

// A CTA's item is `groups` 16-row groups of the output, dealt out evenly to its
// share = 8 / split row parts, R or R - 1 to each, and a tile of tokens; a stage of
// its ring holds `split` consecutive K blocks of them, one for each slice.  Warp
// (part, slice) multiplies its groups of block `slice`.
//   weights: per slice, rows of 64 bytes in the 64-byte swizzle (16-byte chunk c of
//     row r at c ^ (r/2 & 3)), in boxes of at most 256 rows;
//   tokens: rows of split * 256 bytes and a pad;
//   scales and zero points: per box, a row for each group of the stage's blocks.
// How the chunks are read: a step j of the MMA takes 8 consecutive codes (one
// word) a lane and row.  With groups of 64 or 128 k a lane's two words may be
// consecutive, one 8-byte read (WV = 2), else one (WV = 1), since a step may not mix
// groups: step j of quad lane q is word WV q + j % WV of part j / WV.  The pads put
// the tokens' reads on different banks.
template <int R, int FL>
struct Stage {
  static constexpr int kGroups = kBlkK / FL;
  static constexpr int kRows = 16 * R;
  static constexpr int kWords = FL == 32 || R == 4 ? 1 : 2;   // WV (R = 4 has no registers for more)
  static constexpr int kWeightBytes = kWarps * kRows * 64;
  static constexpr int kPad = kWords == 1 ? 64 : 16;
  __host__ __device__ static int up(int v, int to) { return (v + to - 1) / to * to; }
  __host__ __device__ static int boxes(int groups) { return groups > 16 ? 2 : 1; }
  __host__ __device__ static int box_rows(int groups) { return 16 * (groups / boxes(groups)); }
  __host__ __device__ static int x_pitch(int split) { return split * 256 + kPad; }
  __host__ __device__ static int scale_at(int tile, int split) { return up(kWeightBytes + tile * x_pitch(split), 128); }
  __host__ __device__ static int scale_box(int split, int groups, int es) {
    return up(split * kGroups * box_rows(groups) * es, 128);
  }
  __host__ __device__ static int zero_at(int tile, int split, int groups, int es) {
    return scale_at(tile, split) + boxes(groups) * scale_box(split, groups, es);
  }
  __host__ __device__ static int zero_box(int split, int groups) { return up(split * kGroups * box_rows(groups), 128); }
  __host__ __device__ static int bytes(int tile, int split, int groups, int es, bool zeros) {
    return up(zero_at(tile, split, groups, es) + (zeros ? boxes(groups) * zero_box(split, groups) : 0), 1024);
  }
};
template <int R, int NT>
struct Sums {                                  // the warps' partial sums
  static constexpr int kPitch = 8 * NT + 1;
  static int bytes(int split) { return split > 1 ? kWarps * 16 * R * kPitch * 4 : 0; }
};

struct Item {
  int expert, n0, row0, count;
};

template <typename T, int R, int NT, int FL, bool ZP>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1)
    gemv_w4_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap s_map,
                   const __grid_constant__ CUtensorMap z_map, const __grid_constant__ Args p) {
  using S = Stage<R, FL>;
  using C = Codes<T>;
  constexpr int kRows = S::kRows, kPitch = Sums<R, NT>::kPitch;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int part[2][kWarps + 1];
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages];
  __shared__ int abort_flag_s, routed_s;         // rows of an expert: the rest are zeros
  volatile int* abort_flag = &abort_flag_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int split = p.split, share = kWarps / split, item_rows = 16 * p.groups;
  const int es = p.scale_f32 ? 4 : 2;
  const int box_rows = S::box_rows(p.groups), boxes = S::boxes(p.groups), x_pitch = S::x_pitch(split);
  const int stage_bytes = S::bytes(p.tile, split, p.groups, es, ZP);
  const int scale_at = S::scale_at(p.tile, split), scale_box = S::scale_box(split, p.groups, es);
  const int zero_at = S::zero_at(p.tile, split, p.groups, es), zero_box = S::zero_box(split, p.groups);
  const uint32_t ring = smem_addr(smem);
  float* red = reinterpret_cast<float*>(smem + p.stages * stage_bytes);
  // the experts that have rows: number, first and last sorted row, running count of token tiles
  const int room = p.offsets == nullptr ? 1 : min(p.E, p.rows);
  int* act_expert = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(red) + (split > 1 ? kWarps * kRows * kPitch * 4 : 0));
  int* act_row = act_expert + room;
  int* act_end = act_row + room;
  int* act_tile = act_end + room;

  // ------------------------------------------------------------ item list --
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(smem_addr(&full[i]), 1);
      mbar_init(smem_addr(&empty[i]), kWarps);
    }
    abort_flag_s = 0;
    fence_mbar_init();
  }
  int active = 1;
  if (p.offsets == nullptr) {
    if (threadIdx.x == 0) {
      routed_s = p.rows;
      act_expert[0] = 0;
      act_row[0] = 0;
      act_end[0] = p.rows;
      act_tile[0] = 0;
      act_tile[1] = (p.rows + p.tile - 1) / p.tile;
    }
  } else {
    constexpr int kPer = kMaxExperts / (kWarps * 32);
    int tiles[kPer], first[kPer], last[kPer], my_tiles = 0, my_act = 0, bad = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = threadIdx.x * kPer + i;
      tiles[i] = 0;
      if (e < p.E) {
        first[i] = p.offsets[e];
        last[i] = p.offsets[e + 1];
        bad |= (e == 0 ? first[i] != 0 : first[i] < 0) || last[i] < first[i] || last[i] > p.rows;
        if (last[i] > first[i]) tiles[i] = (last[i] - first[i] + p.tile - 1) / p.tile;
      }
      my_tiles += tiles[i];
      my_act += tiles[i] > 0;
    }
    // offsets that do not ascend from 0 within the rows are no plan: nothing is routed
    if (__syncthreads_or(bad)) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) tiles[i] = 0;
      my_tiles = my_act = bad = 0;
      if (threadIdx.x == 0) routed_s = 0;
    } else if (threadIdx.x == 0) {
      routed_s = p.offsets[p.E];
    }
    int st = my_tiles, sa = my_act;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int ot = __shfl_up_sync(0xffffffffu, st, d), oa = __shfl_up_sync(0xffffffffu, sa, d);
      if (lane >= d) {
        st += ot;
        sa += oa;
      }
    }
    if (lane == 31) {
      part[0][warp] = st;
      part[1][warp] = sa;
    }
    __syncthreads();
    st -= my_tiles;
    sa -= my_act;
    active = 0;
    for (int i = 0; i <= kWarps; ++i) {
      st += i < warp ? part[0][i] : 0;
      sa += i < warp ? part[1][i] : 0;
      active += part[1][i];
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (tiles[i] > 0) {
        act_expert[sa] = threadIdx.x * kPer + i;
        act_row[sa] = first[i];
        act_end[sa] = last[i];
        act_tile[sa] = st;
        ++sa;
        st += tiles[i];
      }
    }
    if (threadIdx.x == kThreads - 1) act_tile[sa] = st;
  }
  __syncthreads();
  const int ntiles = (p.N + item_rows - 1) / item_rows;
  const int items = act_tile[active] * ntiles;
  const int KB = (p.K + kBlkK - 1) / kBlkK;

  // Items go expert by expert, then row tile by row tile, token tiles
  // innermost: the tiles that share weights run side by side.
  auto decode = [&](int item, int& at) {
    const int tile = item / ntiles;
    while (at + 1 < active && act_tile[at + 1] <= tile) ++at;
    const int of = act_tile[at + 1] - act_tile[at];
    const int local = item - act_tile[at] * ntiles;
    const int n = local / of, m = local - n * of;
    Item it;
    it.expert = act_expert[at];
    it.n0 = n * item_rows;
    it.row0 = act_row[at] + m * p.tile;
    it.count = min(p.tile, act_end[at] - it.row0);
    return it;
  };
  // x row of sorted row r, -1 where its pair is none
  auto x_row_of = [&](int r) {
    if (p.src == nullptr) return r;
    const int from = p.src[r];
    return from >= 0 && from < p.rows ? from / p.topk : -1;
  };

  int at = 0, s = 0;
  uint32_t phase = 0;
  if (warp == kWarps) {
    // ----------------------------------------------------------- producer --
    // Lane l < split brings the weights of slice l, lane 8 the scales, lane 9 the
    // zero points, lane 16 + m the blocks of token m.  Tokens past the item's
    // count, or without an x row, are not brought: their columns of the MMA touch
    // no other and are not stored.
    const uint64_t once = policy_evict_first();
    const int groups = p.K / p.G, s_rows = split * S::kGroups;
    int issued = 0;
    bool gone = false;
    for (int item = blockIdx.x; item < items && !gone; item += gridDim.x) {
      const Item it = decode(item, at);
      const int x_row = lane >= 16 && lane - 16 < it.count ? x_row_of(it.row0 + lane - 16) : -1;
      const int x_rows = __popc(__ballot_sync(0xffffffffu, x_row >= 0));
      const uint8_t* x = static_cast<const uint8_t*>(p.x) + (x_row < 0 ? 0 : x_row) * p.ldx * 2;
      for (int kb = 0; kb < KB; kb += split) {
        const bool ok = wait_bounded(smem_addr(&empty[s]), phase ^ 1u, abort_flag, p.status, kStW4, p.timeout_ns);
        if (!__all_sync(0xffffffffu, ok)) {
          gone = true;
          break;
        }
        const uint32_t bar = smem_addr(&full[s]), dst = ring + s * stage_bytes;
        const int blocks = min(split, KB - kb);
        const uint32_t x_bytes = min(split * kBlkK, p.K - kb * kBlkK) * 2;
        if (lane == 0)
          mbar_arrive_expect_tx(bar, blocks * item_rows * 64 + boxes * s_rows * box_rows * (es + (ZP ? 1 : 0)) + x_rows * x_bytes);
        __syncwarp();
        const int group = it.expert * groups + (FL == 128 ? kb * kBlkK / p.G : kb * S::kGroups);
        if (lane < blocks) {
          for (int b = 0; b < boxes; ++b)
            tma_load_2d(dst + lane * item_rows * 64 + b * box_rows * 64, &w_map, bar, (kb + lane) * (kBlkK / 2),
                        it.expert * p.N + it.n0 + b * box_rows, once);
        } else if (lane == 8) {
          for (int b = 0; b < boxes; ++b)
            tma_load_2d(dst + scale_at + b * scale_box, &s_map, bar, it.n0 + b * box_rows, group, once);
        } else if (ZP && lane == 9) {
          for (int b = 0; b < boxes; ++b)
            tma_load_2d(dst + zero_at + b * zero_box, &z_map, bar, it.n0 + b * box_rows, group, once);
        } else if (x_row >= 0) {
          bulk_load_1d(dst + S::kWeightBytes + (lane - 16) * x_pitch, x + static_cast<int64_t>(kb) * (kBlkK * 2), x_bytes, bar);
        }
        __syncwarp();
        ++issued;
        if (++s == p.stages) {
          s = 0;
          phase ^= 1u;
        }
      }
    }
    if (gone && lane == 0) {
      // no copy may land after the CTA exits: wait (bounded, fresh deadline) for the last stages issued
      volatile int no_abort = 0;
      for (int i = issued > p.stages ? issued - p.stages : 0; i < issued; ++i)
        wait_bounded(smem_addr(&full[i % p.stages]), (i / p.stages) & 1u, &no_abort, p.status, kStW4, p.timeout_ns);
    }
    __syncwarp();
  } else {
    // ----------------------------------------------------------- consumer --
    // A wait that gave up leaves the control flow as it is (the barriers below
    // count on every warp) and the status word says that the result is none.
    const int slice = warp % split, part_no = warp / split;
    // this part's groups: R or R - 1 of its box's.  The second box deals them out from
    // its other end, so that a scheduler's two warps of a CTA have 2 R - 1 together.
    const int parts = share / boxes, each = box_rows / 16 / parts, more = box_rows / 16 % parts, box = part_no / parts;
    const int in_box = box ? parts - 1 - part_no % parts : part_no % parts;
    const int box_row = 16 * (in_box * each + min(in_box, more)), first_row = box * box_rows + box_row;
    const bool full_part = each + (in_box < more ? 1 : 0) == R;
    // With groups of 128 k a part of R - 1 groups loads for a last one as well, whose products are
    // left out.  Its words lie in the stage; behind the last box of scales or zero points the
    // ring may end, so there it loads those of the group before.
    const uint32_t last = full_part ? R - 1 : R - 2;
    auto loaded = [&](int r) -> uint32_t { return FL == 128 && r == R - 1 ? last : r; };
    const uint32_t w_at = slice * item_rows * 64 + (first_row + g) * 64 +
                          (((S::kWords == 1 ? 0 : q >> 1) ^ ((g >> 1) & 3)) << 4) + (S::kWords == 1 ? q * 4 : (q & 1) * 8);
    // lanes whose token the tile does not have read another's: their columns are not stored
    uint32_t x_at[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
      x_at[n] = S::kWeightBytes + min(8 * n + g, p.tile - 1) * x_pitch + slice * 256 + S::kWords * q * 16;
    const uint32_t s_at = scale_at + box * scale_box + (box_row + g) * es, z_at = zero_at + box * zero_box + box_row + g;
    bool alive = true;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
      const Item it = decode(item, at);
      float acc[R][NT][4];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.0f;
      // the item's K, this warp's R or R - 1 groups of rows.  With groups of 32 or 64 k the
      // loop is compiled for either (a test for the last rows inside it: 65536 x 7168, 13
      // tokens, G = 64, 98 us, now 90); with 128 two loops need more registers (R = 4: 55 -> 57).
      auto multiply = [&](auto groups_here) {
        constexpr int RR = decltype(groups_here)::value;
        for (int kb0 = 0; kb0 < KB; kb0 += split) {
          if (alive) alive = wait_bounded(smem_addr(&full[s]), phase, abort_flag, p.status, kStW4, p.timeout_ns);
          __syncwarp();
          const int kb = kb0 + slice;
          if (kb < KB) {
            const uint32_t st = ring + s * stage_bytes;
            const int left = p.K - kb * kBlkK;    // k of this block inside K
            // the block's first row of scales: its own, or that of the group it lies in
            int srow = slice * S::kGroups;
            if (FL == 128 && p.G != 128)
              srow = kb * kBlkK / p.G - kb0 * kBlkK / p.G;
            float d[RR][NT][4];
            uint32_t mz[RR][2];                    // minus the zero points of rows g, g + 8
            uint32_t wl[RR][S::kWords], wh[RR][S::kWords];   // their words
#pragma unroll (RR == 4 && NT == 1 && (FL == 32 || (FL == 64 && ZP)) ? FL / 32 : 4)
            for (int j = 0; j < 4; ++j) {         // 32 k each
              // past K: no tokens there, and the next expert's scales, which may be infinite
              if (FL < 128 && j / S::kWords * S::kWords * 32 >= left) break;
              const bool first = j * 32 % FL == 0;
              if (first) {
                const uint32_t zp = st + z_at + (srow + j * 32 / FL) * box_rows;
#pragma unroll
                for (int r = 0; r < RR; ++r) {
                  mz[r][0] = mz[r][1] = C::kMinusEight;
                  if (ZP) {
                    mz[r][0] = mul2<T>((lds8(zp + loaded(r) * 16) & 15u) * 0x00010001u, C::kNegate);
                    mz[r][1] = mul2<T>((lds8(zp + loaded(r) * 16 + 8) & 15u) * 0x00010001u, C::kNegate);
                  }
                }
              }
              const int chunk = 4 * S::kWords * (j / S::kWords) + j % S::kWords;   // + WV q: the lane's 8 k
              uint32_t b[NT][4];
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const uint4 v = lds128(st + x_at[n] + chunk * 16);
                b[n][0] = __byte_perm(v.x, v.z, 0x5410);      // x0, x4
                b[n][1] = __byte_perm(v.x, v.z, 0x7632);      // x1, x5
                b[n][2] = __byte_perm(v.y, v.w, 0x5410);      // x2, x6
                b[n][3] = __byte_perm(v.y, v.w, 0x7632);      // x3, x7
              }
              if (j % S::kWords == 0) {
                // part j / WV: 16 bytes on (WV = 1), 32 bytes on (WV = 2)
                const uint32_t wj = (st + w_at) ^ (S::kWords == 1 ? j << 4 : (j >> 1) << 5);
#pragma unroll
                for (int r = 0; r < RR; ++r) {
                  lds_words(wj + r * 1024, wl[r]);
                  lds_words(wj + r * 1024 + 512, wh[r]);
                }
              }
#pragma unroll
              for (int r = 0; r < RR; ++r) {
                if (FL == 128 && r == R - 1 && !full_part) break;
                uint32_t l[4], h[4];
                unpack_codes<T>(wl[r][j % S::kWords], mz[r][0], l);
                unpack_codes<T>(wh[r][j % S::kWords], mz[r][1], h);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  mma_step<T>(d[r][n], first, l[0], h[0], l[1], h[1], b[n][0], b[n][1]);
                  mma_step<T>(d[r][n], false, l[2], h[2], l[3], h[3], b[n][2], b[n][3]);
                }
              }
              if ((j + 1) * 32 % FL == 0) {
                const uint32_t sp = st + s_at + (srow + j * 32 / FL) * box_rows * es;
                float scale[RR][2];
                if (p.scale_f32) {
#pragma unroll
                  for (int r = 0; r < RR; ++r) {
                    scale[r][0] = __uint_as_float(lds32(sp + loaded(r) * 64));
                    scale[r][1] = __uint_as_float(lds32(sp + loaded(r) * 64 + 32));
                  }
                } else {
#pragma unroll
                  for (int r = 0; r < RR; ++r) {
                    scale[r][0] = scale_of(lds16(sp + loaded(r) * 32), static_cast<T*>(nullptr));
                    scale[r][1] = scale_of(lds16(sp + loaded(r) * 32 + 16), static_cast<T*>(nullptr));
                  }
                }
#pragma unroll
                for (int r = 0; r < RR; ++r) {
                  if (FL == 128 && r == R - 1 && !full_part) break;
#pragma unroll
                  for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[r][n][i] = fmaf(scale[r][i / 2], d[r][n][i], acc[r][n][i]);
                }
              }
            }
          }
          __syncwarp();                           // every lane has read the stage
          if (lane == 0) mbar_arrive(smem_addr(&empty[s]));
          if (++s == p.stages) {
            s = 0;
            phase ^= 1u;
          }
        }
      };
      if (FL == 128 || full_part)
        multiply(std::integral_constant<int, R>());
      else
        multiply(std::integral_constant<int, R - 1>());
      const unsigned rows_with_x = __ballot_sync(0xffffffffu, lane < it.count && x_row_of(it.row0 + lane) >= 0);
      T* y = static_cast<T*>(p.y) + static_cast<int64_t>(it.row0) * p.ldy;
      if (split == 1) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int m = 8 * n + 2 * q + (i & 1), row = it.n0 + first_row + 16 * r + g + (i < 2 ? 0 : 8);
              if (m < it.count && row < p.N && (r < R - 1 || full_part))
                y[static_cast<int64_t>(m) * p.ldy + row] = C::from(rows_with_x >> m & 1u ? acc[r][n][i] * C::kScale : 0.0f);
            }
      } else {
        // the slices' partial sums [slice][row of the item], added in slice order
        float* mine = red + (slice * (kRows * share) + first_row + g) * kPitch + 2 * q;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (r == R - 1 && !full_part) break;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float* lo = mine + 16 * r * kPitch + 8 * n;
            float* hi = lo + 8 * kPitch;
            lo[0] = acc[r][n][0];
            lo[1] = acc[r][n][1];
            hi[0] = acc[r][n][2];
            hi[1] = acc[r][n][3];
          }
        }
        bar_sync(1, kWarps * 32);
        for (int o = threadIdx.x; o < item_rows * it.count; o += kWarps * 32) {
          const int m = o / item_rows, row = o - m * item_rows;
          const float* f = red + row * kPitch + m;
          float v = 0.0f;
          for (int w = 0; w < split; ++w) v += f[w * (kRows * share * kPitch)];
          if (it.n0 + row < p.N)
            y[static_cast<int64_t>(m) * p.ldy + it.n0 + row] = C::from(rows_with_x >> m & 1u ? v * C::kScale : 0.0f);
        }
        bar_sync(1, kWarps * 32);               // the partial sums may be overwritten
      }
    }
  }
  // rows of no expert
  for (int64_t r = routed_s + static_cast<int64_t>(blockIdx.x); r < p.rows; r += gridDim.x)
    for (int n = threadIdx.x; n < p.N; n += kThreads) static_cast<T*>(p.y)[r * p.ldy + n] = C::from(0.0f);
}

// ------------------------------------------------------------------- host --

static bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

constexpr int kMaxDevices = 64;
constexpr int kSmemMost = 226 * 1024, kSmemPair = 112 * 1024;   // a CTA alone on its SM, or one of two
static std::mutex g_mu;

// A plan: 16-row groups of a warp (R, or one fewer), slices of K, groups of an item,
// and what it is thought to take.
struct Plan {
  int R, split, groups;
  double us;
};

// Rounds of `items` over `at_once` places.  Where the number of items is a guess
// (`about`), the mean over guesses up to 9 % off.
static double rounds(double items, int at_once, bool about) {
  const double r = items / at_once;
  if (!about) return ceil(r);
  double sum = 0.0;
  for (int off = -9; off <= 9; off += 3) sum += ceil(r * (1.0 + 0.01 * off));
  return sum / 7.0;
}

// The cheapest R, split and item for `tiles` token tiles of up to 8 NT tokens.
// Measured on B200, in microseconds: a step of an item (one K block a warp) costs an
// SM 0.56 (R = 2) or 0.95 (R = 4) with 8 tokens and two CTAs on it, 0.93 or 1.65 with
// 16 tokens and one CTA; one CTA of two, alone on its SM, takes 0.8 of two; joining the
// slices of an item costs 1.0 (R = 2) or 1.7 (R = 4) with eight, 0.8 with two or four,
// 0.3 with one.  (65536 x 7168, one token: R = 4 with two slices 58 us, R = 2 with one
// 68; 7168 x 2048: R = 2 with eight slices 10-11, R = 4 12; 8192 x 7168, 16 tokens:
// R = 4 22, R = 2 29.)
// Items need not be full: N = 65536 makes 256 items of 256 rows, two on 108 SMs and
// one on 40, but 293 of 224 rows, two on nearly all (58 -> 55 us with one token).  A
// warp's last rows cost about half as much as the mean (its other rows hide them).
// The width of a group and zero points are not in it (47 tokens x 6 of 64 experts,
// 7168 x 2048, groups of 32 with zero points: 102 us by the model, 126-143 measured); what
// counts is the order of the plans.  Over 59 calls of all widths the plan was 3 % slower
// than the best of all plans (mean; 23 % at most).
static Plan plan(int NT, double tiles, bool about, int N, int K, int sms) {
  Plan best = {2, kWarps, 2, 1e30};
  const int KB = (K + kBlkK - 1) / kBlkK;
  for (int R = 2; R <= 4; R += 2) {
    const double step = NT == 1 ? (R == 2 ? 0.56 : 0.95) : (R == 2 ? 0.93 : 1.65);
    const int ctas = NT == 1 ? 2 : 1;
    for (int split = kWarps; split >= 1; split /= 2) {
      const int share = kWarps / split, steps = (KB + split - 1) / split;
      const double join = split == kWarps ? (R == 2 ? 1.0 : 1.7) : split > 1 ? 0.8 : 0.3;
      const int least = (R - 1) * share + 1;
      for (int groups = R * share; groups >= least; --groups) {
        if (groups > 16 && (groups % 2 || groups / 2 <= (R - 1) * (share / 2))) continue;   // two even boxes
        const double items = tiles * ((N / 16 + groups - 1) / groups);
        const double work = steps * step * (0.5 + 0.5 * groups / (R * share));
        const double busy = rounds(items, sms, about) * (work + join);
        const double alone = rounds(items, sms * ctas, about) * (0.8 * ctas * work + join);
        const double us = busy > alone ? busy : alone;
        if (us < best.us) best = {R, split, groups, us};
      }
    }
  }
  return best;
}

template <typename T, int R, int NT, int FL, bool ZP>
static int launch(Args& a, int sms, cudaStream_t s) {
  using S = Stage<R, FL>;
  const auto kernel = gemv_w4_kernel<T, R, NT, FL, ZP>;
  const int es = a.scale_f32 ? 4 : 2;
  const int room = a.offsets ? (a.E < a.rows ? a.E : a.rows) : 1;
  const int stage = S::bytes(a.tile, a.split, a.groups, es, ZP);
  const int rest = Sums<R, NT>::bytes(a.split) + (4 * room + 1) * static_cast<int>(sizeof(int));
  const bool pair = NT == 1 && rest + 2 * stage <= kSmemPair;
  a.stages = ((pair ? kSmemPair : kSmemMost) - rest) / stage;
  if (a.stages > kMaxStages) a.stages = kMaxStages;
  if (a.stages < 1) return record_error(FACK_ERR_LAUNCH, "the 4-bit kernel's stage does not fit an SM");
  const int smem = a.stages * stage + rest;
  int dev = 0, per_sm = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return FACK_ERR_CUDA;
  {
    // resident CTAs an SM: host-side queries, kept per device for this variant's last size
    static int last[kMaxDevices][2] = {};
    std::lock_guard<std::mutex> lk(g_mu);
    if (last[dev][0] != smem) {
      cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
      if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, smem);
      if (e != cudaSuccess || per_sm < 1)
        return record_error(FACK_ERR_LAUNCH, e != cudaSuccess ? cudaGetErrorString(e) : "the 4-bit kernel does not fit an SM");
      last[dev][0] = smem;
      last[dev][1] = per_sm;
    }
    per_sm = last[dev][1];
  }
  const int64_t rows = 16 * a.groups, ntiles = (a.N + rows - 1) / rows, slots = static_cast<int64_t>(sms) * per_sm;
  // at most this many items: every expert with rows starts one token tile, every a.tile rows fill one
  const int64_t most = (a.rows / a.tile + static_cast<int64_t>(room) + 1) * ntiles;
  if (most > INT32_MAX - slots) return FACK_ERR_BAD_SHAPE;
  CUtensorMap wm, sm, zm;
  const uint64_t E = a.E, N = a.N, K = a.K, groups = a.K / a.G;
  int st = encode_elems_2d(&wm, a.w, 1, K / 2, E * N, K / 2, kBlkK / 2, S::box_rows(a.groups), true);
  if (st == FACK_OK)
    st = encode_elems_2d(&sm, a.scales, es, N, E * groups, N * es, S::box_rows(a.groups), a.split * S::kGroups, false);
  if (st == FACK_OK) {
    if (ZP)
      st = encode_elems_2d(&zm, a.zeros, 1, N, E * groups, N, S::box_rows(a.groups), a.split * S::kGroups, false);
    else
      zm = sm;                                  // not used
  }
  if (st != FACK_OK) return record_error(st, "the tensor map of the 4-bit weight was refused");
  kernel<<<static_cast<unsigned>(most < slots ? most : slots), kThreads, smem, s>>>(wm, sm, zm, a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? FACK_OK : record_error(FACK_ERR_LAUNCH, cudaGetErrorString(e));
}

template <typename T, int FL, bool ZP>
static int by_plan(Args& a, int NT, int R, int sms, cudaStream_t s) {
  if (NT == 1) return R == 2 ? launch<T, 2, 1, FL, ZP>(a, sms, s) : launch<T, 4, 1, FL, ZP>(a, sms, s);
  return R == 2 ? launch<T, 2, 2, FL, ZP>(a, sms, s) : launch<T, 4, 2, FL, ZP>(a, sms, s);
}

template <typename T, bool ZP>
static int by_group(Args& a, int NT, int R, int sms, cudaStream_t s) {
  if (a.G % 128 == 0) return by_plan<T, 128, ZP>(a, NT, R, sms, s);
  return a.G == 64 ? by_plan<T, 64, ZP>(a, NT, R, sms, s) : by_plan<T, 32, ZP>(a, NT, R, sms, s);
}

// Token tiles that T tokens of topk experts each are expected to take, chosen at
// random without repeats: E times the mean of ceil(x / tile) over a binomial x.
static double expected_tiles(int T, int topk, int E, int tile) {
  const double q = static_cast<double>(topk) / E, mean = q * T;
  if (q >= 1.0) return static_cast<double>(E) * ((static_cast<int64_t>(T) * topk / E + tile - 1) / tile);
  const double none = T * log1p(-q);            // logarithm of the chance that no token takes an expert
  if (mean > 200.0 || none < -700.0) return E * (mean / tile + 0.5);
  double sum = 0.0, p = exp(none);
  for (int x = 1; x <= T && x < 600; ++x) {
    p *= static_cast<double>(T - x + 1) / x * q / (1.0 - q);
    sum += p * ((x + tile - 1) / tile);
  }
  return E * sum;
}

// Tokens per tile (8 NT at most) and the plan.  An expert's rows are known on the
// device alone; it is not likely to have more than there are tokens, and one token has topk.
static void choose(Args& a, bool experts, int tokens, int sms, int* NT, int* R) {
  Plan p[2];
  int tile[2];
  for (int i = 0; i < 2; ++i) {
    const int most = 8 * (i + 1);
    double tiles;
    if (experts) {
      tile[i] = tokens < most ? tokens : most;
      tiles = expected_tiles(tokens, a.topk, a.E, tile[i]);
    } else {
      const int64_t n = (static_cast<int64_t>(a.rows) + most - 1) / most;
      tile[i] = static_cast<int>((a.rows + n - 1) / n);      // evenly filled
      tiles = static_cast<double>(n);
    }
    p[i] = plan(i + 1, tiles, experts && tokens > 1, a.N, a.K, sms);
  }
  const int i = tile[1] > 8 && p[1].us < p[0].us;
  *NT = i + 1;
  *R = p[i].R;
  a.tile = tile[i];
  a.split = p[i].split;
  a.groups = p[i].groups;
}

static int check_shape(const Args& a) {
  if (a.rows < 1 || a.N < 16 || a.N % 16 || a.N > (1 << 24) || a.K < 32 || a.K > (1 << 20)) return FACK_ERR_BAD_SHAPE;
  if ((a.G != 32 && a.G != 64 && (a.G < 128 || a.G % 128)) || a.K % a.G) return FACK_ERR_BAD_ARG;
  return FACK_OK;
}

static int run(Args& a, int dtype, int scale_dtype, int tokens, void* stream) {
  int st = check_shape(a);
  if (st != FACK_OK) return st;
  if (dtype != FACK_DTYPE_BF16 && dtype != FACK_DTYPE_F16) return FACK_ERR_BAD_ARG;
  if (scale_dtype != FACK_DTYPE_F32 && scale_dtype != dtype) return FACK_ERR_BAD_ARG;
  if (!a.x || !a.w || !a.scales || !a.y || !aligned(a.x, 16) || !aligned(a.w, 16) || !aligned(a.scales, 16) ||
      !aligned(a.zeros, 16) || !aligned(a.y, 2))
    return FACK_ERR_BAD_ALIGN;
  if (a.ldx < 0 || a.ldx % 8 || a.ldy < a.N) return FACK_ERR_BAD_STRIDE;
  int sms = 0;
  st = sm100_device(&sms);
  if (st != FACK_OK) return st;
  a.scale_f32 = scale_dtype == FACK_DTYPE_F32;
  a.status = device_status_word();
  a.timeout_ns = 2000000000ull;                // 2 s
  if (!a.status) return FACK_ERR_CUDA;
  // the copies count rows in 32 bits
  if (static_cast<int64_t>(a.E) * a.N > INT32_MAX - 1024 || static_cast<int64_t>(a.E) * (a.K / a.G) > INT32_MAX - 1024)
    return FACK_ERR_BAD_SHAPE;
  int NT, R;
  choose(a, a.offsets != nullptr, tokens, sms, &NT, &R);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == FACK_DTYPE_BF16)
    return a.zeros ? by_group<__nv_bfloat16, true>(a, NT, R, sms, s) : by_group<__nv_bfloat16, false>(a, NT, R, sms, s);
  return a.zeros ? by_group<__half, true>(a, NT, R, sms, s) : by_group<__half, false>(a, NT, R, sms, s);
}

}  // namespace fack_w4

extern "C" {

int fack_gemv_w4_plan(int tokens, int topk, int num_experts, int N, int K, int group, int* tile, int* warp_groups, int* split,
                      int* item_groups) {
  using namespace fack_w4;
  Args a = {};
  const bool experts = topk != 0 || num_experts != 0;
  if (tokens < 1 || (experts && (topk < 1 || topk > kMaxTopk || num_experts < 1 || num_experts > kMaxExperts ||
                                 static_cast<int64_t>(tokens) * topk > INT32_MAX)))
    return FACK_ERR_BAD_SHAPE;
  a.topk = experts ? topk : 1;
  a.E = experts ? num_experts : 1;
  a.rows = tokens * a.topk;
  a.N = N;
  a.K = K;
  a.G = group;
  int st = check_shape(a);
  if (st != FACK_OK) return st;
  if (!tile || !warp_groups || !split || !item_groups) return FACK_ERR_BAD_ARG;
  int sms = 0;
  st = sm100_device(&sms);
  if (st != FACK_OK) return st;
  int NT;
  choose(a, experts, tokens, sms, &NT, warp_groups);
  *tile = a.tile;
  *split = a.split;
  *item_groups = a.groups;
  return FACK_OK;
}

int fack_gemv_w4(const void* x, int dtype, int64_t ldx, const void* w, const void* scales, int scale_dtype,
                 const void* zeros, int group, void* y, int64_t ldy, int M, int N, int K, void* stream) {
  using namespace fack_w4;
  Args a = {};
  a.x = x;
  a.ldx = ldx;
  a.w = static_cast<const uint8_t*>(w);
  a.scales = scales;
  a.zeros = static_cast<const uint8_t*>(zeros);
  a.y = y;
  a.ldy = ldy;
  a.rows = M;
  a.topk = 1;
  a.N = N;
  a.K = K;
  a.G = group;
  a.E = 1;
  return run(a, dtype, scale_dtype, M, stream);
}

int fack_gemv_w4_experts(const void* x, int dtype, int64_t ldx, const void* w, const void* scales, int scale_dtype,
                         const void* zeros, int group, const int32_t* src, const int32_t* offsets, int T, int topk,
                         int num_experts, void* y, int64_t ldy, int N, int K, void* stream) {
  using namespace fack_w4;
  if (T < 1 || topk < 1 || topk > kMaxTopk || num_experts < 1 || num_experts > kMaxExperts ||
      static_cast<int64_t>(T) * topk > INT32_MAX)
    return FACK_ERR_BAD_SHAPE;
  if (!offsets || !aligned(offsets, 4) || !aligned(src, 4)) return FACK_ERR_BAD_ALIGN;
  Args a = {};
  a.x = x;
  a.ldx = ldx;
  a.w = static_cast<const uint8_t*>(w);
  a.scales = scales;
  a.zeros = static_cast<const uint8_t*>(zeros);
  a.y = y;
  a.ldy = ldy;
  a.src = src;
  a.offsets = offsets;
  a.rows = T * topk;
  a.topk = topk;
  a.N = N;
  a.K = K;
  a.G = group;
  a.E = num_experts;
  return run(a, dtype, scale_dtype, T, stream);
}

}  // extern "C"
