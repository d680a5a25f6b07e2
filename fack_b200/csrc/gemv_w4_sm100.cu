// gemv_w4_sm100.cu -- products of a few tokens with 4-bit weights (sm_100a).
//
//   y[m, n] = sum_k x[m, k] * (c[n, k] - z[k/G, n]) * s[k/G, n]
//
// with codes c in 0..15 packed two a byte along K (even k in the low nibble),
// one scale and optionally one zero point (else 8) per output row and group of
// G consecutive k, x and y bf16 or fp16.  With a plan of tokens sorted by
// expert the same for every expert's rows and weights.
//
// The call is the weight stream: N*K/2 bytes that are read once.  Everything
// here serves to keep that stream going:
//   * A CTA owns 16*R output rows; its 8 warps take the 128-wide K blocks in
//     turn (warp w the blocks w, w + 8, ...), so at any time the CTA reads 512
//     contiguous bytes of each row.  CTAs are persistent: each walks a list of
//     (expert, row tile, token tile) items with one running ring of cp.async
//     stages per warp, which goes on into the next item while the last one is
//     summed, and no barrier stands between a warp and its own loads.
//   * The products go to the warp MMA (m16n8k16, fp32 accumulators): 16 weight
//     rows x 8 tokens.  A code is turned into a 16-bit float of c - z exactly (see
//     Codes), so the MMA's products are exact and the only roundings are fp32
//     additions, the fp32 scale per group, and the last one to the output type.
//   * A word of 8 consecutive codes gives the pairs (i, i + 4) by one shift and
//     mask each; the tokens are put in the same order (the MMA does not care
//     which k goes where, if both operands agree).
// The warp MMA, not tcgen05: 8 or 16 tokens fill a fraction of a tcgen05 tile,
// 4-bit codes with arbitrary scales are no operand type of it, and dequantised
// tiles would have to pass through shared memory once more.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>

#include "../../include/fack_gemm.h"
#include "fack_internal.h"
#include "sm100_ptx.cuh"

namespace fack_w4 {

using namespace fack;

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kBlkK = 128;                     // k per stage
constexpr int kMaxExperts = 1024;
constexpr int kMaxTopk = 64;

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
  int scale_f32;
};

// A word's codes 0..7 as four registers of two 16-bit floats each, (c - z) *
// kUnit exactly, codes i and i + 4 together.  A masked code is a subnormal, c or
// 16c units of the type's smallest (in bf16 the top bit of 16c is the exponent's
// lowest, where the normal numbers go on at the same spacing), and one fused
// multiply-add scales it and takes the zero point away: 1 shift, 4 masks, 4 fma
// for 8 codes.  The ALU, which has half the rate of the fma pipe, does the rest
// of the address work too and is what the kernel ran out of with more shifts.
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

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1, __nv_bfloat16*) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1, __half*) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// d (+)= a * b: the first product of a group starts from zero
template <typename T>
__device__ __forceinline__ void mma_step(float (&d)[4], bool first, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  if (first) d[0] = d[1] = d[2] = d[3] = 0.0f;
  mma16816(d, a0, a1, a2, a3, b0, b1, static_cast<T*>(nullptr));
}

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
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

// One warp's stage of the ring: 16R weight rows of 64 bytes (16-byte chunk c of
// row r at c ^ (r/2 & 3): the reads of a word per row and quad lane have no bank
// conflict), the tokens' rows of 256 bytes (chunk c of token m at c ^ 4(m & 1)),
// the groups' scales and zero points of the 16R rows.  A multiple of 256 bytes, so
// that the exclusive-or can be done on addresses.
template <int R, int FL>
struct Stage {
  static constexpr int kGroups = kBlkK / FL;
  static constexpr int kRows = 16 * R;
  static constexpr int kTokenAt = kRows * 64;
  __host__ __device__ static int scale_at(int tile) { return kTokenAt + tile * 256; }
  __host__ __device__ static int zero_at(int tile, int es) { return scale_at(tile) + kGroups * kRows * es; }
  __host__ __device__ static int bytes(int tile, int es, bool zeros) {
    return (zero_at(tile, es) + (zeros ? kGroups * kRows : 0) + 255) / 256 * 256;
  }
};
template <int R, int NT>
struct Sums {                                  // the warps' partial sums
  static constexpr int kPitch = 8 * NT + 1;
  static constexpr int kBytes = kWarps * 16 * R * kPitch * 4;
};

struct Item {
  int expert, n0, row0, count;
};

template <typename T, int R, int NT, int FL, bool ZP, int STAGES>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1) gemv_w4_kernel(const __grid_constant__ Args p) {
  using S = Stage<R, FL>;
  using C = Codes<T>;
  constexpr int kRows = S::kRows, kPitch = Sums<R, NT>::kPitch;
  extern __shared__ __align__(256) uint8_t smem[];
  __shared__ int part[2][kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int es = p.scale_f32 ? 4 : 2;
  const int stage_bytes = S::bytes(p.tile, es, ZP);
  const uint32_t ring = smem_addr(smem) + warp * (STAGES * stage_bytes);
  float* red = reinterpret_cast<float*>(smem + kWarps * STAGES * stage_bytes);
  // the experts that have rows: number, first and last sorted row, running count of token tiles
  const int room = p.offsets == nullptr ? 1 : min(p.E, p.rows);
  int* act_expert = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(red) + Sums<R, NT>::kBytes);
  int* act_row = act_expert + room;
  int* act_end = act_row + room;
  int* act_tile = act_end + room;

  // ------------------------------------------------------------ item list --
  int routed = p.rows, active = 1;
  if (p.offsets == nullptr) {
    if (threadIdx.x == 0) {
      act_expert[0] = 0;
      act_row[0] = 0;
      act_end[0] = p.rows;
      act_tile[0] = 0;
      act_tile[1] = (p.rows + p.tile - 1) / p.tile;
    }
  } else {
    constexpr int kPer = kMaxExperts / kThreads;
    int tiles[kPer], first[kPer], last[kPer], my_tiles = 0, my_act = 0, bad = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = threadIdx.x * kPer + i;
      tiles[i] = 0;
      if (e < p.E) {
        first[i] = p.offsets[e];
        last[i] = p.offsets[e + 1];
        bad |= first[i] < 0 || last[i] < first[i] || last[i] > p.rows;
        if (last[i] > first[i]) tiles[i] = (last[i] - first[i] + p.tile - 1) / p.tile;
      }
      my_tiles += tiles[i];
      my_act += tiles[i] > 0;
    }
    // offsets that do not ascend within the rows are no plan: nothing is routed
    if (__syncthreads_or(bad)) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) tiles[i] = 0;
      my_tiles = my_act = 0;
      routed = 0;
    } else {
      routed = p.offsets[p.E];
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
    for (int i = 0; i < kWarps; ++i) {
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
  const int ntiles = (p.N + kRows - 1) / kRows;
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
    it.n0 = n * kRows;
    it.row0 = act_row[at] + m * p.tile;
    it.count = min(p.tile, act_end[at] - it.row0);
    return it;
  };

  // ------------------------------------------------------------- producer --
  // Weights: lane -> row lane/4 + 8i, chunk lane%4.  Tokens: for at most two of
  // them 16 lanes each, else 4 lanes each and 4 turns (and the same for tokens
  // 8..15).  Tokens past the item's count are not copied: their columns of the
  // MMA touch no other and are not stored.
  const int64_t row_bytes = p.K / 2, row_step = row_bytes * 8;
  const bool pair = p.tile <= 2;
  const int x_tok = pair ? lane >> 4 : lane >> 2, x_chunk = pair ? lane & 15 : lane & 3;
  const uint32_t w_dst = (lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) << 4);
  const uint32_t x_dst = S::kTokenAt + x_tok * 256 + ((x_chunk ^ (4 * (x_tok & 1))) << 4);
  const int s_per = kRows * es / 16;            // chunks of a group's scales
  const int groups = p.K / p.G;
  // a lane's scale chunks (at most two) and zero-point chunk within a block
  const int64_t s_off = static_cast<int64_t>(lane / s_per) * p.N * es + (lane % s_per) * 16;
  const int64_t s_off2 = static_cast<int64_t>((lane + 32) / s_per) * p.N * es + ((lane + 32) % s_per) * 16;
  const int64_t z_off = static_cast<int64_t>(lane / R) * p.N + (lane % R) * 16;
  const uint8_t *w_src = nullptr, *x_src[NT], *s_src = nullptr, *z_src = nullptr;
  uint32_t x_size[NT];                          // 16, or 0 for a row of zeros
  bool x_on[NT];
  int valid16 = 0;                              // 16-row parts of the tile inside N
  int i_item = blockIdx.x, i_kb = warp, i_at = 0;
  uint32_t i_dst = ring;
  auto open = [&]() {                           // the copies turn to item i_item
    const Item in = decode(i_item, i_at);
    valid16 = min(R, (p.N - in.n0) >> 4);
    w_src = p.w + (static_cast<int64_t>(in.expert) * p.N + in.n0 + (lane >> 2)) * row_bytes + i_kb * (kBlkK / 2) + (lane & 3) * 16;
    const int64_t sn = static_cast<int64_t>(in.expert) * groups * p.N + in.n0;
    s_src = static_cast<const uint8_t*>(p.scales) + sn * es;
    z_src = p.zeros + sn;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int m = x_tok + 8 * n;
      x_on[n] = m < in.count;
      x_size[n] = 0;
      int64_t row = 0;
      if (x_on[n]) {
        row = in.row0 + m;
        if (p.src != nullptr) {
          const int from = p.src[row];
          const bool ok = from >= 0 && from < p.rows;
          row = ok ? from / p.topk : 0;
          x_size[n] = ok ? 16 : 0;
        } else {
          x_size[n] = 16;
        }
      }
      x_src[n] = static_cast<const uint8_t*>(p.x) + (row * p.ldx + i_kb * kBlkK + x_chunk * 8) * 2;
    }
  };
  const bool busy = warp < KB;                  // has K blocks at all
  if (busy && i_item < items) open();
  auto issue = [&]() {
    if (busy && i_item < items) {
      const uint32_t s_dst = i_dst + S::scale_at(p.tile) + lane * 16, z_dst = i_dst + S::zero_at(p.tile, es) + lane * 16;
      // a block's groups: its own 128/FL, or the one it lies in
      const int group = FL == 128 && p.G != 128 ? i_kb / (p.G / 128) : i_kb * S::kGroups;
      const uint8_t* sg = s_src + static_cast<int64_t>(group) * p.N * es;
      const uint8_t* zg = z_src + static_cast<int64_t>(group) * p.N;
      if (i_kb * kBlkK + kBlkK <= p.K && valid16 == R) {
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) cp_async16_cg(i_dst + w_dst + i * 512, w_src + i * row_step);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (!x_on[n]) continue;
          const uint32_t dst = i_dst + x_dst + n * (8 * 256);
          cp_async16_cg_fill(dst, x_src[n], x_size[n]);
          if (!pair) {
#pragma unroll
            for (int i = 1; i < 4; ++i) cp_async16_cg_fill(dst ^ (i << 6), x_src[n] + i * 64, x_size[n]);
          }
        }
        if (lane < S::kGroups * s_per) cp_async16_cg(s_dst, sg + s_off);
        if (S::kGroups * R * 4 > 32 && lane + 32 < S::kGroups * s_per) cp_async16_cg(s_dst + 512, sg + s_off2);
        if (ZP && lane < S::kGroups * R) cp_async16_cg(z_dst, zg + z_off);
      } else {
        const int left = p.K - i_kb * kBlkK;    // k of this block inside K
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) {
          const bool ok = (i >> 1) < valid16 && (lane & 3) * 32 < left;
          cp_async16_cg_fill(i_dst + w_dst + i * 512, ok ? w_src + i * row_step : p.w, ok ? 16u : 0u);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (!x_on[n]) continue;
          const uint32_t dst = i_dst + x_dst + n * (8 * 256);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (pair && i) break;
            const bool ok = x_chunk * 8 + i * 32 < left;
            cp_async16_cg_fill(dst ^ (i << 6), ok ? x_src[n] + i * 64 : p.x, ok ? x_size[n] : 0u);
          }
        }
        for (int i = lane; i < S::kGroups * s_per; i += 32) {
          const int gi = i / s_per, c = i - gi * s_per;
          const bool ok = group + gi < groups && (c * (16 / es)) >> 4 < valid16;
          cp_async16_cg_fill(s_dst + (i - lane) * 16, ok ? sg + static_cast<int64_t>(gi) * p.N * es + c * 16 : p.scales,
                             ok ? 16u : 0u);
        }
        if (ZP && lane < S::kGroups * R) {
          const bool ok = group + lane / R < groups && lane % R < valid16;
          cp_async16_cg_fill(z_dst, ok ? zg + z_off : p.zeros, ok ? 16u : 0u);
        }
      }
      i_dst = i_dst + stage_bytes == ring + STAGES * stage_bytes ? ring : i_dst + stage_bytes;
      i_kb += kWarps;
      w_src += kWarps * (kBlkK / 2);
#pragma unroll
      for (int n = 0; n < NT; ++n) x_src[n] += kWarps * kBlkK * 2;
      if (i_kb >= KB) {
        i_kb = warp;
        i_item += gridDim.x;
        if (i_item < items) open();
      }
    }
    cp_async_commit();                          // one group a step, empty past the end, so the counts hold
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue();

  // ------------------------------------------------------------- consumer --
  const uint32_t w_at = g * 64 + (((g >> 1) & 3) << 4) + q * 4;         // ^ 16j
  const uint32_t x_at = S::kTokenAt + g * 256 + ((g & 1) << 6) + q * 16;  // ^ 64j
  int c_at = 0;
  uint32_t st = ring;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const Item it = decode(item, c_at);
    float acc[R][NT][4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.0f;
    for (int kb = warp; kb < KB; kb += kWarps) {
      __syncwarp();                             // every lane has read the stage that is refilled next
      issue();
      cp_async_wait<STAGES - 1>();              // this lane's copies of the block have landed ...
      __syncwarp();                             // ... and every other lane's
      float d[R][NT][4];
      uint32_t mz[R][2];                        // minus the zero points of rows g, g + 8
#pragma unroll
      for (int j = 0; j < 4; ++j) {             // 32 k each
        const bool first = j * 32 % FL == 0;
        if (first) {
          const uint32_t zp = st + S::zero_at(p.tile, es) + (j * 32 / FL) * kRows + g;
#pragma unroll
          for (int r = 0; r < R; ++r) {
            mz[r][0] = mz[r][1] = C::kMinusEight;
            if (ZP) {
              mz[r][0] = mul2<T>((lds8(zp + r * 16) & 15u) * 0x00010001u, C::kNegate);
              mz[r][1] = mul2<T>((lds8(zp + r * 16 + 8) & 15u) * 0x00010001u, C::kNegate);
            }
          }
        }
        uint32_t b[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (8 * n + g < p.tile) v = lds128((st + x_at + n * (8 * 256)) ^ (j << 6));
          b[n][0] = __byte_perm(v.x, v.z, 0x5410);          // x0, x4
          b[n][1] = __byte_perm(v.x, v.z, 0x7632);          // x1, x5
          b[n][2] = __byte_perm(v.y, v.w, 0x5410);          // x2, x6
          b[n][3] = __byte_perm(v.y, v.w, 0x7632);          // x3, x7
        }
        const uint32_t wj = (st + w_at) ^ (j << 4);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          uint32_t l[4], h[4];
          unpack_codes<T>(lds32(wj + r * 1024), mz[r][0], l);
          unpack_codes<T>(lds32(wj + r * 1024 + 512), mz[r][1], h);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_step<T>(d[r][n], first, l[0], h[0], l[1], h[1], b[n][0], b[n][1]);
            mma_step<T>(d[r][n], false, l[2], h[2], l[3], h[3], b[n][2], b[n][3]);
          }
        }
        if ((j + 1) * 32 % FL == 0) {
          const uint32_t sp = st + S::scale_at(p.tile) + ((j * 32 / FL) * kRows + g) * es;
#pragma unroll
          for (int r = 0; r < R; ++r) {
            float sl, sh;
            if (p.scale_f32) {
              sl = __uint_as_float(lds32(sp + r * 64));
              sh = __uint_as_float(lds32(sp + r * 64 + 32));
            } else {
              sl = scale_of(lds16(sp + r * 32), static_cast<T*>(nullptr));
              sh = scale_of(lds16(sp + r * 32 + 16), static_cast<T*>(nullptr));
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[r][n][i] = fmaf(i < 2 ? sl : sh, d[r][n][i], acc[r][n][i]);
          }
        }
      }
      st = st + stage_bytes == ring + STAGES * stage_bytes ? ring : st + stage_bytes;
    }
    // the warps' partial sums, added in warp order
    float* mine = red + warp * (kRows * kPitch);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float* lo = mine + (16 * r + g) * kPitch + 8 * n + 2 * q;
        float* hi = lo + 8 * kPitch;
        lo[0] = acc[r][n][0];
        lo[1] = acc[r][n][1];
        hi[0] = acc[r][n][2];
        hi[1] = acc[r][n][3];
      }
    __syncthreads();
    for (int o = threadIdx.x; o < kRows * it.count; o += kThreads) {
      const int m = o / kRows, row = o - m * kRows;
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) s += red[(w * kRows + row) * kPitch + m];
      if (it.n0 + row < p.N)
        static_cast<T*>(p.y)[static_cast<int64_t>(it.row0 + m) * p.ldy + it.n0 + row] = C::from(s * C::kScale);
    }
    __syncthreads();                            // the partial sums may be overwritten
  }
  cp_async_wait<0>();
  // rows of no expert
  for (int64_t r = routed + static_cast<int64_t>(blockIdx.x); r < p.rows; r += gridDim.x)
    for (int n = threadIdx.x; n < p.N; n += kThreads) static_cast<T*>(p.y)[r * p.ldy + n] = C::from(0.0f);
}

// ------------------------------------------------------------------- host --

static bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

constexpr int kMaxDevices = 64;
constexpr int kSmemMost = 226 * 1024;
static std::mutex g_mu;

template <typename T, int R, int NT, int FL, bool ZP, int STAGES>
static int launch(const Args& a, int sms, cudaStream_t s) {
  const auto kernel = gemv_w4_kernel<T, R, NT, FL, ZP, STAGES>;
  const int room = a.offsets ? (a.E < a.rows ? a.E : a.rows) : 1;
  const int smem = kWarps * STAGES * Stage<R, FL>::bytes(a.tile, a.scale_f32 ? 4 : 2, ZP) + Sums<R, NT>::kBytes +
                   (4 * room + 1) * static_cast<int>(sizeof(int));
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
  // at most this many items: every expert with rows starts one token tile, every a.tile rows fill one
  const int64_t ntiles = (a.N + 16 * R - 1) / (16 * R);
  const int64_t most = (a.rows / a.tile + static_cast<int64_t>(room) + 1) * ntiles;
  if (most > INT32_MAX) return FACK_ERR_BAD_SHAPE;
  const int64_t grid = most < static_cast<int64_t>(sms) * per_sm ? most : static_cast<int64_t>(sms) * per_sm;
  kernel<<<static_cast<unsigned>(grid), kThreads, smem, s>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? FACK_OK : record_error(FACK_ERR_LAUNCH, cudaGetErrorString(e));
}

template <typename T, int FL, bool ZP>
static int by_tokens(Args& a, int per_expert, int tokens, int sms, cudaStream_t s) {
  if (per_expert <= 8) {
    a.tile = tokens < 8 ? tokens : 8;
    return a.tile <= 2 ? launch<T, 2, 1, FL, ZP, 4>(a, sms, s) : launch<T, 2, 1, FL, ZP, 3>(a, sms, s);
  }
  a.tile = tokens < 16 ? tokens : 16;
  return launch<T, 4, 2, FL, ZP, 2>(a, sms, s);
}

template <typename T, bool ZP>
static int by_group(Args& a, int per_expert, int tokens, int sms, cudaStream_t s) {
  if (a.G % 128 == 0) return by_tokens<T, 128, ZP>(a, per_expert, tokens, sms, s);
  return a.G == 64 ? by_tokens<T, 64, ZP>(a, per_expert, tokens, sms, s) : by_tokens<T, 32, ZP>(a, per_expert, tokens, sms, s);
}

static int run(Args& a, int dtype, int scale_dtype, int per_expert, int tokens, void* stream) {
  if (a.rows < 1 || a.N < 16 || a.N % 16 || a.N > (1 << 24) || a.K < 32 || a.K > (1 << 20)) return FACK_ERR_BAD_SHAPE;
  if ((a.G != 32 && a.G != 64 && (a.G < 128 || a.G % 128)) || a.K % a.G) return FACK_ERR_BAD_ARG;
  if (dtype != FACK_DTYPE_BF16 && dtype != FACK_DTYPE_F16) return FACK_ERR_BAD_ARG;
  if (scale_dtype != FACK_DTYPE_F32 && scale_dtype != dtype) return FACK_ERR_BAD_ARG;
  if (!a.x || !a.w || !a.scales || !a.y || !aligned(a.x, 16) || !aligned(a.w, 16) || !aligned(a.scales, 16) ||
      !aligned(a.zeros, 16) || !aligned(a.y, 2))
    return FACK_ERR_BAD_ALIGN;
  if (a.ldx < 0 || a.ldx % 8 || a.ldy < a.N) return FACK_ERR_BAD_STRIDE;
  int sms = 0;
  const int st = sm100_device(&sms);
  if (st != FACK_OK) return st;
  a.scale_f32 = scale_dtype == FACK_DTYPE_F32;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == FACK_DTYPE_BF16)
    return a.zeros ? by_group<__nv_bfloat16, true>(a, per_expert, tokens, sms, s)
                   : by_group<__nv_bfloat16, false>(a, per_expert, tokens, sms, s);
  return a.zeros ? by_group<__half, true>(a, per_expert, tokens, sms, s) : by_group<__half, false>(a, per_expert, tokens, sms, s);
}

}  // namespace fack_w4

extern "C" {

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
  return run(a, dtype, scale_dtype, M, M, stream);
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
  return run(a, dtype, scale_dtype, (a.rows + num_experts - 1) / num_experts, T, stream);
}

}  // extern "C"
