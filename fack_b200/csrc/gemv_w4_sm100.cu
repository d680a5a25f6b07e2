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
//     rows x 8 tokens.  A code is turned into the 16-bit float c - z exactly
//     (c is or-ed into the low mantissa bits of 128 or 1024, one subtraction
//     takes the offset and the zero point away), so the MMA's products are
//     exact and the only roundings are fp32 additions, the fp32 scale per
//     group, and the last one to the output type.
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
  int tokens_held;                             // tokens per tile that have room in a stage (<= 8 NT)
  int scale_f32;
};

template <typename T> struct Num;
template <> struct Num<__nv_bfloat16> {
  using T2 = __nv_bfloat162;
  static constexpr uint32_t kMagic = 0x43004300u;           // 128, one code step is one unit in the last place
  static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Num<__half> {
  using T2 = __half2;
  static constexpr uint32_t kMagic = 0x64006400u;           // 1024
  static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};

template <typename T>
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  using T2 = typename Num<T>::T2;
  const T2 r = __hsub2(*reinterpret_cast<const T2*>(&a), *reinterpret_cast<const T2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16*) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half*) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// One warp's stage of the ring: 16R weight rows of 64 bytes (16-byte chunk c of
// row r at c ^ (r/2 & 3): the reads of a word per row and quad lane have no bank
// conflict), the tokens' rows of 256 bytes (chunk c of token m at c ^ 4(m & 1)),
// the groups' scales and zero points of the 16R rows.
template <int R, int NT, int FL>
struct Stage {
  static constexpr int kGroups = kBlkK / FL;
  static constexpr int kRows = 16 * R;
  static constexpr int kScaleAt = kRows * 64;
  static constexpr int kZeroAt = kScaleAt + kGroups * kRows * 4;
  static constexpr int kTokenAt = kZeroAt + kGroups * kRows;
  static int bytes(int tokens_held) { return kTokenAt + tokens_held * 256; }
  static constexpr int kPitch = 8 * NT + 1;    // of a row in the partial sums
  static constexpr int kRedBytes = kWarps * kRows * kPitch * 4;
};

struct Item {
  int expert, n0, row0, count;
};

template <typename T, int R, int NT, int FL, int STAGES>
__global__ void __launch_bounds__(kThreads) gemv_w4_kernel(const __grid_constant__ Args p) {
  using S = Stage<R, NT, FL>;
  constexpr int kRows = S::kRows, kTok = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  // the experts that have rows: their number, first sorted row, and running count of token tiles
  __shared__ int act_expert[kMaxExperts], act_row[kMaxExperts], act_end[kMaxExperts], act_tile[kMaxExperts + 1];
  __shared__ int part[2][kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int stage_bytes = S::kTokenAt + p.tokens_held * 256;
  float* red = reinterpret_cast<float*>(smem);
  uint8_t* ring = smem + S::kRedBytes + warp * (STAGES * stage_bytes);
  const uint32_t ring_addr = smem_addr(ring);

  // ------------------------------------------------------------ item list --
  int routed = p.rows;
  if (p.offsets == nullptr) {
    if (threadIdx.x == 0) {
      act_expert[0] = 0;
      act_row[0] = 0;
      act_end[0] = p.rows;
      act_tile[0] = 0;
      act_tile[1] = (p.rows + kTok - 1) / kTok;
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
        if (last[i] > first[i]) tiles[i] = (last[i] - first[i] + kTok - 1) / kTok;
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
    for (int i = 0; i < warp; ++i) {
      st += part[0][i];
      sa += part[1][i];
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
  int active = 1;
  if (p.offsets != nullptr) {
    active = 0;
    for (int i = 0; i < kWarps; ++i) active += part[1][i];
  }
  __syncthreads();
  const int ntiles = (p.N + kRows - 1) / kRows;
  const int items = act_tile[active] * ntiles;
  const int KB = (p.K + kBlkK - 1) / kBlkK;
  const int groups = p.K / p.G;

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
    it.row0 = act_row[at] + m * kTok;
    it.count = min(kTok, act_end[at] - it.row0);
    return it;
  };

  // ------------------------------------------------------------- producer --
  const int es = p.scale_f32 ? 4 : 2;
  int i_item = blockIdx.x, i_kb = warp, i_at = 0, i_stage = 0;
  Item in = {0, 0, 0, 0};
  int64_t in_row = -1;                          // x row of token `lane` of the tile (lane < kTok)
  auto open = [&]() {                           // the issue side turns to item i_item
    in = decode(i_item, i_at);
    in_row = -1;
    if (lane < in.count) {
      const int r = in.row0 + lane;
      if (p.src == nullptr) {
        in_row = r;
      } else {
        const int pair = p.src[r];
        if (pair >= 0 && pair < p.rows) in_row = pair / p.topk;
      }
    }
  };
  const bool busy = warp < KB;                  // has K blocks at all
  if (busy && i_item < items) open();
  auto issue = [&]() {
    if (busy && i_item < items) {
      const uint32_t dst = ring_addr + i_stage * stage_bytes;
      const int k0 = i_kb * kBlkK;
      {
        const int r = lane >> 2, c = lane & 3;
        const bool k_in = k0 + 32 * c < p.K;
        const uint8_t* w = p.w + (static_cast<int64_t>(in.expert) * p.N + in.n0 + r) * (p.K / 2) + k0 / 2 + c * 16;
#pragma unroll
        for (int i = 0; i < kRows / 8; ++i) {
          const int row = r + 8 * i;
          const bool ok = k_in && in.n0 + row < p.N;
          cp_async16_cg_fill(dst + row * 64 + ((c ^ ((row >> 1) & 3)) << 4),
                             ok ? w + static_cast<int64_t>(8 * i) * (p.K / 2) : p.w, ok ? 16u : 0u);
        }
      }
      {
        const int c = lane & 15;
        const bool k_in = k0 + 8 * c < p.K;
#pragma unroll
        for (int i = 0; i < kTok / 2; ++i) {
          const int m = 2 * i + (lane >> 4);
          const int64_t row = __shfl_sync(0xffffffffu, in_row, m);
          if (2 * i < p.tokens_held && m < p.tokens_held) {
            const bool ok = k_in && row >= 0;
            const uint8_t* x = static_cast<const uint8_t*>(p.x);
            cp_async16_cg_fill(dst + S::kTokenAt + m * 256 + ((c ^ (4 * (m & 1))) << 4),
                               ok ? x + (row * p.ldx + k0 + 8 * c) * 2 : x, ok ? 16u : 0u);
          }
        }
      }
      {
        const int per = kRows * es / 16;        // chunks of a group's scales
        for (int i = lane; i < S::kGroups * per; i += 32) {
          const int gi = i / per, c = i - gi * per;
          const int k = k0 + gi * FL;
          const bool ok = k < p.K && in.n0 + c * (16 / es) < p.N;
          const uint8_t* s = static_cast<const uint8_t*>(p.scales);
          cp_async16_cg_fill(dst + S::kScaleAt + gi * (kRows * 4) + c * 16,
                             ok ? s + ((static_cast<int64_t>(in.expert) * groups + k / p.G) * p.N + in.n0) * es + c * 16 : s,
                             ok ? 16u : 0u);
        }
        if (p.zeros != nullptr && lane < S::kGroups * R) {
          const int gi = lane / R, c = lane - gi * R;
          const int k = k0 + gi * FL;
          const bool ok = k < p.K && in.n0 + c * 16 < p.N;
          cp_async16_cg_fill(dst + S::kZeroAt + gi * kRows + c * 16,
                             ok ? p.zeros + (static_cast<int64_t>(in.expert) * groups + k / p.G) * p.N + in.n0 + c * 16 : p.zeros,
                             ok ? 16u : 0u);
        }
      }
      i_stage = i_stage + 1 == STAGES ? 0 : i_stage + 1;
      i_kb += kWarps;
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
  int c_at = 0, c_stage = 0;
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
      const uint8_t* st = ring + c_stage * stage_bytes;
      c_stage = c_stage + 1 == STAGES ? 0 : c_stage + 1;
      float d[R][NT][4];
      uint32_t zlo[R], zhi[R];
#pragma unroll
      for (int j = 0; j < 4; ++j) {             // 32 k each
        if (j * 32 % FL == 0) {
          const int gi = j * 32 / FL;
#pragma unroll
          for (int r = 0; r < R; ++r) {
            uint32_t a = 8, b = 8;
            if (p.zeros != nullptr) {
              a = st[S::kZeroAt + gi * kRows + 16 * r + g] & 15u;
              b = st[S::kZeroAt + gi * kRows + 16 * r + g + 8] & 15u;
            }
            zlo[r] = Num<T>::kMagic | a * 0x00010001u;
            zhi[r] = Num<T>::kMagic | b * 0x00010001u;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) d[r][n][i] = 0.0f;
          }
        }
        uint32_t b[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int m = 8 * n + g;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (m < p.tokens_held)
            v = *reinterpret_cast<const uint4*>(st + S::kTokenAt + m * 256 + (((4 * j + q) ^ (4 * (g & 1))) << 4));
          b[n][0] = __byte_perm(v.x, v.z, 0x5410);          // x0, x4
          b[n][1] = __byte_perm(v.x, v.z, 0x7632);          // x1, x5
          b[n][2] = __byte_perm(v.y, v.w, 0x5410);          // x2, x6
          b[n][3] = __byte_perm(v.y, v.w, 0x7632);          // x3, x7
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int lo = 16 * r + g, hi = lo + 8;           // lo/2 and hi/2 agree mod 4
          const int at = ((j ^ ((g >> 1) & 3)) << 4) + q * 4;
          const uint32_t wl = *reinterpret_cast<const uint32_t*>(st + lo * 64 + at);
          const uint32_t wh = *reinterpret_cast<const uint32_t*>(st + hi * 64 + at);
          uint32_t l[4], h[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            l[i] = sub2<T>(((wl >> (4 * i)) & 0x000f000fu) | Num<T>::kMagic, zlo[r]);
            h[i] = sub2<T>(((wh >> (4 * i)) & 0x000f000fu) | Num<T>::kMagic, zhi[r]);
          }
          const uint32_t a0[4] = {l[0], h[0], l[1], h[1]}, a1[4] = {l[2], h[2], l[3], h[3]};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma16816(d[r][n], a0, b[n][0], b[n][1], static_cast<T*>(nullptr));
            mma16816(d[r][n], a1, b[n][2], b[n][3], static_cast<T*>(nullptr));
          }
        }
        if ((j + 1) * 32 % FL == 0) {
          const int gi = j * 32 / FL;
          const uint8_t* sp = st + S::kScaleAt + gi * (kRows * 4);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const int lo = 16 * r + g;
            float sl, sh;
            if (p.scale_f32) {
              sl = reinterpret_cast<const float*>(sp)[lo];
              sh = reinterpret_cast<const float*>(sp)[lo + 8];
            } else {
              sl = Num<T>::to(reinterpret_cast<const T*>(sp)[lo]);
              sh = Num<T>::to(reinterpret_cast<const T*>(sp)[lo + 8]);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              acc[r][n][0] = fmaf(sl, d[r][n][0], acc[r][n][0]);
              acc[r][n][1] = fmaf(sl, d[r][n][1], acc[r][n][1]);
              acc[r][n][2] = fmaf(sh, d[r][n][2], acc[r][n][2]);
              acc[r][n][3] = fmaf(sh, d[r][n][3], acc[r][n][3]);
            }
          }
        }
      }
    }
    // the warps' partial sums, added in warp order
    float* mine = red + warp * (kRows * S::kPitch);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float* lo = mine + (16 * r + g) * S::kPitch + 8 * n + 2 * q;
        float* hi = lo + 8 * S::kPitch;
        lo[0] = acc[r][n][0];
        lo[1] = acc[r][n][1];
        hi[0] = acc[r][n][2];
        hi[1] = acc[r][n][3];
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRows * kTok / kThreads; ++i) {
      const int o = i * kThreads + threadIdx.x, m = o / kRows, row = o - m * kRows;
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) s += red[(w * kRows + row) * S::kPitch + m];
      if (m < it.count && it.n0 + row < p.N)
        static_cast<T*>(p.y)[static_cast<int64_t>(it.row0 + m) * p.ldy + it.n0 + row] = Num<T>::from(s);
    }
    __syncthreads();                            // the partial sums may be overwritten
  }
  cp_async_wait<0>();
  // rows of no expert
  for (int64_t r = routed + static_cast<int64_t>(blockIdx.x); r < p.rows; r += gridDim.x)
    for (int n = threadIdx.x; n < p.N; n += kThreads) static_cast<T*>(p.y)[r * p.ldy + n] = Num<T>::from(0.0f);
}

// ------------------------------------------------------------------- host --

static bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

constexpr int kMaxDevices = 64;
constexpr int kSmemMost = 208 * 1024;     // dynamic; the item list is static beside it
static std::mutex g_mu;

template <typename T, int R, int NT, int FL, int STAGES>
static int launch(const Args& a, int sms, cudaStream_t s) {
  using S = Stage<R, NT, FL>;
  const auto kernel = gemv_w4_kernel<T, R, NT, FL, STAGES>;
  const int smem = S::kRedBytes + kWarps * STAGES * S::bytes(a.tokens_held);
  int dev = 0, per_sm = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return FACK_ERR_CUDA;
  {
    // resident CTAs an SM at this stage size: host-side queries, kept per device for this variant
    static int per_sm_at[kMaxDevices][8 * NT + 1] = {};
    std::lock_guard<std::mutex> lk(g_mu);
    if (!per_sm_at[dev][a.tokens_held]) {
      cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
      if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, smem);
      if (e != cudaSuccess || per_sm < 1)
        return record_error(FACK_ERR_LAUNCH, e != cudaSuccess ? cudaGetErrorString(e) : "the 4-bit kernel does not fit an SM");
      per_sm_at[dev][a.tokens_held] = per_sm;
    }
    per_sm = per_sm_at[dev][a.tokens_held];
  }
  // at most this many items: every expert with rows starts one token tile, every 8 NT rows fill one
  const int64_t ntiles = (a.N + S::kRows - 1) / S::kRows;
  const int64_t most = (a.rows / (8 * NT) + (a.E < a.rows ? a.E : a.rows) + 1) * ntiles;
  if (most > INT32_MAX) return FACK_ERR_BAD_SHAPE;
  const int64_t grid = most < static_cast<int64_t>(sms) * per_sm ? most : static_cast<int64_t>(sms) * per_sm;
  kernel<<<static_cast<unsigned>(grid), kThreads, smem, s>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? FACK_OK : record_error(FACK_ERR_LAUNCH, cudaGetErrorString(e));
}

template <typename T, int FL>
static int by_tokens(Args& a, int per_expert, int sms, cudaStream_t s) {
  if (per_expert <= 8) {
    a.tokens_held = a.rows < 8 ? a.rows : 8;
    return launch<T, 2, 1, FL, 4>(a, sms, s);
  }
  a.tokens_held = a.rows < 16 ? a.rows : 16;
  return launch<T, 2, 2, FL, 3>(a, sms, s);
}

template <typename T>
static int by_group(Args& a, int per_expert, int sms, cudaStream_t s) {
  if (a.G % 128 == 0) return by_tokens<T, 128>(a, per_expert, sms, s);
  return a.G == 64 ? by_tokens<T, 64>(a, per_expert, sms, s) : by_tokens<T, 32>(a, per_expert, sms, s);
}

static int run(Args& a, int dtype, int scale_dtype, int per_expert, void* stream) {
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
  return dtype == FACK_DTYPE_BF16 ? by_group<__nv_bfloat16>(a, per_expert, sms, s) : by_group<__half>(a, per_expert, sms, s);
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
  return run(a, dtype, scale_dtype, (a.rows + num_experts - 1) / num_experts, stream);
}

}  // extern "C"
