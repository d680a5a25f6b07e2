// moe_sm100.cu -- tokens sorted by expert and back (sm_100a).
//
// A routed layer sends token t's slot j to expert e = ids[t, j].  The pair
// p = t*topk + j gets the sorted row
//   r = offsets[e] + #{p' < p : ids[p'] = e},   offsets[e] = #{p' : 0 <= ids[p'] < e}
// (a stable counting sort).  row_of[t, j] = r and src[r] = p are each other's
// inverse; a pair whose id is outside [0, E) has no row (row_of = -1) and the
// rows behind offsets[E] have no pair (src = -1).  On that plan:
//   gather   y[r] = x[src[r] / topk]                        (0 without a pair)
//   quantise the same rows as e4m3 codes and per-128 scales, for the FP8 GEMM
//   combine  out[t] = sum_j w[t, j] * y[row_of[t, j]]        (fp32, slots in order)
//   backward of combine: dy[r] = w[t, j] * dout[t], dw[t, j] = <dout[t], y[r]>
// and the backward of gather is combine without weights.
//
// All of it is byte work.  The row kernels go by token, not by sorted row: a
// token's data is read once and its topk rows are written (or its topk rows
// read, all loads in flight together, and one row written), so each byte
// crosses HBM once and no sum needs an atomic.  Every index read from a plan
// is range-checked before it is used as an address.
//
// Measured on B200 (calls one after another in a replayed graph, share of the 6464 GB/s
// copy): gather 8192 x 8 rows of 7168 bf16 180 us (0.91), 4096 x 6 of 4096 fp16 39.5
// (0.92); combine 155 (1.05) and 39.4 (0.92); combine's gradients 316 (0.98) and 74 (0.91);
// the quantising gather 4095 x 4 of 7168 fp32 39.5 (0.93), 8192 x 2 of 7168 bf16 58 (0.64:
// 25 instructions an element for two bytes in and two out fill 76 % of the issue slots).
// Few tokens are bound by latency: 2.6-3.3 us to 16 tokens.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/fack_gemm.h"
#include "fack_internal.h"

namespace fack_moe {

constexpr int kBlk = 128;
constexpr float kQmax = 240.0f;
constexpr int kMaxExperts = 1024;
constexpr int kMaxTopk = 64;
constexpr int kMaxDim = 1 << 20;

// ------------------------------------------------------------------- sort --

constexpr int kSortRounds = 4;       // pairs per thread and chunk; their ranks stay in registers
constexpr int kSortMaxBlocks = 128;
// Shared memory of sort_place_kernel for `threads` threads; most, for 1024 experts and 1024 threads.
constexpr size_t sort_smem_bytes(int threads, int E) {
  return (E + 1) * sizeof(int) + static_cast<size_t>(threads / 32) * (E + 1) * sizeof(uint16_t);
}
constexpr int kSortSmemMost = static_cast<int>(sort_smem_bytes(1024, kMaxExperts));
constexpr size_t kSortSmemPlain = 47 * 1024;   // beside the kernel's static arrays this needs no opt-in

// Expert of pair p, or E when it is not routed here.  Ids are compared in
// their own width, so a 64-bit id never aliases a small one.
template <typename I>
__device__ __forceinline__ int expert_of(const I* __restrict__ ids, int64_t p, int64_t pairs, int E) {
  if (p >= pairs) return E;
  const I id = ids[p];
  return id >= 0 && id < static_cast<I>(E) ? static_cast<int>(id) : E;
}

// Exclusive scan of v over the block's threads (blockDim a multiple of 32);
// *total gets the sum.  `part` holds one int per warp plus one.
__device__ __forceinline__ int block_scan(int v, int* part, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int s = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, s, d);
    if (lane >= d) s += o;
  }
  if (lane == 31) part[warp] = s;
  __syncthreads();
  if (warp == 0) {
    int w = lane < warps ? part[lane] : 0;
    const int mine = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += o;
    }
    if (lane < warps) part[lane] = w - mine;
    if (lane == 31) part[32] = w;
  }
  __syncthreads();
  *total = part[32];
  return part[warp] + s - v;
}

// Counts of each block's contiguous share of the pairs: hist[block][E].
template <typename I>
__global__ void __launch_bounds__(1024) sort_count_kernel(const I* __restrict__ ids, int64_t pairs, int64_t share, int E,
                                                          int* __restrict__ hist) {
  __shared__ int cnt[kMaxExperts + 1];
  for (int e = threadIdx.x; e <= E; e += blockDim.x) cnt[e] = 0;
  __syncthreads();
  const int64_t begin = blockIdx.x * share;
  const int64_t end = begin + share < pairs ? begin + share : pairs;
  for (int64_t p = begin + threadIdx.x; p < end; p += blockDim.x) atomicAdd(&cnt[expert_of(ids, p, pairs, E)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += blockDim.x) hist[static_cast<int64_t>(blockIdx.x) * E + e] = cnt[e];
}

// Ranks and scatters each block's share, chunk by chunk.  A warp takes a
// contiguous run of a chunk, 32 pairs a round: lanes with the same expert find
// each other by a ballot for each bit of its number (match.any is slower: 9.7
// against 7.9 us for 4096 pairs over 256 experts), their rank is the warp's running
// count plus the lanes before them, so order is kept without an atomic.  A column
// scan over the warps then turns counts into rows.  With one block (hist NULL) the
// counts of the first and only chunk are the histogram.  Bound by latency: 3.1 us
// for one token's pairs, 9.5 us for 524288 over 64 experts in two launches.
template <typename I>
__global__ void __launch_bounds__(1024) sort_place_kernel(const I* __restrict__ ids, int64_t pairs, int64_t share, int E,
                                                          const int* __restrict__ hist, int* __restrict__ row_of,
                                                          int* __restrict__ src, int* __restrict__ offsets) {
  extern __shared__ int sort_smem[];
  __shared__ int part[33];
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* base = sort_smem;                                             // [E + 1] next row of each expert
  uint16_t* cnt = reinterpret_cast<uint16_t*>(sort_smem + E + 1);    // [warps][E + 1]
  uint16_t* mine = cnt + warp * (E + 1);
  const int64_t begin = blockIdx.x * share;
  const int64_t end = begin + share < pairs ? begin + share : pairs;
  const int e0 = threadIdx.x;                                        // blockDim >= E
  const int bits = 32 - __clz(E);                                    // of an expert's number, E itself included

  int routed = 0;
  if (hist != nullptr) {
    // all blocks' counts, and those of the blocks before this one: the threads
    // share out the blocks, blockDim / E of them at a time
    int* all = reinterpret_cast<int*>(sort_smem + E + 1);              // [2][E] in the place of cnt
    for (int i = threadIdx.x; i < 2 * E; i += blockDim.x) all[i] = 0;
    __syncthreads();
    const int at_once = blockDim.x / E, mine_e = threadIdx.x % E;
    if (static_cast<int>(threadIdx.x) < at_once * E) {
      int before = 0, total = 0;
#pragma unroll 8
      for (int b = threadIdx.x / E; b < static_cast<int>(gridDim.x); b += at_once) {
        const int c = hist[static_cast<int64_t>(b) * E + mine_e];
        before += b < static_cast<int>(blockIdx.x) ? c : 0;
        total += c;
      }
      atomicAdd(&all[mine_e], total);
      atomicAdd(&all[E + mine_e], before);
    }
    __syncthreads();
    const int first = block_scan(e0 < E ? all[e0] : 0, part, &routed);
    if (e0 < E) {
      base[e0] = first + all[E + e0];
      if (blockIdx.x == 0) offsets[e0] = first;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) offsets[E] = routed;
  }

  const int chunk = blockDim.x * kSortRounds;
  for (int64_t c0 = begin; c0 < end; c0 += chunk) {
    __syncthreads();                                                 // base is whole; cnt of the last chunk is read
    for (int i = threadIdx.x; i < warps * (E + 1); i += blockDim.x) cnt[i] = 0;
    __syncthreads();
    int expert[kSortRounds], rank[kSortRounds];
    const int64_t w0 = c0 + static_cast<int64_t>(warp) * (32 * kSortRounds) + lane;
#pragma unroll
    for (int i = 0; i < kSortRounds; ++i) expert[i] = expert_of(ids, w0 + 32 * i, end, E);
#pragma unroll
    for (int i = 0; i < kSortRounds; ++i) {
      unsigned same = 0xffffffffu;                                   // lanes with this lane's expert
      for (int bit = 0; bit < bits; ++bit) {
        const bool set = expert[i] >> bit & 1;
        const unsigned those = __ballot_sync(0xffffffffu, set);
        same &= set ? those : ~those;
      }
      const int ahead = __popc(same & ((1u << lane) - 1u));
      rank[i] = mine[expert[i]] + ahead;
      __syncwarp();
      if (ahead == 0) mine[expert[i]] = static_cast<uint16_t>(rank[i] + __popc(same));
      __syncwarp();
    }
    __syncthreads();
    int total = 0;
    if (e0 < E) {
#pragma unroll 8
      for (int w = 0; w < warps; ++w) {
        const int c = cnt[w * (E + 1) + e0];
        cnt[w * (E + 1) + e0] = static_cast<uint16_t>(total);        // this warp's first rank in the chunk
        total += c;
      }
    }
    if (hist == nullptr) {
      const int first = block_scan(total, part, &routed);
      if (e0 < E) {
        base[e0] = first;
        offsets[e0] = first;
      }
      if (threadIdx.x == 0) offsets[E] = routed;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSortRounds; ++i) {
      const int64_t p = w0 + 32 * i;
      if (p >= end) continue;
      int row = -1;
      if (expert[i] < E) {
        row = base[expert[i]] + mine[expert[i]] + rank[i];
        if (row < pairs) src[row] = static_cast<int>(p);             // always, unless the ids changed between the passes
      }
      row_of[p] = row;
    }
    __syncthreads();
    if (e0 < E) base[e0] += total;
  }
  // rows without a pair
  for (int64_t r = routed + blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; r < pairs;
       r += static_cast<int64_t>(gridDim.x) * blockDim.x)
    src[r] = -1;
}

// -------------------------------------------------------------- row kernels --

template <int B> struct Bytes;
template <> struct Bytes<16> { using type = uint4; };
template <> struct Bytes<8> { using type = uint2; };
template <> struct Bytes<4> { using type = uint32_t; };
template <> struct Bytes<2> { using type = uint16_t; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// V elements of T moved as one access of 16, 8 or 4 bytes, or one element.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  uint32_t w[V * sizeof(T) / 4];
};
template <typename T>
struct Pack<T, 1> {
  T v;
};
__device__ __forceinline__ void unpack_word(uint32_t w, float* f, __nv_bfloat16*) {
  f[0] = __uint_as_float(w << 16);
  f[1] = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void unpack_word(uint32_t w, float* f, __half*) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
  f[0] = v.x;
  f[1] = v.y;
}
__device__ __forceinline__ void unpack_word(uint32_t w, float* f, float*) { f[0] = __uint_as_float(w); }
__device__ __forceinline__ uint32_t pack_word(const float* f, __nv_bfloat16*) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(f[0], f[1]);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_word(const float* f, __half*) {
  const __half2 v = __floats2half2_rn(f[0], f[1]);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_word(const float* f, float*) { return __float_as_uint(f[0]); }
template <typename T, int V>
__device__ __forceinline__ void unpack(const Pack<T, V>& p, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = to_f32(p.v);
  } else {
#pragma unroll
    for (int i = 0; i < static_cast<int>(V * sizeof(T) / 4); ++i)
      unpack_word(p.w[i], f + i * (4 / sizeof(T)), static_cast<T*>(nullptr));
  }
}
template <typename T, int V>
__device__ __forceinline__ void pack(Pack<T, V>& p, const float (&f)[V]) {
  if constexpr (V == 1) {
    p.v = from_f32<T>(f[0]);
  } else {
#pragma unroll
    for (int i = 0; i < static_cast<int>(V * sizeof(T) / 4); ++i)
      p.w[i] = pack_word(f + i * (4 / sizeof(T)), static_cast<T*>(nullptr));
  }
}

// Zeros in the rows behind the last routed one, shared out over the grid's x;
// y covers the row in units of U.
template <typename U>
__device__ __forceinline__ void zero_tail(U* y, int64_t ldy, int nvec, int64_t rows, int routed, U zero) {
  const int64_t first = routed < 0 ? 0 : routed;
  for (int64_t r = first + blockIdx.x; r < rows; r += gridDim.x)
    for (int v = blockIdx.y * blockDim.x + threadIdx.x; v < nvec; v += gridDim.y * blockDim.x) y[r * ldy + v] = zero;
}

// y[row_of[t, j]] = x[t], as bytes.  One block (or gridDim.y blocks) a token; the
// next bytes of x are on their way while the last are written.
template <int B>
__global__ void __launch_bounds__(256) gather_kernel(const void* __restrict__ xp, int64_t ldx, int nvec, int topk,
                                                     int64_t rows, const int* __restrict__ row_of,
                                                     const int* __restrict__ routed, void* __restrict__ yp,
                                                     int64_t ldy) {
  using U = typename Bytes<B>::type;
  __shared__ int at[kMaxTopk];
  const U* x = static_cast<const U*>(xp);
  U* y = static_cast<U*>(yp);
  const int64_t t = blockIdx.x;
  const int step = gridDim.y * blockDim.x;
  int v = blockIdx.y * blockDim.x + threadIdx.x;
  U next = v < nvec ? x[t * ldx + v] : U{};       // on its way while the rows are looked up
  for (int j = threadIdx.x; j < topk; j += blockDim.x) {
    const int r = row_of[t * topk + j];
    at[j] = r >= 0 && r < rows ? r : -1;
  }
  __syncthreads();
  for (; v < nvec; v += step) {
    const U val = next;
    if (v + step < nvec) next = x[t * ldx + v + step];
#pragma unroll 4
    for (int j = 0; j < topk; ++j) {
      const int r = at[j];
      if (r >= 0) y[r * ldy + v] = val;
    }
  }
  zero_tail<U>(y, ldy, nvec, rows, *routed, U{});
}

// out[t] = sum_j w[t, j] * y[row_of[t, j]] (w NULL: 1), fp32, slots in order.  A
// thread has SL slots of U places of the row in flight: two of two, four of two or eight
// of one, four to eight 16-byte loads.  With one place the rows of 16384 x 2 experts,
// 1024 wide bf16, came at 0.60 of the copy rate (two loads); with two it is 0.89, 17.5 us.
template <typename T, int V, int SL, int U>
__global__ void __launch_bounds__(256) combine_kernel(const T* __restrict__ y, int64_t ldy, const float* __restrict__ w,
                                                      int nvec, int topk, int64_t rows, const int* __restrict__ row_of,
                                                      T* __restrict__ out, int64_t ldo) {
  using P = Pack<T, V>;
  __shared__ int at[kMaxTopk];
  __shared__ float gate[kMaxTopk];
  const int64_t t = blockIdx.x;
  for (int j = threadIdx.x; j < topk; j += blockDim.x) {
    const int r = row_of[t * topk + j];
    at[j] = r >= 0 && r < rows ? r : -1;
    gate[j] = w ? w[t * topk + j] : 1.0f;
  }
  __syncthreads();
  const int step = gridDim.y * blockDim.x;
  for (int v0 = blockIdx.y * blockDim.x + threadIdx.x; v0 < nvec; v0 += U * step) {
    float acc[U][V];
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[k][i] = 0.0f;
    for (int j0 = 0; j0 < topk; j0 += SL) {
      P p[SL][U];
#pragma unroll
      for (int u = 0; u < SL; ++u)
        if (j0 + u < topk && at[j0 + u] >= 0) {
          const T* row = y + at[j0 + u] * ldy;
#pragma unroll
          for (int k = 0; k < U; ++k)
            if (v0 + k * step < nvec) p[u][k] = *reinterpret_cast<const P*>(row + static_cast<int64_t>(v0 + k * step) * V);
        }
#pragma unroll
      for (int u = 0; u < SL; ++u)
        if (j0 + u < topk && at[j0 + u] >= 0) {
          const float g = gate[j0 + u];
#pragma unroll
          for (int k = 0; k < U; ++k)
            if (v0 + k * step < nvec) {
              float f[V];
              unpack(p[u][k], f);
#pragma unroll
              for (int i = 0; i < V; ++i) acc[k][i] = fmaf(g, f[i], acc[k][i]);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (v0 + k * step < nvec) {
        P o;
        pack(o, acc[k]);
        *reinterpret_cast<P*>(out + t * ldo + static_cast<int64_t>(v0 + k * step) * V) = o;
      }
  }
}

// dy[row_of[t, j]] = w[t, j] * dout[t] and dw[t, j] = <dout[t], y[row_of[t, j]]>
// (either may be NULL), one block a token.  The dot products are fp32: each
// thread's own columns in order, then the lanes, then the warps.  Four slots at a
// time (two places of the row when a token has two): with eight the registers leave
// two blocks an SM and 4096 x 6 x 4096 fp16 takes 85 instead of 74 us.
// dout's load waits for no index.
template <typename T, int V, int SL, int U>
__global__ void __launch_bounds__(256, 3) combine_bwd_kernel(const T* __restrict__ dout, int64_t ldd,
                                                          const T* __restrict__ y, int64_t ldy,
                                                          const float* __restrict__ w, int nvec, int topk, int64_t rows,
                                                          const int* __restrict__ row_of,
                                                          const int* __restrict__ routed, T* __restrict__ dy,
                                                          int64_t lddy, float* __restrict__ dw) {
  using P = Pack<T, V>;
  __shared__ int at[kMaxTopk];
  __shared__ float gate[kMaxTopk];
  __shared__ float sums[8][SL];
  const int64_t t = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  for (int j = threadIdx.x; j < topk; j += blockDim.x) {
    const int r = row_of[t * topk + j];
    at[j] = r >= 0 && r < rows ? r : -1;
    gate[j] = w[t * topk + j];
  }
  __syncthreads();
  const int step = blockDim.x;
  for (int j0 = 0; j0 < topk; j0 += SL) {
    float dot[SL];
#pragma unroll
    for (int u = 0; u < SL; ++u) dot[u] = 0.0f;
    for (int v0 = threadIdx.x; v0 < nvec; v0 += U * step) {
      P dp[U], p[SL][U];
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (v0 + k * step < nvec) dp[k] = *reinterpret_cast<const P*>(dout + t * ldd + static_cast<int64_t>(v0 + k * step) * V);
      if (dw) {
#pragma unroll
        for (int u = 0; u < SL; ++u)
          if (j0 + u < topk && at[j0 + u] >= 0) {
            const T* row = y + at[j0 + u] * ldy;
#pragma unroll
            for (int k = 0; k < U; ++k)
              if (v0 + k * step < nvec) p[u][k] = *reinterpret_cast<const P*>(row + static_cast<int64_t>(v0 + k * step) * V);
          }
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (v0 + k * step >= nvec) break;
        float d[V];
        unpack(dp[k], d);
#pragma unroll
        for (int u = 0; u < SL; ++u) {
          if (j0 + u >= topk || at[j0 + u] < 0) continue;
          if (dw) {
            float f[V];
            unpack(p[u][k], f);
#pragma unroll
            for (int i = 0; i < V; ++i) dot[u] = fmaf(d[i], f[i], dot[u]);
          }
          if (dy) {
            P o;
            float f[V];
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = gate[j0 + u] * d[i];
            pack(o, f);
            *reinterpret_cast<P*>(dy + at[j0 + u] * lddy + static_cast<int64_t>(v0 + k * step) * V) = o;
          }
        }
      }
    }
    if (dw) {
#pragma unroll
      for (int u = 0; u < SL; ++u) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], d);
      }
      if (lane == 0) {
#pragma unroll
        for (int u = 0; u < SL; ++u) sums[warp][u] = dot[u];
      }
      __syncthreads();
      if (threadIdx.x < SL && j0 + threadIdx.x < topk) {
        float s = 0.0f;
        for (int i = 0; i < warps; ++i) s += sums[i][threadIdx.x];
        dw[t * topk + j0 + threadIdx.x] = at[j0 + threadIdx.x] >= 0 ? s : 0.0f;
      }
      __syncthreads();
    }
  }
  if (dy) {
    P zero;
    const float none[V] = {};
    pack(zero, none);
    zero_tail<P>(reinterpret_cast<P*>(dy), lddy / V, nvec, rows, *routed, zero);
  }
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t quant2(float a, float b, float scale) {
  const float qa = max_nan(min_nan(a / scale, kQmax), -kQmax), qb = max_nan(min_nan(b / scale, kQmax), -kQmax);
  return __nv_cvt_float2_to_fp8x2(make_float2(qa, qb), __NV_SATFINITE, __NV_E4M3);
}

// 16 consecutive elements in fp32
__device__ __forceinline__ void load16(const float* p, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 f = reinterpret_cast<const float4*>(p)[i];
    v[4 * i] = f.x;
    v[4 * i + 1] = f.y;
    v[4 * i + 2] = f.z;
    v[4 * i + 3] = f.w;
  }
}
__device__ __forceinline__ void load16(const __nv_bfloat16* p, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float f[8];
    unpack(reinterpret_cast<const Pack<__nv_bfloat16, 8>*>(p)[i], f);
#pragma unroll
    for (int u = 0; u < 8; ++u) v[8 * i + u] = f[u];
  }
}

// The codes and scales of fack_quant_act, computed once a token and written to
// its topk rows.  Eight lanes take a group of 128, 16 elements each, so a lane's
// codes are one 16-byte store.  The magnitudes' bit patterns order as integers
// with NaN on top, so a group that holds one gets scale NaN and NaN codes; a
// group whose scale would round to 0 gets scale 1 and zero codes.  Six blocks an SM
// (40 registers): 8192 x 2 rows of 7168 bf16 61 -> 57 us; loading a group ahead takes
// 60 registers and 71 us.
template <typename T>
__global__ void __launch_bounds__(256, 6) gather_quant_kernel(const T* __restrict__ x, int64_t ldx, int KB, int topk,
                                                           int64_t rows, const int* __restrict__ row_of,
                                                           const int* __restrict__ routed, uint8_t* __restrict__ xq,
                                                           int64_t ldq, float* __restrict__ xs, int64_t lds) {
  __shared__ int at[kMaxTopk];
  const int64_t t = blockIdx.x;
  const int lane8 = threadIdx.x & 7, per_block = blockDim.x >> 3;
  for (int j = threadIdx.x; j < topk; j += blockDim.x) {
    const int r = row_of[t * topk + j];
    at[j] = r >= 0 && r < rows ? r : -1;
  }
  __syncthreads();
  // a whole warp enters or leaves the loop: the shuffles below name all its lanes
  for (int g0 = blockIdx.y * per_block + (threadIdx.x >> 5) * 4; g0 < KB; g0 += gridDim.y * per_block) {
    const int g = g0 + ((threadIdx.x & 31) >> 3);
    const bool live = g < KB;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.0f;
    if (live) load16(x + t * ldx + static_cast<int64_t>(g) * kBlk + lane8 * 16, v);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    float scale = __uint_as_float(top) / kQmax;
    if (scale == 0.0f) scale = 1.0f;
    uint4 q;
    q.x = quant2(v[0], v[1], scale) | quant2(v[2], v[3], scale) << 16;
    q.y = quant2(v[4], v[5], scale) | quant2(v[6], v[7], scale) << 16;
    q.z = quant2(v[8], v[9], scale) | quant2(v[10], v[11], scale) << 16;
    q.w = quant2(v[12], v[13], scale) | quant2(v[14], v[15], scale) << 16;
    if (!live) continue;
#pragma unroll 4
    for (int j = 0; j < topk; ++j)
      if (at[j] >= 0) *reinterpret_cast<uint4*>(xq + at[j] * ldq + static_cast<int64_t>(g) * kBlk + lane8 * 16) = q;
    for (int j = lane8; j < topk; j += 8)
      if (at[j] >= 0) xs[at[j] * lds + g] = scale;
  }
  zero_tail<uint4>(reinterpret_cast<uint4*>(xq), ldq / 16, KB * (kBlk / 16), rows, *routed, uint4{0, 0, 0, 0});
  zero_tail<float>(xs, lds, KB, rows, *routed, 1.0f);
}

// ------------------------------------------------------------------- host --

static bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
static int elem_size(int dtype) {
  return dtype == FACK_DTYPE_F32 ? 4 : dtype == FACK_DTYPE_BF16 || dtype == FACK_DTYPE_F16 ? 2 : 0;
}

static int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? FACK_OK : fack::record_error(FACK_ERR_LAUNCH, cudaGetErrorString(e));
}

// Threads and blocks for rows of `units`: as few passes over the row as 256
// threads allow, evenly filled, and for few tokens the row split over blocks
// until two blocks an SM are busy.
struct RowGrid {
  dim3 grid;
  int threads;
};
static RowGrid row_grid(int64_t tokens, int units, int sms) {
  const int passes = (units + 255) / 256;
  int threads = ((units + passes - 1) / passes + 31) / 32 * 32;
  int split = tokens < 2 * sms ? static_cast<int>((2 * sms + tokens - 1) / tokens) : 1;
  if (split > passes) {            // more blocks than passes: narrower blocks
    const int warps = (units + 31) / 32;
    if (split > warps) split = warps;
    threads = ((units + split - 1) / split + 31) / 32 * 32;
    if (threads > 256) threads = 256;
    split = (units + threads - 1) / threads;
  }
  return {dim3(static_cast<unsigned>(tokens), static_cast<unsigned>(split)), threads};
}

static int check_plan(int T, int topk, const void* row_of, const void* offsets, int E) {
  if (T < 1 || topk < 1 || topk > kMaxTopk || E < 1 || E > kMaxExperts ||
      static_cast<int64_t>(T) * topk > INT32_MAX)
    return FACK_ERR_BAD_SHAPE;
  if (!row_of || !offsets || !aligned(row_of, 4) || !aligned(offsets, 4)) return FACK_ERR_BAD_ALIGN;
  return FACK_OK;
}

static int64_t sort_blocks(int64_t pairs, int* threads, int E) {
  int th = E < 128 ? 128 : (E + 31) / 32 * 32;             // one thread an expert in the scans
  while (th < 1024 && pairs > static_cast<int64_t>(th) * kSortRounds) th = th * 2 < 1024 ? th * 2 : 1024;
  *threads = th;
  const int64_t chunk = static_cast<int64_t>(th) * kSortRounds;
  const int64_t blocks = (pairs + chunk - 1) / chunk;
  return blocks < kSortMaxBlocks ? blocks : kSortMaxBlocks;
}

template <typename I>
static int sort_launch(const void* ids, int64_t pairs, int E, int* row_of, int* src, int* offsets, int* hist,
                       cudaStream_t s) {
  int threads;
  const int64_t blocks = sort_blocks(pairs, &threads, E);
  const int64_t chunk = static_cast<int64_t>(threads) * kSortRounds;
  const int64_t share = ((pairs + blocks - 1) / blocks + chunk - 1) / chunk * chunk;
  const int64_t grid = (pairs + share - 1) / share;
  const size_t smem = sort_smem_bytes(threads, E);
  // Set on every call that needs it, so that each device has it (a host-side attribute, no device
  // work), and always to the same value: it belongs to the function, whichever thread sorts what.
  const cudaError_t e = smem > kSortSmemPlain ? cudaFuncSetAttribute(sort_place_kernel<I>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                                     kSortSmemMost)
                                              : cudaSuccess;
  if (e != cudaSuccess) return fack::record_error(FACK_ERR_LAUNCH, cudaGetErrorString(e));
  if (grid > 1)
    sort_count_kernel<I><<<static_cast<unsigned>(grid), 1024, 0, s>>>(static_cast<const I*>(ids), pairs, share, E, hist);
  sort_place_kernel<I><<<static_cast<unsigned>(grid), threads, smem, s>>>(static_cast<const I*>(ids), pairs, share, E,
                                                                          grid > 1 ? hist : nullptr, row_of, src, offsets);
  return launched();
}

// Widest access that every row of both tensors allows.
static int row_vector(int es, const void* a, int64_t lda, const void* b, int64_t ldb, int D) {
  for (int v = 16; v > es; v /= 2)
    if (aligned(a, v) && aligned(b, v) && lda * es % v == 0 && ldb * es % v == 0 && static_cast<int64_t>(D) * es % v == 0)
      return v;
  return es;
}

template <typename T, int V, int SL, int U>
static void combine_launch(const void* y, int64_t ldy, const float* w, int T_, int topk, int D, const int* row_of,
                           void* out, int64_t ldo, int sms, cudaStream_t s) {
  const RowGrid g = row_grid(T_, (D / V + U - 1) / U, sms);
  combine_kernel<T, V, SL, U><<<g.grid, g.threads, 0, s>>>(static_cast<const T*>(y), ldy, w, D / V, topk,
                                                           static_cast<int64_t>(T_) * topk, row_of, static_cast<T*>(out), ldo);
}

// Places of the row in flight beside the slots: as many as keep two warps a token
// busy, and one when few tokens need every thread.
template <typename T, int V>
static void combine_wide(const void* y, int64_t ldy, const float* w, int T_, int topk, int D, const int* row_of, void* out,
                         int64_t ldo, int sms, cudaStream_t s) {
  const int units = T_ < 2 * sms ? 0 : D / V;
  if (topk <= 2 && units >= 128)
    combine_launch<T, V, 2, 2>(y, ldy, w, T_, topk, D, row_of, out, ldo, sms, s);
  else if (topk <= 4 && units >= 128)
    combine_launch<T, V, 4, 2>(y, ldy, w, T_, topk, D, row_of, out, ldo, sms, s);
  else
    combine_launch<T, V, 8, 1>(y, ldy, w, T_, topk, D, row_of, out, ldo, sms, s);
}

template <typename T>
static void combine_rows(int bytes, const void* y, int64_t ldy, const float* w, int T_, int topk, int D, const int* row_of,
                         void* out, int64_t ldo, int sms, cudaStream_t s) {
  constexpr int es = sizeof(T);
  if (bytes == 16)
    combine_wide<T, 16 / es>(y, ldy, w, T_, topk, D, row_of, out, ldo, sms, s);
  else if (bytes == 8)
    combine_launch<T, 8 / es, 8, 1>(y, ldy, w, T_, topk, D, row_of, out, ldo, sms, s);
  else if (bytes == 4)
    combine_launch<T, 4 / es, 8, 1>(y, ldy, w, T_, topk, D, row_of, out, ldo, sms, s);
  else
    combine_launch<T, 1, 8, 1>(y, ldy, w, T_, topk, D, row_of, out, ldo, sms, s);
}

template <typename T, int V, int SL, int U>
static void combine_bwd_launch(const void* dout, int64_t ldd, const void* y, int64_t ldy, const float* w, int T_,
                               int topk, int D, const int* row_of, const int* routed, void* dy, int64_t lddy, float* dw,
                               cudaStream_t s) {
  const int units = (D / V + U - 1) / U, passes = (units + 255) / 256;
  const int threads = ((units + passes - 1) / passes + 31) / 32 * 32;
  combine_bwd_kernel<T, V, SL, U><<<static_cast<unsigned>(T_), threads, 0, s>>>(
      static_cast<const T*>(dout), ldd, static_cast<const T*>(y), ldy, w, D / V, topk,
      static_cast<int64_t>(T_) * topk, row_of, routed, static_cast<T*>(dy), lddy, dw);
}

template <typename T>
static void combine_bwd_rows(int bytes, const void* dout, int64_t ldd, const void* y, int64_t ldy, const float* w, int T_,
                             int topk, int D, const int* row_of, const int* routed, void* dy, int64_t lddy, float* dw,
                             cudaStream_t s) {
  constexpr int es = sizeof(T), V = 16 / es;
  if (bytes == 16 && topk <= 2 && D / V >= 128)
    combine_bwd_launch<T, V, 2, 2>(dout, ldd, y, ldy, w, T_, topk, D, row_of, routed, dy, lddy, dw, s);
  else if (bytes == 16)
    combine_bwd_launch<T, V, 4, 1>(dout, ldd, y, ldy, w, T_, topk, D, row_of, routed, dy, lddy, dw, s);
  else if (bytes == 8)
    combine_bwd_launch<T, 8 / es, 4, 1>(dout, ldd, y, ldy, w, T_, topk, D, row_of, routed, dy, lddy, dw, s);
  else if (bytes == 4)
    combine_bwd_launch<T, 4 / es, 4, 1>(dout, ldd, y, ldy, w, T_, topk, D, row_of, routed, dy, lddy, dw, s);
  else
    combine_bwd_launch<T, 1, 4, 1>(dout, ldd, y, ldy, w, T_, topk, D, row_of, routed, dy, lddy, dw, s);
}

}  // namespace fack_moe

extern "C" {

int fack_moe_sort_workspace_size(int T, int topk, int num_experts, size_t* bytes) {
  using namespace fack_moe;
  if (!bytes) return FACK_ERR_BAD_ARG;
  if (T < 1 || topk < 1 || topk > kMaxTopk || num_experts < 1 || num_experts > kMaxExperts ||
      static_cast<int64_t>(T) * topk > INT32_MAX)
    return FACK_ERR_BAD_SHAPE;
  int threads;
  const int64_t blocks = sort_blocks(static_cast<int64_t>(T) * topk, &threads, num_experts);
  *bytes = blocks > 1 ? static_cast<size_t>(blocks) * num_experts * sizeof(int) : 0;
  return FACK_OK;
}

int fack_moe_sort(const void* ids, int ids_bytes, int T, int topk, int num_experts, int32_t* row_of, int32_t* src,
                  int32_t* offsets, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace fack_moe;
  size_t need = 0;
  int st = fack_moe_sort_workspace_size(T, topk, num_experts, &need);
  if (st != FACK_OK) return st;
  if (ids_bytes != 4 && ids_bytes != 8) return FACK_ERR_BAD_ARG;
  if (!ids || !row_of || !src || !offsets || !aligned(ids, ids_bytes) || !aligned(row_of, 4) || !aligned(src, 4) ||
      !aligned(offsets, 4))
    return FACK_ERR_BAD_ALIGN;
  if (need && (!workspace || workspace_bytes < need)) return FACK_ERR_WS_TOO_SMALL;
  if (need && !aligned(workspace, 4)) return FACK_ERR_BAD_ALIGN;
  int sms = 0;
  st = fack::sm100_device(&sms);
  if (st != FACK_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t pairs = static_cast<int64_t>(T) * topk;
  return ids_bytes == 4 ? sort_launch<int32_t>(ids, pairs, num_experts, row_of, src, offsets, static_cast<int*>(workspace), s)
                        : sort_launch<int64_t>(ids, pairs, num_experts, row_of, src, offsets, static_cast<int*>(workspace), s);
}

int fack_moe_gather(const void* x, int dtype, int64_t ldx, int T, int topk, int D, const int32_t* row_of,
                    const int32_t* offsets, int num_experts, void* y, int64_t ldy, void* stream) {
  using namespace fack_moe;
  int st = check_plan(T, topk, row_of, offsets, num_experts);
  if (st != FACK_OK) return st;
  if (D < 1 || D > kMaxDim) return FACK_ERR_BAD_SHAPE;
  const int es = elem_size(dtype);
  if (!es) return FACK_ERR_BAD_ARG;
  if (!x || !y || !aligned(x, es) || !aligned(y, es)) return FACK_ERR_BAD_ALIGN;
  if (ldx < 0 || ldy < D) return FACK_ERR_BAD_STRIDE;
  int sms = 0;
  st = fack::sm100_device(&sms);
  if (st != FACK_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int b = row_vector(es, x, ldx, y, ldy, D);
  const int units = static_cast<int>(static_cast<int64_t>(D) * es / b);
  const RowGrid g = row_grid(T, units, sms);
  const int64_t rows = static_cast<int64_t>(T) * topk;
  const int* routed = offsets + num_experts;
  if (b == 16)
    gather_kernel<16><<<g.grid, g.threads, 0, s>>>(x, ldx * es / 16, units, topk, rows, row_of, routed, y, ldy * es / 16);
  else if (b == 8)
    gather_kernel<8><<<g.grid, g.threads, 0, s>>>(x, ldx * es / 8, units, topk, rows, row_of, routed, y, ldy * es / 8);
  else if (b == 4)
    gather_kernel<4><<<g.grid, g.threads, 0, s>>>(x, ldx * es / 4, units, topk, rows, row_of, routed, y, ldy * es / 4);
  else
    gather_kernel<2><<<g.grid, g.threads, 0, s>>>(x, ldx, units, topk, rows, row_of, routed, y, ldy);
  return launched();
}

int fack_moe_gather_quant(const void* x, int dtype, int64_t ldx, int T, int topk, int K, const int32_t* row_of,
                          const int32_t* offsets, int num_experts, void* xq, int64_t ldq, float* x_scale, int64_t lds,
                          void* stream) {
  using namespace fack_moe;
  int st = check_plan(T, topk, row_of, offsets, num_experts);
  if (st != FACK_OK) return st;
  if (K < kBlk || K % kBlk || K > kMaxDim) return FACK_ERR_BAD_SHAPE;
  if (dtype != FACK_DTYPE_F32 && dtype != FACK_DTYPE_BF16) return FACK_ERR_BAD_ARG;
  if (!x || !xq || !x_scale || !aligned(x, 16) || !aligned(xq, 16) || !aligned(x_scale, 4)) return FACK_ERR_BAD_ALIGN;
  if (ldx < 0 || ldx * elem_size(dtype) % 16 || ldq < K || ldq % 16 || lds < K / kBlk) return FACK_ERR_BAD_STRIDE;
  int sms = 0;
  st = fack::sm100_device(&sms);
  if (st != FACK_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const RowGrid g = row_grid(T, K / 16, sms);
  const int64_t rows = static_cast<int64_t>(T) * topk;
  const int* routed = offsets + num_experts;
  if (dtype == FACK_DTYPE_F32)
    gather_quant_kernel<float><<<g.grid, g.threads, 0, s>>>(static_cast<const float*>(x), ldx, K / kBlk, topk, rows, row_of,
                                                           routed, static_cast<uint8_t*>(xq), ldq, x_scale, lds);
  else
    gather_quant_kernel<__nv_bfloat16><<<g.grid, g.threads, 0, s>>>(static_cast<const __nv_bfloat16*>(x), ldx, K / kBlk, topk,
                                                                   rows, row_of, routed, static_cast<uint8_t*>(xq), ldq,
                                                                   x_scale, lds);
  return launched();
}

int fack_moe_combine(const void* y, int dtype, int64_t ldy, const float* weights, int T, int topk, int D,
                     const int32_t* row_of, void* out, int64_t ldo, void* stream) {
  using namespace fack_moe;
  int st = check_plan(T, topk, row_of, row_of, 1);
  if (st != FACK_OK) return st;
  if (D < 1 || D > kMaxDim) return FACK_ERR_BAD_SHAPE;
  const int es = elem_size(dtype);
  if (!es) return FACK_ERR_BAD_ARG;
  if (!y || !out || !aligned(y, es) || !aligned(out, es) || !aligned(weights, 4)) return FACK_ERR_BAD_ALIGN;
  if (ldy < 0 || ldo < D) return FACK_ERR_BAD_STRIDE;
  int sms = 0;
  st = fack::sm100_device(&sms);
  if (st != FACK_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int bytes = row_vector(es, y, ldy, out, ldo, D);
  if (dtype == FACK_DTYPE_F32)
    combine_rows<float>(bytes, y, ldy, weights, T, topk, D, row_of, out, ldo, sms, s);
  else if (dtype == FACK_DTYPE_BF16)
    combine_rows<__nv_bfloat16>(bytes, y, ldy, weights, T, topk, D, row_of, out, ldo, sms, s);
  else
    combine_rows<__half>(bytes, y, ldy, weights, T, topk, D, row_of, out, ldo, sms, s);
  return launched();
}

int fack_moe_combine_bwd(const void* dout, int dtype, int64_t ldd, const void* y, int64_t ldy, const float* weights, int T,
                         int topk, int D, const int32_t* row_of, const int32_t* offsets, int num_experts, void* dy,
                         int64_t lddy, float* dweights, void* stream) {
  using namespace fack_moe;
  int st = check_plan(T, topk, row_of, offsets, num_experts);
  if (st != FACK_OK) return st;
  if (D < 1 || D > kMaxDim) return FACK_ERR_BAD_SHAPE;
  const int es = elem_size(dtype);
  if (!es || (!dy && !dweights)) return FACK_ERR_BAD_ARG;
  if (!dout || !weights || !aligned(dout, es) || !aligned(weights, 4)) return FACK_ERR_BAD_ALIGN;
  if (ldd < 0) return FACK_ERR_BAD_STRIDE;
  if (dweights && (!y || !aligned(y, es) || !aligned(dweights, 4))) return FACK_ERR_BAD_ALIGN;
  if (dweights && ldy < 0) return FACK_ERR_BAD_STRIDE;
  if (dy && !aligned(dy, es)) return FACK_ERR_BAD_ALIGN;
  if (dy && lddy < D) return FACK_ERR_BAD_STRIDE;
  int sms = 0;
  st = fack::sm100_device(&sms);
  if (st != FACK_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int bytes = row_vector(es, dout, ldd, dout, ldd, D);
  if (dweights) {
    const int b = row_vector(es, y, ldy, y, ldy, D);
    bytes = b < bytes ? b : bytes;
  }
  if (dy) {
    const int b = row_vector(es, dy, lddy, dy, lddy, D);
    bytes = b < bytes ? b : bytes;
  }
  const int* routed = offsets + num_experts;
  if (dtype == FACK_DTYPE_F32)
    combine_bwd_rows<float>(bytes, dout, ldd, y, ldy, weights, T, topk, D, row_of, routed, dy, lddy, dweights, s);
  else if (dtype == FACK_DTYPE_BF16)
    combine_bwd_rows<__nv_bfloat16>(bytes, dout, ldd, y, ldy, weights, T, topk, D, row_of, routed, dy, lddy, dweights, s);
  else
    combine_bwd_rows<__half>(bytes, dout, ldd, y, ldy, weights, T, topk, D, row_of, routed, dy, lddy, dweights, s);
  return launched();
}

}  // extern "C"
