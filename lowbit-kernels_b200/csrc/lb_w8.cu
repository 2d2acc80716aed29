// W8A8 linear layer: y[M, N] = (sum_k q[m, k] w[n, k]) s[m] t[n] (+ bias[n]), q and w in [-127, 127] as 8-bit
// integers, s one fp32 scale per token, t one per output channel.
//
// The activations are quantized per token on the way in: with a = max_k |x[m, k]|, q = rint(x (127 / a)) and
// s = a / 127 in fp32 (a row of zeros has q = 0 and s = 0; a row that holds an infinity or a NaN has s = that, and
// its outputs are not finite). The products are summed in int32, so the sum is exact and no order of the additions,
// tile or split changes a bit of it (K <= 131072 keeps it below 2^31); then float(sum) * s * t + bias in fp32 and one
// rounding to the output's type.
#include <atomic>

#include "lb_launch.h"
#include "lb_tc.cuh"
#include "lb_types.cuh"

namespace lb {

// status word of this file's kernels (a bounded wait that gave up); read by w8_device_error()
__device__ int g_w8_status;

namespace {

// ------------------------------------------------------------------------------------------- quantize rows
// 127 / amax of a row of subnormals would overflow: such rows are scaled by `up`, a power of two, first
struct RowScale {
  float up, r, s;
};
__device__ __forceinline__ RowScale row_scale(float amax) {
  RowScale v;
  v.up = amax < 0x1p-100f ? 0x1p100f : 1.f;
  v.r = amax > 0.f ? 127.f / (amax * v.up) : 0.f;
  v.s = amax / 127.f;
  return v;
}

// rint(x r) in the low byte: adding 1.5 * 2^23 rounds to an integer, half to even (|x r| <= 127 but for rows that are
// not finite, whose scale makes the outputs so)
__device__ __forceinline__ uint32_t quant_bits(float x, float r) {
  return __float_as_uint(__fadd_rn(__fmul_rn(x, r), 12582912.f));   // two roundings: not to be fused
}

__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

__device__ __forceinline__ uint2 quant8(const float (&f)[8], const RowScale& v) {
  uint32_t q[8];
  if (v.up == 1.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = quant_bits(f[i], v.r);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = quant_bits(f[i] * v.up, v.r);
  }
  return make_uint2(low_bytes(q[0], q[1], q[2], q[3]), low_bytes(q[4], q[5], q[6], q[7]));
}

// Eight values of a row. Maxima of |x| are taken on the bits without the sign, which order like the magnitudes with NaN
// above all: `amax` keeps them packed, `amax_float` gives the fp32 value.
template <typename T>
struct Vec8 {
  uint32_t v[4];
  // n: values left in the row, zeros behind them; through L2 only (the row may have been written while this kernel was
  // already resident)
  __device__ __forceinline__ void load(const T* p, int n, bool aligned) {
    if (n >= 8 && aligned) {
      const uint4 a = ldg_cg_u128(p);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    } else {
      uint16_t h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = i < n ? ldg_cg_u16(p + i) : (uint16_t)0;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (uint32_t)h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
    }
  }
  __device__ __forceinline__ uint32_t amax(uint32_t a) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) a = __vmaxu2(a, v[i] & 0x7FFF7FFFu);
    return a;
  }
  static __device__ __forceinline__ uint32_t amax_float(uint32_t a) {
    return __float_as_uint(Elem<T>::unpack(max(a & 0xFFFFu, a >> 16)).x);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = Elem<T>::unpack(v[i]);
      f[2 * i] = a.x;
      f[2 * i + 1] = a.y;
    }
  }
};
template <>
struct Vec8<float> {
  float v[8];
  __device__ __forceinline__ void load(const float* p, int n, bool) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? __uint_as_float(ldg_cg_u32(reinterpret_cast<const uint32_t*>(p + i))) : 0.f;
  }
  __device__ __forceinline__ uint32_t amax(uint32_t a) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return a;
  }
  static __device__ __forceinline__ uint32_t amax_float(uint32_t a) { return a; }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = v[i];
  }
};

// GT threads take one row of up to 64 GT values: the row goes into registers once, the maximum is reduced over the
// group, and the bytes are written 8 at a time. Memory bound: 2 K (4 K for fp32) bytes read and K written per row.
constexpr int kQVecs = 8;
enum Release { kAtEnd, kAfterWait, kAtEntry };   // when a quantization lets the next kernel start

template <typename T, int GT>
__global__ void __launch_bounds__(256)
    quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q, int ldq, float* __restrict__ s,
                         int M, int K, int release) {
  constexpr int kRows = 256 / GT;
  __shared__ uint32_t red[kRows][GT / 32];
  if (release == kAtEntry) pdl_launch_dependents();
  pdl_wait();
  if (release == kAfterWait) pdl_launch_dependents();
  const int g = threadIdx.x / GT, tid = threadIdx.x % GT;
  const int64_t row = (int64_t)blockIdx.x * kRows + g;
  const bool on = row < M;
  const T* xr = x + (on ? row : 0) * ldx;
  const int nv = on ? ldq / 8 : 0;
  const bool aligned = ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)(ldx * sizeof(T))) & 15u) == 0;
  Vec8<T> v[kQVecs];
#pragma unroll
  for (int i = 0; i < kQVecs; ++i) {
    const int j = tid + i * GT;
    if (j < nv) v[i].load(xr + 8 * j, K - 8 * j, aligned);
  }
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < kQVecs; ++i)
    if (tid + i * GT < nv) a = v[i].amax(a);
  a = __reduce_max_sync(0xffffffffu, Vec8<T>::amax_float(a));
  if (GT > 32) {
    if ((tid & 31) == 0) red[g][tid >> 5] = a;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < GT / 32; ++w) a = max(a, red[g][w]);
  }
  const RowScale sc = row_scale(__uint_as_float(a));
  if (on && tid == 0) s[row] = sc.s;
  uint2* dst = reinterpret_cast<uint2*>(q + row * ldq);
#pragma unroll
  for (int i = 0; i < kQVecs; ++i) {
    const int j = tid + i * GT;
    if (j < nv) {
      float f[8];
      v[i].get(f);
      dst[j] = quant8(f, sc);
    }
  }
}

// Longer rows, one CTA each: the row (its first `cap` values, if it is longer than that) is copied into shared memory
// in one piece, so that several rows of an SM are in flight whatever the registers; both passes read it there.
constexpr int kQLongThreads = 512;
constexpr int kQLongBytes = 96 * 1024;

template <typename T>
__global__ void __launch_bounds__(kQLongThreads)
    quantize_long_kernel(const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q, int ldq, float* __restrict__ s,
                         int K, int cap, int release) {
  extern __shared__ __align__(128) uint8_t row_bytes[];
  __shared__ uint64_t bar;
  __shared__ uint32_t red[kQLongThreads / 32];
  if (release == kAtEntry) pdl_launch_dependents();
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  const int nv = ldq / 8, held = min(K, cap) / 8;   // vectors in all, and in shared memory
  const bool aligned = ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)(ldx * sizeof(T))) & 15u) == 0;
  if (tid == 0) {
    mbar_init(&bar, 1);
    mbar_fence_init();
  }
  __syncthreads();
  pdl_wait();
  if (release == kAfterWait) pdl_launch_dependents();
  T* mine = reinterpret_cast<T*>(row_bytes);
  if (aligned) {
    if (tid == 0) {
      mbar_arrive_expect_tx(&bar, (uint32_t)(8 * held * sizeof(T)));
      bulk_copy_g2s(mine, xr, (uint32_t)(8 * held * sizeof(T)), &bar);
    }
    wait_bounded(&bar, 0, &g_w8_status);
  } else {
    for (int i = tid; i < held; i += kQLongThreads) {
      Vec8<T> v;
      v.load(xr + 8 * i, 8, false);
#pragma unroll
      for (int h = 0; h < (int)sizeof(T) / 2; ++h) reinterpret_cast<uint4*>(mine + 8 * i)[h] = reinterpret_cast<const uint4*>(&v.v[0])[h];
    }
    __syncthreads();
  }
  auto fetch = [&](int j, Vec8<T>& v) {
    if (j < held) {
      const uint4* src = reinterpret_cast<const uint4*>(mine + 8 * j);
#pragma unroll
      for (int h = 0; h < (int)sizeof(T) / 2; ++h) reinterpret_cast<uint4*>(&v.v[0])[h] = src[h];
    } else {
      v.load(xr + 8 * j, K - 8 * j, aligned);
    }
  };
  uint32_t a = 0;
  for (int j = tid; j < nv; j += kQLongThreads) {
    Vec8<T> v;
    fetch(j, v);
    a = v.amax(a);
  }
  a = __reduce_max_sync(0xffffffffu, Vec8<T>::amax_float(a));
  if ((tid & 31) == 0) red[tid >> 5] = a;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQLongThreads / 32; ++w) a = max(a, red[w]);
  const RowScale sc = row_scale(__uint_as_float(a));
  if (tid == 0) s[row] = sc.s;
  uint2* dst = reinterpret_cast<uint2*>(q + row * ldq);
  for (int j = tid; j < nv; j += kQLongThreads) {
    Vec8<T> v;
    fetch(j, v);
    float f[8];
    v.get(f);
    dst[j] = quant8(f, sc);
  }
}

// ------------------------------------------------------------------------------------------- the product, many rows
// y[m, n] = s_m t_n sum_k q[m, k] w[n, k] + b_n by tcgen05.mma kind::i8, the channels as the A side (128 rows a CTA) and
// a tile of BN tokens as the N side; the int32 accumulators in tensor memory are exact.
//   * loader warp: one thread copies each 128-byte K chunk of the tile (channels, tokens; 128-byte swizzle, rows and
//     columns past the edge read as zeros) into a stage ring; the first stages' weights before the wait on the previous
//     kernel (the quantization), whose rows follow after it.
//   * MMA warp: one elected lane runs the whole loop, four K = 32 MMAs per chunk; a commit per chunk releases the stage,
//     one per tile hands the accumulator to the epilogue. Two accumulators: the next tile's MMAs run under this tile's
//     epilogue.
//   * 16 epilogue warps, four per 32-lane quarter of tensor memory: a lane holds one channel (its scale and bias in
//     registers), a column one token. 16 tokens x the warp's 32 channels are turned in shared memory, so that a lane
//     stores 16 bytes of an output row (N % 8 == 0; else single values): 18 % off the 509-token product, whose outputs
//     left two bytes a lane before. (Tokens as the A side and a row a lane: 22.3 us instead of 18.0.)
// CTAs are persistent over tiles, tokens innermost, so that the CTAs of one moment share weights in L2.
// PAIR: two CTAs work on one tile of 256 channels (cta_group::2): each loads its 128 channels and half of the tokens, and
// the leader's MMAs read both, so that a chunk costs each SM 16 + BN / 16 KB of loads instead of 16 + BN / 8. The loads
// bound the small products (some 64 bytes a clock and SM arrive from L2), and single CTAs keep the grids that pairs and
// wide tiles would leave short of the SMs.
// With `halves` = 2 a pair's tile is up to 512 tokens wide, in two accumulators that fill the tensor memory: 48 bytes a
// clock and SM instead of 64 for 256 x 256; the epilogue, which then only the next tile's loads run under, is short
// beside a long K. 8192 tokens of 18944 values, 3584 channels: 352 us (3.16 POP/s, 0.96 of twice the measured bf16 peak) and
// 77 for the quantization before it, 431 a call, while a burst lasts; 498 a call once the power cap holds the clock, after
// a tenth of a second. 4096 tokens: the tensor pipe works 88 % of the time. 509 tokens of 1536, 17920 channels: 21.3 us.
// Few tiles and long K: a cluster of S single CTAs splits K, each parks its int32 partial tile in its (then idle) ring
// and all sum their share through distributed shared memory -- exact, so the bits do not depend on S.
constexpr int kChunk = 128;               // bytes of K per stage
constexpr int kWBytes = 128 * kChunk;
constexpr int kEpiWarps = 16;
constexpr int kMmaThreads = (2 + kEpiWarps) * 32;   // loader, MMA, epilogue warps
constexpr int kMaxStages = 8;
constexpr int kW8MaxSplits = 8;           // portable cluster size
constexpr int kW8Smem = 227 * 1024;
constexpr int kBarrierBytes = (2 * kMaxStages + 4) * 8 + 16 + kEpiWarps * 64 * 4 + kEpiWarps * 1024;   // + scales, + staging

// A warp's token scales: an accumulator's columns 16 part + 64 i + j, i < 4, j < 16, of its four-warp part, as 16 i + j. Each
// warp keeps its own, so that no epilogue warp waits for another: one whose bounded wait gave up can leave by itself.
__device__ __forceinline__ int scale_at(int column) { return (column >> 6) * 16 + (column & 15); }

struct W8Gemm {
  const float* s;       // token scales
  const float* t;       // channel scales
  const void* bias;
  void* y;
  int M, N, chunks;     // 128-byte chunks of K
  int bn, halves, tiles_m, tiles, splits, stages;
  int columns;          // tensor memory: 2 accumulators (persistent), or 1 (split)
  int acc_stride;       // columns between the accumulators
  int park;             // byte offset behind the ring: barriers, scales, staging
  bool vec;             // output rows take 16-byte stores
};

// This CTA's share of a cluster's outputs: the int32 partial tiles [token][128 channels] at the same offset of every
// CTA's shared memory, summed, scaled and stored. A thread's four channels are the same in every round; their scales and
// biases are under way while the cluster meets.
template <typename T>
__device__ __forceinline__ void sum_partials(uint32_t red, const float* sc, const float* t, const T* bias, T* y, int n0,
                                             int N, int rows, int rank, int S) {
  const int r4 = (threadIdx.x & 31) * 4;
  float tn[4], bn[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool on = n0 + r4 + j < N;
    tn[j] = on ? t[n0 + r4 + j] : 0.f;
    bn[j] = on && bias ? Elem<T>::to_float(bias[n0 + r4 + j]) : 0.f;
  }
  cluster_sync_all();
  const int warps = blockDim.x >> 5;
  const bool vec = n0 + r4 + 4 <= N && N % 4 == 0 && (reinterpret_cast<uintptr_t>(y) & 7u) == 0;
  for (int m = rank * warps + (threadIdx.x >> 5); m < rows; m += S * warps) {
    const uint32_t off = red + (uint32_t)(m * 128 + r4) * 4u;
    const float scale = sc[(m >> 4 & 3) * 256 + scale_at(m)];   // of the first warp of the column's part
    float4 f[kW8MaxSplits];
#pragma unroll
    for (int q = 0; q < kW8MaxSplits; ++q)
      if (q < S) f[q] = ld_dsmem_f4(mapa_shared(off, (uint32_t)q));
    int v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < kW8MaxSplits; ++q)
      if (q < S) {
        v[0] += __float_as_int(f[q].x);
        v[1] += __float_as_int(f[q].y);
        v[2] += __float_as_int(f[q].z);
        v[3] += __float_as_int(f[q].w);
      }
    float o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = fmaf(__int2float_rn(v[j]) * scale, tn[j], bn[j]);
    T* dst = y + (int64_t)m * N + n0 + r4;
    if (vec) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(Elem<T>::pack(o[0], o[1]), Elem<T>::pack(o[2], o[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + r4 + j < N) dst[j] = Elem<T>::from_float(o[j]);
    }
  }
}

template <typename T, bool PAIR>
__global__ void __launch_bounds__(kMmaThreads, 1)
    w8_gemm_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap qmap, const W8Gemm p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + p.park);   // PAIR: the leader's, for both CTAs' copies
  uint64_t* empty = full + kMaxStages;
  uint64_t* acc_full = empty + kMaxStages;
  uint64_t* acc_empty = acc_full + 2;                            // PAIR: the leader's
  uint32_t* slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  float* sc = reinterpret_cast<float*>(slot + 4);   // [epilogue warps][64] token scales
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int own_bn = PAIR ? p.bn / 2 : p.bn;        // tokens this CTA loads
  const int H = PAIR ? p.halves : 1, acc_bn = p.bn / H, box = own_bn / H;
  const int stage_bytes = kWBytes + own_bn * kChunk, S = PAIR ? 1 : p.splits, St = p.stages;
  const int rank = PAIR || S > 1 ? (int)cluster_rank() : 0;
  const int group = PAIR ? 2 : S;
  const int first = blockIdx.x / group, step = gridDim.x / group;
  const int c0 = PAIR ? 0 : p.chunks * rank / S, nc = PAIR ? p.chunks : p.chunks * (rank + 1) / S - c0;
  constexpr int kTileN = PAIR ? 256 : 128;
  const int n_off = PAIR ? 128 * rank : 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < St; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], PAIR ? 2 * kEpiWarps : kEpiWarps);
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    if (PAIR)
      tc::alloc_pair(slot, p.columns);
    else
      tc::alloc(slot, p.columns);
  }
  tc::fence_before();
  if (PAIR)
    cluster_sync_all();   // the peer's barriers exist before a copy or a commit reaches them
  else
    __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *slot;
  pdl_launch_dependents();

  if (warp == 0) {
    if (tc::elect_one()) {
      tma_prefetch_map(&wmap);
      tma_prefetch_map(&qmap);
      // counters instead of quotients: with the integer divisions of a running index this one thread took some 450
      // clocks a chunk and bounded every shape
      struct Place {
        int tile, c, m0, n0;
      };
      auto at = [&](int tile) {
        const int n = tile / p.tiles_m, m = tile - n * p.tiles_m;
        return Place{tile, 0, m * p.bn + (PAIR ? rank * box : 0), n * kTileN + n_off};
      };
      auto next = [&](Place& q) {
        if (++q.c == nc) q = at(q.tile + step);
      };
      auto weights = [&](const Place& q, int s) {
        uint8_t* dst = ring + s * stage_bytes;
        if (PAIR) {
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * stage_bytes);
          tc::tma_load_2d_pair(dst, &wmap, q.c * kChunk, q.n0, mapa_shared(smem_addr(&full[s]), 0));
        } else {
          mbar_arrive_expect_tx(&full[s], stage_bytes);
          tma_load_2d(dst, &wmap, (c0 + q.c) * kChunk, q.n0, &full[s]);
        }
      };
      auto tokens = [&](const Place& q, int s) {
        uint8_t* dst = ring + s * stage_bytes + kWBytes;
        if (PAIR)
          for (int h = 0; h < H; ++h)
            tc::tma_load_2d_pair(dst + h * box * kChunk, &qmap, q.c * kChunk, q.m0 + h * acc_bn,
                                 mapa_shared(smem_addr(&full[s]), 0));
        else
          tma_load_2d(dst, &qmap, (c0 + q.c) * kChunk, q.m0, &full[s]);
      };
      Place w = at(first), q = w;
      int head = 0;
      for (; head < St && w.tile < p.tiles; ++head, next(w)) weights(w, head);
      pdl_wait();
      for (int s = 0; s < head; ++s, next(q)) tokens(q, s);
      int s = 0, phase = 0;   // the stage to fill next, and the parity of its release
      bool ok = true;
      for (; q.tile < p.tiles; next(q)) {
        ok = wait_bounded(&empty[s], phase, &g_w8_status);
        if (!ok) break;
        weights(q, s);
        tokens(q, s);
        if (++s == St) s = 0, phase ^= 1;
      }
      // no copy in flight past this point (a pair's leader's barriers count its peer's copies too): stage s holds the
      // oldest of the last `head` copies, its parity is that of the release before it
      if (rank == 0 || !PAIR)
        for (int i = 0; i < head; ++i) {
          wait_bounded(&full[s], phase, &g_w8_status);
          if (++s == head) s = 0, phase ^= 1;
        }
    }
    __syncwarp();
  } else if (warp == 1) {
    // one elected lane runs the whole loop (measured, four MMAs with their wait and commit: under `if (lane == 0)` 560
    // clocks, more than the 512 that they take at 256 tokens)
    if ((!PAIR || rank == 0) && tc::elect_one()) {
      // int32 accumulator, signed 8-bit A and B, both K-major
      const uint32_t idesc =
          (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(acc_bn >> 3) << 17) | ((uint32_t)(kTileN >> 4) << 24);
      const uint64_t desc0 = tc::desc_sw128(smem_addr(ring), 16, 1024);   // the address field counts 16 bytes
      const uint32_t half_step = (uint32_t)(box * kChunk) >> 4, stage_step = (uint32_t)stage_bytes >> 4;
      int s = 0, phase = 0, a = 0;   // stage, its parity, accumulators used so far
      bool ok = true;
      for (int tile = first; tile < p.tiles && ok; tile += step, a += H) {
        for (int c = 0; c < nc && ok; ++c) {
          ok = wait_bounded(&full[s], phase, &g_w8_status);
          const uint64_t ad = desc0 + s * stage_step;
          for (int h = 0; h < H && ok; ++h) {
            const int u = a + h;
            if (c == 0 && u >= 2) ok = wait_bounded(&acc_empty[u & 1], ((u >> 1) - 1) & 1, &g_w8_status);
            if (!ok) break;
            tc::fence_after();
            const uint32_t d = tmem + (u & 1) * p.acc_stride;
            const uint64_t bd = ad + (kWBytes >> 4) + h * half_step;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (PAIR)
                tc::mma_i8_ss_pair(d, ad + 2 * k, bd + 2 * k, idesc, c > 0 || k > 0);
              else
                tc::mma_i8_ss(d, ad + 2 * k, bd + 2 * k, idesc, c > 0 || k > 0);
            }
          }
          if (!ok) break;
          if (PAIR)
            tc::commit_pair(&empty[s]);
          else
            tc::commit(&empty[s]);
          if (++s == St) s = 0, phase ^= 1;
        }
        // (after a wait that gave up: what has been issued hands its tile over as it is)
        for (int h = 0; h < H; ++h) {
          if (PAIR)
            tc::commit_pair(&acc_full[(a + h) & 1]);
          else
            tc::commit(&acc_full[(a + h) & 1]);
        }
      }
      // no MMA in flight past this point
      for (int b = max(0, a - 2); b < a; ++b) wait_bounded(&acc_full[b & 1], (b >> 1) & 1, &g_w8_status);
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, part = (warp - 2) >> 2, row = 32 * quarter + lane;
    const uint32_t tlane = (uint32_t)(32 * quarter) << 16;
    const T* bias = static_cast<const T*>(p.bias);
    T* y = static_cast<T*>(p.y);
    float* scale = sc + (warp - 2) * 64;
    uint16_t* turn = reinterpret_cast<uint16_t*>(sc + kEpiWarps * 64) + (warp - 2) * 512;
    pdl_wait();
    bool ok = true;   // of this lane: one that gave up waits no more, but stays with its warp's collective instructions
    const int mine = first < p.tiles ? (p.tiles - first + step - 1) / step : 0;
    for (int a = 0; a < mine * H; ++a) {
      const int tile = first + a / H * step;
      const int m0 = tile % p.tiles_m * p.bn + a % H * acc_bn, n = tile / p.tiles_m * kTileN + n_off + row;
      const bool on = n < p.N;
#pragma unroll
      for (int i = lane; i < 64; i += 32) {
        const int j = 64 * (i >> 4) + 16 * part + (i & 15);
        if (j < acc_bn)
          scale[i] = m0 + j < p.M ? __uint_as_float(ldg_cg_u32(reinterpret_cast<const uint32_t*>(p.s + m0 + j))) : 0.f;
      }
      const float tn = on ? p.t[n] : 0.f, bn = on && bias ? Elem<T>::to_float(bias[n]) : 0.f;
      if (ok) ok = wait_bounded(&acc_full[a & 1], (a >> 1) & 1, &g_w8_status);
      __syncwarp();
      tc::fence_after();
      // 16 columns at a time, the next ones on their way from tensor memory under this block's stores
      const uint32_t acc = tmem + tlane + (uint32_t)((a & 1) * p.acc_stride);
      constexpr int kStep = 4 * kEpiWarps;   // columns between a warp's blocks
      uint32_t v[2][16];
      if (16 * part < acc_bn) tc::ld16(acc + 16 * part, v[0]);
      auto block = [&](int j0, const uint32_t (&w)[16]) {
        if (S == 1) {
          const int left = p.M - m0 - j0;   // tokens
          uint32_t h[8];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            h[j] = Elem<T>::pack(fmaf(__int2float_rn((int)w[2 * j]) * scale[scale_at(j0) + 2 * j], tn, bn),
                                 fmaf(__int2float_rn((int)w[2 * j + 1]) * scale[scale_at(j0) + 2 * j + 1], tn, bn));
          if (p.vec) {
            // through the warp's 1 KB: [16 tokens][32 channels], then eight rows of 64 bytes a store
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              turn[2 * j * 32 + lane] = (uint16_t)h[j];
              turn[(2 * j + 1) * 32 + lane] = (uint16_t)(h[j] >> 16);
            }
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int j = 8 * q + (lane >> 2), c = (lane & 3) * 8;
              const uint4 v = *reinterpret_cast<const uint4*>(turn + j * 32 + c);
              if (j < left && n - lane + c < p.N) *reinterpret_cast<uint4*>(y + (int64_t)(m0 + j0 + j) * p.N + n - lane + c) = v;
            }
            __syncwarp();
          } else if (on) {
            uint16_t* dst = reinterpret_cast<uint16_t*>(y) + (int64_t)(m0 + j0) * p.N + n;
#pragma unroll
            for (int j = 0; j < 16; ++j, dst += p.N)
              if (j < left) *dst = (uint16_t)(h[j >> 1] >> (16 * (j & 1)));
          }
        } else {
          int* red = reinterpret_cast<int*>(ring);   // [token][128 channels]
#pragma unroll
          for (int j = 0; j < 16; ++j) red[(j0 + j) * 128 + row] = (int)w[j];
        }
      };
      for (int j0 = 16 * part; j0 < acc_bn; j0 += 2 * kStep) {
        tc::wait_ld();
        if (j0 + kStep < acc_bn) tc::ld16(acc + j0 + kStep, v[1]);
        block(j0, v[0]);
        if (j0 + kStep < acc_bn) {
          tc::wait_ld();
          if (j0 + 2 * kStep < acc_bn) tc::ld16(acc + j0 + 2 * kStep, v[0]);
          block(j0 + kStep, v[1]);
        }
      }
      tc::fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR)
          tc::arrive_cluster(mapa_shared(smem_addr(&acc_empty[a & 1]), 0));
        else
          mbar_arrive(&acc_empty[a & 1]);
      }
    }
  }
  __syncwarp();
  if (!PAIR && S > 1) {
    const int n0 = first / p.tiles_m * 128, m0 = first % p.tiles_m * p.bn;
    sum_partials<T>(smem_addr(ring), sc, p.t, static_cast<const T*>(p.bias),
                    static_cast<T*>(p.y) + (int64_t)m0 * p.N, n0, p.N, min(p.bn, p.M - m0), rank, S);
  }
  tc::fence_before();
  if (PAIR || S > 1)
    cluster_sync_all();   // no CTA leaves while its partner still reads, or signals, its shared memory
  else
    __syncthreads();
  if (warp == 1) {
    tc::fence_after();
    if (PAIR)
      tc::dealloc_pair(tmem, p.columns);
    else
      tc::dealloc(tmem, p.columns);
  }
}

// ------------------------------------------------------------------------------------------- the product, one to eight rows
// A CTA takes 16 channels and all of K: mma.sync m16n8k32 with the weights' fragments loaded straight into registers,
// 64 bytes of K of a row per four lanes and 16-byte load (the order of k inside a fragment is free as long as both
// operands share it). The first loads -- all there are, up to 64 R NW values of K -- are issued at once, with
// `early` before the wait on the previous kernel; the CTA quantizes the token rows while they are under way. Bound by the weights' way from
// memory; a cluster, tensor memory or a second launch would each add about a microsecond of latency to some four.
// One token, weights in L2: 4608 x 3584 (16.5 MB) 4.7 us, 12544 x 1792 (22.5 MB) 5.4 us; the many-rows product takes
// 8.5 and 9.9 with its quantization.
constexpr int kGemvRows = 8;

struct W8Gemv {
  const void* x;
  int64_t ldx;
  const int8_t* w;
  int64_t ldw;
  const float* t;
  const void* bias;
  void* y;
  int M, N, K, pieces;   // 64-byte pieces of K
  int pitch;             // bytes between the quantized rows: 64 modulo 128, so that two rows' reads do not share banks
};

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// MR: the most rows, 1, 4 or 8. R: 64-byte pieces of K a warp has in flight. An SM holds gemv_per_sm of its CTAs.
constexpr int gemv_per_sm(int NW, int MR, int R) {
  return NW == 16 ? (R == 2 && MR < 8 ? 2 : 1) : (MR == 8 ? 2 : 3) + (R == 2);
}
template <typename T, int NW, int MR, int R>
__global__ void __launch_bounds__(32 * NW, gemv_per_sm(NW, MR, R)) w8_gemv_kernel(const W8Gemv p, bool early) {
  extern __shared__ __align__(16) uint8_t rows[];   // [M][pitch] quantized tokens
  __shared__ int part[NW][128];
  __shared__ uint32_t maxima[kGemvRows];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16;
  pdl_launch_dependents();
  if (!early) pdl_wait();
  // rows past N repeat the last one; pieces past K read as zeros (K is padded to 16, a lane's share of a piece)
  const int8_t* w0 = p.w + (int64_t)min(n0 + g, p.N - 1) * p.ldw + 16 * t;
  const int8_t* w1 = p.w + (int64_t)min(n0 + g + 8, p.N - 1) * p.ldw + 16 * t;
  uint4 a[R][2];
  auto fetch = [&](int i, int c) {
    const bool on = 64 * c + 16 * t < p.K;
    a[i][0] = on ? ldg_stream(reinterpret_cast<const uint4*>(w0 + 64 * c)) : make_uint4(0, 0, 0, 0);
    a[i][1] = on ? ldg_stream(reinterpret_cast<const uint4*>(w1 + 64 * c)) : make_uint4(0, 0, 0, 0);
  };
#pragma unroll
  for (int i = 0; i < R; ++i) fetch(i, warp + i * NW);
  const int out_n = n0 + (tid & 15), out_m = tid >> 4;   // the output this thread sums, of 16 x 8
  const bool out_on = tid < 128 && out_n < p.N && out_m < p.M;
  const float tn = out_on ? p.t[out_n] : 0.f;
  const float bn = out_on && p.bias ? Elem<T>::to_float(static_cast<const T*>(p.bias)[out_n]) : 0.f;
  if (tid < kGemvRows) maxima[tid] = 0u;
  __syncthreads();
  if (early) pdl_wait();
  const bool aligned = ((reinterpret_cast<uintptr_t>(p.x) | (uintptr_t)(p.ldx * sizeof(T))) & 15u) == 0;
  const T* x = static_cast<const T*>(p.x);
  const int nv = p.pieces * 8;   // vectors of 8 values of a row
  Vec8<T> v[MR];
  auto tokens = [&](int j) {
#pragma unroll
    for (int m = 0; m < MR; ++m)
      if (m < p.M && j < nv) v[m].load(x + m * p.ldx + 8 * j, p.K - 8 * j, aligned);
  };
  uint32_t mx[MR] = {};
  for (int j = tid; j < nv; j += 32 * NW) {
    tokens(j);
#pragma unroll
    for (int m = 0; m < MR; ++m)
      if (m < p.M) mx[m] = v[m].amax(mx[m]);
  }
#pragma unroll
  for (int m = 0; m < MR; ++m)
    if (m < p.M) {
      const uint32_t am = __reduce_max_sync(0xffffffffu, Vec8<T>::amax_float(mx[m]));
      if (lane == 0) atomicMax(&maxima[m], am);
    }
  __syncthreads();
  const RowScale mine = row_scale(__uint_as_float(maxima[lane & 7]));
  for (int j0 = 0; j0 < nv; j0 += 32 * NW) {
    const int j = j0 + tid;
    if (nv > 32 * NW) tokens(j);
#pragma unroll
    for (int m = 0; m < MR; ++m)
      if (m < p.M) {
        const RowScale rs{__shfl_sync(0xffffffffu, mine.up, m), __shfl_sync(0xffffffffu, mine.r, m), 0.f};
        if (j < nv) {
          float f[8];
          v[m].get(f);
          *reinterpret_cast<uint2*>(rows + m * p.pitch + 8 * j) = quant8(f, rs);
        }
      }
  }
  __syncthreads();
  int d[4] = {0, 0, 0, 0};
  const uint32_t own = smem_addr(rows) + (uint32_t)(min(g, p.M - 1) * p.pitch + 16 * t);   // unused columns repeat a row
  for (int c0 = warp; c0 < p.pieces; c0 += NW * R) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = c0 + i * NW;
      if (c < p.pieces) {
        const uint4 b = lds128(own + 64 * c);
        mma_s8(d, a[i][0].x, a[i][1].x, a[i][0].y, a[i][1].y, b.x, b.y);
        mma_s8(d, a[i][0].z, a[i][1].z, a[i][0].w, a[i][1].w, b.z, b.w);
        fetch(i, c + NW * R);
      }
    }
  }
  // D[g][2t], D[g][2t + 1], D[g + 8][..]: channel x token
  part[warp][(2 * t) * 16 + g] = d[0];
  part[warp][(2 * t + 1) * 16 + g] = d[1];
  part[warp][(2 * t) * 16 + g + 8] = d[2];
  part[warp][(2 * t + 1) * 16 + g + 8] = d[3];
  __syncthreads();
  if (out_on) {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) sum += part[w][tid];
    static_cast<T*>(p.y)[(int64_t)out_m * p.N + out_n] = Elem<T>::from_float(
        fmaf(__int2float_rn(sum) * row_scale(__uint_as_float(maxima[out_m])).s, tn, bn));
  }
}

// ------------------------------------------------------------------------------------------- the product, a few tens of rows
// The same fragments with rows quantized by a kernel before: a CTA takes 16 CT channels, all of K and up to 8 NT tokens,
// its 16 warps the 64-byte pieces of K in turn; the tokens' fragments come straight from L2 like the weights'. Each warp's
// first R pieces of weights are under way before the wait on the quantization (whose own wait covers what wrote the
// weights). The warps' int32 tiles are summed in shared memory. Latency bound: what it saves is the set-up of the tcgen05
// product's ring, tensor memory and cluster sum. (Tokens of the next piece under way under this one's MMAs: 3584 x 3584
// M = 33 9.9 -> 9.6 us, 8960 x 1536 M = 33 13.7 -> 11.6.)
constexpr int kRowsWarps = 16;

struct W8Rows {
  const int8_t* q;      // [M, kp]
  const float* s;
  const int8_t* w;
  int64_t ldw;
  const float* t;
  const void* bias;
  void* y;
  int M, N, kp, pieces;
};

template <typename T, int CT, int NT>
__global__ void __launch_bounds__(32 * kRowsWarps, 1) w8_rows_kernel(const W8Rows p) {
  constexpr int R = CT * NT >= 10 ? 2 : 4, kCh = 16 * CT, kTok = 8 * NT, kPitch = kCh + 4;
  extern __shared__ __align__(16) int rows_part[];   // [warps][kTok][kPitch]
  static_assert(R % 2 == 0, "the two token buffers alternate from round to round");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kCh;
  pdl_launch_dependents();
  const int8_t* w = p.w + 16 * t;
  int64_t row[CT][2];   // rows past N repeat the last one
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int h = 0; h < 2; ++h) row[c][h] = (int64_t)min(n0 + 16 * c + 8 * h + g, p.N - 1) * p.ldw;
  uint4 a[R][CT][2];
  auto fetch = [&](int i, int piece) {   // shares past K as zeros (K is padded to 16, a lane's share)
    const bool on = 64 * piece + 16 * t < p.kp;
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        a[i][c][h] = on ? ldg_stream(reinterpret_cast<const uint4*>(w + row[c][h] + 64 * piece)) : make_uint4(0, 0, 0, 0);
  };
#pragma unroll
  for (int i = 0; i < R; ++i) fetch(i, warp + i * kRowsWarps);
  int d[CT][NT][4] = {};
  const int8_t* q = p.q + 16 * t;
  int tok[NT];   // token rows past M repeat the last one, their columns are not stored
#pragma unroll
  for (int j = 0; j < NT; ++j) tok[j] = min(8 * j + g, p.M - 1) * p.kp;
  pdl_wait();
  uint4 b[2][NT];
  auto tokens = [&](int k, int piece) {
    const bool on = 64 * piece + 16 * t < p.kp;
#pragma unroll
    for (int j = 0; j < NT; ++j) b[k][j] = on ? ldg_cg_u128(q + tok[j] + 64 * piece) : make_uint4(0, 0, 0, 0);
  };
  tokens(0, warp);
  for (int c0 = warp; c0 < p.pieces; c0 += kRowsWarps * R) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int piece = c0 + i * kRowsWarps;
      if (piece < p.pieces) {
        tokens((i + 1) & 1, piece + kRowsWarps);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            const uint4 x = b[i & 1][j];
            mma_s8(d[c][j], a[i][c][0].x, a[i][c][1].x, a[i][c][0].y, a[i][c][1].y, x.x, x.y);
            mma_s8(d[c][j], a[i][c][0].z, a[i][c][1].z, a[i][c][0].w, a[i][c][1].w, x.z, x.w);
          }
        fetch(i, piece + kRowsWarps * R);
      }
    }
  }
  int* mine = rows_part + warp * kTok * kPitch;
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[(8 * j + 2 * t + (e & 1)) * kPitch + 16 * c + g + (e >> 1) * 8] = d[c][j][e];
  __syncthreads();
  for (int i = tid; i < kTok * kCh; i += 32 * kRowsWarps) {
    const int m = i / kCh, c = i % kCh, n = n0 + c;
    if (m < p.M && n < p.N) {
      int sum = 0;
#pragma unroll
      for (int k = 0; k < kRowsWarps; ++k) sum += rows_part[(k * kTok + m) * kPitch + c];
      static_cast<T*>(p.y)[(int64_t)m * p.N + n] = Elem<T>::from_float(
          fmaf(__int2float_rn(sum) * p.s[m], p.t[n], p.bias ? Elem<T>::to_float(static_cast<const T*>(p.bias)[n]) : 0.f));
    }
  }
}

// ------------------------------------------------------------------------------------------- launches
template <typename Kern, typename... Args>
cudaError_t launch_w8(Kern kern, unsigned grid, int threads, size_t smem, int cluster, bool pdl, cudaStream_t st,
                      Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  if (pdl) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = cluster;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Lets a kernel use that much dynamic shared memory, once per device
template <typename Kern>
cudaError_t allow_smem(Kern kern, std::atomic<uint64_t>& done, int bytes = kW8Smem) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// a warp or 128 threads a row where the registers hold it, else a CTA. With few rows the next kernel, the product, is let
// in early: it may read weights before it waits, so where they may still be in the making only once everything before the
// quantization is complete. With many rows it would take the registers of CTAs still to come (measured at 8192 rows of 18944: the quantization ran at
// half its speed under the product's resident CTAs).
template <typename T>
cudaError_t quantize_t(const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* s, int64_t M, int64_t K,
                       Release few, bool pdl, cudaStream_t st) {
  const int64_t nv = ldq / 8;
  const int release = M <= 296 ? few : kAtEnd;
  const T* xt = static_cast<const T*>(x);
  if (nv <= 128 * kQVecs) {
    const int GT = nv <= 32 * kQVecs && M > 512 ? 32 : 128, rows = 256 / GT;
    return launch_w8(GT == 32 ? quantize_rows_kernel<T, 32> : quantize_rows_kernel<T, 128>,
                     (unsigned)((M + rows - 1) / rows), 256, 0, 1, pdl, st, xt, ldx, q, (int)ldq, s, (int)M, (int)K, release);
  }
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(quantize_long_kernel<T>, done, kQLongBytes + 16);
  if (e != cudaSuccess) return e;
  const int cap = (int)min(K, (int64_t)(kQLongBytes / sizeof(T)));
  return launch_w8(quantize_long_kernel<T>, (unsigned)M, kQLongThreads, (size_t)cap * sizeof(T) + 16, 1, pdl, st, xt, ldx,
                   q, (int)ldq, s, (int)K, cap, release);
}

int64_t padded(int64_t k) { return (k + 15) / 16 * 16; }

bool encode_rows(CUtensorMap* map, const void* base, int64_t width, int64_t ld, int64_t rows, int box_rows) {
  return encode_tensor_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, (uint64_t)width, (uint64_t)rows, (uint64_t)ld, kChunk,
                              (uint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

int tmem_columns(int bn) { return bn <= 32 ? 32 : bn <= 64 ? 64 : bn <= 128 ? 128 : 256; }

// Tokens per tile, pairs or single CTAs, K split and stages: the candidate whose estimated time is least, in clocks per
// CTA. A start and an end (measured 2.5 us of setup, first loads and last stores); per wave and 128-byte chunk the MMAs
// (two clocks a token, but 450 at least, the issue's own time) and the loads at 64 bytes a clock -- both, since at large
// sizes the power cap makes either cost the other's clock; the epilogue that nothing runs under; and a cluster's sum,
// 1.5 us, where the cluster's CTAs can all be resident.
struct W8Plan {
  int bn, halves, splits, stages;
  bool pair;
};

template <typename T>
int resident_clusters(int S) {   // of S single CTAs with the whole shared memory each, on the current device
  static std::atomic<int> known[64][kW8MaxSplits + 1];
  int dev = 0;
  cudaGetDevice(&dev);
  std::atomic<int>& k = known[dev & 63][S];
  int v = k.load(std::memory_order_relaxed);
  if (v == 0) {
    static std::atomic<uint64_t> done{0};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(S);
    cfg.blockDim = dim3(kMmaThreads);
    cfg.dynamicSmemBytes = kW8Smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = S;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (allow_smem(w8_gemm_kernel<T, false>, done) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, w8_gemm_kernel<T, false>, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    v = n + 1;
    k.store(v, std::memory_order_relaxed);
  }
  return v - 1;
}

template <typename T>
W8Plan w8_plan(int64_t M, int64_t N, int chunks, int sms) {
  W8Plan best{0, 1, 1, 0, false};
  int64_t least = INT64_MAX;
  auto consider = [&](int bn, bool pair, int S) {
    const int64_t tiles = (M + bn - 1) / bn * (pair ? (N + 255) / 256 : (N + 127) / 128);
    if (S > 1 && tiles > resident_clusters<T>(S)) return;
    const int64_t ctas = tiles * (pair ? 2 : S), waves = (ctas + sms - 1) / sms;
    const int64_t chunk = max(450, 2 * bn) + (kWBytes + (pair ? bn / 2 : bn) * kChunk) / 64;
    const int64_t c = 4700 + waves * ((chunks + S - 1) / S) * chunk + (bn > 256 ? waves * 20 * bn : 20 * bn) + (S > 1 ? 2800 : 0);
    if (c < least) {
      least = c;
      best.bn = bn, best.pair = pair, best.splits = S, best.halves = bn > 256 ? 2 : 1;
    }
  };
  for (int bn = 512; bn >= 64; bn -= bn > 256 ? 64 : 32) consider(bn, true, 1);
  for (int bn = 256; bn >= 16; bn -= 16) {
    if (bn - 16 >= M) continue;   // wider than the tokens
    for (int S = 1; S <= kW8MaxSplits && (S == 1 || chunks >= 2 * S); ++S) consider(bn, false, S);
  }
  best.stages = min(kMaxStages, (kW8Smem - 1024 - kBarrierBytes) / (kWBytes + (best.pair ? best.bn / 2 : best.bn) * kChunk));
  return best;
}

// One to eight rows, while their values are few: every CTA quantizes all of them. Measured, the GEMV against the two
// launches: 11008 x 2048 M = 4 8.2 / 9.0 us, M = 8 13.5 / 9.0; 2048 x 11008 M = 1 8.0 / 8.9, M = 2 9.6 / 8.9;
// 3584 x 18944 M = 1 25.7 / 15.5; 896 x 896 M = 8 3.7 / 5.5.
bool gemv_takes(int64_t M, int64_t K) { return M <= kGemvRows && M * K <= 12288; }

template <typename T>
cudaError_t gemv_t(const W8Params& p, bool pdl, cudaStream_t st) {
  const int pieces = (int)((p.K + 63) / 64), pitch = (pieces * 64 + 127) / 128 * 128 + 64;
  const W8Gemv g{p.x, p.ldx, static_cast<const int8_t*>(p.w), p.ldw, p.w_scales, p.bias, p.y, (int)p.M, (int)p.N, (int)p.K,
                 pieces, pitch};
  // 8 warps where they hold all of K, on wide layers; else 16. R = 4, or R = 2 where the more CTAs an SM then holds save a
  // round (cold weights, M = 2: 11008 x 2048, two rounds either way, R = 4 7.0 us, R = 2 9.1; 8960 x 1536, two rounds or
  // one, 6.0 and 4.4; M = 1: 4608 x 3584 16 warps 6.1 and 4.4; 11008 x 2048 8 warps 5.7, 16 warps 7.7)
  const int warps = pieces > 32 || p.N < 4096 ? 16 : 8, ctas = (int)((p.N + 15) / 16), sms = sm_count();
  auto rounds = [&](int per) { return (ctas + per * sms - 1) / (per * sms); };
#define LB_GEMV(MR)                                                                                                   \
  (warps == 8 ? (rounds(gemv_per_sm(8, MR, 2)) < rounds(gemv_per_sm(8, MR, 4)) ? w8_gemv_kernel<T, 8, MR, 2>           \
                                                                               : w8_gemv_kernel<T, 8, MR, 4>)          \
              : (rounds(gemv_per_sm(16, MR, 2)) < rounds(gemv_per_sm(16, MR, 4)) ? w8_gemv_kernel<T, 16, MR, 2>        \
                                                                                 : w8_gemv_kernel<T, 16, MR, 4>))
  auto kern = p.M == 1 ? LB_GEMV(1) : p.M <= 4 ? LB_GEMV(4) : LB_GEMV(8);
#undef LB_GEMV
  return launch_w8(kern, (unsigned)ctas, 32 * warps, (size_t)p.M * pitch, 1, pdl, st, g, p.early);
}

// Up to 40 rows on layers of one round of 32-channel CTAs, while K is short enough for latency to count for more than the
// tokens' second way through L2 (cold weights, tcgen05 / this, with the quantization: 3584 x 3584 M = 9 9.1 / 7.1 us,
// M = 40 9.9 / 9.8; 4096 x 4096 M = 24 10.5 / 8.6; 4864 x 896 M = 33 9.0 / 7.8; 8960 x 1536 M = 24 10.9 / 10.1,
// M = 40 11.1 / 11.7; 18944 x 3584 M = 9 17.9 / 23.3).
bool rows_takes(int64_t M, int64_t N, int64_t K, int sms) {
  return M <= 40 && N <= 32 * (int64_t)sms && K <= (M <= 24 ? 10240 : 5120);
}

template <typename T, int CT, int NT>
cudaError_t rows_launch(const W8Rows& r, bool pdl, cudaStream_t st) {
  constexpr size_t smem = (size_t)kRowsWarps * 8 * NT * (16 * CT + 4) * sizeof(int);
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(w8_rows_kernel<T, CT, NT>, done, (int)smem);
  if (e != cudaSuccess) return e;
  return launch_w8(w8_rows_kernel<T, CT, NT>, (unsigned)((r.N + 16 * CT - 1) / (16 * CT)), 32 * kRowsWarps, smem, 1, pdl, st, r);
}

template <typename T>
cudaError_t rows_t(const W8Params& p, const int8_t* q, const float* s, int kp, int sms, bool pdl, cudaStream_t st) {
  const W8Rows r{q, s, static_cast<const int8_t*>(p.w), p.ldw, p.w_scales, p.bias, p.y, (int)p.M, (int)p.N, kp, (kp + 63) / 64};
  if (p.N <= 16 * (int64_t)sms)
    return p.M <= 8    ? rows_launch<T, 1, 1>(r, pdl, st)
           : p.M <= 16 ? rows_launch<T, 1, 2>(r, pdl, st)
           : p.M <= 24 ? rows_launch<T, 1, 3>(r, pdl, st)
                       : rows_launch<T, 1, 5>(r, pdl, st);
  return p.M <= 8    ? rows_launch<T, 2, 1>(r, pdl, st)
         : p.M <= 16 ? rows_launch<T, 2, 2>(r, pdl, st)
         : p.M <= 24 ? rows_launch<T, 2, 3>(r, pdl, st)
                     : rows_launch<T, 2, 5>(r, pdl, st);
}

template <typename T>
cudaError_t linear_t(const W8Params& p, bool pdl, cudaStream_t st) {
  if (gemv_takes(p.M, p.K)) return gemv_t<T>(p, pdl, st);
  const int sms = sm_count();
  const int64_t kp = padded(p.K);
  const int chunks = (int)((kp + kChunk - 1) / kChunk);
  int8_t* q = static_cast<int8_t*>(p.workspace);
  float* s = reinterpret_cast<float*>(q + p.M * kp);
  if (rows_takes(p.M, p.N, p.K, sms)) {
    const cudaError_t e = quantize_t<T>(p.x, p.ldx, q, kp, s, p.M, p.K, p.early ? kAtEntry : kAfterWait, pdl, st);
    return e == cudaSuccess ? rows_t<T>(p, q, s, (int)kp, sms, pdl, st) : e;
  }
  CUtensorMap wmap, qmap;
  if (!encode_rows(&wmap, p.w, kp, p.ldw, p.N, 128)) return cudaErrorInvalidValue;
  cudaError_t e = quantize_t<T>(p.x, p.ldx, q, kp, s, p.M, p.K, p.early ? kAtEntry : kAfterWait, pdl, st);
  if (e != cudaSuccess) return e;
  static thread_local struct {   // the last plan of this host thread, for calls of one shape that follow one another
    int64_t M, N, chunks;
    int sms;
    W8Plan plan;
  } last = {};
  if (last.M != p.M || last.N != p.N || last.chunks != chunks || last.sms != sms)
    last = {p.M, p.N, chunks, sms, w8_plan<T>(p.M, p.N, chunks, sms)};
  const W8Plan plan = last.plan;
  const int own_bn = plan.pair ? plan.bn / 2 : plan.bn, tile_n = plan.pair ? 256 : 128;
  const int tiles_m = (int)((p.M + plan.bn - 1) / plan.bn), tiles = (int)((p.N + tile_n - 1) / tile_n) * tiles_m;
  const int stride = tmem_columns(plan.bn / plan.halves), park = plan.stages * (kWBytes + own_bn * kChunk);
  const W8Gemm g{s, p.w_scales, p.bias, p.y, (int)p.M, (int)p.N, chunks, plan.bn, plan.halves, tiles_m, tiles, plan.splits,
                 plan.stages, plan.splits > 1 ? stride : 2 * stride, stride, park,
                 p.N % 8 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15u) == 0};
  if (!encode_rows(&qmap, q, kp, kp, p.M, own_bn / plan.halves)) return cudaErrorInvalidValue;
  const size_t smem = (size_t)park + kBarrierBytes + 1024;
  if (plan.pair) {
    static std::atomic<uint64_t> done{0};
    if ((e = allow_smem(w8_gemm_kernel<T, true>, done)) != cudaSuccess) return e;
    return launch_w8(w8_gemm_kernel<T, true>, (unsigned)(2 * min(tiles, sms / 2)), kMmaThreads, smem, 2, pdl, st, wmap, qmap, g);
  }
  static std::atomic<uint64_t> done{0};
  if ((e = allow_smem(w8_gemm_kernel<T, false>, done)) != cudaSuccess) return e;
  return launch_w8(w8_gemm_kernel<T, false>, (unsigned)(plan.splits > 1 ? tiles * plan.splits : min(tiles, sms)), kMmaThreads,
                   smem, plan.splits, pdl, st, wmap, qmap, g);
}

}  // namespace

// none where the product quantizes by itself
size_t w8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (gemv_takes(M, K)) return 0;
  const int64_t kp = padded(K);
  return (size_t)M * (size_t)kp + (size_t)M * 4;
}

cudaError_t launch_w8_quantize_rows(const void* x, int dtype, int64_t ldx, int8_t* q, int64_t ldq, float* s, int64_t M,
                                    int64_t K, bool pdl, cudaStream_t st) {
  return dtype == 0   ? quantize_t<__half>(x, ldx, q, ldq, s, M, K, kAtEnd, pdl, st)
         : dtype == 1 ? quantize_t<__nv_bfloat16>(x, ldx, q, ldq, s, M, K, kAtEnd, pdl, st)
                      : quantize_t<float>(x, ldx, q, ldq, s, M, K, kAtEnd, pdl, st);
}

cudaError_t launch_w8_linear(const W8Params& p, bool pdl, cudaStream_t st) {
  return p.dtype == 0 ? linear_t<__half>(p, pdl, st) : linear_t<__nv_bfloat16>(p, pdl, st);
}

int w8_device_error() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_w8_status, sizeof(int));
  return v;
}

void w8_clear_device_error() {
  int z = 0;
  cudaMemcpyToSymbol(g_w8_status, &z, sizeof(int));
}

}  // namespace lb
